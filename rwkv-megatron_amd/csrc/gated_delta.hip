// The gated delta rule for MI355X (gfx950): over sequences in chunks of 64 tokens, forward and
// backward, and over a few tokens as the recurrence itself.
//
// For a head with state S [K, V], log decay g and write strength beta, one token is
//   S' = e^g S      e = v - S'^T k      S = S' + beta k e^T      o = scale S^T q
// and a chunk with G = cumsum(g), L_ij = e^{G_i - G_j}, S the state entering it and C its last token
//   T = (1 + [beta_i L_ij k_i.k_j]_{i>j})^-1       n = T beta (v - e^G (k S))      (the values written)
//   o = scale e^G (q S) + P n,   P = [scale L_ij q_i.k_j]_{i>=j}
//   S_out = e^{G_C} S + k^T (e^{G_C - G} n)
// Backward, from d_o and the gradient D of S_out, the same triangle transposed:
//   d_n = P^T d_o + e^{G_C - G} (k D)     r = T^T d_n      d_v = beta r
//   D_in = e^{G_C} D + q^T (scale e^G d_o) - k^T (e^G d_v)
//   d_q = scale e^G (d_o S^T) + p k,      p = [scale L_ij d_o_i.n_j]_{i>=j}
//   d_k = e^{G_C - G} (n D^T) - e^G (d_v S^T) + p^T q + m k + m^T k,   m = [-L_ij d_v_i.n_j]_{i>j}
//   d_beta_i = r_i.(v - e^G k S)_i - sum_j (r_i.n_j) L_ij k_i.k_j
//   d_G: + where e^{G_i} stands (q's rows, the correction's, p's and m's rows), - where e^{-G_j} does;
//   d_g = the suffix sums of d_G in the chunk.
//
// Kernels: `prep` (G and T, a block a chunk), `fwd` (a walk over the chunks), `bwd` (the walk back,
// for d_v and D), `segment` and `join` (where the walks of long sequences of few heads start in the middle),
// `grads` (the rest, a block a chunk), `step` (a few tokens).
//
// A walk.  Only k S, T (..) and k^T (..) follow one another from chunk to chunk, and their columns are
// independent of each other: a wave keeps 16 columns of S in its accumulators, and since an accumulator's rows are
// what the next product contracts over, it hands every intermediate on in registers (the contraction's order is
// permuted to the accumulators' one, see `GD_POS`) and meets the others only for what they share.  Four such
// waves have a block; four more bring the next chunk in and form P, so that the chain's waves issue nothing else: a walk
// is bound by the instructions of that one wave a SIMD.
//
// Numbers.  q, k, v and d_o are bf16 and enter the products as they are.  Everything computed (S, n, T, P,
// ...) is 32 bits and enters as a sum of three bf16 numbers, nothing of it lost: a product that torch would run in
// 32 bits becomes three of bf16 (bf16 times computed) or six (computed times computed, without the halves that
// lie below 2^-24), 5 and 2.5 times the rate of the matrix instructions in 32 bits, which also keep a wave's other
// instructions from running beside them (33 cycles each and 6 for each of five multiply-adds between two of them
// took 61; independent bf16 ones, of 16 cycles, hide theirs).  What ends in a bf16 output alone is no exception: where a
// write takes the place of what is read, o is the small difference of q S and P n, and d_q and d_k are such differences
// too.  All outputs so have the precision of 32-bit arithmetic, rounded once.
// G is summed in 64 bits and kept as a pair of floats: decays between neighbours late in a chunk are
// differences of large sums.
#include <type_traits>

#include "common.h"
#include "../../include/rwkv6_amd.h"

#define GD_C 64                 // tokens of a chunk
#define GD_PAD 8                // elements behind a row of an LDS tile
#define GD_TS (GD_C + GD_PAD)   // row of a bf16 tile of 64 columns
#define GD_BF 16                // row of a 16 x 16 block in 32 bits: what a wave reads of one is adjacent
#define GD_TB 2560              // T in memory: the ten 16 x 16 blocks of its triangle
#define GD_TP 3584              // a part of T in LDS: 32 rows of 32 columns, 32 of 64
#define GD_TROW(i) ((i) < 32 ? (i) * 40 : 1280 + ((i) - 32) * GD_TS)
#define GD_FLOOR (-1024.f)      // log decays below are this one: e^-1024 is 0 in 32 bits
#define GD_STEP_WAVES 4

namespace {

struct GdTensor {               // [B, heads, T, channels], channels adjacent
    const uint16_t* p;
    int64_t sb, sh, st;
};
struct GdShape {
    int H, HV, T, NC, V;        // key heads, value heads, tokens, chunks, value channels
    int64_t BH;                 // sequences times value heads
    int per, segs;              // the forward's chunks of a segment, segments
};
struct Three {                  // a computed operand: h + m + l, exact
    bf16x8 h, m, l;
};

__device__ __forceinline__ uint4 rest8(float* x, uint4 h) {        // x less what h holds of it, and that as bf16
    float f[8];
    unpack8(h, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] -= f[j];
    return pack8(x);
}
__device__ __forceinline__ Three three(f32x4 a, f32x4 b) {
    float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    const uint4 h = pack8(x), m = rest8(x, h), l = rest8(x, m);
    return {__builtin_bit_cast(bf16x8, h), __builtin_bit_cast(bf16x8, m), __builtin_bit_cast(bf16x8, l)};
}
// four values in parts of bf16, 8 bytes each
__device__ __forceinline__ uint2 rest4(float* x, uint2 h) {
    float f[4];
    unpack4(h, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] -= f[j];
    return make_uint2(pk2(x[0], x[1]), pk2(x[2], x[3]));
}
__device__ __forceinline__ f32x4 mm(bf16x8 a, const Three& b, f32x4 c) {
    return mfma32(a, b.h, mfma32(a, b.m, mfma32(a, b.l, c)));
}
__device__ __forceinline__ f32x4 mm(const Three& a, bf16x8 b, f32x4 c) {
    return mfma32(a.h, b, mfma32(a.m, b, mfma32(a.l, b, c)));
}
__device__ __forceinline__ f32x4 mm(const Three& a, const Three& b, f32x4 c) {
    c = mfma32(a.m, b.m, mfma32(a.h, b.l, mfma32(a.l, b.h, c)));
    return mfma32(a.h, b.h, mfma32(a.h, b.m, mfma32(a.m, b.h, c)));
}

// The walks' contraction order: slot 8q + j of 32 stands for index 16 (j / 4) + 4q + j % 4, so that two accumulator
// tiles, whose lane holds rows 4q .. 4q + 3, are an operand as they are.  q and k lie in LDS with their columns in
// that order: column c at place GD_POS(c) of its row.
#define GD_POS(c) (((c) & ~31) + 8 * (((c) >> 2) & 3) + 4 * (((c) >> 4) & 1) + ((c) & 3))
// Operand of 16 rows of such a tile, contracted over its columns c0 .. c0 + 31.
__device__ __forceinline__ bf16x8 prows(const uint16_t* X, int stride, int r0, int c0, int lane) {
    return ld_bf16x8(X + (r0 + (lane & 15)) * stride + c0 + 8 * (lane >> 4));
}
// Its transposed: 16 columns, contracted over the rows r0 .. r0 + 31 in the walks' order.
__device__ __forceinline__ bf16x8 pcols(const uint16_t* X, int stride, int r0, int c0, int lane) {
    const int L = lane & 15, q = lane >> 4;
    const uint16_t* p = X + (r0 + 4 * q + (L >> 2)) * stride + GD_POS(c0) + 8 * (L & 3);
    return cat_bf16x8(lds_tr16(p), lds_tr16(p + 16 * stride));
}
// The same of a tile in plain order.
__device__ __forceinline__ bf16x8 cols(const uint16_t* X, int stride, int r0, int c0, int lane) {
    const int L = lane & 15, q = lane >> 4;
    const uint16_t* p = X + (r0 + 4 * q + (L >> 2)) * stride + c0 + 4 * (L & 3);
    return cat_bf16x8(lds_tr16(p), lds_tr16(p + 16 * stride));
}
// Rows r0 + 4q .. + 3 of column c0 + lr: a bf16 tile's values as an accumulator tile's lane holds them.
__device__ __forceinline__ f32x4 as_acc(const uint16_t* X, int stride, int r0, int c0, int lane) {
    const int L = lane & 15, q = lane >> 4;
    const uint2 x = __builtin_bit_cast(uint2, lds_tr16(X + (r0 + 4 * q + (L >> 2)) * stride + c0 + 4 * (L & 3)));
    float f[4];
    unpack4(x, f);
    return f32x4{f[0], f[1], f[2], f[3]};
}
__device__ __forceinline__ f32x4 at4(const float* p, int i) { return *reinterpret_cast<const f32x4*>(p + i); }
// A 16 x 16 block times an accumulator tile, in 32 bits.  Step r contracts over rows 4q + r.
__device__ __forceinline__ f32x4 mul_f32(const float* B, const f32x4& x, f32x4 c, int lane) {
    const f32x4 t = at4(B, (lane & 15) * GD_BF + 4 * (lane >> 4));
#pragma unroll
    for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(t[r], x[r], c, 0, 0, 0);
    return c;
}
// T's rows 16 I .. against its columns 32 s .., and T^T's.
__device__ __forceinline__ Three t_rows(const uint16_t* T, int I, int s, int lane) {
    const uint16_t* p = T + GD_TROW(16 * I);
    const int st = I < 2 ? 40 : GD_TS;
    return {prows(p, st, 0, 32 * s, lane), prows(p + GD_TP, st, 0, 32 * s, lane), prows(p + 2 * GD_TP, st, 0, 32 * s, lane)};
}
__device__ __forceinline__ Three t_cols(const uint16_t* T, int I, int s, int lane) {
    const uint16_t* p = T + GD_TROW(32 * s);
    const int st = s ? GD_TS : 40;
    return {pcols(p, st, 0, 16 * I, lane), pcols(p + GD_TP, st, 0, 16 * I, lane), pcols(p + 2 * GD_TP, st, 0, 16 * I, lane)};
}
// tiles I0 .. I1 - 1 of c += a b, both computed, side by side
template <int I0, int I1> __device__ __forceinline__ void mm_tiles(const Three* a, const Three& b, f32x4* c) {
#pragma unroll
    for (int I = I0; I < I1; ++I) c[I] = mfma32(a[I].l, b.h, c[I]);
#pragma unroll
    for (int I = I0; I < I1; ++I) c[I] = mfma32(a[I].h, b.l, c[I]);
#pragma unroll
    for (int I = I0; I < I1; ++I) c[I] = mfma32(a[I].m, b.m, c[I]);
#pragma unroll
    for (int I = I0; I < I1; ++I) c[I] = mfma32(a[I].m, b.h, c[I]);
#pragma unroll
    for (int I = I0; I < I1; ++I) c[I] = mfma32(a[I].h, b.m, c[I]);
#pragma unroll
    for (int I = I0; I < I1; ++I) c[I] = mfma32(a[I].h, b.h, c[I]);
}
__device__ __forceinline__ float gd_gap(float2 a, float2 b) { return (a.x - b.x) + (a.y - b.y); }
__device__ __forceinline__ float gd_beta(const void* p, int dt, int64_t i) {
    return dt == RWKV6_BF16 ? bf2f(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ int gd_block_row(int t) { return t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0; }
// Accumulator tiles in memory: [chunk][16 columns][tile][lane][4].
__device__ __forceinline__ void put_tiles(float* p, f32x4 x, int lane) { *reinterpret_cast<f32x4*>(p + 4 * lane) = x; }

// 16-byte pieces of 256 threads of a [64][COLS] tile.  Rows behind the last token read that one and are made zero on
// their way into LDS: loads under a branch would be waited for where it ends.
template <int COLS> struct TileRegs {
    uint4 q[(COLS + 31) / 32];
};
template <int COLS>
__device__ __forceinline__ TileRegs<COLS> tile_load(const uint16_t* p, int64_t st, int t0, int T, int tid) {
    constexpr int per = COLS / 8, step = 256 / per;            // pieces of a row, rows of a step
    TileRegs<COLS> r;
    const int row = t0 + tid / per;
    const uint16_t* x = p + 8 * (tid % per);
#pragma unroll
    for (int i = 0; i < (COLS + 31) / 32; ++i) r.q[i] = *reinterpret_cast<const uint4*>(x + min(row + step * i, T - 1) * st);
    return r;
}
template <int COLS, bool PERMUTED>
__device__ __forceinline__ void tile_store(const TileRegs<COLS>& r, uint16_t* X, int t0, int T, int tid) {
    constexpr int per = COLS / 8, step = 256 / per;
    const int col = 8 * (tid % per), row = t0 + tid / per;
    uint16_t* p = X + (tid / per) * (COLS + GD_PAD) + (PERMUTED ? GD_POS(col) : col);
    if (COLS < 32 && tid >= GD_C * per) return;
#pragma unroll
    for (int i = 0; i < (COLS + 31) / 32; ++i, p += step * (COLS + GD_PAD)) {
        const uint4 z = make_uint4(0, 0, 0, 0), x = row + step * i < T ? r.q[i] : z;
        if constexpr (PERMUTED) {
            *reinterpret_cast<uint2*>(p) = make_uint2(x.x, x.y);
            *reinterpret_cast<uint2*>(p + 8) = make_uint2(x.z, x.w);
        } else {
            *reinterpret_cast<uint4*>(p) = x;
        }
    }
}

// P of a chunk in N parts, tiles [i][j] with j in the walks' order, by four waves: tile t of the triangle's ten by wave
// t % 4, formed transposed, so that a lane has four adjacent j.  The blocks right of the diagonal are zeroed by
// `gd_zero_p`.
template <int K, int N>
__device__ __forceinline__ void gd_p(const uint16_t* Qt, const uint16_t* Kt, const float2* G, float scale, uint16_t* P, int wave,
                                     int lane) {
    const int lr = lane & 15, q = lane >> 4;
#pragma unroll
    for (int u = 0; u < 3; ++u) {
        const int t = wave + 4 * u;
        if (t >= 10) break;
        const int I = gd_block_row(t), J = t - I * (I + 1) / 2, i = 16 * I + lr, j = 16 * J + 4 * q;
        const float2 gi = G[i];
        const f32x4 g0 = *reinterpret_cast<const f32x4*>(G + j), g1 = *reinterpret_cast<const f32x4*>(G + j + 2);
        f32x4 a = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < K / 32; ++s)
            a = mfma32(prows(Kt, K + GD_PAD, 16 * J, 32 * s, lane), prows(Qt, K + GD_PAD, 16 * I, 32 * s, lane), a);
        const float2 gj[4] = {{g0[0], g0[1]}, {g0[2], g0[3]}, {g1[0], g1[1]}, {g1[2], g1[3]}};
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            x[r] = scale * ex2(gd_gap(gi, gj[r])) * a[r];
            x[r] = i >= j + r ? x[r] : 0.f;
        }
        uint2 part = make_uint2(pk2(x[0], x[1]), pk2(x[2], x[3]));
#pragma unroll
        for (int m = 0; m < N; ++m) {
            *reinterpret_cast<uint2*>(P + m * GD_C * GD_TS + i * GD_TS + GD_POS(j)) = part;
            if (m + 1 < N) part = rest4(x, part);
        }
    }
}
template <int N> __device__ __forceinline__ void gd_zero_p(uint16_t* P, int tid) {
    // blocks (0,1) and (2,3): 2 x 16 rows of four 8-byte pieces a part
#pragma unroll
    for (int m = 0; m < N; ++m)
        if (tid < 128) {
            const int row = (tid >> 2) & 15, b = tid >> 6, j = 32 * b + 16 + 4 * (tid & 3);
            *reinterpret_cast<uint2*>(P + m * GD_C * GD_TS + (32 * b + row) * GD_TS + GD_POS(j)) = make_uint2(0, 0);
        }
}

}  // namespace

// G and T of a chunk.  Wave w forms the rows of its 16-token block of A = beta L k k^T, one wave inverts the blocks
// on the diagonal by substitution, and wave w then forms column w of the blocks below it, in the 32-bit matrix instructions:
// T_IJ = -T_II sum_{J<=l<I} A_Il T_lJ.  Bound by the latency of that chain of products and of the substitution, blocks
// side by side filling it: 16384 chunks 82 to 88 us, 323 MB at 3.8 TB/s (K = 64).  Out: G [chunk][64] as pairs of floats in base-2 units, beta
// in 32 bits, T [chunk][10 blocks][16][16].
template <int K>
__global__ void __launch_bounds__(256, K == 64 ? 8 : 4)
rwkv6_gated_delta_prep_kernel(GdTensor k, const float* __restrict__ g, const void* __restrict__ beta, int beta_dt,
                              float2* __restrict__ G_out, float* __restrict__ b_out, float* __restrict__ T_out, GdShape n) {
    // the blocks of the triangles, row by row: A's ten, whose diagonal T's replaces, and T's six below it.  17 KB of LDS leave
    // room for eight blocks a CU (126 us for 16384 chunks with whole squares, four blocks a CU; 101 with padded rows, six)
    __shared__ __attribute__((aligned(16))) float X[16][16 * GD_BF];
    const auto at_A = [](int I, int J) { return X[I * (I + 1) / 2 + J]; };
    const auto at_T = [](int I, int J) { return I == J ? X[I * (I + 3) / 2] : X[10 + I * (I - 1) / 2 + J]; };
    __shared__ float2 G[GD_C];
    __shared__ float be[GD_C];
    // the waves' shares differ: from block to block they move on by a SIMD
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(((tid >> 6) + blockIdx.x) & 3);
    const int64_t chunk = blockIdx.x, bh = blockIdx.x / (unsigned)n.NC;
    const int c = (int)(blockIdx.x % (unsigned)n.NC), b = (int)bh / n.HV, hv = (int)bh % n.HV, t0 = c * GD_C;
    const uint16_t* kp = k.p + b * k.sb + (hv / (n.HV / n.H)) * k.sh;
    bf16x8 f[4][K / 32];
#pragma unroll
    for (int J = 0; J < 4; ++J)
        if (J <= wave) {
            const int t = t0 + 16 * J + lr;
#pragma unroll
            for (int s = 0; s < K / 32; ++s) {
                uint4 x = *reinterpret_cast<const uint4*>(kp + (int64_t)(t < n.T ? t : n.T - 1) * k.st + 32 * s + 8 * q);
                if (t >= n.T) x = make_uint4(0, 0, 0, 0);
                f[J][s] = __builtin_bit_cast(bf16x8, x);
            }
        }
    if (wave == 0) {
        const int t = t0 + lane;
        const float gr = t < n.T ? g[bh * n.T + t] : 0.f;
        double s = (double)(gr < GD_FLOOR ? GD_FLOOR : gr) * 1.4426950408889634;
        for (int d = 1; d < 64; d <<= 1) {
            const double o = __shfl_up(s, d);
            if (lane >= d) s += o;
        }
        const float hi = (float)s;
        G[lane] = make_float2(hi, (float)(s - hi));
        G_out[chunk * GD_C + lane] = G[lane];
        be[lane] = t < n.T ? gd_beta(beta, beta_dt, bh * n.T + t) : 0.f;
        b_out[chunk * GD_C + lane] = be[lane];
    }
    __syncthreads();
#pragma unroll
    for (int I = 0; I < 4; ++I) {
        if (I != wave) continue;
#pragma unroll
        for (int J = 0; J <= I; ++J) {
            f32x4 a = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < K / 32; ++s) a = mfma32(f[J][s], f[I][s], a);        // transposed: row i = lr
            const int i = 16 * I + lr, j = 16 * J + 4 * q;
            const float2 gi = G[i];
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = i > j + r ? be[i] * ex2(gd_gap(gi, G[j + r])) * a[r] : 0.f;
            *reinterpret_cast<f32x4*>(at_A(I, J) + lr * GD_BF + 4 * q) = x;
        }
    }
    __syncthreads();
    if (wave == 3) {                                       // the four blocks on the diagonal, 16 lanes each
        float x[16];
        float* A = at_A(q, q);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float a[16], s0 = r == lr ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
            for (int s = 0; s < r; s += 4) {
                const f32x4 v = at4(A, r * GD_BF + s);
#pragma unroll
                for (int j = 0; j < 4; ++j) a[s + j] = v[j];
            }
#pragma unroll
            for (int s = 0; s < r; ++s) (s & 1 ? s1 : s0) -= a[s] * x[s];
            x[r] = s0 + s1;
            A[r * GD_BF + lr] = x[r];
        }
    }
    __syncthreads();
#pragma unroll
    for (int J = 0; J < 3; ++J) {
        if (J != wave) continue;
        f32x4 t[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) t[J][r] = at_T(J, J)[(4 * q + r) * GD_BF + lr];
#pragma unroll
        for (int I = J + 1; I < 4; ++I) {
            f32x4 a = {0, 0, 0, 0}, d = {0, 0, 0, 0};
#pragma unroll
            for (int l = J; l < I; ++l) a = mul_f32(at_A(I, l), t[l], a, lane);
            d = mul_f32(at_T(I, I), a, d, lane);
            t[I] = -d;
#pragma unroll
            for (int r = 0; r < 4; ++r) at_T(I, J)[(4 * q + r) * GD_BF + lr] = t[I][r];
        }
    }
    __syncthreads();
    for (int i = tid; i < GD_TB / 4; i += 256) {
        const int t = i >> 6, I = gd_block_row(t);
        *reinterpret_cast<f32x4*>(T_out + chunk * GD_TB + 4 * i) = at4(at_T(I, t - I * (I + 1) / 2), 4 * (i & 63));
    }
}

namespace {
// LDS of the walks: two buffers of q, k, v (or d_o), T, G, e^G, e^{G_C - G}, beta; then P in NP parts.
template <int K, int NW, int NP> struct WalkLds {
    static constexpr int qk = GD_C * (K + GD_PAD), t = GD_C * GD_TS, v = GD_C * (16 * NW + GD_PAD);
    static constexpr int buf = 2 * qk + v + 3 * GD_TP + (8 + 3 * 4) / 2 * GD_C;          // in elements of 2 bytes
    static constexpr size_t bytes = (size_t)(2 * buf + NP * t) * 2;
};
struct WalkBuf {
    uint16_t *Q, *K, *V, *T;
    float2* G;
    float *eG, *eL, *be;
};
template <int K, int NW> __device__ __forceinline__ WalkBuf walk_buf(uint16_t* p) {
    using L = WalkLds<K, NW, 0>;
    WalkBuf b;
    b.Q = p;
    b.K = p + L::qk;
    b.V = p + 2 * L::qk;
    b.T = b.V + L::v;
    b.G = reinterpret_cast<float2*>(b.T + 3 * GD_TP);
    b.eG = reinterpret_cast<float*>(b.G + GD_C);
    b.eL = b.eG + GD_C;
    b.be = b.eL + GD_C;
    return b;
}
// One chunk's inputs on their way from memory to LDS, in 256 threads.
template <int K, int NW> struct WalkRegs {
    TileRegs<K> q, k;
    TileRegs<16 * NW> v;
    f32x4 t[3];
    float2 G, GC;
    float be;
};
struct WalkIn {
    const uint16_t *q, *k, *v;
    int64_t qs, ks, vs;
    const float* T;             // of the head's first chunk
    const float* beta;
    const float2* G;
    int tokens;
};
template <int K, int NW, bool Q>
__device__ __forceinline__ WalkRegs<K, NW> walk_load(const WalkIn& w, int c, int tid) {
    WalkRegs<K, NW> r;
    const int t0 = c * GD_C;
    r.k = tile_load<K>(w.k, w.ks, t0, w.tokens, tid);
    if constexpr (Q) r.q = tile_load<K>(w.q, w.qs, t0, w.tokens, tid);
    r.v = tile_load<16 * NW>(w.v, w.vs, t0, w.tokens, tid);
    const f32x4* T = reinterpret_cast<const f32x4*>(w.T + (int64_t)c * GD_TB);
#pragma unroll
    for (int i = 0; i < 3; ++i) r.t[i] = T[min(tid + 256 * i, GD_TB / 4 - 1)];
    r.G = w.G[t0 + (tid & 63)];
    r.GC = w.G[t0 + GD_C - 1];
    r.be = w.beta[t0 + (tid & 63)];
    return r;
}
template <int K, int NW, bool Q>
__device__ __forceinline__ void walk_store(const WalkRegs<K, NW>& r, const WalkIn& w, int c, const WalkBuf& L, int tid) {
    const int t0 = c * GD_C;
    tile_store<K, true>(r.k, L.K, t0, w.tokens, tid);
    if constexpr (Q) tile_store<K, true>(r.q, L.Q, t0, w.tokens, tid);
    tile_store<16 * NW, false>(r.v, L.V, t0, w.tokens, tid);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        if (i == 2 && tid >= GD_TB / 4 - 512) break;
        const int t = (tid >> 6) + 4 * i, I = gd_block_row(t), J = t - I * (I + 1) / 2;
        uint16_t* p = L.T + GD_TROW(16 * I + ((tid >> 2) & 15)) + GD_POS(16 * J + 4 * (tid & 3));
        float x[4] = {r.t[i][0], r.t[i][1], r.t[i][2], r.t[i][3]};
        uint2 part = make_uint2(pk2(x[0], x[1]), pk2(x[2], x[3]));
#pragma unroll
        for (int m = 0; m < 3; ++m) {
            *reinterpret_cast<uint2*>(p + m * GD_TP) = part;
            if (m < 2) part = rest4(x, part);
        }
    }
    if (tid < GD_C) {
        L.G[tid] = r.G;
        L.eG[tid] = ex2(r.G.x);
        L.eL[tid] = ex2(gd_gap(r.GC, r.G));
        L.be[tid] = r.be;
    }
}
// Which head and 16 NW columns a block walks: blocks of a head's other columns follow a multiple of 8 later where the
// heads are one, on the same XCD, and find its q, k and T in that L2.
struct WalkAt {
    int64_t bh, b;
    int hv, hk, v0, seg, i0;    // i0: the map's first column, or -1
};
template <int NW> __device__ __forceinline__ WalkAt walk_at(const GdShape& n) {
    WalkAt w;
    const unsigned heads = (unsigned)n.BH, bh = blockIdx.x % heads;
    w.bh = bh;
    w.b = bh / (unsigned)n.HV;
    w.hv = (int)(bh % (unsigned)n.HV);
    w.hk = w.hv / (n.HV / n.H);
    const int col = (int)(blockIdx.x / heads), cols = n.V / (16 * NW);
    w.v0 = 16 * NW * (col % cols);
    w.seg = col / cols;
    w.i0 = -1;
    return w;
}
// The same of the blocks that go before: the V columns of the first segment, then the V + K of each other one but the last.
template <int K, int NW> __device__ __forceinline__ WalkAt segment_at(const GdShape& n) {
    WalkAt w = walk_at<NW>(n);
    const int vcols = n.V / (16 * NW), cols = vcols + K / (16 * NW);
    int x = (int)(blockIdx.x / (unsigned)n.BH);
    w.seg = 0;
    if (x >= vcols) {
        x -= vcols;
        w.seg = 1 + x / cols;
        x %= cols;
        if (x >= vcols) {
            w.i0 = 16 * NW * (x - vcols);
            x = 0;
        }
    }
    w.v0 = 16 * NW * x;
    return w;
}
// The inputs of a head from chunk c0 on.
__device__ __forceinline__ WalkIn walk_in(const WalkAt& w, const GdShape& n, int c0, const GdTensor& q, const GdTensor& k,
                                          const GdTensor& v, const float* T, const float* beta, const float2* G) {
    const int64_t at = w.bh * n.NC + c0, t = (int64_t)c0 * GD_C;
    return {q.p + w.b * q.sb + w.hk * q.sh + t * q.st, k.p + w.b * k.sb + w.hk * k.sh + t * k.st,
            v.p + w.b * v.sb + w.hv * v.sh + t * v.st + w.v0, q.st, k.st, v.st, T + at * GD_TB, beta + at * GD_C, G + at * GD_C,
            n.T - c0 * GD_C};
}
// What a segment but the last leaves: its map M [K][K] of the state that enters it, and the state it leaves for an empty
// one (the first: for h0), in tiles; `join` makes that the state which the next one starts from.
template <int K> __device__ __forceinline__ float* seg_map(float* E, const GdShape& n, int64_t bh, int seg) {
    return E + (bh * (n.segs - 1) + seg) * K * (K + n.V);
}
template <int K> __device__ __forceinline__ float* seg_state(float* E, const GdShape& n, int64_t bh, int seg, int ct) {
    return seg_map<K>(E, n, bh, seg) + K * K + ct * (K * 16);
}
template <int K>
__device__ __forceinline__ void put_segment(float* E, const GdShape& n, const WalkAt& w, const f32x4* S, int wave, int lane) {
    if (w.i0 >= 0) {
        float* p = seg_map<K>(E, n, w.bh, w.seg) + w.i0 + 16 * wave + (lane & 15);
#pragma unroll
        for (int d = 0; d < K / 16; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) p[(16 * d + 4 * (lane >> 4) + r) * K] = S[d][r];
    } else {
        float* p = seg_state<K>(E, n, w.bh, w.seg, w.v0 / 16 + wave);
#pragma unroll
        for (int d = 0; d < K / 16; ++d) put_tiles(p + 256 * d, S[d], lane);
    }
}
// A block's waves: NW walk (the first), four help.  Wave w runs on SIMD w % 4, so with fewer walking the helpers are
// placed on the other SIMDs and the waves between, which have nothing to do, end at once.
template <int NW> constexpr int walk_threads = NW == 1 ? 384 : 512;
template <int NW> __device__ __forceinline__ int walk_role(int wave) {       // -1: walks, -2: nothing, else the helper's number
    if (wave < NW) return -1;
    if constexpr (NW == 4) return wave - 4;
    if constexpr (NW == 2) return wave < 4 ? wave - 2 : wave < 6 ? -2 : wave - 4;
    return wave < 4 ? wave - 1 : wave == 4 ? -2 : 3;
}
}  // namespace

namespace {
// What the four helper waves of a walk do: chunk c is in LDS before the first barrier of its step and P of it before
// the second; the loads of the chunk after the next are in flight meanwhile.  NP = 0: no q, no P, no second barrier.
template <int K, int NW, int NP, bool BACK>
__device__ __forceinline__ void walk_help(const WalkIn& in, int NC, float scale, uint16_t* lds, int tid) {
    using M = WalkLds<K, NW, NP>;
    uint16_t* const P = lds + 2 * M::buf;
    const int lane = tid & 63, wave = tid >> 6;
    constexpr bool Q = NP > 0;
    const auto at = [&](int x) { return BACK ? NC - 1 - min(x, NC - 1) : min(x, NC - 1); };
    gd_zero_p<NP>(P, tid);
    if (tid < 128)                                         // the blocks of T right of the diagonal that a step of 32 takes in
#pragma unroll
        for (int m = 0; m < 6; ++m) {
            const int b = tid >> 6;
            uint16_t* T = walk_buf<K, NW>(lds + (m / 3) * M::buf).T + (m % 3) * GD_TP;
            *reinterpret_cast<uint2*>(T + GD_TROW(32 * b + ((tid >> 2) & 15)) + GD_POS(32 * b + 16 + 4 * (tid & 3))) = make_uint2(0, 0);
        }
    if (!NC) return;
    walk_store<K, NW, Q>(walk_load<K, NW, Q>(in, at(0), tid), in, at(0), walk_buf<K, NW>(lds), tid);
    WalkRegs<K, NW> next = walk_load<K, NW, Q>(in, at(1), tid);
    for (int x = 0; x < NC; ++x) {
        const int u = x & 1;
        const WalkBuf L = walk_buf<K, NW>(lds + u * M::buf);
        __syncthreads();
        const WalkRegs<K, NW> later = walk_load<K, NW, Q>(in, at(x + 2), tid);
        if constexpr (Q) {
            gd_p<K, NP>(L.Q, L.K, L.G, scale, P, wave, lane);
            __syncthreads();
        }
        if (x + 1 < NC) walk_store<K, NW, Q>(next, in, at(x + 1), walk_buf<K, NW>(lds + (u ^ 1) * M::buf), tid);
        next = later;
    }
}
// Everything before stays before, for the compiler: it would put each LDS read next to its use, and wait for it there.
__device__ __forceinline__ void gd_issued() { __builtin_amdgcn_sched_barrier(0); }
// x is there from here on: or the compiler computes it where the loop uses it, past the branches of the stores.
__device__ __forceinline__ void gd_here(Three& x) { asm volatile("" : "+v"(x.h), "+v"(x.m), "+v"(x.l)); }
// The order of the instructions since: N matrix instructions with V others after each, so that a wave has both pipes at
// work.
template <int N, int V> __device__ __forceinline__ void gd_weave() {
    if constexpr (N > 0) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, V, 0);
        gd_weave<N - 1, V>();
    }
}
}  // namespace

// A block walks a segment of one head's chunks with 16 NW columns of the state.  SAVE: S_save and n_save get the state
// entering each chunk and the values it writes, for the backward.  Bound by the chain's instructions: at 64 channels 144
// matrix instructions of 16 cycles a chunk and some 500 others of 4, 4300 of the 4600 cycles (1.95 us) of a wave with a
// SIMD to itself: what runs under the matrix instructions, waits for LDS, barriers and products cost again (2.9 us at 128 key
// channels).  With four chain waves a block each shares its SIMD with a helper: 6900 cycles, 3.5 us at the 2.0 GHz that a
// full chip runs at; with S_save and n_save 8150, near the memory's rate: 256 heads of 64 chunks, 64 x 64, 237 to 255 us, 1.25
// GB at 4.9 to 5.3 TB/s.
template <int K, int NW, bool SAVE>
__global__ void __launch_bounds__(walk_threads<NW>) __attribute__((amdgpu_waves_per_eu(2, 2)))
rwkv6_gated_delta_fwd_kernel(GdTensor q, GdTensor k, GdTensor v, const float* __restrict__ beta,
                             const float2* __restrict__ G, const float* __restrict__ T, const float* __restrict__ h0,
                             float* __restrict__ E_in, uint16_t* __restrict__ o, float* __restrict__ hT,
                             float* __restrict__ S_save, float* __restrict__ n_save, GdShape n, float scale) {
    extern __shared__ __attribute__((aligned(16))) uint16_t gd_lds[];
    using M = WalkLds<K, NW, 3>;
    uint16_t* const P = gd_lds + 2 * M::buf;
    constexpr int KS = K + GD_PAD, ND = K / 16, NS = K / 32, PS = GD_C * GD_TS, VS = 16 * NW + GD_PAD;
    const int wave = threadIdx.x >> 6;
    int lane = threadIdx.x & 63, lr = lane & 15, lq = lane >> 4;
    const WalkAt w = walk_at<NW>(n);
    const int role = walk_role<NW>(__builtin_amdgcn_readfirstlane(wave));
    if (role == -2) return;
    const int c0 = w.seg * n.per, c1 = min(n.NC, c0 + n.per);
    if (role >= 0) {
        walk_help<K, NW, 3, false>(walk_in(w, n, c0, q, k, v, T, beta, G), c1 - c0, scale, gd_lds, 64 * role + lane);
        return;
    }
    const int ct = w.v0 / 16 + wave, col = w.v0 + 16 * wave + lr;
    f32x4 S[ND];
    if (w.seg == 0)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[d][r] = h0 ? h0[(w.bh * K + 16 * d + 4 * lq + r) * n.V + col] : 0.f;
    else
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = at4(seg_state<K>(E_in, n, w.bh, w.seg - 1, ct), 256 * d + 4 * lane);
    Three Sp[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) Sp[s] = three(S[2 * s], S[2 * s + 1]);
    uint16_t* po = o + (w.bh * n.T + c0 * GD_C + lr) * n.V + w.v0 + 16 * wave + 4 * lq;
    const f32x4 zero = {0, 0, 0, 0};
    for (int c = c0; c < c1; ++c, po += (int64_t)GD_C * n.V) {
        const WalkBuf L = walk_buf<K, NW>(gd_lds + ((c - c0) & 1) * M::buf);
        const int64_t at = (w.bh * n.NC + c) * (n.V / 16) + ct;
        if constexpr (K == 128) {                          // taken anew: no registers for a lane's addresses over the loop
            asm volatile("" : "+v"(lane));
            lr = lane & 15;
            lq = lane >> 4;
        }
        if constexpr (SAVE)
#pragma unroll
            for (int d = 0; d < ND; ++d) put_tiles(S_save + (at * ND + d) * 256, S[d], lane);
        __syncthreads();
        bf16x8 f[NS][4], k0[ND], k1[ND];
        f32x4 E[4], N[4], O[4], x[4], be[4], eg[4], el[4];
        Three t0[4], t1[4];                                // T's columns 0 .. 31 and 32 .. 63
        float qg[4];
        // reads that 128 key channels leave no registers for yet come later there
        const auto read_t0 = [&] {
#pragma unroll
            for (int I = 0; I < 4; ++I) t0[I] = t_rows(L.T, I, 0, lane);
        };
        const auto read_t1 = [&] {
#pragma unroll
            for (int I = 2; I < 4; ++I) t1[I] = t_rows(L.T, I, 1, lane);
        };
        const auto read_k1 = [&] {
#pragma unroll
            for (int d = 0; d < ND; ++d) k1[d] = pcols(L.K, KS, 32, 16 * d, lane);
        };
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int I = 0; I < 4; ++I) f[s][I] = prows(L.K, KS, 16 * I, 32 * s, lane);
        gd_issued();
#pragma unroll
        for (int I = 0; I < 4; ++I) E[I] = N[I] = O[I] = zero;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            if (s == NS / 2) {                             // what comes next, once half of k's registers are free
#pragma unroll
                for (int I = 0; I < 4; ++I) {
                    x[I] = as_acc(L.V, VS, 16 * I, 16 * wave, lane);
                    be[I] = at4(L.be, 16 * I + 4 * lq);
                    eg[I] = at4(L.eG, 16 * I + 4 * lq);
                }
                if constexpr (K == 64) read_t0();
                gd_issued();
            }
#pragma unroll
            for (int I = 0; I < 4; ++I) E[I] = mfma32(f[s][I], Sp[s].l, E[I]);
#pragma unroll
            for (int I = 0; I < 4; ++I) E[I] = mfma32(f[s][I], Sp[s].m, E[I]);
#pragma unroll
            for (int I = 0; I < 4; ++I) E[I] = mfma32(f[s][I], Sp[s].h, E[I]);
        }
        gd_issued();
        const auto read_q = [&](int s0) {
#pragma unroll
            for (int s = s0; s < s0 + 2; ++s)
#pragma unroll
                for (int I = 0; I < 4; ++I) f[s][I] = prows(L.Q, KS, 16 * I, 32 * s, lane);
        };
        // q S (transposed: a lane has four adjacent channels of a token) beside v - e^G k S and its parts
        const auto q_s = [&](int s0) {
#pragma unroll
            for (int s = s0; s < s0 + 2; ++s) {
#pragma unroll
                for (int I = 0; I < 4; ++I) O[I] = mfma32(Sp[s].l, f[s][I], O[I]);
#pragma unroll
                for (int I = 0; I < 4; ++I) O[I] = mfma32(Sp[s].m, f[s][I], O[I]);
#pragma unroll
                for (int I = 0; I < 4; ++I) O[I] = mfma32(Sp[s].h, f[s][I], O[I]);
            }
        };
        read_q(0);
        gd_issued();
        q_s(0);
#pragma unroll
        for (int I = 0; I < 4; ++I) E[I] = be[I] * (x[I] - eg[I] * E[I]);
        const Three e0 = three(E[0], E[1]);
        gd_weave<24, 4>();
        gd_issued();
        if constexpr (K == 128) {
            read_q(2);
            gd_issued();
            q_s(2);
            gd_issued();
        }
        if constexpr (K == 64) read_t1();
        else read_t0();
#pragma unroll
        for (int I = 0; I < 4; ++I) el[I] = at4(L.eL, 16 * I + 4 * lq);
        const float eC = L.eG[GD_C - 1];
#pragma unroll
        for (int d = 0; d < ND; ++d) k0[d] = pcols(L.K, KS, 0, 16 * d, lane);
        gd_issued();
        // T (..): the first two tiles of n, then the other two beside taking the first ones apart
        mm_tiles<0, 2>(t0, e0, N);
        const Three e1 = three(E[2], E[3]);
        gd_weave<12, 4>();
        gd_issued();
        if constexpr (K == 128) read_t1();
        gd_issued();
        mm_tiles<2, 4>(t0, e0, N);
        const Three w0 = three(N[0] * el[0], N[1] * el[1]);
        gd_weave<12, 5>();
        gd_issued();
        if constexpr (K == 64) read_k1();
#pragma unroll
        for (int I = 0; I < 4; ++I) qg[I] = L.eG[16 * I + lr];
        gd_issued();
        mm_tiles<2, 4>(t1, e1, N);
        const Three n0 = three(N[0], N[1]);
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] *= eC;
        gd_weave<12, 4>();
        __syncthreads();                                   // P
        Three pp[4][2];
        const auto read_p = [&](int s) {
#pragma unroll
            for (int I = 2 * s; I < 4; ++I)
                pp[I][s] = {prows(P, GD_TS, 16 * I, 32 * s, lane), prows(P + PS, GD_TS, 16 * I, 32 * s, lane),
                            prows(P + 2 * PS, GD_TS, 16 * I, 32 * s, lane)};
            gd_issued();
        };
        if constexpr (K == 64) read_p(0);                  // (128: its registers are still taken)
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma32(k0[d], w0.l, S[d]);
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma32(k0[d], w0.m, S[d]);
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma32(k0[d], w0.h, S[d]);
        const Three w1 = three(N[2] * el[2], N[3] * el[3]);
        gd_weave<3 * ND, K == 64 ? 5 : 2>();
        gd_issued();
        if constexpr (K == 128) {
            read_k1();
            gd_issued();
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma32(k1[d], w1.l, S[d]);
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma32(k1[d], w1.m, S[d]);
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma32(k1[d], w1.h, S[d]);
        const Three n1 = three(N[2], N[3]);
#pragma unroll
        for (int I = 0; I < 4; ++I) O[I] *= scale * qg[I];
        gd_weave<3 * ND, K == 64 ? 4 : 2>();
        gd_issued();
        if constexpr (SAVE)
#pragma unroll
            for (int I = 0; I < 4; ++I) put_tiles(n_save + (at * 4 + I) * 256, N[I], lane);
        // beside P n the next chunk's state is taken apart
        const auto p_n = [&](const Three& x, int s) {
#pragma unroll
            for (int I = 2 * s; I < 4; ++I) O[I] = mfma32(x.l, pp[I][s].h, O[I]);
#pragma unroll
            for (int I = 2 * s; I < 4; ++I) O[I] = mfma32(x.h, pp[I][s].l, O[I]);
#pragma unroll
            for (int I = 2 * s; I < 4; ++I) O[I] = mfma32(x.m, pp[I][s].m, O[I]);
#pragma unroll
            for (int I = 2 * s; I < 4; ++I) O[I] = mfma32(x.m, pp[I][s].h, O[I]);
#pragma unroll
            for (int I = 2 * s; I < 4; ++I) O[I] = mfma32(x.h, pp[I][s].m, O[I]);
#pragma unroll
            for (int I = 2 * s; I < 4; ++I) O[I] = mfma32(x.h, pp[I][s].h, O[I]);
        };
        const auto part = [&](int s0) {
#pragma unroll
            for (int s = s0; s < s0 + NS / 2; ++s) {
                Sp[s] = three(S[2 * s], S[2 * s + 1]);
                gd_here(Sp[s]);
            }
        };
        if constexpr (K == 128) read_p(0);
        read_p(1);
        p_n(n0, 0);
        part(0);
        gd_weave<24, K == 64 ? 3 : 5>();
        gd_issued();
        p_n(n1, 1);
        part(NS / 2);
        gd_weave<12, K == 64 ? 5 : 9>();
        gd_issued();
        uint2 ob[4];
#pragma unroll
        for (int I = 0; I < 4; ++I) ob[I] = make_uint2(pk2(O[I][0], O[I][1]), pk2(O[I][2], O[I][3]));
        if ((c + 1) * GD_C <= n.T) {                       // one branch, not four
#pragma unroll
            for (int I = 0; I < 4; ++I) *reinterpret_cast<uint2*>(po + (int64_t)16 * I * n.V) = ob[I];
        } else {
#pragma unroll
            for (int I = 0; I < 4; ++I)
                if (c * GD_C + 16 * I + lr < n.T) *reinterpret_cast<uint2*>(po + (int64_t)16 * I * n.V) = ob[I];
        }
    }
    if (hT && c1 == n.NC)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) hT[(w.bh * K + 16 * d + 4 * lq + r) * n.V + col] = S[d][r];
}

// What a segment does to a state, before the segments' walks: S alone is carried through, without q and o.  The map of
// the state that enters it is one more walk, of K columns that begin as the identity and to which nothing is written.
// 1.4 us a chunk, where the whole walk takes 1.95; 32 heads of 512 chunks in eight segments 237 to 254 us, `join` 9.
template <int K, int NW>
__global__ void __launch_bounds__(walk_threads<NW>) __attribute__((amdgpu_waves_per_eu(2, 2)))
rwkv6_gated_delta_segment_kernel(GdTensor q, GdTensor k, GdTensor v, const float* __restrict__ beta,
                                 const float2* __restrict__ G, const float* __restrict__ T, const float* __restrict__ h0,
                                 float* __restrict__ E_out, GdShape n) {
    extern __shared__ __attribute__((aligned(16))) uint16_t gd_lds[];
    using M = WalkLds<K, NW, 0>;
    constexpr int KS = K + GD_PAD, ND = K / 16, NS = K / 32, VS = 16 * NW + GD_PAD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lq = lane >> 4;
    const WalkAt w = segment_at<K, NW>(n);
    const int role = walk_role<NW>(__builtin_amdgcn_readfirstlane(wave));
    if (role == -2) return;
    const int c0 = w.seg * n.per;
    if (role >= 0) {
        walk_help<K, NW, 0, false>(walk_in(w, n, c0, q, k, v, T, beta, G), n.per, 0.f, gd_lds, 64 * role + lane);
        return;
    }
    const int col = (w.i0 < 0 ? w.v0 : w.i0) + 16 * wave + lr;
    f32x4 S[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 16 * d + 4 * lq + r;
            if (w.i0 >= 0) S[d][r] = row == col ? 1.f : 0.f;
            else S[d][r] = w.seg == 0 && h0 ? h0[(w.bh * K + row) * n.V + col] : 0.f;
        }
    Three Sp[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) Sp[s] = three(S[2 * s], S[2 * s + 1]);
    const f32x4 zero = {0, 0, 0, 0};
    for (int c = 0; c < n.per; ++c) {
        const WalkBuf L = walk_buf<K, NW>(gd_lds + (c & 1) * M::buf);
        __syncthreads();
        bf16x8 f[NS][4], k0[ND], k1[ND];
        f32x4 E[4], N[4], x[4], be[4], eg[4], el[4];
        Three t0[4], t1[4];
        const auto read_t0 = [&] {
#pragma unroll
            for (int I = 0; I < 4; ++I) t0[I] = t_rows(L.T, I, 0, lane);
        };
        const auto read_k1 = [&] {
#pragma unroll
            for (int d = 0; d < ND; ++d) k1[d] = pcols(L.K, KS, 32, 16 * d, lane);
        };
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int I = 0; I < 4; ++I) f[s][I] = prows(L.K, KS, 16 * I, 32 * s, lane);
        gd_issued();
        // half the chunk at a time: e0 beside the other half's products
#pragma unroll
        for (int I = 0; I < 4; ++I) E[I] = N[I] = zero;
        const auto read_s = [&](int I0) {
#pragma unroll
            for (int s = 0; s < NS; ++s) {
#pragma unroll
                for (int I = I0; I < I0 + 2; ++I) E[I] = mfma32(f[s][I], Sp[s].l, E[I]);
#pragma unroll
                for (int I = I0; I < I0 + 2; ++I) E[I] = mfma32(f[s][I], Sp[s].m, E[I]);
#pragma unroll
                for (int I = I0; I < I0 + 2; ++I) E[I] = mfma32(f[s][I], Sp[s].h, E[I]);
            }
        };
        const auto written = [&](int I0) {
#pragma unroll
            for (int I = I0; I < I0 + 2; ++I) E[I] = be[I] * (x[I] - eg[I] * E[I]);
            return three(E[I0], E[I0 + 1]);
        };
        read_s(0);
        gd_issued();
#pragma unroll
        for (int I = 0; I < 4; ++I) {
            be[I] = at4(L.be, 16 * I + 4 * lq);
            eg[I] = at4(L.eG, 16 * I + 4 * lq);
            x[I] = as_acc(L.V, VS, 16 * I, 16 * wave, lane);
            if (w.i0 >= 0) x[I] = zero;
        }
        if constexpr (K == 64) read_t0();
        gd_issued();
        read_s(2);
        const Three e0 = written(0);
        gd_weave<6 * NS, 4>();
        gd_issued();
        if constexpr (K == 128) read_t0();
#pragma unroll
        for (int I = 0; I < 4; ++I) el[I] = at4(L.eL, 16 * I + 4 * lq);
        const float eC = L.eG[GD_C - 1];
#pragma unroll
        for (int d = 0; d < ND; ++d) k0[d] = pcols(L.K, KS, 0, 16 * d, lane);
        gd_issued();
        mm_tiles<0, 2>(t0, e0, N);
        const Three e1 = written(2);
        gd_weave<12, 4>();
        gd_issued();
#pragma unroll
        for (int I = 2; I < 4; ++I) t1[I] = t_rows(L.T, I, 1, lane);
        gd_issued();
        mm_tiles<2, 4>(t0, e0, N);
        const Three w0 = three(N[0] * el[0], N[1] * el[1]);
        gd_weave<12, 4>();
        gd_issued();
        if constexpr (K == 64) read_k1();
        gd_issued();
        mm_tiles<2, 4>(t1, e1, N);
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] *= eC;
        gd_weave<12, K / 32>();
        gd_issued();
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma32(k0[d], w0.l, S[d]);
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma32(k0[d], w0.m, S[d]);
#pragma unroll
        for (int d = 0; d < ND; ++d) S[d] = mfma32(k0[d], w0.h, S[d]);
        const Three w1 = three(N[2] * el[2], N[3] * el[3]);
        gd_weave<3 * ND, K == 64 ? 4 : 2>();
        gd_issued();
        if constexpr (K == 128) read_k1();
        gd_issued();
        // two tiles at a time, taken apart for the next chunk beside the next two
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int d = 2 * s; d < 2 * s + 2; ++d) S[d] = mfma32(k1[d], w1.l, S[d]);
#pragma unroll
            for (int d = 2 * s; d < 2 * s + 2; ++d) S[d] = mfma32(k1[d], w1.m, S[d]);
#pragma unroll
            for (int d = 2 * s; d < 2 * s + 2; ++d) S[d] = mfma32(k1[d], w1.h, S[d]);
            Sp[s] = three(S[2 * s], S[2 * s + 1]);
            gd_here(Sp[s]);
        }
        gd_weave<6, 1>();
        gd_weave<6 * (NS - 1), 6>();
        gd_issued();
    }
    put_segment<K>(E_out, n, w, S, wave, lane);
}

// The states that the segments start from, one after the other: a block has 16 columns, a wave a quarter of the rows;
// S_s+1 = M_s S_s + what segment s left for an empty state, in the 32-bit matrix instructions, the next map on its way
// meanwhile.
template <int K>
__global__ void __launch_bounds__(256) rwkv6_gated_delta_join_kernel(float* __restrict__ E, GdShape n) {
    constexpr int ND = K / 16, NR = ND / 4;
    __shared__ f32x4 S[2][ND][64];
    const int lane = threadIdx.x & 63, d0 = NR * (int)(threadIdx.x >> 6), ct = (int)(blockIdx.x / (unsigned)n.BH);
    const int64_t bh = blockIdx.x % (unsigned)n.BH;
    const auto own = [&](int s, int d) { return seg_state<K>(E, n, bh, s, ct) + 256 * (d0 + d) + 4 * lane; };
    f32x4 m[NR][ND], x[NR];
    const auto load = [&](int s) {
        const float* p = seg_map<K>(E, n, bh, s) + (16 * d0 + (lane & 15)) * K + 4 * (lane >> 4);
#pragma unroll
        for (int d = 0; d < NR; ++d) {
            x[d] = at4(own(s, d), 0);
#pragma unroll
            for (int j = 0; j < ND; ++j) m[d][j] = at4(p, 16 * d * K + 16 * j);
        }
    };
#pragma unroll
    for (int d = 0; d < NR; ++d) S[0][d0 + d][lane] = at4(own(0, d), 0);
    const int last = n.segs - 2;
    load(1);
    for (int s = 1; s <= last; ++s) {
        __syncthreads();
        f32x4 y[NR], a[NR][ND];
#pragma unroll
        for (int d = 0; d < NR; ++d) {
            y[d] = x[d];
#pragma unroll
            for (int j = 0; j < ND; ++j) a[d][j] = m[d][j];
        }
        load(min(s + 1, last));
#pragma unroll
        for (int j = 0; j < ND; ++j) {
            const f32x4 t = S[(s - 1) & 1][j][lane];
#pragma unroll
            for (int d = 0; d < NR; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) y[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[d][j][r], t[r], y[d], 0, 0, 0);
        }
#pragma unroll
        for (int d = 0; d < NR; ++d) *reinterpret_cast<f32x4*>(own(s, d)) = S[s & 1][d0 + d][lane] = y[d];
    }
}

// The walk back: d_v, and for the other gradients r and the gradient D of the state that each chunk leaves.
// BEFORE: what the segments but the first do to D, as in `segment`, the last segment being the first to be walked.
// 256 heads of 64 chunks, 64 x 64: 268 to 289 us, 1.25 GB at 4.3 to 4.7 TB/s; 2.8 us a chunk where heads are few: 126 matrix
// instructions and some 530 others are 64 % of its 6470 cycles, waits for LDS and for P, which the chain wants first, the
// rest (8650 cycles on a full chip).
template <int K, int NW, bool BEFORE>
__global__ void __launch_bounds__(walk_threads<NW>) __attribute__((amdgpu_waves_per_eu(2, 2)))
rwkv6_gated_delta_bwd_kernel(GdTensor q, GdTensor k, GdTensor d_o, const float* __restrict__ beta,
                             const float2* __restrict__ G, const float* __restrict__ T, const float* __restrict__ dhT,
                             float* __restrict__ E, uint16_t* __restrict__ dv, float* __restrict__ dh0, float* __restrict__ D_save,
                             float* __restrict__ r_save, GdShape n, float scale) {
    extern __shared__ __attribute__((aligned(16))) uint16_t gd_lds[];
    using M = WalkLds<K, NW, 3>;
    uint16_t* const P = gd_lds + 2 * M::buf;
    constexpr int KS = K + GD_PAD, ND = K / 16, NS = K / 32, PS = GD_C * GD_TS, VS = 16 * NW + GD_PAD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lq = lane >> 4;
    const WalkAt w = BEFORE ? segment_at<K, NW>(n) : walk_at<NW>(n);       // w.seg: from the back
    const int c0 = (n.segs - 1 - w.seg) * n.per, c1 = min(n.NC, c0 + n.per);
    const int role = walk_role<NW>(__builtin_amdgcn_readfirstlane(wave));
    if (role == -2) return;
    if (role >= 0) {
        walk_help<K, NW, 3, true>(walk_in(w, n, c0, q, k, d_o, T, beta, G), c1 - c0, scale, gd_lds, 64 * role + lane);
        return;
    }
    const int ct = w.v0 / 16 + wave, col = w.v0 + 16 * wave + lr;
    f32x4 D[ND];
    if (!BEFORE && w.seg)
#pragma unroll
        for (int d = 0; d < ND; ++d) D[d] = at4(seg_state<K>(E, n, w.bh, w.seg - 1, ct), 256 * d + 4 * lane);
    else if (BEFORE && w.i0 >= 0)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) D[d][r] = 16 * d + 4 * lq + r == w.i0 + 16 * wave + lr ? 1.f : 0.f;
    else
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) D[d][r] = w.seg == 0 && dhT ? dhT[(w.bh * K + 16 * d + 4 * lq + r) * n.V + col] : 0.f;
    Three Dp[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) Dp[s] = three(D[2 * s], D[2 * s + 1]);
    const f32x4 zero = {0, 0, 0, 0};
    for (int c = c1 - 1, u = 0; c >= c0; --c, u ^= 1) {
        const WalkBuf L = walk_buf<K, NW>(gd_lds + u * M::buf);
        const int64_t at = (w.bh * n.NC + c) * (n.V / 16) + ct;
        if constexpr (!BEFORE)
#pragma unroll
            for (int d = 0; d < ND; ++d) put_tiles(D_save + (at * ND + d) * 256, D[d], lane);
        __syncthreads();
        bf16x8 f[NS][4], fc[2][ND], dof[2];
        f32x4 X[4], Y[4], R[4], V[4], el[4], eg[4], be[4]; // X: d_n; Y: scale e^G d_o; V: d_v
        Three t0[4], t1[4], pp[4][2];                      // T^T's columns 0 .. 31 and 32 .. 63; P^T's
#pragma unroll
        for (int I = 0; I < 4; ++I) {
            Y[I] = as_acc(L.V, VS, 16 * I, 16 * wave, lane);
            if (BEFORE && w.i0 >= 0) Y[I] = zero;
            eg[I] = at4(L.eG, 16 * I + 4 * lq);
        }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int I = 0; I < 4; ++I) f[s][I] = prows(L.K, KS, 16 * I, 32 * s, lane);
#pragma unroll
        for (int I = 0; I < 4; ++I) el[I] = at4(L.eL, 16 * I + 4 * lq);
        const float eC = L.eG[GD_C - 1];
        gd_issued();
        // k D beside scale e^G d_o and its parts
#pragma unroll
        for (int I = 0; I < 4; ++I) X[I] = R[I] = zero;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int I = 0; I < 4; ++I) X[I] = mfma32(f[s][I], Dp[s].l, X[I]);
#pragma unroll
            for (int I = 0; I < 4; ++I) X[I] = mfma32(f[s][I], Dp[s].m, X[I]);
#pragma unroll
            for (int I = 0; I < 4; ++I) X[I] = mfma32(f[s][I], Dp[s].h, X[I]);
        }
#pragma unroll
        for (int I = 0; I < 4; ++I) Y[I] *= scale * eg[I];
        const Three Yp[2] = {three(Y[0], Y[1]), three(Y[2], Y[3])};
#pragma unroll
        for (int d = 0; d < ND; ++d) D[d] *= eC;
        gd_weave<12 * NS, K == 64 ? 6 : 3>();
        gd_issued();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            dof[s] = cols(L.V, VS, 32 * s, 16 * wave, lane);
            if (BEFORE && w.i0 >= 0) dof[s] = bf16x8{};
        }
        __syncthreads();                                   // P
#pragma unroll
        for (int s = 1; s >= 0; --s)
#pragma unroll
            for (int I = 2 * s + 1; I >= 0; --I)
                pp[I][s] = {pcols(P, GD_TS, 32 * s, 16 * I, lane), pcols(P + PS, GD_TS, 32 * s, 16 * I, lane),
                            pcols(P + 2 * PS, GD_TS, 32 * s, 16 * I, lane)};
        // reads that 128 key channels leave no registers for yet come later there
        const auto read_q = [&](int s) {
#pragma unroll
            for (int d = 0; d < ND; ++d) fc[s][d] = pcols(L.Q, KS, 32 * s, 16 * d, lane);
        };
        if constexpr (K == 64) read_q(0);
        gd_issued();
#pragma unroll
        for (int I = 0; I < 4; ++I) X[I] *= el[I];
        const auto p_do = [&](int I, int s) {
            X[I] = mfma32(pp[I][s].l, dof[s], X[I]);
            X[I] = mfma32(pp[I][s].m, dof[s], X[I]);
            X[I] = mfma32(pp[I][s].h, dof[s], X[I]);
        };
        p_do(3, 1), p_do(2, 1);
        gd_issued();
        read_q(K == 64 ? 1 : 0);
        gd_issued();
        // the other tiles of P^T d_o, and q^T (..), beside the parts of d_n
        p_do(1, 1), p_do(0, 1), p_do(1, 0), p_do(0, 0);
        const Three x1 = three(X[2], X[3]);
        gd_weave<12, 4>();
        gd_issued();
        const auto read_t1 = [&] {
#pragma unroll
            for (int I = 0; I < 4; ++I) t1[I] = t_cols(L.T, I, 1, lane);
#pragma unroll
            for (int I = 0; I < 4; ++I) be[I] = at4(L.be, 16 * I + 4 * lq);
        };
        if constexpr (K == 64) read_t1();
        else read_q(1);
        gd_issued();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int d = 0; d < ND; ++d) D[d] = mfma32(fc[s][d], Yp[s].l, D[d]);
#pragma unroll
            for (int d = 0; d < ND; ++d) D[d] = mfma32(fc[s][d], Yp[s].m, D[d]);
#pragma unroll
            for (int d = 0; d < ND; ++d) D[d] = mfma32(fc[s][d], Yp[s].h, D[d]);
        }
        const Three x0 = three(X[0], X[1]);
        gd_weave<6 * ND, K == 64 ? 2 : 1>();
        gd_issued();
        if constexpr (K == 128) read_t1();
#pragma unroll
        for (int I = 0; I < 2; ++I) t0[I] = t_cols(L.T, I, 0, lane);
#pragma unroll
        for (int d = 0; d < ND; ++d) fc[0][d] = pcols(L.K, KS, 32, 16 * d, lane);
        gd_issued();
        mm_tiles<2, 4>(t1, x1, R);
        gd_issued();
        mm_tiles<0, 2>(t1, x1, R);
#pragma unroll
        for (int I = 2; I < 4; ++I) {
            V[I] = be[I] * R[I];
            X[I] = -eg[I] * V[I];
        }
        const Three r1 = three(X[2], X[3]);
        gd_weave<12, 5>();
        gd_issued();
#pragma unroll
        for (int d = 0; d < ND; ++d) fc[1][d] = pcols(L.K, KS, 0, 16 * d, lane);
        gd_issued();
        mm_tiles<0, 2>(t0, x0, R);
        gd_issued();
#pragma unroll
        for (int d = 0; d < ND; ++d) D[d] = mfma32(fc[0][d], r1.l, D[d]);
#pragma unroll
        for (int d = 0; d < ND; ++d) D[d] = mfma32(fc[0][d], r1.m, D[d]);
#pragma unroll
        for (int d = 0; d < ND; ++d) D[d] = mfma32(fc[0][d], r1.h, D[d]);
#pragma unroll
        for (int I = 0; I < 2; ++I) {
            V[I] = be[I] * R[I];
            X[I] = -eg[I] * V[I];
        }
        const Three r0 = three(X[0], X[1]);
        gd_weave<3 * ND, K == 64 ? 5 : 3>();
        gd_issued();
        // two tiles at a time, taken apart for the next chunk beside the next two
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
            for (int d = 2 * s; d < 2 * s + 2; ++d) D[d] = mfma32(fc[1][d], r0.l, D[d]);
#pragma unroll
            for (int d = 2 * s; d < 2 * s + 2; ++d) D[d] = mfma32(fc[1][d], r0.m, D[d]);
#pragma unroll
            for (int d = 2 * s; d < 2 * s + 2; ++d) D[d] = mfma32(fc[1][d], r0.h, D[d]);
            Dp[s] = three(D[2 * s], D[2 * s + 1]);
            gd_here(Dp[s]);
        }
        gd_weave<6, 1>();
        gd_weave<6 * (NS - 1), 6>();
        gd_issued();
        if constexpr (BEFORE) continue;
#pragma unroll
        for (int I = 0; I < 4; ++I) put_tiles(r_save + (at * 4 + I) * 256, R[I], lane);
        uint16_t* pv = dv + (w.bh * n.T + c * GD_C + 4 * lq) * n.V + col;
        if ((c + 1) * GD_C <= n.T) {
#pragma unroll
            for (int I = 0; I < 4; ++I)
#pragma unroll
                for (int r = 0; r < 4; ++r) pv[(16 * I + r) * n.V] = f2bf(V[I][r]);
        } else {
#pragma unroll
            for (int I = 0; I < 4; ++I)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (c * GD_C + 16 * I + 4 * lq + r < n.T) pv[(16 * I + r) * n.V] = f2bf(V[I][r]);
        }
    }
    if constexpr (BEFORE) put_segment<K>(E, n, w, D, wave, lane);
    else if (dh0 && c0 == 0)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) dh0[(w.bh * K + 16 * d + 4 * lq + r) * n.V + col] = D[d][r];
}

namespace {
// LDS of the gradients: q and k; 32 value channels of n, r [32][64 tokens] and S, D [32][K] in three parts, in
// whose place p and m [64][64] in three parts come afterwards; sums.
template <int K> struct GradLds {
    static constexpr int qk = GD_C * (K + GD_PAD), nv = 32 * GD_TS, sv = 32 * (K + GD_PAD), pm = GD_C * GD_TS;
    static constexpr int shared_ = 6 * nv + 6 * sv > 6 * pm ? 6 * nv + 6 * sv : 6 * pm;
    static constexpr int sums = 3 + 4 + 2 * 3 + 1;         // of 64: e^G, e^{G_C - G}, beta; columns; rows' three by half; rest
    static constexpr size_t bytes = (size_t)(2 * qk + shared_) * 2 + GD_C * 8 + sums * GD_C * 4;
};
// Two 16-column tiles of 16 TILES rows in 512 threads, and into three parts [32 columns][16 TILES].
template <int TILES>
__device__ __forceinline__ void tiles_load(const float* base, int64_t at, int tid, f32x4* x) {
#pragma unroll
    for (int i = 0; i < TILES / 4; ++i) x[i] = reinterpret_cast<const f32x4*>(base)[at * (64 * TILES) + tid + 512 * i];
}
template <int TILES>
__device__ __forceinline__ void tiles_store(const f32x4* v, uint16_t* X, int tid) {
    constexpr int stride = 16 * TILES + GD_PAD;
#pragma unroll
    for (int i = 0; i < TILES / 4; ++i) {
        const int m = tid + 512 * i, lane = m & 63, d = (m >> 6) % TILES, tile = (m >> 6) / TILES;
        uint16_t* p = X + (16 * tile + (lane & 15)) * stride + 16 * d + 4 * (lane >> 4);
        float x[4] = {v[i][0], v[i][1], v[i][2], v[i][3]};
        uint2 part = make_uint2(pk2(x[0], x[1]), pk2(x[2], x[3]));
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            *reinterpret_cast<uint2*>(p + j * 32 * stride) = part;
            if (j < 2) part = rest4(x, part);
        }
    }
}
// Operand of 16 columns c0 .. of such a tile, contracted over the 32 value channels.
__device__ __forceinline__ Three tr3(const uint16_t* X, int stride, int c0, int lane) {
    return {lds_tr8(X, stride, 0, c0, lane), lds_tr8(X + 32 * stride, stride, 0, c0, lane),
            lds_tr8(X + 64 * stride, stride, 0, c0, lane)};
}
__device__ __forceinline__ float sum16(float v) {          // over the 16 lanes of a row
    v = sum8lanes(v);
    return v + dpp_mov<0x140>(v);
}
__device__ __forceinline__ float sum_rows(float v) {       // over the four rows of 16 lanes
    const RowSums r = row_sums(v);
    return r.lo + r.hi;
}
__device__ __forceinline__ bf16x8 plain_rows(const uint16_t* X, int stride, int r0, int c0, int lane) {
    return ld_bf16x8(X + (r0 + (lane & 15)) * stride + c0 + 8 * (lane >> 4));
}
}  // namespace

// d_q, d_k, d_g and d_beta of a chunk of a key head, its value heads one after the other.  Wave (I, half) has the
// tokens 16 I .. 16 I + 15 against half of the key channels, and of the columns of p and m those of its parity; every
// product is formed transposed, so that a lane has one token and four adjacent channels.  Bound by its other
// instructions (50 % of the cycles: parts of S, D, n, r), LDS (55 %, 25 in bank conflicts), matrix instructions (28 %) and the
// waits between barriers of two blocks a CU: 16384 chunks of 64 x 64 473 to 503 us, 1.90 GB at 3.8 to 4.0 TB/s.  At 128 key
// channels one block a CU leaves each of them below 40 %.  Two value heads a key head and more hold d_q and d_k over
// them, which takes more registers (GROUPED).
template <int K, bool GROUPED>
__global__ void __launch_bounds__(512, K == 64 && !GROUPED ? 4 : 2)
rwkv6_gated_delta_grads_kernel(GdTensor q, GdTensor k, GdTensor v, GdTensor d_o, const float* __restrict__ beta, int beta_dt,
                               const float2* __restrict__ G_in, const float* __restrict__ S_save,
                               const float* __restrict__ n_save, const float* __restrict__ D_save,
                               const float* __restrict__ r_save, uint16_t* __restrict__ dq, uint16_t* __restrict__ dk,
                               float* __restrict__ dg, void* __restrict__ dbeta, GdShape n, float scale) {
    extern __shared__ __attribute__((aligned(16))) uint16_t gd_lds[];
    using M = GradLds<K>;
    constexpr int KS = K + GD_PAD, ND = K / 32, NS = K / 32;              // ND: a half's channel tiles
    uint16_t *Qt = gd_lds, *Kt = Qt + M::qk, *X = Kt + M::qk;
    uint16_t *Nt = X, *Rt = Nt + 3 * M::nv, *St = Rt + 3 * M::nv, *Dt = St + 3 * M::sv;
    uint16_t *pt = X, *mt = pt + 3 * M::pm;
    float2* G = reinterpret_cast<float2*>(X + M::shared_);
    float *eG = reinterpret_cast<float*>(G + GD_C), *eL = eG + GD_C, *be = eL + GD_C, *colsum = be + GD_C;
    float *own_ = colsum + 4 * GD_C, *kept_ = own_ + 2 * GD_C, *db_ = kept_ + 2 * GD_C, *part = db_ + 2 * GD_C;
    // lane and tid are taken anew from an opaque copy where a phase begins: hoisted out of the loops, the addresses
    // of all of them at once would not fit the registers
    int tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lq = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), I = wave & 3, half = wave >> 2;
    const auto put_parts = [](uint16_t* to, float* x) {
        uint2 part = make_uint2(pk2(x[0], x[1]), pk2(x[2], x[3]));
#pragma unroll
        for (int l = 0; l < 3; ++l) {
            *reinterpret_cast<uint2*>(to + l * M::pm) = part;
            if (l < 2) part = rest4(x, part);
        }
    };
    const auto anew = [&] {
        int x = threadIdx.x;
        asm volatile("" : "+v"(x));
        tid = x;
        lane = x & 63;
        lr = x & 15;
        lq = lane >> 4;
    };
    const int group = GROUPED ? n.HV / n.H : 1;
    const int bk = (int)(blockIdx.x / (unsigned)n.NC), c = (int)(blockIdx.x % (unsigned)n.NC), hk = bk % n.H, t0 = c * GD_C;
    const int64_t b = bk / n.H, head = bk;
    const auto tile = half ? tile_load<K>(q.p + b * q.sb + hk * q.sh, q.st, t0, n.T, tid - 256)
                           : tile_load<K>(k.p + b * k.sb + hk * k.sh, k.st, t0, n.T, tid);
    const int d0 = ND * half;
    f32x4 aq[ND], ak[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) aq[d] = ak[d] = f32x4{0, 0, 0, 0};
    for (int e = 0; e < group; ++e) {
        const int hv = hk * group + e;
        const int64_t bh = b * n.HV + hv, chunk = bh * n.NC + c;
        const uint16_t *vp = v.p + b * v.sb + hv * v.sh, *op = d_o.p + b * d_o.sb + hv * d_o.sh;
        anew();
        if (tid < GD_C) {
            const float2 g = G_in[chunk * GD_C + tid], gC = G_in[chunk * GD_C + GD_C - 1];
            G[tid] = g;
            eG[tid] = ex2(g.x);
            eL[tid] = ex2(gd_gap(gC, g));
            be[tid] = beta[chunk * GD_C + tid];
        }
        f32x4 P[2], R[2], Z[ND], Y[ND], W[ND], RV = {0, 0, 0, 0};
        float sd = 0.f;
        P[0] = P[1] = R[0] = R[1] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < ND; ++d) Z[d] = Y[d] = W[d] = f32x4{0, 0, 0, 0};
        f32x4 xn[1], xr[1], xs[K / 64], xd[K / 64];
        uint4 ov, vv;
        const auto load = [&](int vb) {
            const int64_t at = chunk * (n.V / 16) + 2 * vb;
            tiles_load<4>(n_save, at, tid, xn);
            tiles_load<4>(r_save, at, tid, xr);
            tiles_load<K / 16>(S_save, at, tid, xs);
            tiles_load<K / 16>(D_save, at, tid, xd);
            const int row = min(t0 + 16 * I + lr, n.T - 1);
            ov = *reinterpret_cast<const uint4*>(op + row * d_o.st + 32 * vb + 8 * lq);
            vv = *reinterpret_cast<const uint4*>(vp + row * v.st + 32 * vb + 8 * lq);
        };
        load(0);
        if (e == 0) tile_store<K, false>(tile, half ? Qt : Kt, t0, n.T, tid & 255);
        const int blocks = n.V / 32;
        for (int vb = 0; vb < blocks; ++vb) {
#pragma unroll
            for (int j = 0; j < K / 64; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) sd += xs[j][r] * xd[j][r];
            const bool live = t0 + 16 * I + lr < n.T;
            const uint4 none = make_uint4(0, 0, 0, 0);
            const bf16x8 fo = __builtin_bit_cast(bf16x8, live ? ov : none), fv = __builtin_bit_cast(bf16x8, live ? vv : none);
            __syncthreads();                               // the last block's operands, or p and m, are done with
            tiles_store<4>(xn, Nt, tid);
            tiles_store<4>(xr, Rt, tid);
            tiles_store<K / 16>(xs, St, tid);
            tiles_store<K / 16>(xd, Dt, tid);
            __syncthreads();
            load(min(vb + 1, blocks - 1));                 // the next block's, under this one's products
            {
                const Three fr = tr3(Rt, GD_TS, 16 * I, lane);
                if (half) RV = mm(fr, fv, RV);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int J = 2 * u + half;
                    if (J > I) continue;
                    const Three nj = tr3(Nt, GD_TS, 16 * J, lane);
                    P[u] = mm(nj, fo, P[u]);
                    R[u] = mm(nj, fr, R[u]);
                }
                gd_issued();
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const Three sp = tr3(St, KS, 16 * (d0 + d), lane);
                    Z[d] = mm(sp, fo, Z[d]);
                    Y[d] = mm(sp, fr, Y[d]);
                    gd_issued();
                }
            }
            const Three fn = tr3(Nt, GD_TS, 16 * I, lane);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                W[d] = mm(tr3(Dt, KS, 16 * (d0 + d), lane), fn, W[d]);
                gd_issued();
            }
        }
        sd = wave_sum(sd);
        anew();
        if (lane == 0) part[wave] = sd;
        __syncthreads();                                   // p and m take the operands' place
        const int i = 16 * I + lr;                         // this lane's token
        float own = 0.f, kept = 0.f, db = 0.f;
        const float gi = eG[i], bi = be[i], li = eL[i];
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            float qv[4], kv[4];
            unpack4(*reinterpret_cast<const uint2*>(Qt + i * KS + 16 * (d0 + d) + 4 * lq), qv);
            unpack4(*reinterpret_cast<const uint2*>(Kt + i * KS + 16 * (d0 + d) + 4 * lq), kv);
            Z[d] *= scale * gi;
            Y[d] *= gi;
            W[d] *= li;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float yk = Y[d][r] * kv[r];
                db -= yk;
                own += Z[d][r] * qv[r] - bi * yk;
                kept += W[d][r] * kv[r];
            }
            aq[d] += Z[d];
            ak[d] += W[d] - bi * Y[d];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int J = 2 * u + half, j = 16 * J + 4 * lq;
            float cs[4] = {0, 0, 0, 0}, p[4] = {0, 0, 0, 0}, m[4] = {0, 0, 0, 0};
            if (J <= I) {
                f32x4 qk = {0, 0, 0, 0}, kk = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const bf16x8 kj = plain_rows(Kt, KS, 16 * J, 32 * s, lane);
                    qk = mfma32(kj, plain_rows(Qt, KS, 16 * I, 32 * s, lane), qk);
                    kk = mfma32(kj, plain_rows(Kt, KS, 16 * I, 32 * s, lane), kk);
                }
                const float2 g = G[i];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float l = ex2(gd_gap(g, G[j + r])), w = i > j + r ? -l * R[u][r] : 0.f;
                    p[r] = i >= j + r ? scale * l * P[u][r] : 0.f;
                    m[r] = bi * w;
                    // without the diagonal, which no decay enters: its share of row and column would only round
                    cs[r] = i > j + r ? p[r] * qk[r] + m[r] * kk[r] : 0.f;
                    own += cs[r];
                    db += w * kk[r];
                }
            }
            put_parts(pt + i * GD_TS + j, p);
            put_parts(mt + i * GD_TS + j, m);
#pragma unroll
            for (int r = 0; r < 4; ++r) cs[r] = sum16(cs[r]);
            if (lr == 0) *reinterpret_cast<float4*>(colsum + I * GD_C + j) = make_float4(cs[0], cs[1], cs[2], cs[3]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (half && lr == 4 * lq + r) db += RV[r];     // the diagonal of r v^T
        own = sum_rows(own);
        kept = sum_rows(kept);
        db = sum_rows(db);
        if (lq == 0) {
            own_[half * GD_C + i] = own;
            kept_[half * GD_C + i] = kept;
            db_[half * GD_C + i] = db;
        }
        __syncthreads();
        anew();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            // own rows: columns up to the diagonal; transposed: rows from it
            const bool left = 2 * s <= I, right = 2 * s + 1 >= I;
            const auto rows = [&](const uint16_t* x) {
                return Three{plain_rows(x, GD_TS, 16 * I, 32 * s, lane), plain_rows(x + M::pm, GD_TS, 16 * I, 32 * s, lane),
                             plain_rows(x + 2 * M::pm, GD_TS, 16 * I, 32 * s, lane)};
            };
            const auto turned = [&](const uint16_t* x) {
                return Three{lds_tr8(x, GD_TS, 32 * s, 16 * I, lane), lds_tr8(x + M::pm, GD_TS, 32 * s, 16 * I, lane),
                             lds_tr8(x + 2 * M::pm, GD_TS, 32 * s, 16 * I, lane)};
            };
            Three p0, m0, p1, m1;
            if (left) p0 = rows(pt), m0 = rows(mt);
            if (right) p1 = turned(pt), m1 = turned(mt);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const bf16x8 fk = lds_tr8(Kt, KS, 32 * s, 16 * (d0 + d), lane);
                if (left) {
                    aq[d] = mm(fk, p0, aq[d]);
                    ak[d] = mm(fk, m0, ak[d]);
                }
                if (right) {
                    ak[d] = mm(lds_tr8(Qt, KS, 32 * s, 16 * (d0 + d), lane), p1, ak[d]);
                    ak[d] = mm(fk, m1, ak[d]);
                }
            }
        }
        if (wave == 0) {                                   // d_g: suffix sums over the chunk's tokens
            const double kept2 = (double)kept_[lane] + kept_[GD_C + lane];
            double x = (double)own_[lane] + own_[GD_C + lane] - kept2, all = kept2;
            x -= (double)colsum[lane] + colsum[GD_C + lane] + colsum[2 * GD_C + lane] + colsum[3 * GD_C + lane];
            for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d);
            if (lane == GD_C - 1) {
                double s = 0;
                for (int j = 0; j < 8; ++j) s += part[j];
                x += all + (double)eG[GD_C - 1] * s;
            }
            for (int d = 1; d < 64; d <<= 1) {
                const double o = __shfl_down(x, d);
                if (lane + d < 64) x += o;
            }
            if (t0 + lane < n.T) dg[bh * n.T + t0 + lane] = (float)x;
        } else if (wave == 4 && t0 + lane < n.T) {
            const float x = db_[lane] + db_[GD_C + lane];
            const int64_t at = bh * n.T + t0 + lane;
            if (beta_dt == RWKV6_BF16) reinterpret_cast<uint16_t*>(dbeta)[at] = f2bf(x);
            else reinterpret_cast<float*>(dbeta)[at] = x;
        }
        if (GROUPED) __syncthreads();                      // the sums and G are written again
    }
    anew();
    const int row = t0 + 16 * I + lr;
    if (row < n.T)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int64_t at = (head * n.T + row) * K + 16 * (d0 + d) + 4 * lq;
            *reinterpret_cast<uint2*>(dq + at) = make_uint2(pk2(aq[d][0], aq[d][1]), pk2(aq[d][2], aq[d][3]));
            *reinterpret_cast<uint2*>(dk + at) = make_uint2(pk2(ak[d][0], ak[d][1]), pk2(ak[d][2], ak[d][3]));
        }
}

// A few tokens.  A wave has 32 columns of a head's state in registers: lane group lane / 8 has K / 8 adjacent
// rows, a lane four columns of them, so a row is read in 128 bytes and the sums over rows cross the groups only.
// The state is read and written once, whatever the number of tokens, past the caches (a layer's state is next read
// after every other layer's), and that is all that bounds it: 256 x 32 heads of 128 x 128 190 us, 5.7 TB/s, where a
// copy of 1 GiB reaches 5.2; through the caches it takes 20 us more.  The next token's inputs come under this one's
// arithmetic.
template <int K>
__global__ void __launch_bounds__(64 * GD_STEP_WAVES)
rwkv6_gated_delta_step_kernel(GdTensor q, GdTensor k, GdTensor v, const float* __restrict__ g, const void* __restrict__ beta,
                              int beta_dt, float* __restrict__ state, int64_t ssb, int64_t ssh, uint16_t* __restrict__ o,
                              GdShape n, float scale, unsigned waves) {
    constexpr int R = K / 8;
    const int lane = threadIdx.x & 63, grp = lane >> 3;
    const unsigned w = blockIdx.x * GD_STEP_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w >= waves) return;
    const unsigned nb = n.V / 32, head = w / nb;           // fewer than 2^27 waves
    const int64_t bh = head, b = head / (unsigned)n.HV;
    const int hv = (int)(head % (unsigned)n.HV), hk = hv / (n.HV / n.H), c0 = 32 * (int)(w % nb) + 4 * (lane & 7);
    const uint16_t *qp = q.p + b * q.sb + hk * q.sh + R * grp, *kp = k.p + b * k.sb + hk * k.sh + R * grp;
    const uint16_t* vp = v.p + b * v.sb + hv * v.sh + c0;
    float* sp = state + b * ssb + hv * ssh + (int64_t)(R * grp) * n.V + c0;
    f32x4 S[R];
#pragma unroll
    for (int i = 0; i < R; ++i) S[i] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(sp + (int64_t)i * n.V));
    auto over_groups = [](f32x4 x) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] += lane_xor8(x[j]);
            const RowSums r = row_sums(x[j]);
            x[j] = r.lo + r.hi;
        }
        return x;
    };
    uint4 kr[R / 8], qr[R / 8];
    uint2 vr;
    float gr;
    uint16_t bh_, bl_;                                     // beta's halves: a branch on its type would wait for all loads
    const uint16_t* bp = reinterpret_cast<const uint16_t*>(beta);
    const int wide = beta_dt == RWKV6_F32;
    const auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < R / 8; ++i) {
            kr[i] = *reinterpret_cast<const uint4*>(kp + t * k.st + 8 * i);
            qr[i] = *reinterpret_cast<const uint4*>(qp + t * q.st + 8 * i);
        }
        vr = *reinterpret_cast<const uint2*>(vp + t * v.st);
        gr = g[bh * n.T + t];
        bl_ = bp[(bh * n.T + t) << wide];
        bh_ = bp[((bh * n.T + t) << wide) + wide];
    };
    load(0);
    for (int t = 0; t < n.T; ++t) {
        float kf[R], qf[R], x[4];
#pragma unroll
        for (int i = 0; i < R / 8; ++i) {
            unpack8(kr[i], kf + 8 * i);
            unpack8(qr[i], qf + 8 * i);
        }
        unpack4(vr, x);
        const float a = expf(gr), be = __builtin_bit_cast(float, (uint32_t)bh_ << 16 | (wide ? (uint32_t)bl_ : 0u));
        load(min(t + 1, n.T - 1));                         // under this token's arithmetic
        f32x4 e = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < R; ++i) {
            S[i] *= a;
            e += kf[i] * S[i];
        }
        e = over_groups(e);
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = be * (x[j] - e[j]);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            S[i] += kf[i] * e;
            y += qf[i] * S[i];
        }
        y = over_groups(y) * scale;
        if (grp == 0)
            *reinterpret_cast<uint2*>(o + (bh * n.T + t) * n.V + c0) = make_uint2(pk2(y[0], y[1]), pk2(y[2], y[3]));
    }
#pragma unroll
    for (int i = 0; i < R; ++i) __builtin_nontemporal_store(S[i], reinterpret_cast<f32x4*>(sp + (int64_t)i * n.V));
}

namespace {
inline bool gd_al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// How a head's columns are dealt to blocks: a block of 4 waves of 16 columns, or of fewer where all blocks still find a
// CU of their own (256 and 512 tiles).  A wave then has its SIMD and the CU's LDS to itself: 1.08 ms against 1.55 with 4
// for 32 heads of 512 chunks, 32 us against 40 forward and 44 against 50 backward for 16 heads of 8.
inline int gd_waves(int64_t tiles) { return tiles <= 256 ? 1 : tiles <= 512 ? 2 : 4; }
// Microseconds that `chunks` chunks of that many 16-column tiles take, before the segments' walks and in them: a block's
// start, and a chunk as measured for each way to deal the tiles; 1024 have the chip at once.
inline double gd_time(int tiles, int64_t K, bool back, bool before, int chunks) {
    const double pace[2][2][2][3] = {{{{1.95, 2.25, 3.5}, {1.4, 1.55, 1.9}}, {{2.9, 3.3, 4.3}, {2.0, 2.2, 2.6}}},
                                     {{{2.8, 3.1, 4.4}, {2.45, 2.85, 3.8}}, {{3.8, 4.3, 6.2}, {3.4, 3.8, 5.1}}}};
    const double* p = pace[back][K == 128][before];
    return tiles <= 512 ? 4 + chunks * p[tiles > 256] : ((tiles + 1023) >> 10) * (4 + chunks * p[2]);
}
// Segments of a walk.  Few heads leave most of the chip idle and a walk as long as the sequence: p segments walk
// side by side from states that a walk over all but the last has found (with the K columns of its map beside the
// V of its state) and `join` has put together.  The number with the least time by the paces above and what
// two more launches cost is taken, 1 where none beats it (two segments never do by two hundredths).  Forward of 4 heads
// (64 x 64) of 65536 tokens 1980 to 290 us, of 8 and of 32 heads of 32768 1010 to 190 and 1080 to 550; backward of 8 and of 32
// heads of 16384 730 to 203 and 940 to 640; 256 heads of 4096 tokens fill the chip as they are.
void gd_segments(GdShape* n, int64_t K, bool back) {
    n->segs = 1;
    n->per = n->NC;
    if (n->NC < 8 || n->BH * (n->V / 16) > 512) return;   // nothing to win with fewer chunks, a seventh at most with more tiles
    const int vt = (int)n->BH * (n->V / 16), kt = (int)n->BH * ((int)K / 16);
    double best = gd_time(vt, K, back, false, n->NC);
    for (int p = 3; p <= 16; ++p) {
        const int per = (n->NC + p - 1) / p;
        if ((n->NC + per - 1) / per != p) continue;
        const double t = 12 + (p - 2) + gd_time(vt + (p - 2) * (vt + kt), K, back, true, per) + gd_time(vt * p, K, back, false, per);
        if (t < best) {
            best = t;
            n->segs = p;
            n->per = per;
        }
    }
}
int gd_shape(int64_t B, int64_t H, int64_t HV, int64_t T, int64_t K, int64_t V, GdShape* n) {
    if (B < 0 || H < 1 || HV < 1 || T < 0 || K < 1 || V < 1 || HV % H) return RWKV6_ERR_INVALID_ARG;
    if ((K != 64 && K != 128) || V % 64 || V > 512) return RWKV6_ERR_UNSUPPORTED;
    // a launch holds fewer than 2^32 threads: 512 a chunk and head, or a head and 64 value channels
    const int64_t most = ((int64_t)1 << 23) - 1;
    if (HV > most || B > most / HV || T > ((int64_t)1 << 30)) return RWKV6_ERR_UNSUPPORTED;
    const int64_t NC = (T + GD_C - 1) / GD_C;
    if (B * HV * (NC > V / 64 ? NC : V / 64) > most) return RWKV6_ERR_UNSUPPORTED;
    *n = {(int)H, (int)HV, (int)T, (int)NC, (int)V, B * HV, 0, 0};
    gd_segments(n, K, false);
    return RWKV6_OK;
}
// A strided [B, heads, T, C] tensor: its strides, and the bytes from its first to its last element.
int gd_tensor(const void* p, const int64_t* s, int64_t B, int64_t heads, int64_t T, int64_t C, GdTensor* t, Span* span) {
    *t = {static_cast<const uint16_t*>(p), s[0], s[1], s[2]};
    *span = {p, 0};
    if (!B || !T) return RWKV6_OK;
    if (!p || s[0] < 0 || s[1] < 0 || s[2] < 0) return RWKV6_ERR_INVALID_ARG;
    if (!gd_al16(p) || s[0] % 8 || s[1] % 8 || s[2] % 8) return RWKV6_ERR_ALIGNMENT;
    const int64_t most = (int64_t)1 << 40;
    if (s[0] > most / B || s[1] > most / heads || s[2] > most / T) return RWKV6_ERR_UNSUPPORTED;
    span->n = (size_t)((B - 1) * s[0] + (heads - 1) * s[1] + (T - 1) * s[2] + C) * 2;
    return RWKV6_OK;
}
// What the forward uses itself (T, G, beta, the segments' maps and states) and leaves for the backward (and the states and
// written values).
struct GdSaved {
    size_t T, G, B, E, S, N, end;
    GdSaved(const GdShape& n, int64_t K) {
        const size_t chunks = (size_t)n.BH * n.NC;
        T = 0;
        G = T + chunks * 4 * GD_TB;
        B = G + chunks * 8 * GD_C;
        E = B + chunks * 4 * GD_C;
        S = E + (size_t)n.BH * (n.segs - 1) * 4 * K * (K + n.V);
        N = S + chunks * 4 * K * n.V;
        end = N + chunks * 4 * GD_C * n.V;
    }
};
// The backward's workspace: gradients like the states and values, and its own segments' maps and states.
size_t gd_work(const GdSaved& s, GdShape n, int64_t K) {
    gd_segments(&n, K, true);
    return s.end - s.S + (size_t)n.BH * (n.segs - 1) * 4 * K * (K + n.V);
}
// f(integral constants of the key channels and of gd_waves)
template <class F> void gd_walks(int64_t tiles, int64_t K, F&& f) {
    const auto by_waves = [&](auto k) {
        switch (gd_waves(tiles)) {
        case 1: f(k, std::integral_constant<int, 1>()); break;
        case 2: f(k, std::integral_constant<int, 2>()); break;
        default: f(k, std::integral_constant<int, 4>());
        }
    };
    if (K == 64) by_waves(std::integral_constant<int, 64>());
    else by_waves(std::integral_constant<int, 128>());
}
// Columns that are walked before the segments.
inline int64_t gd_before(const GdShape& n, int64_t K) { return n.V + (n.segs - 2) * (n.V + K); }
void gd_join(const GdShape& n, int64_t K, float* E, hipStream_t s) {
    auto join = K == 64 ? rwkv6_gated_delta_join_kernel<64> : rwkv6_gated_delta_join_kernel<128>;
    hipLaunchKernelGGL(join, dim3((unsigned)(n.BH * (n.V / 16))), dim3(256), 0, s, E, n);
}
// The walks' and gradients' LDS is past what a launch gets by itself: raised once on each device.
int gd_limits(hipStream_t stream) {
    static DeviceOnce once[kMaxDevices];
    int dev = 0, cur = 0;
    const int st = stream_device(stream, &dev, &cur);
    if (st) return st;
    return device_once(once[dev], dev, cur, [] {
        hipError_t e = hipSuccess;
        auto raise = [&](const void* f, size_t bytes) {
            if (e == hipSuccess) e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        };
#define GD_RAISE(K, NW)                                                                                              \
    raise(reinterpret_cast<const void*>(rwkv6_gated_delta_fwd_kernel<K, NW, false>), WalkLds<K, NW, 3>::bytes);       \
    raise(reinterpret_cast<const void*>(rwkv6_gated_delta_fwd_kernel<K, NW, true>), WalkLds<K, NW, 3>::bytes);        \
    raise(reinterpret_cast<const void*>(rwkv6_gated_delta_segment_kernel<K, NW>), WalkLds<K, NW, 0>::bytes);          \
    raise(reinterpret_cast<const void*>(rwkv6_gated_delta_bwd_kernel<K, NW, false>), WalkLds<K, NW, 3>::bytes);       \
    raise(reinterpret_cast<const void*>(rwkv6_gated_delta_bwd_kernel<K, NW, true>), WalkLds<K, NW, 3>::bytes);
        GD_RAISE(64, 1) GD_RAISE(64, 2) GD_RAISE(64, 4) GD_RAISE(128, 1) GD_RAISE(128, 2) GD_RAISE(128, 4)
#undef GD_RAISE
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_grads_kernel<64, false>), GradLds<64>::bytes);
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_grads_kernel<64, true>), GradLds<64>::bytes);
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_grads_kernel<128, false>), GradLds<128>::bytes);
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_grads_kernel<128, true>), GradLds<128>::bytes);
        return e;
    });
}
}  // namespace

extern "C" {

size_t rwkv6_gated_delta_saved_bytes(int64_t B, int64_t HV, int64_t T, int64_t K, int64_t V) {
    GdShape n;
    if (gd_shape(B, 1, HV, T, K, V, &n)) return 0;
    return GdSaved(n, K).end;
}

size_t rwkv6_gated_delta_workspace_bytes(int64_t B, int64_t HV, int64_t T, int64_t K, int64_t V, int for_bwd) {
    GdShape n;
    if (gd_shape(B, 1, HV, T, K, V, &n)) return 0;
    const GdSaved s(n, K);
    return for_bwd ? gd_work(s, n, K) : s.S;
}

int rwkv6_gated_delta_fwd(const void* q, const void* k, const void* v, const int64_t* strides, const float* g,
                          const void* beta, int beta_dtype, const float* h0, void* o, float* hT, void* saved,
                          void* workspace, int64_t B, int64_t H, int64_t HV, int64_t T, int64_t K, int64_t V, float scale,
                          void* stream) {
    GdShape n;
    int st = gd_shape(B, H, HV, T, K, V, &n);
    if (st) return st;
    if (!strides || (beta_dtype != RWKV6_F32 && beta_dtype != RWKV6_BF16)) return RWKV6_ERR_INVALID_ARG;
    if (B == 0) return RWKV6_OK;
    GdTensor qt, kt, vt;
    Span qs, ks, vs;
    if ((st = gd_tensor(q, strides, B, H, T, K, &qt, &qs)) || (st = gd_tensor(k, strides + 3, B, H, T, K, &kt, &ks)) ||
        (st = gd_tensor(v, strides + 6, B, HV, T, V, &vt, &vs)))
        return st;
    if (T > 0 && (!g || !beta || !o || (!saved && !workspace))) return RWKV6_ERR_INVALID_ARG;
    for (const void* p : {(const void*)h0, (const void*)o, (const void*)hT, (const void*)saved, (const void*)workspace})
        if (!gd_al16(p)) return RWKV6_ERR_ALIGNMENT;
    const GdSaved at(n, K);
    const size_t tok = (size_t)n.BH * T, states = (size_t)n.BH * K * V * 4;
    if (any_alias({{o, tok * V * 2}, {hT, states}, {saved, at.end}, {saved ? nullptr : workspace, at.S}},
                  {qs, ks, vs, {g, tok * 4}, {beta, tok * param_bytes(beta_dtype)}, {h0, states}}))
        return RWKV6_ERR_INVALID_ARG;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if ((st = gd_limits(s))) return st;
    char* base = static_cast<char*>(saved ? saved : workspace);
    float2* G = reinterpret_cast<float2*>(base + at.G);
    float* Tm = reinterpret_cast<float*>(base);
    float *be = reinterpret_cast<float*>(base + at.B), *S = saved ? reinterpret_cast<float*>(base + at.S) : nullptr,
          *N = saved ? reinterpret_cast<float*>(base + at.N) : nullptr, *E = reinterpret_cast<float*>(base + at.E);
    if (T > 0) {
        auto prep = K == 64 ? rwkv6_gated_delta_prep_kernel<64> : rwkv6_gated_delta_prep_kernel<128>;
        hipLaunchKernelGGL(prep, dim3((unsigned)(n.BH * n.NC)), dim3(256), 0, s, kt, g, beta, beta_dtype, G, be, Tm, n);
    }
    if (n.segs > 1) {
        const int64_t cols = gd_before(n, K);
        gd_walks(n.BH * (cols / 16), K, [&](auto k_, auto w_) {
            constexpr int k = k_, w = w_;
            auto segment = rwkv6_gated_delta_segment_kernel<k, w>;
            const size_t lds = WalkLds<k, w, 0>::bytes;
            hipLaunchKernelGGL(segment, dim3((unsigned)(n.BH * (cols / (16 * w)))), dim3(walk_threads<w>), lds, s, qt, kt, vt, be, G,
                               Tm, h0, E, n);
        });
        gd_join(n, K, E, s);
    }
    if (T > 0 || hT)
        gd_walks(n.BH * (V / 16) * n.segs, K, [&](auto k_, auto w_) {
            constexpr int k = k_, w = w_;
            auto walk = saved ? rwkv6_gated_delta_fwd_kernel<k, w, true> : rwkv6_gated_delta_fwd_kernel<k, w, false>;
            const size_t lds = WalkLds<k, w, 3>::bytes;
            hipLaunchKernelGGL(walk, dim3((unsigned)(n.BH * (V / (16 * w)) * n.segs)), dim3(walk_threads<w>), lds, s, qt, kt, vt, be, G,
                               Tm, h0, E, (uint16_t*)o, hT, S, N, n, scale);
        });
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}

int rwkv6_gated_delta_bwd(const void* q, const void* k, const void* v, const void* d_o, const int64_t* strides,
                          const void* beta, int beta_dtype, const float* dhT, const void* saved, void* dq, void* dk, void* dv,
                          float* dg, void* dbeta, float* dh0, void* workspace, int64_t B, int64_t H, int64_t HV, int64_t T,
                          int64_t K, int64_t V, float scale, void* stream) {
    GdShape n;
    int st = gd_shape(B, H, HV, T, K, V, &n);
    if (st) return st;
    if (!strides || (beta_dtype != RWKV6_F32 && beta_dtype != RWKV6_BF16)) return RWKV6_ERR_INVALID_ARG;
    if (B == 0) return RWKV6_OK;
    GdTensor qt, kt, vt, ot;
    Span qs, ks, vs, os;
    if ((st = gd_tensor(q, strides, B, H, T, K, &qt, &qs)) || (st = gd_tensor(k, strides + 3, B, H, T, K, &kt, &ks)) ||
        (st = gd_tensor(v, strides + 6, B, HV, T, V, &vt, &vs)) || (st = gd_tensor(d_o, strides + 9, B, HV, T, V, &ot, &os)))
        return st;
    if (T > 0 && (!beta || !saved || !dq || !dk || !dv || !dg || !dbeta || !workspace)) return RWKV6_ERR_INVALID_ARG;
    for (const void* p : {(const void*)dhT, saved, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)dh0,
                          (const void*)workspace})
        if (!gd_al16(p)) return RWKV6_ERR_ALIGNMENT;
    const GdSaved at(n, K);
    const size_t tok = (size_t)n.BH * T, states = (size_t)n.BH * K * V * 4, qk = (size_t)(B * H) * T * K * 2;
    if (any_alias({{dq, qk}, {dk, qk}, {dv, tok * V * 2}, {dg, tok * 4}, {dbeta, tok * param_bytes(beta_dtype)}, {dh0, states},
                   {workspace, gd_work(at, n, K)}},
                  {qs, ks, vs, os, {beta, tok * param_bytes(beta_dtype)}, {dhT, states}, {saved, at.end}}))
        return RWKV6_ERR_INVALID_ARG;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if ((st = gd_limits(s))) return st;
    const char* base = static_cast<const char*>(saved);
    const float2* G = reinterpret_cast<const float2*>(base + at.G);
    const float* Tm = reinterpret_cast<const float*>(base);
    const float *be = reinterpret_cast<const float*>(base + at.B), *S = reinterpret_cast<const float*>(base + at.S),
                *N = reinterpret_cast<const float*>(base + at.N);
    float *D = static_cast<float*>(workspace), *R = D + (at.N - at.S) / 4, *E = D + (at.end - at.S) / 4;
    gd_segments(&n, K, true);
    const auto walks = [&](int64_t cols, auto before) {
        gd_walks(n.BH * (cols / 16), K, [&](auto k_, auto w_) {
            constexpr int k = k_, w = w_;
            auto walk = rwkv6_gated_delta_bwd_kernel<k, w, decltype(before)::value>;
            const size_t lds = WalkLds<k, w, 3>::bytes;
            hipLaunchKernelGGL(walk, dim3((unsigned)(n.BH * (cols / (16 * w)))), dim3(walk_threads<w>), lds, s, qt, kt, ot, be, G, Tm,
                               dhT, E, (uint16_t*)dv, dh0, D, R, n, scale);
        });
    };
    if (n.segs > 1) {
        walks(gd_before(n, K), std::true_type());
        gd_join(n, K, E, s);
    }
    if (T > 0 || dh0) walks(V * n.segs, std::false_type());
    if (T > 0) {
        auto grads = K == 64 ? (HV > H ? rwkv6_gated_delta_grads_kernel<64, true> : rwkv6_gated_delta_grads_kernel<64, false>)
                             : (HV > H ? rwkv6_gated_delta_grads_kernel<128, true> : rwkv6_gated_delta_grads_kernel<128, false>);
        hipLaunchKernelGGL(grads, dim3((unsigned)(B * H * n.NC)), dim3(512), K == 64 ? GradLds<64>::bytes : GradLds<128>::bytes, s,
                           qt, kt, vt, ot, be, beta_dtype, G, S, N, D, R, (uint16_t*)dq, (uint16_t*)dk, dg, dbeta, n, scale);
    }
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}

int rwkv6_gated_delta_step(const void* q, const void* k, const void* v, const int64_t* strides, const float* g,
                           const void* beta, int beta_dtype, float* state, const int64_t* state_strides, void* o, int64_t B,
                           int64_t H, int64_t HV, int64_t T, int64_t K, int64_t V, float scale, void* stream) {
    GdShape n;
    int st = gd_shape(B, H, HV, T, K, V, &n);
    if (st) return st;
    if (!strides || !state_strides || (beta_dtype != RWKV6_F32 && beta_dtype != RWKV6_BF16)) return RWKV6_ERR_INVALID_ARG;
    if (B == 0 || T == 0) return RWKV6_OK;
    GdTensor qt, kt, vt;
    Span qs, ks, vs;
    if ((st = gd_tensor(q, strides, B, H, T, K, &qt, &qs)) || (st = gd_tensor(k, strides + 3, B, H, T, K, &kt, &ks)) ||
        (st = gd_tensor(v, strides + 6, B, HV, T, V, &vt, &vs)))
        return st;
    if (!g || !beta || !o || !state) return RWKV6_ERR_INVALID_ARG;
    // states of different sequences and heads lie apart: heads inside a sequence, or the other way round
    const int64_t sb = state_strides[0], sh = state_strides[1], one = K * V, most = (int64_t)1 << 40;
    if (sb < 0 || sh < 0) return RWKV6_ERR_INVALID_ARG;
    if (sb > most / B || sh > most / HV) return RWKV6_ERR_UNSUPPORTED;
    const bool heads_in = (HV == 1 || sh >= one) && (B == 1 || sb >= (HV - 1) * sh + one);
    const bool seqs_in = (B == 1 || sb >= one) && (HV == 1 || sh >= (B - 1) * sb + one);
    if (!heads_in && !seqs_in) return RWKV6_ERR_INVALID_ARG;
    if (!gd_al16(state) || !gd_al16(o) || (B > 1 && sb % 4) || (HV > 1 && sh % 4)) return RWKV6_ERR_ALIGNMENT;
    const size_t tok = (size_t)n.BH * T;
    if (any_alias({{o, tok * V * 2}, {state, (size_t)((B - 1) * sb + (HV - 1) * sh + one) * 4}},
                  {qs, ks, vs, {g, tok * 4}, {beta, tok * param_bytes(beta_dtype)}}))
        return RWKV6_ERR_INVALID_ARG;
    const int64_t waves = n.BH * (V / 32);
    auto step = K == 64 ? rwkv6_gated_delta_step_kernel<64> : rwkv6_gated_delta_step_kernel<128>;
    hipLaunchKernelGGL(step, dim3((unsigned)((waves + GD_STEP_WAVES - 1) / GD_STEP_WAVES)), dim3(64 * GD_STEP_WAVES), 0,
                       reinterpret_cast<hipStream_t>(stream), qt, kt, vt, g, beta, beta_dtype, state, sb, sh, (uint16_t*)o, n, scale,
                       (unsigned)waves);
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}

}  // extern "C"
