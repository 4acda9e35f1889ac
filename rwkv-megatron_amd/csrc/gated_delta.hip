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
// for d_v and D), `grads` (the rest, a block a chunk), `step` (a few tokens).  Only k S, T (..) and k^T (..)
// follow one another in a walk.  Its columns are independent of each other: a wave keeps 16 columns of S in
// its accumulators, and since an accumulator's rows are what the next product contracts over, it hands every
// intermediate on in registers (the contraction's order is permuted to the accumulators' one, see `rows`).
//
// Numbers.  q, k, v and d_o are bf16 and enter the products as they are.  Everything computed (S, T, n,
// P, ...) is 32 bits and enters as a sum of two bf16, 2^-17 of the value off at most: one product where
// torch would run one in 32 bits becomes two (bf16 times computed) or three (computed times computed, without
// the two low halves), 5 to 8 times the rate of the matrix instructions in 32 bits.  Final states and the
// gradients of g and beta so have the precision of 32-bit arithmetic, not of bf16.
// G is summed in 64 bits and kept as a pair of floats: decays between neighbours late in a chunk are
// differences of large sums.
#include "common.h"
#include "../../include/rwkv6_amd.h"

#define GD_C 64                 // tokens of a chunk
#define GD_PAD 8                // elements behind a row of an LDS tile
#define GD_TS (GD_C + GD_PAD)   // row of a tile of 64 columns
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
};
struct Pair {                   // a computed operand: hi + lo
    bf16x8 h, l;
};

__device__ __forceinline__ Pair split8(const float* x) {
    float f[8], d[8];
    const uint4 h = pack8(x);
    unpack8(h, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) d[j] = x[j] - f[j];
    return {__builtin_bit_cast(bf16x8, h), __builtin_bit_cast(bf16x8, pack8(d))};
}
__device__ __forceinline__ Pair split_tiles(f32x4 a, f32x4 b) {
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return split8(x);
}
// one computed operand, one of bf16
__device__ __forceinline__ f32x4 mm(bf16x8 a, const Pair& b, f32x4 c) { return mfma32(a, b.h, mfma32(a, b.l, c)); }
__device__ __forceinline__ f32x4 mm(const Pair& a, bf16x8 b, f32x4 c) { return mfma32(a.h, b, mfma32(a.l, b, c)); }
// both computed
__device__ __forceinline__ f32x4 mm(const Pair& a, const Pair& b, f32x4 c) {
    return mfma32(a.h, b.h, mfma32(a.h, b.l, mfma32(a.l, b.h, c)));
}

// Operand of 16 rows of a row-major tile, contracted over its columns c0 .. c0 + 31 in the accumulators'
// order: slot 8q + j stands for column c0 + 16 (j / 4) + 4q + j % 4, so that two accumulator tiles, whose lane
// holds rows 4q .. 4q + 3, are the other operand as they are.
__device__ __forceinline__ bf16x8 rows(const uint16_t* X, int stride, int r0, int c0, int lane) {
    const uint16_t* p = X + (r0 + (lane & 15)) * stride + c0 + 4 * (lane >> 4);
    return cat_bf16x8(ld_bf16x4(p), ld_bf16x4(p + 16));
}
// The transposed one: 16 columns, contracted over the rows r0 .. r0 + 31, in the same order.
__device__ __forceinline__ bf16x8 cols(const uint16_t* X, int stride, int r0, int c0, int lane) {
    const int L = lane & 15, q = lane >> 4;
    const uint16_t* p = X + (r0 + 4 * q + (L >> 2)) * stride + c0 + 4 * (L & 3);
    return cat_bf16x8(lds_tr16(p), lds_tr16(p + 16 * stride));
}
__device__ __forceinline__ Pair rows2(const uint16_t* H, const uint16_t* L, int stride, int r0, int c0, int lane) {
    return {rows(H, stride, r0, c0, lane), rows(L, stride, r0, c0, lane)};
}
__device__ __forceinline__ Pair cols2(const uint16_t* H, const uint16_t* L, int stride, int r0, int c0, int lane) {
    return {cols(H, stride, r0, c0, lane), cols(L, stride, r0, c0, lane)};
}
// Rows r0 + 4q .. + 3 of column c0 + lr: a bf16 tile's values as an accumulator tile's lane holds them.
__device__ __forceinline__ f32x4 as_acc(const uint16_t* X, int stride, int r0, int c0, int lane) {
    const int L = lane & 15, q = lane >> 4;
    const uint2 x = __builtin_bit_cast(uint2, lds_tr16(X + (r0 + 4 * q + (L >> 2)) * stride + c0 + 4 * (L & 3)));
    float f[4];
    unpack4(x, f);
    return f32x4{f[0], f[1], f[2], f[3]};
}
__device__ __forceinline__ float gd_gap(float2 a, float2 b) { return (a.x - b.x) + (a.y - b.y); }
__device__ __forceinline__ float gd_beta(const void* p, int dt, int64_t i) {
    return dt == RWKV6_BF16 ? bf2f(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
// Operands in memory as the walks hold them: [chunk][16 columns][32 contracted][hi, lo][lane][8].
__device__ __forceinline__ void put_pair(uint16_t* base, int64_t n, int lane, const Pair& p) {
    uint4* d = reinterpret_cast<uint4*>(base) + n * 128 + lane;
    d[0] = __builtin_bit_cast(uint4, p.h);
    d[64] = __builtin_bit_cast(uint4, p.l);
}

// N 16-byte pieces a thread of a [64][8 * per_row] tile (zeros behind the last token), and into LDS.
template <int COLS> struct TileRegs {
    uint4 q[COLS / 32];
};
template <int COLS>
__device__ __forceinline__ TileRegs<COLS> tile_load(const uint16_t* p, int64_t st, int t0, int T, int tid) {
    TileRegs<COLS> r;
#pragma unroll
    for (int i = 0; i < COLS / 32; ++i) {
        const int n = tid + 256 * i, row = n / (COLS / 8), col = 8 * (n % (COLS / 8)), t = t0 + row;
        r.q[i] = *reinterpret_cast<const uint4*>(p + (int64_t)(t < T ? t : T - 1) * st + col);
        if (t >= T) r.q[i] = make_uint4(0, 0, 0, 0);
    }
    return r;
}
template <int COLS>
__device__ __forceinline__ void tile_store(const TileRegs<COLS>& r, uint16_t* X, int tid) {
#pragma unroll
    for (int i = 0; i < COLS / 32; ++i) {
        const int n = tid + 256 * i, row = n / (COLS / 8), col = 8 * (n % (COLS / 8));
        *reinterpret_cast<uint4*>(X + row * (COLS + GD_PAD) + col) = r.q[i];
    }
}

// P of a chunk as hi and lo tiles [i][j], by four waves: tile t of the triangle's ten by wave t % 4, formed
// transposed, so that a lane has four adjacent j.  The blocks right of the diagonal are zeroed by `gd_zero_p`.
template <int K>
__device__ __forceinline__ void gd_p(const uint16_t* Qt, const uint16_t* Kt, const float2* G, float scale, uint16_t* Ph,
                                     uint16_t* Pl, int wave, int lane) {
    const int lr = lane & 15, q = lane >> 4;
#pragma unroll
    for (int u = 0; u < 3; ++u) {
        const int t = wave + 4 * u;
        if (t >= 10) break;
        const int I = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0, J = t - I * (I + 1) / 2;
        f32x4 a = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < K / 32; ++s)
            a = mfma32(rows(Kt, K + GD_PAD, 16 * J, 32 * s, lane), rows(Qt, K + GD_PAD, 16 * I, 32 * s, lane), a);
        const int i = 16 * I + lr, j = 16 * J + 4 * q;
        const float2 gi = G[i];
        float x[4], d[4], f[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = i >= j + r ? scale * ex2(gd_gap(gi, G[j + r])) * a[r] : 0.f;
        const uint2 h = make_uint2(pk2(x[0], x[1]), pk2(x[2], x[3]));
        unpack4(h, f);
#pragma unroll
        for (int r = 0; r < 4; ++r) d[r] = x[r] - f[r];
        *reinterpret_cast<uint2*>(Ph + i * GD_TS + j) = h;
        *reinterpret_cast<uint2*>(Pl + i * GD_TS + j) = make_uint2(pk2(d[0], d[1]), pk2(d[2], d[3]));
    }
}
__device__ __forceinline__ void gd_zero_p(uint16_t* Ph, uint16_t* Pl, int tid) {
    // blocks (0,1) and (2,3): 2 x 16 rows of 32 bytes, hi and lo
    if (tid < 128) {
        const int row = (tid >> 1) & 15, b = (tid >> 5) & 1, half = tid & 1;
        uint16_t* P = tid & 64 ? Pl : Ph;
        *reinterpret_cast<uint4*>(P + (32 * b + row) * GD_TS + 32 * b + 16 + 8 * half) = make_uint4(0, 0, 0, 0);
    }
}

}  // namespace

// G and T of a chunk.  Wave w forms the rows of its 16-token block of A = beta L k k^T, inverts the block
// on the diagonal by substitution, and then column w of the blocks below it, in the 32-bit matrix instructions:
// T_IJ = -T_II sum_{J<=l<I} A_Il T_lJ.  Out: G [chunk][64] as pairs of floats in base-2 units, T [chunk]
// [hi, lo][64][64].
template <int K>
__global__ void __launch_bounds__(256)
rwkv6_gated_delta_prep_kernel(GdTensor k, const float* __restrict__ g, const void* __restrict__ beta, int beta_dt,
                              float2* __restrict__ G_out, uint16_t* __restrict__ T_out, GdShape n) {
    __shared__ __attribute__((aligned(16))) float As[GD_C][GD_C + 4], Ts[GD_C][GD_C + 4];
    __shared__ float2 G[GD_C];
    __shared__ float be[GD_C];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, q = lane >> 4;
    const int64_t chunk = blockIdx.x, bh = chunk / n.NC;
    const int c = (int)(chunk - bh * n.NC), hv = (int)(bh % n.HV), t0 = c * GD_C;
    const uint16_t* kp = k.p + (bh / n.HV) * k.sb + (int64_t)(hv / (n.HV / n.H)) * k.sh;
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
    }
    __syncthreads();
#pragma unroll
    for (int I = 0; I < 4; ++I) {
        if (I != wave) continue;
#pragma unroll
        for (int J = 0; J <= I; ++J) {
            f32x4 a = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < K / 32; ++s) a = mfma32(f[I][s], f[J][s], a);
            const int j = 16 * J + lr;
            const float2 gj = G[j];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * I + 4 * q + r;
                As[i][j] = i > j ? be[i] * ex2(gd_gap(G[i], gj)) * a[r] : 0.f;
            }
        }
    }
    __syncthreads();
    {
        float x[16];
        const int b = 16 * wave;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float a[16], s0 = r == lr ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
            for (int s = 0; s < r; s += 4) {
                const float4 v = *reinterpret_cast<const float4*>(&As[b + r][b + s]);
                a[s] = v.x, a[s + 1] = v.y, a[s + 2] = v.z, a[s + 3] = v.w;
            }
#pragma unroll
            for (int s = 0; s < r; ++s) (s & 1 ? s1 : s0) -= a[s] * x[s];
            x[r] = s0 + s1;
            if ((r >> 2) == q) Ts[b + r][b + lr] = x[r];
        }
    }
    __syncthreads();
#pragma unroll
    for (int J = 0; J < 3; ++J) {
        if (J != wave) continue;
        f32x4 t[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) t[J][r] = Ts[16 * J + 4 * q + r][16 * J + lr];
#pragma unroll
        for (int I = J + 1; I < 4; ++I) {
            f32x4 a = {0, 0, 0, 0}, d = {0, 0, 0, 0};
#pragma unroll
            for (int l = J; l < I; ++l) {
                const float4 v = *reinterpret_cast<const float4*>(&As[16 * I + lr][16 * l + 4 * q]);
                const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int r = 0; r < 4; ++r) a = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r], t[l][r], a, 0, 0, 0);
            }
            const float4 v = *reinterpret_cast<const float4*>(&Ts[16 * I + lr][16 * I + 4 * q]);
            const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) d = __builtin_amdgcn_mfma_f32_16x16x4f32(w[r], a[r], d, 0, 0, 0);
            t[I] = -d;
#pragma unroll
            for (int r = 0; r < 4; ++r) Ts[16 * I + 4 * q + r][16 * J + lr] = t[I][r];
        }
    }
    __syncthreads();
    const int row = tid >> 2, cb = tid & 3;
    uint4* out = reinterpret_cast<uint4*>(T_out + chunk * (2 * GD_C * GD_C) + row * GD_C + 16 * cb);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = cb <= (row >> 4) ? Ts[row][16 * cb + 8 * h + j] : 0.f;
        const Pair p = split8(x);
        out[h] = __builtin_bit_cast(uint4, p.h);
        out[h + GD_C * GD_C / 8] = __builtin_bit_cast(uint4, p.l);
    }
}

namespace {
// LDS of the walks: two buffers of q, k, v (or d_o), T hi and lo, G, e^G, e^{G_C - G}, beta; then P hi and lo.
template <int K> struct WalkLds {
    static constexpr int qk = GD_C * (K + GD_PAD), t = GD_C * GD_TS;
    static constexpr int buf = 2 * qk + 3 * t + (8 + 3 * 4) / 2 * GD_C;          // in elements of 2 bytes
    static constexpr size_t bytes = (size_t)(2 * buf + 2 * t) * 2;
};
struct WalkBuf {
    uint16_t *Q, *K, *V, *Th, *Tl;
    float2* G;
    float *eG, *eL, *be;
};
template <int K> __device__ __forceinline__ WalkBuf walk_buf(uint16_t* p) {
    using L = WalkLds<K>;
    WalkBuf b;
    b.Q = p;
    b.K = p + L::qk;
    b.V = p + 2 * L::qk;
    b.Th = b.V + L::t;
    b.Tl = b.Th + L::t;
    b.G = reinterpret_cast<float2*>(b.Tl + L::t);
    b.eG = reinterpret_cast<float*>(b.G + GD_C);
    b.eL = b.eG + GD_C;
    b.be = b.eL + GD_C;
    return b;
}
// One chunk's inputs on their way from memory to LDS.
template <int K> struct WalkRegs {
    TileRegs<K> q, k;
    TileRegs<64> v, th, tl;
    float2 G, GC;
    float be;
};
template <int K>
__device__ __forceinline__ WalkRegs<K> walk_load(const uint16_t* qp, int64_t qs, const uint16_t* kp, int64_t ks, const uint16_t* vp,
                                                 int64_t vs, const uint16_t* T, const float2* G, const void* beta, int beta_dt,
                                                 int64_t bh, int c, const GdShape& n, int tid) {
    WalkRegs<K> r;
    const int t0 = c * GD_C;
    const int64_t chunk = bh * n.NC + c;
    r.k = tile_load<K>(kp, ks, t0, n.T, tid);
    r.th = tile_load<64>(T + chunk * (2 * GD_C * GD_C), GD_C, 0, GD_C, tid);
    r.tl = tile_load<64>(T + chunk * (2 * GD_C * GD_C) + GD_C * GD_C, GD_C, 0, GD_C, tid);
    r.v = tile_load<64>(vp, vs, t0, n.T, tid);
    r.q = tile_load<K>(qp, qs, t0, n.T, tid);
    if (tid < GD_C) {
        r.G = G[chunk * GD_C + tid];
        r.GC = G[chunk * GD_C + GD_C - 1];
        r.be = t0 + tid < n.T ? gd_beta(beta, beta_dt, bh * n.T + t0 + tid) : 0.f;
    }
    return r;
}
template <int K>
__device__ __forceinline__ void walk_store(const WalkRegs<K>& r, const WalkBuf& L, int tid) {
    tile_store<K>(r.q, L.Q, tid);
    tile_store<K>(r.k, L.K, tid);
    tile_store<64>(r.v, L.V, tid);
    tile_store<64>(r.th, L.Th, tid);
    tile_store<64>(r.tl, L.Tl, tid);
    if (tid < GD_C) {
        L.G[tid] = r.G;
        L.eG[tid] = ex2(r.G.x);
        L.eL[tid] = ex2(gd_gap(r.GC, r.G));
        L.be[tid] = r.be;
    }
}
}  // namespace

// A block walks one head's chunks with 64 columns of the state, a wave 16 of them.  S_save and n_save (the
// backward's, or null) get the state entering each chunk and the values it writes.
template <int K>
__global__ void __launch_bounds__(256)
rwkv6_gated_delta_fwd_kernel(GdTensor q, GdTensor k, GdTensor v, const void* __restrict__ beta, int beta_dt,
                             const float2* __restrict__ G, const uint16_t* __restrict__ T, const float* __restrict__ h0,
                             uint16_t* __restrict__ o, float* __restrict__ hT, uint16_t* __restrict__ S_save,
                             uint16_t* __restrict__ n_save, GdShape n, float scale) {
    extern __shared__ __attribute__((aligned(16))) uint16_t gd_lds[];
    uint16_t *const Ph = gd_lds + 2 * WalkLds<K>::buf, *const Pl = Ph + WalkLds<K>::t;
    constexpr int KS = K + GD_PAD, ND = K / 16, NS = K / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lq = lane >> 4;
    const int64_t bh = blockIdx.x % n.BH, b = bh / n.HV;
    const int hv = (int)(bh % n.HV), hk = hv / (n.HV / n.H), v0 = 64 * (int)(blockIdx.x / n.BH), ct = v0 / 16 + wave;
    const uint16_t *qp = q.p + b * q.sb + hk * q.sh, *kp = k.p + b * k.sb + hk * k.sh, *vp = v.p + b * v.sb + hv * v.sh + v0;
    const int col = v0 + 16 * wave + lr;
    f32x4 S[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[d][r] = h0 ? h0[(bh * K + 16 * d + 4 * lq + r) * n.V + col] : 0.f;
    gd_zero_p(Ph, Pl, tid);
    if (n.NC) walk_store<K>(walk_load<K>(qp, q.st, kp, k.st, vp, v.st, T, G, beta, beta_dt, bh, 0, n, tid), walk_buf<K>(gd_lds), tid);
    for (int c = 0; c < n.NC; ++c) {
        const int u = c & 1;
        const WalkBuf L = walk_buf<K>(gd_lds + u * WalkLds<K>::buf);
        const int64_t chunk = bh * n.NC + c;
        __syncthreads();
        const bool more = c + 1 < n.NC;
        WalkRegs<K> next;
        if (more) next = walk_load<K>(qp, q.st, kp, k.st, vp, v.st, T, G, beta, beta_dt, bh, c + 1, n, tid);
        gd_p<K>(L.Q, L.K, L.G, scale, Ph, Pl, wave, lane);
        Pair Sp[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            Sp[s] = split_tiles(S[2 * s], S[2 * s + 1]);
            if (S_save) put_pair(S_save, (chunk * (n.V / 16) + ct) * NS + s, lane, Sp[s]);
        }
        f32x4 E[4];
#pragma unroll
        for (int I = 0; I < 4; ++I) {
            f32x4 a = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NS; ++s) a = mm(rows(L.K, KS, 16 * I, 32 * s, lane), Sp[s], a);
            const f32x4 x = as_acc(L.V, GD_TS, 16 * I, 16 * wave, lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * I + 4 * lq + r;
                E[I][r] = L.be[i] * (x[r] - L.eG[i] * a[r]);
            }
        }
        Pair Ep[2] = {split_tiles(E[0], E[1]), split_tiles(E[2], E[3])};
        f32x4 N[4];
#pragma unroll
        for (int I = 0; I < 4; ++I) {
            N[I] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s <= I / 2; ++s) N[I] = mm(rows2(L.Th, L.Tl, GD_TS, 16 * I, 32 * s, lane), Ep[s], N[I]);
        }
        Pair Np[2] = {split_tiles(N[0], N[1]), split_tiles(N[2], N[3])};
        if (n_save) {
            put_pair(n_save, (chunk * (n.V / 16) + ct) * 2, lane, Np[0]);
            put_pair(n_save, (chunk * (n.V / 16) + ct) * 2 + 1, lane, Np[1]);
        }
#pragma unroll
        for (int I = 0; I < 4; ++I)
#pragma unroll
            for (int r = 0; r < 4; ++r) N[I][r] *= L.eL[16 * I + 4 * lq + r];
        Ep[0] = split_tiles(N[0], N[1]);
        Ep[1] = split_tiles(N[2], N[3]);
        const float eC = L.eG[GD_C - 1];
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            S[d] *= eC;
#pragma unroll
            for (int s = 0; s < 2; ++s) S[d] = mm(cols(L.K, KS, 32 * s, 16 * d, lane), Ep[s], S[d]);
        }
        __syncthreads();                                   // P
        // o transposed: a lane has four adjacent channels of a token
#pragma unroll
        for (int I = 0; I < 4; ++I) {
            f32x4 a = {0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NS; ++s) a = mm(Sp[s], rows(L.Q, KS, 16 * I, 32 * s, lane), a);
            a *= scale * L.eG[16 * I + lr];
#pragma unroll
            for (int s = 0; s <= I / 2; ++s) a = mm(Np[s], rows2(Ph, Pl, GD_TS, 16 * I, 32 * s, lane), a);
            const int t = c * GD_C + 16 * I + lr;
            if (t < n.T)
                *reinterpret_cast<uint2*>(o + (bh * n.T + t) * n.V + v0 + 16 * wave + 4 * lq) = make_uint2(pk2(a[0], a[1]), pk2(a[2], a[3]));
        }
        if (more) walk_store<K>(next, walk_buf<K>(gd_lds + (u ^ 1) * WalkLds<K>::buf), tid);
    }
    if (hT)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) hT[(bh * K + 16 * d + 4 * lq + r) * n.V + col] = S[d][r];
}

// The walk back: d_v, and for the other gradients r and the gradient D of the state that each chunk leaves.
template <int K>
__global__ void __launch_bounds__(256)
rwkv6_gated_delta_bwd_kernel(GdTensor q, GdTensor k, GdTensor d_o, const void* __restrict__ beta, int beta_dt,
                             const float2* __restrict__ G, const uint16_t* __restrict__ T, const float* __restrict__ dhT,
                             uint16_t* __restrict__ dv, float* __restrict__ dh0, uint16_t* __restrict__ D_save,
                             uint16_t* __restrict__ r_save, GdShape n, float scale) {
    extern __shared__ __attribute__((aligned(16))) uint16_t gd_lds[];
    uint16_t *const Ph = gd_lds + 2 * WalkLds<K>::buf, *const Pl = Ph + WalkLds<K>::t;
    constexpr int KS = K + GD_PAD, ND = K / 16, NS = K / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lq = lane >> 4;
    const int64_t bh = blockIdx.x % n.BH, b = bh / n.HV;
    const int hv = (int)(bh % n.HV), hk = hv / (n.HV / n.H), v0 = 64 * (int)(blockIdx.x / n.BH), ct = v0 / 16 + wave;
    const uint16_t *qp = q.p + b * q.sb + hk * q.sh, *kp = k.p + b * k.sb + hk * k.sh, *op = d_o.p + b * d_o.sb + hv * d_o.sh + v0;
    const int col = v0 + 16 * wave + lr;
    f32x4 D[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) D[d][r] = dhT ? dhT[(bh * K + 16 * d + 4 * lq + r) * n.V + col] : 0.f;
    gd_zero_p(Ph, Pl, tid);
    if (n.NC) walk_store<K>(walk_load<K>(qp, q.st, kp, k.st, op, d_o.st, T, G, beta, beta_dt, bh, n.NC - 1, n, tid), walk_buf<K>(gd_lds), tid);
    for (int c = n.NC - 1, u = 0; c >= 0; --c, u ^= 1) {
        const WalkBuf L = walk_buf<K>(gd_lds + u * WalkLds<K>::buf);
        const int64_t chunk = bh * n.NC + c;
        __syncthreads();
        WalkRegs<K> next;
        if (c) next = walk_load<K>(qp, q.st, kp, k.st, op, d_o.st, T, G, beta, beta_dt, bh, c - 1, n, tid);
        gd_p<K>(L.Q, L.K, L.G, scale, Ph, Pl, wave, lane);
        Pair Dp[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            Dp[s] = split_tiles(D[2 * s], D[2 * s + 1]);
            put_pair(D_save, (chunk * (n.V / 16) + ct) * NS + s, lane, Dp[s]);
        }
        const float eC = L.eG[GD_C - 1];
        f32x4 X[4], Y[4];                                  // d_n; scale e^G d_o
#pragma unroll
        for (int I = 0; I < 4; ++I) {
            X[I] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < NS; ++s) X[I] = mm(rows(L.K, KS, 16 * I, 32 * s, lane), Dp[s], X[I]);
            Y[I] = as_acc(L.V, GD_TS, 16 * I, 16 * wave, lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * I + 4 * lq + r;
                X[I][r] *= L.eL[i];
                Y[I][r] *= scale * L.eG[i];
            }
        }
        const Pair Yp[2] = {split_tiles(Y[0], Y[1]), split_tiles(Y[2], Y[3])};
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            D[d] *= eC;
#pragma unroll
            for (int s = 0; s < 2; ++s) D[d] = mm(cols(L.Q, KS, 32 * s, 16 * d, lane), Yp[s], D[d]);
        }
        __syncthreads();                                   // P
        const bf16x8 dof[2] = {cols(L.V, GD_TS, 0, 16 * wave, lane), cols(L.V, GD_TS, 32, 16 * wave, lane)};
#pragma unroll
        for (int I = 0; I < 4; ++I)
#pragma unroll
            for (int s = I / 2; s < 2; ++s) X[I] = mm(cols2(Ph, Pl, GD_TS, 32 * s, 16 * I, lane), dof[s], X[I]);
        const Pair Xp[2] = {split_tiles(X[0], X[1]), split_tiles(X[2], X[3])};
        f32x4 R[4];
#pragma unroll
        for (int I = 0; I < 4; ++I) {
            R[I] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = I / 2; s < 2; ++s) R[I] = mm(cols2(L.Th, L.Tl, GD_TS, 32 * s, 16 * I, lane), Xp[s], R[I]);
        }
        put_pair(r_save, (chunk * (n.V / 16) + ct) * 2, lane, split_tiles(R[0], R[1]));
        put_pair(r_save, (chunk * (n.V / 16) + ct) * 2 + 1, lane, split_tiles(R[2], R[3]));
#pragma unroll
        for (int I = 0; I < 4; ++I)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * I + 4 * lq + r, t = c * GD_C + i;
                const float x = L.be[i] * R[I][r];
                if (t < n.T) dv[(bh * n.T + t) * n.V + col] = f2bf(x);
                R[I][r] = -L.eG[i] * x;
            }
        const Pair Rp[2] = {split_tiles(R[0], R[1]), split_tiles(R[2], R[3])};
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int s = 0; s < 2; ++s) D[d] = mm(cols(L.K, KS, 32 * s, 16 * d, lane), Rp[s], D[d]);
        if (c) walk_store<K>(next, walk_buf<K>(gd_lds + (u ^ 1) * WalkLds<K>::buf), tid);
    }
    if (dh0)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) dh0[(bh * K + 16 * d + 4 * lq + r) * n.V + col] = D[d][r];
}

namespace {
// LDS of the gradients: q and k; 32 value channels of n, r [32][64 tokens] and S, D [32][K] as hi and lo, in
// whose place p and m [64][64] hi and lo come afterwards; sums.
template <int K> struct GradLds {
    static constexpr int qk = GD_C * (K + GD_PAD), nv = 32 * GD_TS, sv = 32 * (K + GD_PAD), pm = GD_C * GD_TS;
    static constexpr int shared_ = 4 * nv + 4 * sv > 4 * pm ? 4 * nv + 4 * sv : 4 * pm;
    static constexpr size_t bytes = (size_t)(2 * qk + shared_) * 2 + GD_C * 8 + (GD_C * 3 + 4 * GD_C + GD_C + 8) * 4;
};
// Two 16-column tiles of operands in the walks' layout, STEPS steps of 32 each, into tiles [32 columns][contracted].
template <int STEPS> struct PairRegs {
    uint4 q[STEPS];
};
template <int STEPS>
__device__ __forceinline__ PairRegs<STEPS> pairs_load(const uint16_t* base, int64_t n0, int tid) {
    PairRegs<STEPS> r;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) r.q[i] = reinterpret_cast<const uint4*>(base)[n0 * 128 + tid + 256 * i];
    return r;
}
template <int STEPS>
__device__ __forceinline__ void pairs_store(const PairRegs<STEPS>& x, uint16_t* H, uint16_t* Lo, int tid) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int m = tid + 256 * i, lane = m & 63, step = (m >> 7) % STEPS, tile = (m >> 7) / STEPS;
        uint16_t* p = (m & 64 ? Lo : H) + (16 * tile + (lane & 15)) * (32 * STEPS + GD_PAD) + 32 * step + 4 * (lane >> 4);
        *reinterpret_cast<uint2*>(p) = make_uint2(x.q[i].x, x.q[i].y);
        *reinterpret_cast<uint2*>(p + 16) = make_uint2(x.q[i].z, x.q[i].w);
    }
}
__device__ __forceinline__ Pair tr8(const uint16_t* H, const uint16_t* L, int stride, int c0, int lane) {
    return {lds_tr8(H, stride, 0, c0, lane), lds_tr8(L, stride, 0, c0, lane)};
}
__device__ __forceinline__ float sum16(float v) {          // over the 16 lanes of a row
    v = sum8lanes(v);
    return v + dpp_mov<0x140>(v);
}
}  // namespace

// d_q, d_k, d_g and d_beta of a chunk of a key head, its value heads one after the other; wave w has the rows
// of tokens 16w .. 16w + 15.
template <int K>
__global__ void __launch_bounds__(256)
rwkv6_gated_delta_grads_kernel(GdTensor q, GdTensor k, GdTensor v, GdTensor d_o, const void* __restrict__ beta, int beta_dt,
                               const float2* __restrict__ G_in, const uint16_t* __restrict__ S_save,
                               const uint16_t* __restrict__ n_save, const uint16_t* __restrict__ D_save,
                               const uint16_t* __restrict__ r_save, uint16_t* __restrict__ dq, uint16_t* __restrict__ dk,
                               float* __restrict__ dg, void* __restrict__ dbeta, GdShape n, float scale) {
    extern __shared__ __attribute__((aligned(16))) uint16_t gd_lds[];
    using M = GradLds<K>;
    constexpr int KS = K + GD_PAD, ND = K / 16, NS = K / 32;
    uint16_t *Qt = gd_lds, *Kt = Qt + M::qk, *X = Kt + M::qk;
    uint16_t *Nh = X, *Nl = Nh + M::nv, *Rh = Nl + M::nv, *Rl = Rh + M::nv;
    uint16_t *Sh = Rl + M::nv, *Sl = Sh + M::sv, *Dh = Sl + M::sv, *Dl = Dh + M::sv;
    uint16_t *ph = X, *pl = ph + M::pm, *mh = pl + M::pm, *ml = mh + M::pm;
    float2* G = reinterpret_cast<float2*>(X + M::shared_);
    float *eG = reinterpret_cast<float*>(G + GD_C), *eL = eG + GD_C, *be = eL + GD_C, *colsum = be + GD_C, *dG = colsum + 4 * GD_C,
          *part = dG + GD_C;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lq = lane >> 4;
    const int group = n.HV / n.H;
    const int64_t kc = blockIdx.x, bk = kc / n.NC, b = bk / n.H;
    const int c = (int)(kc - bk * n.NC), hk = (int)(bk % n.H), t0 = c * GD_C;
    const uint16_t *qp = q.p + b * q.sb + hk * q.sh, *kp = k.p + b * k.sb + hk * k.sh;
    tile_store<K>(tile_load<K>(qp, q.st, t0, n.T, tid), Qt, tid);
    tile_store<K>(tile_load<K>(kp, k.st, t0, n.T, tid), Kt, tid);
    const int row = t0 + 16 * wave + lr;                   // the token whose operands this lane reads
    f32x4 aq[ND], ak[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) aq[d] = ak[d] = f32x4{0, 0, 0, 0};
    for (int e = 0; e < group; ++e) {
        const int hv = hk * group + e;
        const int64_t bh = b * n.HV + hv, chunk = bh * n.NC + c;
        const uint16_t *vp = v.p + b * v.sb + hv * v.sh, *op = d_o.p + b * d_o.sb + hv * d_o.sh;
        if (tid < GD_C) {
            const float2 g = G_in[chunk * GD_C + tid], gC = G_in[chunk * GD_C + GD_C - 1];
            G[tid] = g;
            eG[tid] = ex2(g.x);
            eL[tid] = ex2(gd_gap(gC, g));
            be[tid] = t0 + tid < n.T ? gd_beta(beta, beta_dt, bh * n.T + t0 + tid) : 0.f;
        }
        f32x4 P[4], R[4], Z[ND], Y[ND], W[ND], RV = {0, 0, 0, 0};
        float sd = 0.f;
#pragma unroll
        for (int J = 0; J < 4; ++J) P[J] = R[J] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < ND; ++d) Z[d] = Y[d] = W[d] = f32x4{0, 0, 0, 0};
        for (int vb = 0; vb < n.V / 32; ++vb) {
            const int64_t ct = chunk * (n.V / 16) + 2 * vb;
            const PairRegs<2> xn = pairs_load<2>(n_save, ct * 2, tid), xr = pairs_load<2>(r_save, ct * 2, tid);
            const PairRegs<NS> xs = pairs_load<NS>(S_save, ct * NS, tid), xd = pairs_load<NS>(D_save, ct * NS, tid);
            uint4 ov = *reinterpret_cast<const uint4*>(op + (int64_t)(row < n.T ? row : n.T - 1) * d_o.st + 32 * vb + 8 * lq);
            uint4 vv = *reinterpret_cast<const uint4*>(vp + (int64_t)(row < n.T ? row : n.T - 1) * v.st + 32 * vb + 8 * lq);
            if (row >= n.T) ov = vv = make_uint4(0, 0, 0, 0);
            const bf16x8 fo = __builtin_bit_cast(bf16x8, ov), fv = __builtin_bit_cast(bf16x8, vv);
            __syncthreads();                               // the last block's operands, or p and m, are done with
            pairs_store<2>(xn, Nh, Nl, tid);
            pairs_store<2>(xr, Rh, Rl, tid);
            pairs_store<NS>(xs, Sh, Sl, tid);
            pairs_store<NS>(xd, Dh, Dl, tid);
            __syncthreads();
            for (int i = tid; i < 32 * K / 4; i += 256) {
                const int at = (i / (K / 4)) * KS + 4 * (i % (K / 4));
                float a[4], a2[4], d[4], d2[4];
                unpack4(*reinterpret_cast<const uint2*>(Sh + at), a);
                unpack4(*reinterpret_cast<const uint2*>(Sl + at), a2);
                unpack4(*reinterpret_cast<const uint2*>(Dh + at), d);
                unpack4(*reinterpret_cast<const uint2*>(Dl + at), d2);
#pragma unroll
                for (int j = 0; j < 4; ++j) sd += (a[j] + a2[j]) * (d[j] + d2[j]);
            }
            const Pair fr = tr8(Rh, Rl, GD_TS, 16 * wave, lane), fn = tr8(Nh, Nl, GD_TS, 16 * wave, lane);
            RV = mm(fr, fv, RV);
#pragma unroll
            for (int J = 0; J < 4; ++J) {
                if (J > wave) continue;
                const Pair nj = tr8(Nh, Nl, GD_TS, 16 * J, lane);
                P[J] = mm(fo, nj, P[J]);
                R[J] = mm(fr, nj, R[J]);
            }
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const Pair sp = tr8(Sh, Sl, KS, 16 * d, lane), dp = tr8(Dh, Dl, KS, 16 * d, lane);
                Z[d] = mm(fo, sp, Z[d]);
                Y[d] = mm(fr, sp, Y[d]);
                W[d] = mm(fn, dp, W[d]);
            }
        }
        sd = wave_sum(sd);
        if (lane == 0) part[wave] = sd;
        __syncthreads();                                   // p and m take the operands' place
        float own[4] = {0, 0, 0, 0}, kept[4] = {0, 0, 0, 0}, db[4] = {0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * wave + 4 * lq + r;
                const float qv = bf2f(Qt[i * KS + 16 * d + lr]), kv = bf2f(Kt[i * KS + 16 * d + lr]);
                Z[d][r] *= scale * eG[i];
                Y[d][r] *= eG[i];
                W[d][r] *= eL[i];
                db[r] -= Y[d][r] * kv;
                own[r] += Z[d][r] * qv - be[i] * Y[d][r] * kv;
                kept[r] += W[d][r] * kv;
                aq[d][r] += Z[d][r];
                ak[d][r] += W[d][r] - be[i] * Y[d][r];
            }
#pragma unroll
        for (int J = 0; J < 4; ++J) {
            const int j = 16 * J + lr;
            float cs = 0.f;
            if (J <= wave) {
                f32x4 qk = {0, 0, 0, 0}, kk = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const bf16x8 kj = rows(Kt, KS, 16 * J, 32 * s, lane);
                    qk = mfma32(rows(Qt, KS, 16 * wave, 32 * s, lane), kj, qk);
                    kk = mfma32(rows(Kt, KS, 16 * wave, 32 * s, lane), kj, kk);
                }
                const float2 gj = G[j];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * wave + 4 * lq + r;
                    const float l = ex2(gd_gap(G[i], gj));
                    const float p = i >= j ? scale * l * P[J][r] : 0.f, w = i > j ? -l * R[J][r] : 0.f, m = be[i] * w;
                    const float x = p * qk[r] + m * kk[r];
                    own[r] += x;
                    cs += x;
                    db[r] += w * kk[r];
                    const uint16_t hp = f2bf(p), hm = f2bf(m);
                    ph[i * GD_TS + j] = hp;
                    pl[i * GD_TS + j] = f2bf(p - bf2f(hp));
                    mh[i * GD_TS + j] = hm;
                    ml[i * GD_TS + j] = f2bf(m - bf2f(hm));
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int at = (16 * wave + 4 * lq + r) * GD_TS + j;
                    ph[at] = pl[at] = mh[at] = ml[at] = 0;
                }
            }
            const RowSums rs = row_sums(cs);
            if (lq == 0) colsum[wave * GD_C + j] = rs.lo + rs.hi;
        }
        float all = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * wave + 4 * lq + r;
            if (lr == 4 * lq + r) db[r] += RV[r];          // the diagonal of r v^T
            own[r] = sum16(own[r]);
            kept[r] = sum16(kept[r]);
            db[r] = sum16(db[r]);
            all += kept[r];
            if (lr == 0) {
                dG[i] = own[r] - kept[r];
                if (t0 + i < n.T) {
                    const int64_t at = bh * n.T + t0 + i;
                    if (beta_dt == RWKV6_BF16) reinterpret_cast<uint16_t*>(dbeta)[at] = f2bf(db[r]);
                    else reinterpret_cast<float*>(dbeta)[at] = db[r];
                }
            }
        }
        const RowSums ks = row_sums(all);
        if (lane == 0) part[4 + wave] = ks.lo + ks.hi;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            // own rows: columns up to the diagonal; transposed: rows from it
            const bool left = 2 * s <= wave, right = 2 * s + 1 >= wave;
            Pair p0, m0, p1, m1;
            if (left) {
                p0 = rows2(ph, pl, GD_TS, 16 * wave, 32 * s, lane);
                m0 = rows2(mh, ml, GD_TS, 16 * wave, 32 * s, lane);
            }
            if (right) {
                p1 = cols2(ph, pl, GD_TS, 32 * s, 16 * wave, lane);
                m1 = cols2(mh, ml, GD_TS, 32 * s, 16 * wave, lane);
            }
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const bf16x8 fk = cols(Kt, KS, 32 * s, 16 * d, lane);
                if (left) {
                    aq[d] = mm(p0, fk, aq[d]);
                    ak[d] = mm(m0, fk, ak[d]);
                }
                if (right) {
                    ak[d] = mm(p1, cols(Qt, KS, 32 * s, 16 * d, lane), ak[d]);
                    ak[d] = mm(m1, fk, ak[d]);
                }
            }
        }
        if (wave == 0) {                                   // d_g: suffix sums over the chunk's tokens
            double x = (double)dG[lane] - ((double)colsum[lane] + colsum[GD_C + lane] + colsum[2 * GD_C + lane] + colsum[3 * GD_C + lane]);
            if (lane == GD_C - 1)
                x += (double)part[4] + part[5] + part[6] + part[7] + (double)eG[GD_C - 1] * ((double)part[0] + part[1] + part[2] + part[3]);
            for (int d = 1; d < 64; d <<= 1) {
                const double o = __shfl_down(x, d);
                if (lane + d < 64) x += o;
            }
            if (t0 + lane < n.T) dg[bh * n.T + t0 + lane] = (float)x;
        }
        __syncthreads();                                   // the sums and G are written again
    }
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = t0 + 16 * wave + 4 * lq + r;
            if (t >= n.T) continue;
            const int64_t at = (bk * n.T + t) * K + 16 * d + lr;
            dq[at] = f2bf(aq[d][r]);
            dk[at] = f2bf(ak[d][r]);
        }
}

// A few tokens.  A wave has 32 columns of a head's state in registers: lane group lane / 8 has K / 8 adjacent
// rows, a lane four columns of them, so a row is read in 128 bytes and the sums over rows cross the groups only.
// The state is read and written once, whatever the number of tokens, and that is all that bounds it.
template <int K>
__global__ void __launch_bounds__(64 * GD_STEP_WAVES)
rwkv6_gated_delta_step_kernel(GdTensor q, GdTensor k, GdTensor v, const float* __restrict__ g, const void* __restrict__ beta,
                              int beta_dt, float* __restrict__ state, int64_t ssb, int64_t ssh, uint16_t* __restrict__ o,
                              GdShape n, float scale, int64_t waves) {
    constexpr int R = K / 8;
    const int lane = threadIdx.x & 63, grp = lane >> 3;
    const int64_t w = (int64_t)blockIdx.x * GD_STEP_WAVES + (threadIdx.x >> 6);
    if (w >= waves) return;
    const int nb = n.V / 32;
    const int64_t bh = w / nb, b = bh / n.HV;
    const int hv = (int)(bh % n.HV), hk = hv / (n.HV / n.H), c0 = 32 * (int)(w % nb) + 4 * (lane & 7);
    const uint16_t *qp = q.p + b * q.sb + hk * q.sh + R * grp, *kp = k.p + b * k.sb + hk * k.sh + R * grp;
    const uint16_t* vp = v.p + b * v.sb + hv * v.sh + c0;
    float* sp = state + b * ssb + hv * ssh + (int64_t)(R * grp) * n.V + c0;
    f32x4 S[R];
#pragma unroll
    for (int i = 0; i < R; ++i) S[i] = *reinterpret_cast<const f32x4*>(sp + (int64_t)i * n.V);
    auto over_groups = [](f32x4 x) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] += lane_xor8(x[j]);
            const RowSums r = row_sums(x[j]);
            x[j] = r.lo + r.hi;
        }
        return x;
    };
    for (int t = 0; t < n.T; ++t) {
        float kf[R], qf[R], x[4];
#pragma unroll
        for (int i = 0; i < R; i += 8) {
            load8(kp + t * k.st + i, kf + i);
            load8(qp + t * q.st + i, qf + i);
        }
        unpack4(*reinterpret_cast<const uint2*>(vp + t * v.st), x);
        const float a = expf(g[bh * n.T + t]), be = gd_beta(beta, beta_dt, bh * n.T + t);
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
    for (int i = 0; i < R; ++i) *reinterpret_cast<f32x4*>(sp + (int64_t)i * n.V) = S[i];
}

namespace {
inline bool gd_al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int gd_shape(int64_t B, int64_t H, int64_t HV, int64_t T, int64_t K, int64_t V, GdShape* n) {
    if (B < 0 || H < 1 || HV < 1 || T < 0 || K < 1 || V < 1 || HV % H) return RWKV6_ERR_INVALID_ARG;
    if ((K != 64 && K != 128) || V % 64 || V > 512) return RWKV6_ERR_UNSUPPORTED;
    // a launch holds fewer than 2^32 threads, 256 a chunk and head, and 64 a wave of a step
    const int64_t most = ((int64_t)1 << 24) - 1;
    if (HV > most || B > most / HV || T > ((int64_t)1 << 30)) return RWKV6_ERR_UNSUPPORTED;
    const int64_t NC = (T + GD_C - 1) / GD_C;
    if (B * HV * (NC > V / 8 ? NC : V / 8) > most) return RWKV6_ERR_UNSUPPORTED;
    *n = {(int)H, (int)HV, (int)T, (int)NC, (int)V, B * HV};
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
// What the forward leaves for the backward (or uses itself): T, G, and the states and written values.
struct GdSaved {
    size_t T, G, S, N, end;
    GdSaved(const GdShape& n, int64_t K) {
        const size_t chunks = (size_t)n.BH * n.NC;
        T = 0;
        G = T + chunks * 4 * GD_C * GD_C;
        S = G + chunks * 8 * GD_C;
        N = S + chunks * 4 * K * n.V;
        end = N + chunks * 4 * GD_C * n.V;
    }
};
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
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_fwd_kernel<64>), WalkLds<64>::bytes);
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_fwd_kernel<128>), WalkLds<128>::bytes);
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_bwd_kernel<64>), WalkLds<64>::bytes);
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_bwd_kernel<128>), WalkLds<128>::bytes);
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_grads_kernel<64>), GradLds<64>::bytes);
        raise(reinterpret_cast<const void*>(rwkv6_gated_delta_grads_kernel<128>), GradLds<128>::bytes);
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
    return for_bwd ? s.end - s.S : s.S;                   // D and r have the sizes of S and N; T and G
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
    uint16_t *Tm = reinterpret_cast<uint16_t*>(base), *S = saved ? reinterpret_cast<uint16_t*>(base + at.S) : nullptr,
             *N = saved ? reinterpret_cast<uint16_t*>(base + at.N) : nullptr;
    if (T > 0) {
        auto prep = K == 64 ? rwkv6_gated_delta_prep_kernel<64> : rwkv6_gated_delta_prep_kernel<128>;
        hipLaunchKernelGGL(prep, dim3((unsigned)(n.BH * n.NC)), dim3(256), 0, s, kt, g, beta, beta_dtype, G, Tm, n);
    }
    if (T > 0 || hT) {
        auto walk = K == 64 ? rwkv6_gated_delta_fwd_kernel<64> : rwkv6_gated_delta_fwd_kernel<128>;
        hipLaunchKernelGGL(walk, dim3((unsigned)(n.BH * (V / 64))), dim3(256), K == 64 ? WalkLds<64>::bytes : WalkLds<128>::bytes, s,
                           qt, kt, vt, beta, beta_dtype, G, Tm, h0, (uint16_t*)o, hT, S, N, n, scale);
    }
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
                   {workspace, at.end - at.S}},
                  {qs, ks, vs, os, {beta, tok * param_bytes(beta_dtype)}, {dhT, states}, {saved, at.end}}))
        return RWKV6_ERR_INVALID_ARG;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if ((st = gd_limits(s))) return st;
    const char* base = static_cast<const char*>(saved);
    const float2* G = reinterpret_cast<const float2*>(base + at.G);
    const uint16_t *Tm = reinterpret_cast<const uint16_t*>(base), *S = reinterpret_cast<const uint16_t*>(base + at.S),
                   *N = reinterpret_cast<const uint16_t*>(base + at.N);
    uint16_t *D = static_cast<uint16_t*>(workspace), *R = D + (at.N - at.S) / 2;
    if (T > 0 || dh0) {
        auto walk = K == 64 ? rwkv6_gated_delta_bwd_kernel<64> : rwkv6_gated_delta_bwd_kernel<128>;
        hipLaunchKernelGGL(walk, dim3((unsigned)(n.BH * (V / 64))), dim3(256), K == 64 ? WalkLds<64>::bytes : WalkLds<128>::bytes, s,
                           qt, kt, ot, beta, beta_dtype, G, Tm, dhT, (uint16_t*)dv, dh0, D, R, n, scale);
    }
    if (T > 0) {
        auto grads = K == 64 ? rwkv6_gated_delta_grads_kernel<64> : rwkv6_gated_delta_grads_kernel<128>;
        hipLaunchKernelGGL(grads, dim3((unsigned)(B * H * n.NC)), dim3(256), K == 64 ? GradLds<64>::bytes : GradLds<128>::bytes, s,
                           qt, kt, vt, ot, beta, beta_dtype, G, S, N, D, R, (uint16_t*)dq, (uint16_t*)dk, dg, dbeta, n, scale);
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
                       waves);
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}

}  // extern "C"
