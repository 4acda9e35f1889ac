// A block's output gated, scaled and added to the residual stream, and the LayerNorm that the next
// block reads, in one pass for MI355X (gfx950), forward and backward.
//
// Reference: the bias-dropout-adds and LayerNorms between the blocks
// (/root/reference/rwkv_megatron/rwkv6_layer_specs.py:543-548) and the channel mix's sigmoid gate
// before them (:533-536).
//   f = (branch + branch_bias) sigmoid(gate)       s = x + scale f
//   y = (s - mean) rstd gamma + beta               statistics of the unrounded s, fp32 inside
//   dS = ds + rstd (g - mean(g) - xh mean(g xh)),  g = dy gamma, xh = (s - mean) rstd
//   dx = dS, d_branch = scale dS sg, d_gate = scale dS (branch + branch_bias) sg (1 - sg)
//   dgamma = sum_rows dy xh, dbeta = sum_rows dy, d_branch_bias = sum_rows d_branch (fixed order)
// s is rounded once, to x's type, on its way out.  The backward forms it again from the inputs: a
// stored bf16 s would put its rounding, 2^-9 of s, into xh and so into an fp32 dgamma.  Where the norm was taken
// of the stored s (stepwise, below) and there is no gate, it can take that s in place of x and the branch.
// `stepwise` gives the numbers of the operators run one by one instead: the sum with the bias, the
// product with the gate and s are rounded (bf16, bf16, x's type) before the next takes them, y is the
// norm of s as it is stored, and the gradients are rounded at the same places.  The layers and the
// model run that, so that fusing them changed no value of theirs by more than the order of a row's
// sums does.
//
// Bound by memory: bytes an element in bf16 8 forward (10 gated), 10 backward (16 gated).  16384 x 2048
// forward and backward 106 us (kernels 47 + 57, and 4 for the parameters' sums), gated 160 us (56 + 101 +
// 4): 5.7 and 5.4 TB/s of those bytes, where a sum of two 1 GiB tensors reaches 6.1; torch's operators in 32
// bits take 1300 and 1950.  Stepwise, the layers' form: 110 to 114 us (51, 59 from the stored sum, 5), gated 167
// (61 + 103 + 5).  Few rows are bound by the launches (8 rows of 2048: 4 us of kernel, 10 a call).
#include "common.h"
#include "../../include/rwkv6_amd.h"

#define RN_PIECE 512      // channels of a wave: 8 a lane
#define RN_MAX_C 8192
#define RN_MAX_WAVES 8
#define RN_FWD_BLOCKS (1 << 20)
#define RN_BLOCKS 512    // blocks of the backward at most, with one run of rows each (see rn_runs)
#define RN_TURN_BLOCKS 768   // and with runs of RN_TURN steps in turn
#define RN_TURN 4

namespace {

template <bool F32>
__device__ __forceinline__ void raw_f32(const WRaw<F32>& r, float* f) {
    if constexpr (F32) {
        const unsigned w[8] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w, r.q[1].x, r.q[1].y, r.q[1].z, r.q[1].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
    } else {
        unpack8(r.q[0], f);
    }
}
// Eight channels of an output; `nt`: past the caches (see rn_stream).
template <bool F32>
__device__ __forceinline__ void store8_as(void* p, int64_t off, const float* f, bool nt = false) {
    if constexpr (F32) {
        f32x4* q = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p) + off);
        const f32x4 a = {f[0], f[1], f[2], f[3]}, b = {f[4], f[5], f[6], f[7]};
        if (nt) {
            __builtin_nontemporal_store(a, q);
            __builtin_nontemporal_store(b, q + 1);
        } else {
            q[0] = a;
            q[1] = b;
        }
    } else if (nt) {
        store8_nt(reinterpret_cast<uint16_t*>(p) + off, f);
    } else {
        store8(reinterpret_cast<uint16_t*>(p) + off, f);
    }
}
// sigmoid of eight values.  `near`: the reciprocal with a Newton step, as near as the separate operator's
// division; without, the hardware's to 2^-23 (gated forward of 16384 x 2048 56 us, 61 with the step and the other
// roundings of `stepwise`).
__device__ __forceinline__ void sigmoid8(float* g, bool near) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = 1.f + ex2(-RW_L2E * g[j]);
        g[j] = __builtin_amdgcn_rcpf(x[j]);
    }
    if (near)
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = x[j] == INFINITY ? 0.f : fmaf(fmaf(-x[j], g[j], 1.f), g[j], g[j]);
}

// Sum over the row's W waves, the same bits in each: `red` is [waves], one of two arrays that the
// caller alternates, so one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float v, float* red, int W, int wv, int w0) {
    v = wave_sum(v);
    if (W == 1) return v;
    if ((threadIdx.x & 63) == 0) red[wv] = v;
    __syncthreads();
    float t = red[w0];
    for (int w = 1; w < W; ++w) t += red[w0 + w];
    return t;
}

struct RnIn {
    const void* x;
    const uint16_t *branch, *gate;
    const void* cbias;
    int cdt;
    float scale;
    int stepwise;
};
// Eight values rounded to bf16.
__device__ __forceinline__ void round8(float* f) { unpack8(pack8(f), f); }

}  // namespace

// A row is W waves' (512 NV channels each, 8 a lane and piece); a block holds RB = 4 / W rows, one at
// least, and strides over the rows.  The pieces of a row stay in registers.
template <int NV, bool XF, bool GATE, bool CB>
__global__ void __launch_bounds__(64 * RN_MAX_WAVES)
rwkv6_residual_norm_fwd_kernel(RnIn in, const void* __restrict__ gamma, const void* __restrict__ beta, int pdt,
                               float eps, void* __restrict__ s, uint16_t* __restrict__ y,
                               float* __restrict__ mean_out, float* __restrict__ rstd_out, float* __restrict__ gamma_used,
                               int64_t N, int C, int W, int RB, bool nt) {
    __shared__ float red[2][RN_MAX_WAVES];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, gr = wv / W, w = wv - gr * W;
    const float inv = 1.f / (float)C;
    int c[NV];
    float ga[NV][8], be[NV][8], cb[CB ? NV : 1][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        c[i] = 8 * (lane + 64 * (w + W * i));
        if (c[i] < C) {
            load_param8(gamma, pdt, c[i], ga[i]);
            load_param8(beta, pdt, c[i], be[i]);
            if constexpr (CB) load_param8(in.cbias, in.cdt, c[i], cb[i]);
            // for a backward after gamma has changed
            if (gamma_used && blockIdx.x == 0 && gr == 0) store8_as<true>(gamma_used, c[i], ga[i]);
        }
    }
    for (int64_t b0 = (int64_t)blockIdx.x * RB; b0 < N; b0 += (int64_t)gridDim.x * RB) {
        const bool live = b0 + gr < N;
        const int64_t n = live ? b0 + gr : N - 1, row = n * C;
        float v[NV][8];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (c[i] < C) {
                float f[8];
                raw_f32<XF>(w_load<XF>(in.x, row + c[i]), v[i]);
                load8(in.branch + row + c[i], f);
                if constexpr (CB) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] += cb[i][j];
                    if (in.stepwise) round8(f);
                }
                if constexpr (GATE) {
                    float g[8];
                    load8(in.gate + row + c[i], g);
                    sigmoid8(g, in.stepwise);
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] *= g[j];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] *= in.scale;
                if (in.stepwise) round8(f);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] += f[j];
                if (!XF && in.stepwise) round8(v[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += v[i][j];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
            }
        }
        const float mean = row_sum(sum, red[0], W, wv, gr * W) * inv;
        float var = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (c[i] < C)
#pragma unroll
                for (int j = 0; j < 8; ++j) var += (v[i][j] - mean) * (v[i][j] - mean);
        const float rstd = rsqrtf(row_sum(var, red[1], W, wv, gr * W) * inv + eps);
        if (!live) continue;                               // the block's last step: nothing follows
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (c[i] >= C) continue;
            store8_as<XF>(s, row + c[i], v[i], nt);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = (v[i][j] - mean) * rstd * ga[i][j] + be[i][j];
            store8(y + row + c[i], v[i]);
        }
        if (mean_out && lane == 0 && w == 0) {
            mean_out[n] = mean;
            rstd_out[n] = rstd;
        }
    }
}

// Steps of RB rows; block p takes `run` of them, then skips the other blocks' runs.  part[p][CB ? 3 : 2][C] = its sums of dgamma, dbeta
// and d_branch_bias (part null: none).  ds null: zero.  db null: d_branch equals dx, not stored twice.  SUM: x is the
// sum s as the stepwise forward stored it, what its norm was taken of, and the branch is not read.
template <int NV, bool XF, bool GATE, bool CB, bool SUM>
__global__ void __launch_bounds__(64 * RN_MAX_WAVES)
rwkv6_residual_norm_bwd_kernel(RnIn in, const void* __restrict__ gamma, int pdt, const float* __restrict__ mean_in,
                               const float* __restrict__ rstd_in, const void* __restrict__ ds,
                               const uint16_t* __restrict__ dy, void* __restrict__ dx, uint16_t* __restrict__ db,
                               uint16_t* __restrict__ dg, float* __restrict__ part, int64_t N, int C, int W, int RB, int run,
                               bool nt) {
    extern __shared__ __attribute__((aligned(16))) float rn_acc[];            // [CB ? 3 : 2][C]
    __shared__ float2 red[2][RN_MAX_WAVES];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, gr = wv / W, w = wv - gr * W;
    const float inv = 1.f / (float)C;
    int c[NV];
    float ga[NV][8], cb[CB ? NV : 1][8], ag[NV][8], ab[NV][8], ac[CB ? NV : 1][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        c[i] = 8 * (lane + 64 * (w + W * i));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            ga[i][j] = ag[i][j] = ab[i][j] = 0.f;
            if constexpr (CB) cb[i][j] = ac[i][j] = 0.f;
        }
        if (c[i] < C) {
            load_param8(gamma, pdt, c[i], ga[i]);
            if constexpr (CB && !SUM) load_param8(in.cbias, in.cdt, c[i], cb[i]);
        }
    }
    int turn = 0;
    const int64_t skip = ((int64_t)gridDim.x - 1) * run * RB;
    int step = 0;
    for (int64_t b0 = (int64_t)blockIdx.x * run * RB; b0 < N; turn ^= 1) {
        const bool live = b0 + gr < N;
        const int64_t n = live ? b0 + gr : N - 1, row = n * C;
        b0 += RB;
        if (++step == run) {
            step = 0;
            b0 += skip;
        }
        const float mean = mean_in[n], rstd = rstd_in[n];
        float xh[NV][8], g[NV][8], f[NV][8], sg[NV][8], dS[NV][8];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) xh[i][j] = g[i][j] = f[i][j] = sg[i][j] = dS[i][j] = 0.f;
            if (c[i] >= C) continue;
            raw_f32<XF>(w_load<XF>(in.x, row + c[i]), xh[i]);
            if constexpr (!SUM) load8(in.branch + row + c[i], f[i]);
            if constexpr (GATE) load8(in.gate + row + c[i], sg[i]);
            load8(dy + row + c[i], g[i]);
            if (ds) raw_f32<XF>(w_load<XF>(ds, row + c[i]), dS[i]);
            float t[8];
            if constexpr (SUM) {
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = xh[i][j];
            } else {
                if constexpr (CB) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[i][j] += cb[i][j];
                    if (in.stepwise) round8(f[i]);
                }
                if constexpr (GATE) sigmoid8(sg[i], in.stepwise);
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = (GATE ? f[i][j] * sg[i][j] : f[i][j]) * in.scale;
                if (in.stepwise) round8(t);
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] += xh[i][j];
                if (!XF && in.stepwise) round8(t);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                xh[i][j] = (t[j] - mean) * rstd;
                if (live) {
                    ag[i][j] += g[i][j] * xh[i][j];
                    ab[i][j] += g[i][j];
                }
                s1 += g[i][j] * ga[i][j];
                s2 += g[i][j] * ga[i][j] * xh[i][j];
            }
        }
        s1 = wave_sum(s1);
        s2 = wave_sum(s2);
        if (W > 1) {
            if (lane == 0) red[turn][wv] = make_float2(s1, s2);
            __syncthreads();
            s1 = s2 = 0.f;
            for (int k = 0; k < W; ++k) {
                const float2 r = red[turn][gr * W + k];
                s1 += r.x;
                s2 += r.y;
            }
        }
        s1 *= inv;
        s2 *= inv;
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (c[i] >= C) continue;
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = rstd * (g[i][j] * ga[i][j] - s1 - xh[i][j] * s2);
            if (!XF && in.stepwise) round8(e);
#pragma unroll
            for (int j = 0; j < 8; ++j) dS[i][j] += e[j];
            if (!XF && in.stepwise) round8(dS[i]);
            store8_as<XF>(dx, row + c[i], dS[i], nt);
            if (!db) continue;
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) dS[i][j] *= in.scale;
            if (in.stepwise) round8(dS[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = GATE ? dS[i][j] * sg[i][j] : dS[i][j];
            if constexpr (CB) {
                if (in.stepwise) round8(o);
#pragma unroll
                for (int j = 0; j < 8; ++j) ac[i][j] += o[j];
            }
            store8_as<false>(db, row + c[i], o, nt);
            if constexpr (GATE) {
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = dS[i][j] * f[i][j] * sg[i][j] * (1.f - sg[i][j]);
                store8_as<false>(dg, row + c[i], o, nt);
            }
        }
    }
    if (!part) return;
    constexpr int K = CB ? 3 : 2;
    float* out = part + (int64_t)blockIdx.x * K * C;
    if (RB == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (c[i] >= C) continue;
            store8_as<true>(out, c[i], ag[i]);
            store8_as<true>(out, C + c[i], ab[i]);
            if constexpr (CB) store8_as<true>(out, 2 * C + c[i], ac[i]);
        }
        return;
    }
    // the row groups' sums, in order (rows of up to 1024 channels)
    for (int r = 0; r < RB; ++r) {
        if (gr == r)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (c[i] >= C) continue;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    rn_acc[c[i] + j] = (r ? rn_acc[c[i] + j] : 0.f) + ag[i][j];
                    rn_acc[C + c[i] + j] = (r ? rn_acc[C + c[i] + j] : 0.f) + ab[i][j];
                    if constexpr (CB) rn_acc[2 * C + c[i] + j] = (r ? rn_acc[2 * C + c[i] + j] : 0.f) + ac[i][j];
                }
            }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < K * C; i += blockDim.x) out[i] = rn_acc[i];
}

// The parameters' gradients: column m of part [P][M] summed in a fixed order, 32 columns a block, 32
// row lanes that take every 32nd row and are then added in order.  P = 0 writes zeros.
__global__ void __launch_bounds__(1024)
rwkv6_residual_norm_sums_kernel(const float* __restrict__ part, int P, int M, int C, void* __restrict__ dgamma,
                                void* __restrict__ dbeta, int pdt, void* __restrict__ dcb, int cdt) {
    __shared__ float acc[32][33];
    const int q = threadIdx.x >> 5, l = threadIdx.x & 31, m = blockIdx.x * 32 + l, mc = m < M ? m : M - 1;
    float t = 0.f;
    for (int p0 = q; p0 < P; p0 += 32 * 8) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = part[(int64_t)min(p0 + 32 * k, P - 1) * M + mc];
#pragma unroll
        for (int k = 0; k < 8; ++k) t += p0 + 32 * k < P ? v[k] : 0.f;
    }
    acc[q][l] = t;
    __syncthreads();
    if (q || m >= M) return;
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += acc[k][l];
    const int which = m / C, i = m - which * C, dt = which == 2 ? cdt : pdt;
    void* dst = which == 0 ? dgamma : which == 1 ? dbeta : dcb;
    if (dt == RWKV6_BF16) reinterpret_cast<uint16_t*>(dst)[i] = f2bf(t);
    else reinterpret_cast<float*>(dst)[i] = t;
}

namespace {
inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool dt_ok(int dt) { return dt == RWKV6_F32 || dt == RWKV6_BF16; }
inline int rn_check(int64_t N, int64_t C) {
    if (N < 0 || C < 1) return RWKV6_ERR_INVALID_ARG;
    // rows: 2^40 elements at most, so that byte offsets and spans stay far inside 64 bits
    if (C % 8 || C > RN_MAX_C || N > ((int64_t)1 << 40) / C) return RWKV6_ERR_UNSUPPORTED;
    return RWKV6_OK;
}
struct RnShape {
    int NV, W, RB;
};
inline RnShape rn_shape(int64_t C) {
    const int NV = C > RN_PIECE * RN_MAX_WAVES ? 2 : 1, W = (int)((C + RN_PIECE * NV - 1) / (RN_PIECE * NV));
    return {NV, W, W >= 4 ? 1 : 4 / W};
}
// Whether the outputs but y are stored past the caches: where the call's tensors do not fit the 256 MB of
// the last one anyway.  Kept in it, they push out what the call still reads: 16384 x 2048 bf16, us, cached
// and streamed: backward 75 and 57, gated 103 and 100, gated forward 64 and 57.  y is the next kernel's
// input: streamed too, the forward and backward one after the other took 109 instead of 112 us, but a training step of
// the 1.6B shape 168.2 instead of 167.5 ms (three runs each).  2049 x 4096, both ways the same.
inline bool rn_stream(int64_t N, int64_t C) { return N * C >= (int64_t)1 << 24; }
// The backward's blocks, each with two steps or more, and the steps that a block takes in a row before it
// leaves as many to each other block.  Without a gate and with work for them 768 blocks (three a CU) take
// runs of 4 in turn, so that the rows in work lie together; otherwise 512 blocks take one run each.  us, in
// turn and in one run: 8192 x 2048 31 and 36, 16384 x 2048 57 to 68 and 66 to 68 (by where the tensors lie),
// 32768 x 2048 125 and 133; gated 57 and 52, 100 to 114 and 100 to 108, 210 and 212.
struct RnRuns {
    int64_t blocks;
    int run;
};
inline RnRuns rn_runs(int64_t N, int RB, bool gate) {
    const int64_t steps = (N + RB - 1) / RB, half = (steps + 1) / 2;
    if (!gate && steps >= 2 * RN_TURN * RN_TURN_BLOCKS) return {RN_TURN_BLOCKS, RN_TURN};
    const int64_t b = half < 1 ? 1 : half < RN_BLOCKS ? half : RN_BLOCKS, run = (steps + b - 1) / b;
    return {b, (int)(run < 1 ? 1 : run)};
}
int rn_fwd(const void* x, int x_dtype, const void* branch, const void* branch_bias, int bias_dtype, const void* gate,
           float scale, int stepwise, const void* gamma, const void* beta, int param_dtype, float eps, void* s, void* y,
           float* mean, float* rstd, float* gamma_used, int64_t N, int64_t C, void* stream) {
    const int st = rn_check(N, C);
    if (st) return st;
    if (!dt_ok(x_dtype) || !dt_ok(param_dtype) || (branch_bias && !dt_ok(bias_dtype)) || (!mean != !rstd))
        return RWKV6_ERR_INVALID_ARG;
    if (N == 0) return RWKV6_OK;
    if (!x || !branch || !gamma || !beta || !s || !y) return RWKV6_ERR_INVALID_ARG;
    for (const void* p : {x, branch, branch_bias, gate, gamma, beta, (const void*)s, (const void*)y, (const void*)gamma_used})
        if (!al16(p)) return RWKV6_ERR_ALIGNMENT;
    const size_t act = (size_t)(N * C) * 2, xs = (size_t)(N * C) * param_bytes(x_dtype), st4 = (size_t)N * 4;
    const size_t par = (size_t)C * param_bytes(param_dtype);
    if (any_alias({{s, xs}, {y, act}, {mean, st4}, {rstd, st4}, {gamma_used, (size_t)C * 4}},
                  {{x, xs}, {branch, act}, {branch_bias, (size_t)C * param_bytes(bias_dtype)}, {gate, act}, {gamma, par}, {beta, par}}))
        return RWKV6_ERR_INVALID_ARG;
    const RnShape h = rn_shape(C);
    const bool xf = x_dtype == RWKV6_F32, gt = gate != nullptr, cb = branch_bias != nullptr;
#define RN_CB(NV, X, G) (cb ? rwkv6_residual_norm_fwd_kernel<NV, X, G, true> : rwkv6_residual_norm_fwd_kernel<NV, X, G, false>)
#define RN_PICK(NV) (xf ? (gt ? RN_CB(NV, true, true) : RN_CB(NV, true, false)) : (gt ? RN_CB(NV, false, true) : RN_CB(NV, false, false)))
    auto k = h.NV == 1 ? RN_PICK(1) : RN_PICK(2);
#undef RN_PICK
#undef RN_CB
    const int64_t blocks = (N + h.RB - 1) / h.RB;
    hipLaunchKernelGGL(k, dim3((unsigned)(blocks < RN_FWD_BLOCKS ? blocks : RN_FWD_BLOCKS)), dim3(64 * h.W * h.RB), 0,
                       reinterpret_cast<hipStream_t>(stream),
                       RnIn{x, (const uint16_t*)branch, (const uint16_t*)gate, branch_bias, bias_dtype, scale, stepwise}, gamma, beta,
                       param_dtype, eps, s, (uint16_t*)y, mean, rstd, gamma_used, N, (int)C, h.W, h.RB, rn_stream(N, C));
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}
}  // namespace

extern "C" {

int rwkv6_residual_norm_fwd(const void* x, int x_dtype, const void* branch, const void* branch_bias, int bias_dtype,
                            const void* gate, float scale, int stepwise, const void* gamma, const void* beta,
                            int param_dtype, float eps, void* s, void* y, float* mean, float* rstd, int64_t N, int64_t C, void* stream) {
    return rn_fwd(x, x_dtype, branch, branch_bias, bias_dtype, gate, scale, stepwise, gamma, beta, param_dtype, eps, s, y, mean, rstd,
                  nullptr, N, C, stream);
}

int rwkv6_residual_norm_train_fwd(const void* x, int x_dtype, const void* branch, const void* branch_bias, int bias_dtype,
                                  const void* gate, float scale, int stepwise, const void* gamma, const void* beta,
                                  int param_dtype, float eps, void* s, void* y, float* mean, float* rstd,
                                  float* gamma_used, int64_t N, int64_t C, void* stream) {
    return rn_fwd(x, x_dtype, branch, branch_bias, bias_dtype, gate, scale, stepwise, gamma, beta, param_dtype, eps, s, y, mean, rstd,
                  gamma_used, N, C, stream);
}

size_t rwkv6_residual_norm_bwd_workspace_bytes(int64_t N, int64_t C) {
    if (rn_check(N, C)) return 0;
    return (size_t)(rn_runs(N, rn_shape(C).RB, false).blocks * 3 * C) * sizeof(float);
}

int rwkv6_residual_norm_bwd(const void* x, int x_dtype, const void* branch, const void* branch_bias, int bias_dtype,
                            const void* gate, float scale, int stepwise, const void* gamma, int gamma_dtype, const float* mean,
                            const float* rstd, const void* ds, const void* dy, void* dx, void* d_branch, void* d_gate,
                            void* dgamma, void* dbeta, int param_dtype, void* d_branch_bias, void* workspace, int64_t N,
                            int64_t C, void* stream) {
    const int st = rn_check(N, C);
    if (st) return st;
    if (!dt_ok(x_dtype) || !dt_ok(gamma_dtype) || !dt_ok(param_dtype) || (branch_bias && !dt_ok(bias_dtype)))
        return RWKV6_ERR_INVALID_ARG;
    const bool sums = dgamma || dbeta, xf = x_dtype == RWKV6_F32, gt = gate != nullptr, cb = branch_bias != nullptr;
    // d_branch is dx itself, and not written, only where the two are the same numbers
    if (N > 0 && !d_branch && (gt || cb || xf || scale != 1.f)) return RWKV6_ERR_INVALID_ARG;
    // no branch: x is the sum that the stepwise forward stored
    if (!gamma || (!dgamma != !dbeta) || (!d_branch_bias != !(cb && sums)) || (sums && !workspace) ||
        (N > 0 && (!x || (!branch && (!stepwise || gt)) || !mean || !rstd || !dy || !dx || !d_gate != !gt)))
        return RWKV6_ERR_INVALID_ARG;
    for (const void* p : {x, branch, branch_bias, gate, gamma, ds, dy, (const void*)dx, (const void*)d_branch,
                          (const void*)d_gate, (const void*)workspace})
        if (!al16(p)) return RWKV6_ERR_ALIGNMENT;
    const size_t act = (size_t)(N * C) * 2, xs = (size_t)(N * C) * param_bytes(x_dtype), st4 = (size_t)N * 4;
    const size_t par = (size_t)C * param_bytes(param_dtype), cbs = cb ? (size_t)C * param_bytes(bias_dtype) : 0;
    if (any_alias({{dx, xs}, {d_branch, act}, {d_gate, act}, {dgamma, par}, {dbeta, par}, {d_branch_bias, cbs},
                   {sums ? workspace : nullptr, rwkv6_residual_norm_bwd_workspace_bytes(N, C)}},
                  {{x, xs}, {branch, act}, {branch_bias, cbs}, {gate, act}, {gamma, (size_t)C * param_bytes(gamma_dtype)},
                   {mean, st4}, {rstd, st4}, {ds, xs}, {dy, act}}))
        return RWKV6_ERR_INVALID_ARG;
    hipStream_t stm = reinterpret_cast<hipStream_t>(stream);
    const RnShape h = rn_shape(C);
    const RnRuns r = rn_runs(N, h.RB, gt);
    const int64_t M = (cb ? 3 : 2) * C;
    float* part = sums ? (float*)workspace : nullptr;
    if (N > 0) {
#define RN_CB(NV, X, G, S) (cb ? rwkv6_residual_norm_bwd_kernel<NV, X, G, true, S> : rwkv6_residual_norm_bwd_kernel<NV, X, G, false, S>)
#define RN_GATE(NV, X) (gt ? RN_CB(NV, X, true, false) : branch ? RN_CB(NV, X, false, false) : RN_CB(NV, X, false, true))
#define RN_PICK(NV) (xf ? RN_GATE(NV, true) : RN_GATE(NV, false))
        auto k = h.NV == 1 ? RN_PICK(1) : RN_PICK(2);
#undef RN_PICK
#undef RN_GATE
#undef RN_CB
        hipLaunchKernelGGL(k, dim3((unsigned)r.blocks), dim3(64 * h.W * h.RB), sums && h.RB > 1 ? (size_t)M * 4 : 0, stm,
                           RnIn{x, (const uint16_t*)branch, (const uint16_t*)gate, branch_bias, bias_dtype, scale, stepwise}, gamma,
                           gamma_dtype, mean, rstd, ds, (const uint16_t*)dy, dx, (uint16_t*)d_branch, (uint16_t*)d_gate, part,
                           N, (int)C, h.W, h.RB, r.run, rn_stream(N, C));
    }
    if (sums)
        hipLaunchKernelGGL(rwkv6_residual_norm_sums_kernel, dim3((unsigned)((M + 31) / 32)), dim3(1024), 0, stm, part,
                           N > 0 ? (int)r.blocks : 0, (int)M, (int)C, dgamma, dbeta, param_dtype, d_branch_bias, bias_dtype);
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}

}  // extern "C"
