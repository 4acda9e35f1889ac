// An AdamW step over many tensors at once for MI355X (gfx950), states in 32 or 8 bits, clipped by the
// norm of all gradients.
//
// Reference: the optimizer step after the backward (/root/reference/example_config.yaml:199-221: AdamW
// with weight decay and a gradient clip; Megatron's training loop runs it, pretrain_rwkv6.py:281-286).
//   norm = sqrt(sum g^2) over all tensors (64-bit sums),  c = min(1, max_norm / (norm + 1e-6))
//   g' = c g;  m' = b1 m + (1 - b1) g';  v' = b2 v + (1 - b2) g'^2;  t = step + 1
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
// Everything is elementwise in 32 bits with one rounding of p at the end; p' takes the unrounded m' and
// v' also where the states are kept in 8 bits.
//
// States in 8 bits: a block of 256 consecutive elements of a tensor holds float8 (e4m3) codes and one
// fp32 scale, the block's largest magnitude over 448; m as code * scale and v by its root, v = (code *
// scale)^2, which doubles the range in the exponent (a code reaches from 448 to 2^-9: 2^-36 of the
// block's largest v).  Values that are not finite do not enter the scale and become NaN codes, so that
// they spoil no other element of the block; a block below 2^-118 stores zeros.
// Codes are rounded to the nearest, or (`stochastic`) up or down so that m and v, not its root, come out
// right on average.  A run of steps wants that: a step moves the root of v by (1 - b2) / 2 of it at most
// downwards, far less than half a code (3 to 6 %), so that the nearest code is the old one step after step
// and an element's v moves with its block's largest alone.  4000 steps of N(0, 1) gradients at b2 = 0.995
// (test_optim_rounding_gpu.py has the like): where half a block's fall to a tenth, their root ends 10.5 times that of
// 32 bits with the nearest codes, and 0.77 to 1.28 times it (5th to 95th percentile) on average right.
// The choice is a hash of the step, the element and its gradient, so that equal calls give equal bits.
//
// The tensors' addresses travel in the kernels' arguments, AW_T tensors a launch: nothing is copied to
// the device or kept between calls, and a captured call replays with the addresses it was made with.
// The step count and the norm stay on the device, for the same reason.
//
// Bound by memory: bytes a parameter 22 (bf16 p and g, fp32 states), 28 (all fp32), 10 and 16 with
// 8-bit states, and once more the gradient where it is clipped.  Four layers of 2048 channels (218 M
// bf16 parameters in 92 tensors): norm 90 us (4.9 TB/s), step 883 us (5.4 TB/s), with 8-bit states 401 us
// (5.5 TB/s), with codes right on average 465 us, whose arithmetic the bytes no longer hide (55 M fp32 parameters
// 160 us either way); two layers of 512 (7.3 M fp32): 7 + 5 + 34 us, the 5 the one block that forms the norm and
// the coefficients.  A sum of two 1 GiB tensors reaches 6.1 TB/s.  torch's operators in 32 bits on the same
// parameters as one tensor take 8.0 ms, 11.7 ms and 313 us.  Tried and left: the step's loads past the
// caches (499 us instead of 457 for 109 M parameters) and its stores (the same), the norm's sums of eight
// squares in 32 bits (the same), the tensors in reverse so that the norm's last ones are still cached
// (the same).
#include "common.h"
#include "../../include/rwkv6_amd.h"

#include <algorithm>
#include <vector>

#define AW_THR 256
#define AW_STEP (8 * AW_THR)    // elements a block takes at once
#define AW_PARTS 8192           // blocks of the norm's sums, at about; below 50 M elements some of them have no run
#define AW_AHEAD 4              // steps of the norm's loads in flight
#define AW_RUN (AW_AHEAD * AW_STEP)
#define AW_T 60                 // tensors a launch: the arguments stay below 4 KB
#define AW_BLK 256              // elements under one 8-bit scale: 32 lanes of 8
#define AW_MAX ((int64_t)1 << 37)   // elements a call
#define AW_BLOCKS ((int64_t)1 << 23)    // blocks a launch, at about: fewer than 2^32 threads
#define AW_F8_MAX 448.f
#define AW_F8_BELOW 447.99988f  // 448 (1 - 2^-22): times a reciprocal and the value itself, below 448 after three roundings
#define AW_TINY 0x1p-118f

namespace {

struct NormTable {
    const void* g[AW_T];
    int64_t n[AW_T];
    int first[AW_T];            // first block of the tensor in this launch
    int dt[AW_T];
    int count, base;            // base: blocks of the launches before
};
struct StepTable {
    void* p[AW_T];
    const void* g[AW_T];
    void *m[AW_T], *v[AW_T];
    float *ms[AW_T], *vs[AW_T];
    int64_t n[AW_T];
    int first[AW_T];
    int dt[AW_T];               // the parameter's type, and the gradient's 8 bits up
    int count;
};
static_assert(sizeof(StepTable) <= 4000 && sizeof(NormTable) <= 4000, "kernel arguments");
// The tables hold no element below 4 bytes.  A uniform index into them becomes scalar loads, whose address
// is a sum of which the hardware drops the two low bits of every term; with byte arrays beside the pointers
// the compiler (ROCm 7.2) shares the byte address between them and forms 8 k as k + 7 k.

// The launch's tensor that holds block b: the last one whose first block is not after it.
__device__ __forceinline__ int aw_find(const int* first, int count, int b) {
    const int lane = threadIdx.x & 63;
    const bool at = lane < count && first[lane < count ? lane : 0] <= b;
    return __popcll(__ballot(at)) - 1;
}

// Eight elements from i of a tensor of n: as vectors where they are all there and aligned (`vec`), else
// one by one, zeros past the end.
__device__ __forceinline__ void aw_load8(const void* p, int dt, int64_t i, int64_t n, bool vec, float* f) {
    if (vec && i + 8 <= n) {
        if (dt == RWKV6_BF16) {
            load8(reinterpret_cast<const uint16_t*>(p) + i, f);
        } else {
            const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
            const float4 a = q[0], b = q[1];
            f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
            f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            f[j] = 0.f;
            if (i + j < n)
                f[j] = dt == RWKV6_BF16 ? bf2f(reinterpret_cast<const uint16_t*>(p)[i + j])
                                        : reinterpret_cast<const float*>(p)[i + j];
        }
    }
}
// Eight aligned elements past the caches.
__device__ __forceinline__ void aw_load8_nt(const void* p, int dt, int64_t i, float* f) {
    if (dt == RWKV6_BF16) {
        const u32x4_t q = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(reinterpret_cast<const uint16_t*>(p) + i));
        unpack8(make_uint4(q.x, q.y, q.z, q.w), f);
    } else {
        const f32x4* q = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(p) + i);
        const f32x4 a = __builtin_nontemporal_load(q), b = __builtin_nontemporal_load(q + 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = a[j];
            f[4 + j] = b[j];
        }
    }
}
__device__ __forceinline__ void aw_store8(void* p, int dt, int64_t i, int64_t n, bool vec, const float* f) {
    if (vec && i + 8 <= n) {
        if (dt == RWKV6_BF16) {
            store8(reinterpret_cast<uint16_t*>(p) + i, f);
        } else {
            float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
            q[0] = make_float4(f[0], f[1], f[2], f[3]);
            q[1] = make_float4(f[4], f[5], f[6], f[7]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j < n) {
                if (dt == RWKV6_BF16) reinterpret_cast<uint16_t*>(p)[i + j] = f2bf(f[j]);
                else reinterpret_cast<float*>(p)[i + j] = f[j];
            }
    }
}
__device__ __forceinline__ bool aw_al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Eight float8 codes.
__device__ __forceinline__ uint2 aw_codes_load(const void* p, int64_t i, int64_t n, bool vec) {
    const uint8_t* b = reinterpret_cast<const uint8_t*>(p) + i;
    if (vec && i + 8 <= n) return *reinterpret_cast<const uint2*>(b);
    uint2 q = make_uint2(0u, 0u);
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (i + j < n) (j < 4 ? q.x : q.y) |= (unsigned)b[j] << (8 * (j & 3));
    return q;
}
__device__ __forceinline__ void aw_codes_store(void* p, int64_t i, int64_t n, bool vec, uint2 q) {
    uint8_t* b = reinterpret_cast<uint8_t*>(p) + i;
    if (vec && i + 8 <= n) {
        *reinterpret_cast<uint2*>(b) = q;
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (i + j < n) b[j] = (uint8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
}
__device__ __forceinline__ void aw_decode(uint2 q, float s, float* f) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, true);
    const f32x2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, true);
    f[0] = a[0] * s; f[1] = a[1] * s; f[2] = b[0] * s; f[3] = b[1] * s;
    f[4] = c[0] * s; f[5] = c[1] * s; f[6] = d[0] * s; f[7] = d[1] * s;
}
__device__ __forceinline__ uint2 aw_encode(const float* f, float inv) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inv, f[1] * inv, 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * inv, f[3] * inv, lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * inv, f[5] * inv, 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * inv, f[7] * inv, hi, true);
    return make_uint2((unsigned)lo, (unsigned)hi);
}
// Largest finite magnitude of the 8 values of each of 32 lanes.
__device__ __forceinline__ float aw_top(const float* f) {
    float t = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float a = fabsf(f[j]);
        t = fmaxf(t, a < INFINITY ? a : 0.f);
    }
    t = fmaxf(t, lane_xor1(t));
    t = fmaxf(t, lane_xor2(t));
    t = fmaxf(t, dpp_mov<0x141>(t));              // the other quad of 8 lanes
    t = fmaxf(t, dpp_mov<0x140>(t));              // the other 8 of 16
    return fmaxf(t, lane_xor_swz<16>(t));
}
// What the random bits of eight elements start from: a multiply and shift hash, every bit of which depends on
// every bit of the step, the element's place and the gradient.
__device__ __forceinline__ uint32_t aw_seed(float t, int64_t i, float g) {
    uint32_t h = (uint32_t)(i >> 3) * 0x9E3779B1u ^ (uint32_t)(i >> 35) * 0xC2B2AE3Du ^ __float_as_uint(t) * 0x85EBCA77u ^ __float_as_uint(g);
    h = (h ^ h >> 16) * 0x7FEB352Du;
    h = (h ^ h >> 15) * 0x846CA68Bu;
    return h ^ h >> 16;
}
// Eight codes each of m and of the roots of v over their scales, rounded up or down to one of the two e4m3
// numbers lo < hi around a value a: m up with probability (a - lo) / (hi - lo), a right on average, a root with
// (a^2 - lo^2) / (hi^2 - lo^2), its square right on average.  The values lie below 448 (see AW_F8_BELOW); one
// that is not finite becomes NaN.  Below 2^-6 the numbers lie 2^-9 apart, as from 2^-6 to 2^-5: `off` moves a
// value there.  An e4m3 number has the low 20 bits of a float zero.  32 random bits an element, m's from the
// top, the root's from the 23rd.
__device__ __forceinline__ void aw_encode_either(const float* m, float im, const float* root, float iv, uint32_t h, uint2* cm,
                                                 uint2* cv) {
    float qm[8], qv[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        h += 0x9E3779B9u;
        const uint32_t r = __umul24(h ^ h >> 15, 0xD1D5F3u);
        {
            // the carry of the random bits below the code's last one
            const float a = fabsf(m[j]) * im, off = a < 0x1p-6f ? 0x1p-6f : 0.f;
            qm[j] = copysignf(__uint_as_float((__float_as_uint(a + off) + (r >> 12)) & 0xfff00000u) - off, m[j]);
        }
        {
            const float a = root[j] * iv, off = a < 0x1p-6f ? 0x1p-6f : 0.f;
            const uint32_t b = __float_as_uint(a + off) & 0xfff00000u;
            const float lo = __uint_as_float(b) - off, hi = __uint_as_float(b + 0x100000u) - off;
            const float low2 = lo * lo, all = fmaf(hi, hi, -low2);
            const float u1 = __uint_as_float((r & 0x7fffffu) | 0x3f800000u);          // 1 + u
            qv[j] = fmaf(u1, all, -all) < fmaf(a, a, -low2) ? hi : lo;
        }
    }
    *cm = aw_encode(qm, 1.f);
    *cv = aw_encode(qv, 1.f);
}
struct Coef {
    float clip, keep, lr, rbc2;                   // c, 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

}  // namespace

// Sums of squares: a tensor's blocks take its runs of AW_RUN elements in turn, so that together they
// sweep it; part[base + block].
__global__ void __launch_bounds__(AW_THR)
rwkv6_grad_square_sums_kernel(const NormTable tab, bool nt, double* __restrict__ part) {
    __shared__ double red[AW_THR / 64];
    const int k = aw_find(tab.first, tab.count, blockIdx.x);
    const int64_t n = tab.n[k];
    const int j0 = (int)blockIdx.x - tab.first[k];
    const int64_t stride = (int64_t)((k + 1 < tab.count ? tab.first[k + 1] : (int)gridDim.x) - tab.first[k]) * AW_RUN;
    const void* g = tab.g[k];
    const int dt = tab.dt[k];
    const bool vec = aw_al16(g);
    double sum[2] = {0., 0.};
    for (int64_t i = (int64_t)j0 * AW_RUN + 8 * threadIdx.x; i < n; i += stride) {
        float f[AW_AHEAD][8];
        if (vec && i + 8 + (AW_AHEAD - 1) * AW_STEP <= n) {
#pragma unroll
            for (int u = 0; u < AW_AHEAD; ++u) {
                if (nt) aw_load8_nt(g, dt, i + u * AW_STEP, f[u]);
                else aw_load8(g, dt, i + u * AW_STEP, n, true, f[u]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < AW_AHEAD; ++u) aw_load8(g, dt, i + u * AW_STEP, n, vec, f[u]);
        }
#pragma unroll
        for (int u = 0; u < AW_AHEAD; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j & 1] = fma((double)f[u][j], (double)f[u][j], sum[j & 1]);
    }
    double acc = sum[0] + sum[1];
#pragma unroll
    for (int o = 1; o < 64; o *= 2) acc += __shfl_xor(acc, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) part[tab.base + blockIdx.x] = ((red[0] + red[1]) + red[2]) + red[3];
}

// One block: the norm from the partial sums (none: c = 1), the step counted, the coefficients.
__global__ void __launch_bounds__(1024)
rwkv6_adamw_coef_kernel(const double* __restrict__ part, int P, float max_norm, float* __restrict__ norm_out,
                        float* __restrict__ step, const float* __restrict__ lr_dev, double lr, double log_b1,
                        double log_b2, double wd, Coef* __restrict__ coef) {
    __shared__ double red[16];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const bool first = wv == 0 && coef;
    // 1 - b^t for b1 in the even lanes and b2 in the odd ones, while the sums come in
    const float t = first ? step[0] + 1.f : 1.f;
    const double bc = first ? -expm1((double)t * (lane & 1 ? log_b2 : log_b1)) : 1.;
    if (first && lr_dev) lr = (double)lr_dev[0];
    double acc = 0.;
    for (int i = threadIdx.x; i < P; i += 4 * 1024) {
        double v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = part[min(i + k * 1024, P - 1)];
#pragma unroll
        for (int k = 0; k < 4; ++k) acc += i + k * 1024 < P ? v[k] : 0.;
    }
#pragma unroll
    for (int o = 1; o < 64; o *= 2) acc += __shfl_xor(acc, o);
    if (lane == 0) red[wv] = acc;
    __syncthreads();
    if (wv) return;
    acc = lane < 16 ? red[lane] : 0.;
#pragma unroll
    for (int o = 1; o < 16; o *= 2) acc += __shfl_xor(acc, o);
    const double bc2 = __shfl_xor(bc, 1);
    if (lane) return;
    const float norm = (float)sqrt(acc), r = max_norm / (norm + 1e-6f);
    if (norm_out) norm_out[0] = norm;
    if (!coef) return;
    step[0] = t;
    // a NaN norm stays one: the whole update is NaN, as clipped gradients would be
    coef[0] = Coef{part && !(r > 1.f) ? r : 1.f, (float)(1. - lr * wd), (float)(lr / bc), (float)(1. / sqrt(bc2))};
}

// Block b: `per` elements of a tensor, 8 a thread and step.  32 lanes hold the 256 elements of one scale.
// SR: codes rounded up or down at random, right on average.
template <bool F8, bool SR>
__global__ void __launch_bounds__(AW_THR)
rwkv6_adamw_step_kernel(const StepTable tab, const Coef* __restrict__ coef, int64_t per, float b1, float ob1, float b2,
                        float ob2, float eps, const float* __restrict__ step) {
    const int k = aw_find(tab.first, tab.count, blockIdx.x);
    const Coef c = coef[0];
    const float t = SR ? step[0] : 0.f;
    const int64_t n = tab.n[k], i0 = (int64_t)((int)blockIdx.x - tab.first[k]) * per, i1 = min(n, i0 + per);
    void *p = tab.p[k], *m = tab.m[k], *v = tab.v[k];
    const void* g = tab.g[k];
    const int pt = tab.dt[k] & 0xff, gt = tab.dt[k] >> 8;
    const bool vec = aw_al16(p) && aw_al16(g) && aw_al16(m) && aw_al16(v);
    // all lanes of a scale's 32 step together, up to the end of its block
    for (int64_t i = i0 + 8 * threadIdx.x; (i & ~(int64_t)(AW_BLK - 1)) < i1; i += AW_STEP) {
        float pf[8], gf[8], mf[8], vf[8];
        aw_load8(p, pt, i, n, vec, pf);
        aw_load8(g, gt, i, n, vec, gf);
        float* ms = nullptr;
        float* vs = nullptr;
        if constexpr (F8) {
            ms = tab.ms[k] + i / AW_BLK;
            vs = tab.vs[k] + i / AW_BLK;
            aw_decode(aw_codes_load(m, i, n, vec), ms[0], mf);
            aw_decode(aw_codes_load(v, i, n, vec), vs[0], vf);
#pragma unroll
            for (int j = 0; j < 8; ++j) vf[j] *= vf[j];
        } else {
            aw_load8(m, RWKV6_F32, i, n, vec, mf);
            aw_load8(v, RWKV6_F32, i, n, vec, vf);
        }
        float root[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // each product and sum rounded, so that a state's value, and the code it falls on, is the
            // formula's in 32 bits and not one of its contractions
#pragma clang fp contract(off)
            const float gc = gf[j] * c.clip;
            mf[j] = mf[j] * b1 + gc * ob1;
            vf[j] = vf[j] * b2 + (gc * gc) * ob2;
            root[j] = sqrtf(vf[j]);
            pf[j] = pf[j] * c.keep - c.lr * (mf[j] * __builtin_amdgcn_rcpf(root[j] * c.rbc2 + eps));
        }
        aw_store8(p, pt, i, n, vec, pf);
        if constexpr (F8) {
            float tm = aw_top(mf), tv = aw_top(root);
            tm = tm < AW_TINY ? 0.f : tm;
            tv = tv < AW_TINY ? 0.f : tv;
            // scale = t (1 / 448), and the codes' factor 448 (1 / t)
            constexpr float top = SR ? AW_F8_BELOW : AW_F8_MAX;
            const float im = tm > 0.f ? (1.f / tm) * top : 0.f, iv = tv > 0.f ? (1.f / tv) * top : 0.f;
            uint2 cm, cv;
            if constexpr (SR) {
                aw_encode_either(mf, im, root, iv, aw_seed(t, i, gf[0]), &cm, &cv);
            } else {
                cm = aw_encode(mf, im);
                cv = aw_encode(root, iv);
            }
            aw_codes_store(m, i, n, vec, cm);
            aw_codes_store(v, i, n, vec, cv);
            if ((threadIdx.x & 31) == 0) {
                ms[0] = tm * (1.f / AW_F8_MAX);
                vs[0] = tv * (1.f / AW_F8_MAX);
            }
        } else {
            aw_store8(m, RWKV6_F32, i, n, vec, mf);
            aw_store8(v, RWKV6_F32, i, n, vec, vf);
        }
    }
}

namespace {
// Elements that a block takes: `blocks` blocks over all tensors, in steps of AW_STEP.
int64_t aw_per(const int64_t* numel, int64_t count, int64_t blocks) {
    int64_t total = 0;
    for (int64_t k = 0; k < count; ++k) total += numel[k];
    const int64_t per = (total / blocks + AW_STEP - 1) / AW_STEP * AW_STEP;
    return per < AW_STEP ? AW_STEP : per;
}
// Of the step: all blocks at once (eight a CU) where that leaves each a few steps, else one step a block, so
// that the blocks that run together sweep the tensors: 109 M parameters, bf16 with fp32 states, us, with 1,
// 2, 4, 8 and 16 steps a block: 423, 447, 458, 469, 488; 55 M with fp32 and 8-bit states 160, 163, 171, 178, 184;
// 7 M, 2 steps all at once and 1 step 33 and 35.
int64_t aw_step_per(const int64_t* numel, int64_t count) {
    int64_t total = 0;
    for (int64_t k = 0; k < count; ++k) total += numel[k];
    int64_t per = aw_per(numel, count, 2048);
    per = per > 2 * AW_STEP ? AW_STEP : per;
    while (total / per > AW_BLOCKS) per *= 2;      // each tensor of a launch adds a block at most
    return per;
}
int64_t aw_blocks(int64_t n, int64_t per) { return (n + per - 1) / per; }
bool aw_dt(int dt) { return dt == RWKV6_F32 || dt == RWKV6_BF16; }
int aw_sizes(const int64_t* numel, int64_t count) {
    if (count < 0 || (count && !numel)) return RWKV6_ERR_INVALID_ARG;
    if (count > (1 << 20)) return RWKV6_ERR_UNSUPPORTED;
    int64_t total = 0;
    for (int64_t k = 0; k < count; ++k) {
        if (numel[k] < 0) return RWKV6_ERR_INVALID_ARG;
        if (numel[k] > AW_MAX) return RWKV6_ERR_UNSUPPORTED;
        total += numel[k];
    }
    return total > AW_MAX ? RWKV6_ERR_UNSUPPORTED : RWKV6_OK;
}
int64_t aw_partials(const int64_t* numel, int64_t count) {
    const int64_t per = aw_per(numel, count, AW_PARTS);
    int64_t P = 0;
    for (int64_t k = 0; k < count; ++k) P += aw_blocks(numel[k], per);
    return P;
}
bool aw_misaligned(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }

// Whether an output of the step overlaps another or an input, over all tensors: a parameter listed
// twice would be updated by two blocks at once.
struct Range {
    uintptr_t from, to;
    bool out;
};
void aw_add(std::vector<Range>& r, const void* p, size_t bytes, bool out) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    if (p && bytes) r.push_back({a, a + bytes, out});
}
bool aw_overlap(std::vector<Range>& r) {
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t outs = 0, any = 0;                  // where the ones before end
    for (const Range& x : r) {
        if (x.from < (x.out ? any : outs)) return true;
        if (x.out) outs = std::max(outs, x.to);
        any = std::max(any, x.to);
    }
    return false;
}
int aw_step(bool stochastic, void* const* param, const int* param_dtype, const void* const* grad, const int* grad_dtype,
            void* const* exp_avg, void* const* exp_avg_sq, float* const* exp_avg_scale,
            float* const* exp_avg_sq_scale, const int64_t* numel, int64_t count, float* step, double lr,
            const float* lr_dev, double beta1, double beta2, double eps, double weight_decay, const double* partials,
            int64_t P, float max_norm, float* norm, void* workspace, void* stream) {
    const int st = aw_sizes(numel, count);
    if (st) return st;
    const bool f8 = exp_avg_scale != nullptr;
    if (!step || !workspace || P < 0 || (P && !partials)) return RWKV6_ERR_INVALID_ARG;
    if (P > (1 << 30)) return RWKV6_ERR_UNSUPPORTED;
    if (!(beta1 >= 0. && beta1 < 1. && beta2 >= 0. && beta2 < 1.)) return RWKV6_ERR_INVALID_ARG;
    if (count && (!param || !param_dtype || !grad || !grad_dtype || !exp_avg || !exp_avg_sq)) return RWKV6_ERR_INVALID_ARG;
    if (f8 != (exp_avg_sq_scale != nullptr)) return RWKV6_ERR_INVALID_ARG;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) || aw_misaligned(partials, 8) || aw_misaligned(step, 4) ||
        aw_misaligned(lr_dev, 4) || aw_misaligned(norm, 4))
        return RWKV6_ERR_ALIGNMENT;
    try {
        std::vector<Range> ranges;
        ranges.reserve((size_t)count * 6 + 5);
        aw_add(ranges, workspace, sizeof(Coef), true);
        aw_add(ranges, step, 4, true);
        aw_add(ranges, norm, 4, true);
        aw_add(ranges, lr_dev, 4, false);
        aw_add(ranges, partials, (size_t)P * 8, false);
        for (int64_t k = 0; k < count; ++k) {
            if (!aw_dt(param_dtype[k]) || !aw_dt(grad_dtype[k])) return RWKV6_ERR_INVALID_ARG;
            if (numel[k] == 0) continue;
            if (!param[k] || !grad[k] || !exp_avg[k] || !exp_avg_sq[k] || (f8 && (!exp_avg_scale[k] || !exp_avg_sq_scale[k])))
                return RWKV6_ERR_INVALID_ARG;
            const size_t n = (size_t)numel[k], ps = param_bytes(param_dtype[k]), gs = param_bytes(grad_dtype[k]), ss = f8 ? 1 : 4;
            if (aw_misaligned(param[k], ps) || aw_misaligned(grad[k], gs) || aw_misaligned(exp_avg[k], ss) ||
                aw_misaligned(exp_avg_sq[k], ss) || (f8 && (aw_misaligned(exp_avg_scale[k], 4) || aw_misaligned(exp_avg_sq_scale[k], 4))))
                return RWKV6_ERR_ALIGNMENT;
            aw_add(ranges, param[k], n * ps, true);
            aw_add(ranges, grad[k], n * gs, false);
            aw_add(ranges, exp_avg[k], n * ss, true);
            aw_add(ranges, exp_avg_sq[k], n * ss, true);
            if (f8) {
                aw_add(ranges, exp_avg_scale[k], (n + AW_BLK - 1) / AW_BLK * 4, true);
                aw_add(ranges, exp_avg_sq_scale[k], (n + AW_BLK - 1) / AW_BLK * 4, true);
            }
        }
        if (aw_overlap(ranges)) return RWKV6_ERR_INVALID_ARG;
    } catch (...) {                               // no host memory for the check
        return RWKV6_ERR_LAUNCH;
    }
    Coef* coef = (Coef*)workspace;
    hipLaunchKernelGGL(rwkv6_adamw_coef_kernel, dim3(1), dim3(1024), 0, reinterpret_cast<hipStream_t>(stream), partials,
                       partials ? (int)P : 0, max_norm, norm, step, lr_dev, lr, log(beta1), log(beta2), weight_decay, coef);
    const int64_t per = aw_step_per(numel, count);
    StepTable tab;
    int64_t blocks = 0;
    tab.count = 0;
    auto launch = [&] {
        if (!blocks) return;
        auto k = !f8 ? rwkv6_adamw_step_kernel<false, false>
                     : stochastic ? rwkv6_adamw_step_kernel<true, true> : rwkv6_adamw_step_kernel<true, false>;
        hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(AW_THR), 0, reinterpret_cast<hipStream_t>(stream), tab, (const Coef*)coef,
                           per, (float)beta1, (float)(1. - beta1), (float)beta2, (float)(1. - beta2), (float)eps, (const float*)step);
        blocks = tab.count = 0;
    };
    for (int64_t k = 0; k < count; ++k) {
        if (numel[k] == 0) continue;
        const int64_t need = aw_blocks(numel[k], per);
        if (tab.count == AW_T) launch();
        const int i = tab.count++;
        tab.p[i] = param[k];
        tab.g[i] = grad[k];
        tab.m[i] = exp_avg[k];
        tab.v[i] = exp_avg_sq[k];
        tab.ms[i] = f8 ? exp_avg_scale[k] : nullptr;
        tab.vs[i] = f8 ? exp_avg_sq_scale[k] : nullptr;
        tab.n[i] = numel[k];
        tab.dt[i] = param_dtype[k] | grad_dtype[k] << 8;
        tab.first[i] = (int)blocks;
        blocks += need;
    }
    launch();
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}
}  // namespace

extern "C" {

int64_t rwkv6_grad_norm_partials(const int64_t* numel, int64_t count) {
    return aw_sizes(numel, count) ? 0 : aw_partials(numel, count);
}

int rwkv6_grad_norm_sums(const void* const* grad, const int* grad_dtype, const int64_t* numel, int64_t count,
                         double* partials, void* stream) {
    const int st = aw_sizes(numel, count);
    if (st) return st;
    if (count && (!grad || !grad_dtype)) return RWKV6_ERR_INVALID_ARG;
    const int64_t per = aw_per(numel, count, AW_PARTS);
    const Span out = {partials, (size_t)aw_partials(numel, count) * 8};
    int64_t bytes = 0;
    for (int64_t k = 0; k < count; ++k) {
        if (!aw_dt(grad_dtype[k]) || (numel[k] && (!grad[k] || !partials))) return RWKV6_ERR_INVALID_ARG;
        if (aw_misaligned(grad[k], param_bytes(grad_dtype[k]))) return RWKV6_ERR_ALIGNMENT;
        bytes += numel[k] * (int64_t)param_bytes(grad_dtype[k]);
        if (spans_overlap(out, {grad[k], (size_t)numel[k] * param_bytes(grad_dtype[k])}))
            return RWKV6_ERR_INVALID_ARG;
    }
    if (aw_misaligned(partials, 8)) return RWKV6_ERR_ALIGNMENT;
    // Gradients that the last cache (256 MB) cannot keep for the step anyway are read past it: kept there they
    // push out what the kernels before have written.  437 MB: 117 us through the caches, 85 past them.
    const bool nt = bytes > ((int64_t)1 << 28);
    NormTable tab;
    int blocks = 0, base = 0;
    tab.count = 0;
    auto launch = [&] {
        if (!blocks) return;
        tab.base = base;
        hipLaunchKernelGGL(rwkv6_grad_square_sums_kernel, dim3((unsigned)blocks), dim3(AW_THR), 0,
                           reinterpret_cast<hipStream_t>(stream), tab, nt, partials);
        base += blocks;
        blocks = tab.count = 0;
    };
    for (int64_t k = 0; k < count; ++k) {
        if (numel[k] == 0) continue;
        if (tab.count == AW_T) launch();
        const int i = tab.count++;
        tab.g[i] = grad[k];
        tab.n[i] = numel[k];
        tab.dt[i] = grad_dtype[k];
        tab.first[i] = blocks;
        blocks += (int)aw_blocks(numel[k], per);
    }
    launch();
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}

int rwkv6_grad_norm(const double* partials, int64_t P, float* norm, void* stream) {
    if (P < 0 || (P && !partials) || !norm) return RWKV6_ERR_INVALID_ARG;
    if (P > (1 << 30)) return RWKV6_ERR_UNSUPPORTED;
    if (aw_misaligned(partials, 8) || aw_misaligned(norm, 4)) return RWKV6_ERR_ALIGNMENT;
    if (any_alias({{norm, 4}}, {{partials, (size_t)P * 8}})) return RWKV6_ERR_INVALID_ARG;
    hipLaunchKernelGGL(rwkv6_adamw_coef_kernel, dim3(1), dim3(1024), 0, reinterpret_cast<hipStream_t>(stream), partials,
                       (int)P, 0.f, norm, nullptr, nullptr, 0., 0., 0., 0., nullptr);
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}

int rwkv6_adamw_step(void* const* param, const int* param_dtype, const void* const* grad, const int* grad_dtype,
                     void* const* exp_avg, void* const* exp_avg_sq, float* const* exp_avg_scale,
                     float* const* exp_avg_sq_scale, const int64_t* numel, int64_t count, float* step, double lr,
                     const float* lr_dev, double beta1, double beta2, double eps, double weight_decay, const double* partials,
                     int64_t P, float max_norm, float* norm, void* workspace, void* stream) {
    return aw_step(false, param, param_dtype, grad, grad_dtype, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, numel, count, step, lr,
                   lr_dev, beta1, beta2, eps, weight_decay, partials, P, max_norm, norm, workspace, stream);
}

int rwkv6_adamw_step_stochastic(void* const* param, const int* param_dtype, const void* const* grad, const int* grad_dtype,
                                void* const* exp_avg, void* const* exp_avg_sq, float* const* exp_avg_scale,
                                float* const* exp_avg_sq_scale, const int64_t* numel, int64_t count, float* step, double lr,
                                const float* lr_dev, double beta1, double beta2, double eps, double weight_decay, const double* partials,
                                int64_t P, float max_norm, float* norm, void* workspace, void* stream) {
    return aw_step(true, param, param_dtype, grad, grad_dtype, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, numel, count, step, lr,
                   lr_dev, beta1, beta2, eps, weight_decay, partials, P, max_norm, norm, workspace, stream);
}

}  // extern "C"
