// Cross entropy of token rows over the vocabulary and its gradient, for MI355X (gfx950).
//
// Reference: the language model's loss a token, which the training driver averages over the unmasked
// tokens (/root/reference/pretrain_rwkv6.py:144-179; the output head's logits, rwkv6_model.py:28-184).
//   loss = log z + (m - l_t),  m = max_j l_j,  z = sum_j exp(l_j - m)     (0 for an ignored target)
//   d_l_j = d_loss (exp(l_j - m) / z - [j = t])                            (0 for an ignored target)
// The forward reads the logits once, each thread with a running maximum and sum that are joined at the
// end, and keeps m and z of a row: (m, 1/z) instead of log z + m keeps the gradient's exponent free of
// the rounding of a number of size 10.
//
// Bound by memory: 2 bytes a logit in bf16 forward, 4 backward.  16384 x 65536: 341 us (6.3 TB/s) and 726
// us (5.9 TB/s); 1024 x 65536: 38 and 40 us, the forward while what ran before it still writes its output
// back (26 us without); 1001 x 50001 in fp32 53 and 70 us.  A sum of two 1 GiB tensors reaches 6.1 TB/s.  torch's
// operators in 32 bits take 9.1 ms, 636 and 410 us for both ways.
#include "common.h"
#include "../../include/rwkv6_amd.h"

#define CE_GRID (1 << 21)      // blocks a launch, of up to 1024 threads: fewer than 2^32 threads

namespace {

template <bool F32> struct CeVec { static constexpr int E = F32 ? 4 : 8; };     // elements of 16 bytes

template <bool F32>
__device__ __forceinline__ void ce_unpack(uint4 q, float* f) {
    if constexpr (F32) {
        f[0] = __uint_as_float(q.x); f[1] = __uint_as_float(q.y);
        f[2] = __uint_as_float(q.z); f[3] = __uint_as_float(q.w);
    } else {
        unpack8(q, f);
    }
}
template <bool F32>
__device__ __forceinline__ float ce_load(const char* row, int j) {
    if constexpr (F32) return reinterpret_cast<const float*>(row)[j];
    else return bf2f(reinterpret_cast<const uint16_t*>(row)[j]);
}
// elements before the row's first 16-byte boundary (rows lie at multiples of the element's size)
template <bool F32>
__device__ __forceinline__ int ce_lead(const void* row, int V) {
    const int off = (int)(reinterpret_cast<uintptr_t>(row) & 15u) / (F32 ? 4 : 2), E = CeVec<F32>::E;
    const int lead = off ? E - off : 0;
    return lead < V ? lead : V;
}

// (m, z) of a set of logits: z = sum exp(l - m).  An empty set, or one of -inf alone, is (-inf, 0).
struct Soft {
    float m, z;
};
__device__ __forceinline__ float ce_ref(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ Soft join(Soft a, Soft b) {
    const float m = fmaxf(a.m, b.m), r = ce_ref(m);
    return {m, a.z * ex2((a.m - r) * RW_L2E) + b.z * ex2((b.m - r) * RW_L2E)};
}
template <int K> __device__ __forceinline__ void ce_take(Soft& s, const float* v) {
    float m = s.m;
#pragma unroll
    for (int k = 0; k < K; ++k) m = fmaxf(m, v[k]);
    const float r = ce_ref(m);
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) t += ex2((v[k] - r) * RW_L2E);
    s.z = s.z * ex2((s.m - r) * RW_L2E) + t;
    s.m = m;
}
}  // namespace

// THR threads a row: a block, or a wave of the block's four (striding over the rows); CE_U pieces of 16
// bytes a thread in flight.
#define CE_U 4
#define CE_BLOCK(THR) ((THR) < 256 ? 256 : (THR))
template <bool F32, int THR>
__global__ void __launch_bounds__(CE_BLOCK(THR))
rwkv6_cross_entropy_fwd_kernel(const void* __restrict__ logits, int64_t ld, const int64_t* __restrict__ target,
                               int64_t ignore, float* __restrict__ loss, float2* __restrict__ stats, int64_t N,
                               int V) {
    constexpr int E = CeVec<F32>::E, ES = F32 ? 4 : 2, ROWS = CE_BLOCK(THR) / THR;
    __shared__ Soft part[THR / 64];
    const int tid = threadIdx.x % THR;
    for (int64_t n = (int64_t)blockIdx.x * ROWS + threadIdx.x / THR; n < N; n += (int64_t)gridDim.x * ROWS) {
        const int64_t t = target[n];
        const bool ignored = t == ignore, bad = !ignored && (t < 0 || t >= V);
        // the same for all threads of the row; a short row is read all the same, its loads do not wait then
        if (THR > 64 && (ignored || bad)) {
            if (tid == 0) {
                loss[n] = ignored ? 0.f : NAN;
                stats[n] = make_float2(0.f, 1.f);
            }
            continue;
        }
        const char* row = reinterpret_cast<const char*>(logits) + n * ld * ES;
        const int lead = ce_lead<F32>(row, V);
        const int pieces = (V - lead) / E, tail = lead + pieces * E;
        const uint4* body = reinterpret_cast<const uint4*>(row + (int64_t)lead * ES);
        Soft s = {-INFINITY, 0.f};
        int i = tid;
        for (; i + (CE_U - 1) * THR < pieces; i += CE_U * THR) {
            float v[CE_U * E];
#pragma unroll
            for (int u = 0; u < CE_U; ++u) ce_unpack<F32>(body[i + u * THR], v + u * E);
            ce_take<CE_U * E>(s, v);
        }
        for (; i < pieces; i += THR) {
            float v[E];
            ce_unpack<F32>(body[i], v);
            ce_take<E>(s, v);
        }
        // fewer than 8 elements at either end
        if (tid < lead) {
            const float v = ce_load<F32>(row, tid);
            ce_take<1>(s, &v);
        }
        if (tid < V - tail) {
            const float v = ce_load<F32>(row, tail + tid);
            ce_take<1>(s, &v);
        }
        // the wave's maximum first, then every lane's sum scaled to it once
        const float m = wave_max(s.m);
        s.z = wave_sum(s.z * ex2((s.m - ce_ref(m)) * RW_L2E));
        s.m = m;
        if constexpr (THR > 64) {
            __syncthreads();                              // the row before has been read from `part`
            if ((tid & 63) == 0) part[tid >> 6] = s;
            __syncthreads();
        }
        if (tid == 0) {
            if constexpr (THR > 64)
                for (int w = 1; w < THR / 64; ++w) s = join(s, part[w]);
            loss[n] = ignored ? 0.f : bad ? NAN : logf(s.z) + (s.m - ce_load<F32>(row, (int)t));
            stats[n] = make_float2(s.m, s.z);
        }
    }
}

// THR threads a row as above, or a part of it: `seg` parts a row, a block each, in the order they lie in
// memory, so that the blocks that run together sweep it.
template <bool F32, int THR>
__global__ void __launch_bounds__(CE_BLOCK(THR))
rwkv6_cross_entropy_bwd_kernel(const void* __restrict__ logits, int64_t ld, const int64_t* __restrict__ target,
                               int64_t ignore, const float2* __restrict__ stats, const float* __restrict__ d_loss,
                               void* __restrict__ d_logits, int64_t N, int V, int seg) {
    constexpr int E = CeVec<F32>::E, ES = F32 ? 4 : 2, ROWS = CE_BLOCK(THR) / THR;
    const int tid = threadIdx.x % THR;
    const int64_t all = (N + ROWS - 1) / ROWS * seg;
    for (int64_t id = blockIdx.x; id < all; id += gridDim.x) {
        const int part = seg > 1 ? (int)(id % seg) : 0;
        const int64_t n = (seg > 1 ? id / seg : id) * ROWS + threadIdx.x / THR;
        if (n >= N) return;
        const int64_t t = target[n];
        const bool ignored = t == ignore, bad = !ignored && (t < 0 || t >= V);
        const char* row = reinterpret_cast<const char*>(logits) + n * ld * ES;
        char* out = reinterpret_cast<char*>(d_logits) + n * V * ES;
        const float2 st = stats[n];
        const float dl = d_loss[n];
        // an ignored row's zeros and a bad one's NaN do not depend on its logits
        const bool fixed = ignored || bad;
        const float w = bad ? NAN : ignored ? 0.f : dl, q = w / st.y, m = st.x;
        const int hit = fixed ? -1 : (int)t;
        auto grad = [&](float l, int j) {
            const float p = q * ex2((l - m) * RW_L2E);
            return fixed ? w : j == hit ? p - w : p;
        };
        auto put = [&](int j, const float* v) {
            if constexpr (F32) *reinterpret_cast<float4*>(out + (int64_t)j * ES) = make_float4(v[0], v[1], v[2], v[3]);
            else store8(reinterpret_cast<uint16_t*>(out) + j, v);
        };
        auto put1 = [&](int j) {
            const float g = grad(ce_load<F32>(row, j), j);
            if constexpr (F32) reinterpret_cast<float*>(out)[j] = g;
            else reinterpret_cast<uint16_t*>(out)[j] = f2bf(g);
        };
        const int lead = ce_lead<F32>(out, V);
        const int pieces = (V - lead) / E, tail = lead + pieces * E;
        const bool vec = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(out)) & 15u) == 0;
        const int per = (pieces + seg - 1) / seg, i0 = min(per * part, pieces);
        const int i1 = min(i0 + per, pieces);
        int i = i0 + tid;
        for (; vec && i + (CE_U - 1) * THR < i1; i += CE_U * THR) {
            uint4 raw[CE_U];
#pragma unroll
            for (int u = 0; u < CE_U; ++u) raw[u] = *reinterpret_cast<const uint4*>(row + (int64_t)(lead + (i + u * THR) * E) * ES);
#pragma unroll
            for (int u = 0; u < CE_U; ++u) {
                const int j = lead + (i + u * THR) * E;
                float v[E];
                ce_unpack<F32>(raw[u], v);
#pragma unroll
                for (int k = 0; k < E; ++k) v[k] = grad(v[k], j + k);
                put(j, v);
            }
        }
        for (; i < i1; i += THR) {
            const int j = lead + i * E;
            float v[E];
            if (vec) {
                ce_unpack<F32>(*reinterpret_cast<const uint4*>(row + (int64_t)j * ES), v);
            } else {
#pragma unroll
                for (int k = 0; k < E; ++k) v[k] = ce_load<F32>(row, j + k);
            }
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] = grad(v[k], j + k);
            put(j, v);
        }
        // fewer than 8 elements at either end
        if (part == 0) {
            if (tid < lead) put1(tid);
            if (tid < V - tail) put1(tail + tid);
        }
    }
}

namespace {
int ce_check(const void* logits, int dtype, int64_t ld, const int64_t* target, int64_t N, int64_t V) {
    if (N < 0 || V < 1 || ld < V) return RWKV6_ERR_INVALID_ARG;
    if (dtype != RWKV6_F32 && dtype != RWKV6_BF16) return RWKV6_ERR_INVALID_ARG;
    if (V > ((int64_t)1 << 30) || ld > ((int64_t)1 << 40) || N > ((int64_t)1 << 50) / ld) return RWKV6_ERR_UNSUPPORTED;
    if (N > 0 && (!logits || !target)) return RWKV6_ERR_INVALID_ARG;
    // rows may start at any element
    if (reinterpret_cast<uintptr_t>(logits) % param_bytes(dtype)) return RWKV6_ERR_ALIGNMENT;
    return RWKV6_OK;
}
// bytes from the first logit to the last
size_t ce_span(int64_t ld, int64_t N, int64_t V, int dtype) { return (size_t)((N - 1) * ld + V) * param_bytes(dtype); }
}  // namespace

extern "C" {

int rwkv6_cross_entropy_fwd(const void* logits, int dtype, int64_t ld, const int64_t* target, int64_t ignore_index,
                            float* loss, float* stats, int64_t N, int64_t V, void* stream) {
    const int st = ce_check(logits, dtype, ld, target, N, V);
    if (st || N == 0) return st;
    if (!loss || !stats) return RWKV6_ERR_INVALID_ARG;
    if (reinterpret_cast<uintptr_t>(stats) & 7u) return RWKV6_ERR_ALIGNMENT;
    if (any_alias({{loss, (size_t)N * 4}, {stats, (size_t)N * 8}},
                  {{logits, ce_span(ld, N, V, dtype)}, {target, (size_t)N * 8}}))
        return RWKV6_ERR_INVALID_ARG;
    const bool f32 = dtype == RWKV6_F32;
    // A wave for a short row, whose cost is the joining of the threads' sums, more for a long one; one row
    // of 1024 threads at a time streams best where the rows fill the device several times over.  Forward, us,
    // with 64, 256, 512, 1024 threads: 65536 x 376 20, 61, 132, 261; 16384 x 4104 26, 35, 52, 86; 16384 x 8192
    // 50, 45, 68, 96; 8192 x 32000 92, 91, 87, 107; 4096 x 65536 103, 94, 92, 86; 1024 x 65536 35, 28, 26, 26;
    // 512 x 65536 24, 13, 13, 14.
    const int64_t pieces = V * (int64_t)param_bytes(dtype) / 16;
    const int thr = pieces < 1024 ? 64 : pieces < 4096 ? 256 : N < 2048 ? 512 : 1024;
#define CE_PICK(F) (thr == 64 ? rwkv6_cross_entropy_fwd_kernel<F, 64> : thr == 256 ? rwkv6_cross_entropy_fwd_kernel<F, 256> \
                    : thr == 512 ? rwkv6_cross_entropy_fwd_kernel<F, 512> : rwkv6_cross_entropy_fwd_kernel<F, 1024>)
    auto k = f32 ? CE_PICK(true) : CE_PICK(false);
#undef CE_PICK
    const int64_t blocks = thr == 64 ? (N + 3) / 4 : N;
    hipLaunchKernelGGL(k, dim3((unsigned)(blocks < CE_GRID ? blocks : CE_GRID)), dim3(CE_BLOCK(thr)), 0,
                       reinterpret_cast<hipStream_t>(stream), logits, ld, target, ignore_index, loss, (float2*)stats, N, (int)V);
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}

int rwkv6_cross_entropy_bwd(const void* logits, int dtype, int64_t ld, const int64_t* target, int64_t ignore_index,
                            const float* stats, const float* d_loss, void* d_logits, int64_t N, int64_t V,
                            void* stream) {
    const int st = ce_check(logits, dtype, ld, target, N, V);
    if (st || N == 0) return st;
    if (!stats || !d_loss || !d_logits) return RWKV6_ERR_INVALID_ARG;
    if ((reinterpret_cast<uintptr_t>(stats) & 7u) || reinterpret_cast<uintptr_t>(d_logits) % param_bytes(dtype))
        return RWKV6_ERR_ALIGNMENT;
    if (any_alias({{d_logits, (size_t)(N * V) * param_bytes(dtype)}},
                  {{logits, ce_span(ld, N, V, dtype)}, {target, (size_t)N * 8}, {stats, (size_t)N * 8}, {d_loss, (size_t)N * 4}}))
        return RWKV6_ERR_INVALID_ARG;
    // A wave for a short row; a long one in parts of 1024 pieces, the CE_U a thread that are in flight at once.
    // 16384 x 65536 bf16, us, with 256, 1024, 2048, 4096 pieces and whole rows a block: 936, 726, 775, 795, 807.
    const int64_t pieces = V * (int64_t)param_bytes(dtype) / 16;
    const bool f32 = dtype == RWKV6_F32, wave = pieces < 1024;
    const int seg = wave ? 1 : (int)((pieces + 1023) / 1024);
    auto k = f32 ? (wave ? rwkv6_cross_entropy_bwd_kernel<true, 64> : rwkv6_cross_entropy_bwd_kernel<true, 256>)
                 : (wave ? rwkv6_cross_entropy_bwd_kernel<false, 64> : rwkv6_cross_entropy_bwd_kernel<false, 256>);
    const int64_t blocks = wave ? (N + 3) / 4 : N * seg;
    hipLaunchKernelGGL(k, dim3((unsigned)(blocks < CE_GRID ? blocks : CE_GRID)), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), logits, ld, target, ignore_index, (const float2*)stats, d_loss,
                       d_logits, N, (int)V, seg);
    return hipGetLastError() == hipSuccess ? RWKV6_OK : RWKV6_ERR_LAUNCH;
}

}  // extern "C"
