// Distillation of a student from a teacher's top logits, and its gradient.  Row r of the (rows, vocab) student logits z has `slots`
// pairs (index, teacher logit t); with temperature T
//     p_i = softmax(t / T) over the row's used slots        q_j = softmax(z / T) over the whole vocabulary
//     loss_r = T^2 sum_i p_i (log p_i - log q_(index i))     dz_j = T u_r (q_j - sum_(i: index i = j) p_i)
// u_r being the upstream gradient of loss_r.  A slot whose index lies outside [0, vocab) or whose teacher logit is -inf is unused;
// a row without a used slot has loss 0 and gradient 0 and its logits are not read.
//
// Bound: HBM.  Forward reads the logits once (online softmax: every thread keeps a running maximum and the sum relative to it),
// backward reads them once more and writes the gradient: 3 * rows * vocab * bytes in all.  Nothing of the vocabulary's length is kept
// between the two, only each row's maximum m and sum s: q = exp((z - m) / T) / s, with the difference taken first so that
// the exponent carries no rounding of a large log-sum.
//
// One CTA works on one row at a time; 16-byte pieces where the row is aligned, single values up to the first
// boundary and behind the last.  Sums are fp32 per thread (at most a few hundred terms) and joined in a fixed order.
#include <cuda_bf16.h>
#include <math_constants.h>

#include "common.cuh"

namespace axs6 {
namespace distill {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxSlots = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
    const void *z, *t;
    const long long *index;
    long long rows, vocab, ldz, ldt, ldi;
    int slots;
    float temperature;
    float *row_loss;        // rows
    float *stats;           // rows x 2: maximum of z, sum of exp((z - maximum) / T); sum 0 = unused row
    // backward
    void *grad;
    long long ldg;
    const float *upstream;
    long long upstream_stride;
    const float *count;     // null, or the number of rows the mean was taken over
};

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }

template <typename T> struct Vec { static constexpr int n = 16 / (int)sizeof(T); union { uint4 raw; T v[n]; }; };

// Values before the first 16-byte boundary of a row (at most vocab).
template <typename T> __device__ __forceinline__ int head_of(const T *row, long long vocab)
{
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    const int h = mis ? Vec<T>::n - mis : 0;
    return (long long)h < vocab ? h : (int)vocab;
}

struct Slots {
    int index[kMaxSlots];   // -1: unused
    float p[kMaxSlots];     // teacher logit, then its probability
};

// Loads a row's slots and turns the teacher's logits into probabilities; sc[0] = sum of exp((t - max) / T) (0: no used slot),
// sc[1] = max.  Called by the whole CTA; ends with a barrier.
template <typename Tt>
__device__ __forceinline__ void load_slots(const Params &p, long long row, Slots &s, float *sc)
{
    const Tt *t = static_cast<const Tt *>(p.t) + row * p.ldt;
    const long long *ix = p.index + row * p.ldi;
    for (int i = threadIdx.x; i < p.slots; i += kThreads) {
        const long long j = ix[i];
        const float v = to_f(t[i]);
        const bool used = j >= 0 && j < p.vocab && v != -CUDART_INF_F;
        s.index[i] = used ? (int)j : -1;
        s.p[i] = used ? v : -CUDART_INF_F;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const float c = kLog2e / p.temperature;
        float m = -CUDART_INF_F, sum = 0.0f;
        for (int i = threadIdx.x; i < p.slots; i += 32) m = fmaxf(m, s.p[i]);
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        if (m != -CUDART_INF_F) {
            for (int i = threadIdx.x; i < p.slots; i += 32) sum += ex2((s.p[i] - m) * c);
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        }
        if (threadIdx.x == 0) { sc[0] = sum; sc[1] = m; }
    }
    __syncthreads();
}

// (m, s) of two parts of a row joined: the sum is relative to the maximum.
__device__ __forceinline__ void join(float &m, float &s, float m2, float s2, float c)
{
    const float top = fmaxf(m, m2), base = top == -CUDART_INF_F ? 0.0f : top;
    s = s * ex2((m - base) * c) + s2 * ex2((m2 - base) * c);
    m = top;
}

template <typename T, typename Tt>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Params p)
{
    __shared__ Slots slots;
    __shared__ float sc[2], part[2 * kWarps];
    const float c = kLog2e / p.temperature;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *z = static_cast<const T *>(p.z) + row * p.ldz;
        load_slots<Tt>(p, row, slots, sc);
        if (sc[0] == 0.0f) {                                        // no used slot
            if (threadIdx.x == 0) { p.row_loss[row] = 0.0f; p.stats[2 * row] = 0.0f; p.stats[2 * row + 1] = 0.0f; }
            __syncthreads();
            continue;
        }
        float m = -CUDART_INF_F, s = 0.0f;
        auto one = [&](float v) {
            if (v > m) { s *= ex2((m - v) * c); m = v; }
            s += v == -CUDART_INF_F ? 0.0f : ex2((v - m) * c);       // m is finite or +inf here unless v is -inf or NaN
        };
        const int head = head_of(z, p.vocab);
        const long long vecs = (p.vocab - head) / Vec<T>::n;
        const uint4 *zv = reinterpret_cast<const uint4 *>(z + head);
        constexpr int kUnroll = 4;
        long long i = threadIdx.x;
        auto piece = [&](const Vec<T> &v) {
            float top = to_f(v.v[0]);
#pragma unroll
            for (int e = 1; e < Vec<T>::n; ++e) top = fmaxf(top, to_f(v.v[e]));
            if (top > m) { s *= ex2((m - top) * c); m = top; }
            const float base = m == -CUDART_INF_F ? 0.0f : m;
#pragma unroll
            for (int e = 0; e < Vec<T>::n; ++e) s += ex2((to_f(v.v[e]) - base) * c);
        };
        for (; i + (kUnroll - 1) * kThreads < vecs; i += kUnroll * kThreads) {
            Vec<T> v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) v[u].raw = __ldg(zv + i + u * kThreads);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) piece(v[u]);
        }
        for (; i < vecs; i += kThreads) { Vec<T> v; v.raw = __ldg(zv + i); piece(v); }
        if ((int)threadIdx.x < head) one(to_f(z[threadIdx.x]));
        for (long long j = head + vecs * Vec<T>::n + threadIdx.x; j < p.vocab; j += kThreads) one(to_f(z[j]));
        for (int o = 16; o; o >>= 1) join(m, s, __shfl_xor_sync(~0u, m, o), __shfl_xor_sync(~0u, s, o), c);
        if ((threadIdx.x & 31) == 0) { part[2 * (threadIdx.x >> 5)] = m; part[2 * (threadIdx.x >> 5) + 1] = s; }
        __syncthreads();
        if (threadIdx.x < 32) {
            m = -CUDART_INF_F; s = 0.0f;
            if (threadIdx.x < kWarps) { m = part[2 * threadIdx.x]; s = part[2 * threadIdx.x + 1]; }
            for (int o = 16; o; o >>= 1) join(m, s, __shfl_xor_sync(~0u, m, o), __shfl_xor_sync(~0u, s, o), c);
            // log p_i - log q_i in bits: (t_i - max t) c - log2 sum - (z_i - m) c + log2 s
            const float lt = log2f(sc[0]), lz = log2f(s), inv = 1.0f / sc[0];
            float loss = 0.0f;
            for (int k = threadIdx.x; k < p.slots; k += 32) {
                if (slots.index[k] < 0) continue;
                const float a = (slots.p[k] - sc[1]) * c, prob = ex2(a) * inv;
                if (prob != 0.0f) loss += prob * ((a - lt) - ((to_f(z[slots.index[k]]) - m) * c - lz));
            }
            for (int o = 16; o; o >>= 1) loss += __shfl_xor_sync(~0u, loss, o);
            if (threadIdx.x == 0) {
                p.row_loss[row] = loss * (kLn2 * p.temperature * p.temperature);
                p.stats[2 * row] = m;
                p.stats[2 * row + 1] = s;
            }
        }
        __syncthreads();
    }
}

// Sum of the rows' losses, or their mean over the rows with a used slot, in 64 bits and in a fixed order; out[1] = that number of rows.
__global__ void __launch_bounds__(1024) reduce_kernel(const float *row_loss, const float *stats, long long rows, int mean, float *out)
{
    __shared__ double sum_s[32];
    __shared__ long long cnt_s[32];
    pdl_wait();
    double sum = 0.0;
    long long cnt = 0;
    for (long long i = threadIdx.x; i < rows; i += 1024) { sum += (double)row_loss[i]; cnt += stats[2 * i + 1] != 0.0f; }
    for (int o = 16; o; o >>= 1) { sum += __shfl_xor_sync(~0u, sum, o); cnt += __shfl_xor_sync(~0u, cnt, o); }
    if ((threadIdx.x & 31) == 0) { sum_s[threadIdx.x >> 5] = sum; cnt_s[threadIdx.x >> 5] = cnt; }
    __syncthreads();
    if (threadIdx.x < 32) {
        sum = sum_s[threadIdx.x]; cnt = cnt_s[threadIdx.x];
        for (int o = 16; o; o >>= 1) { sum += __shfl_xor_sync(~0u, sum, o); cnt += __shfl_xor_sync(~0u, cnt, o); }
        if (threadIdx.x == 0) {
            const double n = cnt ? (double)cnt : 1.0;
            out[0] = (float)(mean ? sum / n : sum);
            out[1] = (float)n;
        }
    }
}

template <typename T, typename Tt>
__global__ void __launch_bounds__(kThreads) backward_kernel(const Params p)
{
    __shared__ Slots slots;
    __shared__ float sc[2];
    const float c = kLog2e / p.temperature;
    for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *z = static_cast<const T *>(p.z) + row * p.ldz;
        T *g = static_cast<T *>(p.grad) + row * p.ldg;
        const float m = p.stats[2 * row], s = p.stats[2 * row + 1];
        const bool used = s != 0.0f;
        const float up = p.upstream[row * p.upstream_stride] * p.temperature / (p.count ? *p.count : 1.0f);
        const float w = used ? up / s : 0.0f;
        const int head = head_of(g, p.vocab);
        // 16-byte pieces of both, if the two rows lie alike
        const bool alike = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(g)) & 15u) == 0;
        const long long vecs = alike || !used ? (p.vocab - head) / Vec<T>::n : 0;
        uint4 *gv = reinterpret_cast<uint4 *>(g + head);
        auto one = [&](long long j) { from_f(used ? ex2((to_f(z[j]) - m) * c) * w : 0.0f, g[j]); };
        if (used) {
            const uint4 *zv = reinterpret_cast<const uint4 *>(z + head);
            auto piece = [&](const Vec<T> &v, long long at) {
                Vec<T> o;
#pragma unroll
                for (int e = 0; e < Vec<T>::n; ++e) from_f(ex2((to_f(v.v[e]) - m) * c) * w, o.v[e]);
                __stcs(gv + at, o.raw);
            };
            constexpr int kUnroll = 4;
            long long i = threadIdx.x;
            for (; i + (kUnroll - 1) * kThreads < vecs; i += kUnroll * kThreads) {
                Vec<T> v[kUnroll];
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) v[u].raw = __ldg(zv + i + u * kThreads);
#pragma unroll
                for (int u = 0; u < kUnroll; ++u) piece(v[u], i + u * kThreads);
            }
            for (; i < vecs; i += kThreads) { Vec<T> v; v.raw = __ldg(zv + i); piece(v, i); }
        } else {
            for (long long i = threadIdx.x; i < vecs; i += kThreads) gv[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        if ((int)threadIdx.x < head) one(threadIdx.x);
        for (long long j = head + vecs * Vec<T>::n + threadIdx.x; j < p.vocab; j += kThreads) one(j);
        if (used) {
            load_slots<Tt>(p, row, slots, sc);                       // its barriers also order the stores above before those below
            const float inv = 1.0f / sc[0];
            // The first slot that names a place writes it, with the probabilities of all the slots that name it in slot order.
            for (int k = threadIdx.x; k < p.slots; k += kThreads) {
                const int j = slots.index[k];
                if (j < 0) continue;
                float prob = 0.0f;
                bool first = true;
                for (int o = 0; o < p.slots; ++o)
                    if (slots.index[o] == j) {
                        if (o < k) { first = false; break; }
                        prob += ex2((slots.p[o] - sc[1]) * c) * inv;
                    }
                if (first) from_f((ex2((to_f(z[j]) - m) * c) / s - prob) * up, g[j]);
            }
            __syncthreads();
        }
    }
}

static bool args_ok(const void *z, int dtype, int64_t rows, int64_t vocab, int64_t ldz, const void *t, int t_dtype, int64_t ldt,
                    const void *index, int64_t ldi, int64_t slots, float temperature)
{
    return valid_dtype(dtype) && valid_dtype(t_dtype) && rows >= 0 && vocab >= 1 && vocab < INT32_MAX && slots >= 1 && ldz >= 0 && ldt >= 0 &&
           ldi >= 0 && temperature > 0.0f && temperature <= 3.402823466e38f && (rows == 0 || (z && t && index));
}

// CTAs: as many as are resident, or one a row.
static unsigned grid_of(const void *kernel, const DeviceInfo &d, int64_t rows)
{
    const int per = cached_occupancy(kernel, kThreads);
    const int64_t most = (int64_t)d.sms * (per > 0 ? per : 1);
    return (unsigned)(rows < most ? rows : most);
}

}  // namespace distill
}  // namespace axs6

AXS6_API int axs6_distill_fwd(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const void *teacher, int teacher_dtype,
                              int64_t ld_teacher, const int64_t *index, int64_t ld_index, int64_t slots, float temperature, int reduction,
                              float *row_loss, float *row_stats, float *reduced, axs6_stream_t stream)
{
    using namespace axs6;
    using namespace axs6::distill;
    if (!args_ok(logits, dtype, rows, vocab, ld, teacher, teacher_dtype, ld_teacher, index, ld_index, slots, temperature) || reduction < 0 ||
        reduction > 2 || (rows && (!row_loss || !row_stats)) || (reduction && !reduced))
        return AXS6_ERR_ARG;
    if (slots > kMaxSlots) return AXS6_ERR_UNSUPPORTED;
    const DeviceInfo &d = device_info();
    if (!d.valid || !d.ok) return AXS6_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Params p = {};
    p.z = logits; p.t = teacher; p.index = reinterpret_cast<const long long *>(index);
    p.rows = rows; p.vocab = vocab; p.ldz = ld; p.ldt = ld_teacher; p.ldi = ld_index; p.slots = (int)slots; p.temperature = temperature;
    p.row_loss = row_loss; p.stats = row_stats;
    if (rows) {
        auto go = [&](auto kernel) {
            kernel<<<grid_of(reinterpret_cast<const void *>(kernel), d, rows), kThreads, 0, st>>>(p);
            count_launch();
            return check_launch();
        };
        const int rc = dtype == AXS6_F32
            ? (teacher_dtype == AXS6_F32 ? go(&forward_kernel<float, float>) : go(&forward_kernel<float, __nv_bfloat16>))
            : (teacher_dtype == AXS6_F32 ? go(&forward_kernel<__nv_bfloat16, float>) : go(&forward_kernel<__nv_bfloat16, __nv_bfloat16>));
        if (rc != AXS6_OK) return rc;
    }
    if (reduction) {
        if (launch_overlapped(true, reduce_kernel, 1, 1024, 0, st, row_loss, row_stats, (long long)rows, reduction == 2, reduced) != cudaSuccess)
            return AXS6_ERR_LAUNCH;
        count_launch();
    }
    return AXS6_OK;
}

AXS6_API int axs6_distill_bwd(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const void *teacher, int teacher_dtype,
                              int64_t ld_teacher, const int64_t *index, int64_t ld_index, int64_t slots, float temperature,
                              const float *row_stats, const float *upstream, int64_t upstream_stride, const float *count, void *grad,
                              int64_t ld_grad, axs6_stream_t stream)
{
    using namespace axs6;
    using namespace axs6::distill;
    if (!args_ok(logits, dtype, rows, vocab, ld, teacher, teacher_dtype, ld_teacher, index, ld_index, slots, temperature) || ld_grad < 0 ||
        (rows && (!row_stats || !upstream || !grad)))
        return AXS6_ERR_ARG;
    if (slots > kMaxSlots) return AXS6_ERR_UNSUPPORTED;
    if (rows == 0) return AXS6_OK;
    const DeviceInfo &d = device_info();
    if (!d.valid || !d.ok) return AXS6_ERR_DEVICE;
    Params p = {};
    p.z = logits; p.t = teacher; p.index = reinterpret_cast<const long long *>(index);
    p.rows = rows; p.vocab = vocab; p.ldz = ld; p.ldt = ld_teacher; p.ldi = ld_index; p.slots = (int)slots; p.temperature = temperature;
    p.stats = const_cast<float *>(row_stats); p.grad = grad; p.ldg = ld_grad;
    p.upstream = upstream; p.upstream_stride = upstream_stride; p.count = count;
    auto go = [&](auto kernel) {
        kernel<<<grid_of(reinterpret_cast<const void *>(kernel), d, rows), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
        count_launch();
        return check_launch();
    };
    if (dtype == AXS6_F32)
        return teacher_dtype == AXS6_F32 ? go(&backward_kernel<float, float>) : go(&backward_kernel<float, __nv_bfloat16>);
    return teacher_dtype == AXS6_F32 ? go(&backward_kernel<__nv_bfloat16, float>) : go(&backward_kernel<__nv_bfloat16, __nv_bfloat16>);
}
