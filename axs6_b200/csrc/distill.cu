// Distillation of a student from a teacher's top logits, and its gradient.  Row r of the (rows, vocab) student logits z has `slots`
// pairs (index, teacher logit t); with temperature T
//     p_i = softmax(t / T) over the row's used slots        q_j = softmax(z / T) over the whole vocabulary
//     loss_r = T^2 sum_i p_i (log p_i - log q_(index i))     dz_j = T u_r (q_j - sum_(i: index i = j) p_i)
// u_r being the upstream gradient of loss_r.  A slot whose index lies outside [0, vocab) or whose teacher logit is -inf is unused;
// a row without a used slot has loss 0 and gradient 0, whatever its logits are.
//
// Bound: HBM.  Forward reads the logits once (online softmax: every thread keeps a running maximum and the sum relative to it),
// backward reads them once more and writes the gradient: 3 * rows * vocab * bytes in all.  Nothing of the vocabulary's length is kept
// between the two, only each row's maximum m and sum s: q = exp((z - m) / T) / s, with the difference taken first so that
// the exponent carries no rounding of a large log-sum.  Backward takes the rows in the other order, since the last of them are still in L2.
//
// One CTA of 256 threads works on a row, or on a segment of it where rows are few (the segments of a row are a thread-block cluster in the
// forward kernel, which joins their maxima and sums through distributed shared memory): several CTAs an SM are in different phases,
// so that the ends of rows hide under the others' loads.  16-byte pieces where the row is aligned, single values up to the first boundary and
// behind the last.  Sums are fp32 per thread (a few hundred terms) and joined in a fixed order.
//
// Measured, 8192 x 32000 bf16, 64 slots: forward 101 us (5.2 TB/s; the exp2 unit is 68 % busy), backward 157-167 us (6.3 TB/s); 1000 x 100001 fp32: 70
// and 150 us; 7 x 32000 bf16: 8.4 and 6.4 us.  Short rows (5000 values) pay 97 us a pass at 16384 rows for 25 us of bytes: the ends of a row.
#include <cuda_bf16.h>
#include <math_constants.h>

#include "common.cuh"

namespace axs6 {
namespace distill {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxSlots = 1024, kSlotRounds = kMaxSlots / kThreads;
constexpr int kMaxSegments = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
    const void *z, *t;
    const long long *index;
    long long rows, vocab, ldz, ldt, ldi;
    int slots;
    float temperature;
    float *row_loss;        // rows
    float4 *stats;          // a row's maximum of z, sum of exp((z - maximum) / T) (0: unused row), the same two of its used teacher logits
    int segments, shift;    // of a row: a power of two, and its logarithm
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

// Two fp32 values in one instruction
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void parts(f32x2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// 16 bytes of a row
template <typename T> struct Vec {
    static constexpr int n = 16 / (int)sizeof(T);
    union { uint4 raw; uint32_t w[4]; T v[n]; };
    __device__ __forceinline__ f32x2 two(int e) const
    {
        if (sizeof(T) == 4) return pair(__uint_as_float(w[(2 * e) & 3]), __uint_as_float(w[(2 * e + 1) & 3]));
        return pair(__uint_as_float(w[e & 3] << 16), __uint_as_float(w[e & 3] & 0xffff0000u));
    }
    __device__ __forceinline__ float top() const
    {
        if (sizeof(T) == 4) return fmaxf(fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])), fmaxf(__uint_as_float(w[2]), __uint_as_float(w[3])));
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(w);
        const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(m), __high2float(m));
    }
    // pair e of values, rounded to the type
    __device__ __forceinline__ void put(int e, float a, float b)
    {
        if (sizeof(T) == 4) { w[(2 * e) & 3] = __float_as_uint(a); w[(2 * e + 1) & 3] = __float_as_uint(b); return; }
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        w[e & 3] = *reinterpret_cast<const uint32_t *>(&h);
    }
};

// Values before the first 16-byte boundary of a row (at most vocab).
template <typename T> __device__ __forceinline__ int head_of(const T *row, long long vocab)
{
    const int mis = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    const int h = mis ? Vec<T>::n - mis : 0;
    return (long long)h < vocab ? h : (int)vocab;
}

// Pieces [from, to) of a row that segment `seg` has; the values before the first boundary are the first segment's, those behind the last
// piece the last one's.
struct Range { int head, pieces, from, to; };
template <typename T> __device__ __forceinline__ Range range_of(const Params &p, const T *row, int seg)
{
    Range r;
    r.head = head_of(row, p.vocab);
    r.pieces = (int)(p.vocab - r.head) / Vec<T>::n;
    r.from = (r.pieces >> p.shift) * seg;
    r.to = seg == p.segments - 1 ? r.pieces : r.from + (r.pieces >> p.shift);
    return r;
}

__device__ __forceinline__ int slot_index(const Params &p, long long j, float t) { return j >= 0 && j < p.vocab && t != -CUDART_INF_F ? (int)j : -1; }

// (m, s) of two parts of a row joined: the sum is relative to the maximum.
__device__ __forceinline__ void join(float &m, float &s, float m2, float s2, float c)
{
    const float top = fmaxf(m, m2), base = top == -CUDART_INF_F ? 0.0f : top;
    s = s * ex2((m - base) * c) + s2 * ex2((m2 - base) * c);
    m = top;
}

__device__ __forceinline__ uint32_t cluster_address(const void *shared, uint32_t rank)
{
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(shared)), "r"(rank));
    return a;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

template <typename T, typename Tt>
__global__ void __launch_bounds__(kThreads, 4) forward_kernel(const Params p)
{
    __shared__ int index_s[kMaxSlots];                              // -1: unused
    __shared__ float teacher_s[kMaxSlots], picked_s[kMaxSlots];
    __shared__ float part[2 * kWarps], teacher_stat[2];
    __shared__ float joined[2 * kMaxSegments];                      // in the first CTA of a row: every segment's maximum and sum
    const long long row = blockIdx.x >> p.shift;
    const int seg = (int)blockIdx.x & (p.segments - 1);
    const float c = kLog2e / p.temperature;
    const T *z = static_cast<const T *>(p.z) + row * p.ldz;
    const Tt *tl = static_cast<const Tt *>(p.t) + row * p.ldt;
    const long long *ix = p.index + row * p.ldi;
    const Range g = range_of(p, z, seg);
    const uint4 *zv = reinterpret_cast<const uint4 *>(z + g.head);

    // the first pieces are under way while the slots arrive
    constexpr int kUnroll = 4;
    Vec<T> v[kUnroll];
    int i = g.from + threadIdx.x;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
        if (i + u * kThreads < g.to) v[u].raw = __ldg(zv + i + u * kThreads);
    bool any = false;
    int mine[kSlotRounds];
#pragma unroll
    for (int x = 0; x < kSlotRounds; ++x) {
        const int k = threadIdx.x + x * kThreads;
        mine[x] = -1;
        if (k >= p.slots) continue;
        const float t = to_f(tl[k]);
        mine[x] = slot_index(p, ix[k], t);
        any |= mine[x] >= 0;
        if (seg == 0) { index_s[k] = mine[x]; teacher_s[k] = t; }
    }
    if (!__syncthreads_or(any)) {                                   // no used slot: the same in all segments of the row
        if (seg == 0 && threadIdx.x == 0) { p.row_loss[row] = 0.0f; p.stats[row] = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
        return;
    }
    if (p.segments > 1) cluster_arrive();                           // the segments' CTAs run: their shared memory may be written to
    float picked[kSlotRounds];
#pragma unroll
    for (int x = 0; x < kSlotRounds; ++x) picked[x] = seg == 0 && mine[x] >= 0 ? to_f(z[mine[x]]) : 0.0f;

    // one warp turns the teacher's logits into probabilities while the others begin
    if (seg == 0 && threadIdx.x >= kThreads - 32) {
        const int lane = threadIdx.x & 31;
        float tm = -CUDART_INF_F, ts = 0.0f;
        for (int k = lane; k < p.slots; k += 32)
            if (index_s[k] >= 0) tm = fmaxf(tm, teacher_s[k]);
        for (int o = 16; o; o >>= 1) tm = fmaxf(tm, __shfl_xor_sync(~0u, tm, o));
        for (int k = lane; k < p.slots; k += 32)
            if (index_s[k] >= 0) ts += ex2((teacher_s[k] - tm) * c);
        for (int o = 16; o; o >>= 1) ts += __shfl_xor_sync(~0u, ts, o);
        if (lane == 0) { teacher_stat[0] = tm; teacher_stat[1] = ts; }
    }

    float m = -CUDART_INF_F;
    f32x2 sum = pair(0.0f, 0.0f);
    const f32x2 c2 = pair(c, c);
    auto raise = [&](float top) {
        if (top > m) {
            const float f = ex2((m - top) * c);
            sum = mul2(sum, pair(f, f));
            m = top;
        }
    };
    auto one = [&](float w) {
        raise(w);
        sum = add2(sum, pair(w == -CUDART_INF_F ? 0.0f : ex2((w - m) * c), 0.0f));       // m is finite or +inf here unless w is -inf or NaN
    };
    auto piece = [&](const Vec<T> &w) {
        raise(w.top());
        const float base = m == -CUDART_INF_F ? 0.0f : m;
        const f32x2 back = pair(-base, -base);
#pragma unroll
        for (int e = 0; e < Vec<T>::n / 2; ++e) {
            float a, b;
            parts(mul2(add2(w.two(e), back), c2), a, b);
            sum = add2(sum, pair(ex2(a), ex2(b)));
        }
    };
    for (; i < g.to; i += kUnroll * kThreads) {
        Vec<T> w[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) w[u] = v[u];
        const int next = i + kUnroll * kThreads;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (next + u * kThreads < g.to) v[u].raw = __ldg(zv + next + u * kThreads);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (i + u * kThreads < g.to) piece(w[u]);
    }
    if (seg == 0 && (int)threadIdx.x < g.head) one(to_f(z[threadIdx.x]));
    if (seg == p.segments - 1)
        for (int j = g.head + g.pieces * Vec<T>::n + threadIdx.x; j < p.vocab; j += kThreads) one(to_f(z[j]));
    float s, s_odd;
    parts(sum, s, s_odd);
    s += s_odd;
    for (int o = 16; o; o >>= 1) join(m, s, __shfl_xor_sync(~0u, m, o), __shfl_xor_sync(~0u, s, o), c);
    if ((threadIdx.x & 31) == 0) { part[2 * (threadIdx.x >> 5)] = m; part[2 * (threadIdx.x >> 5) + 1] = s; }
    if (seg == 0) {
#pragma unroll
        for (int x = 0; x < kSlotRounds; ++x)
            if (threadIdx.x + x * kThreads < p.slots) picked_s[threadIdx.x + x * kThreads] = picked[x];
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        m = part[2 * (threadIdx.x & (kWarps - 1))]; s = part[2 * (threadIdx.x & (kWarps - 1)) + 1];
        for (int o = kWarps / 2; o; o >>= 1) join(m, s, __shfl_xor_sync(~0u, m, o), __shfl_xor_sync(~0u, s, o), c);
    }
    if (p.segments > 1) {
        __syncwarp();
        cluster_wait();
        if (threadIdx.x == 0) {
            const uint32_t a = cluster_address(joined + 2 * seg, 0);
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(m) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a + 4u), "f"(s) : "memory");
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (seg == 0 && threadIdx.x < 32) {
            m = -CUDART_INF_F; s = 0.0f;
            for (int x = 0; x < p.segments; ++x) join(m, s, joined[2 * x], joined[2 * x + 1], c);
        }
    }
    if (seg == 0 && threadIdx.x < 32) {
        const float tm = teacher_stat[0], ts = teacher_stat[1];
        float loss = 0.0f;
        // log p_i - log q_i in bits: (t_i - max t) c - log2 sum t - (z_i - m) c + log2 s
        const float lt = log2f(ts), lz = log2f(s), inv = 1.0f / ts;
        for (int k = threadIdx.x; k < p.slots; k += 32) {
            if (index_s[k] < 0) continue;
            const float a = (teacher_s[k] - tm) * c, prob = ex2(a) * inv;
            if (prob != 0.0f) loss += prob * ((a - lt) - ((picked_s[k] - m) * c - lz));
        }
        for (int o = 16; o; o >>= 1) loss += __shfl_xor_sync(~0u, loss, o);
        if (threadIdx.x == 0) {
            p.row_loss[row] = loss * (kLn2 * p.temperature * p.temperature);
            p.stats[row] = make_float4(m, s, tm, ts);
        }
    }
}

// Sum of the rows' losses, or their mean over the rows with a used slot, in 64 bits and in a fixed order; *count = that number of rows, at least 1.
__global__ void __launch_bounds__(1024) reduce_kernel(const float *row_loss, const float4 *stats, long long rows, int mean, float *out, float *count)
{
    __shared__ double sum_s[32];
    __shared__ long long cnt_s[32];
    pdl_wait();
    double sum = 0.0;
    long long cnt = 0;
#pragma unroll 8
    for (long long i = threadIdx.x; i < rows; i += 1024) { sum += (double)row_loss[i]; cnt += stats[i].y != 0.0f; }
    for (int o = 16; o; o >>= 1) { sum += __shfl_xor_sync(~0u, sum, o); cnt += __shfl_xor_sync(~0u, cnt, o); }
    if ((threadIdx.x & 31) == 0) { sum_s[threadIdx.x >> 5] = sum; cnt_s[threadIdx.x >> 5] = cnt; }
    __syncthreads();
    if (threadIdx.x < 32) {
        sum = sum_s[threadIdx.x]; cnt = cnt_s[threadIdx.x];
        for (int o = 16; o; o >>= 1) { sum += __shfl_xor_sync(~0u, sum, o); cnt += __shfl_xor_sync(~0u, cnt, o); }
        if (threadIdx.x == 0) {
            const double n = cnt ? (double)cnt : 1.0;
            *out = (float)(mean ? sum / n : sum);
            *count = (float)n;
        }
    }
}

template <typename T, typename Tt>
__global__ void __launch_bounds__(kThreads, 4) backward_kernel(const Params p)
{
    __shared__ __align__(16) int index_s[kMaxSlots];
    __shared__ float prob_s[kMaxSlots];
    const long long row = p.rows - 1 - (blockIdx.x >> p.shift);
    const int seg = (int)blockIdx.x & (p.segments - 1);
    const float c = kLog2e / p.temperature;
    const T *z = static_cast<const T *>(p.z) + row * p.ldz;
    T *grad = static_cast<T *>(p.grad) + row * p.ldg;
    const Tt *tl = static_cast<const Tt *>(p.t) + row * p.ldt;
    const long long *ix = p.index + row * p.ldi;
    // segments and boundaries by where the gradient lies; 16-byte pieces of both if the two rows lie alike
    const Range g = range_of(p, grad, seg);
    const uint4 *zv = reinterpret_cast<const uint4 *>(z + g.head);
    const bool alike = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(grad)) & 15u) == 0;
    // the first pieces are under way while the statistics and the slots arrive
    constexpr int kUnroll = 4;
    Vec<T> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
        if (alike && g.from + threadIdx.x + u * kThreads < g.to) v[u].raw = __ldg(zv + g.from + threadIdx.x + u * kThreads);
    const float4 st = p.stats[row];
    const float m = st.x, s = st.y;
    const bool used = s != 0.0f;
    const float up = p.upstream[row * p.upstream_stride] * p.temperature / (p.count ? *p.count : 1.0f);
    const float w = used ? up / s : 0.0f;
    // the row's slots, and the logits that they name, before the row itself
    const int low = seg == 0 ? 0 : g.head + g.from * Vec<T>::n, high = seg == p.segments - 1 ? (int)p.vocab : g.head + g.to * Vec<T>::n;
    int mine[kSlotRounds];
    float picked[kSlotRounds];
#pragma unroll
    for (int x = 0; x < kSlotRounds; ++x) {
        const int k = threadIdx.x + x * kThreads;
        mine[x] = -1;
        picked[x] = 0.0f;
        if (!used || k >= p.slots) { if (k < (p.slots + 3) / 4 * 4) index_s[k] = -1; continue; }
        const float t = to_f(tl[k]);
        const int j = slot_index(p, ix[k], t);
        index_s[k] = j;
        prob_s[k] = j >= 0 ? ex2((t - st.z) * c) / st.w : 0.0f;
        if (j < low || j >= high) continue;                          // -1 among them
        mine[x] = j;
        picked[x] = to_f(z[j]);
    }
    uint4 *gv = reinterpret_cast<uint4 *>(grad + g.head);
    if (!used) {
        for (int i = g.from + threadIdx.x; i < g.to; i += kThreads) __stcs(gv + i, make_uint4(0u, 0u, 0u, 0u));
    } else if (alike) {
        const f32x2 back = pair(-m, -m), c2 = pair(c, c), w2 = pair(w, w);
        for (int i = g.from + threadIdx.x; i < g.to; i += kUnroll * kThreads) {
            const int next = i + kUnroll * kThreads;
            Vec<T> x[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) x[u] = v[u];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (next + u * kThreads < g.to) v[u].raw = __ldg(zv + next + u * kThreads);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (i + u * kThreads >= g.to) continue;
                Vec<T> o;
#pragma unroll
                for (int e = 0; e < Vec<T>::n / 2; ++e) {
                    float a, b;
                    parts(mul2(add2(x[u].two(e), back), c2), a, b);
                    parts(mul2(pair(ex2(a), ex2(b)), w2), a, b);
                    o.put(e, a, b);
                }
                __stcs(gv + i + u * kThreads, o.raw);
            }
        }
    }
    auto one = [&](int j) { from_f(used ? ex2((to_f(z[j]) - m) * c) * w : 0.0f, grad[j]); };
    if (used && !alike)
        for (int j = g.head + g.from * Vec<T>::n + threadIdx.x; j < g.head + g.to * Vec<T>::n; j += kThreads) one(j);
    if (seg == 0 && (int)threadIdx.x < g.head) one(threadIdx.x);
    if (seg == p.segments - 1)
        for (int j = g.head + g.pieces * Vec<T>::n + threadIdx.x; j < p.vocab; j += kThreads) one(j);
    if (!used) return;
    __syncthreads();                                                 // also orders the stores above before those below
    // The first slot that names a place of this segment writes it, with the probabilities of all the slots that name it in slot order.
#pragma unroll
    for (int x = 0; x < kSlotRounds; ++x) {
        const int j = mine[x], k = threadIdx.x + x * kThreads;
        if (j < 0) continue;
        float prob = 0.0f;
        bool first = true;
        for (int o = 0; o < p.slots && first; o += 4) {
            const int4 q = *reinterpret_cast<const int4 *>(index_s + o);
            if (q.x != j && q.y != j && q.z != j && q.w != j) continue;
            const int four[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int y = 0; y < 4; ++y)
                if (four[y] == j) { prob += prob_s[o + y]; first = first && o + y >= k; }
        }
        if (first) from_f((ex2((picked[x] - m) * c) / s - prob) * up, grad[j]);
    }
}

static bool args_ok(const void *z, int dtype, int64_t rows, int64_t vocab, int64_t ldz, const void *t, int t_dtype, int64_t ldt,
                    const void *index, int64_t ldi, int64_t slots, float temperature)
{
    return valid_dtype(dtype) && valid_dtype(t_dtype) && rows >= 0 && vocab >= 1 && vocab < INT32_MAX / 2 && slots >= 1 && ldz >= 0 && ldt >= 0 &&
           ldi >= 0 && temperature > 0.0f && temperature <= 3.402823466e38f && (rows == 0 || (z && t && index));
}

// Segments of a row: doubled while the CTAs would not fill two on every SM and a segment keeps two rounds of a CTA's loads.
static int segments_of(const DeviceInfo &d, int64_t rows, int64_t vocab, int esize)
{
    int n = 1;
    while (n < kMaxSegments && rows * n < 2 * (int64_t)d.sms && vocab * esize / (2 * n) >= 2 * 4 * 16 * kThreads) n *= 2;
    return n;
}

}  // namespace distill
}  // namespace axs6

AXS6_API int axs6_distill_fwd(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t ld, const void *teacher, int teacher_dtype,
                              int64_t ld_teacher, const int64_t *index, int64_t ld_index, int64_t slots, float temperature, int reduction,
                              float *row_loss, float *row_stats, float *reduced, float *count, axs6_stream_t stream)
{
    using namespace axs6;
    using namespace axs6::distill;
    if (!args_ok(logits, dtype, rows, vocab, ld, teacher, teacher_dtype, ld_teacher, index, ld_index, slots, temperature) || reduction < 0 ||
        reduction > 2 || (rows && (!row_loss || !row_stats)) || (reduction && (!reduced || !count)))
        return AXS6_ERR_ARG;
    if (slots > kMaxSlots) return AXS6_ERR_UNSUPPORTED;
    if (!aligned16(row_stats)) return AXS6_ERR_ALIGN;
    const DeviceInfo &d = device_info();
    if (!d.valid || !d.ok) return AXS6_ERR_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Params p = {};
    p.z = logits; p.t = teacher; p.index = reinterpret_cast<const long long *>(index);
    p.rows = rows; p.vocab = vocab; p.ldz = ld; p.ldt = ld_teacher; p.ldi = ld_index; p.slots = (int)slots; p.temperature = temperature;
    p.row_loss = row_loss; p.stats = reinterpret_cast<float4 *>(row_stats);
    p.segments = segments_of(d, rows, vocab, dtype == AXS6_F32 ? 4 : 2);
    while ((1 << p.shift) < p.segments) ++p.shift;
    if (rows * p.segments > INT32_MAX) return AXS6_ERR_ARG;
    if (rows) {
        auto go = [&](auto kernel) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)(rows * p.segments), 1, 1);
            cfg.blockDim = dim3(kThreads, 1, 1);
            cfg.stream = st;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = (unsigned)p.segments;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = p.segments > 1 ? 1 : 0;
            const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
            note_cuda_error(e);
            count_launch();
            return e == cudaSuccess ? AXS6_OK : AXS6_ERR_LAUNCH;
        };
        const int rc = dtype == AXS6_F32
            ? (teacher_dtype == AXS6_F32 ? go(&forward_kernel<float, float>) : go(&forward_kernel<float, __nv_bfloat16>))
            : (teacher_dtype == AXS6_F32 ? go(&forward_kernel<__nv_bfloat16, float>) : go(&forward_kernel<__nv_bfloat16, __nv_bfloat16>));
        if (rc != AXS6_OK) return rc;
    }
    if (reduction) {
        if (launch_overlapped(true, reduce_kernel, 1, 1024, 0, st, row_loss, p.stats, (long long)rows, reduction == 2, reduced, count) != cudaSuccess)
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
    if (!aligned16(row_stats)) return AXS6_ERR_ALIGN;
    if (rows == 0) return AXS6_OK;
    const DeviceInfo &d = device_info();
    if (!d.valid || !d.ok) return AXS6_ERR_DEVICE;
    Params p = {};
    p.z = logits; p.t = teacher; p.index = reinterpret_cast<const long long *>(index);
    p.rows = rows; p.vocab = vocab; p.ldz = ld; p.ldt = ld_teacher; p.ldi = ld_index; p.slots = (int)slots; p.temperature = temperature;
    p.stats = reinterpret_cast<float4 *>(const_cast<float *>(row_stats)); p.segments = segments_of(d, rows, vocab, dtype == AXS6_F32 ? 4 : 2);
    while ((1 << p.shift) < p.segments) ++p.shift;
    if (rows * p.segments > INT32_MAX) return AXS6_ERR_ARG;
    p.grad = grad; p.ldg = ld_grad;
    p.upstream = upstream; p.upstream_stride = upstream_stride; p.count = count;
    auto go = [&](auto kernel) {
        kernel<<<(unsigned)(rows * p.segments), kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
        count_launch();
        return check_launch();
    };
    if (dtype == AXS6_F32)
        return teacher_dtype == AXS6_F32 ? go(&backward_kernel<float, float>) : go(&backward_kernel<float, __nv_bfloat16>);
    return teacher_dtype == AXS6_F32 ? go(&backward_kernel<__nv_bfloat16, float>) : go(&backward_kernel<__nv_bfloat16, __nv_bfloat16>);
}
