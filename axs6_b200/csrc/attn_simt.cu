// Attention on the fp32 pipes: forward, and the backward pass that recomputes the probabilities.  For fp32 tensors, whose products
// the tensor cores would round to 11 bits.
//
// Forward, for 64 queries of one head: keys pass by in tiles of 64, x = scale Q K^T (+ mask), running maximum m and sum l of
// exp(x - m), O rescaled whenever m grows.  Backward with P = exp(x - m) / l recomputed per tile:
//     dV = P^T dO    dP = dO V^T    dS = P (dP - delta), delta = rowsum(dO O)    dQ = scale dS K    dK = scale dS^T Q
// in two kinds of CTAs: one per 64 queries for dQ, one per 64 keys for dK and dV, which also walks the query heads that share the key
// head; so every output has one writer and a fixed order of summation, without atomics.
//
// Bound: fp32 FMA pipe (4 D flops a pair forward; 6 D and 8 D in the two halves of the backward pass, which both recompute S and dP).  256 threads
// as 16 x 16; each owns 4 x 4 scores and 4 x D/16 outputs, operands in shared memory with rows padded by 16 bytes (a quarter warp's
// 16-byte reads of eight rows then fall into different banks): 12 wavefronts of shared memory for 64 FMA instructions.
// Measured: 64 heads of 64, 1024 x 1024: 628 us forward (27 TFLOP/s of 74), 1833 us backward; 16 heads, 512 x 512 with a mask: 84 and 158 us.
#include "attn_common.cuh"

namespace axs6 {
namespace attn {

constexpr int kTile = 64, kThreads = 256;
constexpr int kPStride = kTile + 4;

// rows [r0, r0 + 64) of a (token, value) matrix into shared memory, zeros outside [0, limit) and behind the head's size
template <int DP>
__device__ __forceinline__ void load_tile(float *dst, const float *src, long long stride, int r0, int limit, int d, bool vec)
{
    constexpr int S = DP + 4;
    if (vec) {
        for (int i = threadIdx.x; i < kTile * (DP / 4); i += kThreads) {
            const int r = i / (DP / 4), c = (i - r * (DP / 4)) * 4;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r0 + r < limit && c < d) v = *reinterpret_cast<const float4 *>(src + (r0 + r) * stride + c);
            *reinterpret_cast<float4 *>(dst + r * S + c) = v;
        }
    } else {
        for (int i = threadIdx.x; i < kTile * DP; i += kThreads) {
            const int r = i / DP, c = i - r * DP;
            dst[r * S + c] = (r0 + r < limit && c < d) ? src[(r0 + r) * stride + c] : 0.0f;
        }
    }
}

// acc[a][b] = sum over values of A[ty*4 + a] B[tx + 16 b]
template <int DP>
__device__ __forceinline__ void rows_by_rows(const float *A, const float *B, int ty, int tx, float acc[4][4])
{
    constexpr int S = DP + 4;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[a][b] = 0.0f;
#pragma unroll 4
    for (int c = 0; c < DP; c += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) x[a] = *reinterpret_cast<const float4 *>(A + (ty * 4 + a) * S + c);
#pragma unroll
        for (int b = 0; b < 4; ++b) y[b] = *reinterpret_cast<const float4 *>(B + (tx + 16 * b) * S + c);
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b)
                acc[a][b] = fmaf(x[a].w, y[b].w, fmaf(x[a].z, y[b].z, fmaf(x[a].y, y[b].y, fmaf(x[a].x, y[b].x, acc[a][b]))));
    }
}
// acc[a][e] += sum over k of P[ty*4 + a][k] B[k][column e], columns 64 (e / 4) + tx * 4 + e % 4
template <int DP>
__device__ __forceinline__ void rows_by_cols(const float *P, const float *B, int ty, int tx, float acc[4][DP / 16])
{
    constexpr int S = DP + 4;
#pragma unroll 2
    for (int k = 0; k < kTile; k += 4) {
        float4 w[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) w[a] = *reinterpret_cast<const float4 *>(P + (ty * 4 + a) * kPStride + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int g = 0; g < DP / 64; ++g) {
                const float4 y = *reinterpret_cast<const float4 *>(B + (k + kk) * S + g * 64 + tx * 4);
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const float f = kk == 0 ? w[a].x : kk == 1 ? w[a].y : kk == 2 ? w[a].z : w[a].w;
                    acc[a][4 * g + 0] = fmaf(f, y.x, acc[a][4 * g + 0]);
                    acc[a][4 * g + 1] = fmaf(f, y.y, acc[a][4 * g + 1]);
                    acc[a][4 * g + 2] = fmaf(f, y.z, acc[a][4 * g + 2]);
                    acc[a][4 * g + 3] = fmaf(f, y.w, acc[a][4 * g + 3]);
                }
            }
    }
}
template <int DP>
__device__ __forceinline__ void store_rows(float *dst, long long stride, int r0, int limit, int d, int ty, int tx, const float acc[4][DP / 16], const float f[4])
{
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int r = r0 + ty * 4 + a;
        if (r >= limit) continue;
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) {
            const int c = 64 * (e / 4) + tx * 4 + e % 4;
            if (c < d) dst[r * stride + c] = acc[a][e] * f[a];
        }
    }
}

// Whether every pair of 64 queries from i0 and 64 keys from j0 is visible but for a mask tensor.
__device__ __forceinline__ bool whole_tile(const Params &p, int i0, int j0, int keys)
{
    return i0 + kTile <= p.q_len && j0 + kTile <= keys && (!p.causal || j0 + kTile - 1 <= i0 + p.offset) &&
           (!p.window || j0 > i0 + kTile - 1 + p.offset - p.window);
}
// The mask's values for pairs (i0 + di(a), j0 + dj(c)), fetched before the products that they are added to; -inf hides a pair.
template <typename I, typename J> __device__ __forceinline__ void fetch_mask(const Params &p, int b, int h, float mk[4][4], I query, J key, int keys)
{
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int i = query(a, c), j = key(a, c);
            mk[a][c] = i < p.q_len && j < keys ? masked_score(p, 0.0f, b, h, i, j) : 0.0f;
        }
}

__device__ __forceinline__ bool vec_ok(const View &v, int d)
{
    return ((reinterpret_cast<uintptr_t>(v.p) & 15u) | ((v.b | v.h | v.t | d) & 3)) == 0;
}

template <int DP, bool kMask>
__global__ void __launch_bounds__(kThreads, 2) simt_fwd_kernel(const Params p)
{
    extern __shared__ __align__(16) float sm[];
    constexpr int S = DP + 4;
    float *Qs = sm, *Ks = Qs + kTile * S, *Vs = Ks + kTile * S, *Ps = Vs + kTile * S;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int bh = blockIdx.x % (p.batch * p.q_heads), h = bh % p.q_heads, b = bh / p.q_heads, kh = h / p.group;
    const int i0 = (int)((gridDim.x - 1 - blockIdx.x) / (p.batch * p.q_heads)) * kTile;      // the longest rows of a causal call first
    const int keys = keys_of(p, b);
    const float *q = static_cast<const float *>(p.q.p) + b * p.q.b + h * p.q.h, *k = static_cast<const float *>(p.k.p) + b * p.k.b + kh * p.k.h,
            *v = static_cast<const float *>(p.v.p) + b * p.v.b + kh * p.v.h;
    const bool qv = vec_ok(p.q, p.head_size), kv = vec_ok(p.k, p.head_size), vv = vec_ok(p.v, p.head_size);
    load_tile<DP>(Qs, q, p.q.t, i0, p.q_len, p.head_size, qv);
    float m[4], l[4], acc[4][DP / 16];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        m[a] = -CUDART_INF_F; l[a] = 0.0f;
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) acc[a][e] = 0.0f;
    }
    const int i1 = i0 + kTile < p.q_len ? i0 + kTile : p.q_len;
    const int end = end_key(p, i1, keys);
    for (int j0 = first_key(p, i0) / kTile * kTile; j0 < end; j0 += kTile) {
        __syncthreads();
        load_tile<DP>(Ks, k, p.k.t, j0, keys, p.head_size, kv);
        load_tile<DP>(Vs, v, p.v.t, j0, keys, p.head_size, vv);
        float mk[4][4];
        if (kMask) fetch_mask(p, b, h, mk, [&](int a, int) { return i0 + ty * 4 + a; }, [&](int, int c) { return j0 + tx + 16 * c; }, keys);
        const bool whole = whole_tile(p, i0, j0, keys);
        __syncthreads();
        float s[4][4];
        rows_by_rows<DP>(Qs, Ks, ty, tx, s);
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int i = i0 + ty * 4 + a;
            float top = m[a];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int j = j0 + tx + 16 * c;
                s[a][c] = whole || sees(p, i, j, keys) ? (kMask ? under_mask(s[a][c] * p.scale, mk[a][c]) : s[a][c] * p.scale) : -CUDART_INF_F;
                top = fmaxf(top, s[a][c]);
            }
            for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
            const float base = top == -CUDART_INF_F ? 0.0f : top;
            const float f = ex2((m[a] - base) * kLog2e);
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float e = ex2((s[a][c] - base) * kLog2e);
                Ps[(ty * 4 + a) * kPStride + tx + 16 * c] = e;
                sum += e;
            }
            for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            l[a] = l[a] * f + sum;
            m[a] = top;
#pragma unroll
            for (int e = 0; e < DP / 16; ++e) acc[a][e] *= f;
        }
        __syncwarp();                                                    // a warp reads back only the rows it wrote
        rows_by_cols<DP>(Ps, Vs, ty, tx, acc);
    }
    float inv[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        inv[a] = l[a] == 0.0f ? 0.0f : 1.0f / l[a];
        const int i = i0 + ty * 4 + a;
        if (tx == 0 && i < p.q_len) {
            const long long at = ((long long)b * p.q_heads + h) * p.q_len + i;
            p.row_max[at] = m[a];
            p.row_sum[at] = l[a];
            if (p.lse) p.lse[at] = l[a] == 0.0f ? -CUDART_INF_F : m[a] + log2f(l[a]) * kLn2;
        }
    }
    store_rows<DP>(static_cast<float *>(p.out) + b * p.out_b + h * p.out_h, p.out_t, i0, p.q_len, p.head_size, ty, tx, acc, inv);
}

// delta = rowsum(dO * O): one warp a row.
__global__ void __launch_bounds__(256) delta_kernel(const Params p)
{
    const long long rows = (long long)p.batch * p.q_heads * p.q_len;
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int i = (int)(row % p.q_len), h = (int)(row / p.q_len % p.q_heads), b = (int)(row / p.q_len / p.q_heads);
    const float *o = static_cast<const float *>(p.o.p) + b * p.o.b + h * p.o.h + i * p.o.t;
    const float *g = static_cast<const float *>(p.d_o.p) + b * p.d_o.b + h * p.d_o.h + i * p.d_o.t;
    float s = 0.0f;
    for (int c = threadIdx.x & 31; c < p.head_size; c += 32) s = fmaf(o[c], g[c], s);
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(~0u, s, x);
    if ((threadIdx.x & 31) == 0) p.delta[row] = s;
}

template <int DP, bool kMask> __device__ __forceinline__ void dq_body(const Params &p, float *sm, uint32_t block, uint32_t blocks)
{
    constexpr int S = DP + 4;
    float *Qs = sm, *Gs = Qs + kTile * S, *Ks = Gs + kTile * S, *Vs = Ks + kTile * S, *Ds = Vs + kTile * S;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int bh = block % (p.batch * p.q_heads), h = bh % p.q_heads, b = bh / p.q_heads, kh = h / p.group;
    const int i0 = (int)((blocks - 1 - block) / (p.batch * p.q_heads)) * kTile;
    const int keys = keys_of(p, b);
    const float *q = static_cast<const float *>(p.q.p) + b * p.q.b + h * p.q.h, *k = static_cast<const float *>(p.k.p) + b * p.k.b + kh * p.k.h,
            *v = static_cast<const float *>(p.v.p) + b * p.v.b + kh * p.v.h, *g = static_cast<const float *>(p.d_o.p) + b * p.d_o.b + h * p.d_o.h;
    const bool kv = vec_ok(p.k, p.head_size), vv = vec_ok(p.v, p.head_size);
    load_tile<DP>(Qs, q, p.q.t, i0, p.q_len, p.head_size, vec_ok(p.q, p.head_size));
    load_tile<DP>(Gs, g, p.d_o.t, i0, p.q_len, p.head_size, vec_ok(p.d_o, p.head_size));
    float m[4], inv[4], delta[4], acc[4][DP / 16];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        const int i = i0 + ty * 4 + a;
        const long long at = ((long long)b * p.q_heads + h) * p.q_len + i;
        const float l = i < p.q_len ? p.row_sum[at] : 0.0f;
        m[a] = l == 0.0f ? 0.0f : p.row_max[at];
        inv[a] = l == 0.0f ? 0.0f : 1.0f / l;
        delta[a] = i < p.q_len ? p.delta[at] : 0.0f;
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) acc[a][e] = 0.0f;
    }
    const int i1 = i0 + kTile < p.q_len ? i0 + kTile : p.q_len;
    const int end = end_key(p, i1, keys);
    for (int j0 = first_key(p, i0) / kTile * kTile; j0 < end; j0 += kTile) {
        __syncthreads();
        load_tile<DP>(Ks, k, p.k.t, j0, keys, p.head_size, kv);
        load_tile<DP>(Vs, v, p.v.t, j0, keys, p.head_size, vv);
        __syncthreads();
        float s[4][4], d[4][4], mk[4][4];
        if (kMask) fetch_mask(p, b, h, mk, [&](int a, int) { return i0 + ty * 4 + a; }, [&](int, int c) { return j0 + tx + 16 * c; }, keys);
        const bool whole = whole_tile(p, i0, j0, keys);
        rows_by_rows<DP>(Qs, Ks, ty, tx, s);
        rows_by_rows<DP>(Gs, Vs, ty, tx, d);
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int i = i0 + ty * 4 + a, j = j0 + tx + 16 * c;
                const float x = whole || sees(p, i, j, keys) ? (kMask ? under_mask(s[a][c] * p.scale, mk[a][c]) : s[a][c] * p.scale) : -CUDART_INF_F;
                Ds[(ty * 4 + a) * kPStride + tx + 16 * c] = x == -CUDART_INF_F ? 0.0f : ex2((x - m[a]) * kLog2e) * inv[a] * (d[a][c] - delta[a]);
            }
        __syncwarp();
        rows_by_cols<DP>(Ds, Ks, ty, tx, acc);
    }
    const float f[4] = {p.scale, p.scale, p.scale, p.scale};
    store_rows<DP>(static_cast<float *>(p.dq) + b * p.dq_b + h * p.dq_h, p.dq_t, i0, p.q_len, p.head_size, ty, tx, acc, f);
}

template <int DP, bool kMask> __device__ __forceinline__ void dkv_body(const Params &p, float *sm, uint32_t block)
{
    constexpr int S = DP + 4;
    float *Ks = sm, *Vs = Ks + kTile * S, *Qs = Vs + kTile * S, *Gs = Qs + kTile * S, *Ps = Gs + kTile * S, *Ds = Ps + kTile * kPStride;
    float *Ms = Ds + kTile * kPStride, *Is = Ms + kTile, *Es = Is + kTile;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int bh = block % (p.batch * p.k_heads), kh = bh % p.k_heads, b = bh / p.k_heads;
    const int j0 = (int)(block / (p.batch * p.k_heads)) * kTile;
    const int keys = keys_of(p, b);
    const float *k = static_cast<const float *>(p.k.p) + b * p.k.b + kh * p.k.h, *v = static_cast<const float *>(p.v.p) + b * p.v.b + kh * p.v.h;
    load_tile<DP>(Ks, k, p.k.t, j0, keys, p.head_size, vec_ok(p.k, p.head_size));
    load_tile<DP>(Vs, v, p.v.t, j0, keys, p.head_size, vec_ok(p.v, p.head_size));
    const bool qv = vec_ok(p.q, p.head_size), gv = vec_ok(p.d_o, p.head_size);
    float ak[4][DP / 16], av[4][DP / 16];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) { ak[a][e] = 0.0f; av[a][e] = 0.0f; }
    const int j1 = j0 + kTile < keys ? j0 + kTile : keys;
    const int end = j0 < keys ? end_query(p, j1) : 0;
    for (int h = kh * p.group; h < (kh + 1) * p.group; ++h) {
        const float *q = static_cast<const float *>(p.q.p) + b * p.q.b + h * p.q.h, *g = static_cast<const float *>(p.d_o.p) + b * p.d_o.b + h * p.d_o.h;
        for (int i0 = first_query(p, j0) / kTile * kTile; i0 < end; i0 += kTile) {
            __syncthreads();
            load_tile<DP>(Qs, q, p.q.t, i0, p.q_len, p.head_size, qv);
            load_tile<DP>(Gs, g, p.d_o.t, i0, p.q_len, p.head_size, gv);
            if (threadIdx.x < kTile) {
                const int i = i0 + threadIdx.x;
                const long long at = ((long long)b * p.q_heads + h) * p.q_len + i;
                const float l = i < p.q_len ? p.row_sum[at] : 0.0f;
                Ms[threadIdx.x] = l == 0.0f ? 0.0f : p.row_max[at];
                Is[threadIdx.x] = l == 0.0f ? 0.0f : 1.0f / l;
                Es[threadIdx.x] = i < p.q_len ? p.delta[at] : 0.0f;
            }
            __syncthreads();
            float s[4][4], d[4][4], mk[4][4];
            if (kMask) fetch_mask(p, b, h, mk, [&](int, int c) { return i0 + tx + 16 * c; }, [&](int a, int) { return j0 + ty * 4 + a; }, keys);
            const bool whole = whole_tile(p, i0, j0, keys);
            rows_by_rows<DP>(Ks, Qs, ty, tx, s);
            rows_by_rows<DP>(Vs, Gs, ty, tx, d);
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int n = tx + 16 * c, i = i0 + n, j = j0 + ty * 4 + a;
                    const float x = whole || sees(p, i, j, keys) ? (kMask ? under_mask(s[a][c] * p.scale, mk[a][c]) : s[a][c] * p.scale) : -CUDART_INF_F;
                    const float w = x == -CUDART_INF_F ? 0.0f : ex2((x - Ms[n]) * kLog2e) * Is[n];
                    Ps[(ty * 4 + a) * kPStride + n] = w;
                    Ds[(ty * 4 + a) * kPStride + n] = w == 0.0f ? 0.0f : w * (d[a][c] - Es[n]);
                }
            __syncwarp();
            rows_by_cols<DP>(Ps, Gs, ty, tx, av);
            rows_by_cols<DP>(Ds, Qs, ty, tx, ak);
        }
    }
    const float fk[4] = {p.scale, p.scale, p.scale, p.scale}, fv[4] = {1.f, 1.f, 1.f, 1.f};
    store_rows<DP>(static_cast<float *>(p.dk) + b * p.dk_b + kh * p.dk_h, p.dk_t, j0, p.k_len, p.head_size, ty, tx, ak, fk);
    store_rows<DP>(static_cast<float *>(p.dv) + b * p.dv_b + kh * p.dv_h, p.dv_t, j0, p.k_len, p.head_size, ty, tx, av, fv);
}

// The CTAs of both halves of the backward pass in one launch, those of dK and dV, which do more, first: small calls have no second tail.
template <int DP, bool kMask> __global__ void __launch_bounds__(kThreads, DP == 64 ? 2 : 1) simt_bwd_kernel(const Params p, const uint32_t key_blocks)
{
    extern __shared__ __align__(16) float sm[];
    if (blockIdx.x < key_blocks) dkv_body<DP, kMask>(p, sm, blockIdx.x);
    else dq_body<DP, kMask>(p, sm, blockIdx.x - key_blocks, gridDim.x - key_blocks);
}

template <int DP> static int fwd_t(const Params &p, cudaStream_t st)
{
    const auto kernel = p.mask_kind == kMaskNone ? &simt_fwd_kernel<DP, false> : &simt_fwd_kernel<DP, true>;
    const int smem = (3 * kTile * (DP + 4) + kTile * kPStride) * 4;
    if (!ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), smem)) return AXS6_ERR_LAUNCH;
    const unsigned grid = (unsigned)((p.q_len + kTile - 1) / kTile) * (unsigned)(p.batch * p.q_heads);
    kernel<<<grid, kThreads, smem, st>>>(p);
    count_launch();
    return check_launch();
}
template <int DP> static int bwd_t(const Params &p, cudaStream_t st)
{
    const long long rows = (long long)p.batch * p.q_heads * p.q_len;
    if (rows) {
        delta_kernel<<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p);
        count_launch();
        const int rc = check_launch();
        if (rc != AXS6_OK) return rc;
    }
    const auto kernel = p.mask_kind == kMaskNone ? &simt_bwd_kernel<DP, false> : &simt_bwd_kernel<DP, true>;
    const int smem = (4 * kTile * (DP + 4) + 2 * kTile * kPStride + 3 * kTile) * 4;
    if (!ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), smem)) return AXS6_ERR_LAUNCH;
    const uint32_t key_blocks = (uint32_t)((p.k_len + kTile - 1) / kTile) * (uint32_t)(p.batch * p.k_heads);
    const uint32_t query_blocks = (uint32_t)((p.q_len + kTile - 1) / kTile) * (uint32_t)(p.batch * p.q_heads);
    kernel<<<key_blocks + query_blocks, kThreads, smem, st>>>(p, key_blocks);
    count_launch();
    return check_launch();
}

int fwd_fp32(const Params &p, cudaStream_t st) { return p.head_size <= 64 ? fwd_t<64>(p, st) : fwd_t<128>(p, st); }
int bwd_fp32(const Params &p, cudaStream_t st) { return p.head_size <= 64 ? bwd_t<64>(p, st) : bwd_t<128>(p, st); }

}  // namespace attn
}  // namespace axs6
