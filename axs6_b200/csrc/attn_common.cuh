// What the attention kernels share: the parameters of a call, which keys a query sees, and scores under a mask tensor.
#pragma once
#include <cuda_bf16.h>
#include <math_constants.h>

#include "common.cuh"

namespace axs6 {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
enum { kMaskNone = 0, kMaskKept = 1, kMaskAddF32 = 2, kMaskAddBf16 = 3 };

struct View { const void *p; long long b, h, t; };        // (batch, head, token, value): strides in elements, values adjacent

struct Params {
    View q, k, v, o, d_o;                   // o: forward's output / backward's input
    void *out, *dq, *dk, *dv;               // written tensors, with the strides below
    void *o_low;                            // null, or what rounding left of o (bf16), laid out like it
    long long out_b, out_h, out_t, dq_b, dq_h, dq_t, dk_b, dk_h, dk_t, dv_b, dv_h, dv_t;
    float *row_max, *row_sum, *lse;         // (batch, q_heads, q_len)
    float *delta;                           // the same shape, workspace of the backward pass
    int batch, q_heads, k_heads, group, q_len, k_len, head_size;
    int offset;                             // k_len - q_len: query i stands at key i + offset
    int causal, window;                     // window 0: none
    const int *key_lengths;                 // per batch entry, or null
    float scale;
    const void *mask;
    int mask_kind;
    long long mask_b, mask_h, mask_q, mask_k;
};

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ int keys_of(const Params &p, int b)
{
    if (!p.key_lengths) return p.k_len;
    const int n = p.key_lengths[b];
    return n < 0 ? 0 : (n > p.k_len ? p.k_len : n);
}
// Keys [first_key, end_key) hold everything that queries [i0, i1) can see by causality, window and length.
__device__ __forceinline__ int first_key(const Params &p, int i0)
{
    const int a = p.window ? i0 + p.offset - p.window + 1 : 0;
    return a > 0 ? a : 0;
}
__device__ __forceinline__ int end_key(const Params &p, int i1, int keys)
{
    const int e = p.causal ? i1 + p.offset : keys;
    return e < keys ? (e < 0 ? 0 : e) : keys;
}
// Queries [first_query, end_query) hold everything that sees one of keys [j0, j1).
__device__ __forceinline__ int first_query(const Params &p, int j0)
{
    const int a = p.causal ? j0 - p.offset : 0;
    return a > 0 ? a : 0;
}
__device__ __forceinline__ int end_query(const Params &p, int j1)
{
    const int e = p.window ? j1 - 1 - p.offset + p.window : p.q_len;
    return e < p.q_len ? (e < 0 ? 0 : e) : p.q_len;
}
__device__ __forceinline__ bool sees(const Params &p, int i, int j, int keys)
{
    return i < p.q_len && j < keys && (!p.causal || j <= i + p.offset) && (!p.window || j > i + p.offset - p.window);
}
// Score of a visible pair: scaled product plus mask; -inf where the mask hides it, whatever the product is.
__device__ __forceinline__ float masked_score(const Params &p, float x, int b, int h, int i, int j)
{
    if (p.mask_kind == kMaskNone) return x;
    const long long at = b * p.mask_b + h * p.mask_h + i * p.mask_q + j * p.mask_k;
    if (p.mask_kind == kMaskKept) return static_cast<const unsigned char *>(p.mask)[at] ? x : -CUDART_INF_F;
    const float m = p.mask_kind == kMaskAddF32 ? static_cast<const float *>(p.mask)[at]
                                               : __bfloat162float(static_cast<const __nv_bfloat16 *>(p.mask)[at]);
    return m == -CUDART_INF_F ? m : x + m;
}

// The same with what masked_score gave for a score of 0: the mask's value, 0 where a truth value keeps the pair.
__device__ __forceinline__ float under_mask(float x, float m) { return m == -CUDART_INF_F ? m : x + m; }

// Implemented by the translation units of the kernels.
int fwd_fp32(const Params &p, cudaStream_t st);
int bwd_fp32(const Params &p, cudaStream_t st);

}  // namespace attn
}  // namespace axs6
