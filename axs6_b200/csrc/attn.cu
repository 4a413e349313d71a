// C entry points of attention: checks, parameters, and the choice of kernels by the tensors' type.
#include <math.h>

#include "attn_common.cuh"

namespace axs6 {
namespace attn {

int fwd_bf16(const Params &p, float *ws, int sms, cudaStream_t st);
int64_t fwd_bf16_workspace(int64_t batch, int64_t q_heads, int64_t k_heads, int64_t q_len, int64_t k_len, int64_t head_size, int64_t window);
int bwd_bf16(const Params &p, cudaStream_t st);
int64_t bwd_bf16_workspace(int64_t heads, int64_t q_len, bool mask);

static int64_t rows_of(const axs6_attn_args &a) { return a.batch * a.q_heads * a.q_len; }

static bool sizes_ok(const axs6_attn_args &a)
{
    const int64_t most = 1 << 30;
    return valid_dtype(a.dtype) && a.batch >= 0 && a.q_heads >= 0 && a.k_heads >= 0 && a.q_len >= 0 && a.k_len >= 0 && a.head_size >= 1 &&
           a.batch < most && a.q_heads < most && a.k_heads < most && a.q_len < most && a.k_len < most && a.window >= 0 &&
           (a.k_heads == 0 ? a.q_heads == 0 : a.q_heads % a.k_heads == 0) && a.batch * a.q_heads < most &&
           a.mask_kind >= AXS6_MASK_NONE && a.mask_kind <= AXS6_MASK_ADD_BF16;
}

static int fill(Params &p, const axs6_attn_args &a, bool backward)
{
    if (!sizes_ok(a) || !(a.scale > 0.0f) || !isfinite(a.scale)) return AXS6_ERR_ARG;
    if (a.window && !a.causal) return AXS6_ERR_ARG;
    if (a.head_size > 128) return AXS6_ERR_UNSUPPORTED;
    const bool has_q = a.batch && a.q_heads && a.q_len, has_k = a.batch && a.k_heads && a.k_len;
    if (has_q && (!a.q || !a.o || !a.row_max || !a.row_sum)) return AXS6_ERR_ARG;
    if (has_k && (!a.k || !a.v)) return AXS6_ERR_ARG;
    if (has_q && has_k && a.mask_kind != AXS6_MASK_NONE && !a.mask) return AXS6_ERR_ARG;
    if (backward && ((has_q && (!a.d_o || !a.dq)) || (has_k && (!a.dk || !a.dv)))) return AXS6_ERR_ARG;
    // tiles of 64 rows or more, one CTA each, in one grid dimension
    if ((a.q_len / 64 + 1) * a.batch * a.q_heads >= INT32_MAX || (a.k_len / 64 + 1) * a.batch * a.k_heads >= INT32_MAX) return AXS6_ERR_ARG;
    auto view = [](const void *t, const int64_t *s) { View v; v.p = t; v.b = s[0]; v.h = s[1]; v.t = s[2]; return v; };
    p.q = view(a.q, a.q_strides); p.k = view(a.k, a.k_strides); p.v = view(a.v, a.v_strides);
    p.o = view(a.o, a.o_strides); p.d_o = view(a.d_o, a.d_o_strides);
    p.out = a.o; p.out_b = a.o_strides[0]; p.out_h = a.o_strides[1]; p.out_t = a.o_strides[2];
    p.dq = a.dq; p.dq_b = a.dq_strides[0]; p.dq_h = a.dq_strides[1]; p.dq_t = a.dq_strides[2];
    p.dk = a.dk; p.dk_b = a.dk_strides[0]; p.dk_h = a.dk_strides[1]; p.dk_t = a.dk_strides[2];
    p.dv = a.dv; p.dv_b = a.dv_strides[0]; p.dv_h = a.dv_strides[1]; p.dv_t = a.dv_strides[2];
    p.row_max = a.row_max; p.row_sum = a.row_sum; p.lse = a.lse; p.o_low = a.o_low;
    p.batch = (int)a.batch; p.q_heads = (int)a.q_heads; p.k_heads = (int)a.k_heads; p.group = a.k_heads ? (int)(a.q_heads / a.k_heads) : 1;
    p.q_len = (int)a.q_len; p.k_len = (int)a.k_len; p.head_size = (int)a.head_size; p.offset = p.k_len - p.q_len;
    p.causal = a.causal != 0; p.window = (int)(a.window < a.k_len ? a.window : a.k_len);      // a wider window hides nothing more
    if (a.window && p.window == 0) p.window = 1;
    p.key_lengths = a.key_lengths; p.scale = a.scale;
    p.mask = a.mask; p.mask_kind = a.mask_kind;
    p.mask_b = a.mask_strides[0]; p.mask_h = a.mask_strides[1]; p.mask_q = a.mask_strides[2]; p.mask_k = a.mask_strides[3];
    return AXS6_OK;
}

static int64_t workspace(const axs6_attn_args &a, bool backward)
{
    const int64_t window = a.window < a.k_len ? a.window : a.k_len;          // as in the call
    if (!backward)
        return a.dtype == AXS6_F32 ? 0 : fwd_bf16_workspace(a.batch, a.q_heads, a.k_heads, a.q_len, a.k_len, a.head_size, a.window && !window ? 1 : window);
    return a.dtype == AXS6_F32 ? rows_of(a) * 4 : bwd_bf16_workspace(a.batch * a.q_heads, a.q_len, a.mask_kind != AXS6_MASK_NONE);   // delta, ...
}

}  // namespace attn
}  // namespace axs6

AXS6_API int64_t axs6_attn_workspace_bytes(const axs6_attn_args *args, int backward)
{
    if (!args || !axs6::attn::sizes_ok(*args)) return 0;
    return axs6::attn::workspace(*args, backward != 0);
}

AXS6_API int axs6_attn_fwd(const axs6_attn_args *args, axs6_stream_t stream)
{
    using namespace axs6;
    if (!args) return AXS6_ERR_ARG;
    attn::Params p = {};
    const int rc = attn::fill(p, *args, false);
    if (rc != AXS6_OK) return rc;
    if (attn::rows_of(*args) == 0) return AXS6_OK;
    const DeviceInfo &d = device_info();
    if (!d.valid || !d.ok) return AXS6_ERR_DEVICE;
    const int64_t need = attn::workspace(*args, false);
    if (need && (!args->workspace || args->workspace_bytes < need)) return AXS6_ERR_WORKSPACE;
    if (!aligned16(args->workspace)) return AXS6_ERR_ALIGN;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return args->dtype == AXS6_F32 ? attn::fwd_fp32(p, st) : attn::fwd_bf16(p, static_cast<float *>(args->workspace), d.sms, st);
}

AXS6_API int axs6_attn_bwd(const axs6_attn_args *args, axs6_stream_t stream)
{
    using namespace axs6;
    if (!args) return AXS6_ERR_ARG;
    attn::Params p = {};
    const int rc = attn::fill(p, *args, true);
    if (rc != AXS6_OK) return rc;
    if (attn::rows_of(*args) == 0 && args->batch * args->k_heads * args->k_len == 0) return AXS6_OK;
    const int64_t need = attn::workspace(*args, true);
    if (need && (!args->workspace || args->workspace_bytes < need)) return AXS6_ERR_WORKSPACE;
    if (!aligned16(args->workspace)) return AXS6_ERR_ALIGN;
    const DeviceInfo &d = device_info();
    if (!d.valid || !d.ok) return AXS6_ERR_DEVICE;
    p.delta = static_cast<float *>(args->workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return args->dtype == AXS6_F32 ? attn::bwd_fp32(p, st) : attn::bwd_bf16(p, st);
}
