// Host side of the tensor-core attention kernels: alignment checks, tensor maps, launches.
#include "attn_fwd_kernel.cuh"

namespace axs6 {
namespace attn {
namespace tc {

static bool operand_ok(const View &v, int tokens, int heads, int batch)
{
    return aligned16(v.p) && (tokens <= 1 || (v.t % 8 == 0 && v.t > 0)) && (heads <= 1 || (v.h % 8 == 0 && v.h > 0)) &&
           (batch <= 1 || (v.b % 8 == 0 && v.b > 0));
}

bool aligned_for_tiles(const Params &p, bool backward)
{
    const View out = {p.out, p.out_b, p.out_h, p.out_t};
    bool ok = operand_ok(p.q, p.q_len, p.q_heads, p.batch) && operand_ok(p.k, p.k_len, p.k_heads, p.batch) &&
              operand_ok(p.v, p.k_len, p.k_heads, p.batch) && operand_ok(out, p.q_len, p.q_heads, p.batch);
    if (backward) {
        const View dq = {p.dq, p.dq_b, p.dq_h, p.dq_t}, dk = {p.dk, p.dk_b, p.dk_h, p.dk_t}, dv = {p.dv, p.dv_b, p.dv_h, p.dv_t};
        ok = ok && operand_ok(p.d_o, p.q_len, p.q_heads, p.batch) && operand_ok(dq, p.q_len, p.q_heads, p.batch) &&
             operand_ok(dk, p.k_len, p.k_heads, p.batch) && operand_ok(dv, p.k_len, p.k_heads, p.batch);
    }
    return ok;
}

template <int DP, bool kMask> static int fwd_launch(const Params &p, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t st)
{
    const auto kernel = &fwd_kernel<DP, kMask>;
    if (!ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), FwdSmem<DP>::kBytes)) return AXS6_ERR_LAUNCH;
    const unsigned grid = (unsigned)((p.q_len + 2 * kRows - 1) / (2 * kRows)) * (unsigned)(p.batch * p.q_heads);
    kernel<<<grid, kFwdThreads, FwdSmem<DP>::kBytes, st>>>(mq, mk, mv, p);
    count_launch();
    return check_launch();
}

}  // namespace tc

int fwd_bf16(const Params &p, cudaStream_t st)
{
    using namespace tc;
    if (!aligned_for_tiles(p, false)) return AXS6_ERR_ALIGN;
    CUtensorMap mq, mk, mv;
    // without keys nothing is loaded, and the maps of K and V stand in for tensors that need not exist
    const bool none = p.k_len == 0;
    if (!make_map(&mq, p.q.p, p.head_size, p.q_len, p.q_heads, p.batch, p.q.t, p.q.h, p.q.b)) return AXS6_ERR_DEVICE;
    if (none) { mk = mq; mv = mq; }
    else if (!make_map(&mk, p.k.p, p.head_size, p.k_len, p.k_heads, p.batch, p.k.t, p.k.h, p.k.b) ||
             !make_map(&mv, p.v.p, p.head_size, p.k_len, p.k_heads, p.batch, p.v.t, p.v.h, p.v.b)) return AXS6_ERR_DEVICE;
    const bool mask = p.mask_kind != kMaskNone;
    if (p.head_size <= 64) return mask ? fwd_launch<64, true>(p, mq, mk, mv, st) : fwd_launch<64, false>(p, mq, mk, mv, st);
    return mask ? fwd_launch<128, true>(p, mq, mk, mv, st) : fwd_launch<128, false>(p, mq, mk, mv, st);
}

}  // namespace attn
}  // namespace axs6

AXS6_API int axs6_attn_status(void)
{
    const axs6::DeviceInfo &d = axs6::device_info();
    if (!d.valid || !d.ok) return AXS6_ERR_DEVICE;
    int v = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&v, axs6::attn::tc::g_status, sizeof(v)) != cudaSuccess) return AXS6_ERR_DEVICE;
    if (v && cudaMemcpyToSymbol(axs6::attn::tc::g_status, &zero, sizeof(zero)) != cudaSuccess) return AXS6_ERR_DEVICE;
    return v;
}
