// Host side of the tensor-core attention kernels: alignment checks, tensor maps, launches.
#include "attn_bwd_kernel.cuh"
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
    if (p.o_low && !aligned16(p.o_low)) return false;
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

static RowData row_data(const Params &p)
{
    RowData w;
    w.padded = (p.q_len + kRows - 1) / kRows * kRows;
    const long long n = (long long)p.batch * p.q_heads * w.padded;
    w.shift = p.delta; w.delta = w.shift + n; w.log_sum = w.delta + n;
    return w;
}

template <int DP, bool kMask> static int bwd_launch(const Params &p, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
                                                    const CUtensorMap &mg, cudaStream_t st)
{
    const RowData w = row_data(p);
    const long long rows = (long long)p.batch * p.q_heads * w.padded;
    if (rows) {
        row_data_kernel<<<(unsigned)((rows + 15) / 16), 256, 0, st>>>(p, w, kMask);
        count_launch();
        const int rc = check_launch();
        if (rc != AXS6_OK) return rc;
    }
    if (p.k_len) {
        const auto kernel = &dkv_kernel<DP, kMask>;
        if (!ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), DkvSmem<DP>::kBytes)) return AXS6_ERR_LAUNCH;
        const unsigned grid = (unsigned)((p.k_len + kRows - 1) / kRows) * (unsigned)(p.batch * p.k_heads);
        kernel<<<grid, kBwdThreads, DkvSmem<DP>::kBytes, st>>>(mq, mk, mv, mg, p, w);
        count_launch();
        const int rc = check_launch();
        if (rc != AXS6_OK) return rc;
    }
    if (rows) {
        const auto kernel = &dq_kernel<DP, kMask>;
        if (!ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), DqSmem<DP>::kBytes)) return AXS6_ERR_LAUNCH;
        const unsigned grid = (unsigned)(w.padded / kRows) * (unsigned)(p.batch * p.q_heads);
        kernel<<<grid, kBwdThreads, DqSmem<DP>::kBytes, st>>>(mq, mk, mv, mg, p, w);
        count_launch();
        return check_launch();
    }
    return AXS6_OK;
}

}  // namespace tc

int64_t bwd_bf16_workspace(int64_t heads, int64_t q_len, bool mask)
{
    return heads * ((q_len + tc::kRows - 1) / tc::kRows * tc::kRows) * 4 * (mask ? 3 : 2);
}

int bwd_bf16(const Params &p, cudaStream_t st)
{
    using namespace tc;
    if (!aligned_for_tiles(p, true)) return AXS6_ERR_ALIGN;
    CUtensorMap mq, mk, mv, mg;
    const bool no_q = p.q_len == 0 || p.q_heads == 0, no_k = p.k_len == 0 || p.k_heads == 0;      // their tiles are never loaded
    if (!no_q && (!make_map(&mq, p.q.p, p.head_size, p.q_len, p.q_heads, p.batch, p.q.t, p.q.h, p.q.b) ||
                  !make_map(&mg, p.d_o.p, p.head_size, p.q_len, p.q_heads, p.batch, p.d_o.t, p.d_o.h, p.d_o.b))) return AXS6_ERR_DEVICE;
    if (!no_k && (!make_map(&mk, p.k.p, p.head_size, p.k_len, p.k_heads, p.batch, p.k.t, p.k.h, p.k.b) ||
                  !make_map(&mv, p.v.p, p.head_size, p.k_len, p.k_heads, p.batch, p.v.t, p.v.h, p.v.b))) return AXS6_ERR_DEVICE;
    if (no_q) { mq = mk; mg = mk; }
    if (no_k) { mk = mq; mv = mq; }
    const bool mask = p.mask_kind != kMaskNone;
    if (p.head_size <= 64) return mask ? bwd_launch<64, true>(p, mq, mk, mv, mg, st) : bwd_launch<64, false>(p, mq, mk, mv, mg, st);
    return mask ? bwd_launch<128, true>(p, mq, mk, mv, mg, st) : bwd_launch<128, false>(p, mq, mk, mv, mg, st);
}

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
