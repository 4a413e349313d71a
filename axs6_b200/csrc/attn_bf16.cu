// Host side of the tensor-core attention kernels: alignment checks, tensor maps, launches.
#include "attn_bwd_kernel.cuh"
#include "attn_few_kernel.cuh"
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

// Whether the few-queries kernel takes a call, and how the keys are cut.  It does when the stacked rows of a key head fit one tile, so that
// a key tile is read once instead of once a query head, and when the other kernel's CTAs of 256 queries would leave half of the SMs idle.  Chunks:
// about as many CTAs as are resident, whole key tiles each.  Twice as many even out batch entries of different lengths a little (16 entries of
// 1 to 8 Ki keys, 8 key heads of 128: 70 against 73 us) and cost elsewhere, in prologues and in the join (1 entry of 64 Ki keys, 8 heads of 64:
// 51 against 39 us).
constexpr int kFewPerSm = 2;

struct Plan { bool few; Few f; int64_t rows; };

static Plan plan_of(int64_t batch, int64_t q_heads, int64_t k_heads, int64_t q_len, int64_t k_len, int64_t window, int sms)
{
    Plan pl = {};
    const int64_t group = k_heads ? q_heads / k_heads : 1, rows = q_len * group;
    const int64_t wide = (q_len + 2 * kRows - 1) / (2 * kRows) * batch * q_heads;
    pl.few = rows <= kRows || 2 * wide <= sms;
    pl.rows = batch * k_heads * rows;
    int64_t span = (k_len + kKeys - 1) / kKeys;
    if (window) {                                                  // queries of one tile stand at most this many keys apart
        const int64_t seen = (window + (kRows + group - 1) / group + kKeys - 1) / kKeys + 1;
        if (seen < span) span = seen;
    }
    const int64_t tiles = (rows + kRows - 1) / kRows, ctas = tiles * batch * k_heads;
    int64_t chunks = ctas ? (kFewPerSm * (int64_t)sms + ctas - 1) / ctas : 1;
    if (chunks > span) chunks = span;
    if (chunks < 1) chunks = 1;
    const int64_t chunk = span ? (span + chunks - 1) / chunks : 1;
    pl.f.row_tiles = (int)tiles; pl.f.chunk = (int)chunk; pl.f.chunks = span ? (int)((span + chunk - 1) / chunk) : 1;
    return pl;
}

template <int DP, bool kMask> static int few_launch(const Params &p, Plan &pl, float *ws, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t st)
{
    const auto kernel = &few_kernel<DP, kMask>;
    if (!ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), FewSmem<DP>::kBytes)) return AXS6_ERR_LAUNCH;
    pl.f.out = ws; pl.f.stat = ws + (pl.f.chunks > 1 ? (int64_t)pl.f.chunks * pl.rows * DP : 0);
    const int64_t grid = (int64_t)p.batch * p.k_heads * pl.f.row_tiles * pl.f.chunks;
    if (grid > INT32_MAX) return AXS6_ERR_ARG;
    kernel<<<(unsigned)grid, kFewThreads, FewSmem<DP>::kBytes, st>>>(mk, mv, p, pl.f);
    count_launch();
    const int rc = check_launch();
    if (rc != AXS6_OK || pl.f.chunks == 1) return rc;
    if (launch_overlapped(true, join_kernel<DP>, (unsigned)((pl.rows + 3) / 4), 128, 0, st, p, pl.f) != cudaSuccess) return AXS6_ERR_LAUNCH;
    count_launch();
    return AXS6_OK;
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
        row_data_kernel<DP / 8><<<(unsigned)(rows * (DP / 8) / 1024), 256, 0, st>>>(p, w, kMask);
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
        if (launch_overlapped(p.k_len > 0, kernel, grid, kBwdThreads, DqSmem<DP>::kBytes, st, mq, mk, mv, mg, p, w) != cudaSuccess) return AXS6_ERR_LAUNCH;
        count_launch();
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
    if (no_q) mq = mg = mk;
    if (no_k) mk = mv = mq;
    const bool mask = p.mask_kind != kMaskNone;
    if (p.head_size <= 64) return mask ? bwd_launch<64, true>(p, mq, mk, mv, mg, st) : bwd_launch<64, false>(p, mq, mk, mv, mg, st);
    return mask ? bwd_launch<128, true>(p, mq, mk, mv, mg, st) : bwd_launch<128, false>(p, mq, mk, mv, mg, st);
}

int64_t fwd_bf16_workspace(int64_t batch, int64_t q_heads, int64_t k_heads, int64_t q_len, int64_t k_len, int64_t head_size, int64_t window)
{
    const DeviceInfo &d = device_info();
    if (!d.valid || batch * q_heads * q_len == 0) return 0;
    const tc::Plan pl = tc::plan_of(batch, q_heads, k_heads, q_len, k_len, window, d.sms);
    return pl.few && pl.f.chunks > 1 ? pl.f.chunks * pl.rows * ((head_size <= 64 ? 64 : 128) + 2) * 4 : 0;
}

int fwd_bf16(const Params &p, float *ws, int sms, cudaStream_t st)
{
    using namespace tc;
    if (!aligned_for_tiles(p, false)) return AXS6_ERR_ALIGN;
    CUtensorMap mq, mk, mv;
    // without keys nothing is loaded, and the maps of K and V stand in for tensors that need not exist
    const bool none = p.k_len == 0;
    if (!make_map(&mq, p.q.p, p.head_size, p.q_len, p.q_heads, p.batch, p.q.t, p.q.h, p.q.b)) return AXS6_ERR_DEVICE;
    const bool mask = p.mask_kind != kMaskNone;
    Plan pl = plan_of(p.batch, p.q_heads, p.k_heads, p.q_len, p.k_len, p.window, sms);
    const int box = pl.few ? kKeys : kRows;
    if (none) { mk = mq; mv = mq; }
    else if (!make_map(&mk, p.k.p, p.head_size, p.k_len, p.k_heads, p.batch, p.k.t, p.k.h, p.k.b, box) ||
             !make_map(&mv, p.v.p, p.head_size, p.k_len, p.k_heads, p.batch, p.v.t, p.v.h, p.v.b, box)) return AXS6_ERR_DEVICE;
    if (pl.few) {
        if (p.head_size <= 64) return mask ? few_launch<64, true>(p, pl, ws, mk, mv, st) : few_launch<64, false>(p, pl, ws, mk, mv, st);
        return mask ? few_launch<128, true>(p, pl, ws, mk, mv, st) : few_launch<128, false>(p, pl, ws, mk, mv, st);
    }
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
