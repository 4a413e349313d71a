// Attention forward on the tensor cores (bf16 tensors, fp32 scores, sums and output accumulator).
//
// A CTA owns 256 queries of one head as two tiles of 128 and walks the keys in tiles of 128:
//     S_t = Q_t K_j^T  (tensor memory)    P_t = exp2(c S_t - c m)  (bf16, over S_t's columns)    O_t += P_t V_j  (tensor memory)
// with c = scale log2 e and the running reference m per row.  m is only raised, and O_t and the sum rescaled, when a row's maximum exceeds
// it by more than 8 in base 2: any reference gives the same quotient O / l, exp2 stays below 2^8, and the pass over O runs in the first few
// steps only.  P is rounded to bf16 because the tensor cores multiply it with V; the sum l takes the unrounded values, so the rounding
// errors of a row's P average out instead of shifting it.
//
// Warps 0-15: softmax, two threads a row with 64 scores each: warps 0-3 and 4-7 the two halves of tile 0's keys, warps 8-15 those of tile 1.  The
// two warps that share 32 rows exchange their maxima through shared memory and keep the same reference.  Warp 16: products.  Warp 17: loads.
// (Warps 18 and 19 only complete the warpgroup that hands its registers over.)  A row's softmax is a chain of dependent instructions; with
// one thread a row and two softmax warps on a scheduler the exponential unit was half idle, whatever the length of a tile.
//
// Score tiles (tile 0 and tile 1 in turn) rotate through the tensor memory that two output tiles leave: 2 buffers at D = 128, 3 at D = 64.  The
// scores of unit u + buffers are computed behind P V of unit u; tcgen05 instructions of one thread complete in order, so they may overwrite its P.
// Tiles of 64 keys with twice the buffers were 10 % slower at D = 128: an M = 128, K = 16 product takes 64 clocks for any N up to 128.
//
// Bound: tensor cores, 4 D flops a pair (1024 clocks a tile of 128 x 128 at D = 128, 768 at D = 64), and one exp2 a pair (16 a clock: 1024
// clocks).  Measured: D = 128, 32 / 8 heads, 8192 x 8192: 900 us, 1222 TFLOP/s, where the power cap holds a plain bf16 GEMM to 1393; causal 477 us,
// 1150; D = 64, 64 heads, 4096 x 4096: 375 us, 733 TFLOP/s, exp2 unit 72 % busy.  A CTA's start, end and the gap to the next one take 6 us, which
// is what short sequences pay (16 x 8 heads, 1024 x 1024, causal: 50 us for 15 us of tiles).
#pragma once
#include "attn_tc.cuh"

namespace axs6 {
namespace attn {
namespace tc {

constexpr int kFwdThreads = 640;
// Registers: launched with 96 a thread, 5 x 96 = 480 for the five warpgroups; the softmax warpgroups take 112 each, the one that loads and issues
// keeps 32.
constexpr int kRegsMore = 112, kRegsLess = 32;

template <int DP> struct FwdSmem {
    static constexpr uint32_t kTile = kBox * (DP / 64);
    static constexpr int kStages = DP == 64 ? 8 : 4;
    static constexpr int kBufs = DP == 64 ? 3 : 2;
    static constexpr uint32_t kRing = 2 * kTile, kTops = kRing + kStages * kTile;
    static constexpr uint32_t kBars = kTops + 8 * kRows * 4;                     // maxima (of two steps), then sums, of a row's two halves
    static constexpr uint32_t kBytes = kBars + 512 + 1024;
};

template <int DP, bool kMask>
__global__ void __launch_bounds__(kFwdThreads, 1)
fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Params p)
{
    typedef FwdSmem<DP> L;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t *gen = raw + (base - smem_u32(raw));
    const uint32_t bars = base + L::kBars;
    // of tile t, of score buffer x
    constexpr int kBufs = L::kBufs;
    const auto q_full = [&](int t) { return bars + 8u * t; };
    const auto o_full = [&](int t) { return bars + 16u + 8u * t; };
    const auto o_done = [&](int t, int j) { return bars + 32u + 16u * t + 8u * (j & 1); };
    const auto s_full = [&](int x) { return bars + 64u + 8u * x; };
    const auto p_full = [&](int x) { return bars + 88u + 8u * x; };
    const uint32_t fix = bars + 112u;
    const auto kv_full = [&](int s) { return bars + 120u + 8u * s; };
    const auto kv_empty = [&](int s) { return bars + 120u + 8u * (L::kStages + s); };
    constexpr uint32_t kSlot = 120 + 16 * L::kStages;
    volatile uint32_t *slot = reinterpret_cast<volatile uint32_t *>(gen + L::kBars + kSlot);
    int *status = &g_status;

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int heads = p.batch * p.q_heads;
    const int bh = blockIdx.x % heads, h = bh % p.q_heads, b = bh / p.q_heads, kh = h / p.group;
    const int i0 = (int)((gridDim.x - 1 - blockIdx.x) / heads) * 2 * kRows;       // the longest rows of a causal call first
    const int keys = keys_of(p, b);
    const int kb = first_key(p, i0) / kRows;
    const auto tiles_of = [&](int t) {                                            // key tiles that tile t walks
        const int lo = i0 + t * kRows, hi = lo + kRows < p.q_len ? lo + kRows : p.q_len;
        const int e = lo < p.q_len ? (end_key(p, hi, keys) + kRows - 1) / kRows - kb : 0;
        return e > 0 ? e : 0;
    };
    const int n0 = uniform(tiles_of(0)), n1 = uniform(tiles_of(1)), steps = n0 > n1 ? n0 : n1, both = n0 < n1 ? n0 : n1;
    // Units in the order of their products: both tiles of each step, then what the longer walk has left.
    const auto unit_of = [&](int j, int t) { return j < both ? 2 * j + t : both + j; };

    // the thread that issues the loads sets the barriers up and sends the first loads off before the others are ready
    if (threadIdx.x == 544) {
        failed() = 0;
        for (int t = 0; t < 2; ++t) { acp::mbar_init(q_full(t), 1); acp::mbar_init(o_full(t), 1); acp::mbar_init(o_done(t, 0), 1); acp::mbar_init(o_done(t, 1), 1); }
        for (int x = 0; x < kBufs; ++x) { acp::mbar_init(s_full(x), 1); acp::mbar_init(p_full(x), 256); }
        acp::mbar_init(fix, 1);
        for (int s = 0; s < L::kStages; ++s) { acp::mbar_init(kv_full(s), 1); acp::mbar_init(kv_empty(s), 1); }
        acp::fence_barrier_init();
        acp::fence_async_smem();
        if (steps > 0) {
            for (int t = 0; t < 2; ++t)
                if ((t ? n1 : n0) > 0) {
                    acp::mbar_expect_tx(q_full(t), L::kTile);
                    load_tile<DP>(base + t * L::kTile, &mq, q_full(t), i0 + t * kRows, h, b);
                }
            acp::mbar_expect_tx(kv_full(0), L::kTile);
            load_tile<DP>(base + L::kRing, &mk, kv_full(0), kb * kRows, kh, b);
            prefetch_map(&mv);
        }
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(bars + kSlot) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *slot;
    const auto tS = [&](int x) { return tmem + 128u * x; };
    const auto tO = [&](int t) { return tmem + 128u * kBufs + (uint32_t)DP * t; };

    if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLess));
    if (warp == 17) {
        // ------------------------------------------------------------------ loads: V_0 (Q and K_0 are under way), then K_j, V_j in turn
        bool ok = true;
        int s = 1;
        uint32_t ph = 0;
        for (int x = 1; x < 2 * steps && ok; ++x) {
            const int row = (kb + x / 2) * kRows;
            ok = wait_warp(kv_empty(s), ph ^ 1u, 1, status);
            if (!ok) break;
            const uint32_t dst = base + L::kRing + s * L::kTile;
            const bool cut = (x & 1) && keys < p.k_len && row + kRows > keys;     // V rows behind the length may hold anything
            if (lane == 0) {
                const uint32_t bar = cut ? fix : kv_full(s);
                acp::mbar_expect_tx(bar, L::kTile);
                load_tile<DP>(dst, (x & 1) ? &mv : &mk, bar, row, kh, b);
            }
            if (cut) {                                                           // the last tile of the walk
                ok = wait_warp(fix, 0u, 2, status);
                if (!ok) break;
                clear_rows<DP>(gen + (dst - base), keys - row);
                if (lane == 0) acp::mbar_arrive(kv_full(s));
            }
            __syncwarp();
            if (++s == L::kStages) { s = 0; ph ^= 1u; }
        }
    } else if (warp == 16) {
        // ------------------------------------------------------------------ products
        if (steps > 0) {
            const bool one = elect();
            const int slices = (p.head_size + 15) / 16;
            const auto stage = [&](int x) { return base + L::kRing + (uint32_t)(x % L::kStages) * L::kTile; };
            const auto full = [&](int x, int code) { return wait_warp(kv_full(x % L::kStages), (uint32_t)(x / L::kStages) & 1u, code, status); };
            const int units = n0 + n1, first = n0 > 0 ? 0 : 1;                    // tile 1 alone walks where tile 0 sees nothing
            const auto step_of = [&](int u) { return u < 2 * both ? u / 2 : u - both; };
            const auto tile_of = [&](int u) { return u < 2 * both ? u & 1 : (n0 > n1 ? 0 : 1); };
            const auto last_of_step = [&](int u) { return u >= 2 * both || (u & 1); };
            const auto scores = [&](int u) {                                      // S of unit u
                const int j = step_of(u), t = tile_of(u);
                if (!full(2 * j, 3)) return false;
                fence_after();
                if (one) {
                    product_rows<DP>(tS(u % kBufs), base + t * L::kTile, stage(2 * j), slices);
                    commit(s_full(u % kBufs));
                    if (last_of_step(u)) commit(kv_empty((2 * j) % L::kStages));
                }
                __syncwarp();
                return true;
            };
            bool ok = wait_warp(q_full(first), 0u, 4, status) && (both == 0 || wait_warp(q_full(1), 0u, 5, status));
            for (int u = 0; u < kBufs && u < units && ok; ++u) ok = scores(u);
            for (int u = 0; u < units && ok; ++u) {
                const int j = step_of(u), t = tile_of(u);
                ok = full(2 * j + 1, 6) && wait_warp(p_full(u % kBufs), (uint32_t)(u / kBufs) & 1u, 7, status);
                if (!ok) break;
                fence_after();
                if (one) {
                    product_cols<DP, kRows, 64>(tO(t), tS(u % kBufs), stage(2 * j + 1), j != 0);
                    commit(j + 1 == (t ? n1 : n0) ? o_full(t) : o_done(t, j));
                    if (last_of_step(u)) commit(kv_empty((2 * j + 1) % L::kStages));
                }
                __syncwarp();
                if (u + kBufs < units) ok = scores(u + kBufs);                    // over P of unit u, behind the product that reads it
            }
        }
    }
    } else {
        // ------------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMore));
        const int t = warp >> 3, half = (warp >> 2) & 1, row = threadIdx.x & 127, i = i0 + t * kRows + row;
        const int low = i0 + t * kRows, nt = t ? n1 : n0;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                        // this warp's 32 lanes of tensor memory
        const uint32_t O = tO(t) + lanes;
        const float c = kMask ? kLog2e : p.scale * kLog2e;
        const float slack = 8.0f / c;
        volatile float *tops = reinterpret_cast<float *>(gen + L::kTops) + t * 2 * kRows + row;
        const auto meet = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + 4 * t + (warp & 3)) : "memory"); };      // the two warps of these rows
        float m = -CUDART_INF_F, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < nt; ++j) {
            const int u = unit_of(j, t);
            const uint32_t S = tS(u % kBufs) + lanes + 64u * half;
            uint32_t r[64];
            if (ok) {
                ok = wait_warp(s_full(u % kBufs), (uint32_t)(u / kBufs) & 1u, 8, status);
                fence_after();
                ld32(S, r);
                ld32(S + 32u, r + 32);
                wait_ld();
            }
            const int j0 = (kb + j) * kRows + 64 * half;
            if (kMask) {
#pragma unroll
                for (int e = 0; e < 64; ++e) {
                    const float v = sees(p, i, j0 + e, keys) ? masked_score(p, __uint_as_float(r[e]) * p.scale, b, h, i, j0 + e) : -CUDART_INF_F;
                    r[e] = __float_as_uint(v);
                }
            } else if (j0 + 64 > keys || (p.causal && j0 + 63 > low + p.offset) || (p.window && j0 <= low + kRows - 1 + p.offset - p.window)) {
                int lo = 0, hi = keys - j0;                                       // visible columns [lo, hi) of this row
                if (p.causal && i + p.offset + 1 - j0 < hi) hi = i + p.offset + 1 - j0;
                if (p.window) lo = i + p.offset - p.window + 1 - j0;
#pragma unroll
                for (int e = 0; e < 64; ++e)
                    if (e < lo || e >= hi) r[e] = 0xff800000u;
            }
            float top = row_max<64>(r);
            // two slots a row, this step's and the last one's: a warp may be a step ahead of the other's read
            tops[half * kRows + (j & 1) * 4 * kRows] = top;
            meet();
            top = fmaxf(top, tops[(half ^ 1) * kRows + (j & 1) * 4 * kRows]);
            if (!ok) continue;                                                    // after a failure the warps only keep meeting, so that neither waits alone
            if (__any_sync(~0u, top > m + slack || (m == -CUDART_INF_F && top > m))) {
                const float raised = fmaxf(m, top);
                const float f = m == -CUDART_INF_F ? 0.0f : ex2((m - raised) * c);
                l *= f;
                m = raised;
                if (j > 0) {
                    // P V of the step before is done.  That of three steps before, on the same barrier, was long before: these scores came
                    // behind it, so the parity is unambiguous.  Each half of the warps rescales half of the columns.
                    ok = wait_warp(o_done(t, j - 1), (uint32_t)((j - 1) / 2) & 1u, 9, status);
                    if (!ok) continue;
                    fence_after();
#pragma unroll 1
                    for (int e = half * (DP / 32); e < (half + 1) * (DP / 32); ++e) {
                        uint32_t o[16];
                        ld16(O + 16u * e, o);
                        wait_ld();
#pragma unroll
                        for (int z = 0; z < 16; ++z) o[z] = __float_as_uint(__uint_as_float(o[z]) * f);
                        st16(O + 16u * e, o);
                    }
                }
            }
            Exponentials<kMask> ex(m == -CUDART_INF_F ? 0.0f : m, c);
#pragma unroll
            for (int e = 0; e < 4; ++e) ex.piece(r + 16 * e, S + 8u * e);
            l += ex.sum();
            wait_st();
            fence_before();
            acp::mbar_arrive(p_full(u % kBufs));
        }
        if (ok && nt > 0) {
            ok = wait_warp(o_full(t), 0u, 10, status);
            fence_after();
        }
        meet();                                                                   // the last maxima have been read
        tops[half * kRows] = l;
        meet();
        if (ok && low < p.q_len) {
            l += tops[(half ^ 1) * kRows];
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + b * p.out_b + h * p.out_h + i * p.out_t;
            // each half of the warps writes half of the columns
#pragma unroll 1
            for (int e = half * (DP / 64); e < (half + 1) * (DP / 64); ++e) {
                uint32_t o[32];
                if (nt > 0) { ld32(O + 32u * e, o); wait_ld(); }
                else {
#pragma unroll
                    for (int z = 0; z < 32; ++z) o[z] = 0u;
                }
                if (i < p.q_len) {
                    store_piece(out, 32 * e, p.head_size, o, inv);
                    if (p.o_low) store_rest(static_cast<__nv_bfloat16 *>(p.o_low) + (out - static_cast<__nv_bfloat16 *>(p.out)), 32 * e, p.head_size, o, inv);
                }
            }
            if (half == 0 && i < p.q_len) {
                const long long at = ((long long)b * p.q_heads + h) * p.q_len + i;
                const float top = kMask ? m : m * p.scale;                        // -inf stays -inf
                p.row_max[at] = top;
                p.row_sum[at] = l;
                if (p.lse) p.lse[at] = l == 0.0f ? -CUDART_INF_F : top + log2f(l) * kLn2;
            }
        }
    }
    fence_before();
    __syncthreads();
    linger_if_failed();
    if (warp == 16) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

}  // namespace tc
}  // namespace attn
}  // namespace axs6
