// Attention forward on the tensor cores (bf16 tensors, fp32 scores, sums and output accumulator).
//
// A CTA owns 256 queries of one head as two tiles of 128 and walks the keys in tiles of 64:
//     S_t = Q_t K_j^T  (tensor memory)    P_t = exp2(c S_t - c m)  (bf16, over S_t's columns)    O_t += P_t V_j  (tensor memory)
// with c = scale log2 e and the running reference m per row.  m is only raised, and O_t and the sum rescaled, when a row's maximum exceeds
// it by more than 8 in base 2: any reference gives the same quotient O / l, exp2 stays below 2^8, and the pass over O runs in the first few
// steps only.  P is rounded to bf16 because the tensor cores multiply it with V; the sum l takes the unrounded values, so the rounding
// errors of a row's P average out instead of shifting it.
//
// Warps 0-15: softmax, one thread a row and score buffer (no shuffles): warps 0-3 and 4-7 take the even and odd steps of tile 0, warps 8-11 and
// 12-15 those of tile 1.  Warp 16: products.  Warp 17: loads.  (Warps 18 and 19 only complete the warpgroup that hands its registers over.)
// A step's softmax is a chain of dependent instructions of about 1900 clocks with two softmax warps on a scheduler, and neither longer tiles
// nor exponentials on the fma pipe shortened it; with four warps two steps of each tile run side by side.  What they share is the reference:
// a step reads it when the step before has decided about it (a barrier per step), and raises it, rarely, after that step's PV.  Each tile has
// two score buffers (2 x 2 x 64 columns, next to 2 x D of output: all of tensor memory at D = 128), so S_t(j + 2) is computed under the
// softmax of step j + 1.  tcgen05 instructions of one thread complete in order: S_t(j + 2) may overwrite P_t(j) behind P_t(j) V.
//
// Bound: tensor cores, per 128 x 64 pairs at D = 128 256 clocks for PV and 384 for S (an N = 64 product reads 6 KB of shared memory for 32
// clocks of work), and one exp2 a pair (16 a clock: 512 clocks).
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
    static constexpr uint32_t kQ = kBox * (DP / 64), kTile = kKeys * 128 * (DP / 64);
    static constexpr int kStages = 8;
    static constexpr uint32_t kRing = 2 * kQ, kRefs = kRing + kStages * kTile;
    static constexpr uint32_t kSums = kRefs + 2 * kRows * 4, kBars = kSums + 4 * kRows * 4;      // a row's reference, its sums of even and odd steps
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
    // barriers of tile t and score buffer x
    const auto q_full = [&](int t) { return bars + 8u * t; };
    const auto o_full = [&](int t) { return bars + 16u + 8u * t; };
    const auto s_full = [&](int t, int x) { return bars + 32u + 16u * t + 8u * x; };
    const auto p_full = [&](int t, int x) { return bars + 64u + 16u * t + 8u * x; };
    const auto o_done = [&](int t, int x) { return bars + 96u + 16u * t + 8u * x; };
    const auto turn = [&](int t, int x) { return bars + 128u + 16u * t + 8u * x; };
    const uint32_t fix = bars + 160u;
    const auto kv_full = [&](int s) { return bars + 168u + 8u * s; };
    const auto kv_empty = [&](int s) { return bars + 168u + 8u * (L::kStages + s); };
    constexpr uint32_t kSlot = 168 + 16 * L::kStages;
    volatile uint32_t *slot = reinterpret_cast<volatile uint32_t *>(gen + L::kBars + kSlot);
    int *status = &g_status;

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int heads = p.batch * p.q_heads;
    const int bh = blockIdx.x % heads, h = bh % p.q_heads, b = bh / p.q_heads, kh = h / p.group;
    const int i0 = (int)((gridDim.x - 1 - blockIdx.x) / heads) * 2 * kRows;       // the longest rows of a causal call first
    const int keys = keys_of(p, b);
    const int kb = first_key(p, i0) / kKeys;
    const auto tiles_of = [&](int t) {                                            // key tiles that tile t walks
        const int lo = i0 + t * kRows, hi = lo + kRows < p.q_len ? lo + kRows : p.q_len;
        const int e = lo < p.q_len ? (end_key(p, hi, keys) + kKeys - 1) / kKeys - kb : 0;
        return e > 0 ? e : 0;
    };
    const int n0 = uniform(tiles_of(0)), n1 = uniform(tiles_of(1)), steps = n0 > n1 ? n0 : n1;

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            acp::mbar_init(q_full(t), 1); acp::mbar_init(o_full(t), 1);
            for (int x = 0; x < 2; ++x) { acp::mbar_init(turn(t, x), 128); acp::mbar_init(s_full(t, x), 1); acp::mbar_init(p_full(t, x), 128); acp::mbar_init(o_done(t, x), 1); }
        }
        acp::mbar_init(fix, 1);
        for (int s = 0; s < L::kStages; ++s) { acp::mbar_init(kv_full(s), 1); acp::mbar_init(kv_empty(s), 1); }
        acp::fence_barrier_init();
        acp::fence_async_smem();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(bars + kSlot) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *slot;
    const auto tS = [&](int t, int x) { return tmem + 128u * t + 64u * x; };
    const auto tO = [&](int t) { return tmem + 256u + 128u * t; };

    if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLess));
    if (warp == 17) {
        // ------------------------------------------------------------------ loads: Q, then K_j, V_j in turn
        bool ok = steps > 0;
        if (ok && lane == 0)
            for (int t = 0; t < 2; ++t)
                if ((t ? n1 : n0) > 0) {
                    acp::mbar_expect_tx(q_full(t), L::kQ);
                    load_tile<DP>(base + t * L::kQ, &mq, q_full(t), i0 + t * kRows, h, b);
                }
        int s = 0;
        uint32_t ph = 0;
        for (int x = 0; x < 2 * steps && ok; ++x) {
            const int row = (kb + x / 2) * kKeys;
            ok = wait_warp(kv_empty(s), ph ^ 1u, 1, status);
            if (!ok) break;
            const uint32_t dst = base + L::kRing + s * L::kTile;
            const bool cut = (x & 1) && keys < p.k_len && row + kKeys > keys;     // V rows behind the length may hold anything
            if (lane == 0) {
                const uint32_t bar = cut ? fix : kv_full(s);
                acp::mbar_expect_tx(bar, L::kTile);
                load_tile<DP, kKeys>(dst, (x & 1) ? &mv : &mk, bar, row, kh, b);
            }
            if (cut) {                                                           // the last tile of the walk
                ok = wait_warp(fix, 0u, 2, status);
                if (!ok) break;
                clear_rows<DP, kKeys>(gen + (dst - base), keys - row);
                if (lane == 0) acp::mbar_arrive(kv_full(s));
            }
            __syncwarp();
            if (++s == L::kStages) { s = 0; ph ^= 1u; }
        }
    } else if (warp == 16) {
        // ------------------------------------------------------------------ products
        if (steps > 0) {
            const bool one = elect();
            const auto stage = [&](int x) { return base + L::kRing + (uint32_t)(x % L::kStages) * L::kTile; };
            const auto full = [&](int x, int code) { return wait_warp(kv_full(x % L::kStages), (uint32_t)(x / L::kStages) & 1u, code, status); };
            const auto scores = [&](int t, int j) {
                if (one) {
                    product_rows<DP, kKeys>(tS(t, j & 1), base + t * L::kQ, stage(2 * j));
                    commit(s_full(t, j & 1));
                }
                __syncwarp();
            };
            bool ok = true;
            for (int t = 0; t < 2 && ok; ++t)
                if ((t ? n1 : n0) > 0) ok = wait_warp(q_full(t), 0u, 3, status);
            for (int j = 0; j < 2 && j < steps && ok; ++j) {
                ok = full(2 * j, 4);
                if (!ok) break;
                fence_after();
                for (int t = 0; t < 2; ++t)
                    if (j < (t ? n1 : n0)) scores(t, j);
                if (one) commit(kv_empty((2 * j) % L::kStages));
                __syncwarp();
            }
            for (int j = 0; j < steps && ok; ++j) {
                ok = full(2 * j + 1, 5);
                bool next = false;                                                // K(j + 2) is here
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int nt = t ? n1 : n0;
                    if (!ok || j >= nt) continue;
                    ok = wait_warp(p_full(t, j & 1), (uint32_t)(j / 2) & 1u, 6, status);
                    if (!ok) continue;
                    fence_after();
                    if (one) {
                        product_cols<DP, kKeys>(tO(t), tS(t, j & 1), stage(2 * j + 1), j != 0);
                        commit(j + 1 == nt ? o_full(t) : o_done(t, j & 1));
                    }
                    __syncwarp();
                    if (j + 2 < nt) {                                             // over P_t(j), behind the product that reads it
                        if (!next) { ok = full(2 * (j + 2), 7); next = true; fence_after(); }
                        if (ok) scores(t, j + 2);
                    }
                }
                if (ok && one) {
                    commit(kv_empty((2 * j + 1) % L::kStages));
                    if (j + 2 < steps) commit(kv_empty((2 * (j + 2)) % L::kStages));
                }
                __syncwarp();
            }
        }
    }
    } else {
        // ------------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMore));
        const int t = warp >> 3, x = (warp >> 2) & 1, row = threadIdx.x & 127, i = i0 + t * kRows + row;
        const int low = i0 + t * kRows, nt = t ? n1 : n0;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                        // this warp's 32 lanes of tensor memory
        const uint32_t S = tS(t, x) + lanes, O = tO(t) + lanes;
        const float c = kMask ? kLog2e : p.scale * kLog2e;
        const float slack = 8.0f / c;
        volatile float *refs = reinterpret_cast<float *>(gen + L::kRefs) + t * kRows + row;
        volatile float *sums = reinterpret_cast<float *>(gen + L::kSums) + t * 2 * kRows + row;
        float m = -CUDART_INF_F, l = 0.0f;                                        // l is relative to m, this thread's copy of the reference
        bool ok = true;
        if (x == 0) *refs = -CUDART_INF_F;                                        // read by others only behind a barrier that this thread arrives at
        for (int j = x; j < nt; j += 2) {
            const uint32_t phase = (uint32_t)(j / 2) & 1u, before = (uint32_t)((j - 1) / 2) & 1u;
            ok = wait(s_full(t, x), phase, 8, status);
            if (!__all_sync(~0u, ok)) { ok = false; break; }
            fence_after();
            uint32_t r[kKeys];
            ld32(S, r);
            ld32(S + 32u, r + 32);
            wait_ld();
            const int j0 = (kb + j) * kKeys;
            if (kMask) {
#pragma unroll
                for (int e = 0; e < kKeys; ++e) {
                    const float v = sees(p, i, j0 + e, keys) ? masked_score(p, __uint_as_float(r[e]) * p.scale, b, h, i, j0 + e) : -CUDART_INF_F;
                    r[e] = __float_as_uint(v);
                }
            } else if (j0 + kKeys > keys || (p.causal && j0 + kKeys - 1 > low + p.offset) ||
                       (p.window && j0 <= low + kRows - 1 + p.offset - p.window)) {
                int lo = 0, hi = keys - j0;                                       // visible columns [lo, hi) of this row
                if (p.causal && i + p.offset + 1 - j0 < hi) hi = i + p.offset + 1 - j0;
                if (p.window) lo = i + p.offset - p.window + 1 - j0;
#pragma unroll
                for (int e = 0; e < kKeys; ++e)
                    if (e < lo || e >= hi) r[e] = 0xff800000u;
            }
            const float top = row_max<kKeys>(r);
            float ref = -CUDART_INF_F;
            if (j > 0) {
                ok = wait(turn(t, x ^ 1), before, 9, status);
                if (!__all_sync(~0u, ok)) { ok = false; break; }
                ref = *refs;
            }
            if (__any_sync(~0u, top > ref + slack || (ref == -CUDART_INF_F && top > ref))) {
                const float raised = fmaxf(ref, top);
                if (j > 0) {
                    // O is up to date: P(j - 1) V is done.  P(j - 3) V on the same barrier was long before, since S(j) came behind P(j - 2) V:
                    // the parity is unambiguous.
                    const float f = ref == -CUDART_INF_F ? 0.0f : ex2((ref - raised) * c);
                    ok = wait(o_done(t, x ^ 1), before, 10, status);
                    if (!__all_sync(~0u, ok)) { ok = false; break; }
                    fence_after();
#pragma unroll 1
                    for (int e = 0; e < DP / 16; ++e) {
                        uint32_t o[16];
                        ld16(O + 16u * e, o);
                        wait_ld();
#pragma unroll
                        for (int z = 0; z < 16; ++z) o[z] = __float_as_uint(__uint_as_float(o[z]) * f);
                        st16(O + 16u * e, o);
                    }
                }
                ref = raised;
                *refs = ref;
            }
            acp::mbar_arrive(turn(t, x));
            if (__any_sync(~0u, ref != m)) {
                l *= m == -CUDART_INF_F ? 0.0f : ex2((m - ref) * c);
                m = ref;
            }
            Exponentials<kMask> ex(m == -CUDART_INF_F ? 0.0f : m, c);
#pragma unroll
            for (int e = 0; e < kKeys / 16; ++e) ex.piece(r + 16 * e, S + 8u * e);
            l += ex.sum();
            wait_st();
            fence_before();
            acp::mbar_arrive(p_full(t, x));
        }
        if (ok && nt > 0) {
            ok = wait(o_full(t), 0u, 11, status);
            ok = __all_sync(~0u, ok);
            fence_after();
        }
        // the two threads of a row join their sums, relative to the last reference
        asm volatile("bar.sync %0, 256;" ::"r"(1 + t) : "memory");
        const float ref = *refs;
        sums[x * kRows] = m == -CUDART_INF_F ? 0.0f : l * ex2((m - ref) * c);
        asm volatile("bar.sync %0, 256;" ::"r"(1 + t) : "memory");
        if (ok && low < p.q_len) {
            l = sums[0] + sums[kRows];
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + b * p.out_b + h * p.out_h + i * p.out_t;
            // each writes half of the columns
#pragma unroll 1
            for (int e = x * (DP / 64); e < (x + 1) * (DP / 64); ++e) {
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
            if (x == 0 && i < p.q_len) {
                const long long at = ((long long)b * p.q_heads + h) * p.q_len + i;
                const float top = kMask ? ref : ref * p.scale;                    // -inf stays -inf
                p.row_max[at] = top;
                p.row_sum[at] = l;
                if (p.lse) p.lse[at] = l == 0.0f ? -CUDART_INF_F : top + log2f(l) * kLn2;
            }
        }
    }
    linger_if_failed(status);
    fence_before();
    __syncthreads();
    if (warp == 16) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

}  // namespace tc
}  // namespace attn
}  // namespace axs6
