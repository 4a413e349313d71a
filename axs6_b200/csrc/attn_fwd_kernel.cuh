// Attention forward on the tensor cores (bf16 tensors, fp32 scores, sums and output accumulator).
//
// A CTA owns 256 queries of one head as two tiles of 128 and walks the keys in tiles of 128:
//     S_t = Q_t K_j^T  (tensor memory)    P_t = exp2(c S_t - c m)  (bf16, over S_t's columns)    O_t += P_t V_j  (tensor memory)
// with c = scale log2 e and the running reference m per row.  m is only raised, and O_t and the sum rescaled, when a row's maximum exceeds
// it by more than 8 in base 2: any reference gives the same quotient O / l, exp2 stays below 2^8, and the rescaling pass over O (which costs
// as much as a quarter of a tile) runs in the first few tiles only.  P is rounded to bf16 because the tensor cores multiply it with V; the
// sum l takes the unrounded values, so the rounding errors of a row's P average out instead of shifting it.
//
// Warps 0-3 / 4-7: softmax of tile 0 / 1, one thread a row, 128 scores in registers (no shuffles).  Warp 8: one thread issues all products.
// Warp 9: loads.  (Warps 10 and 11 only complete the warpgroup that hands its registers over.)  The two tiles alternate on the tensor cores: while tile 0 is in its softmax, tile 1's PV and next S run.
// tcgen05 instructions of one thread complete in order, so S_t(j+1), issued behind PV_t(j), also tells that O_t is up to date.
//
// Bound: 4 D flops a pair on the tensor cores (8192 a clock: 1024 clocks a tile and D = 128) and one exp2 a pair (16 a clock: 1024 clocks).
#pragma once
#include "attn_tc.cuh"

namespace axs6 {
namespace attn {
namespace tc {

constexpr int kFwdThreads = 384;
// Registers: launched with 168 a thread, 3 x 168 = 504 for the three warpgroups; the softmax warpgroups take 240 each (a row of 128
// scores and its bf16 form are held at once), the one that loads and issues keeps 24.
constexpr int kRegsMore = 224, kRegsLess = 56;

template <int DP> struct FwdSmem {
    static constexpr uint32_t kTile = kBox * (DP / 64);
    static constexpr int kStages = DP == 64 ? 8 : 4;
    static constexpr uint32_t kRing = 2 * kTile, kBars = kRing + kStages * kTile;
    static constexpr uint32_t kBytes = kBars + 256 + 1024;
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
    const auto q_full = [&](int t) { return bars + 8u * t; };
    const auto s_full = [&](int t) { return bars + 16u + 8u * t; };
    const auto p_full = [&](int t) { return bars + 32u + 8u * t; };
    const auto o_full = [&](int t) { return bars + 48u + 8u * t; };
    const uint32_t fix = bars + 64u;
    const auto kv_full = [&](int s) { return bars + 72u + 8u * s; };
    const auto kv_empty = [&](int s) { return bars + 72u + 8u * (L::kStages + s); };
    volatile uint32_t *slot = reinterpret_cast<volatile uint32_t *>(gen + L::kBars + 72 + 16 * L::kStages);
    int *status = &g_status;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
    const int n0 = tiles_of(0), n1 = tiles_of(1), steps = n0 > n1 ? n0 : n1;

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) { acp::mbar_init(q_full(t), 1); acp::mbar_init(s_full(t), 1); acp::mbar_init(p_full(t), 128); acp::mbar_init(o_full(t), 1); }
        acp::mbar_init(fix, 1);
        for (int s = 0; s < L::kStages; ++s) { acp::mbar_init(kv_full(s), 1); acp::mbar_init(kv_empty(s), 1); }
        acp::fence_barrier_init();
        acp::fence_async_smem();
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(bars + 72u + 16u * L::kStages) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *slot;
    const auto tS = [&](int t) { return tmem + 128u * t; };
    const auto tO = [&](int t) { return tmem + 256u + 128u * t; };

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLess));
    if (warp == 9) {
        // ------------------------------------------------------------------ loads: Q, then K_j, V_j in turn
        bool ok = steps > 0;
        if (ok && lane == 0)
            for (int t = 0; t < 2; ++t)
                if ((t ? n1 : n0) > 0) {
                    acp::mbar_expect_tx(q_full(t), L::kTile);
                    load_tile<DP>(base + t * L::kTile, &mq, q_full(t), i0 + t * kRows, h, b);
                }
        int s = 0;
        uint32_t ph = 0;
        for (int x = 0; x < 2 * steps && ok; ++x) {
            const int row = (kb + x / 2) * kRows;
            ok = wait(kv_empty(s), ph ^ 1u, 1, status);
            if (!ok) break;
            const uint32_t dst = base + L::kRing + s * L::kTile;
            const bool cut = (x & 1) && keys < p.k_len && row + kRows > keys;     // V rows behind the length may hold anything
            if (lane == 0) {
                const uint32_t bar = cut ? fix : kv_full(s);
                acp::mbar_expect_tx(bar, L::kTile);
                load_tile<DP>(dst, (x & 1) ? &mv : &mk, bar, row, kh, b);
            }
            if (cut) {                                                           // the last tile of the walk
                ok = wait(fix, 0u, 2, status);
                if (!ok) break;
                clear_rows<DP>(gen + (dst - base), keys - row);
                if (lane == 0) acp::mbar_arrive(kv_full(s));
            }
            __syncwarp();
            if (++s == L::kStages) { s = 0; ph ^= 1u; }
        }
    } else if (warp == 8) {
        // ------------------------------------------------------------------ products
        if (lane == 0 && steps > 0) {
            bool ok = true;
            const auto stage = [&](int x) { return base + L::kRing + (uint32_t)(x % L::kStages) * L::kTile; };
            const auto full = [&](int x, int code) { return wait(kv_full(x % L::kStages), (uint32_t)(x / L::kStages) & 1u, code, status); };
            ok = full(0, 3);
            for (int t = 0; t < 2 && ok; ++t)
                if ((t ? n1 : n0) > 0) {
                    ok = wait(q_full(t), 0u, 4, status);
                    if (!ok) break;
                    fence_after();
                    product_rows<DP>(tS(t), base + t * L::kTile, stage(0));
                    commit(s_full(t));
                }
            commit(kv_empty(0));
            for (int j = 0; j < steps && ok; ++j) {
                bool v_here = false, k_here = false;
                for (int t = 0; t < 2 && ok; ++t) {
                    const int nt = t ? n1 : n0;
                    if (j >= nt) continue;
                    ok = wait(p_full(t), (uint32_t)j & 1u, 5, status);
                    if (ok && !v_here) { ok = full(2 * j + 1, 6); v_here = true; }
                    if (!ok) break;
                    fence_after();
                    product_cols<DP>(tO(t), tS(t), stage(2 * j + 1), j != 0);
                    if (j + 1 == nt) {
                        commit(o_full(t));
                    } else {
                        if (!k_here) { ok = full(2 * j + 2, 7); k_here = true; }
                        if (!ok) break;
                        product_rows<DP>(tS(t), base + t * L::kTile, stage(2 * j + 2));
                        commit(s_full(t));
                    }
                }
                if (!ok) break;
                commit(kv_empty((2 * j + 1) % L::kStages));
                if (j + 1 < steps) commit(kv_empty((2 * j + 2) % L::kStages));
            }
        }
    }
    } else {
        // ------------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsMore));
        const int t = warp >> 2, row = threadIdx.x & 127, i = i0 + t * kRows + row;
        const int low = i0 + t * kRows, nt = t ? n1 : n0;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                        // this warp's 32 lanes of tensor memory
        const uint32_t S = tS(t) + lanes, O = tO(t) + lanes;
        const float c = kMask ? kLog2e : p.scale * kLog2e;
        const float slack = 8.0f / c;
        float m = -CUDART_INF_F, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < nt; ++j) {
            ok = wait(s_full(t), (uint32_t)j & 1u, 8, status);
            if (!__all_sync(~0u, ok)) { ok = false; break; }
            fence_after();
            uint32_t r[128];
#pragma unroll
            for (int x = 0; x < 4; ++x) ld32(S + 32u * x, r + 32 * x);
            wait_ld();
            const int j0 = (kb + j) * kRows;
            if (kMask) {
#pragma unroll
                for (int x = 0; x < 128; ++x) {
                    const float v = sees(p, i, j0 + x, keys) ? masked_score(p, __uint_as_float(r[x]) * p.scale, b, h, i, j0 + x) : -CUDART_INF_F;
                    r[x] = __float_as_uint(v);
                }
            } else if (j0 + kRows > keys || (p.causal && j0 + kRows - 1 > low + p.offset) ||
                       (p.window && j0 <= low + kRows - 1 + p.offset - p.window)) {
                int lo = 0, hi = keys - j0;                                       // visible columns [lo, hi) of this row
                if (p.causal && i + p.offset + 1 - j0 < hi) hi = i + p.offset + 1 - j0;
                if (p.window) lo = i + p.offset - p.window + 1 - j0;
#pragma unroll
                for (int x = 0; x < 128; ++x)
                    if (x < lo || x >= hi) r[x] = 0xff800000u;
            }
            float top = __uint_as_float(r[0]), top1 = __uint_as_float(r[1]);
#pragma unroll
            for (int x = 2; x < 128; x += 2) { top = fmaxf(top, __uint_as_float(r[x])); top1 = fmaxf(top1, __uint_as_float(r[x + 1])); }
            top = fmaxf(top, top1);
            if (__any_sync(~0u, top > m + slack || (m == -CUDART_INF_F && top > m))) {
                const float raised = fmaxf(m, top);
                const float f = m == -CUDART_INF_F ? 0.0f : ex2((m - raised) * c);
                l *= f;
                m = raised;
                if (j > 0) {
#pragma unroll
                    for (int x = 0; x < DP / 32; ++x) {
                        uint32_t o[32];
                        ld32(O + 32u * x, o);
                        wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        st32(O + 32u * x, o);
                    }
                }
            }
            const float ref = m == -CUDART_INF_F ? 0.0f : m, shift = -ref * c;
            float l1 = 0.0f;
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float u = __uint_as_float(r[16 * x + 2 * e]), v = __uint_as_float(r[16 * x + 2 * e + 1]);
                    const float pu = ex2(kMask ? (u - ref) * c : fmaf(u, c, shift)), pv = ex2(kMask ? (v - ref) * c : fmaf(v, c, shift));
                    l += pu;
                    l1 += pv;
                    w[e] = pack2(pu, pv);
                }
                st8(S + 8u * x, w);
            }
            l += l1;
            wait_st();
            fence_before();
            acp::mbar_arrive(p_full(t));
        }
        if (ok && nt > 0) {
            ok = wait(o_full(t), 0u, 9, status);
            ok = __all_sync(~0u, ok);
            fence_after();
        }
        if (ok && low < p.q_len) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + b * p.out_b + h * p.out_h + i * p.out_t;
#pragma unroll 1
            for (int x = 0; x < DP / 32; ++x) {
                uint32_t o[32];
                if (nt > 0) { ld32(O + 32u * x, o); wait_ld(); }
                else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
                if (i < p.q_len) {
                    store_piece(out, 32 * x, p.head_size, o, inv);
                    if (p.o_low) store_rest(static_cast<__nv_bfloat16 *>(p.o_low) + (out - static_cast<__nv_bfloat16 *>(p.out)), 32 * x, p.head_size, o, inv);
                }
            }
            if (i < p.q_len) {
                const long long at = ((long long)b * p.q_heads + h) * p.q_len + i;
                const float top = kMask ? m : m * p.scale;                        // -inf stays -inf
                p.row_max[at] = top;
                p.row_sum[at] = l;
                if (p.lse) p.lse[at] = l == 0.0f ? -CUDART_INF_F : top + log2f(l) * kLn2;
            }
        }
    }
    linger_if_failed(status);
    fence_before();
    __syncthreads();
    if (warp == 8) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

}  // namespace tc
}  // namespace attn
}  // namespace axs6
