// Attention forward for few queries (a generated token, a short prompt over a long cache), bf16 tensors.
//
// The query heads that share a key head are stacked into one tile of 128 rows (row = query * group + head), so keys and values are
// read once for all of them, and the keys are cut into chunks that CTAs of their own walk.  Each CTA leaves its rows' maximum, sum and
// unnormalised fp32 output in a workspace; a second kernel joins them in chunk order:
//     m = max m_c    l = sum l_c e^(m_c - m)    O = sum O_c e^(m_c - m) / l
// With a single chunk the result is written at once.
//
// Bound: HBM, keys and values once.  Two CTAs live on an SM (half of tensor memory, 97 KB of shared memory each), so that one's products and
// softmax run under the other's loads, and up to 128 KB are in flight on an SM.  Scores are double-buffered in tensor memory: S(j + 1) is
// issued before P(j) V, so that the softmax of one tile runs under the products of its
// neighbours.  Warps 0-3: softmax, one thread a row; warps without rows idle (the lanes of P that they would fill hold anything: a row of A reaches only its own row of the product).  Warp 4: products.
// Warp 5: loads.  Measured: 16 entries of 8192 keys, 32 / 8 heads of 128: 109 us, 4.9 TB/s (0.75 of a copy); with 1 to 8 Ki keys 73 us for 48 us of
// bytes; the tensor cores, which multiply 128 rows where 4 are wanted, are 40 % busy.
#pragma once
#include "attn_tc.cuh"

namespace axs6 {
namespace attn {
namespace tc {

constexpr int kFewThreads = 192;

struct Few {
    int row_tiles, chunks, chunk;     // tiles of 128 stacked rows a key head, chunks of the keys, key tiles (of 64) of a chunk
    float *out, *stat;                // chunks > 1: (chunk, batch, key head, row, DP) and (chunk, batch, key head, row, 2)
};

template <int DP> struct FewSmem {
    static constexpr uint32_t kTile = kKeys * 128 * (DP / 64);
    static constexpr int kStages = DP == 64 ? 8 : 4;
    static constexpr uint32_t kRing = kBox * (DP / 64), kBars = kRing + kStages * kTile;
    static constexpr uint32_t kBytes = kBars + 256 + 1024;
};

template <int DP, bool kMask>
__global__ void __launch_bounds__(kFewThreads, 2)
few_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const Params p, const Few f)
{
    typedef FewSmem<DP> L;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t *gen = raw + (base - smem_u32(raw));
    const uint32_t bars = base + L::kBars;
    const uint32_t q_full = bars, fix = bars + 8, o_full = bars + 16;
    const auto s_full = [&](int x) { return bars + 24u + 8u * x; };
    const auto p_full = [&](int x) { return bars + 40u + 8u * x; };
    const auto o_done = [&](int x) { return bars + 56u + 8u * x; };
    const auto kv_full = [&](int s) { return bars + 72u + 8u * s; };
    const auto kv_empty = [&](int s) { return bars + 72u + 8u * (L::kStages + s); };
    volatile uint32_t *slot = reinterpret_cast<volatile uint32_t *>(gen + L::kBars + 72 + 16 * L::kStages);
    int *status = &g_status;

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int chunk = blockIdx.x % f.chunks, tile = blockIdx.x / f.chunks % f.row_tiles, bk = blockIdx.x / f.chunks / f.row_tiles;
    const int kh = bk % p.k_heads, b = bk / p.k_heads;
    const int rows = p.q_len * p.group, r0 = tile * kRows, r1 = r0 + kRows < rows ? r0 + kRows : rows;
    const int keys = keys_of(p, b);
    const int kb = first_key(p, r0 / p.group) / kKeys, ke = (end_key(p, (r1 - 1) / p.group + 1, keys) + kKeys - 1) / kKeys;
    const int from = kb + chunk * f.chunk, to = from + f.chunk < ke ? from + f.chunk : ke;
    const int steps = uniform(to > from ? to - from : 0);
    if (steps == 0 && chunk > 0) return;                                   // the join does not read this chunk

    // the thread that issues the loads sets the barriers up and sends the first loads off before the others are ready
    if (threadIdx.x == 160) {
        failed() = 0;
        acp::mbar_init(q_full, 128); acp::mbar_init(o_full, 1); acp::mbar_init(fix, 1);
        for (int x = 0; x < 2; ++x) { acp::mbar_init(s_full(x), 1); acp::mbar_init(o_done(x), 1); acp::mbar_init(p_full(x), (uint32_t)(r1 - r0 + 31) / 32u * 32u); }
        for (int s = 0; s < L::kStages; ++s) { acp::mbar_init(kv_full(s), 1); acp::mbar_init(kv_empty(s), 1); }
        acp::fence_barrier_init();
        acp::fence_async_smem();
        if (steps > 0) {
            acp::mbar_expect_tx(kv_full(0), L::kTile);
            load_tile<DP, kKeys>(base + L::kRing, &mk, kv_full(0), from * kKeys, kh, b);
            prefetch_map(&mv);
        }
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(bars + 72u + 16u * L::kStages) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *slot, tO = tmem + 128u;

    if (warp == 5) {
        bool ok = true;
        int s = 1;                                                        // K of the first tile is under way
        uint32_t ph = 0;
        for (int x = 1; x < 2 * steps && ok; ++x) {
            const int row = (from + x / 2) * kKeys;
            ok = wait_warp(kv_empty(s), ph ^ 1u, 1, status);
            if (!ok) break;
            const uint32_t dst = base + L::kRing + s * L::kTile;
            const bool cut = (x & 1) && keys < p.k_len && row + kKeys > keys;
            if (lane == 0) {
                const uint32_t bar = cut ? fix : kv_full(s);
                acp::mbar_expect_tx(bar, L::kTile);
                load_tile<DP, kKeys>(dst, (x & 1) ? &mv : &mk, bar, row, kh, b);
            }
            if (cut) {
                ok = wait_warp(fix, 0u, 2, status);
                if (!ok) break;
                clear_rows<DP, kKeys>(gen + (dst - base), keys - row);
                if (lane == 0) acp::mbar_arrive(kv_full(s));
            }
            __syncwarp();
            if (++s == L::kStages) { s = 0; ph ^= 1u; }
        }
    } else if (warp == 4) {
        if (steps > 0) {
            const bool one = elect();
            const int slices = (p.head_size + 15) / 16;
            const auto stage = [&](int x) { return base + L::kRing + (uint32_t)(x % L::kStages) * L::kTile; };
            const auto full = [&](int x, int code) { return wait_warp(kv_full(x % L::kStages), (uint32_t)(x / L::kStages) & 1u, code, status); };
            const auto scores = [&](int j) {
                if (!full(2 * j, 4)) return false;
                fence_after();
                if (one) {
                    product_rows<DP, kKeys>(tmem + 64u * (j & 1), base, stage(2 * j), slices);
                    commit(s_full(j & 1));
                    commit(kv_empty((2 * j) % L::kStages));
                }
                __syncwarp();
                return true;
            };
            bool ok = wait_warp(q_full, 0u, 3, status) && scores(0);
            for (int j = 0; j < steps && ok; ++j) {
                if (j + 1 < steps) ok = scores(j + 1);                    // over P(j - 1), behind the product that read it
                ok = ok && full(2 * j + 1, 5) && wait_warp(p_full(j & 1), (uint32_t)(j / 2) & 1u, 6, status);
                if (!ok) break;
                fence_after();
                if (one) {
                    product_cols<DP, kKeys>(tO, tmem + 64u * (j & 1), stage(2 * j + 1), j != 0);
                    commit(kv_empty((2 * j + 1) % L::kStages));
                    commit(o_done(j & 1));
                }
                __syncwarp();
            }
            if (ok && one) commit(o_full);
        }
    } else {
        const int r = r0 + threadIdx.x, i = r / p.group, h = kh * p.group + r % p.group;
        const bool live = r0 + 32 * warp < r1;                            // warps without rows take no part
        if (steps > 0) {
            // this row of Q, 16-byte pieces in the 128-byte swizzle (piece c of row x lies at c ^ (x & 7))
            const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(p.q.p) + b * p.q.b + h * p.q.h + i * p.q.t;
            for (int c = 0; c < DP / 8; ++c) {
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (r < r1) {
                    if (c * 8 + 8 <= p.head_size) w = *reinterpret_cast<const uint4 *>(q + c * 8);
                    else {
                        union { uint4 v; __nv_bfloat16 e[8]; } u;
                        u.v = w;
                        for (int e = 0; e < 8; ++e)
                            if (c * 8 + e < p.head_size) u.e[e] = q[c * 8 + e];
                        w = u.v;
                    }
                }
                *reinterpret_cast<uint4 *>(gen + (c / 8) * kBox + threadIdx.x * 128 + ((c % 8) ^ (threadIdx.x & 7)) * 16) = w;
            }
            acp::fence_async_smem();
            acp::mbar_arrive(q_full);
        }
        const uint32_t lanes = (uint32_t)warp << 21;
        const float c = kMask ? kLog2e : p.scale * kLog2e;
        const float slack = 8.0f / c;
        float m = -CUDART_INF_F, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < steps && live; ++j) {
            ok = wait(s_full(j & 1), (uint32_t)(j / 2) & 1u, 7, status);
            if (!__all_sync(~0u, ok)) { ok = false; break; }
            fence_after();
            const int j0 = (from + j) * kKeys;
            const uint32_t tS = tmem + lanes + 64u * (j & 1);
            int lo = 0, hi = keys - j0;                                   // visible columns [lo, hi) of this row
            if (p.causal && i + p.offset + 1 - j0 < hi) hi = i + p.offset + 1 - j0;
            if (p.window) lo = i + p.offset - p.window + 1 - j0;
            uint32_t s[kKeys];
            ld32(tS, s);
            ld32(tS + 32u, s + 32);
            wait_ld();
            if (kMask) {
#pragma unroll
                for (int x = 0; x < kKeys; ++x)
                    s[x] = __float_as_uint(x >= lo && x < hi && r < r1 ? masked_score(p, __uint_as_float(s[x]) * p.scale, b, h, i, j0 + x) : -CUDART_INF_F);
            } else if (__any_sync(~0u, lo > 0 || hi < kKeys)) {
#pragma unroll
                for (int x = 0; x < kKeys; ++x)
                    if (x < lo || x >= hi) s[x] = 0xff800000u;
            }
            const float top = row_max<kKeys>(s);
            if (__any_sync(~0u, top > m + slack || (m == -CUDART_INF_F && top > m))) {
                const float raised = fmaxf(m, top);
                const float g = m == -CUDART_INF_F ? 0.0f : ex2((m - raised) * c);
                l *= g;
                m = raised;
                if (j > 0) {
                    // P(j - 1) V is done.  P(j - 3) V on the same barrier was long before: S(j) came behind it, so the parity is unambiguous.
                    ok = wait(o_done((j - 1) & 1), (uint32_t)((j - 1) / 2) & 1u, 9, status);
                    if (!__all_sync(~0u, ok)) { ok = false; break; }
                    fence_after();
#pragma unroll
                    for (int x = 0; x < DP / 32; ++x) {
                        uint32_t o[32];
                        ld32(tO + lanes + 32u * x, o);
                        wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * g);
                        st32(tO + lanes + 32u * x, o);
                    }
                }
            }
            Exponentials<kMask> ex(m == -CUDART_INF_F ? 0.0f : m, c);
#pragma unroll
            for (int x = 0; x < kKeys / 16; ++x) ex.piece(s + 16 * x, tS + 8u * x);
            l += ex.sum();
            wait_st();
            fence_before();
            acp::mbar_arrive(p_full(j & 1));
        }
        if (ok && live) {
            if (steps > 0) {
                ok = wait(o_full, 0u, 8, status);
                ok = __all_sync(~0u, ok);
                fence_after();
            }
            const float top = kMask ? m : m * p.scale;
            const long long at = ((long long)b * p.q_heads + h) * p.q_len + i;
            const long long part = ((long long)chunk * p.batch * p.k_heads + bk) * rows + r;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out) + b * p.out_b + h * p.out_h + i * p.out_t;
            if (ok && r < r1) {
                if (f.chunks > 1) { f.stat[2 * part] = top; f.stat[2 * part + 1] = l; }
                else {
                    p.row_max[at] = top;
                    p.row_sum[at] = l;
                    if (p.lse) p.lse[at] = l == 0.0f ? -CUDART_INF_F : top + log2f(l) * kLn2;
                }
            }
#pragma unroll 1
            for (int x = 0; x < DP / 32; ++x) {
                uint32_t o[32];
                if (steps > 0) { ld32(tO + lanes + 32u * x, o); wait_ld(); }
                else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
                if (!ok || r >= r1) continue;
                if (f.chunks > 1) {
                    uint4 *dst = reinterpret_cast<uint4 *>(f.out + part * DP + 32 * x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dst[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                } else {
                    store_piece(out, 32 * x, p.head_size, o, inv);
                    if (p.o_low) store_rest(static_cast<__nv_bfloat16 *>(p.o_low) + (out - static_cast<__nv_bfloat16 *>(p.out)), 32 * x, p.head_size, o, inv);
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    linger_if_failed();
    if (warp == 4) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem));
    }
}

// One warp a row: joins the chunks' results in order.
template <int DP> __global__ void __launch_bounds__(128) join_kernel(const Params p, const Few f)
{
    pdl_wait();
    const int rows = p.q_len * p.group;
    const long long total = (long long)p.batch * p.k_heads * rows, row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= total) return;
    const int lane = threadIdx.x & 31, r = (int)(row % rows), bk = (int)(row / rows), kh = bk % p.k_heads, b = bk / p.k_heads;
    const int i = r / p.group, h = kh * p.group + r % p.group;
    // chunks that hold keys of this row's tile; the first always wrote
    const int r0 = r / kRows * kRows, r1 = r0 + kRows < rows ? r0 + kRows : rows;
    const int kb = first_key(p, r0 / p.group) / kKeys, ke = (end_key(p, (r1 - 1) / p.group + 1, keys_of(p, b)) + kKeys - 1) / kKeys;
    int n = ke > kb ? (ke - kb + f.chunk - 1) / f.chunk : 1;
    if (n > f.chunks) n = f.chunks;
    float m = -CUDART_INF_F;
    for (int x = lane; x < n; x += 32) m = fmaxf(m, f.stat[2 * (x * total + row)]);
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const float ref = m == -CUDART_INF_F ? 0.0f : m;
    float l = 0.0f, acc[DP / 32];
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) acc[e] = 0.0f;
    for (int x = 0; x < n; ++x) {
        const float2 s = *reinterpret_cast<const float2 *>(f.stat + 2 * (x * total + row));
        const float g = s.x == -CUDART_INF_F ? 0.0f : ex2((s.x - ref) * kLog2e);
        const float *o = f.out + (x * total + row) * DP + lane * (DP / 32);
        l = fmaf(s.y, g, l);
#pragma unroll
        for (int e = 0; e < DP / 32; ++e) acc[e] = fmaf(o[e], g, acc[e]);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const long long at = b * p.out_b + h * p.out_h + i * p.out_t;
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) {
        const int c = lane * (DP / 32) + e;
        if (c >= p.head_size) continue;
        const __nv_bfloat16 v = __float2bfloat16_rn(acc[e] * inv);
        static_cast<__nv_bfloat16 *>(p.out)[at + c] = v;
        if (p.o_low) static_cast<__nv_bfloat16 *>(p.o_low)[at + c] = __float2bfloat16_rn(acc[e] * inv - __bfloat162float(v));
    }
    if (lane == 0) {
        const long long st = ((long long)b * p.q_heads + h) * p.q_len + i;
        p.row_max[st] = m;
        p.row_sum[st] = l;
        if (p.lse) p.lse[st] = l == 0.0f ? -CUDART_INF_F : m + log2f(l) * kLn2;
    }
}

}  // namespace tc
}  // namespace attn
}  // namespace axs6
