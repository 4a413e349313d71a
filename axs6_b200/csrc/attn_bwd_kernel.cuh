// Attention backward on the tensor cores (bf16 tensors).  With c = scale log2 e and per row L = log2 of the forward's sum of exp2(c s):
//     P = exp2(c S - L)    dV = P^T dO    dP = dO V^T    dS = P (dP - delta), delta = rowsum(dO O)    dQ = scale dS K    dK = scale dS^T Q
// Two kernels, both recomputing S and dP: one per 128 keys (dK, dV; it also walks the query heads that share the key head), one per 128
// queries (dQ).  That is 7 products a tile pair instead of the 5 that one kernel would need, and in return every output has one writer:
// no fp32 copy of dQ in memory, no atomics, the same bits every time.  P and dS are rounded to bf16 as operands; everything else is fp32.
//
// Both kernels: warps 0-15 do the elementwise part (row = lane of tensor memory), warp 16 issues the products, warp 17 loads.  P and dS go back
// to tensor memory over fp32 columns that have been read and are the A operands of the next products, so shared memory holds nothing but
// loaded tiles.  Within a step the probabilities need S, dS needs dP and the next products need both: a chain during which either the
// exponential unit or the tensor cores idle.  Where tensor memory has room for a second S, the warps are two sets of eight that take the even
// and the odd steps: dQ (S, S, dP, dQ), and dK, dV at D = 64 (S, S, dP, dK, dV; P and dS share the columns of S, so that dP is free as
// soon as it is read).  dK, dV at D = 128 has one set of sixteen (S, dP, dK, dV; P over S, dS over dP).  Every barrier that a set waits on
// is its own: with one for both, a parity wait could not tell a step from the one before the other set's.
//
// Bound: tensor cores.  An M = 128, K = 16 product takes 64 clocks for any N up to 128: per 128 x 128 tile dK and dV 2048 clocks at D = 128 and
// 1536 at D = 64, dQ 1536 and 1024; exp2 takes 1024 in each.  (Two sets at D = 128 with S and dP for 64 queries at a time: 3072, and slower.)
// Measured, both kernels and the row sums: D = 128, 32 / 8 heads, 8192 x 8192, causal: 1500 us, 916 TFLOP/s of the five products and 1280 of the
// seven that run, 0.92 of what the power cap leaves a plain GEMM; D = 64, 64 heads, 4096 x 4096: 1162 us; 16 x 8 heads, 1024 x 1024, causal: 151 us.
#pragma once
#include "attn_tc.cuh"

namespace axs6 {
namespace attn {
namespace tc {

constexpr int kBwdThreads = 640;
// Registers: launched with 96 a thread, 5 x 96 = 480; 112 for the four warpgroups that hold up to 64 probabilities a thread, 32 for the last
constexpr int kBwdRegsMore = 112, kBwdRegsLess = 32;

// Per row: what the probabilities are taken relative to, and delta; arrays padded to whole tiles per head, so that they load in bulk.
// Rows behind the last query and rows without keys get L = +inf: probability 0.
struct RowData {
    float *shift;       // without a mask: L; with one: the row's maximum (its score may be the type's lowest value, where adding L is lost)
    float *log_sum;     // with a mask: log2 of the row's sum
    float *delta;
    int padded;         // rows of a head
};

// kLanes threads a row, 8 values each, four rows a thread
template <int kLanes> __global__ void __launch_bounds__(256) row_data_kernel(const Params p, const RowData w, int mask)
{
    constexpr int kStep = 256 / kLanes, kCtaRows = 4 * kStep;              // 64 or 128 rows of one head
    const uint32_t tiles = (uint32_t)(w.padded / kCtaRows);
    const uint32_t bh = blockIdx.x / tiles, h = bh % (uint32_t)p.q_heads, b = bh / (uint32_t)p.q_heads;
    const int first = (int)(blockIdx.x - bh * tiles) * kCtaRows + (int)threadIdx.x / kLanes, part = threadIdx.x % kLanes, c = part * 8;
    const __nv_bfloat16 *o = static_cast<const __nv_bfloat16 *>(p.o.p) + b * p.o.b + h * p.o.h;
    const __nv_bfloat16 *g = static_cast<const __nv_bfloat16 *>(p.d_o.p) + b * p.d_o.b + h * p.d_o.h;
    const __nv_bfloat16 *low = p.o_low ? static_cast<const __nv_bfloat16 *>(p.o_low) + (o - static_cast<const __nv_bfloat16 *>(p.o.p)) : nullptr;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    const bool whole = c + 8 <= p.head_size;
    uint4 x[4], y[4], t[4];
    float m[4], l[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int i = first + kStep * n;
        const long long src = (long long)bh * p.q_len + i;
        m[n] = i < p.q_len ? p.row_max[src] : 0.0f;
        l[n] = i < p.q_len ? p.row_sum[src] : 0.0f;
        const bool here = whole && i < p.q_len;
        x[n] = here ? *reinterpret_cast<const uint4 *>(o + i * p.o.t + c) : none;
        y[n] = here ? *reinterpret_cast<const uint4 *>(g + i * p.d_o.t + c) : none;
        t[n] = here && low ? *reinterpret_cast<const uint4 *>(low + i * p.o.t + c) : none;
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int i = first + kStep * n;
        const uint32_t xs[4] = {x[n].x, x[n].y, x[n].z, x[n].w}, ys[4] = {y[n].x, y[n].y, y[n].z, y[n].w}, ts[4] = {t[n].x, t[n].y, t[n].z, t[n].w};
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s = fmaf(__uint_as_float(xs[e] << 16) + __uint_as_float(ts[e] << 16), __uint_as_float(ys[e] << 16), s);
            s = fmaf(__uint_as_float(xs[e] & 0xffff0000u) + __uint_as_float(ts[e] & 0xffff0000u), __uint_as_float(ys[e] & 0xffff0000u), s);
        }
        if (!whole && i < p.q_len)
            for (int e = c; e < p.head_size; ++e)
                s = fmaf(__bfloat162float(o[i * p.o.t + e]) + (low ? __bfloat162float(low[i * p.o.t + e]) : 0.0f), __bfloat162float(g[i * p.d_o.t + e]), s);
        for (int z = kLanes / 2; z; z >>= 1) s += __shfl_xor_sync(~0u, s, z);
        if (part == 0) {
            float shift = mask ? 0.0f : CUDART_INF_F, log_sum = CUDART_INF_F;
            if (l[n] != 0.0f) { log_sum = log2f(l[n]); shift = mask ? m[n] : fmaf(m[n], kLog2e, log_sum); }
            const long long at = (long long)bh * w.padded + i;
            w.shift[at] = shift;
            if (mask) w.log_sum[at] = log_sum;
            w.delta[at] = s;
        }
    }
}

// ------------------------------------------------------------------------------------------------ dK, dV
template <int DP> struct DkvSmem {
    static constexpr uint32_t kTile = kBox * (DP / 64);
    static constexpr int kStages = DP == 64 ? 4 : 2;
    static constexpr int kSets = DP == 64 ? 2 : 1, kCols = 32 * kSets;         // sets of warps, columns (queries) of a thread
    static constexpr uint32_t kVec = 3 * kRows * 4;                            // shift, log_sum, delta
    static constexpr uint32_t kStage = 2 * kTile;                              // Q, dO
    static constexpr uint32_t kRing = 2 * kTile, kVecs = kRing + kStages * kStage, kBars = kVecs + kStages * kVec;
    static constexpr uint32_t kBytes = kBars + 512 + 1024;
};

template <int DP, bool kMask>
__global__ void __launch_bounds__(kBwdThreads, 1)
dkv_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
           const __grid_constant__ CUtensorMap mg, const Params p, const RowData w)
{
    typedef DkvSmem<DP> L;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t *gen = raw + (base - smem_u32(raw));
    const uint32_t bars = base + L::kBars;
    const uint32_t kv_full = bars, done = bars + 8;
    // of the set that takes step x
    constexpr int kSets = L::kSets, kCols = L::kCols;
    const auto s_full = [&](int x) { return bars + 16u + 8u * (x % kSets); };
    const auto d_full = [&](int x) { return bars + 32u + 8u * (x % kSets); };
    const auto p_full = [&](int x) { return bars + 48u + 8u * (x % kSets); };
    const auto ds_full = [&](int x) { return bars + 64u + 8u * (x % kSets); };
    const auto turn = [&](int x) { return (uint32_t)(x / kSets) & 1u; };        // the phase of step x on them
    const auto q_full = [&](int s) { return bars + 80u + 8u * s; };
    const auto g_full = [&](int s) { return bars + 80u + 8u * (L::kStages + s); };
    const auto empty = [&](int s) { return bars + 80u + 8u * (2 * L::kStages + s); };
    constexpr uint32_t kSlot = 80 + 24 * L::kStages;
    volatile uint32_t *slot = reinterpret_cast<volatile uint32_t *>(gen + L::kBars + kSlot);
    int *status = &g_status;

    pdl_launch_dependents();                                              // the dQ kernel's CTAs may take the SMs that this grid's last ones leave
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int heads = p.batch * p.k_heads;
    const int bh = blockIdx.x % heads, kh = bh % p.k_heads, b = bh / p.k_heads;
    const int j0 = (int)(blockIdx.x / heads) * kRows;                     // the first keys of a causal call have the longest walk: first
    const int keys = keys_of(p, b);
    const int j1 = j0 + kRows < keys ? j0 + kRows : keys;
    const int ib = first_query(p, j0) / kRows;
    const int ie = j0 < keys ? (end_query(p, j1) + kRows - 1) / kRows : 0;
    const int per_head = uniform(ie > ib ? ie - ib : 0), steps = per_head * p.group;

    // the thread that issues the loads sets the barriers up and sends the first loads off before the others are ready
    if (threadIdx.x == 544) {
        failed() = 0;
        acp::mbar_init(kv_full, 1); acp::mbar_init(done, 1);
        for (int x = 0; x < kSets; ++x) { acp::mbar_init(s_full(x), 1); acp::mbar_init(d_full(x), 1); acp::mbar_init(p_full(x), 512 / kSets); acp::mbar_init(ds_full(x), 512 / kSets); }
        for (int s = 0; s < L::kStages; ++s) { acp::mbar_init(q_full(s), 1); acp::mbar_init(g_full(s), 1); acp::mbar_init(empty(s), 1); }
        acp::fence_barrier_init();
        acp::fence_async_smem();
        if (steps > 0) {
            acp::mbar_expect_tx(kv_full, 2 * L::kTile);
            load_tile<DP>(base, &mk, kv_full, j0, kh, b);
            load_tile<DP>(base + L::kTile, &mv, kv_full, j0, kh, b);
            prefetch_map(&mq);
            prefetch_map(&mg);
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
    const auto tS = [&](int x) { return tmem + 128u * (x % kSets); };
    const uint32_t tD = tmem + 128u * kSets, tV = tmem + 512u - 2 * DP, tK = tmem + 512u - DP;
    // P over the first columns that a thread read of S; dS over the columns behind them, or over those of dP
    const auto tG = [&](int x) { return kSets == 2 ? tS(x) + kCols / 2 : tD; };

    if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBwdRegsLess));
    if (warp == 17) {
        if (lane == 0 && steps > 0) {
            int s = 0;
            uint32_t ph = 0;
            for (int x = 0; x < steps; ++x) {
                if (!wait(empty(s), ph ^ 1u, 21, status)) break;
                const int h = kh * p.group + x / per_head, i0 = (ib + x % per_head) * kRows;
                const uint32_t dst = base + L::kRing + s * L::kStage, vec = base + L::kVecs + s * L::kVec;
                const long long at = ((long long)b * p.q_heads + h) * w.padded + i0;
                acp::mbar_expect_tx(q_full(s), L::kTile + (kMask ? 2 : 1) * kRows * 4);
                load_tile<DP>(dst, &mq, q_full(s), i0, h, b);
                acp::bulk_load(vec, w.shift + at, kRows * 4, q_full(s));
                if (kMask) acp::bulk_load(vec + kRows * 4, w.log_sum + at, kRows * 4, q_full(s));
                acp::mbar_expect_tx(g_full(s), L::kTile + kRows * 4);
                load_tile<DP>(dst + L::kTile, &mg, g_full(s), i0, h, b);
                acp::bulk_load(vec + 2 * kRows * 4, w.delta + at, kRows * 4, g_full(s));
                if (++s == L::kStages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 16) {
        if (steps > 0) {
            const bool one = elect();
            const int slices = (p.head_size + 15) / 16;
            const auto stage = [&](int x) { return base + L::kRing + (uint32_t)(x % L::kStages) * L::kStage; };
            const auto scores = [&](int x) {                              // S^T = K Q^T
                if (!wait_warp(q_full(x % L::kStages), (uint32_t)(x / L::kStages) & 1u, 22, status)) return false;
                fence_after();
                if (one) {
                    product_rows<DP>(tS(x), base, stage(x), slices);
                    commit(s_full(x));
                }
                __syncwarp();
                return true;
            };
            const auto grads = [&](int x) {                               // dP^T = V dO^T
                if (!wait_warp(g_full(x % L::kStages), (uint32_t)(x / L::kStages) & 1u, 23, status)) return false;
                fence_after();
                if (one) {
                    product_rows<DP>(tD, base + L::kTile, stage(x) + L::kTile, slices);
                    commit(d_full(x));
                }
                __syncwarp();
                return true;
            };
            bool ok = wait_warp(kv_full, 0u, 24, status);
            for (int x = 0; x < kSets && x < steps && ok; ++x) ok = scores(x);
            ok = ok && grads(0);
            for (int x = 0; x < steps && ok; ++x) {
                ok = wait_warp(p_full(x), turn(x), 25, status);
                if (!ok) break;
                fence_after();
                if (one) product_cols<DP, kRows, kCols>(tV, tS(x), stage(x) + L::kTile, x != 0);      // dV += P^T dO
                __syncwarp();
                if (kSets == 1 && x + 1 < steps) ok = scores(x + 1);
                ok = ok && wait_warp(ds_full(x), turn(x), 26, status);
                if (!ok) break;
                fence_after();
                if (kSets == 2 && x + 1 < steps) ok = grads(x + 1);       // dP of this step has been read
                if (!ok) break;
                if (one) {
                    product_cols<DP, kRows, kCols>(tK, tG(x), stage(x), x != 0);                      // dK += dS^T Q
                    commit(empty(x % L::kStages));
                }
                __syncwarp();
                if (kSets == 1 && x + 1 < steps) ok = grads(x + 1);
                if (kSets == 2 && x + 2 < steps) ok = scores(x + 2);      // over P and dS of this step
            }
            if (ok && one) commit(done);
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBwdRegsMore));
        const int set = kSets == 2 ? warp >> 3 : 0, part = kSets == 2 ? (warp >> 2) & 1 : warp >> 2, row = threadIdx.x & 127, j = j0 + row;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21, mine = lanes + (uint32_t)(kCols * part);      // this warp's lanes and columns
        const float c = p.scale * kLog2e;
        bool ok = true;
        for (int x = set; x < steps; x += kSets) {
            const uint32_t ring = (uint32_t)(x / L::kStages) & 1u;
            const int s = x % L::kStages, h = kh * p.group + x / per_head, i0 = (ib + x % per_head) * kRows;
            const float *vec = reinterpret_cast<const float *>(gen + L::kVecs + s * L::kVec) + kCols * part;
            ok = wait(s_full(x), turn(x), 27, status) && wait(q_full(s), ring, 28, status);
            if (!__all_sync(~0u, ok)) { ok = false; break; }
            fence_after();
            uint32_t r[kCols];
#pragma unroll
            for (int e = 0; e < kCols; e += 32) ld32(tS(x) + mine + (uint32_t)e, r + e);
            wait_ld();
            const int first = i0 + kCols * part;                          // query of this thread's column 0
            if (kMask) {
#pragma unroll
                for (int e = 0; e < kCols; ++e) {
                    const float y = sees(p, first + e, j, keys) ? masked_score(p, __uint_as_float(r[e]) * p.scale, b, h, first + e, j) : -CUDART_INF_F;
                    r[e] = __float_as_uint(y == -CUDART_INF_F ? 0.0f : ex2(fmaf(y - vec[e], kLog2e, -vec[kRows + e])));
                }
            } else {
#pragma unroll
                for (int e = 0; e < kCols; e += 4) {
                    const float4 sh = *reinterpret_cast<const float4 *>(vec + e);
                    r[e] = __float_as_uint(ex2(fmaf(__uint_as_float(r[e]), c, -sh.x)));
                    r[e + 1] = __float_as_uint(ex2(fmaf(__uint_as_float(r[e + 1]), c, -sh.y)));
                    r[e + 2] = __float_as_uint(ex2(fmaf(__uint_as_float(r[e + 2]), c, -sh.z)));
                    r[e + 3] = __float_as_uint(ex2(fmaf(__uint_as_float(r[e + 3]), c, -sh.w)));
                }
                if ((p.causal && j0 + kRows - 1 > i0 + p.offset) || (p.window && j0 <= i0 + kRows - 1 + p.offset - p.window)) {
                    // columns [lo, hi) see this key
                    const int lo = p.causal ? j - p.offset - first : 0, hi = p.window ? j - p.offset + p.window - first : kCols;
#pragma unroll
                    for (int e = 0; e < kCols; ++e)
                        if (e < lo || e >= hi) r[e] = 0u;
                }
            }
#pragma unroll
            for (int e = 0; e < kCols / 16; ++e) {
                uint32_t y[8];
#pragma unroll
                for (int z = 0; z < 8; ++z) y[z] = pack2(__uint_as_float(r[16 * e + 2 * z]), __uint_as_float(r[16 * e + 2 * z + 1]));
                st8(tS(x) + mine + 8u * e, y);
            }
            wait_st();
            fence_before();
            acp::mbar_arrive(p_full(x));
            ok = wait(d_full(x), turn(x), 29, status) && wait(g_full(s), ring, 30, status);
            if (!__all_sync(~0u, ok)) { ok = false; break; }
            fence_after();
            const float *del = vec + 2 * kRows;
#pragma unroll
            for (int n = 0; n < kCols; n += 32) {
                uint32_t d[32];
                ld32(tD + mine + (uint32_t)n, d);
                wait_ld();
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t y[8];
#pragma unroll
                    for (int z = 0; z < 8; z += 2) {
                        const int a = 16 * e + 2 * z;
                        const float4 de = *reinterpret_cast<const float4 *>(del + n + a);
                        y[z] = pack2(__uint_as_float(r[n + a]) * (__uint_as_float(d[a]) - de.x), __uint_as_float(r[n + a + 1]) * (__uint_as_float(d[a + 1]) - de.y));
                        y[z + 1] = pack2(__uint_as_float(r[n + a + 2]) * (__uint_as_float(d[a + 2]) - de.z), __uint_as_float(r[n + a + 3]) * (__uint_as_float(d[a + 3]) - de.w));
                    }
                    st8(tG(x) + mine + (uint32_t)(n / 2 + 8 * e), y);
                }
            }
            wait_st();
            fence_before();
            acp::mbar_arrive(ds_full(x));
        }
        if (ok && steps > 0) {
            ok = wait(done, 0u, 31, status);
            ok = __all_sync(~0u, ok);
            fence_after();
        }
        if (ok) {
            // warps 0-7 write dV, warps 8-15 dK, each half of the columns; keys behind the length get zeros
            const int key = warp >> 3, side = (warp >> 2) & 1;
            const uint32_t acc = (key ? tK : tV) + lanes;
            __nv_bfloat16 *out = key ? static_cast<__nv_bfloat16 *>(p.dk) + b * p.dk_b + kh * p.dk_h + j * p.dk_t
                                     : static_cast<__nv_bfloat16 *>(p.dv) + b * p.dv_b + kh * p.dv_h + j * p.dv_t;
            const float f = key ? p.scale : 1.0f;
#pragma unroll 1
            for (int x = side * (DP / 64); x < (side + 1) * (DP / 64); ++x) {
                uint32_t o[32];
                if (steps > 0) { ld32(acc + 32u * x, o); wait_ld(); }
                if (steps == 0 || j >= keys) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
                if (j < p.k_len) store_piece(out, 32 * x, p.head_size, o, f);
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

// ------------------------------------------------------------------------------------------------ dQ
template <int DP> struct DqSmem {
    static constexpr uint32_t kTile = kBox * (DP / 64);
    static constexpr int kK = DP == 64 ? 4 : 3, kV = DP == 64 ? 4 : 2;
    static constexpr uint32_t kRingK = 2 * kTile, kRingV = kRingK + kK * kTile, kBars = kRingV + kV * kTile;
    static constexpr uint32_t kBytes = kBars + 512 + 1024;
};

template <int DP, bool kMask>
__global__ void __launch_bounds__(kBwdThreads, 1)
dq_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
          const __grid_constant__ CUtensorMap mg, const Params p, const RowData w)
{
    typedef DqSmem<DP> L;
    extern __shared__ uint8_t raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t *gen = raw + (base - smem_u32(raw));
    const uint32_t bars = base + L::kBars;
    const uint32_t q_full = bars, g_full = bars + 8, done = bars + 16, fix = bars + 24;
    // of set x
    const auto s_full = [&](int x) { return bars + 32u + 8u * (x & 1); };
    const auto d_full = [&](int x) { return bars + 48u + 8u * (x & 1); };
    const auto ds_full = [&](int x) { return bars + 64u + 8u * (x & 1); };
    const auto k_full = [&](int s) { return bars + 80u + 8u * s; };
    const auto k_empty = [&](int s) { return bars + 80u + 8u * (L::kK + s); };
    const auto v_full = [&](int s) { return bars + 80u + 8u * (2 * L::kK + s); };
    const auto v_empty = [&](int s) { return bars + 80u + 8u * (2 * L::kK + L::kV + s); };
    constexpr uint32_t kSlot = 80 + 16 * (L::kK + L::kV);
    volatile uint32_t *slot = reinterpret_cast<volatile uint32_t *>(gen + L::kBars + kSlot);
    int *status = &g_status;

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int heads = p.batch * p.q_heads;
    const int bh = blockIdx.x % heads, h = bh % p.q_heads, b = bh / p.q_heads, kh = h / p.group;
    const int i0 = (int)((gridDim.x - 1 - blockIdx.x) / heads) * kRows;
    const int keys = keys_of(p, b);
    const int kb = first_key(p, i0) / kRows;
    const int ke = (end_key(p, i0 + kRows < p.q_len ? i0 + kRows : p.q_len, keys) + kRows - 1) / kRows;
    const int steps = uniform(ke > kb ? ke - kb : 0);

    // the thread that issues the loads sets the barriers up and sends the first loads off before the others are ready
    if (threadIdx.x == 544) {
        failed() = 0;
        acp::mbar_init(q_full, 1); acp::mbar_init(g_full, 1); acp::mbar_init(done, 1); acp::mbar_init(fix, 1);
        for (int x = 0; x < 2; ++x) { acp::mbar_init(s_full(x), 1); acp::mbar_init(d_full(x), 1); acp::mbar_init(ds_full(x), 256); }
        for (int s = 0; s < L::kK; ++s) { acp::mbar_init(k_full(s), 1); acp::mbar_init(k_empty(s), 1); }
        for (int s = 0; s < L::kV; ++s) { acp::mbar_init(v_full(s), 1); acp::mbar_init(v_empty(s), 1); }
        acp::fence_barrier_init();
        acp::fence_async_smem();
        if (steps > 0) {
            acp::mbar_expect_tx(q_full, L::kTile);
            load_tile<DP>(base, &mq, q_full, i0, h, b);
            acp::mbar_expect_tx(g_full, L::kTile);
            load_tile<DP>(base + L::kTile, &mg, g_full, i0, h, b);
            prefetch_map(&mk);
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
    const auto tS = [&](int x) { return tmem + 128u * (x & 1); };
    const uint32_t tD = tmem + 256u, tQ = tmem + 384u;

    if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBwdRegsLess));
    if (warp == 17) {
        bool ok = true;
        for (int x = 0; x < steps && ok; ++x) {
            const int row = (kb + x) * kRows, ks = x % L::kK, vs = x % L::kV;
            const uint32_t kd = base + L::kRingK + ks * L::kTile, vd = base + L::kRingV + vs * L::kTile;
            ok = wait_warp(k_empty(ks), ((uint32_t)(x / L::kK) & 1u) ^ 1u, 21, status);
            if (!ok) break;
            // rows behind the length may hold anything: zeros instead (dS K, and dP where dS is 0)
            const bool cut = keys < p.k_len && row + kRows > keys;
            if (!cut) {
                if (lane == 0) {
                    acp::mbar_expect_tx(k_full(ks), L::kTile);
                    load_tile<DP>(kd, &mk, k_full(ks), row, kh, b);
                }
                ok = wait_warp(v_empty(vs), ((uint32_t)(x / L::kV) & 1u) ^ 1u, 22, status);
                if (!ok) break;
                if (lane == 0) {
                    acp::mbar_expect_tx(v_full(vs), L::kTile);
                    load_tile<DP>(vd, &mv, v_full(vs), row, kh, b);
                }
            } else {                                                      // the last tile of the walk
                ok = wait_warp(v_empty(vs), ((uint32_t)(x / L::kV) & 1u) ^ 1u, 22, status);
                if (!ok) break;
                if (lane == 0) {
                    acp::mbar_expect_tx(fix, 2 * L::kTile);
                    load_tile<DP>(kd, &mk, fix, row, kh, b);
                    load_tile<DP>(vd, &mv, fix, row, kh, b);
                }
                ok = wait_warp(fix, 0u, 23, status);
                if (!ok) break;
                clear_rows<DP>(gen + (kd - base), keys - row);
                clear_rows<DP>(gen + (vd - base), keys - row);
                if (lane == 0) { acp::mbar_arrive(k_full(ks)); acp::mbar_arrive(v_full(vs)); }
            }
            __syncwarp();
        }
    } else if (warp == 16) {
        if (steps > 0) {
            const bool one = elect();
            const int slices = (p.head_size + 15) / 16;
            const auto kt = [&](int x) { return base + L::kRingK + (uint32_t)(x % L::kK) * L::kTile; };
            const auto vt = [&](int x) { return base + L::kRingV + (uint32_t)(x % L::kV) * L::kTile; };
            const auto scores = [&](int x) {                              // S = Q K^T
                if (!wait_warp(k_full(x % L::kK), (uint32_t)(x / L::kK) & 1u, 24, status)) return false;
                fence_after();
                if (one) {
                    product_rows<DP>(tS(x), base, kt(x), slices);
                    commit(s_full(x));
                }
                __syncwarp();
                return true;
            };
            const auto grads = [&](int x) {                               // dP = dO V^T
                if (!wait_warp(v_full(x % L::kV), (uint32_t)(x / L::kV) & 1u, 25, status)) return false;
                fence_after();
                if (one) {
                    product_rows<DP>(tD, base + L::kTile, vt(x), slices);
                    commit(d_full(x));
                    commit(v_empty(x % L::kV));
                }
                __syncwarp();
                return true;
            };
            bool ok = wait_warp(q_full, 0u, 26, status) && scores(0) && wait_warp(g_full, 0u, 27, status) && grads(0);
            if (ok && steps > 1) ok = scores(1);
            for (int x = 0; x < steps && ok; ++x) {
                ok = wait_warp(ds_full(x), (uint32_t)(x / 2) & 1u, 28, status);
                if (!ok) break;
                fence_after();
                if (x + 1 < steps) ok = grads(x + 1);                     // dP of this step has been read; before dQ, since the other set waits for it
                if (!ok) break;
                if (one) {
                    product_cols<DP, kRows, 64>(tQ, tS(x), kt(x), x != 0);                   // dQ += dS K
                    commit(k_empty(x % L::kK));
                }
                __syncwarp();
                if (x + 2 < steps) ok = scores(x + 2);                    // over dS of this step, behind the product that reads it
            }
            if (ok && one) commit(done);
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kBwdRegsMore));
        const int set = warp >> 3, part = (warp >> 2) & 1, row = threadIdx.x & 127, i = i0 + row;
        const uint32_t mine = ((uint32_t)(warp & 3) << 21) + 64u * part;
        const float c = p.scale * kLog2e;
        const long long at = ((long long)b * p.q_heads + h) * w.padded + i;        // padded rows exist
        const float shift = w.shift[at], log_sum = kMask ? w.log_sum[at] : 0.0f, delta = w.delta[at];
        bool ok = true;
        for (int x = set; x < steps; x += 2) {
            const uint32_t phase = (uint32_t)(x / 2) & 1u;
            ok = wait(s_full(x), phase, 29, status);
            if (!__all_sync(~0u, ok)) { ok = false; break; }
            fence_after();
            uint32_t r[64];
            ld32(tS(x) + mine, r);
            ld32(tS(x) + mine + 32u, r + 32);
            wait_ld();
            const int j0 = (kb + x) * kRows, first = j0 + 64 * part;
            if (kMask) {
#pragma unroll
                for (int e = 0; e < 64; ++e) {
                    const float y = sees(p, i, first + e, keys) ? masked_score(p, __uint_as_float(r[e]) * p.scale, b, h, i, first + e) : -CUDART_INF_F;
                    r[e] = __float_as_uint(y == -CUDART_INF_F ? 0.0f : ex2(fmaf(y - shift, kLog2e, -log_sum)));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 64; ++e) r[e] = __float_as_uint(ex2(fmaf(__uint_as_float(r[e]), c, -shift)));
                if (j0 + kRows > keys || (p.causal && j0 + kRows - 1 > i0 + p.offset) || (p.window && j0 <= i0 + kRows - 1 + p.offset - p.window)) {
                    int lo = 0, hi = keys - first;                                 // visible columns [lo, hi)
                    if (p.causal && i + p.offset + 1 - first < hi) hi = i + p.offset + 1 - first;
                    if (p.window) lo = i + p.offset - p.window + 1 - first;
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        if (e < lo || e >= hi) r[e] = 0u;
                }
            }
            ok = wait(d_full(x), phase, 30, status);
            if (!__all_sync(~0u, ok)) { ok = false; break; }
            fence_after();
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                uint32_t d[32];
                ld32(tD + mine + 32u * n, d);
                wait_ld();
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t y[8];
#pragma unroll
                    for (int z = 0; z < 8; ++z) {
                        const int a = 16 * e + 2 * z;
                        y[z] = pack2(__uint_as_float(r[32 * n + a]) * (__uint_as_float(d[a]) - delta),
                                     __uint_as_float(r[32 * n + a + 1]) * (__uint_as_float(d[a + 1]) - delta));
                    }
                    st8(tS(x) + mine + 16u * n + 8u * e, y);
                }
            }
            wait_st();
            fence_before();
            acp::mbar_arrive(ds_full(x));
        }
        if (ok && steps > 0) {
            ok = wait(done, 0u, 31, status);
            ok = __all_sync(~0u, ok);
            fence_after();
        }
        if (ok) {
            // 32 columns for four warps
            __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.dq) + b * p.dq_b + h * p.dq_h + i * p.dq_t;
            const int chunk = warp >> 2;
            if (chunk < DP / 32) {
                uint32_t o[32];
                if (steps > 0) { ld32(tQ + ((uint32_t)(warp & 3) << 21) + 32u * chunk, o); wait_ld(); }
                else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                }
                if (i < p.q_len) store_piece(out, 32 * chunk, p.head_size, o, p.scale);
            }
        }
    }
    // Launched beside the dK, dV kernel, whose results it does not need: what both read was complete when that one began.  Waiting for it here
    // lets work behind this kernel rely on both.
    pdl_wait();
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
