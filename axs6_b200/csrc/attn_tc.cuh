// Tensor-core plumbing of the attention kernels: bounded barrier waits, tensor-memory access, tcgen05.mma with A in shared or in tensor
// memory, and the shared-memory layout of (128 tokens x head) tiles.
//
// A tile is one or two boxes of 128 tokens x 64 values (128 bytes a row, 128-byte swizzle, 16 KB), the second for values 64..127.
// The same bytes serve as a K-major operand (contraction over the head's values) and as an MN-major one (contraction over the
// tokens): only the descriptors differ.
#pragma once
#include <cuda.h>

#include "async_copy.cuh"
#include "attn_common.cuh"

namespace axs6 {
namespace attn {
namespace tc {

using acp::smem_u32;

constexpr int kRows = 128;                       // tokens of a tile
constexpr int kKeys = 64;                        // keys of a tile of the few-queries kernel
constexpr uint32_t kBox = 128 * 128;             // bytes of a box
constexpr uint32_t kWaitPolls = 1u << 20;        // a poll sleeps for as long as the hardware lets it; all of them about a second

static __device__ int g_status;                  // 0, or the code of the first wait that gave up (one translation unit includes this)

// Whether a wait of this CTA gave up
__device__ __forceinline__ int &failed()
{
    __shared__ int f;
    return f;
}
// false: gave up, or somebody else did
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int code, int *status)
{
    for (uint32_t i = 0; i < kWaitPolls; ++i) {
        uint32_t ok;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((i & 63u) == 63u && *(volatile int *)status != 0) break;
    }
    atomicCAS(status, 0, code);
    *(volatile int *)&failed() = 1;
    return false;
}

// The same for a loop that a whole warp runs: one answer for all lanes
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int code, int *status) { return __all_sync(~0u, wait(bar, parity, code, status)); }

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// One lane of a warp, the same every time.  The warp that issues the products runs its loop as a whole, so that addresses and descriptors are
// uniform values, and only the instructions themselves are this lane's (a loop that a single lane runs moved each of the six operand words of
// a product into a uniform register anew, and that loop, not the tensor cores, set the pace).
__device__ __forceinline__ bool elect()
{
    uint32_t e;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(~0u, v, 0); }

// Descriptors: version 1, 128-byte swizzle, 8-row groups 1024 bytes apart.  The low word holds the address and, for MN-major tiles, the
// distance of the 64-value boxes; it advances with the contraction.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t box) { return ((addr & 0x3FFFFu) >> 4) | ((box >> 4) << 16); }

__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.b32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHigh) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc)
{
    asm volatile("{\n .reg .pred p;\n .reg .b64 y;\n setp.ne.b32 p, %4, 0;\n mov.b64 y, {%2, %5};\n"
                 " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}"
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHigh) : "memory");
}
// bf16 operands, fp32 result, M = 128
__host__ __device__ constexpr uint32_t instr(int n, int b_mn)
{
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

// D (128 x kTokens) = A B^T over the head's first 16 `slices` values (behind its size the tiles hold zeros), tiles at shared addresses `a` (128 rows) and `b` (kTokens rows), both K-major
template <int DP, int kTokens = kRows> __device__ __forceinline__ void product_rows(uint32_t d, uint32_t a, uint32_t b, int slices)
{
    const uint32_t al = desc_low(a, 0), bl = desc_low(b, 0);
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
        const uint32_t box = (uint32_t)(k / 4), step = (uint32_t)(k % 4) * 2u;
        if (k < slices) mma_ss(d, al + box * (kBox >> 4) + step, bl + box * (kTokens * 128u >> 4) + step, instr(kTokens, 0), k != 0);
    }
}
// D (128 x DP) (+)= A B over kTokens tokens: A is 128 x kTokens bf16 in tensor memory (two values a column), B a tile, MN-major.  kGroup: A's
// columns in groups of so many tokens, each over the fp32 columns it was made from: token g * kGroup at column g * kGroup.
template <int DP, int kTokens = kRows, int kGroup = kTokens> __device__ __forceinline__ void product_cols(uint32_t d, uint32_t a, uint32_t b, bool acc)
{
    const uint32_t bl = desc_low(b, kTokens * 128u);
#pragma unroll
    for (int k = 0; k < kTokens / 16; ++k)
        mma_ts(d, a + (uint32_t)(k * 16 / kGroup * kGroup) + 8u * (uint32_t)(k % (kGroup / 16)), bl + (uint32_t)k * 128u, instr(DP, 1),
               k != 0 ? 1u : (uint32_t)acc);
}

#define AXS6_REGS32(r) \
    "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), \
    "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),    \
    "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),    \
    "=r"(r[31])
// 32 columns of this thread's lane
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
                 "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];" : AXS6_REGS32(r) : "r"(addr));
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
                 "%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
                 "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr) : "memory");
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t *r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(addr));
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                   "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr) : "memory");
}
__device__ __forceinline__ void st8(uint32_t addr, const uint32_t *r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(addr) : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Maximum of a row's scores: four chains of three-way maxima
template <int kN> __device__ __forceinline__ float row_max(const uint32_t *r)
{
    float t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = __uint_as_float(r[e]);
#pragma unroll
    for (int x = 4; x + 8 <= kN; x += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = fmaxf(t[e], fmaxf(__uint_as_float(r[x + e]), __uint_as_float(r[x + 4 + e])));
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = fmaxf(t[e], __uint_as_float(r[kN - 4 + e]));
    return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
}
// Two fp32 values in one instruction
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void parts(f32x2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// exp2(c (s - ref)) of a row's scores, rounded to bf16 pairs into tensor memory, and their unrounded sum.  Without a mask tensor as one fma a
// score; with one the difference first, since the scores may be as low as the type goes.
template <bool kMask> struct Exponentials {
    float ref, c;
    f32x2 c2, shift2, part[2];
    __device__ __forceinline__ Exponentials(float ref_, float c_) : ref(ref_), c(c_)
    {
        c2 = pair(c, c);
        shift2 = pair(-ref * c, -ref * c);
        part[0] = part[1] = pair(0.0f, 0.0f);
    }
    // 16 scores into 8 columns
    __device__ __forceinline__ void piece(const uint32_t *r, uint32_t S)
    {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float u = __uint_as_float(r[2 * e]), v = __uint_as_float(r[2 * e + 1]);
            float pu, pv;
            if (kMask) {
                pu = ex2((u - ref) * c);
                pv = ex2((v - ref) * c);
            } else {
                const f32x2 x = fma2(pair(u, v), c2, shift2);
                parts(x, pu, pv);
                pu = ex2(pu);
                pv = ex2(pv);
            }
            part[e & 1] = add2(part[e & 1], pair(pu, pv));
            w[e] = pack2(pu, pv);
        }
        st8(S, w);
    }
    __device__ __forceinline__ float sum() const
    {
        float a, b;
        parts(add2(part[0], part[1]), a, b);
        return a + b;
    }
};

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int row, int head, int b)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(row), "r"(head), "r"(b) : "memory");
}
// The tokens of one head that a box holds (kTokens of them); what lies outside the tensor arrives as zeros
template <int DP, int kTokens = kRows> __device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap *map, uint32_t bar, int row, int head, int b)
{
#pragma unroll
    for (int c = 0; c < DP / 64; ++c) load_box(dst + (uint32_t)c * (kTokens * 128u), map, bar, c * 64, row, head, b);
}
// A whole warp: zeros into rows [row, 128) of a tile (0 * NaN would reach every row of a product over the tokens), seen by the tensor cores
template <int DP, int kTokens = kRows> __device__ __forceinline__ void clear_rows(uint8_t *tile, int row)
{
    const int lane = threadIdx.x & 31;
    for (int i = row * 8 + lane; i < kTokens * 8; i += 32)
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) *reinterpret_cast<uint4 *>(tile + (size_t)c * (kTokens * 128) + (size_t)i * 16) = make_uint4(0u, 0u, 0u, 0u);
    acp::fence_async_smem();
    __syncwarp();
}
// One row of a result: 32 fp32 values from column `c0` on, scaled, rounded to bf16, in 16-byte pieces where the head is that long
__device__ __forceinline__ void store_piece(__nv_bfloat16 *row, int c0, int d, const uint32_t *r, float f)
{
#pragma unroll
    for (int e = 0; e < 32; e += 8) {
        if (c0 + e + 8 <= d) {
            uint4 w;
            w.x = pack2(__uint_as_float(r[e]) * f, __uint_as_float(r[e + 1]) * f);
            w.y = pack2(__uint_as_float(r[e + 2]) * f, __uint_as_float(r[e + 3]) * f);
            w.z = pack2(__uint_as_float(r[e + 4]) * f, __uint_as_float(r[e + 5]) * f);
            w.w = pack2(__uint_as_float(r[e + 6]) * f, __uint_as_float(r[e + 7]) * f);
            *reinterpret_cast<uint4 *>(row + c0 + e) = w;
        } else {
            for (int x = e; x < e + 8; ++x)
                if (c0 + x < d) row[c0 + x] = __float2bfloat16_rn(__uint_as_float(r[x]) * f);
        }
    }
}

// What rounding left of the same values, in the same places of another tensor
__device__ __forceinline__ void store_rest(__nv_bfloat16 *row, int c0, int d, uint32_t *r, float f)
{
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        const float v = __uint_as_float(r[e]) * f;
        r[e] = __float_as_uint(v - __bfloat162float(__float2bfloat16_rn(v)));
    }
    store_piece(row, c0, d, r, 1.0f);
}

// On the way out, behind the last barrier: where a wait gave up, loads and products that were issued may still be running; they complete
// within microseconds, so every thread lingers before shared and tensor memory are released.
__device__ __forceinline__ void linger_if_failed()
{
    if (*(volatile int *)&failed() != 0)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// ---------------------------------------------------------------------------------------------- host
// (value, token, head, batch) map of a bf16 tensor, boxes of 64 values x `rows` tokens
inline bool make_map(CUtensorMap *map, const void *ptr, int d, int64_t tokens, int64_t heads, int64_t batch, int64_t st, int64_t sh, int64_t sb,
                     int rows = kRows)
{
    acp::EncodeTiledFn fn = acp::encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)tokens, (cuuint64_t)heads, (cuuint64_t)batch};
    const cuuint64_t any = (cuuint64_t)((d + 7) / 8 * 16);            // stride of an extent of one: never used, but checked
    const cuuint64_t strides[3] = {tokens > 1 ? (cuuint64_t)st * 2 : any, heads > 1 ? (cuuint64_t)sh * 2 : any, batch > 1 ? (cuuint64_t)sb * 2 : any};
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, es[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tc
}  // namespace attn
}  // namespace axs6
