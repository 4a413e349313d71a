// Rotary positions: every pair (a, b) of a head's first `rotated` values is turned by the angle pos * w_i,
//     a' = g (a cos t - b sin t)     b' = g (a sin t + b cos t)     t = pos * w_i,
// the remaining values are copied.  The gradient is the transpose: the same kernel with the sign of sin changed.
//
// Angles.  w_i / (2 pi) is handed over as a 64-bit fraction of a turn, so pos * turns modulo 2^64 IS the phase, exactly, by one
// wrapping integer product: at position 2^20 a product in fp32 would be off by 0.06 rad, this one by 2^-43 turns.  The upper 32
// bits, reduced to the nearest quarter turn, give an angle in [-pi/4, pi/4] with the relative error of one fp32 rounding, and
// sin / cos of it are the Taylor sums up to x^9 / x^10 (remainders (pi/4)^11 / 11! = 1.8e-9 and (pi/4)^12 / 12! = 1.1e-10).
//
// Bound: HBM, 2 * values * bytes (each value read once, written once).  A CTA takes a few tokens, computes the cos / sin of a
// token's pairs once in shared memory for all its query AND key heads, and then streams the heads in 16-byte pieces: one
// launch for q and k.  Halves of a head are two pieces (half layout) or two neighbouring pieces (interleaved).  Measured: 65536 tokens, 32 / 8 heads of
// 128, 64 values rotated: 248 us, 5.4 TB/s (0.83 of a copy); 8 x 1024 tokens, 16 / 16 heads of 64: 16.6 us; 16 tokens: 4.3 us.
#include <cuda_bf16.h>

#include "common.cuh"

namespace axs6 {
namespace rotary {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;         // tokens of a CTA
constexpr int kTableBytes = 16384;     // cos / sin of its tokens' pairs

struct Side {                          // q or k: (batch, head, token) strides in elements
    const void *x;
    void *y;
    long long xb, xh, xt, yb, yh, yt;
    int heads;
};

struct Params {
    Side side[2];
    const void *positions;
    long long pos_b, pos_t;
    const unsigned long long *turns;
    float gain;
    int pos64, interleaved, inverse;
    int tokens, head_size, pairs;      // pairs = rotated / 2
    long long total_tokens;            // batch * tokens
    int tokens_per_cta;
};

__device__ __forceinline__ float2 turn_of(unsigned long long phase, float gain, bool inverse)
{
    const uint32_t u = (uint32_t)(phase >> 32);
    const uint32_t quarter = (u + 0x20000000u) >> 30;
    const float x = (float)(int)(u - (quarter << 30)) * 1.46291807926715968e-9f;      // 2 pi / 2^32
    const float x2 = x * x;
    float s = x2 * (1.0f / 362880.0f) - 1.0f / 5040.0f;
    s = fmaf(s, x2, 1.0f / 120.0f);
    s = fmaf(s, x2, -1.0f / 6.0f);
    s = fmaf(s * x2, x, x);
    float c = x2 * (-1.0f / 3628800.0f) + 1.0f / 40320.0f;
    c = fmaf(c, x2, -1.0f / 720.0f);
    c = fmaf(c, x2, 1.0f / 24.0f);
    c = fmaf(c, x2, -0.5f);
    c = fmaf(c, x2, 1.0f);
    float cs = (quarter & 1u) ? s : c, sn = (quarter & 1u) ? c : s;                    // a quarter turn swaps them
    if (quarter == 1u || quarter == 2u) cs = -cs;
    if (quarter == 2u || quarter == 3u) sn = -sn;
    return make_float2(cs * gain, (inverse ? -sn : sn) * gain);
}

template <int kBytes> struct Piece;
template <> struct Piece<16> { typedef uint4 type; };
template <> struct Piece<8> { typedef uint2 type; };
template <> struct Piece<4> { typedef uint32_t type; };
template <> struct Piece<2> { typedef uint16_t type; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, float &o) { o = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }

// kVec: values of a piece.  A unit is two pieces: kVec pairs of the rotated part, or 2 kVec values (at the end kVec) of the rest.
template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads, 6) rotary_kernel(const Params p)
{
    typedef typename Piece<kVec * (int)sizeof(T)>::type Raw;
    __shared__ __align__(16) float2 table[kTableBytes / sizeof(float2)];
    __shared__ long long origin[kMaxTokens][4];                            // of a token in q, q's result, k, k's result
    const long long first = (long long)blockIdx.x * p.tokens_per_cta;
    const int count = (int)(p.total_tokens - first < p.tokens_per_cta ? p.total_tokens - first : p.tokens_per_cta);

    if ((int)threadIdx.x < count) {
        const long long tok = first + threadIdx.x, b = tok / p.tokens, s = tok - b * p.tokens;
        origin[threadIdx.x][0] = b * p.side[0].xb + s * p.side[0].xt;
        origin[threadIdx.x][1] = b * p.side[0].yb + s * p.side[0].yt;
        origin[threadIdx.x][2] = b * p.side[1].xb + s * p.side[1].xt;
        origin[threadIdx.x][3] = b * p.side[1].yb + s * p.side[1].yt;
    }
    for (int i = threadIdx.x; i < count * p.pairs; i += kThreads) {
        const int t = i / p.pairs, pair = i - t * p.pairs;
        const long long tok = first + t, b = tok / p.tokens, s = tok - b * p.tokens;
        const long long at = b * p.pos_b + s * p.pos_t;
        const long long pos = p.pos64 ? static_cast<const long long *>(p.positions)[at] : (long long)static_cast<const int *>(p.positions)[at];
        table[i] = turn_of((unsigned long long)pos * p.turns[pair], p.gain, p.inverse != 0);
    }
    __syncthreads();

    // (token, head, unit) of this thread's item, advanced by kThreads items at a time in mixed radix
    const uint32_t heads = (uint32_t)(p.side[0].heads + p.side[1].heads), q_heads = (uint32_t)p.side[0].heads;
    const uint32_t turned = p.pairs / kVec, rest = (p.head_size - 2 * p.pairs) / kVec, units = turned + (rest + 1) / 2;
    const uint32_t step_unit = kThreads % units, step_head = kThreads / units % heads, step_token = kThreads / units / heads;
    uint32_t unit = threadIdx.x % units, head = threadIdx.x / units % heads, t = threadIdx.x / units / heads;
    const int apart = p.interleaved ? kVec : p.pairs;
    while (t < (uint32_t)count) {
        const bool is_k = head >= q_heads;
        const Side &sd = p.side[is_k];
        const long long h = is_k ? head - q_heads : head;
        const T *x = static_cast<const T *>(sd.x) + origin[t][is_k ? 2 : 0] + h * sd.xh;
        T *y = static_cast<T *>(sd.y) + origin[t][is_k ? 3 : 1] + h * sd.yh;
        if (unit >= turned) {
            const int at = 2 * p.pairs + (int)(unit - turned) * 2 * kVec;
            const bool two = (unit - turned) * 2 + 1 < rest;
            const Raw u = *reinterpret_cast<const Raw *>(x + at);
            if (two) {
                const Raw w = *reinterpret_cast<const Raw *>(x + at + kVec);
                *reinterpret_cast<Raw *>(y + at + kVec) = w;
            }
            *reinterpret_cast<Raw *>(y + at) = u;
        } else {
            const int at = (int)unit * (p.interleaved ? 2 * kVec : kVec);
            union Buf { Raw raw[2]; T v[2 * kVec]; } in, out;
            in.raw[0] = *reinterpret_cast<const Raw *>(x + at);
            in.raw[1] = *reinterpret_cast<const Raw *>(x + at + apart);
            const float2 *cs = table + t * p.pairs + unit * kVec;
            if (p.interleaved) {
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const float a = to_f(in.v[2 * e]), c = to_f(in.v[2 * e + 1]);
                    const float2 w = cs[e];
                    from_f(fmaf(a, w.x, -(c * w.y)), out.v[2 * e]);
                    from_f(fmaf(a, w.y, c * w.x), out.v[2 * e + 1]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < kVec; ++e) {
                    const float a = to_f(in.v[e]), c = to_f(in.v[kVec + e]);
                    const float2 w = cs[e];
                    from_f(fmaf(a, w.x, -(c * w.y)), out.v[e]);
                    from_f(fmaf(a, w.y, c * w.x), out.v[kVec + e]);
                }
            }
            *reinterpret_cast<Raw *>(y + at) = out.raw[0];
            *reinterpret_cast<Raw *>(y + at + apart) = out.raw[1];
        }
        unit += step_unit; head += step_head; t += step_token;
        if (unit >= units) { unit -= units; ++head; }
        if (head >= heads) { head -= heads; ++t; }
    }
}

// Whether pieces of `vec` values can be used: every address that is touched is a multiple of the piece.
static bool fits(const Params &p, int vec, int esize)
{
    if (p.pairs % vec || (p.head_size - 2 * p.pairs) % vec) return false;
    for (const Side &s : p.side) {
        if (!s.heads) continue;
        const uintptr_t a = reinterpret_cast<uintptr_t>(s.x) | reinterpret_cast<uintptr_t>(s.y);
        if (a % (uintptr_t)(vec * esize)) return false;
        if ((s.xb | s.xh | s.xt | s.yb | s.yh | s.yt) % vec) return false;
    }
    return true;
}

}  // namespace rotary
}  // namespace axs6

AXS6_API int axs6_rotary(const void *q, void *q_out, int64_t q_heads, const int64_t *q_strides, const int64_t *q_out_strides,
                         const void *k, void *k_out, int64_t k_heads, const int64_t *k_strides, const int64_t *k_out_strides,
                         int dtype, int64_t batch, int64_t tokens, int64_t head_size, int64_t rotated,
                         const void *positions, int positions_64, int64_t pos_batch_stride, int64_t pos_token_stride,
                         const uint64_t *turns, float gain, int interleaved, int inverse, axs6_stream_t stream)
{
    using namespace axs6;
    using namespace axs6::rotary;
    if (!valid_dtype(dtype) || batch < 0 || tokens < 0 || q_heads < 0 || k_heads < 0 || head_size < 1 || rotated < 0 ||
        rotated > head_size || rotated % 2 || head_size > 4096 || q_heads > 65536 || k_heads > 65536 || tokens > INT32_MAX)
        return AXS6_ERR_ARG;
    if (q_heads + k_heads == 0 || batch == 0 || tokens == 0) return AXS6_OK;
    if ((q_heads && (!q || !q_out || !q_strides || !q_out_strides)) || (k_heads && (!k || !k_out || !k_strides || !k_out_strides)) ||
        (rotated && (!positions || !turns)))
        return AXS6_ERR_ARG;
    const DeviceInfo &d = device_info();
    if (!d.valid || !d.ok) return AXS6_ERR_DEVICE;
    Params p = {};
    auto fill = [](Side &s, const void *x, void *y, int64_t heads, const int64_t *xs, const int64_t *ys) {
        s.x = x; s.y = y; s.heads = (int)heads;
        if (heads) { s.xb = xs[0]; s.xh = xs[1]; s.xt = xs[2]; s.yb = ys[0]; s.yh = ys[1]; s.yt = ys[2]; }
    };
    fill(p.side[0], q, q_out, q_heads, q_strides, q_out_strides);
    fill(p.side[1], k, k_out, k_heads, k_strides, k_out_strides);
    p.positions = positions; p.pos64 = positions_64 != 0; p.pos_b = pos_batch_stride; p.pos_t = pos_token_stride;
    p.turns = reinterpret_cast<const unsigned long long *>(turns);
    p.gain = gain; p.interleaved = interleaved != 0; p.inverse = inverse != 0;
    p.tokens = (int)tokens; p.head_size = (int)head_size; p.pairs = (int)(rotated / 2);
    p.total_tokens = batch * tokens;
    const int esize = dtype == AXS6_F32 ? 4 : 2;
    int vec = 16 / esize;
    while (vec > 1 && !fits(p, vec, esize)) vec >>= 1;
    // Enough tokens for about four units a thread, at most what the table holds, and no fewer CTAs than SMs while tokens last.
    const int64_t per_token = (q_heads + k_heads) * (p.pairs / vec + ((head_size - rotated) / vec + 1) / 2);
    int64_t tpc = (4 * kThreads + per_token - 1) / per_token;
    if (tpc > kMaxTokens) tpc = kMaxTokens;
    if (p.pairs && tpc > kTableBytes / (int64_t)(p.pairs * sizeof(float2))) tpc = kTableBytes / (int64_t)(p.pairs * sizeof(float2));
    const int64_t even = (p.total_tokens + 2 * d.sms - 1) / (2 * d.sms);
    if (tpc > even) tpc = even;
    p.tokens_per_cta = (int)(tpc < 1 ? 1 : tpc);
    const int64_t ctas = (p.total_tokens + p.tokens_per_cta - 1) / p.tokens_per_cta;
    if (ctas > INT32_MAX) return AXS6_ERR_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned g = (unsigned)ctas;
    if (dtype == AXS6_F32) {
        if (vec == 4) rotary_kernel<float, 4><<<g, kThreads, 0, st>>>(p);
        else if (vec == 2) rotary_kernel<float, 2><<<g, kThreads, 0, st>>>(p);
        else rotary_kernel<float, 1><<<g, kThreads, 0, st>>>(p);
    } else {
        if (vec == 8) rotary_kernel<__nv_bfloat16, 8><<<g, kThreads, 0, st>>>(p);
        else if (vec == 4) rotary_kernel<__nv_bfloat16, 4><<<g, kThreads, 0, st>>>(p);
        else if (vec == 2) rotary_kernel<__nv_bfloat16, 2><<<g, kThreads, 0, st>>>(p);
        else rotary_kernel<__nv_bfloat16, 1><<<g, kThreads, 0, st>>>(p);
    }
    count_launch();
    return check_launch();
}
