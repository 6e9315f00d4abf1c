// The 8-bit latent cache: e4m3 pages whose blocks of 16 rows have one power-of-two
// scale per part (512 latent, 64 rotary columns), held as exponents.
//
// Why powers of two: x * 2^-e is exact, so a stored value is x rounded once, to
// e4m3, and re-expressing a block's earlier rows under a larger scale rounds only
// what falls into e4m3's subnormals. The choice of e and the stored bytes are
// then the same on any machine, in any order of sums.
#pragma once

#include <cuda_fp8.h>

#include "mla_common.cuh"

namespace mla {

constexpr int kBlock8 = MLA_SCALE_BLOCK;             // 16
constexpr int kBlocks8 = kPage / kBlock8;            // 4 blocks per page
constexpr int kPage8 = MLA_PAGE8_BYTES;              // 36,864
constexpr int kPage8Rope = kPage * kLora;            // offset of the rotary part in a page

// The query of a request as the split-KV kernel's B operand: e4m3 rows n = head (hi) and 16 + head (lo),
// value = (hi + lo / 16) * q_scale, laid out as it lies in shared memory: [4 column blocks][32 rows]
// [128 B] with the 128-byte swizzle, then the rotary part [32 rows][64 B] with the 64-byte swizzle.
constexpr int kQ8N = 2 * kHeads;
constexpr int kQ8C = kQ8N * kLora, kQ8R = kQ8N * kRope;  // 16,384 and 2,048 bytes
static_assert(kQ8C + kQ8R == kQRows * kRow * 2, "the image takes the bf16 query's place in the workspace");
__device__ __forceinline__ int q8_offset(int n, int col) {  // latent column
    return (col >> 7) * (kQ8N * 128) + n * 128 + ((((col & 127) >> 4) ^ (n & 7)) << 4) + (col & 15);
}
__device__ __forceinline__ int q8_offset_rope(int n, int col) {
    return kQ8C + n * kRope + (((col >> 4) ^ ((n >> 1) & 3)) << 4) + (col & 15);
}

// The smallest e >= MLA_SCALE_MIN_EXP with amax <= 448 * 2^e = 1.75 * 2^(8 + e), amax finite.
__device__ __forceinline__ int scale_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u);
    return max(e, MLA_SCALE_MIN_EXP);
}

// 2^k as f32; 0 below the normal range (k <= 127).
__device__ __forceinline__ float pow2i(int k) { return k < -126 ? 0.f : __uint_as_float((uint32_t)(k + 127) << 23); }

// |x| for a block's largest magnitude: infinities and NaN do not set a scale.
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.f;
}
// What is encoded in place of x: e4m3 has no infinity, and saturating one would make it a number.
__device__ __forceinline__ float nan_if_inf(float x) { return fabsf(x) <= 3.402823466e38f ? x : __int_as_float(0x7FC00000); }

// Two values as e4m3 (nearest, ties to even), lo in the low byte. |values| <= 448 or NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)v, __NV_E4M3);
    return __half22float2(__half2(h));
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}

// Two values, |values| <= 448 or NaN, as a pair of e4m3 values each: x = hi + lo / 16 to about 2^-9 of
// x for |x| >= 2^-6 (its own rounding to f16 on the way is 2^-12), to 2^-14 for smaller ones. hi and lo hold
// both values, the first in the low byte.
__device__ __forceinline__ void e4m3_pairs(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    hi = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(h), __NV_SATFINITE, __NV_E4M3);
    const __half2 back(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)hi, __NV_E4M3));
    const __half2 r = __hmul2(__hsub2(h, back), __float2half2_rn(16.f));  // exact
    lo = __nv_cvt_halfraw2_to_fp8x2(static_cast<__half2_raw>(r), __NV_SATFINITE, __NV_E4M3);
}

// Four stored values, held anew under a scale larger by 1 / f (f a power of two <= 1).
__device__ __forceinline__ uint32_t rescale_e4m3x4(uint32_t v, float f) {
    const float2 a = from_e4m3x2(v & 0xFFFFu), b = from_e4m3x2(v >> 16);
    return e4m3x4(a.x * f, a.y * f, b.x * f, b.y * f);
}
__device__ __forceinline__ uint4 rescale_e4m3x16(uint4 v, float f) {
    return make_uint4(rescale_e4m3x4(v.x, f), rescale_e4m3x4(v.y, f), rescale_e4m3x4(v.z, f), rescale_e4m3x4(v.w, f));
}

// The first n rows of block blk of a page, held anew under scales larger by 1 / f_c and
// 1 / f_r (1: left alone); thread t of nt.
__device__ __forceinline__ void rescale_rows(uint8_t* page, int blk, int n, float f_c, float f_r, int t, int nt) {
    if (f_c != 1.f) {
        uint4* c = reinterpret_cast<uint4*>(page + blk * kBlock8 * kLora);
        for (int i = t; i < n * (kLora / 16); i += nt) c[i] = rescale_e4m3x16(c[i], f_c);
    }
    if (f_r != 1.f) {
        uint4* r = reinterpret_cast<uint4*>(page + kPage8Rope + blk * kBlock8 * kRope);
        for (int i = t; i < n * (kRope / 16); i += nt) r[i] = rescale_e4m3x16(r[i], f_r);
    }
}

// One lane's share of a bf16 row: 16 latent columns 16 lane .., rotary columns lane and 32 + lane.
struct RowShare {
    alignas(16) __nv_bfloat162 c[8];  // loaded 16 bytes at a time
    __nv_bfloat16 lo, hi;
};

// The largest finite magnitudes of a share, into ac and ar; true if it holds an infinity.
__device__ __forceinline__ bool share_amax(const RowShare& x, float& ac, float& ar) {
    __nv_bfloat162 m = __habs2(x.c[0]);
#pragma unroll
    for (int k = 1; k < 8; ++k) m = __hmax2(m, __habs2(x.c[k]));  // a NaN loses to a number
    float c = fmaxf(__low2float(m), __high2float(m));
    float r = fmaxf(fabsf(__bfloat162float(x.lo)), fabsf(__bfloat162float(x.hi)));
    bool inf = false;
    if (!(fmaxf(c, r) <= 3.4e38f)) {  // an infinity, or nothing but NaN: look at every value
        c = 0.f;
        r = fmaxf(finite_abs(__bfloat162float(x.lo)), finite_abs(__bfloat162float(x.hi)));
#pragma unroll
        for (int k = 0; k < 8; ++k) c = fmaxf(c, fmaxf(finite_abs(__low2float(x.c[k])), finite_abs(__high2float(x.c[k]))));
        inf = true;
    }
    ac = fmaxf(ac, c);
    ar = fmaxf(ar, r);
    return inf;
}

// A share under the exponents e_c, e_r into slot `slot` of a page. inf: it may hold an infinity.
// The scaling is a bf16 multiply of both halves: a power of two in bf16's range, so it is exact, but
// for results below 2^-126, which e4m3 rounds to zero anyway.
__device__ __forceinline__ void store_share(uint8_t* page, int slot, const RowShare& x, bool inf, int e_c, int e_r,
                                            int lane) {
    const __nv_bfloat162 f = __float2bfloat162_rn(pow2i(-e_c));
    const float g = pow2i(-e_r);
    uint32_t w[4];
    float lo = __bfloat162float(x.lo), hi = __bfloat162float(x.hi);
    if (!inf) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const __nv_bfloat162 a = __hmul2(x.c[2 * k], f), b = __hmul2(x.c[2 * k + 1], f);
            w[k] = e4m3x4(__low2float(a), __high2float(a), __low2float(b), __high2float(b));
        }
    } else {
        const float s = pow2i(-e_c);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w[k] = e4m3x4(nan_if_inf(__low2float(x.c[2 * k])) * s, nan_if_inf(__high2float(x.c[2 * k])) * s,
                          nan_if_inf(__low2float(x.c[2 * k + 1])) * s, nan_if_inf(__high2float(x.c[2 * k + 1])) * s);
        lo = nan_if_inf(lo);
        hi = nan_if_inf(hi);
    }
    *reinterpret_cast<uint4*>(page + slot * kLora + 16 * lane) = make_uint4(w[0], w[1], w[2], w[3]);
    const uint32_t r = e4m3x2(lo * g, hi * g);
    uint8_t* rope = page + kPage8Rope + slot * kRope + lane;
    rope[0] = (uint8_t)r;
    rope[32] = (uint8_t)(r >> 8);
}

// One warp appends a row to its slot of a page: the block's scales (exps = its pair of
// exponents) grow if the row needs it, and the block's earlier rows with them.
__device__ __forceinline__ void append_row8(uint8_t* page, int8_t* page_exps, int slot, const RowShare& x, int lane) {
    float ac = 0.f, ar = 0.f;
    const bool inf = share_amax(x, ac, ar);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        ac = fmaxf(ac, __shfl_xor_sync(0xffffffffu, ac, o));
        ar = fmaxf(ar, __shfl_xor_sync(0xffffffffu, ar, o));
    }
    int e_c = scale_exponent(ac), e_r = scale_exponent(ar);
    const int blk = slot / kBlock8, before = slot % kBlock8;
    char2* exps = reinterpret_cast<char2*>(page_exps) + blk;
    if (before) {
        const char2 old = *exps;
        e_c = max(e_c, (int)old.x);
        e_r = max(e_r, (int)old.y);
        rescale_rows(page, blk, before, pow2i((int)old.x - e_c), pow2i((int)old.y - e_r), lane, 32);
        __syncwarp();  // every lane has read the exponents
    }
    if (lane == 0) *exps = make_char2((signed char)e_c, (signed char)e_r);
    store_share(page, slot, x, inf, e_c, e_r, lane);
}

}  // namespace mla
