// Codes of the paged 8-bit KV cache: layout and conversions shared by the
// kernels that write, read and attend it.
#pragma once

#include "vxh_internal.h"

// Byte of (token, dim) inside one page and head of the keys: 32 tokens x 32
// dims are 1 KiB, lane 16 g + n of which holds dims 8g..8g+7 of token n, then
// of token n + 16 -- the A operands of two 16x16x32 MFMAs in 16 bytes.
__device__ __forceinline__ int vx_kvq_k_byte(int t, int d, int hd)
{
    return (t >> 5) * 32 * hd + (d >> 5) * 1024 + (((d >> 3) & 3) * 16 + (t & 15)) * 16 + ((t >> 4) & 1) * 8 + (d & 7);
}

// The same of the values: lane 16 g + n holds, of dim n and then of dim
// n + 16, tokens 4g..4g+3 and 16+4g..16+4g+3 -- the order in which a score
// MFMA leaves the probabilities in that lane's registers.
__device__ __forceinline__ int vx_kvq_v_byte(int t, int d, int hd)
{
    return (t >> 5) * 32 * hd + (d >> 5) * 1024 + (((t >> 2) & 3) * 16 + (d & 15)) * 16 + ((d >> 4) & 1) * 8 +
           ((t >> 4) & 1) * 4 + (t & 3);
}

// Value of one code: int8 is stored with an offset of 128.
template <int TYPE>
__device__ __forceinline__ float vx_kvq_value(uint32_t byte)
{
    if (TYPE == VXH_KVQ_INT8) return (float)((int)byte - 128);
    return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
}

// y (the fp32 rounding of a quotient) moved to the neighbour with an odd last
// bit when the quotient is not y itself (above: it lies above y): a later
// rounding to fewer bits then rounds the quotient, not y.
__device__ __forceinline__ float vx_round_odd(float y, bool above, bool exact)
{
    const int b = __float_as_int(y);
    if (exact || (b & 1) || y == 0.0f) return y;
    return __int_as_float(above == (y > 0.0f) ? b + 1 : b - 1);
}

// Code of x at the scale s > 0, inv = 1/s: the exact quotient x/s rounded to
// the nearest code, ties to even, saturating; NaN becomes zero.
template <int TYPE>
__device__ __forceinline__ uint32_t vx_kvq_code(float x, float s, float inv)
{
    if (TYPE == VXH_KVQ_INT8) {
        // t may be one off where x * inv lies next to a half; the remainder
        // x - t s is exact (a multiple of s's or x's last bit below 2^24 of it)
        float t = rintf(x * inv);
        t = fminf(fmaxf(t, -127.0f), 127.0f);            // NaN: -127, zeroed below
        const float r = fmaf(-t, s, x), h = 0.5f * s;
        const bool odd = (int)t & 1;
        if (r > h || (r == h && odd)) t += 1.0f;
        if (r < -h || (r == -h && odd)) t -= 1.0f;
        t = fminf(fmaxf(t, -127.0f), 127.0f);
        return x != x ? 128u : (uint32_t)((int)t + 128);
    }
    float y = x / s;
    const float r = fmaf(-y, s, x);
    y = fabsf(y) < 448.0f ? vx_round_odd(y, r > 0.0f, r == 0.0f) : copysignf(448.0f, y);
    return x != x ? 0u : (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, 0.0f, 0, false) & 0xFFu;
}

// The same from a product with inv for finite x of |x| <= top s: the low byte,
// and *sure false where that product lies so near a border between two codes
// (or so near zero, e4m3) that only vx_kvq_code can tell.
template <int TYPE>
__device__ __forceinline__ uint32_t vx_kvq_code_fast(float x, float s, float inv, bool *sure)
{
    const float y = x * inv;
    if (TYPE == VXH_KVQ_INT8) {
        const float t = rintf(y);
        *sure &= fabsf(y - t) < 0.4999f;
        return (uint32_t)((int)t + 128);
    }
    // an e4m3 code has 3 of 23 mantissa bits: a border is a half of the other 20
    const int b = __float_as_int(y);
    *sure &= fabsf(y) >= 0x1p-6f && abs((b & 0xFFFFF) - 0x80000) > 4;
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, 0.0f, 0, false) & 0xFFu;
}

// Code of a stored code's value v (at the scale s0 <= s) at the scale s.
template <int TYPE>
__device__ __forceinline__ uint32_t vx_kvq_recode(float v, float s0, float s)
{
    const double y = (double)v * (double)s0 / (double)s;   // far more bits than a tie needs
    if (TYPE == VXH_KVQ_INT8) {
        const double t = fmin(fmax(rint(y), -127.0), 127.0);
        return (uint32_t)((int)t + 128);
    }
    float f = (float)y;
    f = vx_round_odd(f, y > (double)f, y == (double)f);
    f = fminf(fmaxf(f, -448.0f), 448.0f);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f, 0.0f, 0, false) & 0xFFu;
}

// Host-side checks of a cache handle shared by every entry point.
const char *vx_kvq_bad(const vxh_kvq *c);
