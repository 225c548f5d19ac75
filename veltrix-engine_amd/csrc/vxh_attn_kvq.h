// Device code shared by the kernels that attend the paged 8-bit KV cache.
#pragma once

#include "vxh_kvq.h"

typedef float vx_f32x4 __attribute__((ext_vector_type(4)));

struct vx_kvq_batch {
    const int *row0, *len;
    int B, max_rows, n_kv, G, cap, limit;    // limit: tokens a table row can name
    int few;                                 // queries per kv head up to which a request is the decode kernel's
};

struct vx_kvq_seq {
    int row, m, n, end, nq;      // first row, rows, tokens, tokens any row reads, queries per kv head
};

// Request b as one of the kernels sees it: without rows when it is the other's.
template <bool MANY>
__device__ __forceinline__ vx_kvq_seq vx_kvq_request(const vx_kvq_batch &a, int b)
{
    vx_kvq_seq s;
    s.row = min(max(a.row0[b], 0), a.max_rows);
    s.m = max(min(a.row0[b + 1], a.max_rows) - s.row, 0);
    s.n = min(max(a.len[b], 0), a.limit);
    s.end = a.cap > 0 ? min(s.n, a.cap) : s.n;
    if (((int64_t)s.m * a.G > a.few) != MANY) s.m = 0;
    s.nq = s.m * a.G;
    return s;
}

// 32-token groups of a request (at least one: a tile that reads nothing still
// writes its zeros).
__device__ __forceinline__ int vx_kvq_groups(const vx_kvq_seq &s) { return max((s.end + 31) >> 5, 1); }

// Positions that query qi of a request reads.
__device__ __forceinline__ int vx_kvq_limit(const vx_kvq_batch &a, const vx_kvq_seq &s, int qi)
{
    const int t = s.n - s.m + qi / a.G + 1;
    return a.cap > 0 ? min(t, a.cap) : t;
}

// 8 codes to fp16, exactly.
template <int TYPE>
__device__ __forceinline__ vx_half8 vx_kvq_half8(uint32_t a, uint32_t b)
{
    vx_half2 h[4];
    if (TYPE == VXH_KVQ_INT8) {
        // 0x64xx is 1024 + xx
        const vx_half2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        h[0] = __builtin_bit_cast(vx_half2, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) + off;
        h[1] = __builtin_bit_cast(vx_half2, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) + off;
        h[2] = __builtin_bit_cast(vx_half2, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) + off;
        h[3] = __builtin_bit_cast(vx_half2, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) + off;
    } else {
        h[0] = __builtin_bit_cast(vx_half2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false));
        h[1] = __builtin_bit_cast(vx_half2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true));
        h[2] = __builtin_bit_cast(vx_half2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false));
        h[3] = __builtin_bit_cast(vx_half2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true));
    }
    return vx_half8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// x = hi + lo to 22 bits (both truncated, so the two add up with one sign).
__device__ __forceinline__ void vx_split(float a, float b, vx_half2 *hi, vx_half2 *lo)
{
    *hi = __builtin_bit_cast(vx_half2, __builtin_amdgcn_cvt_pkrtz(a, b));
    *lo = __builtin_bit_cast(vx_half2, __builtin_amdgcn_cvt_pkrtz(a - (float)(*hi)[0], b - (float)(*hi)[1]));
}

// MFMA sources stay live past the instruction: a destination in VGPRs that
// overlaps them gives wrong values.
#define AK_KEEP(D, A, B) asm("" : "+v"(D) : "v"(A), "v"(B))

__device__ __forceinline__ vx_half8 vx_join8(const vx_half2 (&h)[4])
{
    return vx_half8{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// One query's dims 32 j + 8 g4 .. + 7 in every lane (query n = lane & 15, g4 =
// lane / 16).
template <int NJ>
struct vx_kvq_query {
    float4 x0[NJ], x1[NJ];
    __device__ __forceinline__ void load(const float *p)
    {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            x0[j] = *(const float4 *)(p + 32 * j);
            x1[j] = *(const float4 *)(p + 32 * j + 4);
        }
    }
    // The power of two that takes the row below 2^14 (so that the low parts stay
    // normal numbers for long), and what a product of the parts is times to be a
    // score in powers of two.
    __device__ __forceinline__ float scale(float *back) const
    {
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x0[j].x), fabsf(x0[j].y)), fmaxf(fabsf(x0[j].z), fabsf(x0[j].w))));
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x1[j].x), fabsf(x1[j].y)), fmaxf(fabsf(x1[j].z), fabsf(x1[j].w))));
        }
        amax = vx_max_x32(vx_max_x16(amax));
        const float f = vx_row_scale(amax, back) * 16384.0f;
        *back *= 1.44269504088896340736f / 16384.0f / sqrtf(32.0f * NJ);
        return f;
    }
    __device__ __forceinline__ void parts(int j, float f, vx_half2 (&h)[4], vx_half2 (&l)[4]) const
    {
        vx_split(x0[j].x * f, x0[j].y * f, &h[0], &l[0]);
        vx_split(x0[j].z * f, x0[j].w * f, &h[1], &l[1]);
        vx_split(x1[j].x * f, x1[j].y * f, &h[2], &l[2]);
        vx_split(x1[j].z * f, x1[j].w * f, &h[3], &l[3]);
    }
};

// Scores of tokens 4g4 + (0..3) + 16 (0..1) behind t0 that lie past lim: -inf.
__device__ __forceinline__ void vx_kvq_mask(vx_f32x4 (&S)[2], int t0, int lim)
{
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (t0 + (e >> 2) * 16 + (e & 3) >= lim) S[e >> 2][e & 3] = -INFINITY;
}

// 16 value codes of a lane, those of tokens past hi zeroed (an e4m3 code that
// no query reads may be NaN, and 0 times it is).
__device__ __forceinline__ uint4 vx_kvq_mask_codes(uint4 v, int t0, int hi)
{
    uint32_t mk[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; e++)
        if (t0 + (e >> 2) * 16 + (e & 3) < hi) mk[e >> 2] |= 0xFFu << (8 * (e & 3));
    return make_uint4(v.x & mk[0], v.y & mk[1], v.z & mk[0], v.w & mk[1]);
}

__device__ __forceinline__ float vx_max8(const vx_f32x4 (&S)[2])
{
    return fmaxf(fmaxf(fmaxf(S[0][0], S[0][1]), fmaxf(S[0][2], S[0][3])),
                 fmaxf(fmaxf(S[1][0], S[1][1]), fmaxf(S[1][2], S[1][3])));
}

// Scores S cs less their reference, each product rounded before the difference:
// past VX_KVQ_FAR a fused one would leave the largest score above its own
// rounded reference by more than a probability's range.
#define VX_KVQ_FAR 0x1p20f
__device__ __forceinline__ void vx_kvq_far(vx_f32x4 (&S)[2], float cs, float ref)
{
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float p = S[e >> 2][e & 3] * cs;
        S[e >> 2][e & 3] = p - ref;
    }
}

__device__ __forceinline__ vx_f32x4 vx_mfma(vx_half8 a, vx_half8 b, vx_f32x4 c)
{
    vx_f32x4 d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    AK_KEEP(d, a, b);
    return d;
}

// What the kernels share of a call.
struct vx_kvq_call {
    vx_kvq_batch a;
    const float *q;
    int ldq;
    const int *table;
    int ld_table;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    int shift, n_pages;              // tokens of a page as a power of two
    float *out;
    int ld_out;
    float *part;
};

// Requests with many queries (vxh_attn_kvq_many.hip): whether a call should give
// them to their own kernel, and that kernel's launch.
bool vx_kvq_many_wanted(const vx_kvq_batch &a, int max_seq_rows);
int vx_kvq_many(const vx_kvq_call &c, int type, int head_dim, hipStream_t s);
