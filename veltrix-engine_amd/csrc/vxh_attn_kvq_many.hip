// Attention over the paged 8-bit KV cache for requests with many queries
// (prompt chunks, large verify batches).
//
// Bound by the matrix and vector units and LDS, about equally: by count, in a
// 32-token step of 16 wavefronts with heads of 128, a CU's LDS reads and writes
// take 2560 clocks, a SIMD's MFMAs 2048 and its other instructions about 2240
// (counters: the vector unit busy 68% of the time).  A workgroup takes a tile of 64 queries
// of one kv head: SK streams of four wavefronts, 16 queries a wavefront, stream
// i on every SK-th group from the i-th.  A stream converts 32 tokens of K and V
// once, and they stand in LDS as MFMA operands (double-buffered) that its four
// wavefronts read.  The values' scale goes into the probabilities, as a factor
// of the largest one met (U), so that P V sums up inside the MFMAs.
// Measured: 2048 rows from an empty cache, 32/32 heads of 128, 83 us for 34.4
// GFLOP of products in two parts (2 x 34.4 / 83 us = 830 TFLOP/s; a large fp16
// product reaches 1079); two chunks of 500 rows over 2036 positions, 32/4 heads
// of 64, 43 us.
#include "vxh_attn_kvq.h"

#define AM_QT 64                 // queries of a tile
#define AM_P 2048.0f             // what a probability is times in the matrix products
#define AM_SLACK 4.0f            // powers of two a score may pass the reference by

struct vx_kvq_unit {
    vx_kvq_seq s;
    int b, kvh, tile, hi, groups;
};

// Unit u of the list: requests in order, each one's tiles from the last (the
// longest) to the first, kv heads fastest.  False past the end.
__device__ __forceinline__ bool vx_kvq_find_unit(const vx_kvq_batch &a, int u, int *s_found, vx_kvq_unit *un)
{
    const int tid = threadIdx.x;
    int b = 0, rel = u;
    if (a.B > 1) {
        // a wavefront walks the requests, 64 at a time
        if (tid == 0) s_found[0] = -1;
        __syncthreads();
        if (tid < 64) {
            int64_t before = 0;
            for (int c = 0; c < a.B; c += 64) {
                int64_t w = 0;
                if (c + tid < a.B) {
                    const vx_kvq_seq r = vx_kvq_request<true>(a, c + tid);
                    w = (int64_t)((r.nq + AM_QT - 1) / AM_QT) * a.n_kv;
                }
                int64_t at = w;
                for (int o = 1; o < 64; o <<= 1) {
                    const int64_t v = __shfl_up(at, o);
                    if (tid >= o) at += v;
                }
                at += before;
                if (u >= at - w && u < at) {
                    s_found[0] = c + tid;
                    s_found[1] = (int)(u - (at - w));
                }
                before = __shfl(at, 63);
                if (before > u) break;
            }
        }
        __syncthreads();
        b = __builtin_amdgcn_readfirstlane(s_found[0]);
        rel = __builtin_amdgcn_readfirstlane(s_found[1]);
        if (b < 0) return false;
    }
    const vx_kvq_seq s = vx_kvq_request<true>(a, b);
    const int T = (s.nq + AM_QT - 1) / AM_QT;
    if (rel >= (int64_t)T * a.n_kv) return false;
    un->s = s;
    un->b = b;
    un->kvh = rel % a.n_kv;
    un->tile = T - 1 - rel / a.n_kv;
    un->hi = vx_kvq_limit(a, s, min(un->tile * AM_QT + AM_QT - 1, s.nq - 1));
    un->groups = max((un->hi + 31) >> 5, 1);
    return true;
}

// Pages and scales of the groups g0, g0 + stride, .. below g1 of a request and
// kv head: lane i holds the i-th's, so that a loop over them waits for the page
// table and the scales once in 64 groups.  Page -1: none.
struct vx_kvq_pages {
    int page;
    float ks, vs;
};

__device__ __forceinline__ vx_kvq_pages vx_kvq_lookup(const vx_kvq_call &c, int b, int kvh, int g0, int stride, int g1)
{
    const int g = g0 + (int)(threadIdx.x & 63) * stride;
    vx_kvq_pages p;
    p.page = g < g1 ? c.table[(size_t)b * c.ld_table + (g >> (c.shift - 5))] : -1;
    if ((unsigned)p.page >= (unsigned)c.n_pages) p.page = -1;
    const size_t hp = (size_t)max(p.page, 0) * c.a.n_kv + kvh;
    p.ks = p.page < 0 ? 0.0f : c.ks[hp];
    p.vs = p.page < 0 ? 0.0f : c.vs[hp];
    if (p.vs < 0x1p-120f) p.vs = 0.0f;            // (its reciprocal must be a number)
    return p;
}

__device__ __forceinline__ float vx_lane(float v, int i)
{
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
}

template <int TYPE, int HD, int SK>
__global__ __launch_bounds__(256 * SK, 4) void vx_attention_kvq_many_kernel(vx_kvq_call c)
{
    constexpr int QT = AM_QT, NJ = HD / 32, ND = HD / 16, PS = HD + 4, NC = (2 * NJ + 3) / 4;
    // a stream's groups, [buffer][keys by 32 dims, values by 32 dims][MFMA][lane];
    // after the last one the streams' results, [query][values, maximum, sum]
    __shared__ union {
        uint4 kv[SK][2][2 * NJ][2][64];
        float o[SK - 1][QT][PS];
    } sh;
    __shared__ int s_found[2];
    const vx_kvq_batch &a = c.a;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3, strm = __builtin_amdgcn_readfirstlane(tid >> 8);
    vx_kvq_unit un;
    if (!vx_kvq_find_unit(a, blockIdx.x, s_found, &un)) return;
    const vx_kvq_seq s = un.s;
    const int kvh = un.kvh, g_end = un.groups;

    // this wavefront's share of a group: 1 KiB chunks of 16 codes a lane
    uint4 st[NC];
    vx_kvq_pages pages = vx_kvq_lookup(c, un.b, kvh, strm, SK, g_end);
    int page2;                                    // of the group loaded last
    float ks2, vs2;
    auto load = [&](int g) {
        const int at = (g - strm) / SK & 63;
        if (at == 0 && g > strm) pages = vx_kvq_lookup(c, un.b, kvh, g, SK, g_end);
        page2 = __builtin_amdgcn_readlane(pages.page, at);
        ks2 = vx_lane(pages.ks, at);
        vs2 = vx_lane(pages.vs, at);
        const size_t base = ((((size_t)max(page2, 0) * a.n_kv + kvh) << c.shift) +
                             (size_t)(g & ((1 << (c.shift - 5)) - 1)) * 32) * HD + lane * 16;
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const int ch = wave + 4 * i;
            if (2 * NJ % 4 == 0 || ch < 2 * NJ)
                st[i] = *(const uint4 *)((ch < NJ ? c.kc : c.vc) + base + 1024 * (ch < NJ ? ch : ch - NJ));
        }
    };
    auto store = [&](int buf, int g, bool none) {
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const int ch = wave + 4 * i;
            if (2 * NJ % 4 == 0 || ch < 2 * NJ) {
                if (TYPE == VXH_KVQ_E4M3 && ch >= NJ && (none || 32 * g + 32 > un.hi))
                    st[i] = vx_kvq_mask_codes(st[i], 32 * g + 4 * g4, none ? 0 : un.hi);
                sh.kv[strm][buf][ch][0][lane] = __builtin_bit_cast(uint4, vx_kvq_half8<TYPE>(st[i].x, st[i].y));
                sh.kv[strm][buf][ch][1][lane] = __builtin_bit_cast(uint4, vx_kvq_half8<TYPE>(st[i].z, st[i].w));
            }
        }
    };
    load(strm);

    // queries, in registers
    const int w0 = un.tile * QT + 16 * wave, qi = w0 + n;
    const bool ok = qi < s.nq;
    const size_t row = s.row + (ok ? qi / a.G : 0);
    const int col = (kvh * a.G + (ok ? qi % a.G : 0)) * HD;
    // the wavefront's own range: its queries all read lo positions, none passes hi
    const int lo = vx_kvq_limit(a, s, min(w0, s.nq - 1));
    const int hi = w0 < s.nq ? vx_kvq_limit(a, s, min(w0 + 15, s.nq - 1)) : 0;
    vx_half8 qh[NJ], ql[NJ];
    const int lim = ok ? vx_kvq_limit(a, s, qi) : un.hi;      // (a query that is none sees what the others see)
    float qs;
    {
        vx_kvq_query<NJ> x;
        x.load(c.q + row * c.ldq + col + 8 * g4);
        const float f = x.scale(&qs);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            vx_half2 h[4], w[4];
            x.parts(j, f, h, w);
            qh[j] = vx_join8(h);
            ql[j] = vx_join8(w);
        }
    }

    vx_f32x4 O[ND];
    float m = -INFINITY, l = 0.0f, U = 0.0f, inv_U = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; d++) O[d] = vx_f32x4{};
    int page = page2;
    float ksc = ks2, vsc = vs2;
    store(0, strm, page < 0);
    if (strm + SK < g_end) load(strm + SK);
    __syncthreads();
    for (int g = strm, buf = 0; g < g_end + strm; g += SK, buf ^= 1) {
        // (as often in every stream: the first one's count)
        const bool none = page < 0, live = 32 * g < hi && g < g_end;
        const int page1 = page2;
        const float ks1 = ks2, vs1 = vs2;
        vx_f32x4 S[2];
        if (live) {
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const vx_half8 k0 = __builtin_bit_cast(vx_half8, sh.kv[strm][buf][j][0][lane]);
                const vx_half8 k1 = __builtin_bit_cast(vx_half8, sh.kv[strm][buf][j][1][lane]);
                S[0] = vx_mfma(k0, ql[j], j ? S[0] : vx_f32x4{});
                S[1] = vx_mfma(k1, ql[j], j ? S[1] : vx_f32x4{});
                S[0] = vx_mfma(k0, qh[j], S[0]);
                S[1] = vx_mfma(k1, qh[j], S[1]);
            }
        }
        if (g + SK < g_end) {
            store(buf ^ 1, g + SK, page1 < 0);
            if (g + 2 * SK < g_end) load(g + 2 * SK);
        }
        if (live) {
            // the scale's factor: in [2^-10, 1] of U, or U follows (below 2^-60 of
            // it a page's values count for nothing next to the others)
            float r = vsc * inv_U, fo = 1.0f;
            if (vsc > U || (r < 0x1p-10f && r > 0x1p-60f)) {
                fo = U / vsc;
                U = vsc;
                inv_U = 1.0f / vsc;
                r = vsc * inv_U;
            }
            if (32 * g + 32 > lo || none) vx_kvq_mask(S, 32 * g + 4 * g4, none ? 0 : lim);
            float cs = fmaxf(qs * ksc, 1e-37f);               // -inf must not meet a zero
            // the reference follows the maximum when that is 2^4 past it
            const float nm = vx_max_x32(vx_max_x16(vx_max8(S))) * cs;
            if (__any(nm > m + AM_SLACK) || fo != 1.0f) {
                const float to = fmaxf(m, nm), f = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.0f : to));
                l *= f;
#pragma unroll
                for (int d = 0; d < ND; d++) O[d] *= f * fo;
                m = to;
            }
            // probabilities times 2^11 (AM_P): their low parts stay normal numbers
            const float ref = m == -INFINITY ? 0.0f : m;
            float sub = 11.0f - ref;
            if (__any(fabsf(ref) > VX_KVQ_FAR)) {
                vx_kvq_far(S, cs, ref);
                cs = 1.0f;
                sub = 11.0f;
            }
            vx_half2 h[4], w[4];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(S[e >> 2][e & 3], cs, sub));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(S[e >> 2][(e & 3) + 1], cs, sub));
                l += p0 + p1;
                vx_split(p0 * r, p1 * r, &h[e / 2], &w[e / 2]);
            }
            const vx_half8 ph = vx_join8(h), pl = vx_join8(w);
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const vx_half8 v0 = __builtin_bit_cast(vx_half8, sh.kv[strm][buf][NJ + j][0][lane]);
                const vx_half8 v1 = __builtin_bit_cast(vx_half8, sh.kv[strm][buf][NJ + j][1][lane]);
                O[2 * j] = vx_mfma(v0, pl, O[2 * j]);
                O[2 * j + 1] = vx_mfma(v1, pl, O[2 * j + 1]);
                O[2 * j] = vx_mfma(v0, ph, O[2 * j]);
                O[2 * j + 1] = vx_mfma(v1, ph, O[2 * j + 1]);
            }
        }
        __syncthreads();
        page = page1;
        ksc = ks1;
        vsc = vs1;
    }
    l = vx_sum_x32(vx_sum_x16(l));
#pragma unroll
    for (int d = 0; d < ND; d++) O[d] *= U * (1.0f / AM_P);
    if (strm > 0) {
        float *so = sh.o[strm - 1][16 * wave + n];
#pragma unroll
        for (int d = 0; d < ND; d++) *(vx_f32x4 *)(so + 16 * d + 4 * g4) = O[d];
        if (g4 == 0) *(float2 *)(so + HD) = make_float2(m, l);
    }
    __syncthreads();
    if (strm > 0) return;
    const int qt = 16 * wave + n;
    // the other streams' results join the first's
    float nm = m;
#pragma unroll
    for (int t = 0; t < SK - 1; t++) nm = fmaxf(nm, sh.o[t][qt][HD]);
    const float ref = nm == -INFINITY ? 0.0f : nm, f0 = __builtin_amdgcn_exp2f(m - ref);
    m = nm;
    l *= f0;
#pragma unroll
    for (int d = 0; d < ND; d++) O[d] *= f0;
#pragma unroll
    for (int t = 0; t < SK - 1; t++) {
        const float *so = sh.o[t][qt];
        const float f = __builtin_amdgcn_exp2f(so[HD] - ref);
        l = fmaf(so[HD + 1], f, l);
#pragma unroll
        for (int d = 0; d < ND; d++) O[d] += *(const vx_f32x4 *)(so + 16 * d + 4 * g4) * f;
    }
    if (!ok) return;
    const float inv = l != 0.0f ? AM_P / l : 0.0f;
    float *o = c.out + row * c.ld_out + col + 4 * g4;
#pragma unroll
    for (int d = 0; d < ND; d++) *(vx_f32x4 *)(o + 16 * d) = O[d] * inv;
}

// Units are tiles; with few of them a workgroup walks a tile in four streams
// (256 units of 512 rows over 2000 positions, 32/4 heads of 64: 42 us in two
// streams, 34 in four; 1024 units of a 2048-row prompt, 32/32 heads of 128: 97
// and 120).
static int64_t vx_kvq_many_units(const vx_kvq_batch &a)
{
    return ((int64_t)a.max_rows * a.G + AM_QT - 1) / AM_QT * a.n_kv;
}

// Workgroups: a tile more per request with rows, for its last, partly filled one.
static int64_t vx_kvq_many_grid(const vx_kvq_batch &a)
{
    const int with_rows = a.B < a.max_rows ? a.B : a.max_rows;
    return vx_kvq_many_units(a) + (a.B > 1 ? (int64_t)with_rows * a.n_kv : 0);
}

// From 192 tiles on this kernel fills the card and beats the other one (200 tiles
// of 1600 rows over 1900, 8/2 heads of 96: 36 us against 47; 192 of 768 rows,
// 16/16 of 128: 23 against 30; 192 of 130 rows over 4130, 64/64 of 64: 52 against
// 55); below, the other spreads the tiles' lengths too (128 tiles of 70 rows over
// 3070, 64/64 of 64: 31 against 40; 96 of 192 over 2192, 32/32 of 128: 39
// against 45).  A launch holds less than 2^32 threads: 2^22 tiles.
bool vx_kvq_many_wanted(const vx_kvq_batch &a, int max_seq_rows)
{
    return (int64_t)max_seq_rows * a.G > AM_QT && vx_kvq_many_units(a) >= 192 && vx_kvq_many_grid(a) <= 1 << 22;
}

int vx_kvq_many(const vx_kvq_call &c, int type, int head_dim, hipStream_t s)
{
    const int64_t units = vx_kvq_many_units(c.a);
    const unsigned grid = (unsigned)vx_kvq_many_grid(c.a);
#define VX_CALL(T, HD)                                                                                                \
    if (units < 384) vx_attention_kvq_many_kernel<T, HD, 4><<<grid, 1024, 0, s>>>(c);                                 \
    else vx_attention_kvq_many_kernel<T, HD, 2><<<grid, 512, 0, s>>>(c);
#define VX_HD(T)                                                                                                      \
    switch (head_dim) {                                                                                               \
    case 32: VX_CALL(T, 32) break;                                                                                    \
    case 64: VX_CALL(T, 64) break;                                                                                    \
    case 96: VX_CALL(T, 96) break;                                                                                    \
    default: VX_CALL(T, 128)                                                                                          \
    }
    if (type == VXH_KVQ_INT8) {
        VX_HD(VXH_KVQ_INT8)
    } else {
        VX_HD(VXH_KVQ_E4M3)
    }
#undef VX_HD
#undef VX_CALL
    VXH_LAUNCHED();
    return VXH_OK;
}
