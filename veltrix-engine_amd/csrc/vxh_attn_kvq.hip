// Attention of a ragged batch over the paged 8-bit KV cache: the entry point,
// and the kernel of requests with few queries (decode, verify).
//
// A request's rows and the G = n_heads / n_kv_heads query heads of one kv head
// make up its queries there (query i: row i / G, head i % G), taken 16 to a
// tile.  The work is the list of all (request, kv head, tile, 32-token group);
// every workgroup takes an equal, consecutive piece of it, so lengths may
// differ as they like: a long request spreads over many workgroups, short ones
// share one.  A tile cut by a piece's ends leaves partial results (maximum,
// sum, weighted values) in the workspace, joined in order by the last
// workgroup that contributes to it.
#include "vxh_attn_kvq.h"

#define AK_WAVES 4
#define AK_THREADS (64 * AK_WAVES)
#define AK_WG 512                // pieces: two workgroups per CU (640 and 768 pieces: the same or slower)
#define AK_BEGIN 8               // what beginning and ending a tile costs, in 32-token groups (12: the same)
#define AK_SMALL 8               // tiles of up to this many groups take a wavefront each
#define AK_SNAP 12               // most groups a piece's end moves to a tile's
#define AK_FEW 64                // queries per kv head up to which a request is this kernel's (a tile of the other)
#define AK_P 16384.0f            // what a probability is times in the matrix products
#define AK_JOIN 8                // parts whose loads are in flight together (12, 16: one long request 62-64 us, not 60)
#define AK_BLOCK 16              // parts one workgroup joins

// Items of a tile: its groups, behind AK_BEGIN that stand for what beginning
// and ending a tile cost.
__device__ __forceinline__ int vx_kvq_weight(const vx_kvq_seq &s) { return vx_kvq_groups(s) + AK_BEGIN; }

// Partial results, that workgroups of other XCDs read: past this one's L2
// (coherent over the device).  Offsets in floats: of a slot, and in it.
typedef __amdgpu_buffer_rsrc_t vx_part;
typedef unsigned int vx_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int vx_u32x2 __attribute__((ext_vector_type(2)));
#define AK_DEVICE 16             // the load's or store's scope
__device__ __forceinline__ void vx_part_store(vx_part p, int slot, int at, vx_f32x4 v)
{
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(vx_u32x4, v), p, 4 * at, 4 * slot, AK_DEVICE);
}
__device__ __forceinline__ void vx_part_store2(vx_part p, int slot, int at, float a, float b)
{
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(vx_u32x2, make_float2(a, b)), p, 4 * at, 4 * slot, AK_DEVICE);
}
__device__ __forceinline__ vx_f32x4 vx_part_load(vx_part p, int slot, int at)
{
    return __builtin_bit_cast(vx_f32x4, __builtin_amdgcn_raw_buffer_load_b128(p, 4 * at, 4 * slot, AK_DEVICE));
}
__device__ __forceinline__ float2 vx_part_load2(vx_part p, int slot, int at)
{
    return __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(p, 4 * at, 4 * slot, AK_DEVICE));
}

// Quotient of two counts; 64-bit division only where they need it.
__device__ __forceinline__ int64_t vx_quot(int64_t a, int64_t b)
{
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ int64_t vx_uniform(int64_t v)
{
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// A place in the list: a tile of a request and kv head, and its first item.
struct vx_kvq_found {
    vx_kvq_seq s;
    int b, nth;                  // request; tile of the request, over its kv heads
    int64_t first;
};

// The list, counted anew by every workgroup from the lengths (they are on the
// device only): a thread sums a run of requests, the runs are scanned.
struct vx_kvq_list {
    int64_t at[AK_THREADS + 1];      // items before each thread's run of requests
    vx_kvq_seq one[AK_THREADS];      // a run's last request (its only one up to AK_THREADS requests)
    int64_t wave[AK_WAVES];
    int tiles[AK_WAVES];
    vx_kvq_found found[2];
};

__device__ __forceinline__ void vx_kvq_run(const vx_kvq_batch &a, int *b0, int *b1)
{
    const int E = (a.B + AK_THREADS - 1) / AK_THREADS;
    *b0 = min((int)threadIdx.x * E, a.B);
    *b1 = min(*b0 + E, a.B);
}

// Items of the whole list.
__device__ __forceinline__ int64_t vx_kvq_scan(const vx_kvq_batch &a, vx_kvq_list &list, int64_t *n_tiles)
{
    if (a.B == 1) {
        const vx_kvq_seq s = vx_kvq_request<false>(a, 0);
        *n_tiles = (s.nq + 15) / 16 * a.n_kv;
        return *n_tiles * vx_kvq_weight(s);
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int b0, b1, tiles = 0;
    vx_kvq_run(a, &b0, &b1);
    int64_t mine = 0;
    for (int b = b0; b < b1; b++) {
        const vx_kvq_seq s = vx_kvq_request<false>(a, b);
        const int t = (s.nq + 15) / 16 * a.n_kv;
        mine += (int64_t)t * vx_kvq_weight(s);
        tiles += t;
        list.one[tid] = s;
    }
    int64_t at = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up(at, o);
        const int t = __shfl_up(tiles, o);
        if (lane >= o) {
            at += u;
            tiles += t;
        }
    }
    if (lane == 63) {
        list.wave[wave] = at;
        list.tiles[wave] = tiles;
    }
    __syncthreads();
    int64_t total = 0, nt = 0;
    for (int w = 0; w < AK_WAVES; w++) {
        if (w < wave) at += list.wave[w];
        total += list.wave[w];
        nt += list.tiles[w];
    }
    list.at[tid + 1] = at;
    if (tid == 0) list.at[0] = 0;
    __syncthreads();
    *n_tiles = vx_uniform(nt);
    return vx_uniform(total);
}

// What stands at item x of request b, whose items begin at base.
__device__ __forceinline__ vx_kvq_found vx_kvq_place(const vx_kvq_seq &s, int b, int64_t base, int64_t x)
{
    vx_kvq_found f;
    const int w = vx_kvq_weight(s);
    f.s = s;
    f.b = b;
    f.nth = (int)vx_quot(x - base, w);
    f.first = base + (int64_t)f.nth * w;
    return f;
}

// The thread whose run holds item x writes what is there to list.found[k]
// (of one request, each thread finds it by itself: vx_kvq_get).
__device__ __forceinline__ void vx_kvq_find(const vx_kvq_batch &a, vx_kvq_list &list, int64_t x, int k)
{
    if (a.B == 1) return;
    const int tid = threadIdx.x;
    int64_t base = list.at[tid];
    if (x < base || x >= list.at[tid + 1]) return;
    int b0, b1;
    vx_kvq_run(a, &b0, &b1);
    for (int b = b0; b < b1; b++) {
        const vx_kvq_seq s = b1 - b0 == 1 ? list.one[tid] : vx_kvq_request<false>(a, b);
        const int64_t w = (int64_t)((s.nq + 15) / 16) * vx_kvq_weight(s) * a.n_kv;
        if (x < base + w) {
            list.found[k] = vx_kvq_place(s, b, base, x);
            return;
        }
        base += w;
    }
}

// The same in every thread, behind a barrier, in scalar registers.
__device__ __forceinline__ vx_kvq_found vx_kvq_get(const vx_kvq_batch &a, const vx_kvq_list &list, int64_t x, int k)
{
    if (a.B == 1) return vx_kvq_place(vx_kvq_request<false>(a, 0), 0, 0, x);
    vx_kvq_found f;
    f.s.row = __builtin_amdgcn_readfirstlane(list.found[k].s.row);
    f.s.m = __builtin_amdgcn_readfirstlane(list.found[k].s.m);
    f.s.n = __builtin_amdgcn_readfirstlane(list.found[k].s.n);
    f.s.end = __builtin_amdgcn_readfirstlane(list.found[k].s.end);
    f.s.nq = f.s.m * a.G;
    f.b = __builtin_amdgcn_readfirstlane(list.found[k].b);
    f.nth = __builtin_amdgcn_readfirstlane(list.found[k].nth);
    f.first = vx_uniform(list.found[k].first);
    return f;
}

// Boundary y of two pieces, moved to an end of its tile when that is near.
__device__ __forceinline__ int64_t vx_kvq_snap(const vx_kvq_found &f, int64_t y, int snap)
{
    const int64_t end = f.first + vx_kvq_weight(f.s);
    return y - f.first <= snap + AK_BEGIN ? f.first : end - y <= snap ? end : y;
}

// Counts the workgroup in after its partial results have reached memory;
// true for the last of n, which sets the counter back.
__device__ __forceinline__ bool vx_arrive(unsigned *counter, int n, unsigned *s_last)
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        *s_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (*s_last == (unsigned)(n - 1)) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *s_last == (unsigned)(n - 1);
}

// Parts i0..i1-1 of nv queries joined, in order, AK_JOIN at a time: their
// loads wait for memory once.
template <int HD, typename Slot, typename Out>
__device__ __forceinline__ void vx_kvq_join(vx_part part, Slot slot, int i0, int i1, int nv, Out put)
{
    constexpr int PS = HD + 4;
    for (int u = threadIdx.x; u < nv * (HD / 4); u += AK_THREADS) {
        const int qq = u / (HD / 4), d = u % (HD / 4) * 4;
        float mx = -INFINITY, sum = 0.0f;
        vx_f32x4 o = vx_f32x4{};
        for (int p = i0; p < i1; p += AK_JOIN) {
            float2 ml[AK_JOIN];
            vx_f32x4 v[AK_JOIN];
            float nm = mx;
#pragma unroll
            for (int i = 0; i < AK_JOIN; i++) {
                const int at = slot(min(p + i, i1 - 1)) * (16 * PS);
                ml[i] = vx_part_load2(part, at, qq * PS + HD);
                v[i] = vx_part_load(part, at, qq * PS + d);
            }
#pragma unroll
            for (int i = 0; i < AK_JOIN; i++) {
                if (p + i >= i1) ml[i] = make_float2(-INFINITY, 0.0f);
                nm = fmaxf(nm, ml[i].x);
            }
            const float ref = nm == -INFINITY ? 0.0f : nm, fo = __builtin_amdgcn_exp2f(mx - ref);
            sum *= fo;
            o *= fo;
#pragma unroll
            for (int i = 0; i < AK_JOIN; i++) {
                const float f = __builtin_amdgcn_exp2f(ml[i].x - ref);
                sum = fmaf(ml[i].y, f, sum);
                if (p + i < i1) o += v[i] * f;
            }
            mx = nm;
        }
        put(qq, d, o, mx, sum);
    }
}

// ---------------------------------------------------------------------------
// Bound by the cache's bytes.  Per 32 tokens a wavefront loads K and V straight
// into MFMA operand order (16 bytes a lane), converts them to fp16 exactly and
// multiplies 16 queries kept as two fp16 parts (22 bits).  S = K Q^T leaves a
// lane with tokens 4g..4g+3, 16+4g.. of query n, which is the operand P V
// wants: no exchange between lanes but the maximum's.  The four wavefronts take
// every fourth group and join in LDS; short tiles take a wavefront each.
// Measured (28/4 heads of 128 unless said, kernel times): two requests of 128K
// tokens 52 us for 269 MB (5.1 TB/s), 64 requests of up to 8K 50 us for 261 MB,
// 16 requests of 9 rows at up to 2K with 32/32 heads 37 us for 150 MB: the
// cache's bytes, and 2-3 us a tile begun and ended.  One request: 9 rows over
// 8K 19 us, one row over 2K (32/4 heads of 64) 9 us: the chain of list, first
// loads, groups, partial results, arrival and join.
// ---------------------------------------------------------------------------
template <int TYPE, int HD>
__global__ __launch_bounds__(AK_THREADS, 2) void vx_attention_kvq_kernel(
    vx_kvq_call c, const float *__restrict__ q, const int *__restrict__ table, const uint8_t *__restrict__ kc,
    const uint8_t *__restrict__ vc, const float *__restrict__ ks, const float *__restrict__ vs, float *__restrict__ out,
    float *__restrict__ parts, unsigned *__restrict__ counter)
{
    constexpr int NJ = HD / 32, ND = HD / 16, PS = HD + 4;
    // the queries' operands, [tile][hi, lo][32 dims][lane]; after the last group
    // the wavefronts' results, [wave][query][values, maximum, sum]
    __shared__ union {
        uint4 q[AK_WAVES][2][NJ][64];
        float o[AK_WAVES][16][PS];
    } sh;
    __shared__ vx_kvq_list list;
    __shared__ unsigned s_last;
    const vx_kvq_batch &a = c.a;
    const vx_part part = __builtin_amdgcn_make_buffer_rsrc((void *)parts, (short)0, 2 * AK_WG * 16 * PS * 4, 0x00020000);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g4 = lane >> 4;

    int64_t n_tiles;
    const int64_t total = vx_kvq_scan(a, list, &n_tiles);
    if (total == 0) return;
    // Pieces of whole rounds of the wavefronts.  Where there is too little work for
    // all, 8 groups at least, or what one block of parts a tile takes if that is no
    // more than 20: a long tile's chain of groups costs more than a second level of
    // joins, a short one's less (one request of 9 rows over 8192, 28/4 heads of 128:
    // 19 us in 14 parts a tile, 23 in 22; 3 rows over 13000, 2/2 heads: 16 in 15
    // parts, 13 in 52).
    int64_t piece = vx_quot(total + gridDim.x - 1, gridDim.x);
    int64_t least = vx_quot(total + n_tiles * AK_BLOCK - 1, n_tiles * AK_BLOCK);
    least = least > 20 ? 8 : max(least, (int64_t)8);
    piece = vx_uniform((max(piece, least) + AK_WAVES - 1) / AK_WAVES * AK_WAVES);
    // a boundary this near a tile's end moves there: beginning a tile costs more
    const int snap = __builtin_amdgcn_readfirstlane((int)min(piece / 4, (int64_t)AK_SNAP));
    const int64_t start = (int64_t)blockIdx.x * piece;
    if (start >= total) return;
    vx_kvq_find(a, list, start, 0);
    vx_kvq_find(a, list, start + piece, 1);
    __syncthreads();
    int64_t w_end = total;
    if (start + piece < total) w_end = vx_kvq_snap(vx_kvq_get(a, list, start + piece, 1), start + piece, snap);
    int64_t x = vx_kvq_snap(vx_kvq_get(a, list, start, 0), start, snap);
    if (x != start && x < w_end) {
        __syncthreads();
        vx_kvq_find(a, list, x, 0);
        __syncthreads();
    }

    while (x < w_end) {
        const vx_kvq_found f = vx_kvq_get(a, list, x, 0);
        const vx_kvq_seq s = f.s;
        const int b = f.b, groups = vx_kvq_groups(s), tiles = (s.nq + 15) / 16;
        const int64_t first = f.first;                        // the tile's items: [first, first + weight)
        const int g_begin = max((int)(x - first) - AK_BEGIN, 0);
        const int g_end = (int)min((int64_t)groups, w_end - first - AK_BEGIN);
        // short tiles of one request: a wavefront each
        int few = 1;
        if (groups <= AK_SMALL && g_begin == 0 && g_end == groups)
            few = min(min(AK_WAVES, tiles * a.n_kv - f.nth), (int)vx_quot(w_end - first, groups + AK_BEGIN));
        const int nth = f.nth + (few > 1 ? min(wave, few - 1) : 0), kvh = nth / tiles, tile = nth % tiles;
        const int stride = few > 1 ? 1 : AK_WAVES, qw = few > 1 ? wave : 0;

        const int q0 = 16 * tile;
        // what every query of the tile reads, and what none passes
        const int lo = vx_kvq_limit(a, s, q0), hi = vx_kvq_limit(a, s, min(q0 + 15, s.nq - 1));
        const int qi = q0 + n;
        const bool ok = qi < s.nq;
        const int lim = ok ? vx_kvq_limit(a, s, qi) : hi;             // (a query that is none sees what the others see)
        vx_kvq_query<NJ> x0;
        x0.load(q + (size_t)(s.row + (ok ? qi / a.G : 0)) * c.ldq + (size_t)(kvh * a.G + (ok ? qi % a.G : 0)) * HD + 8 * g4);

        const int pgs = c.shift - 5;                          // groups of a page, as a shift
        const int g_stop = few > 1 && wave >= few ? 0 : min(g_end, (hi + 31) >> 5);
        // the page and the byte of a group's keys and values; page -1: none
        auto locate = [&](int g, size_t *base) {
            int page = table[(size_t)b * c.ld_table + (g >> pgs)];
            if ((unsigned)page >= (unsigned)c.n_pages) page = -1;
            *base = ((((size_t)max(page, 0) * a.n_kv + kvh) << c.shift) + (size_t)(g & ((1 << pgs) - 1)) * 32) * HD;
            return page;
        };
        uint4 kr[NJ], vr[NJ];
        int g = few > 1 ? 0 : g_begin + wave, page = -1;
        if (g < g_stop) {
            size_t base;
            page = locate(g, &base);
#pragma unroll
            for (int j = 0; j < NJ; j++) kr[j] = *(const uint4 *)(kc + base + lane * 16 + 1024 * j);
#pragma unroll
            for (int j = 0; j < NJ; j++) vr[j] = *(const uint4 *)(vc + base + lane * 16 + 1024 * j);
        }

        // the queries' parts: each wavefront stores some dims, or its own tile
        float qs;
        const float qf = x0.scale(&qs);
#pragma unroll
        for (int j = 0; j < NJ; j++) {
            if (few == 1 && j % AK_WAVES != wave) continue;
            vx_half2 h[4], l[4];
            x0.parts(j, qf, h, l);
            sh.q[qw][0][j][lane] = *(const uint4 *)h;
            sh.q[qw][1][j][lane] = *(const uint4 *)l;
        }
        __syncthreads();
        vx_f32x4 O[ND];
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; d++) O[d] = vx_f32x4{};
        for (; g < g_stop; g += stride) {
            // the next group's loads go out as this one's registers come free
            const bool more = g + stride < g_stop;
            size_t base;
            const int next = locate(more ? g + stride : g, &base);
            const uint8_t *kn = kc + base + lane * 16, *vn = vc + base + lane * 16;
            const size_t hp = (size_t)max(page, 0) * a.n_kv + kvh;
            const bool none = page < 0;
            const float ksc = none ? 0.0f : ks[hp], vsc = none ? 0.0f : vs[hp] * (1.0f / AK_P);
            page = next;
            vx_f32x4 S[2], L[2];                              // of the high and of the low parts
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const vx_half8 k0 = vx_kvq_half8<TYPE>(kr[j].x, kr[j].y), k1 = vx_kvq_half8<TYPE>(kr[j].z, kr[j].w);
                kr[j] = *(const uint4 *)(kn + 1024 * j);
                const vx_half8 qh = __builtin_bit_cast(vx_half8, sh.q[qw][0][j][lane]);
                const vx_half8 ql = __builtin_bit_cast(vx_half8, sh.q[qw][1][j][lane]);
                S[0] = vx_mfma(k0, qh, j ? S[0] : vx_f32x4{});
                S[1] = vx_mfma(k1, qh, j ? S[1] : vx_f32x4{});
                L[0] = vx_mfma(k0, ql, j ? L[0] : vx_f32x4{});
                L[1] = vx_mfma(k1, ql, j ? L[1] : vx_f32x4{});
            }
            S[0] += L[0];
            S[1] += L[1];
            const int t0 = 32 * g + 4 * g4;
            if (32 * g + 32 > lo || none) vx_kvq_mask(S, t0, none ? 0 : lim);
            float cs = fmaxf(qs * ksc, 1e-37f);         // -inf must not meet a zero
            const float nm = fmaxf(m, vx_max_x32(vx_max_x16(vx_max8(S))) * cs), ref = nm == -INFINITY ? 0.0f : nm;
            if (__any(nm > m)) {
                const float f = __builtin_amdgcn_exp2f(m - ref);
                l *= f;
#pragma unroll
                for (int d = 0; d < ND; d++) O[d] *= f;
                m = nm;
            }
            // probabilities times 2^14 (AK_P): their low parts stay normal numbers
            float sub = 14.0f - ref;
            if (__any(fabsf(ref) > VX_KVQ_FAR)) {
                vx_kvq_far(S, cs, ref);
                cs = 1.0f;
                sub = 14.0f;
            }
            vx_half2 h[4], w[4];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(S[e >> 2][e & 3], cs, sub));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(S[e >> 2][(e & 3) + 1], cs, sub));
                l += p0 + p1;
                vx_split(p0, p1, &h[e / 2], &w[e / 2]);
            }
            const vx_half8 ph = vx_join8(h), pl = vx_join8(w);
            if (TYPE == VXH_KVQ_E4M3 && (none || 32 * g + 32 > hi)) {
#pragma unroll
                for (int j = 0; j < NJ; j++) vr[j] = vx_kvq_mask_codes(vr[j], t0, none ? 0 : hi);
            }
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const vx_half8 v0 = vx_kvq_half8<TYPE>(vr[j].x, vr[j].y), v1 = vx_kvq_half8<TYPE>(vr[j].z, vr[j].w);
                vr[j] = *(const uint4 *)(vn + 1024 * j);
                vx_f32x4 t = vx_mfma(v0, pl, vx_f32x4{}), u = vx_mfma(v1, pl, vx_f32x4{});
                t = vx_mfma(v0, ph, t);
                u = vx_mfma(v1, ph, u);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    O[2 * j][e] = fmaf(t[e], vsc, O[2 * j][e]);
                    O[2 * j + 1][e] = fmaf(u[e], vsc, O[2 * j + 1][e]);
                }
            }
        }

        auto finish = [&](int qi, int d, vx_f32x4 o, float sum) {
            const float inv = sum != 0.0f ? AK_P / sum : 0.0f;
            *(vx_f32x4 *)(out + (size_t)(s.row + qi / a.G) * c.ld_out + (size_t)(kvh * a.G + qi % a.G) * HD + d) = o * inv;
        };
        l = vx_sum_x32(vx_sum_x16(l));
        if (few > 1) {
            if (wave < few && ok)
#pragma unroll
                for (int d = 0; d < ND; d++) finish(qi, 16 * d + 4 * g4, O[d], l);
            x = first + (int64_t)few * (groups + AK_BEGIN);
            __syncthreads();
            if (x < w_end) {
                vx_kvq_find(a, list, x, 0);
                __syncthreads();
            }
            continue;
        }
        // the wavefronts' parts meet in LDS
        __syncthreads();
        {
            float *so = sh.o[wave][n];
#pragma unroll
            for (int d = 0; d < ND; d++) *(vx_f32x4 *)(so + 16 * d + 4 * g4) = O[d];
            if (g4 == 0) *(float2 *)(so + HD) = make_float2(m, l);
        }
        __syncthreads();
        const bool whole = g_begin == 0 && g_end == groups;
        // a piece holds at most one tile begun before it and one that goes on behind it
        const int mine = (2 * (int)blockIdx.x + (g_begin == 0)) * (16 * PS);
        const int nv = min(16, s.nq - q0);
        for (int u = tid; u < nv * (HD / 4); u += AK_THREADS) {
            const int qq = u / (HD / 4), d = u % (HD / 4) * 4;
            float mx = sh.o[0][qq][HD];
#pragma unroll
            for (int w = 1; w < AK_WAVES; w++) mx = fmaxf(mx, sh.o[w][qq][HD]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            float sum = 0.0f;
            vx_f32x4 o = vx_f32x4{};
#pragma unroll
            for (int w = 0; w < AK_WAVES; w++) {
                const float f = __builtin_amdgcn_exp2f(sh.o[w][qq][HD] - ref);
                sum = fmaf(sh.o[w][qq][HD + 1], f, sum);
                o += *(const vx_f32x4 *)(&sh.o[w][qq][d]) * f;
            }
            if (whole)
                finish(q0 + qq, d, o, sum);
            else {
                vx_part_store(part, mine, qq * PS + d, o);
                if (d == 0) vx_part_store2(part, mine, qq * PS + HD, mx, sum);
            }
        }
        if (!whole) {
            // the pieces p0..p1 that hold a part of this tile join in blocks of
            // AK_BLOCK, and the blocks: each time the last one to finish does it
            // (its inner boundaries lie past first + AK_BEGIN + snap and before end - snap)
            const int p0 = (int)vx_quot(first + AK_BEGIN + snap, piece);
            const int p1 = max((int)vx_quot(first + AK_BEGIN + groups - snap + piece - 1, piece) - 1, p0);
            const int me = (int)blockIdx.x - p0, blk = me / AK_BLOCK, n_blk = (p1 - p0) / AK_BLOCK + 1;
            const int c0 = blk * AK_BLOCK, c1 = min(c0 + AK_BLOCK, p1 - p0 + 1);
            // a piece inside the tile has a second slot: a block's joint result goes
            // to its first piece's (the first block's to its second, the first may
            // hold the end of another tile)
            auto slot0 = [&](int i) { return 2 * (p0 + i) + (i == 0); };
            auto slot1 = [&](int i) {
                const int f = i * AK_BLOCK;
                return f == p1 - p0 ? slot0(f) : 2 * (p0 + f + (i == 0)) + 1;
            };
            bool last = c1 - c0 == 1 || vx_arrive(counter + p0 + blk, c1 - c0, &s_last);
            if (last && n_blk > 1) {
                if (c1 - c0 > 1)
                    vx_kvq_join<HD>(part, slot0, c0, c1, nv, [&](int qq, int d, vx_f32x4 o, float mx, float sum) {
                        vx_part_store(part, slot1(blk) * (16 * PS), qq * PS + d, o);
                        if (d == 0) vx_part_store2(part, slot1(blk) * (16 * PS), qq * PS + HD, mx, sum);
                    });
                last = vx_arrive(counter + AK_WG + p0, n_blk, &s_last);
            }
            auto put = [&](int qq, int d, vx_f32x4 o, float mx, float sum) { finish(q0 + qq, d, o, sum); };
            if (last && n_blk > 1) vx_kvq_join<HD>(part, slot1, 0, n_blk, nv, put);
            else if (last) vx_kvq_join<HD>(part, slot0, 0, c1, nv, put);
        }
        x = first + AK_BEGIN + g_end;
        if (x < w_end) {
            __syncthreads();
            vx_kvq_find(a, list, x, 0);
            __syncthreads();
        }
    }
}

extern "C" size_t vxh_attention_kvq_workspace_floats(int max_rows, int n_seqs, int n_heads, int n_kv_heads,
                                                     int head_dim)
{
    // two parts a piece, whatever the batch
    (void)max_rows, (void)n_seqs, (void)n_heads, (void)n_kv_heads;
    return (size_t)2 * AK_WG * 16 * (head_dim + 4);
}

extern "C" int vxh_attention_kvq(const float *q, int ldq, const int *row0, const int *len, int n_seqs, int max_rows,
                                 int max_seq_rows, const int *table, int ld_table, int n_heads, const vxh_kvq *c,
                                 int cap, float *out, int ld_out, vxh_workspace *ws, vxh_stream s)
{
    if (const char *bad = vx_kvq_bad(c)) return vxh_fail(VXH_ERR_PARAM, "attention_kvq: %s", bad);
    // (no row count times head count passes 32 bits in the kernels)
    const int64_t w = (int64_t)n_heads * c->head_dim;
    if (!q || !row0 || !len || !table || !out || !ws || !ws->acc || !ws->part || n_seqs < 1 || n_seqs > VXH_PAGE_MAX_SEQS ||
        max_rows < 1 || max_rows > VXH_PAGE_MAX_ROWS || max_seq_rows < 1 || ld_table < 1 || cap < 0 || n_heads < 1 ||
        (int64_t)max_rows * n_heads > 0x7FFFFFFF || n_heads % c->n_kv_heads || ldq < w || ldq % 4 || ld_out < w || ld_out % 4 || ((uintptr_t)q & 15) ||
        ((uintptr_t)out & 15) ||
        ws->part_floats < vxh_attention_kvq_workspace_floats(max_rows, n_seqs, n_heads, c->n_kv_heads, c->head_dim))
        return vxh_fail(VXH_ERR_PARAM, "attention_kvq: %d requests, %d rows, %d/%d heads of %d (ld %d, %d)", n_seqs,
                        max_rows, n_heads, c->n_kv_heads, c->head_dim, ldq, ld_out);
    const int64_t limit = (int64_t)ld_table * c->page;
    vx_kvq_call call;
    call.a.row0 = row0;
    call.a.len = len;
    call.a.B = n_seqs;
    call.a.max_rows = max_rows;
    call.a.n_kv = c->n_kv_heads;
    call.a.G = n_heads / c->n_kv_heads;
    call.a.cap = cap;
    call.a.limit = limit > 0x7FFFFF00 ? 0x7FFFFF00 : (int)limit;
    call.a.few = 0x7FFFFFFF;
    call.q = q;
    call.ldq = ldq;
    call.table = table;
    call.ld_table = ld_table;
    call.kc = (const uint8_t *)c->k;
    call.vc = (const uint8_t *)c->v;
    call.ks = c->ks;
    call.vs = c->vs;
    call.shift = c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
    call.n_pages = c->n_pages;
    call.out = out;
    call.ld_out = ld_out;
    call.part = ws->part;
    if (vx_kvq_many_wanted(call.a, max_seq_rows)) {
        // of one request the host knows the rows: nothing is left for the other kernel
        call.a.few = n_seqs == 1 ? 0 : AK_FEW;
        int rc = vx_kvq_many(call, c->type, c->head_dim, vxh_hs(s));
        if (rc || n_seqs == 1) return rc;
    }
    unsigned *counter = (unsigned *)(ws->acc + ws->acc_elems);
#define VX_CALL(T, HD) vx_attention_kvq_kernel<T, HD><<<AK_WG, AK_THREADS, 0, vxh_hs(s)>>>( \
        call, call.q, call.table, call.kc, call.vc, call.ks, call.vs, call.out, call.part, counter)
#define VX_HD(T)                                                                                                      \
    switch (c->head_dim) {                                                                                            \
    case 32: VX_CALL(T, 32); break;                                                                                   \
    case 64: VX_CALL(T, 64); break;                                                                                   \
    case 96: VX_CALL(T, 96); break;                                                                                   \
    default: VX_CALL(T, 128);                                                                                         \
    }
    if (c->type == VXH_KVQ_INT8) {
        VX_HD(VXH_KVQ_INT8)
    } else {
        VX_HD(VXH_KVQ_E4M3)
    }
#undef VX_HD
#undef VX_CALL
    VXH_LAUNCHED();
    return VXH_OK;
}
