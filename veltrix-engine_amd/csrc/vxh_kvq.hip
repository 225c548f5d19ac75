// Paged KV cache in 8 bits: page tables and slots of a step, the write of new
// rows and their read-back (the attention over it is in vxh_attn_kvq.hip).
#include <string.h>

#include "vxh_kvq.h"

const char *vx_kvq_bad(const vxh_kvq *c)
{
    if (!c || !c->k || !c->v || !c->ks || !c->vs) return "no cache";
    if (c->type != VXH_KVQ_INT8 && c->type != VXH_KVQ_E4M3) return "type";
    if (c->page != 32 && c->page != 64 && c->page != 128) return "page size";
    if (c->head_dim % 32 || c->head_dim < 32 || c->head_dim > 128) return "head_dim";
    if (c->n_pages < 1 || c->n_kv_heads < 1 || (int64_t)c->n_pages * c->page > 0x7FFFFFFF ||
        (int64_t)c->n_kv_heads * c->head_dim > 0x3FFFFFFF)
        return "size";
    if (((uintptr_t)c->k & 15) || ((uintptr_t)c->v & 15) || ((uintptr_t)c->ks & 3) || ((uintptr_t)c->vs & 3))
        return "alignment";
    return nullptr;
}

extern "C" int vxh_kvq_alloc(vxh_kvq *c, int type, int page, int n_pages, int n_kv_heads, int head_dim)
{
    if (!c) return vxh_fail(VXH_ERR_PARAM, "kvq_alloc: no handle");
    memset(c, 0, sizeof(*c));
    float *const some = (float *)16;                     // the arrays come once the rest is known to be good
    vxh_kvq t = {type, page, n_pages, n_kv_heads, head_dim, some, some, some, some};
    if (const char *bad = vx_kvq_bad(&t))
        return vxh_fail(VXH_ERR_PARAM, "kvq_alloc: %s (type %d, %d pages of %d, %d heads of %d)", bad, type, n_pages,
                        page, n_kv_heads, head_dim);
    const size_t bytes = (size_t)n_pages * page * n_kv_heads * head_dim, ns = (size_t)n_pages * n_kv_heads;
    t.k = t.v = nullptr;
    t.ks = t.vs = nullptr;
    int rc = vxh_malloc(&t.k, bytes);
    if (!rc) rc = vxh_malloc(&t.v, bytes);
    if (!rc) rc = vxh_malloc((void **)&t.ks, ns * sizeof(float));
    if (!rc) rc = vxh_malloc((void **)&t.vs, ns * sizeof(float));
    // scales of zero: a cache that holds zeros, whatever its bytes
    if (!rc) rc = vxh_fill_f32((float *)t.k, 0.0f, bytes / 4, nullptr);
    if (!rc) rc = vxh_fill_f32((float *)t.v, 0.0f, bytes / 4, nullptr);
    if (!rc) rc = vxh_fill_f32(t.ks, 0.0f, ns, nullptr);
    if (!rc) rc = vxh_fill_f32(t.vs, 0.0f, ns, nullptr);
    if (!rc) rc = vxh_stream_sync(nullptr);
    if (rc) {
        vxh_kvq_free(&t);
        return rc;
    }
    *c = t;
    return VXH_OK;
}

extern "C" int vxh_kvq_free(vxh_kvq *c)
{
    if (!c) return VXH_OK;
    vxh_free(c->k);
    vxh_free(c->v);
    vxh_free(c->ks);
    vxh_free(c->vs);
    memset(c, 0, sizeof(*c));
    return VXH_OK;
}

// ---------------------------------------------------------------------------
// Page tables.  Every workgroup scans all requests (rows and pages before
// each, in LDS) and then does its share of the rows and entries, so the step
// is one launch: no workgroup waits for another.  The totals are 64-bit; the
// sums kept in 32 are used only by a step that fits.
// Bound by the chain of its dependent loads, scan and searches: 2.8 us for one
// request of 9 rows, 5.0 for 1012 requests with 12 prompt chunks among them
// (their bytes at the copy rate: 0.02 us).
// ---------------------------------------------------------------------------
#define PT_THREADS 256

__global__ __launch_bounds__(PT_THREADS) void vx_page_tables_kernel(
    const int *__restrict__ len, const int *__restrict__ add, int B, int shift, const int *__restrict__ free_pages,
    int n_free, int *__restrict__ table, int ld_table, int *__restrict__ len_out, int *__restrict__ row0,
    int *__restrict__ row_pos, int *__restrict__ slot, int max_rows, int *__restrict__ counts)
{
    extern __shared__ int s_scan[];
    int *s_row = s_scan, *s_new = s_scan + B + 1;        // exclusive sums, [B] = totals
    __shared__ int64_t s_wave[2][PT_THREADS / 64];
    __shared__ int s_flag;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, mask = (1 << shift) - 1;
    if (tid == 0) s_flag = 0;
    __syncthreads();
    // a run of E requests per thread
    const int E = (B + PT_THREADS - 1) / PT_THREADS, b0 = min(tid * E, B), b1 = min(b0 + E, B);
    int64_t rows = 0, fresh = 0;
    bool wide = false;
    for (int b = b0; b < b1; b++) {
        const int64_t n = max(len[b], 0), a = max(add[b], 0), need = (n + a + mask) >> shift;
        wide |= need > ld_table;
        s_row[b] = (int)rows;
        s_new[b] = (int)fresh;
        rows += a;
        fresh += need - ((n + mask) >> shift);
    }
    if (wide) s_flag = 4;
    int64_t r_in = rows, f_in = fresh;                   // inclusive over the wavefront
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t r = __shfl_up(r_in, o), f = __shfl_up(f_in, o);
        if (lane >= o) {
            r_in += r;
            f_in += f;
        }
    }
    if (lane == 63) {
        s_wave[0][wave] = r_in;
        s_wave[1][wave] = f_in;
    }
    __syncthreads();
    int64_t r_at = r_in - rows, f_at = f_in - fresh, r_sum = 0, f_sum = 0;
    for (int w = 0; w < PT_THREADS / 64; w++) {
        if (w < wave) {
            r_at += s_wave[0][w];
            f_at += s_wave[1][w];
        }
        r_sum += s_wave[0][w];
        f_sum += s_wave[1][w];
    }
    for (int b = b0; b < b1; b++) {
        s_row[b] += (int)r_at;
        s_new[b] += (int)f_at;
    }
    const int r_all = (int)r_sum, f_all = (int)f_sum;
    if (tid == 0) {
        s_row[B] = r_all;
        s_new[B] = f_all;
    }
    const int flag = s_flag | (f_sum > n_free ? 1 : 0) | (r_sum > max_rows ? 2 : 0);
    __syncthreads();
    const bool ok = flag == 0;
    const int step = gridDim.x * PT_THREADS, first = blockIdx.x * PT_THREADS + tid;
    if (first == 0) {
        counts[0] = ok ? r_all : 0;
        counts[1] = ok ? f_all : 0;
        counts[2] = flag;
        counts[3] = f_sum > 0x7FFFFFFF ? 0x7FFFFFFF : f_all;
    }
    for (int b = first; b <= B; b += step) {
        row0[b] = ok ? s_row[b] : 0;
        if (b < B) len_out[b] = max(len[b], 0) + (ok ? s_row[b + 1] - s_row[b] : 0);
    }
    auto find = [&](const int *s, int i) {               // last b with s[b] <= i: skips requests of nothing
        int lo = 0, hi = B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s[mid] <= i) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    for (int i = first; ok && i < f_all; i += step) {
        const int b = find(s_new, i);
        const int have = (int)(((int64_t)max(len[b], 0) + mask) >> shift);
        table[(size_t)b * ld_table + have + i - s_new[b]] = free_pages[i];
    }
    for (int r = first; r < max_rows; r += step) {
        int pos = -1, sl = -1;
        if (ok && r < r_all) {
            const int b = find(s_row, r), n = max(len[b], 0);
            pos = n + r - s_row[b];
            const int col = pos >> shift, have = (int)(((int64_t)n + mask) >> shift);
            // a page of this step comes from the free list: its entry may not be written yet
            const int page = col < have ? table[(size_t)b * ld_table + col] : free_pages[s_new[b] + col - have];
            sl = page < 0 || page > (0x7FFFFFFF >> shift) - 1 ? -1 : (page << shift) + (pos & mask);
        }
        row_pos[r] = pos;
        slot[r] = sl;
    }
}

static bool vx_overlap(const void *a, size_t na, const void *b, size_t nb)
{
    return (const char *)a < (const char *)b + nb && (const char *)b < (const char *)a + na;
}

extern "C" int vxh_page_tables(const int *len, const int *add, int n_seqs, int page, const int *free_pages, int n_free,
                               int *table, int ld_table, int *len_out, int *row0, int *row_pos, int *slot, int max_rows,
                               int *counts, vxh_stream s)
{
    if (!len || !add || !table || !len_out || !row0 || !row_pos || !slot || !counts || (n_free > 0 && !free_pages))
        return vxh_fail(VXH_ERR_PARAM, "page_tables: missing array");
    if (n_seqs < 1 || n_seqs > VXH_PAGE_MAX_SEQS || (page != 32 && page != 64 && page != 128) || n_free < 0 ||
        ld_table < 1 || (int64_t)ld_table * page > 0x7FFFFFFF || max_rows < 1 || max_rows > VXH_PAGE_MAX_ROWS)
        return vxh_fail(VXH_ERR_PARAM, "page_tables: %d requests, pages of %d, %d free, %d columns, %d rows", n_seqs,
                        page, n_free, ld_table, max_rows);
    const size_t nb = (size_t)n_seqs * sizeof(int);
    if (vx_overlap(len, nb, len_out, nb) || vx_overlap(add, nb, len_out, nb))
        return vxh_fail(VXH_ERR_PARAM, "page_tables: len_out lies over len or add");
    const int shift = page == 32 ? 5 : page == 64 ? 6 : 7;
    int grid = (max_rows + PT_THREADS - 1) / PT_THREADS;
    if (grid > 64) grid = 64;
    vx_page_tables_kernel<<<grid, PT_THREADS, 2 * (n_seqs + 1) * sizeof(int), vxh_hs(s)>>>(
        len, add, n_seqs, shift, free_pages, n_free, table, ld_table, len_out, row0, row_pos, slot, max_rows, counts);
    VXH_LAUNCHED();
    return VXH_OK;
}

// ---------------------------------------------------------------------------
// Write.  A workgroup owns pages of K or V of some heads: the first of the
// batch's rows on a page names it, and every other row of the page, wherever it
// stands, is found by one pass over the slots.  So a scale has one writer and
// the result does not depend on the order of workgroups.  The rows are read
// once, into registers; their codes meet in LDS in the cache's order and leave
// as whole 16-byte lanes, blended with the page's other tokens.
// Bound by HBM for a prompt: 2048 rows, 32 heads of 128, 29 us for 84 MB (2.9
// TB/s; 65 pages x 16 workgroups, 4 parts each in turn, are four workgroups a
// CU, and twice as many, each with its pass over the slots, are no faster), and
// by latency below it: 4.8 us for one row of 4 heads, 8.0 for 64 rows on 64
// pages (the slots, the rows, the old codes; the old codes asked for with the
// rows, or the slots with the first rows': the same).
// ---------------------------------------------------------------------------
#define KW_THREADS 256
#define KW_PIECES 128            // of the rows
#define KW_WG 2048               // workgroups; heads past that in turn

// x is taken as new here: what follows from it is worked out again, not kept in
// registers (16 items' conditions, for every part) from before the loop.
#define KW_HERE(x) asm("" : "+v"(x))

// Bytes of a word whose bits 0..3 are set in nib.
__device__ __forceinline__ uint32_t vx_spread(uint32_t nib) { return (((nib & 15u) * 0x00204081u) & 0x01010101u) * 0xFFu; }

template <int TYPE, int PG>
__global__ __launch_bounds__(KW_THREADS) void vx_kvq_write_kernel(vxh_kvq c, const float *__restrict__ k, int ldk,
                                                                  const float *__restrict__ v, int ldv,
                                                                  const int *__restrict__ slot, int R, int chunk)
{
    constexpr int P = 32 * PG, SHIFT = PG == 1 ? 5 : PG == 2 ? 6 : 7, NI = 4 * PG;
    __shared__ int s_src[P], s_first;
    __shared__ uint32_t s_has[PG];                       // the page's tokens that come, a bit each
    __shared__ float s_amax[KW_THREADS / 64];
    __shared__ uint4 s_code[P * 128 / 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hd = c.head_dim;
    const unsigned n_pages = c.n_pages;
    const int n4 = hd / 4;                               // items of 4 dims a token
    const float per4 = 1.0f / n4;
    auto token = [&](int it) { return (int)(((float)it + 0.5f) * per4); };
    auto page_of = [&](int sl) { return sl < 0 || (unsigned)(sl >> SHIFT) >= n_pages ? -1 : sl >> SHIFT; };
    const int r1 = min((int)(blockIdx.y + 1) * chunk, R);
    uint64_t leads = 0;                                  // of 64 rows from base: those that may lead a page
    int here = -1;                                       // the lane's row's page
    for (int base = blockIdx.y * chunk - 64;;) {
        if (!leads) {
            // (a row behind another of its page is that one's)
            base += 64;
            if (base >= r1) break;
            const int r = base + lane;
            here = r < r1 ? page_of(slot[r]) : -1;
            const int before = r < r1 && r > 0 ? page_of(slot[r - 1]) : -1;
            leads = __ballot(here >= 0 && here != before);
            continue;
        }
        const int at = __ffsll((unsigned long long)leads) - 1, lead = base + at, page = __builtin_amdgcn_readlane(here, at);
        leads &= leads - 1;
        __syncthreads();
        if (tid == 0) s_first = R;
        for (int i = tid; i < P; i += KW_THREADS) s_src[i] = -1;
        if (tid < PG) s_has[tid] = 0;
        __syncthreads();
        for (int r0 = tid; r0 < R; r0 += 8 * KW_THREADS) {
            int sl[8];
#pragma unroll
            for (int i = 0; i < 8; i++) sl[i] = r0 + i * KW_THREADS < R ? slot[r0 + i * KW_THREADS] : -1;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (page_of(sl[i]) == page) {
                    const int r = r0 + i * KW_THREADS, t = sl[i] & (P - 1);
                    atomicMin(&s_first, r);
                    atomicMax(&s_src[t], r);             // the same slot twice: the later row
                    atomicOr(&s_has[t >> 5], 1u << (t & 31));
                }
        }
        __syncthreads();
        if (s_first != lead) continue;                   // an earlier row has this page

        // a part's rows, this thread's items of 4 dims; the next part's are on
        // their way while one is worked on
        float4 val[NI];
        unsigned live = 0;                               // items whose token comes, a bit each
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int t = token(tid + i * KW_THREADS);
            if (t < P && s_src[t] >= 0) live |= 1u << i;
        }
        auto fetch = [&](int part) {
            const bool is_v = part >= c.n_kv_heads;
            const int ldx = is_v ? ldv : ldk;
            const float *x = is_v ? v + (part - c.n_kv_heads) * hd : k + part * hd;
            KW_HERE(live);
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int it = tid + i * KW_THREADS, t = token(it);
                val[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (live >> i & 1) val[i] = *(const float4 *)(x + (size_t)s_src[t] * ldx + 4 * (it - t * n4));
            }
        };
        fetch(blockIdx.x);
        for (int part = blockIdx.x; part < 2 * c.n_kv_heads; part += gridDim.x) {
            const bool is_v = part >= c.n_kv_heads;
            const int head = is_v ? part - c.n_kv_heads : part;
            const size_t hp = (size_t)page * c.n_kv_heads + head;
            uint4 *dst = (uint4 *)((uint8_t *)(is_v ? c.v : c.k) + hp * (size_t)(P * hd));
            float *sp = (is_v ? c.vs : c.ks) + hp;
            const float held = *sp;
            float amax = 0.0f;
            bool finite = true;
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const float a[4] = {val[i].x, val[i].y, val[i].z, val[i].w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool f = fabsf(a[e]) < INFINITY;
                    finite &= f;
                    amax = fmaxf(amax, f ? fabsf(a[e]) : 0.0f);
                }
            }
            amax = vx_wave_max64(amax);
            if (lane == 0) s_amax[wave] = amax;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < KW_THREADS / 64; w++) amax = fmaxf(amax, s_amax[w]);
            const float fit = amax >= 0x1p-100f ? amax / (TYPE == VXH_KVQ_INT8 ? 127.0f : 448.0f) : 0.0f;
            const bool start = s_has[0] & 1;             // the page's first token starts it anew
            const float s_old = start ? 0.0f : held, sc = fmaxf(s_old, fit), inv = sc > 0.0f ? 1.0f / sc : 0.0f;
            const bool grown = sc > s_old && !start;
            KW_HERE(live);
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int it = tid + i * KW_THREADS, t = token(it), d = 4 * (it - t * n4);
                if (live >> i & 1) {
                    const float a[4] = {val[i].x, val[i].y, val[i].z, val[i].w};
                    uint32_t code[4];
                    bool sure = finite && sc > 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; e++) code[e] = vx_kvq_code_fast<TYPE>(a[e], sc, inv, &sure);
                    if (!sure) {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            code[e] = sc > 0.0f ? vx_kvq_code<TYPE>(a[e], sc, inv) : TYPE == VXH_KVQ_INT8 ? 128u : 0u;
                    }
                    if (is_v) {
#pragma unroll
                        for (int e = 0; e < 4; e++) ((uint8_t *)s_code)[vx_kvq_v_byte(t, d + e, hd)] = (uint8_t)code[e];
                    } else
                        *(uint32_t *)((uint8_t *)s_code + vx_kvq_k_byte(t, d, hd)) =
                            code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
                }
            }
            if (part + (int)gridDim.x < 2 * c.n_kv_heads) fetch(part + gridDim.x);
            __syncthreads();
            if (tid == 0) *sp = sc;
            // lanes of 16 codes: K holds 8 dims of two tokens, V 8 tokens of two dims
            for (int u = tid; u < P * hd / 16; u += KW_THREADS) {
                const uint32_t has = s_has[(u >> 6) / (hd / 32)];
                const int g = (u >> 4) & 3, n = u & 15;
                uint32_t m0, m1, m2, m3;
                if (is_v) {
                    m0 = m2 = vx_spread(has >> (4 * g));
                    m1 = m3 = vx_spread(has >> (16 + 4 * g));
                } else {
                    m0 = m1 = has >> n & 1 ? ~0u : 0u;
                    m2 = m3 = has >> (n + 16) & 1 ? ~0u : 0u;
                }
                if (!(m0 | m1 | m2) && !grown) continue;
                uint4 w = s_code[u];
                if ((m0 & m1 & m2) != ~0u) {
                    uint4 old = dst[u];
                    if (grown) {
                        uint32_t o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int sh = 8 * (e & 3);
                            const uint32_t code = vx_kvq_recode<TYPE>(vx_kvq_value<TYPE>((o[e >> 2] >> sh) & 0xFFu), s_old, sc);
                            o[e >> 2] = (o[e >> 2] & ~(0xFFu << sh)) | (code << sh);
                        }
                        old = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                    w = make_uint4((w.x & m0) | (old.x & ~m0), (w.y & m1) | (old.y & ~m1), (w.z & m2) | (old.z & ~m2),
                                   (w.w & m3) | (old.w & ~m3));
                }
                dst[u] = w;
            }
        }
    }
}

static int vx_kvq_rows_check(const char *what, const vxh_kvq *c, const void *k, int ldk, const void *v, int ldv,
                             const int *slot, int R)
{
    if (const char *bad = vx_kvq_bad(c)) return vxh_fail(VXH_ERR_PARAM, "%s: %s", what, bad);
    const int w = c->n_kv_heads * c->head_dim;
    if (!k || !v || !slot || R < 1 || R > VXH_KVQ_MAX_ROWS || ldk < w || ldv < w || ldk % 4 || ldv % 4 ||
        ((uintptr_t)k & 15) || ((uintptr_t)v & 15))
        return vxh_fail(VXH_ERR_PARAM, "%s: %d rows of %d (ld %d, %d)", what, R, w, ldk, ldv);
    return VXH_OK;
}

extern "C" int vxh_kvq_write(const vxh_kvq *c, const float *k, int ldk, const float *v, int ldv, const int *slot, int R,
                             vxh_stream s)
{
    int rc = vx_kvq_rows_check("kvq_write", c, k, ldk, v, ldv, slot, R);
    if (rc) return rc;
    // A prompt's pages begin every 32nd row or so: an odd piece length keeps the
    // workgroups that find one off one XCD (2048 rows, 32 heads of 128: 153 us
    // with all on one, 29 spread).  More pieces find the pages sooner, fewer
    // leave each page to more workgroups: write and read-back of 2048 rows took
    // 52 us with 256 pieces, 46 with 128, 46 with 64; of 1500 rows, 32 heads of
    // 64, pages of 64: 51, 40, 39; of 2048 rows, 4 heads of 128: 16, 15, 19.
    const int chunk = R <= KW_PIECES ? 1 : (R + KW_PIECES - 1) / KW_PIECES | 1, gy = (R + chunk - 1) / chunk;
    int gx = 2 * c->n_kv_heads;
    if (gx > KW_WG / gy) gx = KW_WG / gy;
    const dim3 grid(gx, gy);
#define VX_CALL(T, PG) vx_kvq_write_kernel<T, PG><<<grid, KW_THREADS, 0, vxh_hs(s)>>>(*c, k, ldk, v, ldv, slot, R, chunk)
#define VX_PAGE(T)                                                                                                    \
    if (c->page == 32) VX_CALL(T, 1);                                                                                 \
    else if (c->page == 64) VX_CALL(T, 2);                                                                            \
    else VX_CALL(T, 4);
    if (c->type == VXH_KVQ_INT8) {
        VX_PAGE(VXH_KVQ_INT8)
    } else {
        VX_PAGE(VXH_KVQ_E4M3)
    }
#undef VX_PAGE
#undef VX_CALL
    VXH_LAUNCHED();
    return VXH_OK;
}

// ---------------------------------------------------------------------------
// Read-back.  A workgroup takes 32 rows of one kv head's K or V.  Rows that are
// 32 tokens of a page in order (a request read from its start) come as whole
// lanes of the cache through LDS; any others code by code.
// Bound by HBM: 2048 rows, 32 heads of 128, 14.7 us for 84 MB, 5.7 TB/s (36 us
// when every value fetched its own byte); 64 single rows 6.0 us, latency.
// ---------------------------------------------------------------------------
template <int TYPE>
__global__ __launch_bounds__(256) void vx_kvq_read_kernel(vxh_kvq c, const int *__restrict__ slot, int R,
                                                          float *__restrict__ k, int ldk, float *__restrict__ v, int ldv,
                                                          int shift)
{
    __shared__ float s_row[32][128 + 4];
    const int tid = threadIdx.x, hd = c.head_dim, n4 = hd / 4, r0 = blockIdx.y * 32;
    const bool is_v = (int)blockIdx.x >= c.n_kv_heads;
    const int head = is_v ? blockIdx.x - c.n_kv_heads : blockIdx.x, ldx = is_v ? ldv : ldk;
    float *x = (is_v ? v : k) + head * hd;
    const uint8_t *codes = (const uint8_t *)(is_v ? c.v : c.k);
    const float *scales = is_v ? c.vs : c.ks;
    const int s0 = slot[r0], mine = r0 + (tid & 31) < R ? slot[r0 + (tid & 31)] : -1;
    const bool whole = __all(mine == s0 + (tid & 31)) && s0 >= 0 && s0 % 32 == 0 && (s0 >> shift) < c.n_pages;
    if (whole) {                                         // (the same in every wavefront)
        const size_t hp = (size_t)(s0 >> shift) * c.n_kv_heads + head;
        const float sc = scales[hp];
        const uint4 *src = (const uint4 *)(codes + (hp << shift) * hd + (size_t)(s0 & ((1 << shift) - 1)) * hd);
        for (int u = tid; u < 2 * hd; u += 256) {        // 64 lanes for each 32 dims
            const uint4 w = src[u];
            const uint32_t word[4] = {w.x, w.y, w.z, w.w};
            const int g = (u >> 4) & 3, n = u & 15, d0 = u / 64 * 32;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float f = vx_kvq_value<TYPE>((word[e >> 2] >> (8 * (e & 3))) & 0xFFu) * sc;
                if (is_v) s_row[((e >> 2) & 1) * 16 + 4 * g + (e & 3)][d0 + (e >> 3) * 16 + n] = f;
                else s_row[(e >> 3) * 16 + n][d0 + 8 * g + (e & 7)] = f;
            }
        }
        __syncthreads();
        for (int i = tid; i < 32 * n4; i += 256)
            *(float4 *)(x + (size_t)(r0 + i / n4) * ldx + 4 * (i % n4)) = *(const float4 *)&s_row[i / n4][4 * (i % n4)];
        return;
    }
    // (head_dim / 32 items a thread: the loads of all of them go out together)
    int sl[4];
    float sc[4];
    uint32_t code[4][4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = tid + j * 256, r = r0 + i / n4;
        sl[j] = i < 32 * n4 && r < R ? slot[r] : -1;
        if (sl[j] >= 0 && (sl[j] >> shift) >= c.n_pages) sl[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (sl[j] >= 0) {
            const int d = 4 * ((tid + j * 256) % n4), t = sl[j] & ((1 << shift) - 1);
            const size_t hp = (size_t)(sl[j] >> shift) * c.n_kv_heads + head;
            const uint8_t *p = codes + (hp << shift) * hd;
            sc[j] = scales[hp];
            if (is_v) {
#pragma unroll
                for (int e = 0; e < 4; e++) code[j][e] = p[vx_kvq_v_byte(t, d + e, hd)];
            } else {
                const uint32_t w = *(const uint32_t *)(p + vx_kvq_k_byte(t, d, hd));
#pragma unroll
                for (int e = 0; e < 4; e++) code[j][e] = w >> (8 * e) & 0xFFu;
            }
        }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (sl[j] >= 0) {
            const int i = tid + j * 256;
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = vx_kvq_value<TYPE>(code[j][e]) * sc[j];
            *(float4 *)(x + (size_t)(r0 + i / n4) * ldx + 4 * (i % n4)) = make_float4(f[0], f[1], f[2], f[3]);
        }
}

extern "C" int vxh_kvq_read(const vxh_kvq *c, const int *slot, int R, float *k, int ldk, float *v, int ldv,
                            vxh_stream s)
{
    int rc = vx_kvq_rows_check("kvq_read", c, k, ldk, v, ldv, slot, R);
    if (rc) return rc;
    const int shift = c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
    const dim3 grid(2 * c->n_kv_heads, (R + 31) / 32);
    if (c->type == VXH_KVQ_INT8)
        vx_kvq_read_kernel<VXH_KVQ_INT8><<<grid, 256, 0, vxh_hs(s)>>>(*c, slot, R, k, ldk, v, ldv, shift);
    else
        vx_kvq_read_kernel<VXH_KVQ_E4M3><<<grid, 256, 0, vxh_hs(s)>>>(*c, slot, R, k, ldk, v, ldv, shift);
    VXH_LAUNCHED();
    return VXH_OK;
}
