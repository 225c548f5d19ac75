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
    if (c->n_pages < 1 || c->n_kv_heads < 1 || (int64_t)c->n_pages * c->page > 0x7FFFFFFF) return "size";
    return nullptr;
}

extern "C" int vxh_kvq_alloc(vxh_kvq *c, int type, int page, int n_pages, int n_kv_heads, int head_dim)
{
    if (!c) return vxh_fail(VXH_ERR_PARAM, "kvq_alloc: no handle");
    memset(c, 0, sizeof(*c));
    vxh_kvq t = {type, page, n_pages, n_kv_heads, head_dim, c, c, (float *)c, (float *)c};
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
        const int have = (max(len[b], 0) + mask) >> shift;
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
        ld_table < 1 || max_rows < 1 || max_rows > VXH_PAGE_MAX_ROWS)
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
// Write.  A workgroup owns one (page, kv head) of K or of V: a page's first
// row in the batch names it, and every other row of the page, wherever it
// stands, is found by one pass over the slots.  So a scale has one writer and
// the result does not depend on the order of workgroups.  The rows are read
// once, into registers; their codes meet in LDS and leave as whole 16-byte
// lanes of the cache's layout.
// ---------------------------------------------------------------------------
#define KW_THREADS 256

template <int TYPE>
__global__ __launch_bounds__(KW_THREADS) void vx_kvq_write_kernel(vxh_kvq c, const float *__restrict__ k, int ldk,
                                                                  const float *__restrict__ v, int ldv,
                                                                  const int *__restrict__ slot, int R)
{
    __shared__ int s_src[KVQ_MAX_PAGE], s_first, s_count[KW_THREADS / 64], s_lead;
    __shared__ float s_amax[KW_THREADS / 64];
    __shared__ __align__(16) uint8_t s_code[KVQ_MAX_PAGE * (128 + 16)];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int P = c.page, hd = c.head_dim, head = blockIdx.y, ldc = hd + 16;
    const bool is_v = blockIdx.z;
    const float *x = is_v ? v : k;
    const int ldx = is_v ? ldv : ldk;
    uint8_t *cache = (uint8_t *)(is_v ? c.v : c.k);
    float *scales = is_v ? c.vs : c.ks;
    auto page_of = [&](int r) {
        const int sl = slot[r];
        return sl < 0 || sl / P >= c.n_pages ? -1 : sl / P;
    };
    // candidates: rows whose predecessor lies on another page, counted in order
    const int E = (R + KW_THREADS - 1) / KW_THREADS, r0 = min(tid * E, R), r1 = min(r0 + E, R);
    int mine = 0;
    {
        int before = r0 > 0 && r0 < R ? page_of(r0 - 1) : -1;
        for (int r = r0; r < r1; r++) {
            const int p = page_of(r);
            mine += p >= 0 && p != before;
            before = p;
        }
    }
    int at = mine;
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(at, o);
        if (lane >= o) at += u;
    }
    if (lane == 63) s_count[wave] = at;
    __syncthreads();
    int total = 0;
    at -= mine;
    for (int w = 0; w < KW_THREADS / 64; w++) {
        if (w < wave) at += s_count[w];
        total += s_count[w];
    }
    for (int cand = blockIdx.x; cand < total; cand += gridDim.x) {
        __syncthreads();
        if (cand >= at && cand < at + mine) {            // the thread that counted it finds its row
            int i = at, before = r0 > 0 ? page_of(r0 - 1) : -1;
            for (int r = r0; r < r1; r++) {
                const int p = page_of(r);
                if (p >= 0 && p != before && i++ == cand) {
                    s_lead = r;
                    break;
                }
                before = p;
            }
        }
        if (tid == 0) s_first = R;
        for (int i = tid; i < P; i += KW_THREADS) s_src[i] = -1;
        __syncthreads();
        const int lead = s_lead, page = page_of(lead);
        for (int r = tid; r < R; r += KW_THREADS)
            if (page_of(r) == page) {
                atomicMin(&s_first, r);
                atomicMax(&s_src[slot[r] % P], r);       // the same slot twice: the later row
            }
        __syncthreads();
        if (s_first != lead) continue;                   // an earlier candidate has this page

        const size_t base = ((size_t)page * c.n_kv_heads + head) * (size_t)(P * hd);
        float *sp = scales + (size_t)page * c.n_kv_heads + head;
        const int n4 = hd / 4, items = P * n4;           // 16 items a thread at most
        float4 val[KVQ_MAX_PAGE * 128 / 4 / KW_THREADS];
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < KVQ_MAX_PAGE * 128 / 4 / KW_THREADS; i++) {
            const int it = tid + i * KW_THREADS;
            val[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (it < items) {
                const int src = s_src[it / n4];
                if (src >= 0) val[i] = *(const float4 *)(x + (size_t)src * ldx + head * hd + 4 * (it % n4));
            }
            const float a[4] = {val[i].x, val[i].y, val[i].z, val[i].w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (fabsf(a[e]) < INFINITY) amax = fmaxf(amax, fabsf(a[e]));
        }
        amax = vx_wave_max64(amax);
        if (lane == 0) s_amax[wave] = amax;
        __syncthreads();
        for (int w = 0; w < KW_THREADS / 64; w++) amax = fmaxf(amax, s_amax[w]);
        const float fit = amax >= 0x1p-100f ? amax / (TYPE == VXH_KVQ_INT8 ? 127.0f : 448.0f) : 0.0f;
        const bool start = s_src[0] >= 0;
        const float s_old = start ? 0.0f : *sp;
        const float sc = fmaxf(s_old, fit), inv = sc > 0.0f ? 1.0f / sc : 0.0f;
        const bool grown = sc > s_old && !start;
#pragma unroll
        for (int i = 0; i < KVQ_MAX_PAGE * 128 / 4 / KW_THREADS; i++) {
            const int it = tid + i * KW_THREADS;
            if (it < items && s_src[it / n4] >= 0) {
                const float a[4] = {val[i].x, val[i].y, val[i].z, val[i].w};
                uint32_t w = 0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    w |= (sc > 0.0f ? vx_kvq_code<TYPE>(a[e], sc, inv) : TYPE == VXH_KVQ_INT8 ? 128u : 0u) << (8 * e);
                *(uint32_t *)(s_code + (it / n4) * ldc + 4 * (it % n4)) = w;
            }
        }
        __syncthreads();
        if (tid == 0) *sp = sc;
        // lanes of 16 codes: K holds 8 dims of two tokens, V 8 tokens of two dims
        for (int u = tid; u < P * hd / 16; u += KW_THREADS) {
            const int ln = u & 63, g = ln >> 4, n = ln & 15, grp = u >> 6;
            const int t0 = grp / (hd / 32) * 32, d0 = grp % (hd / 32) * 32;
            uint8_t *dst = cache + base + (size_t)u * 16;
            int tok[16], dim[16];
            bool any = false, all = true;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                tok[e] = is_v ? t0 + ((e >> 2) & 1) * 16 + 4 * g + (e & 3) : t0 + (e >> 3) * 16 + n;
                dim[e] = is_v ? d0 + (e >> 3) * 16 + n : d0 + 8 * g + (e & 7);
                const bool in = s_src[tok[e]] >= 0;
                any |= in;
                all &= in;
            }
            if (!any && !grown) continue;
            uint4 old = make_uint4(0, 0, 0, 0);
            if (!all) old = *(const uint4 *)dst;
            uint32_t w[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int sh = 8 * (e & 3);
                uint32_t code = (w[e >> 2] >> sh) & 0xFFu;
                if (s_src[tok[e]] >= 0) code = s_code[tok[e] * ldc + dim[e]];
                else if (grown) code = vx_kvq_recode<TYPE>(vx_kvq_value<TYPE>(code), s_old, sc);
                w[e >> 2] = (w[e >> 2] & ~(0xFFu << sh)) | (code << sh);
            }
            *(uint4 *)dst = make_uint4(w[0], w[1], w[2], w[3]);
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
    int gx = 4096 / (2 * c->n_kv_heads);
    gx = gx < 1 ? 1 : gx > R ? R : gx;
    const dim3 grid(gx, c->n_kv_heads, 2);
    if (c->type == VXH_KVQ_INT8)
        vx_kvq_write_kernel<VXH_KVQ_INT8><<<grid, KW_THREADS, 0, vxh_hs(s)>>>(*c, k, ldk, v, ldv, slot, R);
    else
        vx_kvq_write_kernel<VXH_KVQ_E4M3><<<grid, KW_THREADS, 0, vxh_hs(s)>>>(*c, k, ldk, v, ldv, slot, R);
    VXH_LAUNCHED();
    return VXH_OK;
}

// ---------------------------------------------------------------------------
// Read-back: one thread per 8 dims of a row's K and V head.
// ---------------------------------------------------------------------------
template <int TYPE>
__global__ __launch_bounds__(256) void vx_kvq_read_kernel(vxh_kvq c, const int *__restrict__ slot, int R,
                                                          float *__restrict__ k, int ldk, float *__restrict__ v, int ldv)
{
    const int hd = c.head_dim, per_row = c.n_kv_heads * hd / 8;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int r = (int)(i / per_row), u = (int)(i % per_row), head = u / (hd / 8), d = u % (hd / 8) * 8;
    if (r >= R) return;
    const int sl = slot[r], page = sl / c.page, t = sl % c.page;
    if (sl < 0 || page >= c.n_pages) return;
    const size_t hp = (size_t)page * c.n_kv_heads + head, base = hp * (size_t)(c.page * hd);
    const float ks = c.ks[hp], vs = c.vs[hp];
    const uint8_t *kp = (const uint8_t *)c.k + base, *vp = (const uint8_t *)c.v + base;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        k[(size_t)r * ldk + head * hd + d + e] = vx_kvq_value<TYPE>(kp[vx_kvq_k_byte(t, d + e, hd)]) * ks;
        v[(size_t)r * ldv + head * hd + d + e] = vx_kvq_value<TYPE>(vp[vx_kvq_v_byte(t, d + e, hd)]) * vs;
    }
}

extern "C" int vxh_kvq_read(const vxh_kvq *c, const int *slot, int R, float *k, int ldk, float *v, int ldv,
                            vxh_stream s)
{
    int rc = vx_kvq_rows_check("kvq_read", c, k, ldk, v, ldv, slot, R);
    if (rc) return rc;
    const int64_t n = (int64_t)R * c->n_kv_heads * c->head_dim / 8;
    const unsigned grid = (unsigned)((n + 255) / 256);
    if (c->type == VXH_KVQ_INT8)
        vx_kvq_read_kernel<VXH_KVQ_INT8><<<grid, 256, 0, vxh_hs(s)>>>(*c, slot, R, k, ldk, v, ldv);
    else
        vx_kvq_read_kernel<VXH_KVQ_E4M3><<<grid, 256, 0, vxh_hs(s)>>>(*c, slot, R, k, ldk, v, ldv);
    VXH_LAUNCHED();
    return VXH_OK;
}
