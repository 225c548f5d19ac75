// Attention of a ragged batch over the paged 8-bit KV cache.
#include "vxh_kvq.h"

// One wavefront per (row, head): lane l keeps a running maximum, sum and
// output over tokens l, l + 64, ..; the lanes join at the end.
template <int TYPE, int HD>
__global__ __launch_bounds__(64) void vx_attention_kvq_kernel(const float *__restrict__ q, int ldq,
                                                              const int *__restrict__ row0, const int *__restrict__ len,
                                                              int B, int max_rows, const int *__restrict__ table,
                                                              int ld_table, int n_heads, vxh_kvq c, int cap,
                                                              float *__restrict__ out, int ld_out)
{
    const int r = blockIdx.x, h = blockIdx.y, kvh = h / (n_heads / c.n_kv_heads), lane = threadIdx.x;
    int b = -1;
    for (int i = 0; i < B; i++)
        if (row0[i] <= r && r < row0[i + 1]) b = i;
    if (b < 0) return;
    const int n = min(len[b], (int)min((int64_t)ld_table * c.page, (int64_t)0x7FFFFFFF));
    int end = n - (row0[b + 1] - r) + 1;
    if (cap > 0) end = min(end, cap);
    const float *qr = q + (size_t)r * ldq + h * HD;
    float m = -INFINITY, l = 0.0f, o[HD];
#pragma unroll
    for (int d = 0; d < HD; d++) o[d] = 0.0f;
    for (int t = lane; t < end; t += 64) {
        const int page = table[(size_t)b * ld_table + t / c.page];
        if ((unsigned)page >= (unsigned)c.n_pages) continue;
        const size_t hp = (size_t)page * c.n_kv_heads + kvh, base = hp * (size_t)(c.page * HD);
        const uint8_t *kp = (const uint8_t *)c.k + base, *vp = (const uint8_t *)c.v + base;
        float s = 0.0f;
#pragma unroll 8
        for (int d = 0; d < HD; d++) s = fmaf(qr[d], vx_kvq_value<TYPE>(kp[vx_kvq_k_byte(t % c.page, d, HD)]), s);
        s *= c.ks[hp] / sqrtf((float)HD);
        const float nm = fmaxf(m, s), f = expf(m - nm), p = expf(s - nm);
        m = nm;
        l = l * f + p;
#pragma unroll
        for (int d = 0; d < HD; d++)
            o[d] = o[d] * f + p * (vx_kvq_value<TYPE>(vp[vx_kvq_v_byte(t % c.page, d, HD)]) * c.vs[hp]);
    }
    const float all = vx_wave_max64(m), f = m > -INFINITY ? expf(m - all) : 0.0f;
    l = vx_wave_sum64(l * f);
#pragma unroll
    for (int d = 0; d < HD; d++) {
        const float v = vx_wave_sum64(o[d] * f);
        if (lane == 0) out[(size_t)r * ld_out + h * HD + d] = l > 0.0f ? v / l : 0.0f;
    }
}

extern "C" size_t vxh_attention_kvq_workspace_floats(int max_rows, int n_seqs, int n_heads, int n_kv_heads,
                                                     int head_dim)
{
    return 64;
}

extern "C" int vxh_attention_kvq(const float *q, int ldq, const int *row0, const int *len, int n_seqs, int max_rows,
                                 int max_seq_rows, const int *table, int ld_table, int n_heads, const vxh_kvq *c,
                                 int cap, float *out, int ld_out, vxh_workspace *ws, vxh_stream s)
{
    if (const char *bad = vx_kvq_bad(c)) return vxh_fail(VXH_ERR_PARAM, "attention_kvq: %s", bad);
    const int w = n_heads * c->head_dim;
    if (!q || !row0 || !len || !table || !out || !ws || n_seqs < 1 || n_seqs > VXH_PAGE_MAX_SEQS || max_rows < 1 ||
        max_rows > VXH_PAGE_MAX_ROWS || max_seq_rows < 1 || ld_table < 1 || cap < 0 || n_heads < 1 ||
        n_heads % c->n_kv_heads || ldq < w || ldq % 4 || ld_out < w || ld_out % 4 || ((uintptr_t)q & 15) || ((uintptr_t)out & 15))
        return vxh_fail(VXH_ERR_PARAM, "attention_kvq: %d requests, %d rows, %d/%d heads of %d (ld %d, %d)", n_seqs,
                        max_rows, n_heads, c->n_kv_heads, c->head_dim, ldq, ld_out);
    const dim3 grid(max_rows, n_heads);
#define VX_CALL(T, HD)                                                                                                \
    vx_attention_kvq_kernel<T, HD><<<grid, 64, 0, vxh_hs(s)>>>(q, ldq, row0, len, n_seqs, max_rows, table, ld_table,  \
                                                               n_heads, *c, cap, out, ld_out)
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
