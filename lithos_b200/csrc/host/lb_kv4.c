/* Launches of the 4-bit KV cache: rows in and out, attention of a batch. */
#include "lb_internal.h"
#include <math.h>

static int shape_ok(int n_seqs, int max_ctx, int kv_heads, int dim) {
    return n_seqs >= 1 && n_seqs < 1 << 20 && max_ctx >= 16 && max_ctx <= 1 << 20 && max_ctx % 16 == 0 && kv_heads >= 1 && kv_heads <= 32 &&
           (dim == 64 || dim == 128 || dim == 256);
}

LB_API size_t lb_kv4_bytes(int n_seqs, int max_ctx, int kv_heads, int dim) {
    return shape_ok(n_seqs, max_ctx, kv_heads, dim) ? (size_t)n_seqs * (size_t)(max_ctx / 16) * (size_t)kv_heads * (size_t)LB_KV4_BLOCK(dim) : 0;
}

/* the checks that the three calls share, and their view of cache and batch */
static int view(lb_ctx* c, const char* call, const lb_kv4_cache* k, const lb_kv4_batch* b, lb_kv4_view* v) {
    if (!c) return LB_ERR_INVALID;
    if (!k || !b || !k->data || !b->pos) return lb_fail(c, LB_ERR_INVALID, "%s: NULL cache, batch or pos", call);
    if (!shape_ok(k->n_seqs, k->max_ctx, k->kv_heads, k->dim) || k->data % 16)
        return lb_fail(c, LB_ERR_INVALID, "%s: cache of %d x %d rows, %d heads of %d (max_ctx %% 16, up to 2^20; 1..32 heads of 64, 128 or 256; 16-byte aligned)", call, k->n_seqs,
                       k->max_ctx, k->kv_heads, k->dim);
    if (b->n_reqs < 1 || b->n_reqs > LB_KV4_REQS || b->rows < 1 || b->rows > LB_KV4_ROWS || (!b->starts && b->rows != b->n_reqs))
        return lb_fail(c, LB_ERR_INVALID, "%s: %d requests, %d token rows (1..%d requests, 1..2^24 rows; without starts one row each)", call, b->n_reqs, b->rows, LB_KV4_REQS);
    if (((b->pos | b->seqs | b->starts) & 3) != 0) return lb_fail(c, LB_ERR_INVALID, "%s: arrays of 32-bit numbers must be 4-byte aligned", call);
    memset(v, 0, sizeof *v);
    v->cache = (unsigned char*)k->data;
    v->seqs = (const int32_t*)b->seqs; v->pos = (const int32_t*)b->pos; v->starts = (const int32_t*)b->starts;
    v->status = (uint32_t*)c->dev_status;
    v->n_seqs = k->n_seqs; v->max_ctx = k->max_ctx; v->HKV = k->kv_heads; v->n_reqs = b->n_reqs; v->rows = b->rows; v->max_new = b->rows;
    return LB_OK;
}

static int size_of(int type) { return type == LB_IN_F32 ? 4 : 2; }

static int rotation(lb_ctx* c, const char* call, int dim, int rot_dims, float theta, float eps, double* freq) {
    if (rot_dims < 0 || rot_dims > dim || rot_dims % 8 || (rot_dims && !(theta > 0.f && isfinite(theta))) || !(eps >= 0.f && isfinite(eps)))
        return lb_fail(c, LB_ERR_INVALID, "%s: rot_dims %d of %d (a multiple of 8), theta %g, eps %g", call, rot_dims, dim, (double)theta, (double)eps);
    for (int i = 0; i < rot_dims / 2; i++) freq[i] = exp2(-log2((double)theta) * (double)i / (double)(rot_dims / 2));
    return LB_OK;
}

/* Rows of a CTA: as many as its 256 threads take at a time (D / 8 threads for a key or value vector), more where that would make more than four CTAs an SM */
static unsigned rows_grid(const lb_ctx* c, lb_kv4_rows_params* p) {
    const int units = 256 / (p->D / 8), per_row = 2 * p->b.HKV, fill = per_row < units ? units / per_row : 1, even = (p->b.rows + 4 * c->sm_count - 1) / (4 * c->sm_count);
    p->chunk = even > fill ? even : fill;
    return (unsigned)((p->b.rows + p->chunk - 1) / p->chunk);
}

static int by_dim(int dim, int k64, int k128, int k256) { return dim == 64 ? k64 : dim == 128 ? k128 : k256; }

LB_API int lb_kv4_append(lb_ctx* c, const lb_kv4_cache* cache, const lb_kv4_batch* batch, uint64_t k, uint64_t v, int64_t stride, int type, uint64_t k_norm_w, int rot_dims,
                         float rope_theta, float eps) {
    lb_kv4_rows_params p;
    memset(&p, 0, sizeof p);
    LB_TRY(view(c, "lb_kv4_append", cache, batch, &p.b));
    const int64_t width = (int64_t)cache->kv_heads * cache->dim;
    if (stride == 0) stride = width;
    if (!k || !v || type < 0 || type > 2 || (k | v) % size_of(type) || k_norm_w % 2 || stride < width)
        return lb_fail(c, LB_ERR_INVALID, "lb_kv4_append: k, v of an element type (0..2), aligned to it, rows at least kv_heads * dim apart");
    LB_TRY(rotation(c, "lb_kv4_append", cache->dim, rot_dims, rope_theta, eps, p.freq));
    p.k = (const void*)k; p.v = (const void*)v; p.norm_w = (const uint16_t*)k_norm_w;
    p.stride = stride; p.D = cache->dim; p.type = type; p.rot_dims = rot_dims; p.eps = (double)eps;
    p.wide = ((k | v | (uint64_t)stride * (uint64_t)size_of(type)) & 15) == 0;
    void* params[] = {&p};
    return lb_launch(c, by_dim(cache->dim, LBK_kv4_append_64, LBK_kv4_append_128, LBK_kv4_append_256), rows_grid(c, &p), 1, 1, 256, 0, params, 1);
}

LB_API int lb_kv4_read(lb_ctx* c, const lb_kv4_cache* cache, const lb_kv4_batch* batch, uint64_t k_out, uint64_t v_out, int type) {
    lb_kv4_rows_params p;
    memset(&p, 0, sizeof p);
    LB_TRY(view(c, "lb_kv4_read", cache, batch, &p.b));
    if (!k_out || !v_out || type < 0 || type > 2 || (k_out | v_out) % size_of(type)) return lb_fail(c, LB_ERR_INVALID, "lb_kv4_read: k_out, v_out of an element type (0..2), aligned to it");
    p.k = (const void*)k_out; p.v = (const void*)v_out;
    p.D = cache->dim; p.type = type;
    p.wide = ((k_out | v_out) & 15) == 0;
    void* params[] = {&p};
    return lb_launch(c, by_dim(cache->dim, LBK_kv4_read_64, LBK_kv4_read_128, LBK_kv4_read_256), rows_grid(c, &p), 1, 1, 256, 0, params, 1);
}

LB_API int lb_kv4_attention(lb_ctx* c, const lb_kv4_cache* cache, const lb_kv4_batch* batch, uint64_t q, uint64_t gate, int64_t row_stride, int64_t head_stride, int type,
                            uint64_t q_norm_w, uint64_t out, int n_heads, int max_new, int rot_dims, float rope_theta, float eps) {
    lb_kv4_attn_params p;
    memset(&p, 0, sizeof p);
    LB_TRY(view(c, "lb_kv4_attention", cache, batch, &p.b));
    const int D = cache->dim, HKV = cache->kv_heads;
    if (n_heads < HKV || n_heads % HKV || n_heads / HKV > 16) return lb_fail(c, LB_ERR_INVALID, "lb_kv4_attention: %d heads over %d (1 to 16 each)", n_heads, HKV);
    if (max_new < 1 || max_new > LB_KV4_NEW) return lb_fail(c, LB_ERR_INVALID, "lb_kv4_attention: max_new %d (1..%d)", max_new, LB_KV4_NEW);
    if (head_stride == 0) head_stride = D;
    if (row_stride == 0) row_stride = n_heads * head_stride;
    if (!q || !out || type < 0 || type > 2 || (q | gate) % size_of(type) || (q_norm_w | out) % 2 || head_stride < D || row_stride < 0)
        return lb_fail(c, LB_ERR_INVALID, "lb_kv4_attention: q, gate of an element type (0..2), aligned to it, heads at least dim apart; out");
    LB_TRY(rotation(c, "lb_kv4_attention", D, rot_dims, rope_theta, eps, p.freq));
    const int G = n_heads / HKV, sets = (max_new * G + LB_KV4_COLS - 1) / LB_KV4_COLS;
    p.b.max_new = max_new;
    p.q = (const void*)q; p.gate = (const void*)gate; p.norm_w = (const uint16_t*)q_norm_w; p.out = (uint16_t*)out;
    p.records = (float*)c->kv4_records; p.joins = (lb_kv4_join*)c->kv4_joins;
    p.row_stride = row_stride; p.head_stride = head_stride;
    p.HQ = n_heads; p.type = type; p.rot_dims = rot_dims; p.eps = eps;
    p.wide = ((q | gate | (uint64_t)row_stride * (uint64_t)size_of(type) | (uint64_t)head_stride * (uint64_t)size_of(type)) & 15) == 0;
    p.out_wide = out % 16 == 0;
    /* full sequences' items: places in the kernel's line of work, which it counts in 32 bits; no more CTAs than they have work for */
    const int64_t items = (int64_t)batch->n_reqs * HKV * sets, tiles = (cache->max_ctx + LB_KV4_TILE(D) - 1) / LB_KV4_TILE(D);
    if (items * (LB_KV4_STEP * tiles + LB_KV4_ITEM) > UINT32_MAX)
        return lb_fail(c, LB_ERR_INVALID, "lb_kv4_attention: %d requests of up to %d rows, %d KV heads, %d columns: more work than a call can count", batch->n_reqs, cache->max_ctx, HKV, max_new * G);
    const int64_t most = items * (tiles + LB_KV4_ITEM / LB_KV4_STEP + 1);
    int ctas = c->sm_count * LB_KV4_CTAS < LB_KV4_MAX_CTAS ? c->sm_count * LB_KV4_CTAS : LB_KV4_MAX_CTAS;
    if (ctas > most) ctas = (int)most;
    void* params[] = {&p, &ctas};
    LB_TRY(lb_launch(c, by_dim(D, LBK_kv4_attn_64, LBK_kv4_attn_128, LBK_kv4_attn_256), (unsigned)ctas, 1, 1, 256,
                     LB_KV4_SMEM, params, 1));
    return lb_launch(c, by_dim(D, LBK_kv4_merge_64, LBK_kv4_merge_128, LBK_kv4_merge_256), 2u * (unsigned)c->sm_count, 1, 1, 256, 0, params, 1);
}
