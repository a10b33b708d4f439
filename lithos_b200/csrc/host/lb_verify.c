/* Launches of lb_verify_drafts. */
#include "lb_internal.h"
#include <math.h>

/* CTAs of a row or request: as many as have 4096 logits each */
static unsigned cluster_of(int vocab) {
    unsigned c = LB_VD_CLUSTER;
    while (c > 1 && vocab / (int)c < 4096) c /= 2;
    return c;
}

LB_API int lb_verify_drafts(lb_ctx* c, uint64_t logits, int vocab, uint64_t starts, int n_reqs, int rows, uint64_t drafts, uint64_t draft_probs, uint64_t u_accept, uint64_t u_pick,
                            uint64_t tokens, uint64_t accepted, double temperature, int top_k, uint64_t p_out) {
    if (!c) return LB_ERR_INVALID;
    if (!logits || !starts || !drafts || !u_accept || !u_pick || !tokens || !accepted || ((logits | starts | drafts | draft_probs | u_accept | u_pick | tokens | accepted | p_out) & 3))
        return lb_fail(c, LB_ERR_INVALID, "lb_verify_drafts: NULL or unaligned array");
    if (vocab < 1 || vocab > 1 << 24 || n_reqs < 1 || n_reqs > LB_VD_REQS || rows < 1 || rows > LB_VD_ROWS)
        return lb_fail(c, LB_ERR_INVALID, "lb_verify_drafts: %d requests, %d rows of %d (1..%d requests, 1..%d rows, up to 2^24 logits)", n_reqs, rows, vocab, LB_VD_REQS, LB_VD_ROWS);
    if (!isfinite(temperature) || top_k < 0 || top_k > LB_VD_TOPK)
        return lb_fail(c, LB_ERR_INVALID, "lb_verify_drafts: temperature %g, top_k %d (0..%d)", temperature, top_k, LB_VD_TOPK);
    lb_vd_params p;
    memset(&p, 0, sizeof p);
    p.logits = (const float*)logits; p.starts = (const int32_t*)starts; p.drafts = (const int32_t*)drafts; p.probs = (const float*)draft_probs;
    p.u_accept = (const float*)u_accept; p.u_pick = (const float*)u_pick; p.tokens = (int32_t*)tokens; p.accepted = (int32_t*)accepted; p.p_out = (float*)p_out;
    p.stat = (lb_vd_row*)c->vd_stat;
    p.list_val = (float*)(c->vd_stat + (size_t)LB_VD_ROWS * sizeof(lb_vd_row));
    p.list_idx = (int32_t*)(c->vd_stat + (size_t)LB_VD_ROWS * (sizeof(lb_vd_row) + LB_VD_TOPK * 4));
    p.status = (uint32_t*)c->dev_status;
    p.temperature = temperature; p.V = vocab; p.n_reqs = n_reqs; p.rows = rows; p.top_k = temperature > 0 ? top_k : 0;
    void* params[] = {&p};
    const unsigned cl = cluster_of(vocab);
    LB_TRY(lb_launch_cluster(c, p.top_k ? LBK_vd_rows_topk : LBK_vd_rows, (unsigned)rows, cl, 1, p.top_k ? 1024 : 512, 0, params, 1, cl));
    if (p.top_k || temperature <= 0) return lb_launch(c, LBK_vd_pick_short, (unsigned)n_reqs, 1, 1, LB_VD_TOPK, 0, params, 1);
    return lb_launch_cluster(c, LBK_vd_pick, (unsigned)n_reqs, cl, 1, 1024, 0, params, 1, cl);
}
