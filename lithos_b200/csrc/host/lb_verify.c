/* Launches of lb_verify_drafts. */
#include "lb_internal.h"
#include <math.h>

/* CTAs of a cluster for each of n rows or requests: 4096 logits each or more, and the number that fills whole waves of `slots` CTAs best */
static unsigned cluster_of(int n, int vocab, int slots) {
    int best = 1;
    double least = 1e30;
    for (int k = 1; k <= LB_VD_CLUSTER && (k == 1 || vocab / k >= 4096); k++) {
        const double time = (double)((n * k + slots - 1) / slots) * (1.0 / k + 0.06); /* waves of a share and of what a CTA costs besides */
        if (time < least) { least = time; best = k; }
    }
    return (unsigned)best;
}

LB_API int lb_verify_drafts(lb_ctx* c, uint64_t logits, int vocab, uint64_t starts, int n_reqs, int rows, uint64_t drafts, uint64_t draft_probs, uint64_t u_accept, uint64_t u_pick,
                            uint64_t tokens, uint64_t accepted, double temperature, int top_k, uint64_t p_out) {
    if (!c) return LB_ERR_INVALID;
    if (!logits || !starts || !drafts || !u_accept || !u_pick || !tokens || !accepted || ((logits | starts | drafts | draft_probs | u_accept | u_pick | tokens | accepted | p_out) & 3))
        return lb_fail(c, LB_ERR_INVALID, "lb_verify_drafts: NULL or unaligned array");
    if (vocab < 1 || vocab > 1 << 24 || n_reqs < 1 || n_reqs > LB_VD_REQS || rows < 1 || rows > LB_VD_ROWS)
        return lb_fail(c, LB_ERR_INVALID, "lb_verify_drafts: %d requests, %d rows of %d (1..%d requests, 1..%d rows, up to 2^24 logits)", n_reqs, rows, vocab, LB_VD_REQS, LB_VD_ROWS);
    if (!isfinite(temperature) || (temperature > 0 && (temperature < 1e-6 || temperature > 1e6)) || top_k < 0 || top_k > LB_VD_TOPK)
        return lb_fail(c, LB_ERR_INVALID, "lb_verify_drafts: temperature %g (up to 0, or 1e-6..1e6), top_k %d (0..%d)", temperature, top_k, LB_VD_TOPK);
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
    const int kernel = p.top_k ? LBK_vd_rows_topk : temperature > 0 ? LBK_vd_rows : LBK_vd_rows_greedy;
    unsigned cl = cluster_of(rows, vocab, 3 * c->sm_count);
    LB_TRY(lb_launch_cluster(c, kernel, (unsigned)rows, cl, 1, 512, 0, params, 1, cl));
    if (kernel != LBK_vd_rows) return lb_launch(c, LBK_vd_pick_short, (unsigned)n_reqs, 1, 1, 32, 0, params, 1);
    cl = cluster_of(n_reqs, vocab, 2 * c->sm_count); /* one a time on an SM; requests take one pass or two, so that two waves even out: 48 requests 88 us as 6 CTAs each, 90 as 3; but 30 requests 68 as 8 where 4 would take 62 */
    return lb_launch_cluster(c, LBK_vd_pick, (unsigned)n_reqs, cl, 1, 512, 0, params, 1, cl);
}
