// Drafted tokens held against the target's probabilities, with given uniform numbers.
//   p = softmax(logits / T) over the whole vocabulary or the top_k largest, q the draft's probabilities (or 1 at the draft).
//   Draft x of a row stands while  u q(x) < p(x).  The first row of a request that does not stand, or its last row, which has no draft, gives the token: the
//   first one whose cumulative weight exceeds u' times their sum, the weights being max(p - q, 0) (at the last row p).
// What a token's choice depends on is computed in 64 bits: a border between two of 250 000 tokens lies within 2^-24 of some number often enough that 32 bits would pick a neighbour
// in one draw of a hundred.  Whether a draft stands has a single border; there the sum of a row is one of 32-bit exponentials in 64 bits (2^-24 of it).
// Two launches: every row by a cluster of up to 8 CTAs, then every request.  The first reads the logits once and is bound by that; the second reads one row of each request
// again, mostly from L2, and of q the row of a draft that fell.
#include <cooperative_groups.h>

#include "common.cuh"
#include "params.h"
namespace cg = cooperative_groups;

#define VD_THREADS 512
#define VD_WARPS (VD_THREADS / 32)
#define VD_LOG2E 1.4426950408889634

struct vd_place { int covered, last; }; // the row belongs to a request; it is the request's last one

// every thread of the CTA gets the answer; requests that name rows that are not there are not a row's
__device__ __forceinline__ vd_place vd_find(const lb_vd_params& p, int row) {
    int in = 0, last = 0;
    for (int r = threadIdx.x; r < p.n_reqs; r += blockDim.x) {
        const int a = p.starts[r], b = p.starts[r + 1];
        if (a < 0 || b > p.rows || row < a || row >= b) continue;
        in = 1;
        last |= row == b - 1;
    }
    vd_place v;
    v.covered = __syncthreads_or(in);
    v.last = __syncthreads_or(last);
    return v;
}
__device__ __forceinline__ bool vd_better(float v, int i, float bv, int bi) { return v > bv || (v == bv && i < bi); }

// exp((l - max) / T) in 64 bits; an infinite maximum leaves those that share it, -infinity and NaN count as no logit
__device__ __forceinline__ double vd_exp(float l, float max, double inv_t) { return !(l > -INFINITY) ? 0.0 : l == max ? 1.0 : l < max ? exp(((double)l - (double)max) * inv_t) : 0.0; }

// Whether the row's draft stands, and the target's probability of it (from thread 0).  px: that probability
__device__ __forceinline__ void vd_decide(const lb_vd_params& p, int row, bool last, double px, lb_vd_row st) {
    const int x = p.drafts[row];
    const bool there = !last && x >= 0 && x < p.V;
    if (!there) px = 0.0;
    st.stands = 0;
    if (there) {
        double q = 1.0;
        if (p.temperature > 0.0 && p.probs) q = (double)p.probs[(size_t)row * p.V + x];
        st.stands = p.temperature > 0.0 ? (double)p.u_accept[row] * q < px : px > 0.0;
    }
    p.stat[row] = st;
    if (p.p_out) p.p_out[row] = (float)px;
}

// Rows over the whole vocabulary: maximum, its first index, sum of exponentials.  grid (rows, cluster)
extern "C" __global__ void __launch_bounds__(VD_THREADS) vd_rows(const __grid_constant__ lb_vd_params p) {
    __shared__ float sm[VD_WARPS + LB_VD_CLUSTER];
    __shared__ int si[VD_WARPS + LB_VD_CLUSTER];
    __shared__ double ss[VD_WARPS + LB_VD_CLUSTER];
    cg::cluster_group cluster = cg::this_cluster();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, row = blockIdx.x, C = gridDim.y, rank = blockIdx.y;
    pdl_wait();
    const vd_place at = vd_find(p, row);
    if (!at.covered) return; // the same for the whole cluster
    cluster.barrier_arrive(); // waited for before the first word to another CTA
    const float* x = p.logits + (size_t)row * p.V;
    const int per = (((p.V + C - 1) / C) + 3) & ~3, a = min(p.V, rank * per), b = min(p.V, a + per);
    const float k = p.temperature > 0.0 ? (float)(VD_LOG2E / p.temperature) : 0.f;
    float m = -INFINITY, sum = 0.f;
    int best = 0x7fffffff;
    auto take = [&](const float (&v)[8], const int (&id)[8]) { // index order within a thread
        float mx = m;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (v[j] > mx) { mx = v[j]; best = id[j]; }
        if (mx > m) {
            sum *= exp2f((m - mx) * k);
            m = mx;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += v[j] == m ? 1.f : v[j] < m ? exp2f((v[j] - m) * k) : 0.f;
    };
    if ((((size_t)x + 4 * (size_t)a) & 15) == 0) {
        for (int i0 = a + 4 * t; i0 < b; i0 += 8 * VD_THREADS) {
            float v[8];
            int id[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = i0 + 4 * h * VD_THREADS;
                float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (i + 3 < b) f = __ldg(reinterpret_cast<const float4*>(x + i));
                else {
                    if (i < b) f.x = x[i];
                    if (i + 1 < b) f.y = x[i + 1];
                    if (i + 2 < b) f.z = x[i + 2];
                }
                v[4 * h] = f.x; v[4 * h + 1] = f.y; v[4 * h + 2] = f.z; v[4 * h + 3] = f.w;
#pragma unroll
                for (int j = 0; j < 4; ++j) id[4 * h + j] = i + j;
            }
            take(v, id);
        }
    } else {
        for (int i0 = a + t; i0 < b; i0 += 8 * VD_THREADS) {
            float v[8];
            int id[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                id[j] = i0 + j * VD_THREADS;
                v[j] = id[j] < b ? x[id[j]] : -INFINITY;
            }
            take(v, id);
        }
    }
    // the CTA's, then the cluster's: maxima first, then the sums brought to it
    float M = m;
    int I = best;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, M, o);
        const int oi = __shfl_xor_sync(0xffffffffu, I, o);
        if (vd_better(ov, oi, M, I)) { M = ov; I = oi; }
    }
    if (lane == 0) { sm[warp] = M; si[warp] = I; }
    __syncthreads();
    M = sm[0];
    I = si[0];
    for (int w = 1; w < VD_WARPS; ++w)
        if (vd_better(sm[w], si[w], M, I)) { M = sm[w]; I = si[w]; }
    double S = sum > 0.f ? (double)sum * (double)(m == M ? 1.f : exp2f((m - M) * k)) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
    if (lane == 0) ss[warp] = S;
    __syncthreads();
    cluster.barrier_wait();
    if (t == 0) {
        S = 0.0;
        for (int w = 0; w < VD_WARPS; ++w) S += ss[w];
        *cluster.map_shared_rank(&sm[VD_WARPS + rank], 0) = M;
        *cluster.map_shared_rank(&si[VD_WARPS + rank], 0) = I;
        *cluster.map_shared_rank(&ss[VD_WARPS + rank], 0) = S;
    }
    cluster.sync();
    if (rank == 0 && t == 0) {
        M = sm[VD_WARPS];
        I = si[VD_WARPS];
        for (int w = 1; w < C; ++w)
            if (vd_better(sm[VD_WARPS + w], si[VD_WARPS + w], M, I)) { M = sm[VD_WARPS + w]; I = si[VD_WARPS + w]; }
        S = 0.0;
        for (int w = 0; w < C; ++w) {
            const float o = sm[VD_WARPS + w];
            if (ss[VD_WARPS + w] > 0.0) S += ss[VD_WARPS + w] * (o == M ? 1.0 : exp2(((double)o - (double)M) * (double)k));
        }
        lb_vd_row st = {S, M, I == 0x7fffffff ? 0 : I, 0, 0};
        const int d = p.drafts[row];
        double px = 0.0;
        if (d >= 0 && d < p.V) px = p.temperature > 0.0 ? (S > 0.0 ? vd_exp(x[d], M, 1.0 / p.temperature) / S : 0.0) : (d == st.best && M > -INFINITY ? 1.0 : 0.0);
        vd_decide(p, row, at.last, px, st);
    }
}

// ---- rows over the top_k largest ------------------------------------------------------------------------------------------------------------
#define VT_THREADS 1024
#define VT_EACH 32   // logits a thread holds
#define VT_CAND 1024 // candidates that are sorted at once
// a float's bits in an order that unsigned numbers have; 0 stands for -infinity and NaN, which are no candidates
__device__ __forceinline__ uint32_t vt_key(float v) {
    if (!(v > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v); // -0 = 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float vt_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// VT_CAND numbers in shared memory, descending
__device__ __forceinline__ void vt_sort(unsigned long long* s) {
    const int t = threadIdx.x;
    unsigned long long v = s[t];
    for (int size = 2; size <= VT_CAND; size <<= 1)
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            unsigned long long o;
            if (stride >= 32) {
                __syncthreads();
                s[t] = v;
                __syncthreads();
                o = s[t ^ stride];
            } else o = __shfl_xor_sync(0xffffffffu, v, stride);
            const bool down = (t & size) == 0, lower = (t & stride) == 0; // this place keeps the larger one
            v = (down == lower) == (v > o) ? v : o;
        }
    __syncthreads();
    s[t] = v;
    __syncthreads();
}

// The rows' top_k candidates in order (larger logit, then smaller index), as lb_sample_topk takes them.  A thread holds VT_EACH logits; the k-th largest of the threads' maxima
// bounds the k-th largest from below, and what reaches it is sorted: about k.  Where more than VT_CAND reach it (many equal ones, or a few threads with all of the large ones) the
// exact bound is found by halving, first of the value, then of the index among the equal ones.  grid (rows, cluster)
extern "C" __global__ void __launch_bounds__(VT_THREADS) vd_rows_topk(const __grid_constant__ lb_vd_params p) {
    __shared__ unsigned long long cand[VT_CAND];
    __shared__ unsigned long long from[LB_VD_CLUSTER * LB_VD_TOPK]; // the cluster's lists, at its first CTA
    __shared__ int n_cand;
    cg::cluster_group cluster = cg::this_cluster();
    const int t = threadIdx.x, row = blockIdx.x, C = gridDim.y, rank = blockIdx.y, K = p.top_k;
    pdl_wait();
    const vd_place at = vd_find(p, row);
    if (!at.covered) return;
    cluster.barrier_arrive();
    const float* x = p.logits + (size_t)row * p.V;
    const int per = (p.V + C - 1) / C, a = min(p.V, rank * per), b = min(p.V, a + per);
    cand[t] = 0ull;
    __syncthreads();
    for (int base = a; base < b; base += VT_THREADS * VT_EACH) { // the list so far is in cand[0 .. K)
        uint32_t key[VT_EACH], top = 0u;
#pragma unroll
        for (int j = 0; j < VT_EACH; ++j) {
            const int i = base + j * VT_THREADS + t;
            key[j] = i < b ? vt_key(__ldg(x + i)) : 0u;
        }
#pragma unroll
        for (int j = 0; j < VT_EACH; ++j) top = max(top, key[j]);
        // the largest bound that K of the threads' maxima reach (0: fewer than K do, all candidates count)
        uint32_t bound = 0u;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t trial = bound | 1u << bit;
            if (__syncthreads_count(top >= trial) >= K) bound = trial;
        }
        const uint32_t before = (uint32_t)(cand[K - 1] >> 32); // nothing below the list's end comes in
        if (before > bound) bound = before;
        if (bound == 0u) bound = 1u;
        uint32_t last = 0xffffffffu; // of those equal to the bound: indices up to this one
        int mine = 0;
#pragma unroll
        for (int j = 0; j < VT_EACH; ++j) mine += key[j] >= bound;
        if (t == 0) n_cand = K;
        __syncthreads();
        if (mine) atomicAdd(&n_cand, mine);
        __syncthreads();
        if (n_cand > VT_CAND) {
            auto count = [&](auto f) { // over all of the CTA's logits
                int n = 0;
#pragma unroll
                for (int j = 0; j < VT_EACH; ++j) n += f(key[j], (uint32_t)(base + j * VT_THREADS + t));
                __syncthreads();
                if (t == 0) n_cand = 0;
                __syncthreads();
                n = __reduce_add_sync(0xffffffffu, n);
                if ((t & 31) == 0 && n) atomicAdd(&n_cand, n);
                __syncthreads();
                return n_cand;
            };
            bound = 0u;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t trial = bound | 1u << bit;
                if (count([&](uint32_t k, uint32_t) { return k >= trial; }) >= K) bound = trial;
            }
            const int above = count([&](uint32_t k, uint32_t) { return k > bound; });
            last = 0u; // the smallest index with K - above equal ones up to it
            for (int bit = 30; bit >= 0; --bit) {
                const uint32_t trial = last | 1u << bit;
                if (count([&](uint32_t k, uint32_t i) { return k == bound && i < trial; }) < K - above) last = trial;
            }
        }
        __syncthreads();
        if (t >= K) cand[t] = 0ull;
        if (t == 0) n_cand = K;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < VT_EACH; ++j) {
            const uint32_t i = (uint32_t)(base + j * VT_THREADS + t);
            if (key[j] > bound || (key[j] == bound && i <= last)) {
                const int o = atomicAdd(&n_cand, 1);
                if (o < VT_CAND) cand[o] = (unsigned long long)key[j] << 32 | (0xffffffffu - i);
            }
        }
        __syncthreads();
        vt_sort(cand);
    }
    cluster.barrier_wait();
    if (t < K) cluster.map_shared_rank(from, 0)[rank * K + t] = cand[t];
    cluster.sync();
    if (rank) return;
    cand[t] = t < C * K ? from[t] : 0ull;
    __syncthreads();
    if (C > 1) vt_sort(cand);
    double* e = reinterpret_cast<double*>(from);
    const float top = cand[0] ? vt_value((uint32_t)(cand[0] >> 32)) : -INFINITY;
    if (t < K) {
        const float v = vt_value((uint32_t)(cand[t] >> 32));
        e[t] = cand[t] ? vd_exp(v, top, 1.0 / p.temperature) : 0.0;
        p.list_val[(size_t)row * LB_VD_TOPK + t] = v;
        p.list_idx[(size_t)row * LB_VD_TOPK + t] = (int)(0xffffffffu - (uint32_t)cand[t]);
    }
    __syncthreads();
    if (t == 0) {
        lb_vd_row st = {0.0, top, cand[0] ? (int)(0xffffffffu - (uint32_t)cand[0]) : 0, 0, 0};
        double px = 0.0;
        const int d = p.drafts[row];
        for (; st.n < K && cand[st.n]; ++st.n) {
            st.z += e[st.n];
            if ((int)(0xffffffffu - (uint32_t)cand[st.n]) == d) px = e[st.n];
        }
        vd_decide(p, row, at.last, st.z > 0.0 ? px / st.z : 0.0, st);
    }
}

// ---- requests ------------------------------------------------------------------------------------------------------------------------------
// The request's row that gives its token (every thread gets it); -1: it has no rows
__device__ __forceinline__ int vd_stop(const lb_vd_params& p, int r, int& first, int& last) {
    __shared__ int s_at;
    first = p.starts[r];
    const int end = p.starts[r + 1];
    last = end - 1;
    if (first < 0 || end > p.rows || end <= first) {
        if (threadIdx.x == 0) {
            if (end != first) atomicExch(p.status, LB_DEV_BATCH);
            p.accepted[r] = -1;
        }
        return -1;
    }
    if (threadIdx.x == 0) s_at = last;
    __syncthreads();
    for (int i = first + threadIdx.x; i < last; i += blockDim.x)
        if (!p.stat[i].stands) {
            atomicMin(&s_at, i);
            break;
        }
    __syncthreads();
    return s_at;
}
__device__ __forceinline__ void vd_write(const lb_vd_params& p, int r, int first, int last, int at, int token) {
    for (int i = first + threadIdx.x; i <= last; i += blockDim.x) p.tokens[i] = i < at ? p.drafts[i] : i == at ? token : -1;
    if (threadIdx.x == 0) p.accepted[r] = at - first;
}

// Greedy, or from the rows' lists: one CTA of LB_VD_TOPK threads per request
extern "C" __global__ void __launch_bounds__(LB_VD_TOPK) vd_pick_short(const __grid_constant__ lb_vd_params p) {
    __shared__ double w[LB_VD_TOPK];
    __shared__ int token;
    const int t = threadIdx.x, r = blockIdx.x;
    pdl_wait();
    int first, last;
    const int at = vd_stop(p, r, first, last);
    if (at < 0) return;
    const lb_vd_row st = p.stat[at];
    if (t == 0) token = st.best;
    if (p.temperature > 0.0) {
        const int idx = t < st.n ? p.list_idx[(size_t)at * LB_VD_TOPK + t] : -1;
        double e = 0.0, left = 0.0;
        if (t < st.n) {
            e = vd_exp(p.list_val[(size_t)at * LB_VD_TOPK + t], st.max, 1.0 / p.temperature) / st.z;
            left = e;
            if (at < last) {
                const double q = p.probs ? (double)p.probs[(size_t)at * p.V + idx] : idx == p.drafts[at] ? 1.0 : 0.0;
                left = q > 0.0 ? fmax(e - q, 0.0) : e;
            }
        }
        if (!__syncthreads_or(left > 0.0)) left = e; // rounding left nothing
        w[t] = left;
        __syncthreads();
        if (t == 0 && st.n) {
            double total = 0.0, sum = 0.0;
            for (int i = 0; i < st.n; ++i) total += w[i];
            const double goal = (double)p.u_pick[r] * total;
            int i = 0, pick = 0;
            for (; i < st.n; ++i) {
                sum += w[i];
                if (w[i] > 0.0) pick = i;
                if (sum > goal) break;
            }
            token = p.list_idx[(size_t)at * LB_VD_TOPK + pick];
        }
    }
    __syncthreads();
    vd_write(p, r, first, last, at, token);
}

// From the whole vocabulary: a cluster per request, its CTAs and their warps taking neighbouring ranges in index order.  grid (requests, cluster)
#define VP_THREADS 1024
#define VP_WARPS 32
extern "C" __global__ void __launch_bounds__(VP_THREADS) vd_pick(const __grid_constant__ lb_vd_params p) {
    __shared__ double part[2];           // this CTA's sum: of the exponentials, of the weights
    __shared__ double ws[VP_WARPS];
    __shared__ int s_token;
    cg::cluster_group cluster = cg::this_cluster();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, r = blockIdx.x, C = gridDim.y, rank = blockIdx.y;
    pdl_wait();
    int first, last;
    const int at = vd_stop(p, r, first, last);
    if (at < 0) return;
    const lb_vd_row st = p.stat[at];
    const float* x = p.logits + (size_t)at * p.V;
    const bool inner = at < last;
    const float* q = inner && p.probs ? p.probs + (size_t)at * p.V : nullptr;
    const int gone = inner && !p.probs ? p.drafts[at] : -1; // a certain draft
    const double inv_t = 1.0 / p.temperature;
    const int per = (p.V + C * VP_WARPS - 1) / (C * VP_WARPS), a = min(p.V, (rank * VP_WARPS + warp) * per), b = min(p.V, a + per); // this warp's range
    auto all = [&](double v, int which) { // sum over the CTA into part[which] (ws: the warps'), then over the cluster in its order
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) ws[warp] = v;
        __syncthreads();
        if (t == 0) {
            double s = 0.0;
            for (int w = 0; w < VP_WARPS; ++w) s += ws[w];
            part[which] = s;
        }
        cluster.sync();
        double s = 0.0;
        for (int c = 0; c < C; ++c) s += *cluster.map_shared_rank(&part[which], c);
        return s;
    };
    double z = 1.0;
    if (q) {
        double s = 0.0;
        for (int i = a + lane; i < b; i += 32) s += vd_exp(x[i], st.max, inv_t);
        z = 1.0 / all(s, 0);
    }
    bool rest = inner;
    auto weight = [&](int i) {
        const double e = vd_exp(x[i], st.max, inv_t) * z;
        if (!rest) return e;
        if (!q) return i == gone ? 0.0 : e;
        const float o = q[i];
        return o > 0.f ? fmax(e - (double)o, 0.0) : e;
    };
    double s = 0.0;
    for (int i = a + lane; i < b; i += 32) s += weight(i);
    double total = all(s, 1);
    if (rest && !(total > 0.0)) { // rounding left nothing: from p itself
        rest = false;
        cluster.sync(); // the sums have been read
        s = 0.0;
        for (int i = a + lane; i < b; i += 32) s += weight(i);
        total = all(s, 1);
    }
    const double goal = (double)p.u_pick[r] * total;
    double before = 0.0;
    int owner = 0; // the CTA whose range the goal lies in: the last one with weight where rounding has left it behind them all
    for (int c = 0; c < C; ++c) {
        const double v = *cluster.map_shared_rank(&part[1], c);
        if (!(v > 0.0)) continue;
        double sum = 0.0;
        for (int k = 0; k < c; ++k) sum += *cluster.map_shared_rank(&part[1], k);
        owner = c;
        before = sum;
        if (sum + v > goal) break;
    }
    cluster.sync(); // nobody leaves while its sums are read
    if (rank != owner) return;
    int w0 = 0;
    double sum = before, base = before;
    for (int w = 0; w < VP_WARPS; ++w) {
        if (!(ws[w] > 0.0)) continue;
        w0 = w;
        base = sum;
        sum += ws[w];
        if (sum > goal) break;
    }
    // the range of warp w0, one value a thread, 1024 at a time
    if (t == 0) s_token = -1;
    __syncthreads();
    const int lo = min(p.V, (rank * VP_WARPS + w0) * per), hi = min(p.V, lo + per);
    int fallback = st.best; // the last token with weight
    for (int i0 = lo; i0 < hi; i0 += VP_THREADS) {
        const int i = i0 + t;
        const double v = i < hi ? weight(i) : 0.0;
        double run = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double u = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += u;
        }
        __syncthreads(); // ws has been read
        if (lane == 31) ws[warp] = run;
        __syncthreads();
        double add = base;
        for (int w = 0; w < warp; ++w) add += ws[w];
        const uint32_t hit = __ballot_sync(0xffffffffu, v > 0.0 && add + run > goal), some = __ballot_sync(0xffffffffu, v > 0.0);
        __shared__ int s_hit[VP_WARPS], s_some[VP_WARPS];
        if (lane == 0) {
            s_hit[warp] = hit ? __ffs(hit) - 1 : -1;
            s_some[warp] = some ? 31 - __clz(some) : -1;
        }
        __syncthreads();
        if (t == 0)
            for (int w = 0; w < VP_WARPS; ++w) {
                if (s_some[w] >= 0) fallback = i0 + 32 * w + s_some[w];
                if (s_hit[w] >= 0) {
                    s_token = i0 + 32 * w + s_hit[w];
                    break;
                }
            }
        for (int w = 0; w < VP_WARPS; ++w) base += ws[w];
        __syncthreads();
        if (s_token >= 0) break;
    }
    if (t == 0 && s_token < 0) s_token = fallback;
    __syncthreads();
    vd_write(p, r, first, last, at, s_token);
}
