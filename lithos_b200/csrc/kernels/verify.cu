// Drafted tokens held against the target's probabilities, with given uniform numbers.
//   p = softmax(logits / T) over the whole vocabulary or the top_k largest, q the draft's probabilities (or 1 at the draft).
//   Draft x of a row stands while  u q(x) < p(x).  The first row of a request that does not stand, or its last row, which has no draft, gives the token: the
//   first one whose cumulative weight exceeds u' times their sum, the weights being max(p - q, 0) (at the last row p).
// What a token's choice depends on is computed in 64 bits (exponentials of a whole row to 2^-42): a border between two of 250 000 tokens lies within 2^-24 of some number often enough that 32 bits would pick a neighbour
// in one draw of a hundred.  Whether a draft stands has a single border; there the sum of a row is one of 32-bit exponentials, four to a 64-bit addition.  Where logits x
// under the maximum in log2 units carry it, it is off by 2^-22 for the exponential, 2^-24.5 x for its argument's factor and up to 2^-20.5 (x < 32) for the argument: 2^-19 of itself at most.
// Two launches: every row by a cluster of up to 8 CTAs, then every request.  The first reads the logits once and is bound by that where there are many rows (5 TB/s at 188 rows of
// 248 320); the second reads one row of each request again, and of q the row of a draft that fell, and is bound by the issue slots of its exponentials, 45 a logit and warp.
// us a call at a vocabulary of 248 320: 1 request with 4 drafts 19; 48 with up to 5 and the draft's probabilities 86 (37 and 49); 16 with up to 4, top 50, 28; greedy, 32 with up to
// 3 over 32 768, 7.5.
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

__device__ __forceinline__ float vd_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// a finite float as a double, by its bits (conversions run at a quarter of the rate): 0 and denormal ones come out as some number below 2^-126
__device__ __forceinline__ double vd_double(float v) {
    const uint32_t b = __float_as_uint(v);
    return __hiloint2double((((int)b >> 3) & (int)0x8fffffffu) + 0x38000000, (int)(b << 29));
}

// exp of many differences l - max in 64 bits: y = (l - max) 256 / (T ln 2) = 256 a + j + f with |f| <= 1/2, exp = 2^a 2^(j/256) e^(f ln 2 / 256), the last factor by its series, whose
// fourth term is below 2e-13.  Eight operations in 64 bits, two issue slots each; the library's exp also serves arguments that do not occur here and makes the pick twice as long.
#define VD_STEPS 256
struct vd_exps {
    double scale, less; // y = l * scale - less
    const double* table;
    float low;          // what lies below, 2^-969, adds nothing (above it a probability, 2^-24 and less of that, has an exponent); a NaN where there is no logit at all
    __device__ __forceinline__ static void fill(double* table) { // a barrier follows
        for (int i = threadIdx.x; i < VD_STEPS; i += blockDim.x) table[i] = exp2((double)i / VD_STEPS);
    }
    __device__ __forceinline__ vd_exps(const double* t, float max, double temperature) : table(t) {
        // an infinite maximum, or one so far from 0 that the type's next number is 2^15 T off: those that share it have exp = 1, the others 0
        // (up to there the rounding of `less`, a factor that all exponentials share, is within a step)
        const bool alone = max == INFINITY || fabs((double)max) > 1099511627776.0 * temperature;
        scale = alone ? 0.0 : VD_STEPS * VD_LOG2E / temperature;
        less = alone ? 0.0 : (double)max * scale;
        low = !(max > -INFINITY) ? NAN : alone ? max : __double2float_ru((double)max - 672.0 * temperature);
    }
    // N at a time, step by step: every operation waits for the one before, so others have to be under way
    template <int N>
    __device__ __forceinline__ void operator()(const float (&l)[N], double (&e)[N]) const {
        constexpr double L = 0.69314718055994530942 / VD_STEPS, magic = 6755399441055744.0; // 1.5 * 2^52: what is added to it is rounded to a whole number
        double f[N];
        int n[N];
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = fma(vd_double(l[i]), scale, -less);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const double whole = f[i] + magic;
            n[i] = __double2loint(whole);
            e[i] = whole - magic;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] -= e[i];
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = fma(f[i], L * L * L / 6.0, L * L / 2.0);
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = fma(f[i], e[i], L);
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = fma(f[i], e[i], 1.0);
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] *= table[n[i] & (VD_STEPS - 1)];
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = l[i] >= low ? __hiloint2double(__double2hiint(e[i]) + ((n[i] >> 8) << 20), __double2loint(e[i])) : 0.0; // a NaN is not
    }
};

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

// f(four logits, index of the first) over a thread's share of logits a..b-1 of x, a % 4 == 0; what lies behind b comes as -infinity
template <int THREADS, class F>
__device__ __forceinline__ void vd_each(const float* x, int a, int b, F f) {
    int i = a + 4 * threadIdx.x;
    if ((((size_t)x + 4 * (size_t)a) & 15) == 0) {
        for (; i + 12 * THREADS + 3 < b; i += 16 * THREADS) {
            float4 v[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) v[h] = __ldg(reinterpret_cast<const float4*>(x + i + 4 * h * THREADS));
#pragma unroll
            for (int h = 0; h < 4; ++h) f(v[h], i + 4 * h * THREADS);
        }
        for (; i + 3 < b; i += 4 * THREADS) f(__ldg(reinterpret_cast<const float4*>(x + i)), i);
    }
    for (; i < b; i += 4 * THREADS) {
        float4 v = make_float4(x[i], -INFINITY, -INFINITY, -INFINITY);
        if (i + 1 < b) v.y = x[i + 1];
        if (i + 2 < b) v.z = x[i + 2];
        if (i + 3 < b) v.w = x[i + 3];
        f(v, i);
    }
}

// Rows over the whole vocabulary.  Greedy: maximum and its first index; else maximum and sum of exponentials.  The sum is one of 2^(l k - c), k = log2(e) / T, against a reference c that
// only moves when an exponent would pass 2^24: a multiply-add, an exponential, an addition and a maximum per logit.  What the row's sum is in the end is told
// in exponents of 2^(max k), with c known exactly.  Where that is not good enough (a NaN among the logits, infinities, exponents beyond 2^24) the sum is taken again with
// differences from the maximum.  grid (rows, cluster)
template <bool GREEDY>
__device__ __forceinline__ void vd_rows_body(const lb_vd_params& p) {
    __shared__ float sm[VD_WARPS + LB_VD_CLUSTER];
    __shared__ int si[VD_WARPS + LB_VD_CLUSTER];
    __shared__ double ss[VD_WARPS + LB_VD_CLUSTER];
    cg::cluster_group cluster = cg::this_cluster();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, row = blockIdx.x, C = gridDim.y, rank = blockIdx.y;
    pdl_wait();
    const float* x = p.logits + (size_t)row * p.V;
    const int per = (((p.V + C - 1) / C) + 3) & ~3, a = min(p.V, rank * per), b = min(p.V, a + per);
    const float k = GREEDY ? 0.f : (float)(VD_LOG2E / p.temperature);
    float m = -INFINITY;
    double sum = 0.0, ref = 0.0; // the sum and its reference
    int best = 0x7fffffff;
    if (GREEDY) {
        vd_each<VD_THREADS>(x, a, b, [&](const float4& v, int i) {
            const float mx = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
            if (mx > m) { // the first of them: index order within a thread
                m = mx;
                best = v.x == mx ? i : v.y == mx ? i + 1 : v.z == mx ? i + 2 : i + 3;
            }
        });
    } else {
        float c = 0.f;
        vd_each<VD_THREADS>(x, a, b, [&](const float4& v, int) {
            const float mx = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
            if (mx > m) {
                const float now = fmaxf(-3.4e38f, mx * k), d = c - now;
                if (m == -INFINITY || d < -24.f) { // four of 2^24 fit fp32
                    sum *= m == -INFINITY ? 0.0 : (double)vd_exp2(d);
                    c = now;
                }
                m = mx;
            }
            sum += (double)((vd_exp2(fmaf(v.x, k, -c)) + vd_exp2(fmaf(v.y, k, -c))) + (vd_exp2(fmaf(v.z, k, -c)) + vd_exp2(fmaf(v.w, k, -c))));
        });
        ref = (double)c;
        if (!(sum < INFINITY) || !(fabsf(m * k) < 16777216.f)) { // NaN logits; infinite ones, of which only those that share the maximum count; a c that is known to whole numbers only
            sum = 0.0;
            ref = (double)m * (double)k;
            auto one = [&](float l) { return l == m ? 1.f : l < m ? vd_exp2((l - m) * k) : 0.f; };
            vd_each<VD_THREADS>(x, a, b, [&](const float4& v, int) { sum += (double)((one(v.x) + one(v.y)) + (one(v.z) + one(v.w))); });
        }
        if (m == -INFINITY) sum = 0.0;
    }
    const vd_place at = vd_find(p, row);
    if (!at.covered) return; // the same for the whole cluster
    cluster.barrier_arrive(); // waited for before the first word to another CTA
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
    M = sm[lane & (VD_WARPS - 1)];
    I = si[lane & (VD_WARPS - 1)];
#pragma unroll
    for (int o = VD_WARPS / 2; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, M, o);
        const int oi = __shfl_xor_sync(0xffffffffu, I, o);
        if (vd_better(ov, oi, M, I)) { M = ov; I = oi; }
    }
    double S = 0.0;
    if (!GREEDY) {
        if (sum > 0.0) S = M == INFINITY ? (m == M ? sum : 0.0) : sum * exp2(ref - (double)M * (double)k);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) S += __shfl_xor_sync(0xffffffffu, S, o);
        if (lane == 0) ss[warp] = S;
        __syncthreads();
    }
    cluster.barrier_wait();
    if (t == 0) {
        S = 0.0;
        for (int w = 0; w < VD_WARPS && !GREEDY; ++w) S += ss[w];
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
        for (int w = 0; w < C && !GREEDY; ++w) {
            const float o = sm[VD_WARPS + w];
            if (ss[VD_WARPS + w] > 0.0) S += ss[VD_WARPS + w] * (o == M ? 1.0 : exp2(((double)o - (double)M) * (double)k));
        }
        const lb_vd_row st = {S, M, I == 0x7fffffff ? 0 : I, 0, 0};
        const int d = p.drafts[row];
        double px = 0.0;
        if (d >= 0 && d < p.V) px = GREEDY ? (d == st.best && M > -INFINITY ? 1.0 : 0.0) : S > 0.0 ? vd_exp(x[d], M, 1.0 / p.temperature) / S : 0.0;
        vd_decide(p, row, at.last, px, st);
    }
}
extern "C" __global__ void __launch_bounds__(VD_THREADS, 3) vd_rows(const __grid_constant__ lb_vd_params p) { vd_rows_body<false>(p); }
extern "C" __global__ void __launch_bounds__(VD_THREADS, 3) vd_rows_greedy(const __grid_constant__ lb_vd_params p) { vd_rows_body<true>(p); }

// ---- rows over the top_k largest ------------------------------------------------------------------------------------------------------------
#define VT_THREADS 512
#define VT_CAND 512   // candidates that are ranked at once
#define VT_GROUPS 256 // groups of threads whose maxima give the bound
// a float's bits in an order that unsigned numbers have; what is not above 0 stands for -infinity and NaN, which are no candidates
__device__ __forceinline__ uint32_t vt_key(float v) {
    const uint32_t b = __float_as_uint(fmaxf(v, -INFINITY) + 0.f); // -0 = 0
    return (b ^ (uint32_t)((int)b >> 31 | (int)0x80000000u)) - 0x007fffffu;
}
__device__ __forceinline__ float vt_value(uint32_t key) {
    key += 0x007fffffu;
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ unsigned long long vt_pack(uint32_t key, int i) { return (unsigned long long)key << 32 | (0xffffffffu - (uint32_t)i); }

// The K largest of n different numbers (n <= VT_CAND) in descending order, the rest of `out` 0: a number's place is how many are larger
__device__ __forceinline__ void vt_rank(const unsigned long long* in, int n, unsigned long long* out, int K) {
    const int t = threadIdx.x;
    if (t < K) out[t] = 0ull;
    __syncthreads();
    if (t < n) {
        const unsigned long long mine = in[t];
        int place = 0;
#pragma unroll 8
        for (int i = 0; i < n; ++i) place += in[i] > mine;
        if (place < K && mine) out[place] = mine;
    }
    __syncthreads();
}
// the same of C lists of K in descending order: what is larger in another list is found by halving
__device__ __forceinline__ void vt_merge(const unsigned long long* in, int C, unsigned long long* out, int K) {
    const int t = threadIdx.x;
    if (t < K) out[t] = 0ull;
    __syncthreads();
    if (t < C * K) {
        const unsigned long long mine = in[t];
        int place = t % K;
        for (int c = 0; c < C; ++c) {
            if (c == t / K) continue;
            int lo = 0, hi = K; // the first place whose number is not larger
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (in[c * K + mid] > mine) lo = mid + 1;
                else hi = mid;
            }
            place += lo;
        }
        if (place < K && mine) out[place] = mine;
    }
    __syncthreads();
}

// The rows' top_k candidates in order (larger logit, then smaller index), as lb_sample_topk takes them.  The K-th largest of the maxima of pairs of threads bounds the K-th
// largest from below; what reaches it is collected in a second pass, from L2, and ranked: K and a few.  Where more than VT_CAND reach it (many equal ones, or a few threads
// with all of the large ones) the exact bound is found by halving, first of the value, then of the index among the equal ones, a pass each.  grid (rows, cluster)
extern "C" __global__ void __launch_bounds__(VT_THREADS, 3) vd_rows_topk(const __grid_constant__ lb_vd_params p) {
    __shared__ unsigned long long cand[VT_CAND], best[LB_VD_TOPK];
    __shared__ unsigned long long from[LB_VD_CLUSTER * LB_VD_TOPK]; // the cluster's lists, at its first CTA
    __shared__ uint32_t tops[VT_GROUPS], s_bound;
    __shared__ int n_cand;
    cg::cluster_group cluster = cg::this_cluster();
    const int t = threadIdx.x, lane = t & 31, row = blockIdx.x, C = gridDim.y, rank = blockIdx.y, K = p.top_k;
    pdl_wait();
    const float* x = p.logits + (size_t)row * p.V;
    const int per = (((p.V + C - 1) / C) + 3) & ~3, a = min(p.V, rank * per), b = min(p.V, a + per);
    // f(logit, index) over this thread's share of the range
    auto each = [&](auto f) {
        vd_each<VT_THREADS>(x, a, b, [&](const float4& v, int i) { f(v.x, i); f(v.y, i + 1); f(v.z, i + 2); f(v.w, i + 3); });
    };
    float top = -INFINITY;
    each([&](float v, int) { top = fmaxf(top, v); });
    const vd_place at = vd_find(p, row);
    if (!at.covered) return;
    cluster.barrier_arrive();
    const float pair = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    if ((t & 1) == 0) tops[t >> 1] = vt_key(pair);
    if (t == 0) n_cand = 0;
    __syncthreads();
    if (t < 32) { // the largest 20-bit bound that K of the maxima reach; 0: fewer than K do, all candidates count
        uint32_t g[VT_GROUPS / 32], bound = 0u;
#pragma unroll
        for (int i = 0; i < VT_GROUPS / 32; ++i) g[i] = tops[i * 32 + lane];
        for (int bit = 31; bit >= 12; --bit) {
            const uint32_t trial = bound | 1u << bit;
            int n = 0;
#pragma unroll
            for (int i = 0; i < VT_GROUPS / 32; ++i) n += g[i] >= trial;
            if ((int)__reduce_add_sync(0xffffffffu, n) >= K) bound = trial;
        }
        if (lane == 0) s_bound = max(bound, 1u);
    }
    __syncthreads();
    uint32_t bound = s_bound;
    auto collect = [&](int last) { // those above the bound, and of those equal to it the ones up to index `last`
        const float low = vt_value(bound);
        if (top >= low)
            each([&](float v, int i) {
                if (v > low || (v == low && i <= last)) {
                    const int o = atomicAdd(&n_cand, 1);
                    if (o < VT_CAND) cand[o] = vt_pack(vt_key(v), i);
                }
            });
        __syncthreads();
    };
    collect(0x7fffffff);
    if (n_cand > VT_CAND) { // what lies behind the range comes as -infinity, whose key is 0
        auto count = [&](auto f) { // over all of the CTA's logits
            int n = 0;
            each([&](float v, int i) { n += f(vt_key(v), i); });
            __syncthreads();
            if (t == 0) n_cand = 0;
            __syncthreads();
            n = __reduce_add_sync(0xffffffffu, n);
            if (lane == 0 && n) atomicAdd(&n_cand, n);
            __syncthreads();
            return n_cand;
        };
        bound = 0u;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t trial = bound | 1u << bit;
            if (count([&](uint32_t k, int) { return k >= trial; }) >= K) bound = trial;
        }
        const int above = count([&](uint32_t k, int) { return k > bound; });
        int last = 0; // the smallest index with K - above equal ones up to it
        for (int bit = 24; bit >= 0; --bit) {
            const int trial = last | 1 << bit;
            if (count([&](uint32_t k, int i) { return k == bound && i < trial; }) < K - above) last = trial;
        }
        __syncthreads();
        if (t == 0) n_cand = 0;
        __syncthreads();
        collect(last);
    }
    vt_rank(cand, n_cand, best, K);
    cluster.barrier_wait();
    __syncthreads();
    if (t < K) cluster.map_shared_rank(from, 0)[rank * K + t] = best[t];
    cluster.sync();
    if (rank) return;
    if (C > 1) vt_merge(from, C, best, K);
    double* e = reinterpret_cast<double*>(cand);
    const float first = best[0] ? vt_value((uint32_t)(best[0] >> 32)) : -INFINITY;
    if (t < K) {
        const float v = vt_value((uint32_t)(best[t] >> 32));
        e[t] = best[t] ? vd_exp(v, first, 1.0 / p.temperature) : 0.0;
        p.list_val[(size_t)row * LB_VD_TOPK + t] = v;
        p.list_idx[(size_t)row * LB_VD_TOPK + t] = (int)(0xffffffffu - (uint32_t)best[t]);
    }
    __syncthreads();
    if (t < 32) { // the sum, and the draft's place, by one warp
        const int d = p.drafts[row];
        double z = 0.0, px = 0.0;
        int n = 0;
        for (int i = lane; i < K; i += 32) {
            if (!best[i]) continue;
            ++n;
            z += e[i];
            if ((int)(0xffffffffu - (uint32_t)best[i]) == d) px = e[i];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            z += __shfl_xor_sync(0xffffffffu, z, o);
            px += __shfl_xor_sync(0xffffffffu, px, o); // one lane's, the others' 0
        }
        n = __reduce_add_sync(0xffffffffu, n);
        if (t == 0) {
            const lb_vd_row st = {z, first, best[0] ? (int)(0xffffffffu - (uint32_t)best[0]) : 0, 0, n};
            vd_decide(p, row, at.last, z > 0.0 ? px / z : 0.0, st);
        }
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

// Greedy, or from the rows' lists: a warp per request, a lane two neighbouring ranks
extern "C" __global__ void __launch_bounds__(32) vd_pick_short(const __grid_constant__ lb_vd_params p) {
    const int lane = threadIdx.x, r = blockIdx.x;
    pdl_wait();
    int first, last;
    const int at = vd_stop(p, r, first, last);
    if (at < 0) return;
    const lb_vd_row st = p.stat[at];
    int token = st.best;
    if (p.temperature > 0.0 && st.n) {
        double e[2], w[2];
        int idx[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * lane + j;
            idx[j] = i < st.n ? p.list_idx[(size_t)at * LB_VD_TOPK + i] : -1;
            e[j] = w[j] = 0.0;
            if (i < st.n) {
                e[j] = w[j] = vd_exp(p.list_val[(size_t)at * LB_VD_TOPK + i], st.max, 1.0 / p.temperature) / st.z;
                if (at < last) {
                    const double q = p.probs ? (double)p.probs[(size_t)at * p.V + idx[j]] : idx[j] == p.drafts[at] ? 1.0 : 0.0;
                    if (q > 0.0) w[j] = fmax(e[j] - q, 0.0);
                }
            }
        }
        if (!__any_sync(0xffffffffu, w[0] > 0.0 || w[1] > 0.0)) { // rounding left nothing
            w[0] = e[0];
            w[1] = e[1];
        }
        double run = w[0] + w[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        const double goal = (double)p.u_pick[r] * __shfl_sync(0xffffffffu, run, 31), half = run - w[1];
        const bool hit0 = w[0] > 0.0 && half > goal, hit1 = w[1] > 0.0 && run > goal;
        const uint32_t hit = __ballot_sync(0xffffffffu, hit0 || hit1), some = __ballot_sync(0xffffffffu, w[0] > 0.0 || w[1] > 0.0);
        // the first lane behind the goal; none: the last with weight
        const int lane_of = hit ? __ffs(hit) - 1 : 31 - __clz(some);
        token = __shfl_sync(0xffffffffu, (hit ? hit0 : !(w[1] > 0.0)) ? idx[0] : idx[1], lane_of);
    }
    vd_write(p, r, first, last, at, token);
}

// From the whole vocabulary: a cluster per request, its CTAs and their warps taking neighbouring ranges in index order.  Against certain drafts, and in a last row, the weights are
// exponentials as they are (one pass); against the draft's probabilities they have to be divided by their sum first (a pass for it).  grid (requests, cluster)
#define VP_THREADS 512
#define VP_WARPS (VP_THREADS / 32)
extern "C" __global__ void __launch_bounds__(VP_THREADS, 1) vd_pick(const __grid_constant__ lb_vd_params p) {
    __shared__ double part[2];           // this CTA's sum: of the exponentials, of the weights
    __shared__ double ws[VP_WARPS], table[VD_STEPS];
    __shared__ int s_token, s_last;
    cg::cluster_group cluster = cg::this_cluster();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, r = blockIdx.x, C = gridDim.y, rank = blockIdx.y;
    vd_exps::fill(table);
    __syncthreads();
    pdl_wait();
    int first, last;
    const int at = vd_stop(p, r, first, last);
    if (at < 0) return;
    const lb_vd_row st = p.stat[at];
    const float* x = p.logits + (size_t)at * p.V;
    const bool inner = at < last;
    const float* q = inner && p.probs ? p.probs + (size_t)at * p.V : nullptr;
    const int gone = inner && !p.probs ? p.drafts[at] : -1; // a certain draft
    const vd_exps expo(table, st.max, p.temperature);
    const int per = ((p.V + C * VP_WARPS - 1) / (C * VP_WARPS) + 3) & ~3, a = min(p.V, (rank * VP_WARPS + warp) * per), b = min(p.V, a + per); // this warp's range
    double sums[LB_VD_CLUSTER];
    auto all = [&](double v, int which) { // sum over the CTA into part[which] (ws: the warps'), then over the cluster in its order; sums: the CTAs'
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) ws[warp] = v;
        __syncthreads();
        if (warp == 0) {
            double s = lane < VP_WARPS ? ws[lane] : 0.0;
#pragma unroll
            for (int o = VP_WARPS / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (lane == 0) part[which] = s;
        }
        cluster.sync();
        double s = 0.0;
#pragma unroll
        for (int c = 0; c < LB_VD_CLUSTER; ++c) sums[c] = c < C ? *cluster.map_shared_rank(&part[which], c) : 0.0;
#pragma unroll
        for (int c = 0; c < LB_VD_CLUSTER; ++c) s += sums[c];
        return s;
    };
    // weights of four logits at i, i + step, ..: p; p without a certain draft; max(p - q, 0), a q that is no positive number being 0
    auto plain = [&](int, int, const float (&l)[4], const float (&)[4], double (&w)[4]) { expo(l, w); };
    auto without = [&](int i, int step, const float (&l)[4], const float (&)[4], double (&w)[4]) {
        expo(l, w);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j * step == gone) w[j] = 0.0;
    };
    auto rest = [&](int, int, const float (&l)[4], const float (&o)[4], double (&w)[4]) {
        expo(l, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double d = w[j] - vd_double(fmaxf(o[j], 0.f));
            w[j] = o[j] < INFINITY && __double2hiint(d) >= 0 ? d : o[j] >= 0.f ? 0.0 : w[j];
        }
    };
    // their sum over a warp's range: four neighbours a lane and load, the next loads on their way while the values of the last ones are worked on
    auto over = [&](auto f, const float* other) {
        constexpr int H = 3;
        double s[4] = {0.0, 0.0, 0.0, 0.0};
        float4 l[H], o[H];
        const bool wide = (((size_t)(x + a) | (other ? (size_t)(other + a) : 0)) & 15) == 0;
        auto four = [&](const float* v, int i, float none) {
            if (i + 3 < b && wide) return __ldg(reinterpret_cast<const float4*>(v + i));
            return make_float4(i < b ? v[i] : none, i + 1 < b ? v[i + 1] : none, i + 2 < b ? v[i + 2] : none, i + 3 < b ? v[i + 3] : none);
        };
        auto load = [&](int i) {
#pragma unroll
            for (int h = 0; h < H; ++h) {
                l[h] = four(x, i + 128 * h, -INFINITY);
                if (other) o[h] = four(other, i + 128 * h, 0.f);
            }
        };
        load(a + 4 * lane);
        for (int i = a + 4 * lane; i < a + 4 * lane + per; i += 128 * H) { // the whole warp goes on while any lane does
            float4 l0[H], o0[H];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                l0[h] = l[h];
                o0[h] = other ? o[h] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            load(i + 128 * H); // behind the range: nothing is read
#pragma unroll
            for (int h = 0; h < H; ++h) {
                if (i + 128 * h - 4 * lane >= b) break; // the same for the warp
                const float lv[4] = {l0[h].x, l0[h].y, l0[h].z, l0[h].w}, ov[4] = {o0[h].x, o0[h].y, o0[h].z, o0[h].w};
                double w[4];
                f(i + 128 * h, 1, lv, ov, w);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] += w[j];
            }
        }
        return (s[0] + s[1]) + (s[2] + s[3]);
    };
    double total;
    bool whole = !inner; // the weights are p
    if (q) {
        const double z = 1.0 / all(over(plain, nullptr), 0);
        for (int i = t; i < VD_STEPS; i += VP_THREADS) table[i] *= z; // from here on the exponentials are probabilities
        __syncthreads();
        total = all(over(rest, q), 1);
    } else total = all(gone >= 0 ? over(without, nullptr) : over(plain, nullptr), 1);
    if (!whole && !(total > 0.0)) { // rounding left nothing: from p itself
        whole = true;
        cluster.sync(); // the sums have been read
        total = all(over(plain, nullptr), 1);
    }
    cluster.sync(); // nobody leaves while its sums are read
    const double goal = (double)p.u_pick[r] * total;
    double base = 0.0, sum = 0.0;
    int owner = 0; // the CTA whose range the goal lies in: the last one with weight where rounding has left it behind them all
    bool found = false;
#pragma unroll
    for (int c = 0; c < LB_VD_CLUSTER; ++c) {
        if (!found && sums[c] > 0.0) {
            owner = c;
            base = sum;
            found = sum + sums[c] > goal;
        }
        sum += sums[c];
    }
    if (rank != owner) return;
    int w0 = 0;
    sum = base;
    for (int w = 0; w < VP_WARPS; ++w) {
        if (!(ws[w] > 0.0)) continue;
        w0 = w;
        base = sum;
        sum += ws[w];
        if (sum > goal) break;
    }
    // the range of warp w0, four neighbours a thread, 4 VP_THREADS at a time; s_token the first behind the goal, s_last the last with weight
    if (t == 0) {
        s_token = 0x7fffffff;
        s_last = -1;
    }
    const int lo = min(p.V, (rank * VP_WARPS + w0) * per), hi = min(p.V, lo + per);
    for (int i0 = lo; i0 < hi; i0 += 4 * VP_THREADS) {
        const int i = i0 + 4 * t;
        float l[4], o[4];
        double v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            l[j] = i + j < hi ? x[i + j] : -INFINITY;
            o[j] = q && i + j < hi ? q[i + j] : 0.f;
        }
        if (whole) plain(i, 1, l, o, v);
        else if (q) rest(i, 1, l, o, v);
        else without(i, 1, l, o, v);
        double run = (v[0] + v[1]) + (v[2] + v[3]);
        const double mine = run;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double u = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += u;
        }
        __syncthreads(); // ws has been read
        if (lane == 31) ws[warp] = run;
        __syncthreads();
        double upto = base + (run - mine), all_of = 0.0;
        int end = -1;
        for (int w = 0; w < VP_WARPS; ++w) {
            if (w < warp) upto += ws[w];
            all_of += ws[w];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            upto += v[j];
            if (v[j] > 0.0) {
                if (upto > goal) {
                    atomicMin(&s_token, i + j);
                    break;
                }
                end = i + j;
            }
        }
        end = __reduce_max_sync(0xffffffffu, end);
        if (lane == 0) atomicMax(&s_last, end);
        base += all_of;
        __syncthreads();
        if (s_token != 0x7fffffff) break;
    }
    __syncthreads();
    vd_write(p, r, first, last, at, s_token != 0x7fffffff ? s_token : s_last >= 0 ? s_last : st.best);
}
