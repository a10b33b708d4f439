// Grouped-query attention of a batch's new tokens over the 4-bit KV cache (layout: kv4.cuh).
//   out[j, h] = sum_t p_t v_t * sigmoid(gate[j, h]),  p = softmax over the rows t <= position of token j of  q[j, h] . k_t / sqrt(D),
// q normalised and rotated as the decode attention does it.  The columns of an item (a request's KV head) are its new tokens times the query heads that share the
// head; eight of them are taken at a time.
//   * The codes are the products' operands without a conversion: bits 4..7 of a half are the subnormal c 2^-20, which the tensor cores take at their full rate; a shift (for three of
//     four codes) and a mask for two.  A product's additions are cut off 2^-25 below the largest operand times 2^-14, the least normal number, whatever the codes are: at 2^-19 of a code.
//     (Codes in bits 0..3, where a byte's second one is had by difference without a shift, are 4 to 5 % faster and cut off at 2^-15 of a code: results were off by 2^-17 of the
//     values where one row has most of the weight, and queries kept 15 bits, not 22.  In bits 6..9, another shift and 1.5 %, they would be cut off at 2^-21.)
//     scores = sum over groups of scale_t (q . c_t) + lowest_t sum(q); read-out = sum of (p_t scale_t) c_t + p_t lowest_t.
//   * q, p and p scale go in as two fp16 terms, the leading one in rows 0..7 of a product and what it leaves in rows 8..15: 22 bits of each, for the price of rows that eight
//     columns would leave empty.  Weights are 2^9 at their reference and their second terms go in 2^11 up, so that the 22 bits reach down to 2^-23 of it; below that 2^-45 of
//     it stays, which many rows far below one that has the top score and small values need.  A query is scaled by a power of two to [2^13, 2^14) at its largest.  Scores, sums and
//     read-outs are fp32, a tile's read-outs added up by themselves (the products' own additions cut off); the output is fp16, what lb_gemm_int4 takes.
//   * lowest_t sum(q) is one product more per 8 rows, p_t lowest_t and the sum of p one per 16.
//   * A tile is 32768 / D rows, 36 KB, one bulk copy, requested by whichever warp is the last to be done with the place it goes to.  A warp does the scores of 256 / D blocks of
//     16 rows and leaves their probabilities in shared memory; after a barrier it reads a group's 64 features out over its part of the tile, weights - probabilities times that
//     group's scales, multiplied in 32 bits - as operands (with the products written for all groups by whoever has the scores 100 001 rows took 8 % longer).  References are standing:
//     probabilities are taken against the largest score, and a warp's weights of a column against the largest of them, at the last time that one passed its reference by 2^6, for
//     which fp16 has room; so a tile usually costs one barrier and no exchange of maxima.  (A reference from the scales alone, 2 % faster, lost the bits of all rows
//     that have weight where a row that has none is of large scale.)  Tiles whose rows are all there and seen by every column, most, take a path
//     without those checks (5 %).
//   * All tiles of all items are dealt evenly to the CTAs in one line, with places of one and a half tiles for an item's queries and results, so that ragged batches balance (32
//     sequences in an earlier kernel: 74 us without such places, 61 with a tile's, 57 so); an item cut by a border leaves records that kv4_merge joins in order.
// mma.sync rather than tcgen05: the columns are few (6 for one token of 24 heads on 4), and codes would have to be widened into shared or tensor memory for it.
// Bound by the latency of a tile's steps, with 16 warps an SM (as many as 128 registers leave) to hide it: per tile and SM some 720 instructions a warp (issue slots 48 %
// busy), 180 passes through shared memory a warp (half of its time: queries 64, codes 32, copies in 36, scales 36, probabilities 20), the tensor pipe 34 %.
// us a call with the merge, 24 / 4 heads of 256: one sequence of 4096 rows 11.2, of 100 001 43.9 (2.6 TB/s); 32 of 40 to 16 000 rows 54.4 (2.6 TB/s); 16 of 500 to 9001 rows with up
// to 5 new tokens 79.3; 64 of 17 to 3001 rows, 32 / 8 heads of 128: 38.5, of 64: 31.  Tried without gain, with the time of the kernel of then: warps of their own for scores and
// read-outs (8 + 8 with the queries in registers 66 us at 100 001 rows, two CTAs of 6 + 2 60, both where 48); 16 columns at a time on half as many warps (150 where passes of eight took
// 118); three CTAs of four warps with the queries in registers (54 where 48); maxima exchanged for every tile (52 where 48); barriers and references of the warps that share blocks
// alone (41.5 where 41.0); a block's scales by shuffles (41.3 where 41.0); the next launch let in early (13.9 at 4096 rows where 12.4: its waiting CTAs are in the way).
#include "kv4.cuh"

#define KA_WARPS 8
#define KA_THREADS (32 * KA_WARPS)
#define KA_COLS LB_KV4_COLS

__device__ __forceinline__ void ka_mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// the same onto nothing
__device__ __forceinline__ void ka_mma0(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t ka_pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 ka_pair(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float ka_pow2(int e) { return __int_as_float((127 + e) << 23); } // -126 <= e <= 127
__device__ __forceinline__ float ka_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two at a time
__device__ __forceinline__ float2 ka_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 ka_mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 ka_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
// has the phase completed?  (no waiting)
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// fp16 pairs of (x, y) and of what the rounding left
__device__ __forceinline__ void ka_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = ka_pack(x, y);
    const float2 h = ka_pair(hi);
    lo = ka_pack(x - h.x, y - h.y);
}

// the same with the second term carried 2^11 up, where a small number's still has its bits: its products have sums of their own
#define KA_REST 4.8828125e-04f // 2^-11
__device__ __forceinline__ void ka_split_up(float2 v, uint32_t& hi, uint32_t& lo) {
    hi = ka_pack(v.x, v.y);
    const float2 up = make_float2(1.f / KA_REST, 1.f / KA_REST), r = ka_fma2(ka_pair(hi), make_float2(-1.f / KA_REST, -1.f / KA_REST), ka_mul2(v, up));
    lo = ka_pack(r.x, r.y);
}

// code j of both halves of a word as fp16 numbers 2^-20 c
__device__ __forceinline__ uint32_t ka_codes(uint32_t v, int j) { return (j == 0 ? v << 4 : j == 1 ? v : j == 2 ? v >> 4 : v >> 8) & 0x00f000f0u; }

struct ka_item { int r, kv, z, tile, tiles; }; // a place in the line of tiles

#define KA_STEP ((uint32_t)LB_KV4_STEP)
#define KA_ITEM ((uint32_t)LB_KV4_ITEM)
#define KA_LIFT 9.f  // probabilities are 2^9 at their reference
#define KA_OVER 6.f  // and may pass it by 2^6
#define KA_WEIGHT 9  // a column's largest weight, probability times scale, is brought to [2^9, 2^10)
#define KA_ROOM 6    // and later ones may be as large as 2^15
#define KA_LEAST -110 // weights count as no smaller than 2^-110 for that

template <int D>
struct ka {
    static constexpr int S = D / 64, PARTS = KA_WARPS / S, BLK = LB_KV4_BLOCK(D), NS = LB_KV4_STAGES;
    static constexpr int BW = 4 / S, TILE = LB_KV4_TILE(D), BLOCKS = TILE / 16; // blocks of a warp; block w + 8 k is warp w's
    static constexpr int P_BUFS = D == 64 ? 1 : 2; // what there is room for
    struct alignas(128) smem {
        unsigned char ring[NS][BLOCKS * BLK];
        union {
            float4 p[P_BUFS][BLOCKS][32];       // probabilities, a block's as a lane has them
            float sum[PARTS][KA_COLS][D + 4];   // at an item's end
        };
        uint4 q[4 * S][32];             // queries likewise: step 4 group + 2 word + u
        uint2 qsum[32];                 // sums of a query's groups as the operand that meets (scale, lowest)
        float part[KA_WARPS][KA_COLS][S + 1];
        alignas(16) float max[KA_COLS][KA_WARPS];
        double freq[D / 2];
        float factor[KA_COLS], m[KA_COLS], l[KA_COLS], low[KA_COLS][S];
        uint64_t full[NS], pfree;
        ka_item ahead;                  // the last tile that was requested
        uint32_t pre[LB_KV4_REQS + 1];  // places in the line before request r
        int len[LB_KV4_REQS], n[LB_KV4_REQS], start[LB_KV4_REQS], seq[LB_KV4_REQS], limit[KA_COLS];
        uint32_t requested, warp_sum[KA_WARPS]; // requested: tiles of this CTA
    };
    static_assert(sizeof(smem) <= LB_KV4_SMEM && (LB_KV4_SMEM + 1024) * LB_KV4_CTAS <= 228 * 1024, "shared memory");
    const lb_kv4_attn_params& p;
    smem& s;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, ft = lane & 3, G;

    __device__ __forceinline__ ka(const lb_kv4_attn_params& p_, smem& s_) : p(p_), s(s_), G(p_.HQ / p_.b.HKV) {}

    __device__ __forceinline__ int sets(int n) const { return (n * G + KA_COLS - 1) / KA_COLS; }

    // The line of work: for every item (request, KV head, set of columns) KA_ITEM places for its queries and its results, which take about one and a half times as long as a tile, and
    // KA_STEP for every tile, which belongs to the CTA that has its first.
    __device__ __forceinline__ uint32_t places(int tiles) const { return KA_STEP * (uint32_t)tiles + KA_ITEM; }
    // the requests, and how many places lie before each
    __device__ __forceinline__ uint32_t read_batch() {
        kv4_request q = {0, 0, 0, 0};
        if (t < p.b.n_reqs) q = kv4_get(p.b, t);
        const int len = q.n > 0 ? q.pos + q.n : 0;
        s.len[t] = len; s.n[t] = q.n; s.start[t] = q.start; s.seq[t] = q.seq;
        uint32_t sum = q.n > 0 ? places((len + TILE - 1) / TILE) * p.b.HKV * sets(q.n) : 0u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) s.warp_sum[warp] = sum;
        __syncthreads();
        uint32_t before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < KA_WARPS; ++w) {
            if (w < warp) before += s.warp_sum[w];
            total += s.warp_sum[w];
        }
        s.pre[t + 1] = before + sum;
        if (t == 0) s.pre[0] = 0;
        __syncthreads();
        return total;
    }
    __device__ __forceinline__ int request_at(uint32_t x) const { // the last request with pre <= x that has tiles
        int lo = 0, hi = p.b.n_reqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s.pre[mid] <= x) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
    // the first tile that begins at place x of the line or behind it; base: the first place of the item that x lies in
    __device__ __forceinline__ ka_item place(uint32_t x, uint32_t& base) const {
        ka_item it;
        it.r = request_at(x);
        it.tiles = (s.len[it.r] + TILE - 1) / TILE;
        const uint32_t each = places(it.tiles), item = (x - s.pre[it.r]) / each, z = (uint32_t)sets(s.n[it.r]);
        base = s.pre[it.r] + item * each;
        it.kv = (int)(item / z);
        it.z = (int)item - it.kv * (int)z;
        it.tile = before(x - base);
        if (it.tile == it.tiles) {
            --it.tile;
            next(it);
        }
        return it;
    }
    // how many tiles of an item begin before its place v
    static __device__ __forceinline__ int before(uint32_t v) { return v <= KA_ITEM ? 0 : (int)((v - KA_ITEM + KA_STEP - 1) / KA_STEP); }
    // how many tiles begin at places x0 .. x1 - 1
    __device__ __forceinline__ uint32_t tiles_of(uint32_t x0, uint32_t x1) const {
        uint32_t n = 0;
        for (int r = request_at(x0); r < p.b.n_reqs && s.pre[r] < x1; ++r) {
            if (s.pre[r + 1] <= max(s.pre[r], x0)) continue;
            const int tiles = (s.len[r] + TILE - 1) / TILE;
            const uint32_t each = places(tiles), from = max(x0, s.pre[r]) - s.pre[r], to = min(x1, s.pre[r + 1]) - s.pre[r], i0 = from / each, i1 = to / each;
            n += (i1 - i0) * (uint32_t)tiles + (uint32_t)before(to - i1 * each) - (uint32_t)before(from - i0 * each);
        }
        return n;
    }
    __device__ __forceinline__ void next(ka_item& it) const {
        if (++it.tile < it.tiles) return;
        it.tile = 0;
        if (++it.z < sets(s.n[it.r])) return;
        it.z = 0;
        if (++it.kv < p.b.HKV) return;
        it.kv = 0;
        do ++it.r; while (it.r < p.b.n_reqs && s.n[it.r] <= 0);
        it.tiles = it.r < p.b.n_reqs ? (s.len[it.r] + TILE - 1) / TILE : 0;
    }
    __device__ __forceinline__ int blocks(const ka_item& it) const { return min(BLOCKS, (s.len[it.r] - it.tile * TILE + 15) >> 4); }
    // tile number i of this CTA
    __device__ __forceinline__ void copy(const ka_item& it, uint32_t i) const {
        const uint32_t bytes = (uint32_t)blocks(it) * BLK;
        mbar_arrive_expect_tx(&s.full[i % NS], bytes);
        bulk_g2s_plain(s.ring[i % NS], p.b.cache + kv4_block(p.b, D, s.seq[it.r], it.kv, it.tile * TILE), bytes, &s.full[i % NS]);
    }

    // the queries of an item's columns: norm, rotation, 22 bits, as operands; a column per warp, a lane 8 features
    __device__ __forceinline__ void queries(const ka_item& it) {
        const int n = s.n[it.r], pos = s.len[it.r] - n, c = warp, col = it.z * KA_COLS + c, i = col / G, h = it.kv * G + col - i * G;
        const bool on = col < n * G, mine = on && lane < D / 8;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
        if (mine) kv4_load8(p.q, (size_t)(s.start[it.r] + i) * (size_t)p.row_stride + (size_t)h * (size_t)p.head_stride + lane * 8, p.type, p.wide, x);
        // while the queries are on their way: angles in 64 bits, reduced to a turn, sine and cosine of at most pi in 32; a pair of features per lane, handed to the lane that has it
        float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
        if (on)
#pragma unroll
            for (int k = 0; k < D / 64; ++k) {
                if (64 * k >= p.rot_dims) break;
                float c1 = 1.f, s1 = 0.f;
                if (2 * (32 * k + lane) < p.rot_dims) {
                    const double a = (double)(pos + i) * s.freq[32 * k + lane];
                    sincosf((float)fma(-rint(a * 0.15915494309189535), 6.283185307179586, a), &s1, &c1);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) { // pairs 4 lane + j: of the eight lanes from 8 k on
                    const float c2 = __shfl_sync(0xffffffffu, c1, (4 * lane + j) & 31), s2 = __shfl_sync(0xffffffffu, s1, (4 * lane + j) & 31);
                    if (lane >> 3 == k) { cs[j] = c2; sn[j] = s2; }
                }
            }
        if (p.norm_w && on) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
            ss = warp_sum(ss);
            float r = rsqrtf(ss * (1.0f / D) + p.eps);
            if (!(ss < INFINITY)) { // squares beyond fp32: of 2^-80 x, beside which eps is nothing
                ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    x[j] *= 8.27180612553028e-25f;
                    ss = fmaf(x[j], x[j], ss);
                }
                r = rsqrtf(warp_sum(ss) * (1.0f / D));
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] * r * (mine ? bf16_bits_to_f32(p.norm_w[lane * 8 + j]) : 0.f);
        }
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float u = x[2 * j], v = x[2 * j + 1];
            x[2 * j] = u * cs[j] - v * sn[j];
            x[2 * j + 1] = u * sn[j] + v * cs[j];
            top = fmaxf(top, fmaxf(fabsf(x[2 * j]), fabsf(x[2 * j + 1])));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        int e = 13 - ((__float_as_int(top) >> 23) - 127); // largest to [2^13, 2^14)
        e = top == 0.f ? 0 : min(120, max(-114, e));
        const float up = ka_pow2(e);
        float sum = 0.f;
        if (lane < D / 8) {
#pragma unroll
            for (int u = 0; u < 2; ++u) { // codes 2 u and 2 u + 1 of a word's halves
                uint4 w;
                ka_split(x[2 * u] * up, x[2 * u + 4] * up, w.x, w.y);
                ka_split(x[2 * u + 1] * up, x[2 * u + 5] * up, w.z, w.w);
                const float2 a = ka_pair(w.x), b = ka_pair(w.y), c2 = ka_pair(w.z), d = ka_pair(w.w);
                sum += ((a.x + a.y) + (b.x + b.y)) + ((c2.x + c2.y) + (d.x + d.y));
                s.q[(lane >> 3) * 4 + 2 * (lane & 1) + u][c * 4 + ((lane & 7) >> 1)] = w;
            }
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        sum = __shfl_sync(0xffffffffu, sum, (lane & 3) * 8); // of group lane % 4, at most 2^20
        if (lane < 4) {
            uint2 w;
            ka_split(0.f, lane < S ? sum * 0.015625f : 0.f, w.x, w.y);
            s.qsum[c * 4 + lane] = w;
        }
        if (lane == 0) {
            s.factor[c] = ka_pow2(min(20 - e, 127)) * (rsqrtf((float)D) * 1.4426950408889634f); // scores in log2 units; of queries beyond 2^119 less than those: one row has all the weight
            s.limit[c] = on ? pos + i : -1;
        }
    }

    float m;            // reference of column g's scores: one of them, so that its own difference is 0 whatever its size
    float low[4];       // of this warp's rows, column g, from first and from second terms: sums of p lowest of groups 2 ft, 2 ft + 1; ft = 2: the sum of p
    float acc[8][2];    // of this warp's group and part, column g: features 8 (2 ft, 2 ft + 1) + j
    float room;         // of column g's weights in this warp: how large they may be, a power of two, or 0 before the first
    float up;           // what brings them to fp16's range: 2^15 / room, or 0
    float f;            // of column g's scores, to log2 units
    int len, first_new; // rows of the item, the first of its new ones

    __device__ __forceinline__ void begin(const ka_item& it) {
        len = s.len[it.r];
        first_new = len - s.n[it.r];
        m = -INFINITY;
        low[0] = low[1] = low[2] = low[3] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j][0] = acc[j][1] = 0.f;
        room = up = 0.f;
    }

    // (scale, lowest) of four rows, of those that are there
    static __device__ __forceinline__ uint4 there(uint4 v, int row0, int len) {
        return make_uint4(row0 < len ? v.x : 0u, row0 + 1 < len ? v.y : 0u, row0 + 2 < len ? v.z : 0u, row0 + 3 < len ? v.w : 0u);
    }
    static __device__ __forceinline__ uint32_t lowest_or_0(uint32_t pair) { return (pair & 0x7fff0000u) < 0x7c000000u ? pair : 0u; }
    // a thread's scores of a block of 16 rows: rows 4 ft .. 4 ft + 3, column g; probabilities in two terms
    struct rows {
        float sc[4];
        uint2 hi, lo;
    };

    // scores -> probabilities, for whoever reads the block out
    __device__ __forceinline__ void weigh(rows& r, float4* to) {
        const float from = m == -INFINITY ? 0.f : m; // a column that has seen nothing yet
        float2 pr[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 x = ka_fma2(ka_add2(make_float2(r.sc[2 * i], r.sc[2 * i + 1]), make_float2(-from, -from)), make_float2(f, f), make_float2(KA_LIFT, KA_LIFT));
            pr[i] = make_float2(ka_exp2(x.x), ka_exp2(x.y));
        }
        ka_split_up(pr[0], r.hi.x, r.lo.x);
        ka_split_up(pr[1], r.hi.y, r.lo.y);
        to[lane] = make_float4(pr[0].x, pr[0].y, pr[1].x, pr[1].y);
    }
    // `top`: the largest of this thread's weights of a tile.  A new reference for the columns where it is beyond what there is room for
    __device__ __forceinline__ void widen(float top) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (!(top > room)) return;
        const int e = max((__float_as_int(top) >> 23) - 127, KA_LEAST);
        const float shrink = room * ka_pow2(-(e + KA_ROOM)); // 0 before the first, when there are no sums yet
        room = ka_pow2(e + KA_ROOM);
        up = ka_pow2(KA_WEIGHT - e);
#pragma unroll
        for (int j = 0; j < 8; ++j) { acc[j][0] *= shrink; acc[j][1] *= shrink; }
    }

    // one tile; false: the wait for it gave up.  FULL: all of its rows are there and every column sees them
    template <bool FULL>
    __device__ __forceinline__ bool tile(const ka_item& it, uint32_t i_tile, uint32_t tiles) {
        const int slot = i_tile % NS, nb = FULL ? BLOCKS : min(BLOCKS, (len - it.tile * TILE + 15) >> 4), row0 = it.tile * TILE + 4 * ft, group = warp % S, part = warp / S;
        float4 (*const pw)[32] = s.p[P_BUFS == 2 ? i_tile & 1 : 0];
        const unsigned char* ring = s.ring[slot];
        rows r[BW];
        bool landed = mbar_wait(&s.full[slot], (i_tile / NS) & 1), over = !landed;
        if (FULL || (warp < nb && landed)) {
            float a[BW][S][2][4];
            uint2 w[BW][S][2];
            uint32_t pair[BW][2];
#pragma unroll
            for (int k = 0; k < BW; ++k) { // blocks that are not there hold what was there before them: their scores are masked
                const unsigned char* blk = ring + (warp + 8 * k) * BLK;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int q = 0; q < S; ++q) w[k][q][i] = *reinterpret_cast<const uint2*>(blk + ((i * S + q) * 32 + lane) * 8);
                    pair[k][i] = *reinterpret_cast<const uint32_t*>(blk + 16 * D + ((ft % S) * 16 + 4 * (g >> 1) + 2 * i + (g & 1)) * 4);
                }
            }
#pragma unroll
            for (int st = 0; st < 4; ++st) // blocks and groups are chains of their own
#pragma unroll
                for (int q = 0; q < S; ++q) {
                    const uint4 qa = s.q[q * 4 + st][lane];
#pragma unroll
                    for (int k = 0; k < BW; ++k)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t v = st < 2 ? w[k][q][i].x : w[k][q][i].y, b0 = ka_codes(v, 2 * (st & 1)), b1 = ka_codes(v, 2 * (st & 1) + 1);
                            if (st == 0) ka_mma0(a[k][q][i], qa, b0, b1);
                            else ka_mma(a[k][q][i], qa, b0, b1);
                        }
                }
            const uint2 qs = s.qsum[lane];
#pragma unroll
            for (int k = 0; k < BW; ++k) {
                const unsigned char* blk = ring + (warp + 8 * k) * BLK;
#pragma unroll
                for (int i = 0; i < 2; ++i) { // lowest sum(q)
                    float d[4];
                    ka_mma0(d, make_uint4(qs.x, qs.y, 0u, 0u), pair[k][i], 0u);
                    r[k].sc[2 * i] = (d[0] + d[2]) * 6.103515625e-05f; // 2^-14: the codes' 2^-20 over the sums' 2^-6
                    r[k].sc[2 * i + 1] = (d[1] + d[3]) * 6.103515625e-05f;
                }
#pragma unroll
                for (int q = 0; q < S; ++q) {
                    const uint4 pr = *reinterpret_cast<const uint4*>(blk + 16 * D + (q * 16 + 4 * ft) * 4);
                    const float scale[4] = {ka_pair(pr.x).x, ka_pair(pr.y).x, ka_pair(pr.z).x, ka_pair(pr.w).x};
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float2 sum = ka_add2(make_float2(a[k][q][i][0], a[k][q][i][1]), make_float2(a[k][q][i][2], a[k][q][i][3]));
                        const float2 sc = ka_fma2(make_float2(scale[2 * i], scale[2 * i + 1]), sum, make_float2(r[k].sc[2 * i], r[k].sc[2 * i + 1]));
                        r[k].sc[2 * i] = sc.x;
                        r[k].sc[2 * i + 1] = sc.y;
                    }
                }
                if (!FULL) { // rows that the column does not see, or that are not there
                    const int lim = s.limit[g] - row0 - 16 * (warp + 8 * k);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i > lim) r[k].sc[i] = -INFINITY;
                }
                over |= (fmaxf(fmaxf(r[k].sc[0], r[k].sc[1]), fmaxf(r[k].sc[2], r[k].sc[3])) - m) * f > KA_OVER;
            }
        } else {
#pragma unroll
            for (int k = 0; k < BW; ++k) {
                r[k].sc[0] = r[k].sc[1] = r[k].sc[2] = r[k].sc[3] = -INFINITY;
                r[k].hi = r[k].lo = make_uint2(0u, 0u);
            }
        }
        // the tile before has been read out; with two buffers the one before that, which everybody had done at the tile before's barrier
        if (P_BUFS == 1 && i_tile) landed = mbar_wait(&s.pfree, (i_tile - 1) & 1) && landed;
        if (FULL || warp < nb)
#pragma unroll
            for (int k = 0; k < BW; ++k) weigh(r[k], pw[warp + 8 * k]);
        // the values' scales of the blocks that this warp reads out
        uint32_t s01[4], s23[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int b = k * PARTS + part;
            s01[k] = s23[k] = 0u;
            if (!FULL && b >= nb) continue;
            uint4 v = *reinterpret_cast<const uint4*>(ring + b * BLK + 17 * D + (group * 16 + 4 * ft) * 4);
            if (!FULL) v = there(v, row0 + 16 * b, len);
            s01[k] = __byte_perm(v.x, v.y, 0x5410);
            s23[k] = __byte_perm(v.z, v.w, 0x5410);
            if (!FULL) { // a NaN's group reaches the columns that see its row, and no other as 0 times NaN
                const int lim = s.limit[g] - row0 - 16 * b;
                s01[k] &= (lim >= 0 ? 0xffffu : 0u) | (lim >= 1 ? 0xffff0000u : 0u);
                s23[k] &= (lim >= 2 ? 0xffffu : 0u) | (lim >= 3 ? 0xffff0000u : 0u);
            }
        }
        if (__syncthreads_or(over || !landed)) {
            if (__syncthreads_or(!landed)) return false;
            renew(r, FULL || warp < nb, pw);
        }
        uint32_t lv[BW][2]; // p lowest and the sum of p: lowest values as an operand, ones in its fifth column
#pragma unroll
        for (int k = 0; k < BW; ++k) {
            uint4 vr = *reinterpret_cast<const uint4*>(ring + (warp + 8 * k) * BLK + 17 * D + ((g % S) * 16 + 4 * ft) * 4);
            if (!FULL) { // blocks that are not there, too; where a column sees a NaN's row, p scale is NaN
                vr = there(vr, row0 + 16 * (warp + 8 * k), len);
                vr.x = lowest_or_0(vr.x); vr.y = lowest_or_0(vr.y); vr.z = lowest_or_0(vr.z); vr.w = lowest_or_0(vr.w);
            }
            lv[k][0] = g == 4 ? 0x3c003c00u : __byte_perm(vr.x, vr.y, 0x7632);
            lv[k][1] = g == 4 ? 0x3c003c00u : __byte_perm(vr.z, vr.w, 0x7632);
        }
        auto lowest = [&] {
#pragma unroll
            for (int k = 0; k < BW; ++k) {
                float d[4];
                ka_mma0(d, make_uint4(r[k].hi.x, r[k].lo.x, r[k].hi.y, r[k].lo.y), lv[k][0], lv[k][1]);
#pragma unroll
                for (int i = 0; i < 4; ++i) low[i] += d[i];
            }
        };
        if (BW > 2) lowest(); // frees their registers
        if (FULL || part < nb) {
            // weights, in 32 bits: a scale says nothing about them where the probability is small.  A NaN has no say in their reference
            float2 w[4][2];
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int b = k * PARTS + part;
                const float4 pk = !FULL && b >= nb ? make_float4(0.f, 0.f, 0.f, 0.f) : pw[b][lane];
                w[k][0] = ka_mul2(make_float2(pk.x, pk.y), ka_pair(s01[k]));
                w[k][1] = ka_mul2(make_float2(pk.z, pk.w), ka_pair(s23[k]));
                top = fmaxf(fmaxf(top, fmaxf(w[k][0].x, w[k][0].y)), fmaxf(w[k][1].x, w[k][1].y));
            }
            if (__any_sync(0xffffffffu, top > room)) widen(top);
            float d[8][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int b = k * PARTS + part;
                if (!FULL && k && b >= nb) break;
                const uint4 v = *reinterpret_cast<const uint4*>(ring + b * BLK + 8 * D + group * 512 + lane * 16);
                const uint32_t a0 = __byte_perm(v.x, v.y, 0x5410), a1 = __byte_perm(v.x, v.y, 0x7632), c0 = __byte_perm(v.z, v.w, 0x5410), c1 = __byte_perm(v.z, v.w, 0x7632);
                uint4 pa;
                ka_split_up(ka_mul2(w[k][0], make_float2(up, up)), pa.x, pa.y);
                ka_split_up(ka_mul2(w[k][1], make_float2(up, up)), pa.z, pa.w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t y = ka_codes(j < 4 ? a0 : a1, j & 3), z = ka_codes(j < 4 ? c0 : c1, j & 3);
                    if (k == 0) ka_mma0(d[j], pa, y, z);
                    else ka_mma(d[j], pa, y, z);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float2 sum = ka_add2(make_float2(acc[j][0], acc[j][1]), ka_fma2(make_float2(d[j][2], d[j][3]), make_float2(KA_REST, KA_REST), make_float2(d[j][0], d[j][1])));
                acc[j][0] = sum.x;
                acc[j][1] = sum.y;
            }
        }
        if (BW <= 2) lowest();
        __syncwarp();
        if (lane == 0) { // whoever finds that all warps are done, the last one at least, requests what comes to this place next
            mbar_arrive(&s.pfree);
            if (i_tile + NS < tiles && mbar_try(&s.pfree, i_tile & 1) && atomicExch(&s.requested, i_tile + NS + 1) != i_tile + NS + 1) {
                ka_item a = s.ahead;
                next(a);
                s.ahead = a;
                copy(a, i_tile + NS);
            }
        }
        return true;
    }

    // new references: the exchange of maxima, and the probabilities again
    __device__ __forceinline__ void renew(rows (&r)[BW], bool live, float4 (*pw)[32]) {
        float best = -INFINITY;
#pragma unroll
        for (int k = 0; k < BW; ++k) best = fmaxf(best, fmaxf(fmaxf(r[k].sc[0], r[k].sc[1]), fmaxf(r[k].sc[2], r[k].sc[3])));
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
        if (ft == 0) s.max[g][warp] = best;
        __syncthreads();
        const float4 a = *reinterpret_cast<const float4*>(s.max[g]), b = *reinterpret_cast<const float4*>(s.max[g] + 4);
        const float now = fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w))), top = fmaxf(m, now);
        const float corr = top == -INFINITY ? 0.f : ka_exp2((m - top) * f);
        // weights to come are smaller by as much: where there are some, their reference follows, and the sums so far stay as large as they are
        const int down = room > 0.f ? min(min((int)((top - m) * f), (__float_as_int(room) >> 23) - 127 - (KA_LEAST + KA_ROOM)), 100) : 0;
        const float keep = corr * ka_pow2(down);
        room *= ka_pow2(-down);
        up *= ka_pow2(down);
        m = top;
#pragma unroll
        for (int i = 0; i < 4; ++i) low[i] *= corr;
#pragma unroll
        for (int j = 0; j < 8; ++j) { acc[j][0] *= keep; acc[j][1] *= keep; }
        if (live)
#pragma unroll
            for (int k = 0; k < BW; ++k) weigh(r[k], pw[warp + 8 * k]);
        __syncthreads();
    }

    // eight features of a column: out, or a record
    __device__ __forceinline__ void put(const ka_item& it, bool whole, float* rec, int c, int f, const float (&v)[8], float inv) const {
        if (!whole) {
            float4* d = reinterpret_cast<float4*>(rec + c * LB_KV4_REC(D) + f);
            d[0] = make_float4(v[0], v[1], v[2], v[3]);
            d[1] = make_float4(v[4], v[5], v[6], v[7]);
            return;
        }
        const int col = it.z * KA_COLS + c, i = col / G, h = it.kv * G + col - i * G;
        const size_t row = (size_t)(s.start[it.r] + i);
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = v[j] * inv;
        if (p.gate) {
            float x[8];
            kv4_load8(p.gate, row * (size_t)p.row_stride + (size_t)h * (size_t)p.head_stride + f, p.type, p.wide, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] *= sigmoidf_dev(x[j]);
        }
        uint16_t* d = p.out + (row * p.HQ + h) * D + f;
        const uint4 w = make_uint4(ka_pack(o[0], o[1]), ka_pack(o[2], o[3]), ka_pack(o[4], o[5]), ka_pack(o[6], o[7]));
        if (p.out_wide) *reinterpret_cast<uint4*>(d) = w;
        else {
#pragma unroll
            for (int j = 0; j < 8; ++j) d[j] = (uint16_t)((j < 2 ? w.x : j < 4 ? w.y : j < 6 ? w.z : w.w) >> (16 * (j & 1)));
        }
    }
    // The item's columns, whole or this CTA's share of them.  `first`: the item's first tile was this CTA's, `last`: its last
    __device__ __forceinline__ void finish(const ka_item& it, bool first, bool last) {
        const int group = warp % S, part = warp / S, cols = min(KA_COLS, s.n[it.r] * G - it.z * KA_COLS);
        if (2 * ft < S) s.part[warp][g][2 * ft] = fmaf(low[2], KA_REST, low[0]);
        if (2 * ft + 1 < S) s.part[warp][g][2 * ft + 1] = fmaf(low[3], KA_REST, low[1]);
        if (ft == 2) s.part[warp][g][S] = fmaf(low[2], KA_REST, low[0]);
        if (ft == 0 && warp == 0) s.m[g] = m;
        const float unit = room * ka_pow2(20 - KA_WEIGHT - KA_ROOM); // 2^20 / up
        __syncthreads(); // the probabilities have been read
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 8; j += 4)
                *reinterpret_cast<float4*>(&s.sum[part][g][group * 64 + 8 * (2 * ft + i) + j]) =
                    make_float4(acc[j][i] * unit, acc[j + 1][i] * unit, acc[j + 2][i] * unit, acc[j + 3][i] * unit);
        __syncthreads();
        float* rec = p.records + ((size_t)blockIdx.x * 2 + (first ? 1 : 0)) * KA_COLS * LB_KV4_REC(D);
        for (int o = t; o < KA_COLS * D / 8; o += KA_THREADS) { // eight features a thread
            const int c = o / (D / 8), f = o % (D / 8) * 8;
            if (c >= cols) break;
            float lo = 0.f, l = 0.f, v[8];
#pragma unroll
            for (int w = 0; w < KA_WARPS; ++w) {
                lo += s.part[w][c][f >> 6];
                l += s.part[w][c][S];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll
            for (int q = 0; q < PARTS; ++q) { // the parts of a tile in their order
                const float4 a = *reinterpret_cast<const float4*>(&s.sum[q][c][f]), b = *reinterpret_cast<const float4*>(&s.sum[q][c][f + 4]);
                v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
                v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += lo;
            put(it, first && last, rec, c, f, v, 1.f / l);
            if (!(first && last) && f == 0) {
                rec[c * LB_KV4_REC(D) + D] = s.m[c];
                rec[c * LB_KV4_REC(D) + D + 1] = l;
                rec[c * LB_KV4_REC(D) + D + 2] = s.factor[c];
            }
        }
        __syncthreads(); // the sums' place and the queries are free for the next item
    }

    __device__ __forceinline__ void body() {
        if (t == 0) {
#pragma unroll
            for (int i = 0; i < NS; ++i) mbar_init(&s.full[i], 1);
            mbar_init(&s.pfree, KA_WARPS);
            mbar_fence_init();
        }
        for (int i = t; i < p.rot_dims / 2; i += KA_THREADS) s.freq[i] = p.freq[i];
        pdl_wait();
        const uint32_t total = read_batch(); // its barriers also show the mbarriers to everybody
        const uint32_t ctas = min(gridDim.x, total / KA_STEP); // whoever has places within an item has a tile of it
        lb_kv4_join* join = p.joins + blockIdx.x;
        if (blockIdx.x >= ctas) {
            if (t == 0) join->first = -1;
            return;
        }
        const uint32_t share = total / ctas, more = total - share * ctas; // the first `more` CTAs have one place more
        const uint32_t from = blockIdx.x * share + min(blockIdx.x, more), to = from + share + (blockIdx.x < more), x1 = tiles_of(from, to);
        uint32_t base;
        ka_item it = place(from, base);
        if (t == 32) { // does an item begin in the CTA before and go on here?  (another warp than the copies')
            lb_kv4_join j;
            j.first = -1;
            if (x1 && it.tile > 0) {
                const uint32_t begin = base + KA_ITEM, last = begin + KA_STEP * (uint32_t)(it.tiles - 1); // where its first and its last tile begin
                if (begin >= from - share - (blockIdx.x - 1 < more)) {
                    j.first = (int)blockIdx.x - 1;
                    j.last = (int)(last < more * (share + 1) ? last / (share + 1) : more + (last - more * (share + 1)) / share);
                    j.row0 = s.start[it.r];
                    j.kv = it.kv;
                    j.col0 = it.z * KA_COLS;
                    j.cols = min(KA_COLS, s.n[it.r] * G - j.col0);
                }
            }
            *join = j;
        }
        if (!x1) return; // an item's first places alone
        if (t == 0) {
            ka_item a = it;
            uint32_t i = 0;
            for (; i < NS && i < x1; ++i) {
                if (i) next(a);
                copy(a, i);
            }
            s.ahead = a;
            s.requested = i;
        }
        bool first = true;
        for (uint32_t x = 0; x < x1; ++x) {
            if (x == 0 || it.tile == 0) {
                first = it.tile == 0;
                queries(it);
                begin(it);
                __syncthreads();
                f = s.factor[g];
            }
            if (!(it.tile * TILE + TILE - 1 <= first_new ? tile<true>(it, x, x1) : tile<false>(it, x, x1))) { // a copy never landed: say so, let the others land, leave
                if (t == 0) {
                    atomicExch(p.b.status, KV_FAIL_FULL);
                    for (uint32_t y = x; y < s.requested; ++y) mbar_wait(&s.full[y % NS], (y / NS) & 1);
                }
                __syncthreads();
                return;
            }
            if (it.tile == it.tiles - 1 || x == x1 - 1) finish(it, first, it.tile == it.tiles - 1);
            if (x + 1 < x1) next(it);
        }
    }
};

#define KA_KERNEL(D)                                                                                                                             \
    extern "C" __global__ void __launch_bounds__(KA_THREADS, LB_KV4_CTAS) kv4_attn_##D(const __grid_constant__ lb_kv4_attn_params p) {         \
        extern __shared__ __align__(128) unsigned char ka_sm[];                                                                                 \
        ka<D> k(p, *reinterpret_cast<ka<D>::smem*>(ka_sm));                                                                                     \
        k.body();                                                                                                                                \
    }
KA_KERNEL(64)
KA_KERNEL(128)
KA_KERNEL(256)

// Joins the records of the items that were cut.  Every CTA counts the joins' columns; a unit is 64 features of a column, for 16 threads: dealt to groups of 16, or to whole CTAs in which
// the groups take runs of neighbouring records where there are few.  Records are added in the order of the rows, so results are the same from run to run.
#define KM_THREADS 256
#define KM_GROUPS (KM_THREADS / 16)
__device__ __forceinline__ void km_add(float4& A, float& L, float4 a, float l, float w) {
    L = fmaf(l, w, L);
    A.x = fmaf(a.x, w, A.x); A.y = fmaf(a.y, w, A.y); A.z = fmaf(a.z, w, A.z); A.w = fmaf(a.w, w, A.w);
}
template <int D>
__device__ __forceinline__ void kv4_merge_body(const lb_kv4_attn_params& p, int ctas) {
    constexpr int S = D / 64;
    __shared__ float4 red[KM_THREADS];
    __shared__ float red_m[KM_GROUPS], red_l[KM_GROUPS];
    __shared__ int pre[LB_KV4_MAX_CTAS + 1], s_warp[KM_THREADS / 32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, sub = t >> 4, G = p.HQ / p.b.HKV;
    pdl_wait();
    int base = 0;
    if (t == 0) pre[0] = 0;
    for (int c0 = 0; c0 < ctas; c0 += KM_THREADS) { // columns before every join
        int sum = 0;
        if (c0 + t < ctas) {
            const int first = p.joins[c0 + t].first, cols = p.joins[c0 + t].cols;
            sum = first >= 0 ? cols : 0;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) s_warp[warp] = sum;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < KM_THREADS / 32; ++w) {
            if (w < warp) sum += s_warp[w];
            all += s_warp[w];
        }
        if (c0 + t < ctas) pre[c0 + t + 1] = base + sum;
        base += all;
        __syncthreads();
    }
    const int units = base * S;
    const bool few = units <= (int)gridDim.x; // a CTA for each
    for (int first = few ? (int)blockIdx.x : (int)blockIdx.x * KM_GROUPS; first < units; first += few ? (int)gridDim.x : (int)gridDim.x * KM_GROUPS) {
        const int unit = few ? first : first + sub, pair = unit / S, f = unit % S * 64 + (t & 15) * 4;
        float M = -INFINITY, L = 0.f, F = 0.f;
        float4 A = make_float4(0.f, 0.f, 0.f, 0.f), gate = A;
        uint16_t* out = nullptr;
        if (unit < units) {
            int lo = 0, hi = ctas - 1; // the last join with pre <= pair
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (pre[mid] <= pair) lo = mid;
                else hi = mid - 1;
            }
            const lb_kv4_join j = p.joins[lo];
            const int c = pair - pre[lo], col = j.col0 + c, i = col / G, h = j.kv * G + col - i * G;
            const size_t row = (size_t)(j.row0 + i);
            const int n = j.last - j.first + 1, per = few ? (n + KM_GROUPS - 1) / KM_GROUPS : n, b0 = j.first + (few ? sub * per : 0), b1 = min(j.last + 1, b0 + per);
            if (!few || sub == 0) {
                out = p.out + (row * p.HQ + h) * D + f;
                if (p.gate) {
                    const size_t at = row * (size_t)p.row_stride + (size_t)h * (size_t)p.head_stride + f;
                    gate = make_float4(kv4_load1(p.gate, at, p.type), kv4_load1(p.gate, at + 1, p.type), kv4_load1(p.gate, at + 2, p.type), kv4_load1(p.gate, at + 3, p.type));
                }
            }
            F = __ldcg(p.records + (((size_t)j.first * 2 + 1) * KA_COLS + c) * LB_KV4_REC(D) + D + 2); // the same in all of them
            for (int b = b0; b < b1; b += 8) {
                float mv[8], lv[8], mx = M;
                float4 av[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const bool on = b + k < b1;
                    const float* rec = p.records + (((size_t)(on ? b + k : b) * 2 + (b + k == j.first ? 1 : 0)) * KA_COLS + c) * LB_KV4_REC(D);
                    mv[k] = on ? __ldcg(rec + D) : -INFINITY;
                    lv[k] = on ? __ldcg(rec + D + 1) : 0.f;
                    av[k] = on ? __ldcg(reinterpret_cast<const float4*>(rec + f)) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) mx = fmaxf(mx, mv[k]);
                const float use = mx == -INFINITY ? 0.f : mx, w = ka_exp2((M - use) * F);
                L *= w;
                A.x *= w; A.y *= w; A.z *= w; A.w *= w;
#pragma unroll
                for (int k = 0; k < 8; ++k) km_add(A, L, av[k], lv[k], ka_exp2((mv[k] - use) * F));
                M = mx;
            }
        }
        if (few) {
            red[t] = A;
            if ((t & 15) == 0) { red_m[sub] = M; red_l[sub] = L; }
            __syncthreads();
            if (sub == 0) {
#pragma unroll
                for (int q = 1; q < KM_GROUPS; ++q) M = fmaxf(M, red_m[q]);
                const float use = M == -INFINITY ? 0.f : M;
                L = 0.f;
                A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int q = 0; q < KM_GROUPS; ++q) km_add(A, L, red[q * 16 + t], red_l[q], ka_exp2((red_m[q] - use) * F));
            }
            __syncthreads();
        }
        if (out) {
            const float inv = 1.f / L;
            float v[4] = {A.x * inv, A.y * inv, A.z * inv, A.w * inv};
            if (p.gate) { v[0] *= sigmoidf_dev(gate.x); v[1] *= sigmoidf_dev(gate.y); v[2] *= sigmoidf_dev(gate.z); v[3] *= sigmoidf_dev(gate.w); }
#pragma unroll
            for (int k = 0; k < 4; ++k) out[k] = __half_as_ushort(__float2half_rn(v[k]));
        }
    }
}
extern "C" __global__ void __launch_bounds__(KM_THREADS) kv4_merge_64(const __grid_constant__ lb_kv4_attn_params p, int ctas) { kv4_merge_body<64>(p, ctas); }
extern "C" __global__ void __launch_bounds__(KM_THREADS) kv4_merge_128(const __grid_constant__ lb_kv4_attn_params p, int ctas) { kv4_merge_body<128>(p, ctas); }
extern "C" __global__ void __launch_bounds__(KM_THREADS) kv4_merge_256(const __grid_constant__ lb_kv4_attn_params p, int ctas) { kv4_merge_body<256>(p, ctas); }
