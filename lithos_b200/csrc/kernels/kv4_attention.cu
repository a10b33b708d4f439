// Grouped-query attention of a batch's new tokens over the 4-bit KV cache (layout: kv4.cuh).
//   out[j, h] = sum_t p_t v_t * sigmoid(gate[j, h]),  p = softmax over the rows t <= position of token j of  q[j, h] . k_t / sqrt(D),
// q normalised and rotated as the decode attention does it.  The columns of an item (a request's KV head) are its new tokens times the query heads that share the
// head; 8 MT of them are taken at a time.
//   * The codes are the products' operands as they are: four bits in the low end of a half are the subnormal c 2^-24, four bits above them c 2^-20, and the tensor cores
//     take subnormals exactly, at their full rate.  A word of 8 codes costs a shift and four ANDs, no conversion; the 2^4 between neighbours is taken out of the query
//     (keys) and of the sums (values).  scores = sum over groups of scale_t (q . c_t) + lowest_t sum(q); read-out = sum of (p_t scale_t) c_t + p_t lowest_t.
//   * q and p scale go in as two fp16 terms, the leading one in rows 0..7 of a product and what it leaves in rows 8..15: 22 bits of each, for the price of rows that a
//     group of up to 8 columns would leave empty.  A query is scaled by a power of two to [2^13, 2^14) at its largest; p (2^14 at the maximum) times scale by one per group, the
//     largest scale so far becoming [1/2, 1): weights keep their bits down to 2^-27 of the largest.  Scores, maxima, sums and read-outs are fp32; the output is
//     fp16, what lb_gemm_int4 takes.
//   * lowest_t sum(q) is one product more per 8 rows, p_t lowest_t and the sum of p one per 16.
//   * A tile is 128 rows, one bulk copy; a warp does the scores of 16 of them, the warps exchange maxima, leave p scale in shared memory as operands, and each adds up a
//     group's 64 features over its part of the tile.
//   * All tiles of all items are dealt evenly to the CTAs in one line, so that ragged batches balance; an item cut by a border leaves records that kv4_merge joins in order.
#include "kv4.cuh"

#define KA_THREADS 256
#define KA_WARPS 8

__device__ __forceinline__ void ka_mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
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
// fp16 pairs of (x, y) and of what the rounding left
__device__ __forceinline__ void ka_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = ka_pack(x, y);
    const float2 h = ka_pair(hi);
    lo = ka_pack(x - h.x, y - h.y);
}
// 2^(a - e) for scales below 2^(e + 1), whose fp16 bits are at most `bits`; scales below 2^-14 count as that
__device__ __forceinline__ float ka_against(int a, uint32_t bits) { return ka_pow2(a + 15 - max((int)(bits >> 10), 1)); }

struct ka_item { int r, kv, z, tile, tiles; }; // a place in the line of tiles

template <int D, int MT>
struct ka {
    static constexpr int S = D / 64, PARTS = KA_WARPS / S, COLS = LB_KV4_COLS(MT), BLK = LB_KV4_BLOCK(D), NS = LB_KV4_STAGES(D, MT);
    struct alignas(128) smem {
        unsigned char ring[NS][8 * BLK];
        uint4 q[MT][4 * S][32];         // queries as operands of the products: step 4 group + 2 word + u
        uint4 p[S][MT][8][32];          // p scale, likewise: [group][..][16 rows of the tile]
        uint2 qsum[MT][32];             // sums of a query's groups as the operand that meets (scale, lowest)
        float part[KA_WARPS][COLS][S + 1];
        float max[COLS][KA_WARPS];
        float factor[COLS], m[COLS], l[COLS], low[COLS][S];
        uint2 scale[KA_WARPS];
        uint64_t full[NS];
        uint32_t pre[LB_KV4_REQS + 1];  // tiles before request r
        int len[LB_KV4_REQS], n[LB_KV4_REQS], start[LB_KV4_REQS], seq[LB_KV4_REQS], limit[COLS];
        uint32_t warp_sum[KA_WARPS];
    };

    static_assert(sizeof(smem) <= LB_KV4_SMEM(D, MT) && LB_KV4_SMEM(D, MT) * LB_KV4_CTAS(D, MT) <= 227 * 1024 - 1024 * (LB_KV4_CTAS(D, MT) - 1), "shared memory");
    const lb_kv4_attn_params& p;
    smem& s;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, ft = lane & 3, G;

    __device__ __forceinline__ ka(const lb_kv4_attn_params& p_, smem& s_) : p(p_), s(s_), G(p_.HQ / p_.b.HKV) {}

    __device__ __forceinline__ int sets(int n) const { return (n * G + COLS - 1) / COLS; }

    // the requests, and how many tiles lie before each
    __device__ __forceinline__ uint32_t read_batch() {
        kv4_request q = {0, 0, 0, 0};
        if (t < p.b.n_reqs) q = kv4_get(p.b, t);
        const int len = q.n > 0 ? q.pos + q.n : 0;
        s.len[t] = len; s.n[t] = q.n; s.start[t] = q.start; s.seq[t] = q.seq;
        const uint32_t mine = q.n > 0 ? (uint32_t)((len + LB_KV4_TILE - 1) / LB_KV4_TILE) * p.b.HKV * sets(q.n) : 0u;
        uint32_t sum = mine;
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
    __device__ __forceinline__ ka_item place(uint32_t x) const {
        int lo = 0, hi = p.b.n_reqs - 1; // the last request with pre <= x that has tiles
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s.pre[mid] <= x) lo = mid;
            else hi = mid - 1;
        }
        ka_item it;
        it.r = lo;
        it.tiles = (s.len[lo] + LB_KV4_TILE - 1) / LB_KV4_TILE;
        const int local = (int)(x - s.pre[lo]), item = local / it.tiles, z = sets(s.n[lo]);
        it.tile = local - item * it.tiles;
        it.kv = item / z;
        it.z = item - it.kv * z;
        return it;
    }
    __device__ __forceinline__ void next(ka_item& it) const {
        if (++it.tile < it.tiles) return;
        it.tile = 0;
        if (++it.z < sets(s.n[it.r])) return;
        it.z = 0;
        if (++it.kv < p.b.HKV) return;
        it.kv = 0;
        do ++it.r; while (it.r < p.b.n_reqs && s.n[it.r] <= 0);
        it.tiles = it.r < p.b.n_reqs ? (s.len[it.r] + LB_KV4_TILE - 1) / LB_KV4_TILE : 0;
    }
    __device__ __forceinline__ int blocks(const ka_item& it) const { return min(8, (s.len[it.r] - it.tile * LB_KV4_TILE + 15) >> 4); }
    __device__ __forceinline__ void fetch(const ka_item& it, int slot) const {
        const uint32_t bytes = (uint32_t)blocks(it) * BLK;
        mbar_arrive_expect_tx(&s.full[slot], bytes);
        bulk_g2s_plain(s.ring[slot], p.b.cache + kv4_block(p.b, D, s.seq[it.r], it.kv, it.tile * LB_KV4_TILE), bytes, &s.full[slot]);
    }

    // the queries of an item's columns: norm, rotation, 11 bits, as operands; a warp takes whole columns, a lane 8 features
    __device__ __forceinline__ void queries(const ka_item& it) {
        const int n = s.n[it.r], pos = s.len[it.r] - n;
        for (int c = warp; c < COLS; c += KA_WARPS) {
            const int col = it.z * COLS + c, i = col / G, h = it.kv * G + col - i * G;
            const bool on = col < n * G, mine = on && lane < D / 8;
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.f;
            if (mine) kv4_load8(p.q, (size_t)(s.start[it.r] + i) * (size_t)p.row_stride + (size_t)h * (size_t)p.head_stride + lane * 8, p.type, p.wide, x);
            if (p.norm_w && on) {
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
                ss = warp_sum(ss);
                const float r = rsqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = x[j] * r * (mine ? bf16_bits_to_f32(p.norm_w[lane * 8 + j]) : 0.f);
            }
            if (mine && lane * 8 < p.rot_dims) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int f = lane * 4 + j;
                    if (2 * f < p.rot_dims) { // the angle in 64 bits, reduced to a turn; sine and cosine of at most pi in 32
                        const double a = (double)(pos + i) * p.freq[f];
                        float cs, sn;
                        sincosf((float)fma(-rint(a * 0.15915494309189535), 6.283185307179586, a), &sn, &cs);
                        const float u = x[2 * j], v = x[2 * j + 1];
                        x[2 * j] = u * cs - v * sn;
                        x[2 * j + 1] = u * sn + v * cs;
                    }
                }
            }
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            int e = 13 - ((__float_as_int(top) >> 23) - 127); // largest to [2^13, 2^14)
            e = top == 0.f ? 0 : min(120, max(-100, e));
            const float up = ka_pow2(e);
            float sum = 0.f;
            if (lane < D / 8) {
#pragma unroll
                for (int u = 0; u < 2; ++u) { // codes n0 n4 | n1 n5 of a word's lower bytes, n2 n6 | n3 n7: the second of a byte comes 2^4 too large
                    uint4 w;
                    ka_split(x[2 * u] * up, x[2 * u + 4] * up, w.x, w.y);
                    ka_split(x[2 * u + 1] * up * 0.0625f, x[2 * u + 5] * up * 0.0625f, w.z, w.w);
                    const float2 a = ka_pair(w.x), b = ka_pair(w.y), c2 = ka_pair(w.z), d = ka_pair(w.w);
                    sum += (a.x + a.y) + (b.x + b.y) + 16.f * ((c2.x + c2.y) + (d.x + d.y));
                    s.q[c >> 3][(lane >> 3) * 4 + 2 * (lane & 1) + u][(c & 7) * 4 + ((lane & 7) >> 1)] = w;
                }
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            sum = __shfl_sync(0xffffffffu, sum, (lane & 3) * 8); // of group lane % 4, at most 2^20
            if (lane < 4) {
                uint2 w;
                ka_split(0.f, lane < S ? sum * 0.015625f : 0.f, w.x, w.y);
                s.qsum[c >> 3][(c & 7) * 4 + lane] = w;
            }
            if (lane == 0) {
                s.factor[c] = ka_pow2(24 - e) * (rsqrtf((float)D) * 1.4426950408889634f); // scores in log2 units
                s.limit[c] = on ? pos + i : -1;
            }
        }
    }

    float m[MT];            // maximum of column 8 mt + g, before its factor
    float low[MT][4];       // of this warp's rows, columns 8 mt + g in two terms: sums of p lowest of groups 2 ft, 2 ft + 1; ft = 2: the sum of p
    float acc[MT][8][4];    // [feature 8 (2 ft, 2 ft + 1) + j of the group], likewise in two terms
    uint2 top;              // fp16 bits of the groups' largest scales so far

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            m[mt] = -INFINITY;
            low[mt][0] = low[mt][1] = low[mt][2] = low[mt][3] = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[mt][j][0] = acc[mt][j][1] = acc[mt][j][2] = acc[mt][j][3] = 0.f;
        }
        top = make_uint2(0, 0);
    }

    // one tile; false: the wait for it gave up
    __device__ __forceinline__ bool tile(const ka_item& it, int slot, uint32_t parity, bool more, const ka_item& ahead, int ahead_slot) {
        const unsigned char* ring = s.ring[slot];
        const int len = s.len[it.r], first_new = len - s.n[it.r];
        const int nb = blocks(it), row0 = it.tile * LB_KV4_TILE + warp * 16 + 4 * ft; // this thread's rows: row0 .. row0 + 3
        const bool edge = it.tile * LB_KV4_TILE + warp * 16 + 15 > first_new;           // rows that not every column sees, or that are not there
        const unsigned char* blk = ring + warp * BLK;
        float sc[MT][4];
        uint4 scale[S / 2 < 1 ? 1 : S / 2]; // values' scales of rows row0 .. row0 + 3 as fp16 pairs, two groups each
        uint2 mx = make_uint2(0, 0);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) sc[mt][0] = sc[mt][1] = sc[mt][2] = sc[mt][3] = -INFINITY;
#pragma unroll
        for (int q = 0; q < (S + 1) / 2; ++q) scale[q] = make_uint4(0, 0, 0, 0);
        const bool landed = mbar_wait(&s.full[slot], parity);
        if (warp < nb && landed) {
            {   // lowest sum(q)
                uint32_t b[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) b[i] = *reinterpret_cast<const uint32_t*>(blk + 16 * D + ((ft % S) * 16 + 4 * (g >> 1) + 2 * i + (g & 1)) * 4);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const uint2 a = s.qsum[mt][lane];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
                        ka_mma(d, make_uint4(a.x, a.y, 0u, 0u), b[i], 0u);
                        sc[mt][2 * i] = (d[0] + d[2]) * 3.814697265625e-06f; // 2^-18: the codes' 2^-24 over the sums' 2^-6
                        sc[mt][2 * i + 1] = (d[1] + d[3]) * 3.814697265625e-06f;
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < S; ++q) {
                const uint4 pr = *reinterpret_cast<const uint4*>(blk + 16 * D + (q * 16 + 4 * ft) * 4);
                float a[MT][2][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) a[mt][i][0] = a[mt][i][1] = a[mt][i][2] = a[mt][i][3] = 0.f;
                uint2 w[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) w[i] = *reinterpret_cast<const uint2*>(blk + ((i * S + q) * 32 + lane) * 8);
#pragma unroll
                for (int st = 0; st < 4; ++st)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const uint4 qa = s.q[mt][q * 4 + st][lane];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t v = (st < 2 ? w[i].x : w[i].y) >> (st & 1 ? 8 : 0);
                            ka_mma(a[mt][i], qa, v & 0x000f000fu, v & 0x00f000f0u);
                        }
                    }
                const float k0 = ka_pair(pr.x).x, k1 = ka_pair(pr.y).x, k2 = ka_pair(pr.z).x, k3 = ka_pair(pr.w).x;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    sc[mt][0] = fmaf(k0, a[mt][0][0] + a[mt][0][2], sc[mt][0]);
                    sc[mt][1] = fmaf(k1, a[mt][0][1] + a[mt][0][3], sc[mt][1]);
                    sc[mt][2] = fmaf(k2, a[mt][1][0] + a[mt][1][2], sc[mt][2]);
                    sc[mt][3] = fmaf(k3, a[mt][1][1] + a[mt][1][3], sc[mt][3]);
                }
                uint4 vr = *reinterpret_cast<const uint4*>(blk + 17 * D + (q * 16 + 4 * ft) * 4);
                if (edge) vr = there(vr, row0, len);
                uint32_t& s01 = q & 1 ? scale[q >> 1].z : scale[q >> 1].x;
                uint32_t& s23 = q & 1 ? scale[q >> 1].w : scale[q >> 1].y;
                s01 = __byte_perm(vr.x, vr.y, 0x5410);
                s23 = __byte_perm(vr.z, vr.w, 0x5410);
            }
            // the largest scale of each group over these rows; scales are not negative
            auto most = [&](uint4 v) {
                if (edge) { // a NaN has no say: columns before its row are not to notice it
                    v.x &= __vcmpltu2(v.x, 0x7c007c00u); v.y &= __vcmpltu2(v.y, 0x7c007c00u);
                    v.z &= __vcmpltu2(v.z, 0x7c007c00u); v.w &= __vcmpltu2(v.w, 0x7c007c00u);
                }
                const uint32_t a = __vmaxu2(v.x, v.y), b = __vmaxu2(v.z, v.w);
                return __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
            };
            mx.x = most(scale[0]);
            if (S > 2) mx.y = most(scale[S / 2 < 1 ? 0 : S / 2 - 1]);
            if (edge) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const int lim = s.limit[8 * mt + g];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (row0 + i > lim) sc[mt][i] = -INFINITY;
                }
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float v = fmaxf(fmaxf(sc[mt][0], sc[mt][1]), fmaxf(sc[mt][2], sc[mt][3]));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
            if (ft == 0) s.max[8 * mt + g][warp] = v;
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            mx.x = __vmaxu2(mx.x, __shfl_xor_sync(0xffffffffu, mx.x, o));
            if (S > 2) mx.y = __vmaxu2(mx.y, __shfl_xor_sync(0xffffffffu, mx.y, o));
        }
        if (lane == 0) s.scale[warp] = mx;
        if (__syncthreads_or(!landed)) return false;
        // everybody is done with the tile before: its slot is free
        if (t == 0 && more) fetch(ahead, ahead_slot);
        const uint2 old = top;
#pragma unroll
        for (int w = 0; w < KA_WARPS; ++w) {
            const uint2 v = s.scale[w];
            top.x = __vmaxu2(top.x, v.x);
            if (S > 2) top.y = __vmaxu2(top.y, v.y);
        }
        const int group = warp % S, part = warp / S;
        auto bits = [](const uint2& v, int q) { return ((q & 2 ? v.y : v.x) >> (16 * (q & 1))) & 0xffffu; };
        const float shrink = ka_against(0, bits(top, group)) * ka_pow2(max((int)(bits(old, group) >> 10), 1) - 15); // this warp's group is taken against a larger scale from here on
        float corr[MT];
        uint2 hi[MT], lo[MT]; // probabilities, times 2^14
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float* row = s.max[8 * mt + g];
            const float4 a = *reinterpret_cast<const float4*>(row), b = *reinterpret_cast<const float4*>(row + 4);
            const float f = s.factor[8 * mt + g], now = fmaxf(fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w))), m[mt]);
            const float less = now == -INFINITY ? 0.f : -now * f; // a column that has seen nothing yet
            corr[mt] = ka_exp2(fmaf(m[mt], f, less));
            m[mt] = now;
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[mt][i] = ka_exp2(fmaf(sc[mt][i], f, less + 14.f));
            ka_split(sc[mt][0], sc[mt][1], hi[mt].x, lo[mt].x);
            ka_split(sc[mt][2], sc[mt][3], hi[mt].y, lo[mt].y);
        }
        if (__any_sync(0xffffffffu, differs(corr, shrink))) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float c = corr[mt] * shrink;
#pragma unroll
                for (int i = 0; i < 4; ++i) low[mt][i] *= corr[mt];
#pragma unroll
                for (int j = 0; j < 8; ++j) { acc[mt][j][0] *= c; acc[mt][j][1] *= c; acc[mt][j][2] *= c; acc[mt][j][3] *= c; }
            }
        }
        if (warp < nb) {
            uint4 vr = *reinterpret_cast<const uint4*>(blk + 17 * D + ((g % S) * 16 + 4 * ft) * 4);
            if (edge) { // NaNs of rows that a column does not see must not reach it as 0 times NaN; where it does, p scale is NaN
                vr = there(vr, row0, len);
                vr.x = lowest_or_0(vr.x); vr.y = lowest_or_0(vr.y); vr.z = lowest_or_0(vr.z); vr.w = lowest_or_0(vr.w);
            }
            const uint32_t b0 = g == 4 ? 0x3c003c00u : __byte_perm(vr.x, vr.y, 0x7632), b1 = g == 4 ? 0x3c003c00u : __byte_perm(vr.z, vr.w, 0x7632);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) ka_mma(low[mt], make_uint4(hi[mt].x, lo[mt].x, hi[mt].y, lo[mt].y), b0, b1);
#pragma unroll
            for (int q = 0; q < S; ++q) {
                const float up = ka_against(-1, bits(top, q));
                const float2 s01 = ka_pair(q & 1 ? scale[q >> 1].z : scale[q >> 1].x), s23 = ka_pair(q & 1 ? scale[q >> 1].w : scale[q >> 1].y);
                const float v[4] = {s01.x * up, s01.y * up, s23.x * up, s23.y * up};
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = sc[mt][i] * v[i];
                    if (edge) {
                        const int lim = s.limit[8 * mt + g];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (row0 + i > lim) w[i] = 0.f;
                    }
                    uint4 o;
                    ka_split(w[0], w[1], o.x, o.y);
                    ka_split(w[2], w[3], o.z, o.w);
                    s.p[q][mt][warp][lane] = o;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int b = part * S + k;
            if (b >= nb) break;
            const uint4 v = *reinterpret_cast<const uint4*>(ring + b * BLK + 8 * D + group * 512 + lane * 16);
            const uint32_t a0 = __byte_perm(v.x, v.y, 0x5410), a1 = __byte_perm(v.x, v.y, 0x7632), c0 = __byte_perm(v.z, v.w, 0x5410), c1 = __byte_perm(v.z, v.w, 0x7632);
            uint4 pa[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) pa[mt] = s.p[group][mt][b][lane];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint32_t x = (j < 4 ? a0 : a1) >> (j & 2 ? 8 : 0), y = (j < 4 ? c0 : c1) >> (j & 2 ? 8 : 0);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    ka_mma(acc[mt][j], pa[mt], x & 0x000f000fu, y & 0x000f000fu);
                    ka_mma(acc[mt][j + 1], pa[mt], x & 0x00f000f0u, y & 0x00f000f0u);
                }
            }
        }
        return true;
    }
    static __device__ __forceinline__ bool differs(const float (&corr)[MT], float shrink) {
        bool d = shrink != 1.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) d |= corr[mt] != 1.f;
        return d;
    }
    // (scale, lowest) of four rows, of those that are there
    static __device__ __forceinline__ uint4 there(uint4 v, int row0, int len) {
        return make_uint4(row0 < len ? v.x : 0u, row0 + 1 < len ? v.y : 0u, row0 + 2 < len ? v.z : 0u, row0 + 3 < len ? v.w : 0u);
    }
    static __device__ __forceinline__ uint32_t lowest_or_0(uint32_t pair) { return (pair & 0x7fff0000u) < 0x7c000000u ? pair : 0u; }

    // The item's columns, whole or this CTA's share of them: out, or a record.  `first`: the item's first tile was this CTA's, `last`: its last
    __device__ __forceinline__ void finish(const ka_item& it, bool first, bool last) {
        float* sum = reinterpret_cast<float*>(&s.p[0][0][0][0]); // [COLS][D]
        const int group = warp % S, part = warp / S, cols = min(COLS, s.n[it.r] * G - it.z * COLS);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const int c = 8 * mt + g;
            if (2 * ft < S) s.part[warp][c][2 * ft] = low[mt][0] + low[mt][2];
            if (2 * ft + 1 < S) s.part[warp][c][2 * ft + 1] = low[mt][1] + low[mt][3];
            if (ft == 2) s.part[warp][c][S] = low[mt][0] + low[mt][2];
            if (ft == 0 && warp == 0) s.m[c] = m[mt] == -INFINITY ? m[mt] : m[mt] * s.factor[c];
        }
        const int e = max((int)(((group & 2 ? top.y : top.x) >> (16 * (group & 1)) & 0xffffu) >> 10), 1) - 15;
        const float even = ka_pow2(e + 25), odd = ka_pow2(e + 21); // 2^24 (2^20) over 2^(-1 - e)
        for (int turn = 0; turn < PARTS; ++turn) { // the parts of a tile one after the other
            __syncthreads();
            if (part == turn)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float& x = sum[(8 * mt + g) * D + group * 64 + 8 * (2 * ft + i) + j];
                            const float y = (acc[mt][j][i] + acc[mt][j][2 + i]) * (j & 1 ? odd : even);
                            x = turn ? x + y : y;
                        }
        }
        __syncthreads();
        for (int o = t; o < COLS * (S + 1); o += KA_THREADS) {
            const int c = o / (S + 1), q = o - c * (S + 1);
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < KA_WARPS; ++w) v += s.part[w][c][q];
            if (q == S) s.l[c] = v;
            else s.low[c][q] = v;
        }
        __syncthreads();
        if (first && last) {
            for (int o = t; o < cols * D; o += KA_THREADS) {
                const int c = o / D, f = o - c * D, col = it.z * COLS + c, i = col / G, h = it.kv * G + col - i * G;
                const size_t row = (size_t)(s.start[it.r] + i);
                float v = (sum[o] + s.low[c][f >> 6]) / s.l[c];
                if (p.gate) v *= sigmoidf_dev(kv4_load1(p.gate, row * (size_t)p.row_stride + (size_t)h * (size_t)p.head_stride + f, p.type));
                p.out[(row * p.HQ + h) * D + f] = __half_as_ushort(__float2half_rn(v));
            }
        } else {
            float* rec = p.records + ((size_t)blockIdx.x * 2 + (first ? 1 : 0)) * COLS * LB_KV4_REC(D);
            for (int o = t; o < cols * D; o += KA_THREADS) {
                const int c = o / D, f = o - c * D;
                rec[c * LB_KV4_REC(D) + f] = sum[o] + s.low[c][f >> 6];
            }
            if (t < cols) {
                rec[t * LB_KV4_REC(D) + D] = s.m[t];
                rec[t * LB_KV4_REC(D) + D + 1] = s.l[t];
            }
        }
        __syncthreads(); // the sums' place and the queries are free for the next item
    }

    __device__ __forceinline__ void body() {
        if (t == 0) {
#pragma unroll
            for (int i = 0; i < NS; ++i) mbar_init(&s.full[i], 1);
            mbar_fence_init();
        }
        pdl_wait();
        const uint32_t total = read_batch(); // its barriers also show the mbarriers to everybody
        const uint32_t ctas = min(gridDim.x, total);
        lb_kv4_join* join = p.joins + blockIdx.x;
        if (blockIdx.x >= ctas) {
            if (t == 0) join->first = -1;
            return;
        }
        const uint32_t x0 = (uint32_t)((uint64_t)blockIdx.x * total / ctas), x1 = (uint32_t)((uint64_t)(blockIdx.x + 1) * total / ctas);
        ka_item it = place(x0), ahead = it;
        uint32_t fetched = x0;
        if (t == 0) {
            for (; fetched < x1 && fetched < x0 + NS - 1; ++fetched) {
                if (fetched > x0) next(ahead);
                fetch(ahead, (int)(fetched - x0));
            }
            // does an item begin in the CTA before and go on here?
            lb_kv4_join j;
            j.first = -1;
            const uint32_t begin = x0 - (uint32_t)it.tile, end = begin + (uint32_t)it.tiles;
            if (it.tile > 0 && begin >= (uint32_t)((uint64_t)(blockIdx.x - 1) * total / ctas)) {
                j.first = (int)blockIdx.x - 1;
                j.last = (int)(((uint64_t)end * ctas - 1) / total); // the CTA of tile end - 1: the last c with c total / ctas <= end - 1
                j.row0 = s.start[it.r];
                j.kv = it.kv;
                j.col0 = it.z * COLS;
                j.cols = min(COLS, s.n[it.r] * G - j.col0);
            }
            *join = j;
        }
        int slot = 0;
        uint32_t parity = 0;
        bool first = true;
        for (uint32_t x = x0; x < x1; ++x) {
            if (x == x0 || it.tile == 0) {
                first = it.tile == 0;
                queries(it);
                begin();
                __syncthreads();
            }
            const bool more = fetched < x1;
            if (t == 0 && more) next(ahead);
            const int ahead_slot = slot ? slot - 1 : NS - 1;
            if (!tile(it, slot, parity, more, ahead, ahead_slot)) { // a copy never landed: say so, let the others land, leave
                if (t == 0) {
                    atomicExch(p.b.status, KV_FAIL_FULL);
                    for (uint32_t y = x; y < fetched; ++y) {
                        mbar_wait(&s.full[slot], parity);
                        if (++slot == NS) { slot = 0; parity ^= 1u; }
                    }
                }
                __syncthreads();
                return;
            }
            if (t == 0 && more) ++fetched;
            if (++slot == NS) { slot = 0; parity ^= 1u; }
            if (it.tile == it.tiles - 1 || x == x1 - 1) {
                __syncthreads();
                finish(it, first, it.tile == it.tiles - 1);
            }
            if (x + 1 < x1) next(it);
        }
        pdl_launch_dependents();
    }
};

#define KA_KERNEL(D, MT)                                                                                                                             \
    extern "C" __global__ void __launch_bounds__(KA_THREADS, LB_KV4_CTAS(D, MT)) kv4_attn_##D##_##MT(const __grid_constant__ lb_kv4_attn_params p) {   \
        extern __shared__ __align__(128) unsigned char ka_sm[];                                                                                     \
        ka<D, MT> k(p, *reinterpret_cast<ka<D, MT>::smem*>(ka_sm));                                                                                  \
        k.body();                                                                                                                                    \
    }
KA_KERNEL(64, 1)
KA_KERNEL(128, 1)
KA_KERNEL(256, 1)
KA_KERNEL(64, 2)
KA_KERNEL(128, 2)
KA_KERNEL(256, 2)
KA_KERNEL(64, 4)
KA_KERNEL(128, 4)
KA_KERNEL(256, 4)

// Joins the records of the items that were cut.  Every CTA lists the joins; (join, column) pairs are dealt to the CTAs.  Records are added in the order of the rows, in runs
// of neighbours side by side, so results are the same from run to run.
#define KM_THREADS 1024
#define KM_JOINS 512 /* CTAs of the attention kernel at most */
template <int D>
__device__ __forceinline__ void kv4_merge_body(const lb_kv4_attn_params& p, int ctas, int slots) {
    constexpr int SUB = KM_THREADS / D; // runs of records side by side
    __shared__ float red[3][KM_THREADS];
    __shared__ int s_join[KM_JOINS], s_before[KM_JOINS + 1], s_warp[KM_JOINS / 32][2];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    pdl_wait();
    int cols = 0;
    if (t < ctas && p.joins[t].first >= 0) cols = p.joins[t].cols;
    const uint32_t on = __ballot_sync(0xffffffffu, cols > 0);
    int sum = cols;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
    }
    if (lane == 31 && warp < KM_JOINS / 32) {
        s_warp[warp][0] = __popc(on);
        s_warp[warp][1] = sum;
    }
    __syncthreads();
    int joins = 0, pairs = 0, at = __popc(on & ((1u << lane) - 1u)), before = sum - cols;
#pragma unroll
    for (int w = 0; w < KM_JOINS / 32; ++w) {
        if (w == warp) { at += joins; before += pairs; }
        joins += s_warp[w][0];
        pairs += s_warp[w][1];
    }
    if (cols > 0) {
        s_join[at] = t;
        s_before[at] = before;
    }
    __syncthreads();
    const int f = t % D, sub = t / D, G = p.HQ / p.b.HKV;
    int k = 0;
    for (int pair = blockIdx.x; pair < pairs; pair += gridDim.x) {
        while (k + 1 < joins && s_before[k + 1] <= pair) ++k;
        const lb_kv4_join j = p.joins[s_join[k]];
        const int c = pair - s_before[k], per = (j.last - j.first + SUB) / SUB; // records of a run
        float M = -INFINITY, L = 0.f, A = 0.f;
        const int b0 = j.first + sub * per, b1 = min(j.last + 1, b0 + per);
        for (int b = b0; b < b1; b += 8) {
            float mv[8], lv[8], av[8], mx = M;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool there = b + i < b1;
                const float* rec = p.records + (((size_t)(there ? b + i : b) * 2 + (b + i == j.first ? 1 : 0)) * slots + c) * LB_KV4_REC(D);
                mv[i] = there ? __ldcg(rec + D) : -INFINITY;
                lv[i] = there ? __ldcg(rec + D + 1) : 0.f;
                av[i] = there ? __ldcg(rec + f) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) mx = fmaxf(mx, mv[i]);
            const float use = mx == -INFINITY ? 0.f : mx, w = ka_exp2(M - use);
            L *= w;
            A *= w;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = ka_exp2(mv[i] - use);
                L = fmaf(lv[i], v, L);
                A = fmaf(av[i], v, A);
            }
            M = mx;
        }
        red[0][t] = M;
        red[1][t] = L;
        red[2][t] = A;
        __syncthreads();
        if (sub == 0) {
            float mx = M;
#pragma unroll
            for (int q = 1; q < SUB; ++q) mx = fmaxf(mx, red[0][q * D + f]);
            const float use = mx == -INFINITY ? 0.f : mx;
            L = A = 0.f;
#pragma unroll
            for (int q = 0; q < SUB; ++q) {
                const float v = ka_exp2(red[0][q * D + f] - use);
                L = fmaf(red[1][q * D + f], v, L);
                A = fmaf(red[2][q * D + f], v, A);
            }
            const int col = j.col0 + c, i = col / G, h = j.kv * G + col - i * G;
            const size_t row = (size_t)(j.row0 + i);
            float v = A / L;
            if (p.gate) v *= sigmoidf_dev(kv4_load1(p.gate, row * (size_t)p.row_stride + (size_t)h * (size_t)p.head_stride + f, p.type));
            p.out[(row * p.HQ + h) * D + f] = __half_as_ushort(__float2half_rn(v));
        }
        __syncthreads();
    }
}
extern "C" __global__ void __launch_bounds__(KM_THREADS) kv4_merge_64(const __grid_constant__ lb_kv4_attn_params p, int ctas, int slots) { kv4_merge_body<64>(p, ctas, slots); }
extern "C" __global__ void __launch_bounds__(KM_THREADS) kv4_merge_128(const __grid_constant__ lb_kv4_attn_params p, int ctas, int slots) { kv4_merge_body<128>(p, ctas, slots); }
extern "C" __global__ void __launch_bounds__(KM_THREADS) kv4_merge_256(const __grid_constant__ lb_kv4_attn_params p, int ctas, int slots) { kv4_merge_body<256>(p, ctas, slots); }
