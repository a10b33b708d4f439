// Grouped-query attention of a batch's new tokens over the 4-bit KV cache (layout: kv4.cuh).
//   out[j, h] = sum_t p_t v_t * sigmoid(gate[j, h]),  p = softmax over the rows t <= position of token j of  q[j, h] . k_t / sqrt(D),
// q normalised and rotated as the decode attention does it.  The columns of an item (a request's KV head) are its new tokens times the query heads that share the
// head; they are the 16 rows of the products (MT times 16), the cache's rows their other side.
//   * The codes are the products' operands as they are: four bits in the low end of a half are the subnormal c 2^-24, four bits above them c 2^-20, and the tensor cores
//     take subnormals exactly.  A word of 8 codes costs a shift and four ANDs, no conversion; the 2^4 between neighbours is taken out of the query (keys) and of the sums
//     (values).  scores = sum over groups of scale_t (q . c_t) + lowest_t sum(q); read-out = sum of (p_t scale_t) c_t + (p_t lowest_t), the second terms in fp32.
//   * q goes in as fp16, a row scaled by a power of two to [2^13, 2^14) at its largest: 11 bits, as a fp16 projection gives them.  p scale goes in as fp16 too, scaled by a
//     power of two per group and slice of the cache (its largest scale so far becomes [2^13, 2^14)), so that weights keep their 11 bits down to 2^-27 of the largest.
//     Scores, running maxima, sums and read-outs are fp32; the output is fp16, what lb_gemm_int4 takes.
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
// exponent of the largest scale, whose fp16 bits are `bits` (16 of them): 2^e <= scale
__device__ __forceinline__ int ka_exponent(uint32_t bits) {
    const int e = (__float_as_int(__half2float(__ushort_as_half((unsigned short)bits))) >> 23) - 127;
    return e < -40 ? -40 : e;
}

struct ka_item { int r, kv, z, tile, tiles; }; // a place in the line of tiles

template <int D, int MT>
struct ka {
    static constexpr int S = D / 64, PARTS = KA_WARPS / S, COLS = 16 * MT, BLK = LB_KV4_BLOCK(D), NS = LB_KV4_STAGES(D, MT);
    struct alignas(128) smem {
        unsigned char ring[NS][8 * BLK];
        uint4 q[MT][4 * S][32];         // queries as operands of the products: step 4 group + 2 word + u
        uint4 p[S][MT][8][32];          // p scale, likewise: [group][..][16 rows of the tile]
        float part[KA_WARPS][COLS][S + 1];
        float max[COLS][KA_WARPS];
        float factor[COLS], qsum[COLS][S];
        float m[COLS], l[COLS], low[COLS][S];
        uint2 scale[KA_WARPS];
        uint64_t full[NS];
        uint32_t pre[LB_KV4_REQS + 1];  // tiles before request r
        int len[LB_KV4_REQS], n[LB_KV4_REQS], start[LB_KV4_REQS], seq[LB_KV4_REQS], limit[COLS];
        uint32_t warp_sum[KA_WARPS];
    };

    static_assert(sizeof(smem) <= LB_KV4_SMEM(D, MT) && LB_KV4_SMEM(D, MT) * LB_KV4_CTAS(MT) <= 227 * 1024 - 1024 * LB_KV4_CTAS(MT), "shared memory");
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
        int lo = 0, hi = LB_KV4_REQS - 1; // the last request with pre <= x that has tiles
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
        do ++it.r; while (it.r < LB_KV4_REQS && s.n[it.r] <= 0);
        it.tiles = it.r < LB_KV4_REQS ? (s.len[it.r] + LB_KV4_TILE - 1) / LB_KV4_TILE : 0;
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
                    const uint32_t even = ka_pack(x[2 * u] * up, x[2 * u + 4] * up), odd = ka_pack(x[2 * u + 1] * up * 0.0625f, x[2 * u + 5] * up * 0.0625f);
                    const float2 a = ka_pair(even), b = ka_pair(odd);
                    sum += (a.x + a.y) + 16.f * (b.x + b.y);
                    uint32_t* dst = reinterpret_cast<uint32_t*>(&s.q[c >> 4][(lane >> 3) * 4 + 2 * (lane & 1) + u][(c & 7) * 4 + ((lane & 7) >> 1)]) + ((c >> 3) & 1);
                    dst[0] = even;
                    dst[2] = odd;
                }
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane < D / 8 && (lane & 7) == 0) s.qsum[c][lane >> 3] = sum * ka_pow2(-24);
            if (lane == 0) {
                s.factor[c] = ka_pow2(24 - e) * (rsqrtf((float)D) * 1.4426950408889634f); // scores in log2 units
                s.limit[c] = on ? pos + i : -1;
            }
        }
    }

    float m[2 * MT], l[2 * MT], low[2 * MT][S]; // of columns 16 mt + g (even) and + 8 (odd): maximum; sums over this thread's rows
    float acc[MT][8][4];                        // [feature 8 g' + j of the group][columns]
    int ex[S];                                  // exponent that a group's scales are taken against

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
#pragma unroll
            for (int q = 0; q < S; ++q) low[i][q] = 0.f;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[mt][j][0] = acc[mt][j][1] = acc[mt][j][2] = acc[mt][j][3] = 0.f;
#pragma unroll
        for (int q = 0; q < S; ++q) ex[q] = -40;
    }

    // one tile; false: the wait for it gave up
    __device__ __forceinline__ bool tile(const ka_item& it, int slot, uint32_t parity, bool more, const ka_item& ahead, int ahead_slot) {
        const bool landed = mbar_wait(&s.full[slot], parity);
        const unsigned char* ring = s.ring[slot];
        const int nb = blocks(it), row0 = it.tile * LB_KV4_TILE + warp * 16 + 4 * ft, len = s.len[it.r]; // this thread's rows: row0 .. row0 + 3
        const unsigned char* blk = ring + warp * BLK;
        float sc[MT][2][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) sc[mt][i][0] = sc[mt][i][1] = sc[mt][i][2] = sc[mt][i][3] = 0.f;
        uint32_t top[2] = {0u, 0u};
        if (warp < nb && landed) {
#pragma unroll
            for (int q = 0; q < S; ++q) {
                const uint4 pr = *reinterpret_cast<const uint4*>(blk + 16 * D + (q * 16 + 4 * ft) * 4);
                const float2 k0 = ka_pair(pr.x), k1 = ka_pair(pr.y), k2 = ka_pair(pr.z), k3 = ka_pair(pr.w);
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
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const float q0 = s.qsum[16 * mt + g][q], q1 = s.qsum[16 * mt + 8 + g][q];
                    sc[mt][0][0] = fmaf(k0.x, a[mt][0][0], fmaf(k0.y, q0, sc[mt][0][0]));
                    sc[mt][0][1] = fmaf(k1.x, a[mt][0][1], fmaf(k1.y, q0, sc[mt][0][1]));
                    sc[mt][0][2] = fmaf(k0.x, a[mt][0][2], fmaf(k0.y, q1, sc[mt][0][2]));
                    sc[mt][0][3] = fmaf(k1.x, a[mt][0][3], fmaf(k1.y, q1, sc[mt][0][3]));
                    sc[mt][1][0] = fmaf(k2.x, a[mt][1][0], fmaf(k2.y, q0, sc[mt][1][0]));
                    sc[mt][1][1] = fmaf(k3.x, a[mt][1][1], fmaf(k3.y, q0, sc[mt][1][1]));
                    sc[mt][1][2] = fmaf(k2.x, a[mt][1][2], fmaf(k2.y, q1, sc[mt][1][2]));
                    sc[mt][1][3] = fmaf(k3.x, a[mt][1][3], fmaf(k3.y, q1, sc[mt][1][3]));
                }
                const uint4 vr = *reinterpret_cast<const uint4*>(blk + 17 * D + (q * 16 + 4 * ft) * 4);
                uint32_t mx = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t b = (i == 0 ? vr.x : i == 1 ? vr.y : i == 2 ? vr.z : vr.w) & 0xffffu; // scales are not negative; a NaN's group has no say here
                    if (row0 + i < len && b < 0x7c00u) mx = max(mx, b);
                }
                top[q >> 1] |= mx << (16 * (q & 1));
            }
        }
        float mx[2 * MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) { // columns 16 mt + g + 8 e: the scores of rows row0 .. row0 + 3
                const int c = 16 * mt + 8 * e + g, lim = warp < nb ? s.limit[c] : -1;
                const float f = s.factor[c];
                float v = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float& x = sc[mt][i >> 1][2 * e + (i & 1)];
                    x = row0 + i <= lim ? x * f : -INFINITY;
                    v = fmaxf(v, x);
                }
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
                mx[2 * mt + e] = v;
                if (ft == 0) s.max[c][warp] = v;
            }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            top[0] = __vmaxu2(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
            if (S > 2) top[1] = __vmaxu2(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
        }
        if (lane == 0) s.scale[warp] = make_uint2(top[0], top[1]);
        if (__syncthreads_or(!landed)) return false;
        // everybody is done with the tile before: its slot is free
        if (t == 0 && more) fetch(ahead, ahead_slot);
        float corr[2 * MT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            const float* row = s.max[16 * (i >> 1) + 8 * (i & 1) + g];
            const float4 a = *reinterpret_cast<const float4*>(row), b = *reinterpret_cast<const float4*>(row + 4);
            const float now = fmaxf(fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w))), m[i]);
            mx[i] = now == -INFINITY ? 0.f : now; // a column that has seen nothing yet
            corr[i] = ka_exp2(m[i] - mx[i]);
            m[i] = now;
            l[i] *= corr[i];
        }
        uint2 tp = s.scale[0];
#pragma unroll
        for (int w = 1; w < KA_WARPS; ++w) {
            const uint2 v = s.scale[w];
            tp.x = __vmaxu2(tp.x, v.x);
            if (S > 2) tp.y = __vmaxu2(tp.y, v.y);
        }
        const int group = warp % S, part = warp / S;
        float shrink = 1.f; // of this warp's group: its scales are taken against a larger one from here on
#pragma unroll
        for (int q = 0; q < S; ++q) {
            const int e = max(ex[q], ka_exponent(((q & 2 ? tp.y : tp.x) >> (16 * (q & 1))) & 0xffffu));
            if (q == group) shrink = ka_pow2(ex[q] - e);
            ex[q] = e;
        }
        // probabilities
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& x = sc[mt][i >> 1][2 * e + (i & 1)];
                    x = ka_exp2(x - mx[2 * mt + e]);
                    l[2 * mt + e] += x;
                }
#pragma unroll
        for (int q = 0; q < S; ++q) {
            uint4 vr = make_uint4(0, 0, 0, 0);
            if (warp < nb) vr = *reinterpret_cast<const uint4*>(blk + 17 * D + (q * 16 + 4 * ft) * 4);
            if (row0 + 3 >= len) { // rows behind the last one may hold anything
                if (row0 >= len) vr.x = 0;
                if (row0 + 1 >= len) vr.y = 0;
                if (row0 + 2 >= len) vr.z = 0;
                vr.w = 0;
            }
            if (row0 + 3 > len - s.n[it.r]) { // new rows, which not every column sees: a NaN's group reaches those that do, and no other by way of 0 times NaN
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t& v = i == 0 ? vr.x : i == 1 ? vr.y : i == 2 ? vr.z : vr.w;
                    if ((v & 0x7fffu) < 0x7c00u) continue;
                    v = 0;
#pragma unroll
                    for (int c = 0; c < 2 * MT; ++c)
                        if (row0 + i <= s.limit[16 * (c >> 1) + 8 * (c & 1) + g]) low[c][q] = NAN;
                }
            }
            const float2 v0 = ka_pair(vr.x), v1 = ka_pair(vr.y), v2 = ka_pair(vr.z), v3 = ka_pair(vr.w);
            const float up = ka_pow2(13 - ex[q]);
            const float s0 = v0.x * up, s1 = v1.x * up, s2 = v2.x * up, s3 = v3.x * up;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& lo = low[2 * mt + e][q];
                    lo = fmaf(sc[mt][0][2 * e], v0.y, fmaf(sc[mt][0][2 * e + 1], v1.y, fmaf(sc[mt][1][2 * e], v2.y, fmaf(sc[mt][1][2 * e + 1], v3.y, lo * corr[2 * mt + e]))));
                }
                if (warp < nb)
                    s.p[q][mt][warp][lane] = make_uint4(ka_pack(sc[mt][0][0] * s0, sc[mt][0][1] * s1), ka_pack(sc[mt][0][2] * s0, sc[mt][0][3] * s1),
                                                        ka_pack(sc[mt][1][0] * s2, sc[mt][1][1] * s3), ka_pack(sc[mt][1][2] * s2, sc[mt][1][3] * s3));
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float c0 = corr[2 * mt] * shrink, c1 = corr[2 * mt + 1] * shrink;
            if (__any_sync(0xffffffffu, c0 != 1.f || c1 != 1.f)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) { acc[mt][j][0] *= c0; acc[mt][j][1] *= c0; acc[mt][j][2] *= c1; acc[mt][j][3] *= c1; }
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

    // The item's columns, whole or this CTA's share of them: out, or a record.  `first`: the item's first tile was this CTA's, `last`: its last
    __device__ __forceinline__ void finish(const ka_item& it, bool first, bool last) {
        float* sum = reinterpret_cast<float*>(&s.p[0][0][0][0]); // [COLS][D]
        const int group = warp % S, part = warp / S, cols = min(COLS, s.n[it.r] * G - it.z * COLS);
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            const int c = 16 * (i >> 1) + 8 * (i & 1) + g;
            float v = l[i];
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            if (ft == 0) s.part[warp][c][S] = v;
#pragma unroll
            for (int q = 0; q < S; ++q) {
                v = low[i][q];
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                if (ft == 0) s.part[warp][c][q] = v;
            }
            if (ft == 0 && warp == 0) s.m[c] = m[i];
        }
        int e = 0;
#pragma unroll
        for (int q = 0; q < S; ++q)
            if (q == group) e = ex[q];
        const float even = ka_pow2(e + 11), odd = ka_pow2(e + 7); // 2^24 (2^20) over 2^(13 - e)
        for (int turn = 0; turn < PARTS; ++turn) { // the parts of a tile one after the other
            __syncthreads();
            if (part == turn)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float& x = sum[(16 * mt + g + (i & 2 ? 8 : 0)) * D + group * 64 + 8 * (2 * ft + (i & 1)) + j];
                            const float y = acc[mt][j][i] * (j & 1 ? odd : even);
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
                fetch(ahead, (int)(fetched - x0));
                next(ahead);
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
            if (t == 0 && more) {
                ++fetched;
                next(ahead);
            }
            if (++slot == NS) { slot = 0; parity ^= 1u; }
            if (it.tile == it.tiles - 1 || x == x1 - 1) {
                __syncthreads();
                finish(it, first, it.tile == it.tiles - 1);
            }
            next(it);
        }
        pdl_launch_dependents();
    }
};

#define KA_KERNEL(D, MT)                                                                                                                             \
    extern "C" __global__ void __launch_bounds__(KA_THREADS, LB_KV4_CTAS(MT)) kv4_attn_##D##_##MT(const __grid_constant__ lb_kv4_attn_params p) {   \
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

// Joins the records of the items that were cut: CTA (b, y) those of the item whose first cut is the border before CTA b, columns y, y + gridDim.y, ...
// Records are added in the order of the rows, so results are the same from run to run.
#define KM_THREADS 1024
template <int D>
__device__ __forceinline__ void kv4_merge_body(const lb_kv4_attn_params& p, int slots) {
    constexpr int SUB = KM_THREADS / D; // runs of records side by side
    __shared__ float red[3][KM_THREADS];
    pdl_wait();
    const lb_kv4_join j = p.joins[blockIdx.x];
    if (j.first < 0) return;
    const int f = threadIdx.x % D, sub = threadIdx.x / D, G = p.HQ / p.b.HKV, per = (j.last - j.first + SUB) / SUB; // records of a run
    for (int c = blockIdx.y; c < j.cols; c += gridDim.y) {
        float M = -INFINITY, L = 0.f, A = 0.f;
        const int b0 = j.first + sub * per, b1 = min(j.last + 1, b0 + per);
        for (int b = b0; b < b1; b += 8) {
            float mv[8], lv[8], av[8], mx = M;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool on = b + i < b1;
                const float* rec = p.records + (((size_t)(on ? b + i : b) * 2 + (b + i == j.first ? 1 : 0)) * slots + c) * LB_KV4_REC(D);
                mv[i] = on ? __ldcg(rec + D) : -INFINITY;
                lv[i] = on ? __ldcg(rec + D + 1) : 0.f;
                av[i] = on ? __ldcg(rec + f) : 0.f;
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
        red[0][threadIdx.x] = M;
        red[1][threadIdx.x] = L;
        red[2][threadIdx.x] = A;
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
extern "C" __global__ void __launch_bounds__(KM_THREADS) kv4_merge_64(const __grid_constant__ lb_kv4_attn_params p, int slots) { kv4_merge_body<64>(p, slots); }
extern "C" __global__ void __launch_bounds__(KM_THREADS) kv4_merge_128(const __grid_constant__ lb_kv4_attn_params p, int slots) { kv4_merge_body<128>(p, slots); }
extern "C" __global__ void __launch_bounds__(KM_THREADS) kv4_merge_256(const __grid_constant__ lb_kv4_attn_params p, int slots) { kv4_merge_body<256>(p, slots); }
