// Rows into and out of the 4-bit KV cache (layout: kv4.cuh).
#include "kv4.cuh"

#define KC_THREADS 256
#define KC_ROWS 16 // rows that a CTA looks up at a time

// Rows row0 .. row0 + n - 1 of a batch (n <= KC_ROWS): their sequences (-1: no request's, or given way to a later request's) and positions.  The requests' first look is kept in
// shared memory by kc_requests.  Barriers before and behind.
struct kc_batch { int start[LB_KV4_REQS], n[LB_KV4_REQS], seq[LB_KV4_REQS], pos[LB_KV4_REQS], row_seq[KC_ROWS], row_pos[KC_ROWS], row_req[KC_ROWS]; };
__device__ __forceinline__ void kc_requests(const lb_kv4_view& b, kc_batch& s) {
    const int t = threadIdx.x;
    kv4_request q = {0, 0, 0, 0};
    if (t < b.n_reqs) q = kv4_get(b, t);
    s.start[t] = q.start; s.n[t] = q.n; s.seq[t] = q.seq; s.pos[t] = q.pos;
}
template <bool LAST>
__device__ __forceinline__ void kc_rows(const lb_kv4_view& b, kc_batch& s, int row0, int n) {
    const int t = threadIdx.x, q_start = s.start[t], q_n = s.n[t], q_seq = s.seq[t], q_pos = s.pos[t];
    if (t < n) s.row_seq[t] = -1;
    __syncthreads();
    for (int i = max(0, q_start - row0); i < n && row0 + i < q_start + q_n; ++i) { // a row is one request's, unless `starts` is not ascending: then some request's that has it
        s.row_seq[i] = q_seq;
        s.row_pos[i] = q_pos + row0 + i - q_start;
        s.row_req[i] = t;
    }
    __syncthreads();
    if (LAST && b.n_reqs > 1) { // where two requests bring the same row of the same sequence, the later one's is stored
        uint32_t gone = 0;
        if (q_n > 0)
            for (int i = 0; i < n; ++i) gone |= (uint32_t)(s.row_seq[i] == q_seq && t > s.row_req[i] && s.row_pos[i] >= q_pos && s.row_pos[i] < q_pos + q_n) << i;
        __syncthreads();
        for (; gone; gone &= gone - 1) s.row_seq[__ffs(gone) - 1] = -1;
        __syncthreads();
    }
}

// The codes of 8 features: nearest to (x - lowest) / scale, halves to the even one.  The quotient is taken as a product with 1 / scale (from 32 bits, one step of Newton's); where that
// lies within 2^-21 of a half, which side it is on is decided by the division that the definition has.
__device__ __forceinline__ uint32_t kc_codes(const double (&x)[8], double lo, float scale) {
    constexpr double magic = 6755399441055744.0; // 1.5 * 2^52: what is added to it is rounded to a whole number
    const double s = (double)scale, guess = (double)(1.0f / scale), inv = fma(guess, fma(-s, guess, 1.0), guess);
    uint32_t word = 0;
    bool near = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const double y = (x[j] - lo) * inv, n = y + magic;
        near |= (__double2hiint(y - (n - magic)) & 0x7fffffff) >= 0x3fdffffe; // 1/2 - 2^-21 or more off
        word |= (uint32_t)min(max(__double2loint(n), 0), 15) << (4 * j);
    }
    if (near) {
        word = 0;
#pragma unroll 1
        for (int j = 0; j < 8; ++j) {
            double v = x[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) v = j == i ? x[i] : v;
            word |= (uint32_t)min(max(__double2loint((v - lo) / s + magic), 0), 15) << (4 * j);
        }
    }
    return word;
}

// A batch's new rows: keys normalised and rotated as the decode attention does it, keys and values rounded to 4 bits, stored at their positions.
// Everything between the input and the codes is in 64 bits: a code flips where a value's error reaches over a border, and at 2^-53 none does in practice, so the
// cache holds the codes of the exact rows whatever order an implementation computes in.  The (scale, lowest) pairs go to fp32 and then to fp16.
// A unit is one row's key or value vector of a head: D / 8 lanes with 8 features each, a group of 64 is 8 lanes.  A CTA takes `chunk` rows, KC_ROWS at a time: the requests are
// looked at once, sines and cosines are those of a row for all of its heads.  Bound by instructions, some 450 for 8 features of each of 32 lanes, 60 of them in 64 bits.  4001 rows of
// 4 heads of 256: 22 us; 32 rows, one for each of 32 sequences, 5 us.  A division for every code instead of a product took 1.4 times as long.
template <int D>
__device__ __forceinline__ void kv4_append_body(const lb_kv4_rows_params& p) {
    constexpr int L = D / 8, U = KC_THREADS / L; // lanes of a unit, units at a time
    __shared__ kc_batch s;
    __shared__ double2 s_rot[KC_ROWS * (D / 2)];  // cos, sin
    const int t = threadIdx.x, sub = t % L, per_row = 2 * p.b.HKV, half = p.rot_dims / 2, step_rows = U / per_row, step_at = U - step_rows * per_row;
    const int begin = blockIdx.x * p.chunk, end = min(p.b.rows, begin + p.chunk);
    pdl_wait();
    kc_requests(p.b, s);
    for (int row0 = begin; row0 < end; row0 += KC_ROWS) {
        const int rows = min(KC_ROWS, end - row0);
        kc_rows<true>(p.b, s, row0, rows);
        for (int i = t; i < rows * half; i += KC_THREADS) {
            const int r = i / half, f = i - r * half;
            if (s.row_seq[r] < 0) continue;
            double2 cs;
            sincos((double)s.row_pos[r] * p.freq[f], &cs.y, &cs.x);
            s_rot[r * (D / 2) + f] = cs;
        }
        __syncthreads();
        // units in the order (row, keys / values, head); the next one's features are on their way while this one is worked on
        float ahead[8];
        int r_next = (t / L) / per_row, at_next = t / L - r_next * per_row;
        auto load = [&] {
#pragma unroll
            for (int j = 0; j < 8; ++j) ahead[j] = 0.f;
            if (r_next < rows && s.row_seq[r_next] >= 0)
                kv4_load8(at_next >= p.b.HKV ? p.v : p.k, (size_t)(row0 + r_next) * (size_t)p.stride + (size_t)((at_next >= p.b.HKV ? at_next - p.b.HKV : at_next) * D + sub * 8), p.type, p.wide,
                          ahead);
        };
        load();
        for (int u0 = 0; u0 < rows * per_row; u0 += U) {
            const int r = min(r_next, rows - 1), part = at_next >= p.b.HKV, kv = part ? at_next - p.b.HKV : at_next;
            const bool on = r_next < rows && s.row_seq[r] >= 0;
            float in[8];
            double x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                in[j] = ahead[j];
                x[j] = (double)in[j];
            }
            r_next += step_rows;
            at_next += step_at;
            if (at_next >= per_row) { at_next -= per_row; ++r_next; }
            load();
            if (p.norm_w && __any_sync(0xffffffffu, part == 0)) {
                double ss = 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fma(x[j], x[j], ss);
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const double rms = rsqrt(ss * (1.0 / D) + p.eps);
                if (part == 0)
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = x[j] * rms * (double)bf16_bits_to_f32(p.norm_w[sub * 8 + j]);
            }
            if (part == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int f = sub * 4 + j;
                    if (f < half) {
                        const double2 cs = s_rot[r * (D / 2) + f];
                        const double a = x[2 * j], b = x[2 * j + 1];
                        x[2 * j] = a * cs.x - b * cs.y;
                        x[2 * j + 1] = a * cs.y + b * cs.x;
                    }
                }
            }
            float lo_f = INFINITY, size = 0.f, none = 0.f; // rounding keeps the order: the least of the rounded values is the least value rounded
            double hi = 0.0;
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = part ? in[j] : (float)x[j];
                lo_f = fminf(lo_f, v);
                size = fmaxf(size, fabsf(v));
                none = fmaf(v, 0.f, none); // a NaN if one of them is, or is infinite
                hi = j == 0 || x[j] > hi ? x[j] : hi;
            }
            if (size >= 65504.f || none != 0.f) { // what fp16 holds: a value beyond it is cut off
                hi = -65504.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    bad |= !(fabs(x[j]) <= 1.7976931348623157e308);
                    x[j] = fmin(fmax(x[j], -65504.0), 65504.0);
                    hi = fmax(hi, x[j]);
                }
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) {
                lo_f = fminf(lo_f, __shfl_xor_sync(0xffffffffu, lo_f, o));
                const double other = __shfl_xor_sync(0xffffffffu, hi, o);
                hi = other > hi ? other : hi;
            }
            bad = (__ballot_sync(0xffffffffu, bad) >> (t & 24)) & 0xffu; // of the group's eight lanes
            __half lowest = __float2half_rn(fminf(fmaxf(lo_f, -65504.f), 65504.f));
            const double lo = (double)__half2float(lowest);
            const double span = hi - lo, near = span * (1.0 / 15.0), step = fma(fma(-15.0, near, span), 1.0 / 15.0, near); // span / 15
            __half scale = __float2half_rn(fmaxf((float)step, 0.f));
            const float sf = __half2float(scale);
            const uint32_t word = sf > 0.f && !bad ? kc_codes(x, lo, sf) : 0u;
            if (bad) scale = lowest = __ushort_as_half(0x7fff); // a group with an infinity or a NaN stands for NaN
            if (on) {
                const int pos = s.row_pos[r], row = pos & 15;
                unsigned char* blk = p.b.cache + kv4_block(p.b, D, s.row_seq[r], kv, pos);
                *reinterpret_cast<uint32_t*>(blk + (part ? kv4_value_word(D, row, sub) : kv4_key_word(D, row, sub))) = word;
                if ((sub & 7) == 0) *reinterpret_cast<__half2*>(blk + kv4_pair(D, part, row, sub >> 3)) = __halves2half2(scale, lowest);
            }
        }
        __syncthreads(); // the rows have been read
    }
}

// 8 features of a row's key or value vector
template <int D>
__device__ __forceinline__ void kc_read(const lb_kv4_rows_params& p, const kc_batch& s, int token, int r, int part, int kv, int sub) {
    const int row = s.row_pos[r] & 15;
    const unsigned char* blk = p.b.cache + kv4_block(p.b, D, s.row_seq[r], kv, s.row_pos[r]);
    const uint32_t word = *reinterpret_cast<const uint32_t*>(blk + (part ? kv4_value_word(D, row, sub) : kv4_key_word(D, row, sub)));
    const float2 pair = __half22float2(*reinterpret_cast<const __half2*>(blk + kv4_pair(D, part, row, sub >> 3)));
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = fmaf(pair.x, (float)((word >> (4 * j)) & 15u), pair.y);
    const size_t o = ((size_t)token * p.b.HKV + kv) * D + sub * 8;
    void* out = const_cast<void*>(part ? p.v : p.k);
    if (p.type == 1) {
        float* f = reinterpret_cast<float*>(out) + o;
        if (p.wide) {
            *reinterpret_cast<float4*>(f) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(f + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = x[j];
        }
        return;
    }
    uint16_t h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = p.type == 0 ? __bfloat16_as_ushort(__float2bfloat16_rn(x[j])) : __half_as_ushort(__float2half_rn(x[j]));
    uint16_t* d = reinterpret_cast<uint16_t*>(out) + o;
    if (p.wide) {
        *reinterpret_cast<uint4*>(d) = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) d[j] = h[j];
    }
}

// The rows that a batch names, as the values that the cache stands for: lowest + scale * c with one rounding to the output's type.
template <int D>
__device__ __forceinline__ void kv4_read_body(const lb_kv4_rows_params& p) {
    constexpr int L = D / 8, U = KC_THREADS / L;
    __shared__ kc_batch s;
    const int t = threadIdx.x, sub = t % L, per_row = 2 * p.b.HKV, step_rows = U / per_row, step_at = U - step_rows * per_row, begin = blockIdx.x * p.chunk, end = min(p.b.rows, begin + p.chunk);
    pdl_wait();
    kc_requests(p.b, s);
    for (int row0 = begin; row0 < end; row0 += KC_ROWS) {
        const int rows = min(KC_ROWS, end - row0);
        kc_rows<false>(p.b, s, row0, rows);
        int r = (t / L) / per_row, at = t / L - r * per_row;
        while (r < rows) {
            const int part = at >= p.b.HKV;
            if (s.row_seq[r] >= 0) kc_read<D>(p, s, row0 + r, r, part, part ? at - p.b.HKV : at, sub);
            r += step_rows;
            at += step_at;
            if (at >= per_row) { at -= per_row; ++r; }
        }
        __syncthreads();
    }
}

#define KC_KERNELS(D)                                                                                                                                  \
    extern "C" __global__ void __launch_bounds__(KC_THREADS) kv4_append_##D(const __grid_constant__ lb_kv4_rows_params p) { kv4_append_body<D>(p); } \
    extern "C" __global__ void __launch_bounds__(KC_THREADS) kv4_read_##D(const __grid_constant__ lb_kv4_rows_params p) { kv4_read_body<D>(p); }
KC_KERNELS(64)
KC_KERNELS(128)
KC_KERNELS(256)
