// Rows into and out of the 4-bit KV cache (layout: kv4.cuh).
#include "kv4.cuh"

#define KC_THREADS 256

// A batch's new rows: keys normalised and rotated as the decode attention does it, keys and values rounded to 4 bits, stored at their positions.
// All arithmetic between the input and the codes is in 64 bits: a code flips where a value's error reaches over a border, and at 2^-53 none does in practice, so the
// cache holds the codes of the exact rows whatever order an implementation computes in.  The (scale, lowest) pairs go to fp32 and then to fp16.
// A unit is one row's key or value vector of a head: D / 8 lanes with 8 features each, a group of 64 is 8 lanes.  A CTA takes as many rows as fill it.
// Where two requests bring the same row of the same sequence, the later request's is the one that is stored.
template <int D>
__device__ __forceinline__ void kv4_append_body(const lb_kv4_rows_params& p) {
    constexpr int L = D / 8, U = KC_THREADS / L; // lanes of a unit, units at a time
    __shared__ int s_seq[U], s_pos[U], s_drop[U];
    __shared__ double2 s_rot[U * (D / 2)];       // cos, sin
    const int t = threadIdx.x, sub = t % L, per_row = 2 * p.b.HKV, rows = per_row < U ? U / per_row : 1, row0 = blockIdx.x * rows;
    if (t < rows) s_seq[t] = -1, s_drop[t] = 0;
    __syncthreads();
    pdl_wait();
    kv4_request q = {0, 0, 0, 0};
    if (t < p.b.n_reqs) q = kv4_get(p.b, t);
    for (int i = 0; i < rows; ++i) // requests cover rows once unless `starts` is not ascending: then any one of them has the row
        if (row0 + i >= q.start && row0 + i < q.start + q.n) {
            s_pos[i] = q.pos + row0 + i - q.start;
            s_seq[i] = q.seq | t << 20;
        }
    __syncthreads();
    if (q.n > 0)
        for (int i = 0; i < rows; ++i)
            if (s_seq[i] >= 0 && t > s_seq[i] >> 20 && q.seq == (s_seq[i] & 0xfffff) && s_pos[i] >= q.pos && s_pos[i] < q.pos + q.n) s_drop[i] = 1;
    const int half = p.rot_dims / 2;
    for (int i = t; i < rows * half; i += KC_THREADS) {
        const int r = i / half, f = i - r * half;
        if (s_seq[r] < 0) continue;
        double2 cs;
        sincos((double)s_pos[r] * p.freq[f], &cs.y, &cs.x);
        s_rot[r * (D / 2) + f] = cs;
    }
    __syncthreads();
    for (int u0 = 0; u0 < rows * per_row; u0 += U) {
        const int unit = min(u0 + t / L, rows * per_row - 1), r = unit / per_row, part = unit % per_row / p.b.HKV, kv = unit % p.b.HKV;
        const bool on = u0 + t / L < rows * per_row && s_seq[r] >= 0 && !s_drop[r];
        float in[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) in[j] = 0.f;
        if (on) kv4_load8(part ? p.v : p.k, (size_t)(row0 + r) * (size_t)p.stride + (size_t)kv * D + sub * 8, p.type, p.wide, in);
        double x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (double)in[j];
        if (part == 0) {
            if (p.norm_w) {
                double ss = 0.0;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss = fma(x[j], x[j], ss);
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const double rms = 1.0 / sqrt(ss / D + p.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = x[j] * rms * (double)bf16_bits_to_f32(p.norm_w[sub * 8 + j]);
            }
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
        double lo = x[0], hi = x[0];
        int bad = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            lo = fmin(lo, x[j]);
            hi = fmax(hi, x[j]);
            bad |= !(fabs(x[j]) <= 1.7976931348623157e308);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            lo = fmin(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmax(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            bad |= __shfl_xor_sync(0xffffffffu, bad, o);
        }
        lo = fmin(fmax(lo, -65504.0), 65504.0); // what fp16 holds: a value beyond it is cut off
        hi = fmin(fmax(hi, -65504.0), 65504.0);
        __half lowest = __float2half_rn((float)lo);
        lo = (double)__half2float(lowest);
        __half scale = __float2half_rn((float)fmax((hi - lo) / 15.0, 0.0));
        const double s = (double)__half2float(scale);
        uint32_t word = 0;
        if (s > 0.0 && !bad) {
#pragma unroll
            for (int j = 0; j < 8; ++j) word |= (uint32_t)fmin(fmax(rint((x[j] - lo) / s), 0.0), 15.0) << (4 * j);
        }
        if (bad) scale = lowest = __ushort_as_half(0x7fff); // a group with an infinity or a NaN stands for NaN
        if (on) {
            const int row = s_pos[r] & 15;
            unsigned char* blk = p.b.cache + kv4_block(p.b, D, s_seq[r] & 0xfffff, kv, s_pos[r]);
            *reinterpret_cast<uint32_t*>(blk + (part ? kv4_value_word(D, row, sub) : kv4_key_word(D, row, sub))) = word;
            if ((sub & 7) == 0) *reinterpret_cast<__half2*>(blk + kv4_pair(D, part, row, sub >> 3)) = __halves2half2(scale, lowest);
        }
    }
}

// The rows that a batch names, as the values that the cache stands for: lowest + scale * c with one rounding to the output's type.
template <int D>
__device__ __forceinline__ void kv4_read_body(const lb_kv4_rows_params& p) {
    constexpr int L = D / 8, U = KC_THREADS / L;
    __shared__ int s_seq[U], s_pos[U];
    const int t = threadIdx.x, sub = t % L, per_row = 2 * p.b.HKV, rows = per_row < U ? U / per_row : 1, row0 = blockIdx.x * rows;
    if (t < rows) s_seq[t] = -1;
    __syncthreads();
    pdl_wait();
    kv4_request q = {0, 0, 0, 0};
    if (t < p.b.n_reqs) q = kv4_get(p.b, t);
    for (int i = 0; i < rows; ++i)
        if (row0 + i >= q.start && row0 + i < q.start + q.n) {
            s_pos[i] = q.pos + row0 + i - q.start;
            s_seq[i] = q.seq;
        }
    __syncthreads();
    for (int unit = t / L; unit < rows * per_row; unit += U) {
        const int r = unit / per_row, part = unit % per_row / p.b.HKV, kv = unit % p.b.HKV;
        if (s_seq[r] < 0) continue;
        const int row = s_pos[r] & 15;
        const unsigned char* blk = p.b.cache + kv4_block(p.b, D, s_seq[r], kv, s_pos[r]);
        const uint32_t word = *reinterpret_cast<const uint32_t*>(blk + (part ? kv4_value_word(D, row, sub) : kv4_key_word(D, row, sub)));
        const float2 pair = __half22float2(*reinterpret_cast<const __half2*>(blk + kv4_pair(D, part, row, sub >> 3)));
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fmaf(pair.x, (float)((word >> (4 * j)) & 15u), pair.y);
        const size_t o = ((size_t)(row0 + r) * p.b.HKV + kv) * D + sub * 8;
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
            continue;
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
}

#define KC_KERNELS(D)                                                                                                                                  \
    extern "C" __global__ void __launch_bounds__(KC_THREADS) kv4_append_##D(const __grid_constant__ lb_kv4_rows_params p) { kv4_append_body<D>(p); } \
    extern "C" __global__ void __launch_bounds__(KC_THREADS) kv4_read_##D(const __grid_constant__ lb_kv4_rows_params p) { kv4_read_body<D>(p); }
KC_KERNELS(64)
KC_KERNELS(128)
KC_KERNELS(256)
