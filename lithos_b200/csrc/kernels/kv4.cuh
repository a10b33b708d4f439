// The 4-bit KV cache: its layout, the requests of a batch, loads of 8 features in the three input types.
//
// A value stands as one of 16 codes: x ~ lowest + scale * c, c = 0..15, with a (scale, lowest) pair in fp16 for every row, KV head and group of 64
// features: 4.5 bits a value.  lowest = the group's minimum, scale = (maximum - lowest) / 15, each rounded to fp32 and then to fp16, c the nearest code
// (halves to the even one) against the rounded pair.
// A block holds 16 rows of one sequence and KV head, keys and values, 18 D bytes in one piece, S = D / 64 groups:
//   keys    [2][S][8 rows][32 bytes]   half i, place g: row 4 (g / 2) + 2 i + g % 2.  A lane (g, t) of a product with 8 rows as columns reads 8 bytes, its neighbours the next
//   values  [S][8][16 rows][4 bytes]   word g of a group: features 8 g .. 8 g + 7.  Lane (g, t) reads the words of rows 4 t .. 4 t + 3 as 16 bytes
//   (scale, lowest) of the keys [S][16 rows], of the values [S][16 rows]
// The rows' order is the one in which scores leave the first product and enter the second as its operand: a lane of row group t has rows 4 t .. 4 t + 3.
#pragma once
#include "common.cuh"
#include "params.h"

__device__ __forceinline__ size_t kv4_block(const lb_kv4_view& b, int D, int seq, int kv, int row) {
    return (((size_t)seq * b.HKV + kv) * (size_t)(b.max_ctx >> 4) + (size_t)(row >> 4)) * (size_t)LB_KV4_BLOCK(D);
}
// byte offsets inside a block: the 4 bytes of features 8 w .. 8 w + 7 of row r, and its groups' (scale, lowest)
__device__ __forceinline__ int kv4_key_word(int D, int r, int w) {
    return ((((r >> 1) & 1) * (D >> 6) + (w >> 3)) * 8 + 2 * (r >> 2) + (r & 1)) * 32 + (w & 7) * 4;
}
__device__ __forceinline__ int kv4_value_word(int D, int r, int w) { return 8 * D + (w * 16 + r) * 4; }
__device__ __forceinline__ int kv4_pair(int D, int part, int r, int group) { return (16 + part) * D + (group * 16 + r) * 4; }

struct kv4_request { int seq, pos, start, n; };
// Request r of a batch; n = 0 where it names rows or a sequence that are not there, which the status word then says.
__device__ __forceinline__ kv4_request kv4_get(const lb_kv4_view& b, int r) {
    kv4_request q;
    q.start = b.starts ? b.starts[r] : r;
    const int end = b.starts ? b.starts[r + 1] : r + 1;
    q.seq = b.seqs ? b.seqs[r] : r;
    q.pos = b.pos[r];
    q.n = end - q.start;
    if (end == q.start) return q;
    uint32_t bad = 0;
    if (q.start < 0 || end < q.start || end > b.rows || q.n > b.max_new || q.seq < 0 || q.seq >= b.n_seqs) bad = LB_DEV_BATCH;
    else if (q.pos < 0 || q.pos > b.max_ctx - q.n) bad = LB_DEV_POS_RANGE;
    if (bad) {
        atomicExch(b.status, bad);
        q.n = q.start = 0;
    }
    return q;
}

// 8 neighbouring elements; wide: 16 bytes at a time
__device__ __forceinline__ void kv4_load8(const void* p, size_t i, int type, int wide, float (&x)[8]) {
    if (type == 1) {
        const float* f = reinterpret_cast<const float*>(p) + i;
        if (wide) {
            const float4 a = *reinterpret_cast<const float4*>(f), c = *reinterpret_cast<const float4*>(f + 4);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = c.x; x[5] = c.y; x[6] = c.z; x[7] = c.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = f[j];
        }
        return;
    }
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + i;
    uint32_t w[4];
    if (wide) {
        const uint4 a = *reinterpret_cast<const uint4*>(h);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (uint32_t)h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 v = type == 0 ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j])) : __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        x[2 * j] = v.x;
        x[2 * j + 1] = v.y;
    }
}
__device__ __forceinline__ float kv4_load1(const void* p, size_t i, int type) {
    if (type == 1) return reinterpret_cast<const float*>(p)[i];
    const uint16_t h = reinterpret_cast<const uint16_t*>(p)[i];
    return type == 0 ? bf16_bits_to_f32(h) : __half2float(__ushort_as_half(h));
}
