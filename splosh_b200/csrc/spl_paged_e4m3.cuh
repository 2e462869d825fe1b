// spl_paged_e4m3.cuh — attention of the new rows over a paged cache of e4m3 codes with a scale a token and kv head.
#pragma once
#include "spl_paged.cuh"

__device__ __forceinline__ float2 spl_unpack_e4m3(uint16_t v) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"(v));
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

struct SplPagedAttendE4m3 {
    const uint16_t *q; const unsigned char *k, *v; const float *k_scale, *v_scale; void *out; int out_f32;
    const int *lengths;          // of the sequences
};

// A warp a row and head, the tokens one after the other: a lane has the channels 64 j + 2 lane and the next.
template <int HD>
__global__ void __launch_bounds__(256)
spl_paged_attend_e4m3_kernel(SplPagedTables t, SplPagedShape s, SplPagedAttendE4m3 a) {
    spl_grid_begin();
    const int job = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, row = job / s.heads, head = job % s.heads, kv = head / s.group;
    if (row >= *t.count) return;
    const int sequence = t.row_sequence[row], position = t.row_position[row], first = spl_paged_first(s, position), last = spl_paged_last(s, position, a.lengths[sequence]);
    float2 q[HD / 64], o[HD / 64];
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) { q[j] = spl_unpack16<true>(*reinterpret_cast<const uint32_t *>(a.q + (size_t(row) * s.heads + head) * HD + 64 * j + 2 * lane)); o[j] = make_float2(0.0f, 0.0f); }
    float m = -INFINITY, sum = 0.0f;
    const float c = s.scale * 1.4426950408889634f;
    for (int token = first; token < last; ++token) {
        const size_t page = t.table[size_t(sequence) * s.max_pages + token / s.page_tokens];
        const int inside = token % s.page_tokens;
        const size_t at = page * s.page_stride + size_t(kv) * s.head_stride + size_t(inside) * s.token_stride + 2 * lane, scale_at = (page * s.kv_heads + kv) * s.page_tokens + inside;
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) { const float2 k = spl_unpack_e4m3(*reinterpret_cast<const uint16_t *>(a.k + at + 64 * j)); dot += q[j].x * k.x + q[j].y * k.y; }
        const float x = spl_warp_sum(dot) * a.k_scale[scale_at] * c, now = fmaxf(m, x), old = exp2f(m - now), p = exp2f(x - now), pv = p * a.v_scale[scale_at];
        m = now; sum = sum * old + p;
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
            const float2 v = spl_unpack_e4m3(*reinterpret_cast<const uint16_t *>(a.v + at + 64 * j));
            o[j] = make_float2(o[j].x * old + pv * v.x, o[j].y * old + pv * v.y);
        }
    }
    const float inv = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) {
        const size_t place = (size_t(row) * s.heads + head) * HD + 64 * j + 2 * lane;
        if (a.out_f32) *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + place) = make_float2(o[j].x * inv, o[j].y * inv);
        else *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.out) + place) = spl_pack16<true>(o[j].x * inv, o[j].y * inv);
    }
}
