// spl_paged.cuh — new keys and values into a paged cache of the caller's own, with the rotation applied on the way, and
// attention of the new rows over that cache.
//
// What DraftModel builds for its own layers beside Engine.gemm / norm / mlpIn (its K/V store and its attention,
// Sources/Shaders/draft.metal:59-100 and Sources/SploshRuntime/DraftModel.swift:418-468), for any pass over the caller's own
// tensors: 16-bit keys and values, any page size and head layout, sequences of any length.
//
// Cache: element (page, kv head, token in page, channel) of K and of V lies at
//   page * page_stride + head * head_stride + token * token_stride + channel     (16-bit elements)
// A batch: sequence s has rows[s] new tokens, the last of its lengths[s]; row r of a pass belongs to sequence row_sequence[r] and
// sits at position row_position[r]. Token t of sequence s is in page table[s * max_pages + t / page_tokens].
#pragma once
#include "spl_common.cuh"

struct SplPagedShape {
    int heads, kv_heads, group, head_dim, page_tokens, max_pages;
    long long page_stride, head_stride, token_stride;
    int rotary, causal, window;
    float scale;
};
// The batch as the kernels read it (device memory).
struct SplPagedTables {
    const int *counts;            // rows, sequences
    const int *row_sequence, *row_position;
    const int *rows, *lengths;    // per sequence
    const int *table;             // [sequences][max_pages]
};

// 16-bit element types. A value is rounded once, to nearest even.
template <bool BF16> __device__ __forceinline__ uint32_t spl_pack16(float lo, float hi) {
    if constexpr (BF16) { const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const uint32_t *>(&v); }
    else { const __half2 v = __floats2half2_rn(lo, hi); return *reinterpret_cast<const uint32_t *>(&v); }
}
template <bool BF16> __device__ __forceinline__ float2 spl_unpack16(uint32_t v) {
    if constexpr (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
// Two neighbouring elements of a row of type SPL_F32 (0), SPL_F16 (1) or SPL_BF16 (2).
template <int TYPE> __device__ __forceinline__ float2 spl_load_pair(const void *base, size_t element) {
    if constexpr (TYPE == 0) return *reinterpret_cast<const float2 *>(static_cast<const float *>(base) + element);
    else return spl_unpack16<TYPE == 2>(*reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(base) + element));
}

// ---- append -----------------------------------------------------------------------------------
// y = x (* rsqrt(mean x^2 + eps) * w, the head's channels, where a weight is given); channels i and i + rotary/2, i < rotary/2, turned
// by the angle position * theta^(-2i / rotary); queries to their rows, keys and values to their place in the cache, all rounded once to
// 16 bits. The angle is formed in 64 bits as turns (position * theta^(-2i/rotary) / 2 pi): at position 200,000 a 32-bit product is
// off by 6e-3 of a radian, a 64-bit one by 1e-11; what is left of the whole turns fits 32 bits.
// Grid (rows, head ranges), 256 threads: the angles' sines and cosines once a block, then a warp a head.
struct SplPagedRows { const void *q, *k, *v; long long q_ld, k_ld, v_ld; };

template <int TYPE, bool BF16>
__global__ void __launch_bounds__(256)
spl_paged_append_kernel(SplPagedRows in, const uint16_t *__restrict__ q_norm, const uint16_t *__restrict__ k_norm, const double *__restrict__ turns,
                        SplPagedTables t, SplPagedShape s, float eps, uint16_t *q_out, uint16_t *k_cache, uint16_t *v_cache) {
    __shared__ float2 turn[128];                 // (cos, sin) of channel pair i
    __shared__ float2 vector[8][128];
    spl_grid_begin();
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half = s.rotary / 2, hd = s.head_dim, vectors = s.heads + 2 * s.kv_heads;
    if (row >= t.counts[0]) return;
    const int sequence = t.row_sequence[row], position = t.row_position[row];
    if (threadIdx.x < half) {
        const double a = double(position) * turns[threadIdx.x];
        float sn, cs;
        sincospif(2.0f * float(a - rint(a)), &sn, &cs);
        turn[threadIdx.x] = make_float2(cs, sn);
    }
    __syncthreads();
    const int page = t.table[size_t(sequence) * s.max_pages + position / s.page_tokens];
    const size_t place = size_t(page) * s.page_stride + size_t(position % s.page_tokens) * s.token_stride;
    float *mine = reinterpret_cast<float *>(vector[warp]);
    const int per = (vectors + gridDim.y - 1) / gridDim.y, last = min(vectors, int(blockIdx.y + 1) * per);
    for (int n = blockIdx.y * per + warp; n < last; n += 8) {
        const bool is_q = n < s.heads, is_v = n >= s.heads + s.kv_heads;
        const int head = is_q ? n : is_v ? n - s.heads - s.kv_heads : n - s.heads;
        const void *src = is_q ? in.q : is_v ? in.v : in.k;
        const size_t from = size_t(row) * (is_q ? in.q_ld : is_v ? in.v_ld : in.k_ld) + size_t(head) * hd + 2 * lane;
        uint16_t *dst = is_q ? q_out + (size_t(row) * s.heads + head) * hd : (is_v ? v_cache : k_cache) + place + size_t(head) * s.head_stride;
        const uint16_t *weight = is_q ? q_norm : is_v ? nullptr : k_norm;
        float2 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) if (64 * j < hd) x[j] = spl_load_pair<TYPE>(src, from + 64 * j);
        if (weight) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) if (64 * j < hd) ss += x[j].x * x[j].x + x[j].y * x[j].y;
            const float inv = 1.0f / sqrtf(spl_warp_sum(ss) / float(hd) + eps);
#pragma unroll
            for (int j = 0; j < 4; ++j) if (64 * j < hd) {
                const uint32_t w = *reinterpret_cast<const uint32_t *>(weight + 64 * j + 2 * lane);
                x[j].x = x[j].x * inv * __uint_as_float(w << 16); x[j].y = x[j].y * inv * __uint_as_float(w & 0xffff0000u);
            }
        }
        if (!is_v && half) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) if (64 * j < s.rotary) vector[warp][32 * j + lane] = x[j];
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) if (64 * j < s.rotary) {
                auto turned = [&](int i, float own) {
                    if (i >= s.rotary) return own;
                    const bool first = i < half;
                    const float2 c = turn[first ? i : i - half];
                    const float other = mine[first ? i + half : i - half];
                    return first ? own * c.x - other * c.y : own * c.x + other * c.y;
                };
                const int i = 64 * j + 2 * lane;
                x[j] = make_float2(turned(i, x[j].x), turned(i + 1, x[j].y));
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) if (64 * j < hd) *reinterpret_cast<uint32_t *>(dst + 64 * j + 2 * lane) = spl_pack16<BF16>(x[j].x, x[j].y);
    }
}

// ---- attention --------------------------------------------------------------------------------
// Tokens that the row at `position` of a sequence of `length` tokens sees: [first, last).
__host__ __device__ __forceinline__ int spl_paged_first(const SplPagedShape &s, int position) { return s.window > 0 && position + 1 > s.window ? position + 1 - s.window : 0; }
__host__ __device__ __forceinline__ int spl_paged_last(const SplPagedShape &s, int position, int length) { return s.causal ? position + 1 : length; }

// o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - m), one pass with the running maximum m. A warp a (row, head), a lane the
// channels 64j + 2 lane and the next. Grid (ceil(heads / 4), rows), 128 threads.
template <bool BF16, bool F32_OUT>
__global__ void __launch_bounds__(128)
spl_paged_attend_kernel(const uint16_t *__restrict__ q, const uint16_t *__restrict__ k_cache, const uint16_t *__restrict__ v_cache, SplPagedTables t, SplPagedShape s, void *out) {
    spl_grid_begin();
    const int row = blockIdx.y, head = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, hd = s.head_dim;
    if (row >= t.counts[0] || head >= s.heads) return;
    const int sequence = t.row_sequence[row], position = t.row_position[row];
    const int first = spl_paged_first(s, position), last = spl_paged_last(s, position, t.lengths[sequence]);
    const int *pages = t.table + size_t(sequence) * s.max_pages;
    float2 x[4], acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        acc[j] = make_float2(0.0f, 0.0f);
        if (64 * j < hd) x[j] = spl_load_pair<BF16 ? 2 : 1>(q, (size_t(row) * s.heads + head) * hd + 64 * j + 2 * lane);
    }
    float m = -INFINITY, sum = 0.0f;
    for (int token = first; token < last; ++token) {
        const size_t at = size_t(pages[token / s.page_tokens]) * s.page_stride + size_t(head / s.group) * s.head_stride + size_t(token % s.page_tokens) * s.token_stride + 2 * lane;
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (64 * j < hd) { const float2 y = spl_load_pair<BF16 ? 2 : 1>(k_cache, at + 64 * j); dot += x[j].x * y.x + x[j].y * y.y; }
        const float score = spl_warp_sum(dot) * s.scale;
        if (score > m) {
            const float f = expf(m - score);
            m = score; sum *= f;
#pragma unroll
            for (int j = 0; j < 4; ++j) { acc[j].x *= f; acc[j].y *= f; }
        }
        const float p = expf(score - m);
        sum += p;
#pragma unroll
        for (int j = 0; j < 4; ++j) if (64 * j < hd) { const float2 y = spl_load_pair<BF16 ? 2 : 1>(v_cache, at + 64 * j); acc[j].x += p * y.x; acc[j].y += p * y.y; }
    }
    const float inv = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) if (64 * j < hd) {
        const size_t at = (size_t(row) * s.heads + head) * hd + 64 * j + 2 * lane;
        if constexpr (F32_OUT) *reinterpret_cast<float2 *>(static_cast<float *>(out) + at) = make_float2(acc[j].x * inv, acc[j].y * inv);
        else *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(out) + at) = spl_pack16<BF16>(acc[j].x * inv, acc[j].y * inv);
    }
}
