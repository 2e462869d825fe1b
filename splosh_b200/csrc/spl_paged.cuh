// spl_paged.cuh — new keys and values into a paged cache of the caller's own, with the rotation applied on the way, and
// attention of the new rows over that cache.
//
// What DraftModel builds for its own layers beside Engine.gemm / norm / mlpIn (its K/V store and its attention,
// Sources/Shaders/draft.metal:59-100 and Sources/SploshRuntime/DraftModel.swift:418-468), for any pass over the caller's own
// tensors: 16-bit keys and values, any page size and head layout, sequences of any length.
//
// Cache: element (page, kv head, token in page, channel) of K and of V lies at
//   page * page_stride + head * head_stride + token * token_stride + channel     (16-bit elements)
// A batch: row r of a pass belongs to sequence row_sequence[r] and sits at position row_position[r], the last of its sequence's rows at the sequence's last token. Token t of sequence s is in page table[s * max_pages + t / page_tokens].
#pragma once
#include <cuda.h>

#include "spl_attention.cuh"
#include "spl_common.cuh"
#include "spl_paged_plan.h"

struct SplPagedShape {
    int heads, kv_heads, group, head_dim, page_tokens, max_pages;
    long long page_stride, head_stride, token_stride;
    int rotary, causal, window;
    float scale;
};
// The batch as the kernels read it (device memory).
struct SplPagedTables {
    const int *count;             // rows
    const int *row_sequence, *row_position;
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
// Grid (rows, head ranges), 256 threads: the angles' sines and cosines once a block, then a warp a head, a lane the channels 64 j + 2 lane and the next, the next head's on their way.
// A channel's partner is in another register or lane where rotary / 2 is a power of two from 2 on, else it comes by way of shared memory. Bound: the instructions of a head, then HBM: 2,048
// rows of 24/4 heads of 256 (101 MB) took 25 us at 320 instructions a head, 21 at 250, a block's start among them.
struct SplPagedRows { const void *q, *k, *v; long long q_ld, k_ld, v_ld; };

template <int TYPE, bool BF16, int HD>
__global__ void __launch_bounds__(256, 5)
spl_paged_append_kernel(SplPagedRows in, const uint16_t *__restrict__ q_norm, const uint16_t *__restrict__ k_norm, const double *__restrict__ turns,
                        SplPagedTables t, SplPagedShape s, float eps, uint16_t *q_out, uint16_t *k_cache, uint16_t *v_cache) {
    constexpr int J = HD / 64, SIZE = TYPE == 0 ? 4 : 2;
    __shared__ __align__(16) float2 turn[128];   // (cos, sin) of channel pair i
    __shared__ float2 vector[8][32 * J];
    spl_grid_begin();
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = s.rotary / 2, vectors = s.heads + 2 * s.kv_heads;
    const int rows = *t.count, sequence = t.row_sequence[row], position = t.row_position[row];
    if (row >= rows) return;
    const int per = (vectors + gridDim.y - 1) / gridDim.y, begin = blockIdx.y * per + warp, last = min(vectors, int(blockIdx.y + 1) * per);
    // Where head n of the row's queries, keys and values begins, for this lane.
    const char *q_from = static_cast<const char *>(in.q) + (size_t(row) * in.q_ld + 2 * lane) * SIZE, *k_from = static_cast<const char *>(in.k) + (size_t(row) * in.k_ld + 2 * lane) * SIZE,
               *v_from = static_cast<const char *>(in.v) + (size_t(row) * in.v_ld + 2 * lane) * SIZE;
    auto load = [&](int n, float2 (&x)[J]) {
        const int k = n - s.heads, v = k - s.kv_heads;
        const char *from = k < 0 ? q_from + n * (HD * SIZE) : v < 0 ? k_from + k * (HD * SIZE) : v_from + v * (HD * SIZE);
#pragma unroll
        for (int j = 0; j < J; ++j) x[j] = spl_load_pair<TYPE>(from, 64 * j);
    };
    float2 ahead[J];
    if (begin < last) load(begin, ahead);
    const int page = t.table[size_t(sequence) * s.max_pages + position / s.page_tokens];
    if (threadIdx.x < half) {
        const double a = double(position) * turns[threadIdx.x];
        float sn, cs;
        sincospif(2.0f * float(a - rint(a)), &sn, &cs);
        turn[threadIdx.x] = make_float2(cs, sn);
    }
    __syncthreads();
    const bool square = (half & (half - 1)) == 0 && half > 1;
    const size_t place = size_t(page) * s.page_stride + size_t(position % s.page_tokens) * s.token_stride + 2 * lane;
    uint16_t *q_to = q_out + size_t(row) * s.heads * HD + 2 * lane, *k_to = k_cache + place, *v_to = v_cache + place;
    const uint16_t *held = nullptr;              // the weight in registers: a warp's queries come first, then its keys
    float2 w[J];
    for (int n = begin; n < last; n += 8) {
        const int k = n - s.heads, v = k - s.kv_heads;
        uint16_t *dst = k < 0 ? q_to + n * HD : v < 0 ? k_to + size_t(k) * s.head_stride : v_to + size_t(v) * s.head_stride;
        float2 x[J];
#pragma unroll
        for (int j = 0; j < J; ++j) x[j] = ahead[j];
        if (n + 8 < last) load(n + 8, ahead);
        const uint16_t *weight = k < 0 ? q_norm : v < 0 ? k_norm : nullptr;
        if (weight) {
            if (weight != held) {
                held = weight;
#pragma unroll
                for (int j = 0; j < J; ++j) w[j] = spl_unpack16<true>(*reinterpret_cast<const uint32_t *>(weight + 64 * j + 2 * lane));
            }
            float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int j = 0; j < J; ++j) ss = spl_fma2(x[j], x[j], ss);
            const float inv = rsqrtf(spl_warp_sum(ss.x + ss.y) * (1.0f / HD) + eps);
#pragma unroll
            for (int j = 0; j < J; ++j) x[j] = spl_mul2(spl_mul2(x[j], make_float2(inv, inv)), w[j]);
        }
        if (v < 0 && half) {
            if (square) {
                float2 other[J];
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    if (half >= 64) other[j] = half == 64 ? x[j ^ (J > 1 ? 1 : 0)] : x[j ^ (J > 2 ? 2 : 0)];
                    else if (64 * j < s.rotary) other[j] = make_float2(__shfl_xor_sync(0xffffffffu, x[j].x, half / 2), __shfl_xor_sync(0xffffffffu, x[j].y, half / 2));
                }
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const int i = 64 * j + 2 * lane;
                    if (i < s.rotary) {          // (rotary and i are even: a lane's two channels turn together)
                        const float4 a = *reinterpret_cast<const float4 *>(&turn[i & (half - 1)]);
                        const float sign = i & half ? 1.0f : -1.0f;
                        x[j] = make_float2(x[j].x * a.x + sign * other[j].x * a.y, x[j].y * a.z + sign * other[j].y * a.w);
                    }
                }
            } else {
                float *mine = reinterpret_cast<float *>(vector[warp]);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < J; ++j) vector[warp][32 * j + lane] = x[j];
                __syncwarp();
                auto turned = [&](int i, float own) {
                    if (i >= s.rotary) return own;
                    const float2 c = turn[i < half ? i : i - half];
                    return i < half ? own * c.x - mine[i + half] * c.y : own * c.x + mine[i - half] * c.y;
                };
#pragma unroll
                for (int j = 0; j < J; ++j) x[j] = make_float2(turned(64 * j + 2 * lane, x[j].x), turned(64 * j + 2 * lane + 1, x[j].y));
            }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) *reinterpret_cast<uint32_t *>(dst + 64 * j) = spl_pack16<BF16>(x[j].x, x[j].y);
    }
}

// ---- attention --------------------------------------------------------------------------------
// o = sum_j p_j v_j / sum_j p_j with p_j = exp(scale q.k_j - m), in one pass over the tokens with a running reference m.
//
// A block takes pieces (SplPagedItem) of 128 packed query rows (the new tokens of a sequence times the heads that share a kv head: single
// tokens, verify blocks and prompt chunks are one kernel) against tiles of 128 tokens. Per tile
//   S[128 rows x 128 tokens]   = Q[128 x HD] K^T          A = Q, B = K          (shared memory, K-major)
//   O[128 rows x HD]          += P[128 x 128] V           A = P (tensor memory), B = V (shared memory, tokens along the contraction)
// with the softmax between them. Keys come as chunks of 128 tokens x up to 128 channels, values as chunks of up to 128 tokens x all channels (a tile at HD of 64
// and 128, half a tile at 256; 128-byte swizzle), a ring for each (a ring's barriers tell a phase from the one before it and no more, so a ring has one reader); they are asked for in the
// order the products take them: K of tile 0; K of tile i + 1, V of tile i; ... A page smaller than a chunk's tokens is a copy
// of its own, so page sizes and head layouts are the tensor maps' business alone.
// An instruction of the value product spans all HD columns of O: with values in chunks of 64 channels it took HD / 64 times as many instructions of 64 columns, and the
// issuing warp (some 100 cycles an instruction) was the block's pace: 5,000 of 6,450 cycles a tile at HD = 256.
//
// Warps 0-7 softmax (thread: a row and half of the tile's tokens; the pair of warps of 32 rows agrees on the maximum), warps 8 and 11 copy (a chunk is
// some 800 cycles of waiting and asking: with one warp for both that was the block's pace at HD = 256), warps 9 and 10 issue the products: S of tile i + 1 runs under the softmax of tile i. The reference is raised only when a row's maximum exceeds it by 2^8, so the sums in
// tensor memory are rescaled a few times a piece, not every tile. Rows that are not there cost no softmax work.
// Tensor memory: S / P two buffers of 128 columns (P, 16 bits, over the S it came from), O HD columns from 256. (At HD = 128 there is room for P beside S: with the next tile's
// scores loaded under a tile's exponentials 2,048 rows over 8,192 tokens of 32/8 heads took 303 us instead of 264, with two groups of four warps taking turns at the tiles 282.)
//
// Rounding: P to the cache's type (what the tensor core takes beside V); S, m, the sums of P and O are fp32. In fp16 P is scaled by 2^7 (the factor
// cancels), so that probabilities down to 2^-21 of the reference keep all bits and one 2^8 above it stays finite.
//
// What is masked may be anything: a masked score is replaced before it is used, and because 0 x inf is no number, tokens that no row of the piece
// sees (behind the sequence's last token, in front of the window) have their values zeroed in shared memory or are left out of the product.
#define SPL_PAGED_THREADS 384
#define SPL_PAGED_HEADROOM 8.0f
__host__ __device__ constexpr int spl_paged_chunk(int hd) { return hd == 64 ? 16384 : 32768; }
__host__ __device__ constexpr int spl_paged_ring_k(int hd) { return hd == 64 ? 6 : 3; }
__host__ __device__ constexpr int spl_paged_ring_v(int hd) { return hd == 64 ? 6 : hd == 128 ? 3 : 2; }
__host__ __device__ constexpr int spl_paged_ring(int hd) { return spl_paged_ring_k(hd) + spl_paged_ring_v(hd); }
__host__ __device__ constexpr size_t spl_paged_smem_bytes(int hd) {
    return size_t(hd) * 256 + size_t(spl_paged_ring(hd)) * spl_paged_chunk(hd) + 2 * 2 * 128 * 4 /* maxima, sums */ + 512 /* barriers */;
}

// Tokens that the row at `position` of a sequence of `length` tokens sees: [first, last).
__device__ __forceinline__ int spl_paged_first(const SplPagedShape &s, int position) { return s.window > 0 && position + 1 > s.window ? position + 1 - s.window : 0; }
__device__ __forceinline__ int spl_paged_last(const SplPagedShape &s, int position, int length) { return s.causal ? position + 1 : length; }

// D[tmem] (+)= A * B with A and B in shared memory, or A in tensor memory; issued by the lane with `elected` set, in the converged warp's control flow: descriptors are
// formed in uniform registers, which a branch around the instructions prevents (150 cycles an instruction).
__device__ __forceinline__ void spl_tc_mma_ss_if(uint32_t elected, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
__device__ __forceinline__ void spl_tc_mma_ts_if(uint32_t elected, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
__device__ __forceinline__ void spl_tc_commit_if(uint32_t elected, uint64_t *bar) {
    asm volatile("{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(spl_smem_addr(bar)), "r"(elected) : "memory");
}
// The instruction descriptor of spl_tc_idesc for either type; the value product's B has its tokens (the contraction) in rows: MN-major.
__host__ __device__ constexpr uint32_t spl_paged_idesc(int n, bool bf16, bool b_mn) {
    return spl_tc_idesc(n) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}
__device__ __forceinline__ void spl_tc_ld32(uint32_t (&r)[32], uint32_t taddr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 "tcgen05.wait::ld.sync.aligned;\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
                   "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
                   "=r"(r[31]) : "r"(taddr));
}
__device__ __forceinline__ void spl_tma_prefetch(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory"); }
__device__ __forceinline__ void spl_tma_load5(void *smem, const CUtensorMap *map, int x, int token, int block, int head, int page, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];\n"
                 ::"r"(spl_smem_addr(smem)), "l"(map), "r"(x), "r"(token), "r"(block), "r"(head), "r"(page), "r"(spl_smem_addr(bar)) : "memory");
}
// A box into L2 alone.
__device__ __forceinline__ void spl_tma_prefetch5(const CUtensorMap *map, int x, int token, int block, int head, int page) {
    asm volatile("cp.async.bulk.prefetch.tensor.5d.L2.global.tile [%0, {%1, %2, %3, %4, %5}];\n" ::"l"(map), "r"(x), "r"(token), "r"(block), "r"(head), "r"(page) : "memory");
}
// MN-major, 128-byte swizzle: rows of 64 elements (128 bytes) along the contraction, eight-row groups 1,024 bytes apart, the next 64 elements of a row `block_bytes` on.
__device__ __forceinline__ uint64_t spl_tc_desc_mn_sw128(uint32_t smem_byte_addr, uint32_t block_bytes) {
    return (spl_tc_desc_sw128(smem_byte_addr) & ~(uint64_t(0x3FFF) << 16)) | uint64_t(block_bytes >> 4) << 16;
}
// The two warps of 32 rows (w and w + 4): barriers 1 to 4.
__device__ __forceinline__ void spl_paged_pair_barrier(int quarter) {
    if (quarter == 0) spl_named_barrier<1, 64>();
    else if (quarter == 1) spl_named_barrier<2, 64>();
    else if (quarter == 2) spl_named_barrier<3, 64>();
    else spl_named_barrier<4, 64>();
}

// 2^z for two z of at most 2^7 on the fp32 pipe: z = n + f with n = rint(z) (1.5 * 2^23 added leaves n in the low bits), 2^f = exp(f ln 2) by its series to the fifth power (|f| <= 1/2:
// the next term is 2.5e-6 of it, a hundredth of fp16's step), times 2^n. Below -125 zero (a masked score's weight is nothing, whatever its value); what is no number stays none.
__device__ __forceinline__ float2 spl_paged_exp2(float2 z) {
    const float2 t = spl_add2(z, make_float2(12582912.0f, 12582912.0f)), n = spl_add2(t, make_float2(-12582912.0f, -12582912.0f)), f = spl_fma2(n, make_float2(-1.0f, -1.0f), z);
    constexpr float l = 0.6931471805599453f;
    auto twice = [](float v) { return make_float2(v, v); };
    float2 e = spl_fma2(f, twice(l * l * l * l * l / 120.0f), twice(l * l * l * l / 24.0f));
    e = spl_fma2(f, e, twice(l * l * l / 6.0f));
    e = spl_fma2(f, e, twice(l * l / 2.0f));
    e = spl_fma2(f, e, twice(l));
    e = spl_fma2(f, e, twice(1.0f));
    e = spl_mul2(e, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
    return make_float2(z.x < -125.0f ? 0.0f : e.x, z.y < -125.0f ? 0.0f : e.y);
}

struct SplPagedAttend {
    const uint16_t *q; void *out; int out_f32;
    const SplPagedItem *starts, *items; const int *block_begin; int *arrived;
    float *partial;              // [slot][slot_rows][HD] sums
    float2 *partial_ml;          // [slot][slot_rows] reference (log2), sum of p
    int slot_rows;
    int *error_flag;
};

// The pieces of a tile of query rows joined by 256 threads: o = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s. First m and 1 / sum of every row, to shared memory (`scratch`,
// 256 floats); then the sums, four channels a thread, as many on their way as there are registers for: UP groups of 1024 channels times UN pieces.
template <int HD, bool BF16, int UP, int UN>
__device__ __forceinline__ void spl_paged_join_sums(const SplPagedShape &s, const SplPagedAttend &a, const SplPagedItem &it, int row0, int head0, uint32_t per_group, const float *scratch) {
    const int fours = it.q_count * (HD / 4);
    for (int base = threadIdx.x; base < fours; base += UP * 256) {
        float4 acc[UP];
#pragma unroll
        for (int u = 0; u < UP; ++u) acc[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int n0 = 0; n0 < it.pieces; n0 += UN) {
            float4 v[UP][UN];
            float ref[UP][UN];
#pragma unroll
            for (int u = 0; u < UP; ++u)
#pragma unroll
                for (int n = 0; n < UN; ++n) {
                    const int idx = min(base + u * 256, fours - 1), r = idx / (HD / 4);
                    const size_t row = size_t(it.slot0 + min(n0 + n, it.pieces - 1)) * a.slot_rows + r;
                    v[u][n] = __ldcg(reinterpret_cast<const float4 *>(a.partial + row * HD) + idx % (HD / 4));
                    ref[u][n] = __ldcg(&a.partial_ml[row].x);
                }
#pragma unroll
            for (int u = 0; u < UP; ++u)
#pragma unroll
                for (int n = 0; n < UN; ++n) {
                    const int r = min(base + u * 256, fours - 1) / (HD / 4);
                    if (n0 + n >= it.pieces || ref[u][n] == -INFINITY) continue;      // (a piece of whose tokens this row sees none)
                    const float f = exp2f(ref[u][n] - scratch[r]);
                    acc[u].x += f * v[u][n].x; acc[u].y += f * v[u][n].y; acc[u].z += f * v[u][n].z; acc[u].w += f * v[u][n].w;
                }
        }
#pragma unroll
        for (int u = 0; u < UP; ++u) {
            const int idx = base + u * 256;
            if (idx >= fours) continue;
            const int r = idx / (HD / 4), x = head0 + r, row = int(x * per_group >> 16);
            const float inv = scratch[128 + r];
            const size_t place = (size_t(row0 + row) * s.heads + it.kv_head * s.group + x - row * s.group) * HD + idx % (HD / 4) * 4;
            if (a.out_f32) *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + place) = make_float4(acc[u].x * inv, acc[u].y * inv, acc[u].z * inv, acc[u].w * inv);
            else *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + place) = make_uint2(spl_pack16<BF16>(acc[u].x * inv, acc[u].y * inv), spl_pack16<BF16>(acc[u].z * inv, acc[u].w * inv));
        }
    }
}
template <int HD, bool BF16>
__device__ __forceinline__ void spl_paged_join(const SplPagedShape &s, const SplPagedAttend &a, const SplPagedItem &it, int row0, int head0, uint32_t per_group, float *scratch) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto at = [&](int n, int r) { return __ldcg(&a.partial_ml[size_t(it.slot0 + n) * a.slot_rows + r]); };
    if (it.q_count <= 8) {
        // A row a warp (a single token's heads): nothing to exchange. A running reference, eight pieces on their way.
        if (warp >= it.q_count) return;
        const int x = head0 + warp, row = int(x * per_group >> 16);
        float2 acc[HD / 64];
        float m = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) acc[j] = make_float2(0.0f, 0.0f);
        for (int n0 = 0; n0 < it.pieces; n0 += 8) {
            float2 ml[8], v[8][HD / 64];
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int p = min(n0 + n, it.pieces - 1);
                ml[n] = at(p, warp);
#pragma unroll
                for (int j = 0; j < HD / 64; ++j) v[n][j] = __ldcg(reinterpret_cast<const float2 *>(a.partial + (size_t(it.slot0 + p) * a.slot_rows + warp) * HD + 64 * j + 2 * lane));
            }
            float now = m;
#pragma unroll
            for (int n = 0; n < 8; ++n) if (n0 + n < it.pieces) now = fmaxf(now, ml[n].x);
            if (now == -INFINITY) continue;
            const float old = exp2f(m - now);
            sum *= old;
#pragma unroll
            for (int j = 0; j < HD / 64; ++j) { acc[j].x *= old; acc[j].y *= old; }
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                if (n0 + n >= it.pieces || ml[n].x == -INFINITY) continue;      // (a piece of whose tokens this row sees none)
                const float f = exp2f(ml[n].x - now);
                sum += f * ml[n].y;
#pragma unroll
                for (int j = 0; j < HD / 64; ++j) { acc[j].x += f * v[n][j].x; acc[j].y += f * v[n][j].y; }
            }
            m = now;
        }
        const float inv = 1.0f / sum;
        const size_t place = (size_t(row0 + row) * s.heads + it.kv_head * s.group + x - row * s.group) * HD;
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
            if (a.out_f32) *reinterpret_cast<float2 *>(static_cast<float *>(a.out) + place + 64 * j + 2 * lane) = make_float2(acc[j].x * inv, acc[j].y * inv);
            else *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.out) + place + 64 * j + 2 * lane) = spl_pack16<BF16>(acc[j].x * inv, acc[j].y * inv);
        }
        return;
    }
    if (it.pieces <= 4) {                                     // a thread a row
        const int r = threadIdx.x;
        if (r < it.q_count) {
            float2 ml[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) ml[n] = n < it.pieces ? at(n, r) : make_float2(-INFINITY, 0.0f);
            const float m = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < 4; ++n) if (ml[n].x > -INFINITY) sum += exp2f(ml[n].x - m) * ml[n].y;
            scratch[r] = m; scratch[128 + r] = 1.0f / sum;
        }
    } else for (int r = warp; r < it.q_count; r += 8) {       // a warp a row
        float m = -INFINITY, sum = 0.0f;
        for (int n = lane; n < it.pieces; n += 32) m = fmaxf(m, at(n, r).x);
        m = spl_warp_max(m);
        for (int n = lane; n < it.pieces; n += 32) { const float2 ml = at(n, r); if (ml.x > -INFINITY) sum += exp2f(ml.x - m) * ml.y; }
        sum = spl_warp_sum(sum);
        if (lane == 0) { scratch[r] = m; scratch[128 + r] = 1.0f / sum; }
    }
    spl_named_barrier<5, 256>();
    if (it.pieces <= 2) spl_paged_join_sums<HD, BF16, 6, 2>(s, a, it, row0, head0, per_group, scratch);
    else spl_paged_join_sums<HD, BF16, 2, 6>(s, a, it, row0, head0, per_group, scratch);
}

// Tiles a block asks for while the kernel in front ends: 0 and 2 take 24.7 and 23.4 us for eight blocks of 16 rows over a window of 2,048 tokens of 32/8 heads of 128. (12 rows over 3,000 tokens of
// 24/4 heads of 256: 33.2 and 33.1 where every call has other data; 0 to 4 take 32.1, 31.0, 30.7, 31.0 and 31.6 where they have the same.)
#define SPL_PAGED_EARLY 2
template <int HD, bool BF16>
__global__ void __launch_bounds__(SPL_PAGED_THREADS, 1)
spl_paged_attend_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, SplPagedTables t, SplPagedShape s, SplPagedAttend a) {
    constexpr int C = HD / 64, NK = spl_paged_ring_k(HD), NV = spl_paged_ring_v(HD), CHUNK = spl_paged_chunk(HD), PARTS = HD * 256 / CHUNK, KB = C / PARTS, VT = 128 / PARTS;      // chunks a tile; blocks of 64 channels in one of keys, tokens in one of values
    constexpr float PBIAS = BF16 ? 0.0f : 7.0f;
    extern __shared__ __align__(1024) unsigned char spl_paged_raw[];
    if (spl_smem_addr(spl_paged_raw) % 1024) { if (threadIdx.x == 0) a.error_flag[0] = 299; return; }      // (the swizzle's unit; there is no room to round up)
    unsigned char *q_tile = spl_paged_raw, *ring = q_tile + HD * 256, *v_ring = ring + NK * CHUNK;
    float *xmax = reinterpret_cast<float *>(v_ring + NV * CHUNK);      // [tile parity][half][row]
    uint64_t *bars = reinterpret_cast<uint64_t *>(xmax + 2 * 2 * 128);
    uint64_t *full_k = bars, *empty_k = full_k + NK, *full_v = empty_k + NK, *empty_v = full_v + NV, *s_full = empty_v + NV, *p_full = s_full + 2, *o_done = p_full + 2, *q_full = o_done + 2, *drained = q_full + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drained + 2);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1), *joins = abort + 1;
    // (Broadcasts tell the compiler what is the same in a warp: the issuing warp's descriptors then stay in uniform registers.)
    auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < 2 * NK + 2 * NV; ++i) spl_mbar_init(&bars[i], 1);
        for (int i = 0; i < 2; ++i) { spl_mbar_init(&s_full[i], 1); spl_mbar_init(&p_full[i], 8); spl_mbar_init(&o_done[i], 1); }
        spl_mbar_init(q_full, 8); spl_mbar_init(&drained[0], 1); spl_mbar_init(&drained[1], 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (tid == 256) { spl_tma_prefetch(&k_map); spl_tma_prefetch(&v_map); }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(spl_smem_addr(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    spl_tc_fence_before();
    __syncthreads();
    spl_tc_fence_after();
    const uint32_t tmem = uint32_t(uniform(int(*tmem_slot))), tmem_o = tmem + 256;
    // The block's range, its first item and the first tile's pages are there before the kernel in front is done: a batch is set by copies, which are over before the first kernel
    // behind them begins. (The first item comes with the range, not after it.)
    union { SplPagedItem item; int4 four[sizeof(SplPagedItem) / 16]; } first;
#pragma unroll
    for (int i = 0; i < int(sizeof(SplPagedItem) / 16); ++i) first.four[i] = __ldcg(reinterpret_cast<const int4 *>(a.starts + blockIdx.x) + i);
    const SplPagedItem first_item = first.item;
    const int item0 = uniform(__ldcg(a.block_begin + blockIdx.x)), item1 = uniform(__ldcg(a.block_begin + blockIdx.x + 1));
    const int box = min(s.page_tokens, 128), boxes = 128 / box;      // a tile's boxes of tokens: a page, or half a page of 256
    auto page_of = [&](const SplPagedItem &it, int tile) {
        return tile < it.tile_end && lane < min(boxes, (it.length - tile * 128 + box - 1) / box) ? __ldcg(t.table + size_t(it.sequence) * s.max_pages + (s.page_tokens > 128 ? tile >> 1 : tile * boxes + lane)) : 0;
    };
    const int first_page = (warp == 8 || warp == 11) && item0 < item1 ? page_of(first_item, first_item.tile_begin) : 0;
    // The boxes of a tile's chunk, a lane a box. Keys: a page's tokens by 64 channels, or by the chunk's channels where the box is a tile's tokens. Values: tokens by all channels, boxes of at
    // most the chunk's tokens.
    const int whole = boxes == 1 ? KB : 1, block = boxes == 1 ? lane * KB : lane / boxes, b = lane % boxes;
    const int vbox = min(s.page_tokens, VT), vboxes = VT / vbox, per_page = box / vbox;      // values: boxes a chunk, boxes a lane's page
    auto inside_page = [&](int tile) { return s.page_tokens > 128 ? (tile & 1) * 128 : 0; };
    auto tile_tokens = [&](const SplPagedItem &it, int tile) { return min(128, it.length - tile * 128); };
    auto key_boxes = [&](int tokens) { return (tokens + box - 1) / box; };
    auto value_boxes = [&](int tokens, int c) { return min(vboxes, max(0, (tokens - c * VT + vbox - 1) / vbox)); };
    auto value_page = [&](int page, int c) { return __shfl_sync(0xffffffffu, page, lane < vboxes ? (c * vboxes + lane) / per_page : 0); };
    // The first tiles into L2 while the kernel in front ends. (What it still writes there, a new token, is written to L2 too; the copies into shared memory come after it.)
    if ((warp == 8 || warp == 11) && item0 < item1) {
        int page = first_page;
        for (int tile = first_item.tile_begin; tile < min(first_item.tile_end, first_item.tile_begin + SPL_PAGED_EARLY); ++tile) {
            const int ahead = page_of(first_item, tile + 1), inside = inside_page(tile), tokens = tile_tokens(first_item, tile);
            const int from = __shfl_sync(0xffffffffu, page, b);
            for (int c = 0; c < PARTS; ++c) {
                if (warp == 8) {
                    if (block + whole <= KB && b < key_boxes(tokens)) spl_tma_prefetch5(&k_map, 0, inside, c * KB + block, first_item.kv_head, from);
                } else {
                    const int v_from = value_page(page, c);
                    if (lane < value_boxes(tokens, c)) spl_tma_prefetch5(&v_map, 0, inside + (c * vboxes + lane) % per_page * vbox, 0, first_item.kv_head, v_from);
                }
            }
            page = ahead;
        }
    }
    spl_grid_begin();
    auto item_at = [&](int i) { return i == item0 ? first_item : a.items[i]; };
    // A wait tells a phase from the one before it and no more, so a barrier is waited for only by roles that know its last but one use to be over: S, P and O have one a tile
    // parity (tile i's S is issued after the product of tile i - 2 was waited for; whoever has seen that S may wait for the product of tile i - 1 or i).
    // A role whose wait ran out goes through the rest of its loops without waiting: barriers among warps are met by all of them whatever happened.
    bool ok = true;
    auto gave_up = [&](int code) { ok = false; if (!*abort && lane == 0) { spl_note_wait(a.error_flag, code, 0); a.error_flag[0] = 200 + warp; } *abort = 1; };

    if (warp == 8 || warp == 11) {
        // ---- copies, keys (warp 8) and values (warp 11). Lane b holds the page of the tile's b-th box of tokens; a chunk's barrier counts the boxes that hold tokens.
        const bool keys = warp == 8;
        uint64_t *full = keys ? full_k : full_v, *empty = keys ? empty_k : empty_v;
        const int slots = keys ? NK : NV;
        int n = 0, st = 0;                                    // chunks so far, and the next one's place
        auto room = [&]() {
            if (ok && !spl_mbar_wait_warp(&empty[st], ((n / slots) & 1) ^ 1, const_cast<const int *>(abort))) gave_up(60);
            return ok;
        };
        for (int i = item0; i < item1 && ok; ++i) {
            const SplPagedItem it = item_at(i);
            int page = i == item0 ? first_page : page_of(it, it.tile_begin);
            for (int tile = it.tile_begin; tile < it.tile_end && ok; ++tile) {
                const int ahead = page_of(it, tile + 1), inside = inside_page(tile), tokens = tile_tokens(it, tile);
                if (keys) {
                    const int present = key_boxes(tokens), from = __shfl_sync(0xffffffffu, page, b);
                    for (int c = 0; c < PARTS && room(); ++c) {
                        if (lane == 0) spl_mbar_expect_tx(&full[st], uint32_t(present * box) * 128 * KB);
                        __syncwarp();
                        if (block + whole <= KB && b < present) spl_tma_load5(ring + st * CHUNK + block * 16384 + b * box * 128, &k_map, 0, inside, c * KB + block, it.kv_head, from, &full[st]);
                        ++n; st = st + 1 == slots ? 0 : st + 1;
                    }
                } else {
                    for (int c = 0; c < PARTS && room(); ++c) {
                        const int there = value_boxes(tokens, c), from = value_page(page, c);
                        if (lane == 0) spl_mbar_expect_tx(&full[st], uint32_t(there) * vbox * HD * 2);
                        __syncwarp();
                        if (lane < there) spl_tma_load5(v_ring + st * CHUNK + lane * vbox * HD * 2, &v_map, 0, inside + (c * vboxes + lane) % per_page * vbox, 0, it.kv_head, from, &full[st]);
                        ++n; st = st + 1 == slots ? 0 : st + 1;
                    }
                }
                page = ahead;
            }
        }
        // Nothing may still be on its way into the block's shared memory when it is handed on.
        for (int z = 0; z < slots && z < n; ++z) spl_mbar_wait(&full[z], ((z + (n - 1 - z) / slots * slots) / slots) & 1);
    } else if (warp == 9 || warp == 10) {
        // ---- the products, a warp each (a wait is 110 cycles even when it is over: in one warp six a tile were a third of its time), issued by one elected lane of
        // a converged warp.
        const uint32_t elected = spl_elect_one() ? 1u : 0u;
        const bool first_product = warp == 9;
        constexpr uint32_t s_idesc = spl_paged_idesc(128, BF16, false), o_idesc = spl_paged_idesc(HD, BF16, true);
        const uint64_t q_desc = spl_tc_desc_sw128(spl_smem_addr(q_tile)), ring_desc = spl_tc_desc_sw128(spl_smem_addr(ring)), v_desc = spl_tc_desc_mn_sw128(spl_smem_addr(v_ring), vbox * 128);
        const uint32_t v_box_step = uint32_t(vbox) * HD * 2, vlog = 31 - __clz(vbox);
        int n = 0, tiles = 0;                                 // chunks of its ring and tiles so far
        for (int i = item0; i < item1 && ok; ++i) {
            const SplPagedItem it = item_at(i);
            const int tile_begin = uniform(it.tile_begin), count = uniform(it.tile_end) - tile_begin;
            if (first_product) {
                if (!spl_mbar_wait_warp(q_full, (i - item0) & 1, const_cast<const int *>(abort))) { gave_up(63); break; }
                for (int tile = 0; tile < count && ok; ++tile) {
                    const int at = tiles + tile;
                    // The first keys may be there long before the place of the scores is: it held the P of tile at - 2, which has to have been read.
                    if (!spl_mbar_wait_warp(&full_k[n % NK], (n / NK) & 1, const_cast<const int *>(abort))) { gave_up(62); break; }
                    if (at >= 2 && !spl_mbar_wait_warp(&o_done[at & 1], ((at - 2) >> 1) & 1, const_cast<const int *>(abort))) { gave_up(61); break; }
#pragma unroll
                    for (int c = 0; c < PARTS; ++c, ++n) {
                        const int st = n % NK;
                        if (c > 0 && ok && !spl_mbar_wait_warp(&full_k[st], (n / NK) & 1, const_cast<const int *>(abort))) gave_up(62);
                        if (!ok) break;
                        spl_tc_fence_after();
#pragma unroll
                        for (int ks = 0; ks < 4 * KB; ++ks)
                            spl_tc_mma_ss_if(elected, tmem + (at & 1) * 128, q_desc + uint64_t(((c * KB + ks / 4) * 16384 + ks % 4 * 32) >> 4),
                                             ring_desc + uint64_t((st * CHUNK + ks / 4 * 16384 + ks % 4 * 32) >> 4), s_idesc, c + ks > 0 ? 1u : 0u);
                        spl_tc_commit_if(elected, &empty_k[st]);
                        if (c == PARTS - 1) spl_tc_commit_if(elected, &s_full[at & 1]);
                    }
                }
            } else {
                // Tokens that some row of the piece sees.
                const int seen_first = uniform(spl_paged_first(s, it.base + it.q0 / s.group)), seen_last = uniform(spl_paged_last(s, it.base + (it.q0 + it.q_count - 1) / s.group, it.length));
                for (int tile = 0; tile < count && ok; ++tile) {
                    const int at = tiles + tile, token0 = (tile_begin + tile) * 128;
                    const int from = max(0, seen_first - token0), to = min(128, seen_last - token0);
                    const uint32_t p_at = tmem + (at & 1) * 128;
                    for (int c = 0; c < PARTS && ok; ++c, ++n) {
                        const int st = n % NV;
                        if (!spl_mbar_wait_warp(&full_v[st], (n / NV) & 1, const_cast<const int *>(abort))) { gave_up(65); break; }
                        const int f = min(max(from - c * VT, 0), VT), e = min(max(to - c * VT, 0), VT), k0 = f / 16, k1 = (e + 15) / 16;      // the chunk's tokens that some row sees
                        if (f % 16 || e % 16) {
                            // Values of unseen tokens in the first and last groups of sixteen: zero, whatever the cache holds there.
                            const int before = f % 16, after = (16 - e % 16) % 16;
                            for (int z = lane; z < (before + after) * C * 8; z += 32) {
                                const int row = z / (C * 8), token = row < before ? k0 * 16 + row : e + row - before, piece = z % (C * 8);
                                *reinterpret_cast<uint4 *>(v_ring + st * CHUNK + token / vbox * v_box_step + (piece >> 3) * vbox * 128 + token % vbox * 128 + (piece & 7) * 16) = make_uint4(0, 0, 0, 0);
                            }
                            spl_fence_proxy_async();
                            __syncwarp();
                        }
                        if (c == 0 && !spl_mbar_wait_warp(&p_full[at & 1], (at >> 1) & 1, const_cast<const int *>(abort))) { gave_up(64); break; }
                        spl_tc_fence_after();
                        const uint64_t chunk = v_desc + uint64_t((st * CHUNK) >> 4);
                        // The piece's first product overwrites what O held.
                        const uint32_t onto = tile > 0 || c * VT + k0 * 16 > from / 16 * 16 ? 1u : 0u;
                        auto place = [&](int ks) { return chunk + uint64_t((((ks * 16) >> vlog) * v_box_step + ((ks * 16) & (vbox - 1)) * 128) >> 4); };
                        if (k0 == 0 && k1 == VT / 16) {
#pragma unroll
                            for (int ks = 0; ks < VT / 16; ++ks) spl_tc_mma_ts_if(elected, tmem_o, p_at + (c * (VT / 16) + ks) * 8, place(ks), o_idesc, ks > 0 ? 1u : onto);
                        } else {
                            for (int ks = k0; ks < k1; ++ks) spl_tc_mma_ts_if(elected, tmem_o, p_at + (c * (VT / 16) + ks) * 8, place(ks), o_idesc, ks > k0 ? 1u : onto);
                        }
                        spl_tc_commit_if(elected, &empty_v[st]);
                        if (c == PARTS - 1) spl_tc_commit_if(elected, &o_done[at & 1]);
                    }
                }
            }
            tiles += count;
        }
        // No product may still read shared or write tensor memory when they are handed on.
        spl_tc_commit_if(elected, &drained[first_product ? 0 : 1]);
        spl_mbar_wait(&drained[first_product ? 0 : 1], 0);
    } else if (warp < 8) {
        // ---- softmax: row r of the piece, tokens [64 half, 64 half + 64) of a tile.
        const int quarter = warp & 3, half = warp >> 2, r = quarter * 32 + lane;
        const uint32_t lanes = uint32_t(quarter * 32) << 16;
        const float c = s.scale * 1.4426950408889634f;
        const uint32_t per_group = (65536u + s.group - 1) / s.group;      // x / group = x * per_group >> 16 for x below 192
        int tiles = 0;
        // A piece's queries into the swizzled operand tile: 16-byte pieces of eight channels, eight on their way a thread. (What lies in rows without a query does not reach the others.)
        auto bring_q = [&](const SplPagedItem &it) {
            const int row0 = it.row0 + it.q0 / s.group, head0 = it.q0 % s.group, pieces = it.q_count * (HD / 8);
            for (int base = tid; base < pieces; base += 8 * 256) {
                uint4 v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int idx = base + u * 256, x = head0 + idx / (HD / 8), row = int(x * per_group >> 16);
                    if (idx < pieces) v[u] = *reinterpret_cast<const uint4 *>(a.q + (size_t(row0 + row) * s.heads + it.kv_head * s.group + (x - row * s.group)) * HD + idx % (HD / 8) * 8);
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int idx = base + u * 256, piece = idx % (HD / 8);
                    if (idx < pieces) *reinterpret_cast<uint4 *>(q_tile + (piece >> 3) * 16384 + spl_sw128_offset(idx / (HD / 8), (piece & 7) * 8)) = v[u];
                }
            }
            spl_fence_proxy_async();
            spl_tc_fence_before();
            __syncwarp();
            if (lane == 0) spl_mbar_arrive(q_full);
        };
        SplPagedItem it = first_item;
        if (item0 < item1) bring_q(it);
        for (int i = item0; i < item1; ++i) {
            const bool busy = quarter * 32 < it.q_count;             // whether this warp's rows hold a query
            const SplPagedItem next = i + 1 < item1 ? a.items[i + 1] : it;
            const int row0 = it.row0 + it.q0 / s.group, mine = it.q0 % s.group + min(r, it.q_count - 1), row = int(mine * per_group >> 16), head = it.kv_head * s.group + mine - row * s.group;
            const int position = it.base + it.q0 / s.group + row;
            const int first = spl_paged_first(s, position), last = spl_paged_last(s, position, it.length);
            float ref = -INFINITY, sum = 0.0f;
            for (int tile = it.tile_begin; tile < it.tile_end; ++tile, ++tiles) {
                const int buf = tiles & 1;
                if (ok && !spl_mbar_wait_warp(&s_full[buf], (tiles >> 1) & 1, const_cast<const int *>(abort))) gave_up(66);
                if (busy) {
                    spl_tc_fence_after();
                    const uint32_t at = tmem + lanes + buf * 128;
                    uint32_t x0[32], x1[32];
                    spl_tc_ld32(x0, at + half * 64);
                    spl_tc_ld32(x1, at + half * 64 + 32);
                    const int t0 = tile * 128 + half * 64;
                    // Masked scores are -inf; a tile that all rows see whole has none.
                    if (__any_sync(0xffffffffu, t0 < first || t0 + 64 > last)) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            if (t0 + j < first || t0 + j >= last) x0[j] = 0xff800000u;
                            if (t0 + 32 + j < first || t0 + 32 + j >= last) x1[j] = 0xff800000u;
                        }
                    }
                    float m = -INFINITY, n = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        m = fmaxf(m, fmaxf(__uint_as_float(x0[j]), __uint_as_float(x0[j + 1])));
                        n = fmaxf(n, fmaxf(__uint_as_float(x1[j]), __uint_as_float(x1[j + 1])));
                    }
                    m = fmaxf(m, n);
                    xmax[(buf * 2 + half) * 128 + r] = m;
                    spl_paged_pair_barrier(quarter);
                    m = fmaxf(m, xmax[(buf * 2 + (half ^ 1)) * 128 + r]) * c;
                    const bool raise = m > ref + SPL_PAGED_HEADROOM;
                    if (__any_sync(0xffffffffu, raise)) {
                        const float factor = raise ? exp2f(ref - m) : 1.0f;
                        if (tile > it.tile_begin) {
                            // The product before has to be done with these sums; the next waits for this warp's probabilities.
                            if (ok && !spl_mbar_wait_warp(&o_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, const_cast<const int *>(abort))) gave_up(67);
                            spl_tc_fence_after();
#pragma unroll 1
                            for (int o = 0; o < HD / 2; o += 16) {
                                uint32_t y[16];
                                spl_tc_ld16(y, tmem_o + lanes + half * (HD / 2) + o);
#pragma unroll
                                for (int j = 0; j < 16; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * factor);
                                spl_tc_st16(tmem_o + lanes + half * (HD / 2) + o, y);
                            }
                        }
                        if (raise) { sum *= factor; ref = m; }
                    }
                    const float offset = (ref == -INFINITY ? 0.0f : -ref) + PBIAS;      // a row that has seen nothing yet: all its scores are -inf
                    const float2 c2 = make_float2(c, c), offset2 = make_float2(offset, offset);
                    float2 part = make_float2(0.0f, 0.0f);
                    uint32_t p[32];
                    // (A quarter of the exponentials on the fp32 pipe: the unit for them has 16 lanes an SM and is the tile's pace at HD of 64 and 128. 2,048 rows over 8,192
                    // tokens of 32/8 heads of 128 253 -> 241 us, of 64 242 -> 228.)
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const uint32_t *x = j < 16 ? x0 + 2 * j : x1 + 2 * (j - 16);
                        const float2 z = spl_fma2(make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])), c2, offset2), e = j % 4 == 3 ? spl_paged_exp2(z) : make_float2(spl_ex2(z.x), spl_ex2(z.y));
                        part = spl_add2(part, e);
                        p[j] = spl_pack16<BF16>(e.x, e.y);
                    }
                    sum += part.x + part.y;
                    spl_tc_st32(at + half * 32, p);
                    spl_tc_st_wait();
                    spl_tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) spl_mbar_arrive(&p_full[buf]);
            }
            // The next piece's queries: all scores of this one have been seen, so its own are no longer read. (O is overwritten by a product that waits for this warp.)
            if (i + 1 < item1) bring_q(next);
            // The piece's sums.
            if (ok && !spl_mbar_wait_warp(&o_done[(tiles - 1) & 1], ((tiles - 1) >> 1) & 1, const_cast<const int *>(abort))) gave_up(68);
            const size_t slot_row = size_t(it.slot) * a.slot_rows + r;
            if (busy) {
                spl_tc_fence_after();
                // (Exchanged where the maxima of the tile before the last were: nobody reads those any more.)
                float *xsum = xmax + (tiles & 1) * 2 * 128;
                xsum[half * 128 + r] = sum;
                spl_paged_pair_barrier(quarter);
                sum += xsum[(half ^ 1) * 128 + r];
                const bool here = r < it.q_count;
                const size_t place = (size_t(row0 + row) * s.heads + head) * HD + half * (HD / 2);
                const float inv = it.slot < 0 ? 1.0f / sum : 1.0f;
#pragma unroll 1
                for (int o = 0; o < HD / 2; o += 32) {
                    uint32_t y[32];
                    spl_tc_ld32(y, tmem_o + lanes + half * (HD / 2) + o);
#pragma unroll
                    for (int j = 0; j < 32; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * inv);
                    if (!here) {
                    } else if (it.slot >= 0 || a.out_f32) {
                        float *dst = it.slot >= 0 ? a.partial + slot_row * HD + half * (HD / 2) + o : static_cast<float *>(a.out) + place + o;
#pragma unroll
                        for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4 *>(dst + 4 * j) = make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
                    } else {
                        uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + place + o);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int u = 0; u < 4; ++u) w[u] = spl_pack16<BF16>(__uint_as_float(y[8 * j + 2 * u]), __uint_as_float(y[8 * j + 2 * u + 1]));
                            dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                    __syncwarp();
                }
                if (here && it.slot >= 0 && half == 0) a.partial_ml[slot_row] = make_float2(ref, sum);
                spl_tc_fence_before();
                spl_paged_pair_barrier(quarter);              // the sums in shared memory are read before the next piece's
            }
            if (it.slot >= 0) {
                // Whichever block is the last to leave a piece of these rows joins them, in the order of the pieces whoever it is.
                __threadfence();
                spl_named_barrier<5, 256>();
                if (tid == 0) {
                    const bool all = atomicAdd(&a.arrived[it.merge], 1) == it.pieces - 1;
                    if (all) a.arrived[it.merge] = 0;          // for the next launch
                    *joins = all;
                }
                spl_named_barrier<5, 256>();
                if (*joins) {
                    __threadfence();
                    spl_paged_join<HD, BF16>(s, a, it, row0, it.q0 % s.group, per_group, xmax + (tiles & 1) * 2 * 128);
                    spl_named_barrier<5, 256>();               // before the next piece's maxima
                }
            }
            it = next;
        }
    }
    spl_tc_fence_before();
    __syncthreads();
    spl_tc_fence_after();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}
