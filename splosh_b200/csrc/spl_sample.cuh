// spl_sample.cuh — a token a row from its logits: temperature, top-k, top-p, min-p, and one given uniform number.
//
// Sampler.sample (Sources/SploshRuntime/Sampler.swift:128-156) over the whole vocabulary, on the device. The values of [0, limit) stand
// in descending order, the lower index first among equal values; NaN and -inf are never picked. With w = exp((x - max x) / T):
//   top-k   the first k stay                                                      (k <= 0: all)
//   top-p   of those the smallest prefix whose w reaches p times their sum        (p >= 1: all)
//   min-p   of those the ones with w >= m                                         (m <= 0: all)
//   draw    the first whose running sum of w reaches u times the sum of what stays
// T <= 0 takes the largest value. Everything that stays is a prefix of the order, so nothing is sorted: a cut is found
// by its place or by its weight, eight bits of the values' keys at a time.
//
// The token has to be the definition's, so the sums have to be right where a boundary between tokens is close: 32-bit sums of a flat
// vocabulary of 250K would pick another token in one row of fifty. Weights are formed in 64-bit floating point and summed as whole numbers of
// 2^-44 (the largest is 2^44, 2^19 of them fit 64 bits): the sums do not depend on the order of the additions.
#pragma once
#include "spl_elementwise.cuh"

#define SPL_SAMPLE_UNIT 17592186044416.0       // 2^44
#define SPL_SAMPLE_VOCAB (1 << 19)

struct SplSampleArgs {
    const float *logits; long long ld; int limit;
    const float *temperature; const int *top_k; const float *top_p, *min_p, *uniform;      // per row; null: 1, all, 1, 0
    int *ids;
};

__device__ __forceinline__ float spl_topk_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
// The weight of a value, a whole number of 2^-44. (inf - inf is no number: the maximum itself has weight one.)
__device__ __forceinline__ unsigned long long spl_sample_weight(float x, float max, double inv_t) {
    if (x == max) return 1ull << 44;
    return static_cast<unsigned long long>(exp((double(x) - double(max)) * inv_t) * SPL_SAMPLE_UNIT + 0.5);
}

// Grid (rows), 1,024 threads.
__global__ void __launch_bounds__(1024)
spl_sample_kernel(SplSampleArgs a) {
    __shared__ unsigned long long mass[256];
    __shared__ unsigned int count[256], warp_count[32];
    __shared__ unsigned long long found_before;
    __shared__ unsigned int found_digit, shared_max;
    spl_grid_begin();
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *x = a.logits + size_t(row) * a.ld;
    const float t = a.temperature ? a.temperature[row] : 1.0f, p = a.top_p ? a.top_p[row] : 1.0f, u = a.uniform[row];
    const float m = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    if (tid == 0) shared_max = 0u;
    __syncthreads();
    uint32_t top = 0u;
    for (int i = tid; i < a.limit; i += 1024) top = max(top, spl_topk_key(x[i]));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) atomicMax(&shared_max, top);
    __syncthreads();
    top = shared_max;
    if (top == 0u) { if (tid == 0) a.ids[row] = 0; return; }                 // nothing to pick from: as an untouched slot of a top-k
    const float max_value = spl_topk_value(top);
    const bool greedy = !(t > 0.0f);
    const double inv_t = greedy ? 1.0 : 1.0 / double(t);

    // What stays: keys above cut_key, and of cut_key itself the cut_ties lowest indices; and weights of at least `least`.
    uint32_t cut_key = 1u;
    unsigned long long cut_ties = ~0ull, least = 0ull;
    // The place in the order where the running count (by_count) or the running weight reaches `target` (at least the first place):
    // its key, and how many of the key's values the prefix takes.
    auto find = [&](bool by_count, unsigned long long target, uint32_t *key_out, unsigned long long *ties_out) {
        uint32_t prefix = 0u;
        unsigned long long before = 0ull;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) { mass[tid] = 0ull; count[tid] = 0u; }
            __syncthreads();
            for (int i = tid; i < a.limit; i += 1024) {
                const float v = x[i];
                const uint32_t key = spl_topk_key(v);
                if (key < cut_key || key == 0u || (shift < 24 && (key >> (shift + 8)) != prefix)) continue;
                const uint32_t digit = key >> shift & 255u;
                if (by_count) atomicAdd(&count[digit], 1u);
                else {
                    const unsigned long long w = spl_sample_weight(v, max_value, inv_t);
                    if (w < least) continue;
                    atomicAdd(&mass[digit], w);
                    atomicAdd(&count[digit], 1u);
                }
            }
            __syncthreads();
            if (tid == 0) {
                unsigned long long sum = before;
                int last = -1;
                for (int d = 255; d >= 0; --d) {
                    if (!count[d]) continue;
                    const uint32_t reached = prefix << 8 | uint32_t(d);
                    unsigned long long here = by_count ? count[d] : mass[d];
                    // The key that an earlier cut goes through keeps only its lowest indices.
                    if (!by_count && shift == 0 && reached == cut_key && count[d] > cut_ties) here = mass[d] / count[d] * cut_ties;
                    last = d;
                    found_before = sum;
                    sum += here;
                    if (sum >= target) break;
                }
                found_digit = uint32_t(last);
            }
            __syncthreads();
            prefix = prefix << 8 | found_digit;
            before = found_before;
            __syncthreads();
        }
        *key_out = prefix;
        const unsigned long long each = by_count ? 1ull : spl_sample_weight(spl_topk_value(prefix), max_value, inv_t);
        *ties_out = target <= before + 1ull || each == 0ull ? 1ull : (target - before + each - 1ull) / each;
    };
    // The weight of all that stays.
    auto total = [&]() {
        if (tid == 0) { mass[0] = 0ull; count[0] = 0u; }
        __syncthreads();
        unsigned long long sum = 0ull;
        unsigned int ties = 0u;
        for (int i = tid; i < a.limit; i += 1024) {
            const float v = x[i];
            const uint32_t key = spl_topk_key(v);
            if (key < cut_key || key == 0u) continue;
            if (key == cut_key) { ++ties; continue; }
            const unsigned long long w = spl_sample_weight(v, max_value, inv_t);
            if (w >= least) sum += w;
        }
        if (sum) atomicAdd(&mass[0], sum);
        if (ties) atomicAdd(&count[0], ties);
        __syncthreads();
        const unsigned long long each = spl_sample_weight(spl_topk_value(cut_key), max_value, inv_t);
        sum = mass[0];
        if (count[0] && each >= least) sum += each * min((unsigned long long)count[0], cut_ties);
        __syncthreads();
        return sum;
    };
    uint32_t pick_key = top;
    unsigned long long pick_tie = 1ull;
    if (!greedy) {
        if (k > 0 && k < a.limit) find(true, (unsigned long long)k, &cut_key, &cut_ties);
        if (p < 1.0f) {
            const unsigned long long target = p > 0.0f ? (unsigned long long)ceil(double(p) * double(total())) : 0ull;
            uint32_t key; unsigned long long ties;
            find(false, target, &key, &ties);
            if (key > cut_key || ties < cut_ties) { cut_key = key; cut_ties = ties; }
        }
        if (m > 0.0f) least = (unsigned long long)ceil(double(m) * SPL_SAMPLE_UNIT);
        const unsigned long long all = total();
        const unsigned long long target = u > 0.0f ? min(all, (unsigned long long)ceil(double(u) * double(all))) : 0ull;
        find(false, target, &pick_key, &pick_tie);
    }
    // The pick_tie-th lowest index of pick_key: the block walks the row in order.
    unsigned long long seen = 0ull;
    for (int base = 0; base < a.limit; base += 1024) {
        const int i = base + tid;
        const bool hit = i < a.limit && spl_topk_key(x[i]) == pick_key;
        const unsigned int votes = __ballot_sync(0xffffffffu, hit);
        if (lane == 0) warp_count[warp] = __popc(votes);
        __syncthreads();
        unsigned int before = 0u, all = 0u;
        for (int w = 0; w < 32; ++w) { if (w < warp) before += warp_count[w]; all += warp_count[w]; }
        if (hit && seen + before + __popc(votes & ((1u << lane) - 1u)) + 1u == pick_tie) a.ids[row] = i;
        seen += all;
        if (seen >= pick_tie) return;
        __syncthreads();
    }
}
