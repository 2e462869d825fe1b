// spl_sample.cuh — a token a row from its logits: temperature, top-k, top-p, min-p, and one given uniform number.
//
// Sampler.sample (Sources/SploshRuntime/Sampler.swift:128-156) over the whole vocabulary, on the device. The values of [0, limit) stand
// in descending order, the lower index first among equal values; NaN and -inf are never picked. With w = exp((x - max x) / T):
//   top-k   the first k stay                                                      (k <= 0: all)
//   top-p   of those the smallest prefix whose w reaches p times their sum        (p >= 1: all)
//   min-p   of those the ones with w >= m                                         (m <= 0: all)
//   draw    the first whose running sum of w reaches u times the sum of what stays
// T <= 0 takes the largest value. Everything that stays is a prefix of the order, so a row is never sorted: a place in the order
// (the k-th, the one where the weight reaches p, the draw) lies in one bin of a histogram over the values, and only that bin's values are.
//
// The token has to be the definition's, so the sums have to be right where a boundary between tokens is close: 32-bit sums of a flat
// vocabulary of 250K would pick another token in one row of fifty. Weights are formed in 64-bit floating point and summed as whole numbers of
// 2^-44 (the largest is 2^44, 2^19 of them fit 64 bits): the sums do not depend on the order of the additions, and over n values they are off by at most n 2^-45 of the largest weight.
#pragma once
#include <cooperative_groups.h>

#include "spl_elementwise.cuh"

#define SPL_SAMPLE_UNIT 17592186044416.0       // 2^44
#define SPL_SAMPLE_VOCAB (1 << 19)

struct SplSampleArgs {
    const float *logits; long long ld; int limit;
    const float *temperature; const int *top_k; const float *top_p, *min_p, *uniform;      // per row; null: 1, all, 1, 0
    int *ids;
};

__device__ __forceinline__ float spl_topk_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
// The weight of a value, a whole number of 2^-44: 2^44 exp(z), z = (x - max) / T <= 0, rounded. With n = rint(64 z / ln 2) and f = z - n ln 2 / 64 (at most
// 0.0055 in size), exp(z) = 2^(n / 64) exp(f): the power from a table of 64 (powers[j] = 2^(j / 64)) and an exponent, exp(f) its series to f^5 (the next term is 4e-17), all in
// 64 bits; 2^52 added leaves the rounded whole number in the low bits. scale = 64 / (T ln 2). (inf - inf is no number: the maximum itself has weight one, beside an
// infinite one nothing has any. Below -32 nothing is left of 2^44.)
struct SplSampleWeigh { float max; double scale; const double *powers; };
// (The value is the maximum or less than 33 below it times T.)
__device__ __forceinline__ unsigned long long spl_sample_weight_near(float x, const SplSampleWeigh &w) {
    const double d = double(x) - double(w.max);
    const double magic = 6755399441055744.0, shifted = fma(d, w.scale, magic);      // 1.5 * 2^52: the low word of the sum is n
    const int n = __double2loint(shifted);
    const double g = fma(d, w.scale, magic - shifted);                              // f = g ln 2 / 64; the series in g
    constexpr double c = 0.693147180559945309417 / 64.0;
    double e = fma(g, c * c * c * c * c / 120.0, c * c * c * c / 24.0);
    e = fma(g, e, c * c * c / 6.0);
    e = fma(g, e, c * c / 2.0);
    e = fma(g, e, c);
    e = fma(g, e, 1.0);
    const double power = w.powers[n & 63];
    const double scaled = __hiloint2double(__double2hiint(power) + ((n >> 6) + 44) * (1 << 20), __double2loint(power));      // 2^(44 + n / 64), at least 2^-4
    return (unsigned long long)__double_as_longlong(fma(scaled, e, 4503599627370496.0)) & ((1ull << 52) - 1ull);
}
// Whether a value other than the maximum has no weight.
__device__ __forceinline__ bool spl_sample_weightless(float x, const SplSampleWeigh &w) {
    return w.max == INFINITY || !((double(x) - double(w.max)) * w.scale > -32.0 * 64.0 / 0.693147180559945309417);
}
__device__ __forceinline__ unsigned long long spl_sample_weight(float x, const SplSampleWeigh &w) {
    if (x == w.max) return 1ull << 44;
    if (spl_sample_weightless(x, w)) return 0ull;
    return spl_sample_weight_near(x, w);
}

// A cluster of blocks a row, 32,768 values a block in shared memory (a vocabulary of more than eight blocks' is read anew in every pass): the row comes
// from memory once. The histogram has 4,096 bins of 1/128 in (max - x) / T, so that bins hold a few hundred values where a vocabulary's are densest; what is
// 31.98 and more below the maximum has no weight in whole numbers of 2^-44 and is the last bin (no place that matters lies there, and it is never set aside but in a list that it fits). The first block of the cluster adds the blocks' bins, finds the bin
// that a place lies in, and sorts that bin's values, which the blocks have set aside:
//   top-k         counts; the bins down to the k-th value's are sorted whole where they fit (SPL_SAMPLE_LIST), and everything else is decided on
//                 that list; a larger k sorts its own bin alone and leaves a cut for what follows
//   then          weights; the bins of top-p's place and of min-p's bound are sorted for the exact end of what stays, and then the draw's bin
// Where top-p's and min-p's bins and the draw's do not fit one list together, the draw's come in a turn of their own. Bins that do not fit alone (equal logits, very high temperatures: more than
// 4,096 values in a 128th of a unit, or in the three at min-p's bound) leave the row to the first block, which finds places eight bits of the
// values' keys at a time (spl_sample_slow): 12 rows of 248,077 at temperature 10,000 with top-p take 7.2 ms, at 10 still 0.09.
#define SPL_SAMPLE_BINS 4096
#define SPL_SAMPLE_BINS_NAT 128.0f             // bins a natural unit of (max - x) / T
#define SPL_SAMPLE_SCALE_MAX 3.0e38f           // of a row's bin_scale, twice the bins a unit of max - x: at temperatures below 8.6e-37 bins are wider, and values of no weight lie in front of the last one, too
#define SPL_SAMPLE_LIST 4096
#define SPL_SAMPLE_STRETCH 32768
#define SPL_SAMPLE_CLUSTER 8

struct __align__(128) SplSampleShared {
    unsigned int lo[SPL_SAMPLE_BINS], hi[SPL_SAMPLE_BINS];      // the bins: counts in lo, or weights in both
    unsigned long long list[SPL_SAMPLE_LIST];                   // values set aside: key << 32 | ~index, so that descending order is the definition's
    unsigned long long sums[SPL_SAMPLE_LIST];                   // running sums of bins or of the sorted list (first block)
    unsigned long long best[SPL_SAMPLE_CLUSTER];                // the blocks' largest values
    unsigned long long warp_sum[32], value[4];
    double powers[64];                                          // 2^(j / 64)
    unsigned int listed, found;
    // The first block's decision, in every block: which bins to set aside, or what has been decided.
    int step, first_bin, last_bin, also_first, also_last;
    unsigned long long cut;
};
enum { SPL_SAMPLE_DONE = 0, SPL_SAMPLE_FINISH, SPL_SAMPLE_CUT, SPL_SAMPLE_END, SPL_SAMPLE_DRAW, SPL_SAMPLE_WEIGH, SPL_SAMPLE_SLOW };

struct SplSampleRow { float t, p, u, m, bin_scale; SplSampleWeigh w; unsigned long long least; int k; };

__device__ __forceinline__ unsigned long long spl_sample_entry(uint32_t key, uint32_t index) { return (unsigned long long)key << 32 | uint32_t(~index); }

// Sum over the block's threads before this one (exclusive), and of all in *total.
__device__ __forceinline__ unsigned long long spl_sample_scan(unsigned long long v, SplSampleShared &sh, unsigned long long *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long run = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned long long y = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += y; }
    __syncthreads();
    if (lane == 31) sh.warp_sum[warp] = run;
    __syncthreads();
    if (warp == 0) {
        unsigned long long w = sh.warp_sum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const unsigned long long y = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += y; }
        sh.warp_sum[lane] = w;
    }
    __syncthreads();
    *total = sh.warp_sum[31];
    return (warp ? sh.warp_sum[warp - 1] : 0ull) + run - v;
}
// A block's share of the bins, all blocks' added, into the first block's sums. (A block past the last is the first again, left out: the loads of all are on
// their way together.)
__device__ __forceinline__ void spl_sample_add_blocks(SplSampleShared &sh, cooperative_groups::cluster_group &cluster, int rank, int blocks) {
    const int share = SPL_SAMPLE_BINS / blocks;
    unsigned long long *sums = cluster.map_shared_rank(&sh, 0)->sums;
    for (int i = rank * share + threadIdx.x; i < (rank + 1) * share; i += 1024) {
        unsigned int lo[SPL_SAMPLE_CLUSTER], hi[SPL_SAMPLE_CLUSTER];
#pragma unroll
        for (int b = 0; b < SPL_SAMPLE_CLUSTER; ++b) {
            const SplSampleShared *peer = cluster.map_shared_rank(&sh, b < blocks ? b : 0);
            lo[b] = peer->lo[i]; hi[b] = peer->hi[i];
        }
        unsigned long long sum = 0ull;
#pragma unroll
        for (int b = 0; b < SPL_SAMPLE_CLUSTER; ++b) if (b < blocks) sum += (unsigned long long)hi[b] << 32 | lo[b];
        sums[i] = sum;
    }
}
// The first block's sums of bins into running sums.
__device__ __forceinline__ void spl_sample_running(SplSampleShared &sh, unsigned long long *total) {
    unsigned long long v[SPL_SAMPLE_BINS / 1024], run = 0ull;
#pragma unroll
    for (int q = 0; q < SPL_SAMPLE_BINS / 1024; ++q) { v[q] = sh.sums[SPL_SAMPLE_BINS / 1024 * threadIdx.x + q]; run += v[q]; }
    run = spl_sample_scan(run, sh, total);
#pragma unroll
    for (int q = 0; q < SPL_SAMPLE_BINS / 1024; ++q) { run += v[q]; sh.sums[SPL_SAMPLE_BINS / 1024 * threadIdx.x + q] = run; }
    __syncthreads();
}
// The first place of [0, n) whose sums[] reaches `target` (n: none); the sums do not fall. All threads get it.
__device__ __forceinline__ int spl_sample_place(SplSampleShared &sh, int n, unsigned long long target) {
    __syncthreads();
    if (threadIdx.x == 0) sh.found = unsigned(n);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 1024) if (sh.sums[i] >= target && (i == 0 || sh.sums[i - 1] < target)) sh.found = unsigned(i);
    __syncthreads();
    return int(sh.found);
}
__device__ __forceinline__ unsigned long long spl_sample_target(float fraction, unsigned long long sum) {
    return fraction > 0.0f ? min(sum, (unsigned long long)ceil(double(fraction) * double(sum))) : 0ull;
}

// Places found on the row itself, eight bits of the keys at a time, by one block.
__device__ __noinline__ void spl_sample_slow(const SplSampleArgs &a, const SplSampleRow &r, SplSampleShared &sh, int row) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *x = a.logits + size_t(row) * a.ld;
    unsigned long long *mass = sh.sums;
    unsigned int *count = sh.lo, *warp_count = sh.hi;
    // What stays: keys above cut_key, and of cut_key itself the cut_ties lowest indices; and weights of at least `least`.
    uint32_t cut_key = 1u;
    unsigned long long cut_ties = ~0ull, least = 0ull;
    // The place in the order where the running count (by_count) or the running weight reaches `target` (at least the first place):
    // its key, and how many of the key's values the prefix takes.
    auto find = [&](bool by_count, unsigned long long target, uint32_t *key_out, unsigned long long *ties_out) {
        uint32_t prefix = 0u;
        unsigned long long before = 0ull;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) { mass[tid] = 0ull; count[tid] = 0u; }
            __syncthreads();
            for (int base = 0; base < a.limit; base += 1024) {
                const int i = base + tid;
                const float v = i < a.limit ? x[i] : -INFINITY;
                const uint32_t key = spl_topk_key(v);
                const unsigned long long w = by_count ? 1ull : spl_sample_weight(v, r.w);
                const bool counts = key >= cut_key && key != 0u && (shift == 24 || (key >> (shift + 8)) == prefix) && (by_count || w >= least);
                const unsigned int votes = __ballot_sync(0xffffffffu, counts);
                if (!votes) continue;
                const uint32_t digit = key >> shift & 255u, first = __shfl_sync(0xffffffffu, digit, __ffs(votes) - 1);
                // Rows come here because many values are equal: those of a warp are added before they meet the others'.
                if (__all_sync(0xffffffffu, !counts || digit == first)) {
                    unsigned long long sum = counts ? w : 0ull;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (lane == 0) { atomicAdd(&mass[first], sum); atomicAdd(&count[first], __popc(votes)); }
                } else if (counts) { atomicAdd(&mass[digit], w); atomicAdd(&count[digit], 1u); }
            }
            __syncthreads();
            if (tid == 0) {
                unsigned long long sum = before;
                int last = -1;
                for (int d = 255; d >= 0; --d) {
                    if (!count[d]) continue;
                    unsigned long long here = mass[d];
                    // The key that an earlier cut goes through keeps only its lowest indices.
                    if (shift == 0 && (prefix << 8 | uint32_t(d)) == cut_key && count[d] > cut_ties) here = mass[d] / count[d] * cut_ties;
                    last = d;
                    sh.value[0] = sum;
                    sum += here;
                    if (sum >= target) break;
                }
                sh.found = unsigned(last);
            }
            __syncthreads();
            prefix = prefix << 8 | sh.found;
            before = sh.value[0];
        }
        *key_out = prefix;
        const unsigned long long each = by_count ? 1ull : spl_sample_weight(spl_topk_value(prefix), r.w);
        *ties_out = target <= before + 1ull || each == 0ull ? 1ull : (target - before + each - 1ull) / each;
    };
    // The weight of all that stays.
    auto total = [&]() {
        __syncthreads();
        if (tid == 0) { mass[0] = 0ull; count[0] = 0u; }
        __syncthreads();
        unsigned long long sum = 0ull;
        unsigned int ties = 0u;
        for (int i = tid; i < a.limit; i += 1024) {
            const float v = x[i];
            const uint32_t key = spl_topk_key(v);
            if (key < cut_key || key == 0u) continue;
            if (key == cut_key) { ++ties; continue; }
            const unsigned long long w = spl_sample_weight(v, r.w);
            if (w >= least) sum += w;
        }
        if (sum) atomicAdd(&mass[0], sum);
        if (ties) atomicAdd(&count[0], ties);
        __syncthreads();
        const unsigned long long each = spl_sample_weight(spl_topk_value(cut_key), r.w);
        sum = mass[0];
        if (count[0] && each >= least) sum += each * min((unsigned long long)count[0], cut_ties);
        return sum;
    };
    if (r.k > 0 && r.k < a.limit) find(true, (unsigned long long)r.k, &cut_key, &cut_ties);
    if (r.p < 1.0f) {
        uint32_t key; unsigned long long ties;
        find(false, spl_sample_target(r.p, total()), &key, &ties);
        if (key > cut_key || ties < cut_ties) { cut_key = key; cut_ties = ties; }
    }
    least = r.least;
    uint32_t pick_key; unsigned long long pick_tie;
    find(false, spl_sample_target(r.u, total()), &pick_key, &pick_tie);
    // The pick_tie-th lowest index of pick_key: the block walks the row in order.
    unsigned long long seen = 0ull;
    for (int base = 0; base < a.limit; base += 1024) {
        const int i = base + tid;
        const bool hit = i < a.limit && spl_topk_key(x[i]) == pick_key;
        const unsigned int votes = __ballot_sync(0xffffffffu, hit);
        __syncthreads();
        if (lane == 0) warp_count[warp] = __popc(votes);
        __syncthreads();
        unsigned int before = 0u, all = 0u;
        for (int w = 0; w < 32; ++w) { if (w < warp) before += warp_count[w]; all += warp_count[w]; }
        if (hit && seen + before + __popc(votes & ((1u << lane) - 1u)) + 1u == pick_tie) a.ids[row] = i;
        seen += all;
        if (seen >= pick_tie) return;
    }
}

// The first block: the blocks' lists into its own, sorted, with running sums of weights that begin at `base`. Returns the entries, or -1 where
// they do not fit.
__device__ __forceinline__ int spl_sample_sorted(SplSampleShared &sh, cooperative_groups::cluster_group &cluster, int blocks, const SplSampleRow &r, unsigned long long base) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // Each warp works out where the blocks' lists go; the lists of the others are copied side by side, four warps each.
    unsigned int n = lane < blocks ? cluster.map_shared_rank(&sh, lane)->listed : 0u;
    const unsigned int mine = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const unsigned int y = __shfl_up_sync(0xffffffffu, n, o); if (lane >= o) n += y; }
    const unsigned int from = warp / 4, start = __shfl_sync(0xffffffffu, n - mine, from), more = __shfl_sync(0xffffffffu, mine, from);
    n = __shfl_sync(0xffffffffu, n, 31);
    if (n > SPL_SAMPLE_LIST) return -1;
    if (from > 0 && int(from) < blocks) {
        const SplSampleShared *peer = cluster.map_shared_rank(&sh, from);
        for (unsigned int i = (warp & 3) * 32 + lane; i < more; i += 128) sh.list[start + i] = peer->list[i];
    }
    unsigned int width = 32;
    while (width < n) width <<= 1;
    for (unsigned int i = n + tid; i < width; i += 1024) sh.list[i] = 0ull;
    __syncthreads();
    // Bitonic, descending: what meets within 32 entries in registers, the rest through shared memory.
    auto within = [&](unsigned int size, unsigned int first_stride) {
        for (unsigned int i = tid; i < width; i += 1024) {
            unsigned long long v = sh.list[i];
            for (unsigned int stride = first_stride; stride > 0; stride >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, v, stride);
                const bool larger = ((i & stride) == 0) == ((i & size) == 0);      // this entry takes the larger of the two
                v = (v > other) == larger ? v : other;
            }
            sh.list[i] = v;
        }
    };
    for (unsigned int i = tid; i < width; i += 1024) {
        unsigned long long v = sh.list[i];
#pragma unroll
        for (unsigned int size = 2; size <= 32; size <<= 1)
#pragma unroll
            for (unsigned int stride = size >> 1; stride > 0; stride >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, v, stride);
                const bool larger = ((i & stride) == 0) == ((i & size) == 0);
                v = (v > other) == larger ? v : other;
            }
        sh.list[i] = v;
    }
    for (unsigned int size = 64; size <= width; size <<= 1) {
        for (unsigned int stride = size >> 1; stride >= 32; stride >>= 1) {
            __syncthreads();
            for (unsigned int q = tid; q < width / 2; q += 1024) {
                const unsigned int i = 2 * q - (q & (stride - 1)), j = i + stride;
                const unsigned long long x = sh.list[i], y = sh.list[j];
                if ((x < y) == ((i & size) == 0)) { sh.list[i] = y; sh.list[j] = x; }
            }
        }
        __syncthreads();
        within(size, 16);
    }
    __syncthreads();
    unsigned long long w[SPL_SAMPLE_LIST / 1024], run = 0ull, all;
    const int per = width <= 1024 ? 1 : int(width / 1024);
#pragma unroll
    for (int e = 0; e < SPL_SAMPLE_LIST / 1024; ++e) {
        const unsigned int i = tid * per + e;
        w[e] = e < per && i < n ? spl_sample_weight(spl_topk_value(uint32_t(sh.list[i] >> 32)), r.w) : 0ull;
        run += w[e];
    }
    run = base + spl_sample_scan(run, sh, &all);
#pragma unroll
    for (int e = 0; e < SPL_SAMPLE_LIST / 1024; ++e) {
        run += w[e];
        const unsigned int i = tid * per + e;
        if (e < per && i < n) sh.sums[i] = run;
    }
    __syncthreads();
    return int(n);
}

// Grid (blocks a row, rows) in clusters of a row's blocks, 1,024 threads.
template <bool HELD>
__global__ void __launch_bounds__(1024, 1)
spl_sample_kernel(SplSampleArgs a) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(128) unsigned char spl_sample_raw[];
    SplSampleShared &sh = *reinterpret_cast<SplSampleShared *>(spl_sample_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int row = blockIdx.y, rank = blockIdx.x, blocks = gridDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float *x = a.logits + size_t(row) * a.ld;
    const int stretch = ((a.limit + blocks - 1) / blocks + 31) / 32 * 32, begin = rank * stretch, end = min(a.limit, begin + stretch);
    float *held = reinterpret_cast<float *>(spl_sample_raw + sizeof(SplSampleShared));
    const float *mine = x + begin;
    const int count = max(0, end - begin);
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");      // (a block's shared memory may be reached when it has begun)
    for (int i = tid; i < SPL_SAMPLE_BINS; i += 1024) { sh.lo[i] = 0u; sh.hi[i] = 0u; }
    if (tid == 0) sh.listed = 0u;
    if (tid < 64) sh.powers[tid] = exp2(double(tid) / 64.0);
    spl_grid_begin();
    // Every thread of the block runs f(four values, index of the first, step of the index) for its values; past the row's end a value is -inf.
    auto each = [&](auto &&f) {
        if constexpr (HELD) {
#pragma unroll 2
            for (int i = 4 * tid; i < stretch; i += 4096) {
                const float4 four = *reinterpret_cast<const float4 *>(held + i);
                const float value[4] = {four.x, four.y, four.z, four.w};
                f(value, begin + i, 1);
            }
        } else {
            for (int i = tid; i < count; i += 16384) {          // sixteen loads on their way
                float value[4][4];
#pragma unroll
                for (int q = 0; q < 16; ++q) value[q / 4][q % 4] = i + q * 1024 < count ? mine[i + q * 1024] : -INFINITY;
#pragma unroll
                for (int q = 0; q < 4; ++q) f(value[q], begin + i + q * 4096, 1024);
            }
        }
    };
    SplSampleRow r;
    r.t = a.temperature ? a.temperature[row] : 1.0f; r.p = a.top_p ? a.top_p[row] : 1.0f; r.u = a.uniform[row];
    // (At an infinite temperature every weight is one, or none beside an infinite value: min-p takes nothing away.)
    r.m = a.min_p && a.min_p[row] > 0.0f && r.t < INFINITY ? fminf(a.min_p[row], 1.0f) : 0.0f; r.k = a.top_k ? a.top_k[row] : 0;
    r.least = r.m > 0.0f ? (unsigned long long)ceil(double(r.m) * SPL_SAMPLE_UNIT) : 0ull;

    // The largest value and its lowest index.
    {
        uint32_t key = 0u, index = 0u;
        for (int base = 0; base < (HELD ? stretch : count); base += 16 * 1024) {      // sixteen loads on their way
            float value[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) { const int i = base + e * 1024 + tid; value[e] = i < count ? mine[i] : -INFINITY; }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int i = base + e * 1024 + tid;
                if (HELD && i < stretch) held[i] = value[e];
                const uint32_t y = spl_topk_key(value[e]);
                if (y > key) { key = y; index = uint32_t(begin + i); }
            }
        }
        const uint32_t all = __reduce_max_sync(0xffffffffu, key);
        const uint32_t first = __reduce_min_sync(0xffffffffu, key == all ? index : 0xffffffffu);
        if (lane == 0) sh.warp_sum[warp] = spl_sample_entry(all, first);
        __syncthreads();
        unsigned long long best = 0ull;
        if (warp == 0) {
            best = sh.warp_sum[lane];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        }
        asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        if (warp == 0 && lane < blocks) cluster.map_shared_rank(&sh, lane)->best[rank] = best;
        cluster.sync();
    }
    unsigned long long top = sh.best[0];
    for (int b = 1; b < blocks; ++b) top = max(top, sh.best[b]);
    const bool nothing = (top >> 32) == 0ull;          // id 0, as an untouched slot of a top-k
    if (nothing || !(r.t > 0.0f)) {
        if (rank == 0 && tid == 0) a.ids[row] = nothing ? 0 : int32_t(~uint32_t(top));
        return;
    }
    r.w.max = spl_topk_value(uint32_t(top >> 32));
    r.w.scale = 64.0 / 0.693147180559945309417 / double(r.t);
    r.w.powers = sh.powers;
    r.bin_scale = fminf(fmaxf(2.0f * SPL_SAMPLE_BINS_NAT / r.t, 1.0e-38f), SPL_SAMPLE_SCALE_MAX);      // (never zero: an infinite value's bin would be no number at an infinite temperature)
    // The bin of a value that may be picked: halved values do not overflow, and rounding keeps the order (it may put a value in the next bin, no more). Beside an
    // infinite maximum the finite values are binned as beside the largest one (they have no weight), and the infinite ones come to bin 0 by way of -inf.
    const float half_max = 0.5f * fminf(r.w.max, 3.402823466e38f);
    auto bin_of = [&](float value) {
        return __float_as_int(fminf(fmaf(-0.5f, value, half_max) * r.bin_scale, float(SPL_SAMPLE_BINS - 1)) + 8388608.0f) & (SPL_SAMPLE_BINS - 1);
    };
    unsigned long long cut = 0ull;                     // entries below it are out
    // The values of the bins [first, last] and [also_first, also_last] (in front of them; none where also_first is negative) into the block's list.
    auto set_aside = [&](int first, int last, int also_first, int also_last) {
        // Most values are told by comparisons: bounds a bin and the roundings outside the bins asked for.
        const float width = 2.0f / r.bin_scale, slack = 2.0f * width + 1e-6f * fabsf(r.w.max);
        auto top_of = [&](int b) { return r.w.max - float(b) * width + slack; };
        auto bottom_of = [&](int b) { return b == SPL_SAMPLE_BINS - 1 ? -INFINITY : r.w.max - float(b + 1) * width - slack; };
        const float high = top_of(first), low = bottom_of(last), also_high = also_first < 0 ? -INFINITY : top_of(also_first), also_low = also_first < 0 ? INFINITY : bottom_of(also_last);
        auto near = [&](float value) { return !(value > high || value < low) || !(value > also_high || value < also_low); };
        auto keep = [&](float value, int i) {
            const uint32_t key = spl_topk_key(value);
            const int b = bin_of(value);
            if (key == 0u || ((b < first || b > last) && (also_first < 0 || b < also_first || b > also_last))) return;
            const unsigned long long entry = spl_sample_entry(key, uint32_t(i));
            if (entry < cut) return;
            const unsigned int at = atomicAdd(&sh.listed, 1u);
            if (at < SPL_SAMPLE_LIST) sh.list[at] = entry;
        };
        each([&](const float (&value)[4], int i, int step) {
            if (!(near(value[0]) | near(value[1]) | near(value[2]) | near(value[3]))) return;
#pragma unroll
            for (int q = 0; q < 4; ++q) keep(value[q], i + q * step);
        });
        cluster.sync();
    };
    // The first block's decision goes to all of them; what their lists held has been read.
    auto decide = [&](int step, int first_bin, int last_bin, unsigned long long new_cut, int also_first = -1, int also_last = -1) {
        __syncthreads();
        if (tid < blocks) {
            SplSampleShared *peer = cluster.map_shared_rank(&sh, tid);
            peer->step = step; peer->first_bin = first_bin; peer->last_bin = last_bin; peer->also_first = also_first; peer->also_last = also_last; peer->cut = new_cut; peer->listed = 0u;
        }
    };
    int step = SPL_SAMPLE_WEIGH;
    if (r.k > 0 && r.k < a.limit) {
        unsigned int last = 0u;                        // values of the last bin are many: counted apart
        each([&](const float (&value)[4], int, int) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int b = bin_of(value[q]);
                if (value[q] > -INFINITY) { if (b == SPL_SAMPLE_BINS - 1) ++last; else atomicAdd(&sh.lo[b], 1u); }
            }
        });
        last = __reduce_add_sync(0xffffffffu, last);
        if (lane == 0 && last) atomicAdd(&sh.lo[SPL_SAMPLE_BINS - 1], last);
        cluster.sync();
        spl_sample_add_blocks(sh, cluster, rank, blocks);
        cluster.sync();
        if (rank == 0) {
            unsigned long long all;
            spl_sample_running(sh, &all);
            const int b = spl_sample_place(sh, SPL_SAMPLE_BINS, (unsigned long long)r.k);
            if (b < SPL_SAMPLE_BINS && sh.sums[b] <= SPL_SAMPLE_LIST) decide(SPL_SAMPLE_FINISH, 0, b, 0ull);
            else if (b >= SPL_SAMPLE_BINS - 1) decide(SPL_SAMPLE_WEIGH, 0, 0, 0ull);      // fewer values than k, or fewer with a weight: a cut among those without takes nothing away
            else {
                if (tid == 0) sh.value[1] = b ? sh.sums[b - 1] : 0ull;
                decide(SPL_SAMPLE_CUT, b, b, 0ull);
            }
        }
        cluster.sync();
        step = sh.step;
        if (step != SPL_SAMPLE_WEIGH) {
            set_aside(sh.first_bin, sh.last_bin, -1, -1);
            if (rank == 0) {
                const int n = spl_sample_sorted(sh, cluster, blocks, r, 0ull);
                if (n < 0) decide(SPL_SAMPLE_SLOW, 0, 0, 0ull);
                else if (step == SPL_SAMPLE_CUT) decide(SPL_SAMPLE_WEIGH, 0, 0, sh.list[r.k - int(sh.value[1]) - 1]);
                else {
                    int stay = min(n, r.k);
                    if (r.p < 1.0f) stay = min(stay, spl_sample_place(sh, stay, spl_sample_target(r.p, sh.sums[stay - 1])) + 1);
                    if (r.least) {
                        // Weights do not rise along the list.
                        __syncthreads();
                        if (tid == 0) sh.found = unsigned(stay);
                        __syncthreads();
                        for (int i = tid; i < stay; i += 1024)
                            if (sh.sums[i] - (i ? sh.sums[i - 1] : 0ull) < r.least && (i == 0 || sh.sums[i - 1] - (i > 1 ? sh.sums[i - 2] : 0ull) >= r.least)) sh.found = unsigned(i);
                        __syncthreads();
                        stay = int(sh.found);
                    }
                    const int pick = spl_sample_place(sh, stay, spl_sample_target(r.u, sh.sums[stay - 1]));
                    if (tid == 0) a.ids[row] = int32_t(~uint32_t(sh.list[pick]));
                    decide(SPL_SAMPLE_DONE, 0, 0, 0ull);
                }
            }
            cluster.sync();
            step = sh.step;
            cut = sh.cut;
        }
    }
    if (step == SPL_SAMPLE_WEIGH) {
        for (int i = tid; i < SPL_SAMPLE_BINS; i += 1024) { sh.lo[i] = 0u; sh.hi[i] = 0u; }
        __syncthreads();
        // Values that cannot count are passed over: without top-p nothing below min-p's bound is in any sum (a bin and the roundings of slack). Beside an infinite maximum the bound
        // would be no number, which nothing reaches: there all values are looked at.
        const float least_value = r.least && !(r.p < 1.0f) && r.w.max < INFINITY ? r.w.max - (-logf(r.m) + 4.0f / SPL_SAMPLE_BINS_NAT) * r.t - 1e-6f * fabsf(r.w.max) : -INFINITY;
        const bool guarded = r.w.max == INFINITY || r.bin_scale == SPL_SAMPLE_SCALE_MAX;      // the last bin does not hold all values of no weight
        each([&](const float (&value)[4], int i, int step) {
            if (!(value[0] >= least_value) & !(value[1] >= least_value) & !(value[2] >= least_value) & !(value[3] >= least_value)) return;
            // The four weights side by side (a weight is a chain of ten 64-bit operations), whatever of them counts.
            unsigned long long w[4];
            int b[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) { b[q] = bin_of(value[q]); w[q] = spl_sample_weight_near(value[q], r.w); }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (!(value[q] > -INFINITY) || b[q] == SPL_SAMPLE_BINS - 1) continue;
                if (cut && spl_sample_entry(spl_topk_key(value[q]), uint32_t(i + q * step)) < cut) continue;
                if (guarded) { if (value[q] == r.w.max) w[q] = 1ull << 44; else if (spl_sample_weightless(value[q], r.w)) continue; }
                // Two words a bin, the carry taken by whoever makes the lower one overflow.
                const unsigned int low = unsigned(w[q]), was = atomicAdd(&sh.lo[b[q]], low), high = unsigned(w[q] >> 32) + (was + low < was ? 1u : 0u);
                if (high) atomicAdd(&sh.hi[b[q]], high);
            }
        });
        cluster.sync();
        spl_sample_add_blocks(sh, cluster, rank, blocks);
        cluster.sync();
        // The first block: what stays ends in the bins [c0, c1], or nowhere before the last value.
        int c0 = SPL_SAMPLE_BINS, c1 = -1, p_bin = SPL_SAMPLE_BINS, also = -1, also_last = -1;
        unsigned long long p_target = 0ull, all = 0ull;
        if (rank == 0) {
            spl_sample_running(sh, &all);
            // The bins' sums, here for the places below and, where the bins were, for the draw.
            unsigned long long *keep = reinterpret_cast<unsigned long long *>(sh.lo);      // lo and hi
            for (int i = tid; i < SPL_SAMPLE_BINS; i += 1024) keep[i] = sh.sums[i];
            if (r.p < 1.0f) { p_target = spl_sample_target(r.p, all); p_bin = spl_sample_place(sh, SPL_SAMPLE_BINS, p_target); }
            if (p_bin < SPL_SAMPLE_BINS) c0 = c1 = p_bin;
            if (r.least) {
                // Weights of m lie -ln m below the maximum; the bins next to that one may hold some, too, for the rounding of their place.
                const int m_bin = int(fminf(fmaxf(-logf(r.m) * (0.5f * r.bin_scale * r.t), 0.0f), float(SPL_SAMPLE_BINS - 2))), m0 = max(m_bin - 1, 0), m1 = min(m_bin + 1, SPL_SAMPLE_BINS - 2);      // (the last bin's have no weight)
                if (p_bin > m1) { c0 = m0; c1 = m1; p_bin = SPL_SAMPLE_BINS; }      // top-p's place comes later
                else if (p_bin >= m0) { c0 = m0; c1 = m1; }
            }
            if (c1 >= 0) {
                // Whatever of the bins [c0, c1] stays, the draw mostly lies in one and the same bin, or one of a few: set aside with them, it is found in the same list. (With one bin
                // alone a fifth of the rows of a vocabulary of 248,077 needed another turn.)
                const unsigned long long least_sum = c0 ? sh.sums[c0 - 1] : 0ull;
                const int d0 = spl_sample_place(sh, SPL_SAMPLE_BINS, spl_sample_target(r.u, least_sum)), d1 = spl_sample_place(sh, SPL_SAMPLE_BINS, spl_sample_target(r.u, sh.sums[c1]));
                if (d0 < c0 && min(d1, c0 - 1) - d0 < 8) { also = d0; also_last = min(d1, c0 - 1); }
                decide(SPL_SAMPLE_END, c0, c1, cut, also, also_last);
            } else {
                const int b = spl_sample_place(sh, SPL_SAMPLE_BINS, spl_sample_target(r.u, all));
                decide(SPL_SAMPLE_DRAW, b, b, cut);
            }
        }
        cluster.sync();
        step = sh.step;
        const unsigned long long *kept = reinterpret_cast<const unsigned long long *>(sh.lo);
        unsigned long long target = rank == 0 && step == SPL_SAMPLE_DRAW ? spl_sample_target(r.u, all) : 0ull;
        while (step == SPL_SAMPLE_END) {                                               // (twice at most)
            set_aside(sh.first_bin, sh.last_bin, sh.also_first, sh.also_last);
            if (rank == 0) {
                // The list: the draw's bins where they came along (entries [0, front)), then the bins what stays ends in, running sums from `base`.
                const unsigned long long base = c0 ? kept[c0 - 1] : 0ull, also_base = also > 0 ? kept[also - 1] : 0ull, also_sum = also < 0 ? 0ull : kept[also_last] - also_base;
                const int n = spl_sample_sorted(sh, cluster, blocks, r, base - also_sum);
                if (n < 0 && also >= 0) { also = -1; decide(SPL_SAMPLE_END, c0, c1, cut); }      // too many together: the draw has a turn of its own
                else if (n < 0) decide(SPL_SAMPLE_SLOW, 0, 0, 0ull);
                else {
                    int front = 0;
                    if (also >= 0) {
                        __syncthreads();
                        if (tid == 0) sh.found = unsigned(n);
                        __syncthreads();
                        for (int i = tid; i < n; i += 1024) {
                            auto in_front = [&](int e) { return bin_of(spl_topk_value(uint32_t(sh.list[e] >> 32))) <= also_last; };
                            if (!in_front(i) && (i == 0 || in_front(i - 1))) sh.found = unsigned(i);
                        }
                        __syncthreads();
                        front = int(sh.found);
                    }
                    int stay = n;
                    if (p_bin < SPL_SAMPLE_BINS && n > front) {
                        __syncthreads();
                        if (tid == 0) sh.found = unsigned(n);
                        __syncthreads();
                        for (int i = front + tid; i < n; i += 1024) if (sh.sums[i] >= p_target && (i == front || sh.sums[i - 1] < p_target)) sh.found = unsigned(i);
                        __syncthreads();
                        stay = min(n, int(sh.found) + 1);
                    }
                    if (r.least) {
                        __syncthreads();
                        if (tid == 0) sh.found = unsigned(stay);
                        __syncthreads();
                        auto weight_of = [&](int e) { return spl_sample_weight(spl_topk_value(uint32_t(sh.list[e] >> 32)), r.w); };      // does not rise along the list
                        for (int i = front + tid; i < stay; i += 1024) if (weight_of(i) < r.least && (i == front || weight_of(i - 1) >= r.least)) sh.found = unsigned(i);
                        __syncthreads();
                        stay = int(sh.found);
                    }
                    target = spl_sample_target(r.u, stay > front ? sh.sums[stay - 1] : base);
                    int from = -1, to = stay;
                    unsigned long long shift = 0ull;
                    if (target > base || base == 0ull) from = front;
                    else if (also >= 0 && target > also_base && target <= also_base + also_sum) { from = 0; to = front; shift = base - also_sum - also_base; }
                    else if (also == 0) { from = 0; to = front; shift = base - also_sum; }      // a target of nothing: the first value
                    if (from >= 0) {
                        __syncthreads();
                        if (tid == 0) sh.found = unsigned(to - 1);
                        __syncthreads();
                        for (int i = from + tid; i < to; i += 1024) if (sh.sums[i] - shift >= target && (i == from || sh.sums[i - 1] - shift < target)) sh.found = unsigned(i);
                        __syncthreads();
                        if (tid == 0) a.ids[row] = int32_t(~uint32_t(sh.list[sh.found]));
                        decide(SPL_SAMPLE_DONE, 0, 0, 0ull);
                    } else {
                        __syncthreads();
                        for (int i = tid; i < SPL_SAMPLE_BINS; i += 1024) sh.sums[i] = kept[i];
                        const int b = spl_sample_place(sh, SPL_SAMPLE_BINS, target);
                        decide(SPL_SAMPLE_DRAW, b, b, cut);
                    }
                }
            }
            cluster.sync();
            step = sh.step;
        }
        if (step == SPL_SAMPLE_DRAW) {
            const int b = sh.first_bin;
            set_aside(b, b, -1, -1);
            if (rank == 0) {
                const int n = spl_sample_sorted(sh, cluster, blocks, r, b ? kept[b - 1] : 0ull);
                if (n < 0) decide(SPL_SAMPLE_SLOW, 0, 0, 0ull);
                else {
                    const int pick = spl_sample_place(sh, n, target);
                    if (tid == 0) a.ids[row] = int32_t(~uint32_t(sh.list[pick]));
                    decide(SPL_SAMPLE_DONE, 0, 0, 0ull);
                }
            }
            cluster.sync();
            step = sh.step;
        }
    }
    if (step == SPL_SAMPLE_SLOW && rank == 0) spl_sample_slow(a, r, sh, row);
}
