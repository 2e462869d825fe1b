// spl_paged_e4m3.cuh — attention of the new rows over a paged cache of e4m3 codes with a scale a token and kv head.
//
// o = sum_t p_t vs_t V_t / sum_t p_t with p_t = exp(scale ks_t q.K_t - m), K and V codes, ks and vs their scales: spl_paged_attend_kernel's pieces, tiles, roles and joins, with half its bytes.
// What differs:
//   S = Q K^T      in 8 bits, K as it lies in the cache. A bf16 query is the sum of two e4m3 (four significant bits each) once its row is scaled by the power of two that puts its largest
//                  channel in [128, 256): both are rows of the A operand's tile, and a tile's scores are 2 HD / 32 instructions of 32 channels, as long as a 16-bit product's HD / 16. What is lost is
//                  below 2^-17 of the row's largest channel.
//   O += P V       in fp16, which holds every code exactly. Two pairs of warps turn the values of a chunk into fp16 on their way to the products, each every second chunk (V as 8-bit operand would want P in 8 bits, too: a
//                  weight below 2^-17 of the row's largest would be lost, and many tokens of small weight are not a small matter).
// The value scales go into the exponent: y_t = log2 of p_t vs_t = x_t + log2 vs_t has the running reference, so that P = 2^(y - ref) uses fp16's range for what counts in the row's sum, whatever the
// sizes of values that do not (a running maximum of x alone would leave tokens of small values in the subnormals beside one of large ones); the denominator adds P / vs. The warp that copies keys writes each
// token's ks, log2 vs and 1 / vs beside them.
// Values behind the sequence's last token and in front of every row's window are zeros in fp16, whatever the cache holds there.
#pragma once
#include "spl_paged.cuh"

#define SPL_PAGED8_SOFTMAX 16          // warps: four of 32 tokens a quarter of the rows
#define SPL_PAGED8_THREADS (32 * (SPL_PAGED8_SOFTMAX + 8))
__host__ __device__ constexpr int spl_paged8_k_chunk(int hd) { return hd == 64 ? 8192 : 16384; }          // 128 tokens by up to 128 channels
__host__ __device__ constexpr int spl_paged8_v_tokens(int hd) { return hd == 256 ? 64 : 128; }            // a chunk of values: tokens by all channels
__host__ __device__ constexpr int spl_paged8_ring_k(int hd) { return hd == 64 ? 6 : hd == 128 ? 5 : 3; }
// Chunks of values, as they lie and in fp16: even numbers, for two pairs of warps take turns at them and a pair has to meet every phase of its places' barriers.
__host__ __device__ constexpr int spl_paged8_ring_v(int hd) { return hd == 64 ? 6 : 2; }
__host__ __device__ constexpr int spl_paged8_ring_w(int hd) { return hd == 64 ? 4 : 2; }
static_assert(spl_paged8_ring_v(64) % 2 == 0 && spl_paged8_ring_v(128) % 2 == 0 && spl_paged8_ring_v(256) % 2 == 0 && spl_paged8_ring_w(64) % 2 == 0 && spl_paged8_ring_w(128) % 2 == 0 && spl_paged8_ring_w(256) % 2 == 0, "");
// Tiles of scales. Those of tile j are written behind its first keys, which waited for the scores of the tile a ring before, and these for the softmax of the tile two before that.
__host__ __device__ constexpr int spl_paged8_scales(int hd) { return (spl_paged8_ring_k(hd) + (hd == 256 ? 1 : 0)) / (hd == 256 ? 2 : 1) + 2; }
__host__ __device__ constexpr size_t spl_paged8_smem_bytes(int hd) {
    return size_t(hd) * 256 /* Q, two parts */ + size_t(spl_paged8_ring_k(hd)) * spl_paged8_k_chunk(hd) + size_t(spl_paged8_ring_v(hd) + 2 * spl_paged8_ring_w(hd)) * spl_paged8_v_tokens(hd) * hd +
           spl_paged8_scales(hd) * 3 * 512 + 2 * 512 /* the rows' factors */ + 2 * 4 * 512 /* maxima, sums */ + 512 /* barriers */;
}

// A weight P / vs has to be there beside the row's largest product P = p vs, and fp32 ends at 2^-126: value scales count as 2^-60 at least (what they stand for is below 4e-16 then) and are no numbers above 2^40, which
// leaves weights down to 2^-33 of the largest.
#define SPL_PAGED8_SCALE_LEAST 8.673617379884035e-19f
#define SPL_PAGED8_SCALE_MOST 1.099511627776e12f
struct SplPagedScaled { const float *k, *v; };

__device__ __forceinline__ void spl_tc_mma8_ss_if(uint32_t elected, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n @e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected) : "memory");
}
// K-major rows of 128 bytes (128-byte swizzle), or of 64 (64-byte swizzle: eight-row groups 512 bytes apart).
template <int HD> __device__ __forceinline__ uint64_t spl_paged8_desc(uint32_t addr) {
    if constexpr (HD >= 128) return spl_tc_desc_sw128(addr);
    else return uint64_t((addr & 0x3FFFFu) >> 4) | uint64_t(1) << 16 | uint64_t(512 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(4) << 61;
}
__device__ __forceinline__ uint32_t spl_halves_of_e4m3(uint16_t v) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"(v));
    return h;
}

// Sixteen rows by 32 columns of fp32 from tensor memory in the shape 16x256b: register 4 j + e is row lane / 4 + 8 (e / 2), column 8 j + 2 (lane % 4) + e % 2; and 16 rows by 16 words into it in
// 16x128b: register 2 j + e is row lane / 4 + 8 e, word 4 j + lane % 4.
__device__ __forceinline__ void spl_tc_ld_rows(uint32_t *r, uint32_t taddr) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
// The registers of loads are defined behind this.
__device__ __forceinline__ void spl_tc_ld_done(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) : : "memory");
    asm volatile("" : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) : : "memory");
}
__device__ __forceinline__ void spl_tc_st_rows(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// Four values a lane, each to be reduced over the four lanes of lane / 4: lane % 4 = i gets value i's.
template <typename Op> __device__ __forceinline__ float spl_paged8_reduce(const float (&v)[4], int lane, Op &&op) {
    const bool high = lane & 2, odd = lane & 1;
    const float a = op(high ? v[2] : v[0], __shfl_xor_sync(0xffffffffu, high ? v[0] : v[2], 2)), b = op(high ? v[3] : v[1], __shfl_xor_sync(0xffffffffu, high ? v[1] : v[3], 2));
    return op(odd ? b : a, __shfl_xor_sync(0xffffffffu, odd ? a : b, 1));
}
// Four warps meet: barriers 1 to 4; and whether any of their threads says so.
__device__ __forceinline__ void spl_paged8_barrier(int which) {
    if (which == 0) spl_named_barrier<1, 128>();
    else if (which == 1) spl_named_barrier<2, 128>();
    else if (which == 2) spl_named_barrier<3, 128>();
    else spl_named_barrier<4, 128>();
}
template <int ID> __device__ __forceinline__ bool spl_named_barrier_or(bool mine) {
    uint32_t any;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(any) : "r"(uint32_t(mine)), "n"(ID) : "memory");
    return any;
}
__device__ __forceinline__ bool spl_paged8_barrier_or(int which, bool mine) {
    return which == 0 ? spl_named_barrier_or<1>(mine) : which == 1 ? spl_named_barrier_or<2>(mine) : which == 2 ? spl_named_barrier_or<3>(mine) : spl_named_barrier_or<4>(mine);
}
// A row's P are 2^(y + offset), offset = 7 - reference. While no y + offset of a tile is above SPL_PAGED8_MOST the reference may stay, and nobody looks for a maximum; a row that has seen nothing has an offset that takes any number above that: the largest of fp32, so that scores far below zero raise it, too.
#define SPL_PAGED8_MOST 15.0f
#define SPL_PAGED8_UNSEEN 3.402823466e38f
__device__ __forceinline__ float spl_lg2(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float spl_rcp(float x) { float y; asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x)); return y; }

template <int HD>
__global__ void __launch_bounds__(SPL_PAGED8_THREADS, 1)
spl_paged_attend_e4m3_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, SplPagedTables t, SplPagedShape s, SplPagedAttend a, SplPagedScaled scales) {
    constexpr int NK = spl_paged8_ring_k(HD), NV = spl_paged8_ring_v(HD), NW = spl_paged8_ring_w(HD), NS = spl_paged8_scales(HD), KCHUNK = spl_paged8_k_chunk(HD), VT = spl_paged8_v_tokens(HD);
    constexpr int KPARTS = HD == 256 ? 2 : 1, VPARTS = 128 / VT, VCHUNK = VT * HD, WCHUNK = 2 * VCHUNK, QPART = HD * 128, ROW = HD == 64 ? 64 : 128;      // ROW: bytes of a K-major row
    constexpr float PBIAS = 7.0f;
    constexpr int COPY_K = SPL_PAGED8_SOFTMAX, SCORES = COPY_K + 1, VALUES = COPY_K + 2, COPY_V = COPY_K + 3, CONVERT = COPY_K + 4;      // the roles' warps
    extern __shared__ __align__(1024) unsigned char spl_paged8_raw[];
    if (spl_smem_addr(spl_paged8_raw) % 1024) { if (threadIdx.x == 0) a.error_flag[0] = 299; return; }
    unsigned char *q_tile = spl_paged8_raw, *ring = q_tile + 2 * QPART, *v_ring = ring + NK * KCHUNK, *w_ring = v_ring + NV * VCHUNK;
    float *scale_ring = reinterpret_cast<float *>(w_ring + NW * WCHUNK);      // [tile % NS][ks, log2 vs, 1 / vs][token]
    float *factor = scale_ring + NS * 3 * 128;                                // [item parity][row]
    float *xmax = factor + 2 * 128;                                           // [tile parity][quarter of the tokens][row]
    uint64_t *bars = reinterpret_cast<uint64_t *>(xmax + 2 * 4 * 128);
    uint64_t *full_k = bars, *empty_k = full_k + NK, *full_v = empty_k + NK, *empty_v = full_v + NV, *full_w = empty_v + NV, *empty_w = full_w + NW, *scaled = empty_w + NW, *s_full = scaled + NS, *p_full = s_full + 2,
             *o_done = p_full + 2, *q_full = o_done + 2, *drained = q_full + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drained + 2);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1), *joins = abort + 1;
    auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < NK; ++i) { spl_mbar_init(&full_k[i], 1); spl_mbar_init(&empty_k[i], 1); }
        for (int i = 0; i < NV; ++i) { spl_mbar_init(&full_v[i], 1); spl_mbar_init(&empty_v[i], 2); }
        for (int i = 0; i < NW; ++i) { spl_mbar_init(&full_w[i], 2); spl_mbar_init(&empty_w[i], 1); }
        for (int i = 0; i < NS; ++i) spl_mbar_init(&scaled[i], 1);
        for (int i = 0; i < 2; ++i) { spl_mbar_init(&s_full[i], 1); spl_mbar_init(&p_full[i], SPL_PAGED8_SOFTMAX); spl_mbar_init(&o_done[i], 1); }
        spl_mbar_init(q_full, SPL_PAGED8_SOFTMAX); spl_mbar_init(&drained[0], 1); spl_mbar_init(&drained[1], 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (tid == 32 * COPY_K) { spl_tma_prefetch(&k_map); spl_tma_prefetch(&v_map); }
    if (warp == SCORES) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(spl_smem_addr(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    spl_tc_fence_before();
    __syncthreads();
    spl_tc_fence_after();
    const uint32_t tmem = uint32_t(uniform(int(*tmem_slot))), tmem_o = tmem + 256;
    // What the batch's copies brought is read before the kernel in front is done, and the first tiles are asked for, as in spl_paged_attend_kernel.
    union { SplPagedItem item; int4 four[sizeof(SplPagedItem) / 16]; } first;
#pragma unroll
    for (int i = 0; i < int(sizeof(SplPagedItem) / 16); ++i) first.four[i] = __ldcg(reinterpret_cast<const int4 *>(a.starts + blockIdx.x) + i);
    const SplPagedItem first_item = first.item;
    const int item0 = uniform(__ldcg(a.block_begin + blockIdx.x)), item1 = uniform(__ldcg(a.block_begin + blockIdx.x + 1));
    // A tile's boxes of tokens: a page, or half a page of 256. Keys: a box's tokens by a chunk's channels. Values: boxes of at most the chunk's tokens by all channels. Lane b holds the page of the tile's b-th box.
    const int box = min(s.page_tokens, 128), boxes = 128 / box, vbox = min(s.page_tokens, VT), vboxes = VT / vbox, per_page = box / vbox;
    auto page_of = [&](const SplPagedItem &it, int tile) {
        return tile < it.tile_end && lane < min(boxes, (it.length - tile * 128 + box - 1) / box) ? __ldcg(t.table + size_t(it.sequence) * s.max_pages + (s.page_tokens > 128 ? tile >> 1 : tile * boxes + lane)) : 0;
    };
    auto inside_page = [&](int tile) { return s.page_tokens > 128 ? (tile & 1) * 128 : 0; };
    auto key_boxes = [&](const SplPagedItem &it, int tile) { return (min(128, it.length - tile * 128) + box - 1) / box; };
    auto value_boxes = [&](const SplPagedItem &it, int tile, int c) { return min(vboxes, max(0, (min(128, it.length - tile * 128) - c * VT + vbox - 1) / vbox)); };
    auto value_page = [&](int page, int c) { return __shfl_sync(0xffffffffu, page, lane < vboxes ? (c * vboxes + lane) / per_page : 0); };
    const int first_page = (warp == COPY_K || warp == COPY_V) && item0 < item1 ? page_of(first_item, first_item.tile_begin) : 0;
    if ((warp == COPY_K || warp == COPY_V) && item0 < item1) {
        int page = first_page;
        for (int tile = first_item.tile_begin; tile < min(first_item.tile_end, first_item.tile_begin + SPL_PAGED_EARLY); ++tile) {
            const int ahead = page_of(first_item, tile + 1), inside = inside_page(tile);
            if (warp == COPY_K) {
                for (int c = 0; c < KPARTS; ++c) if (lane < key_boxes(first_item, tile)) spl_tma_prefetch5(&k_map, 0, inside, c, first_item.kv_head, page);
            } else for (int c = 0; c < VPARTS; ++c) {
                const int from = value_page(page, c);
                if (lane < value_boxes(first_item, tile, c)) spl_tma_prefetch5(&v_map, 0, inside + (c * vboxes + lane) % per_page * vbox, 0, first_item.kv_head, from);
            }
            page = ahead;
        }
    }
    spl_grid_begin();
    // Waits and what gives them up: as in spl_paged_attend_kernel.
    int ok = 1;
    auto gave_up = [&](int code) { ok = 0; if (!*abort && lane == 0) { spl_note_wait(a.error_flag, code, 0); a.error_flag[0] = 200 + warp; } *abort = 1; };
    auto wait = [&](uint64_t *bar, int phase, int code) { if (ok && !spl_mbar_wait_warp(bar, phase & 1, const_cast<const int *>(abort))) gave_up(code); return ok != 0; };
    // The softmax's waits: the empty statement keeps the compiler from making a second loop for the case that a wait has run out. With the loop twice as large its instructions came too late: 2,048 rows over
    // 8,192 tokens of 32/8 heads of 128 took 671 us instead of 390. (The products' loops are faster without it.)
    auto meet = [&](uint64_t *bar, int phase, int code) { wait(bar, phase, code); asm volatile("" : "+r"(ok)); };
    // Tokens that some row of a piece sees.
    auto seen_first = [&](const SplPagedItem &it) { return spl_paged_first(s, it.base + it.q0 / s.group); };
    auto seen_last = [&](const SplPagedItem &it) { return spl_paged_last(s, it.base + (it.q0 + it.q_count - 1) / s.group, it.length); };

    if (warp == COPY_K || warp == COPY_V) {
        // ---- copies, a warp for keys and one for values.
        const bool keys = warp == COPY_K;
        uint64_t *full = keys ? full_k : full_v, *empty = keys ? empty_k : empty_v;
        const int slots = keys ? NK : NV;
        int n = 0, st = 0, tiles = 0;
        SplPagedItem it = first_item;
        int page = first_page;
        for (int i = item0; i < item1 && ok; ++i) {
            if (i > item0) { it = a.items[i]; page = page_of(it, it.tile_begin); }
            const int seen0 = seen_first(it), seen1 = seen_last(it);
            for (int tile = it.tile_begin; tile < it.tile_end && ok; ++tile, ++tiles) {
                const int ahead = page_of(it, tile + 1), inside = inside_page(tile);
                for (int c = 0; c < (keys ? KPARTS : VPARTS) && wait(&empty[st], (n / slots) + 1, 60); ++c) {
                    const int there = keys ? key_boxes(it, tile) : value_boxes(it, tile, c), from = keys ? page : value_page(page, c);
                    if (lane == 0) spl_mbar_expect_tx(&full[st], uint32_t(there) * (keys ? box * ROW : vbox * HD));
                    __syncwarp();
                    if (lane < there) {
                        if (keys) spl_tma_load5(ring + st * KCHUNK + lane * box * ROW, &k_map, 0, inside, c, it.kv_head, from, &full[st]);
                        else spl_tma_load5(v_ring + st * VCHUNK + lane * vbox * HD, &v_map, 0, inside + (c * vboxes + lane) % per_page * vbox, 0, it.kv_head, from, &full[st]);
                    }
                    ++n; st = st + 1 == slots ? 0 : st + 1;
                    if (keys && c == 0) {
                        // The tile's scales, four tokens a lane (of one page); what no row sees is masked.
                        const int mine = 4 * lane, token = tile * 128 + mine;
                        const size_t at = (size_t(__shfl_sync(0xffffffffu, page, mine / box)) * s.kv_heads + it.kv_head) * s.page_tokens + inside + mine % box;
                        float k[4] = {0.0f, 0.0f, 0.0f, 0.0f}, l[4] = {0.0f, 0.0f, 0.0f, 0.0f}, inv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        if (token + 4 > seen0 && token < seen1) {
                            const float4 ks = __ldcg(reinterpret_cast<const float4 *>(scales.k + at)), vs = __ldcg(reinterpret_cast<const float4 *>(scales.v + at));
                            const float given_k[4] = {ks.x, ks.y, ks.z, ks.w}, given_v[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if (token + e < seen0 || token + e >= seen1) continue;
                                const float v = given_v[e] >= 0.0f && given_v[e] <= SPL_PAGED8_SCALE_MOST ? fmaxf(given_v[e], SPL_PAGED8_SCALE_LEAST) : __int_as_float(0x7fffffff);
                                k[e] = given_k[e]; l[e] = spl_lg2(v); inv[e] = spl_rcp(v);
                            }
                        }
                        float *put = scale_ring + (tiles % NS) * 3 * 128 + mine;
                        *reinterpret_cast<float4 *>(put) = make_float4(k[0], k[1], k[2], k[3]);
                        *reinterpret_cast<float4 *>(put + 128) = make_float4(l[0], l[1], l[2], l[3]);
                        *reinterpret_cast<float4 *>(put + 256) = make_float4(inv[0], inv[1], inv[2], inv[3]);
                        __syncwarp();
                        if (lane == 0) spl_mbar_arrive(&scaled[tiles % NS]);
                    }
                }
                page = ahead;
            }
        }
        // Nothing may still be on its way into the block's shared memory when it is handed on.
        for (int z = 0; z < slots && z < n; ++z) spl_mbar_wait(&full[z], ((z + (n - 1 - z) / slots * slots) / slots) & 1);
    } else if (warp == SCORES || warp == VALUES) {
        // ---- the products, a warp each, issued by one elected lane of a converged warp.
        const uint32_t elected = spl_elect_one() ? 1u : 0u;
        const bool first_product = warp == SCORES;
        constexpr uint32_t s_idesc = spl_tc_idesc(128), o_idesc = spl_paged_idesc(HD, false, true);      // (e4m3 is format 0 of its kind, as fp16 is of the other)
        const uint64_t q_desc = spl_paged8_desc<HD>(spl_smem_addr(q_tile)), k_desc = spl_paged8_desc<HD>(spl_smem_addr(ring)), w_desc = spl_tc_desc_mn_sw128(spl_smem_addr(w_ring), VT * 128);
        int n = 0, tiles = 0;
        for (int i = item0; i < item1 && ok; ++i) {
            const int count = uniform(a.items[i].tile_end) - uniform(a.items[i].tile_begin);
            if (first_product) {
                if (!wait(q_full, i - item0, 63)) break;
                for (int tile = 0; tile < count && ok; ++tile) {
                    const int at = tiles + tile;
                    if (!wait(&full_k[n % NK], n / NK, 62)) break;
                    if (at >= 2 && !wait(&o_done[at & 1], (at - 2) >> 1, 61)) break;      // the place of the scores held the P of tile at - 2
#pragma unroll
                    for (int c = 0; c < KPARTS; ++c, ++n) {
                        const int st = n % NK;
                        if (c > 0 && !wait(&full_k[st], n / NK, 62)) break;
                        spl_tc_fence_after();
#pragma unroll
                        for (int part = 0; part < 2; ++part)
#pragma unroll
                            for (int ks = 0; ks < ROW / 32; ++ks)
                                spl_tc_mma8_ss_if(elected, tmem + (at & 1) * 128, q_desc + uint64_t((part * QPART + c * 16384 + ks * 32) >> 4), k_desc + uint64_t((st * KCHUNK + ks * 32) >> 4), s_idesc,
                                                  c + part + ks > 0 ? 1u : 0u);
                        spl_tc_commit_if(elected, &empty_k[st]);
                        if (c == KPARTS - 1) spl_tc_commit_if(elected, &s_full[at & 1]);
                    }
                }
            } else {
                for (int tile = 0; tile < count && ok; ++tile) {
                    const int at = tiles + tile;
                    for (int c = 0; c < VPARTS && ok; ++c, ++n) {
                        const int st = n % NW;
                        if (!wait(&full_w[st], n / NW, 65) || (c == 0 && !wait(&p_full[at & 1], at >> 1, 64))) break;
                        spl_tc_fence_after();
#pragma unroll
                        for (int ks = 0; ks < VT / 16; ++ks)      // (the piece's first product overwrites what O held)
                            spl_tc_mma_ts_if(elected, tmem_o, tmem + (at & 1) * 128 + (c * (VT / 16) + ks) * 8, w_desc + uint64_t((st * WCHUNK + ks * 2048) >> 4), o_idesc, tile + c + ks > 0 ? 1u : 0u);
                        spl_tc_commit_if(elected, &empty_w[st]);
                        if (c == VPARTS - 1) spl_tc_commit_if(elected, &o_done[at & 1]);
                    }
                }
            }
            tiles += count;
        }
        // No product may still read shared or write tensor memory when they are handed on.
        spl_tc_commit_if(elected, &drained[first_product ? 0 : 1]);
        spl_mbar_wait(&drained[first_product ? 0 : 1], 0);
    } else if (warp >= CONVERT) {
        // ---- values into fp16, two warps a chunk, the other two the next.
        // A quarter of a warp turns 64 channels of two tokens a step: four lanes a token, 16 channels each. The tokens of a pair differ by 5 in the low three bits of their number, so that neither the
        // reads (16-byte pieces of swizzled rows) nor the writes (two pieces a lane) of a quarter meet in a bank. A warp has half of the channels where there are blocks of 64 to share, else half of the tokens.
        constexpr int GROUPS = HD / 64, EACH = GROUPS > 1 ? GROUPS / 2 : 1, EIGHTS = GROUPS > 1 ? 1 : 2, STEPS = VT / 8 / EIGHTS;
        const int side = (warp - CONVERT) & 1, low = lane >> 3, pair_token = (lane & 4) ? low ^ 5 : low, quarter = lane & 3, eight0 = GROUPS > 1 ? 0 : side, vlog = 31 - __clz(vbox);
        const int write_lo = ((2 * quarter) ^ pair_token) * 16;
        int n = 0;
        for (int i = item0; i < item1 && ok; ++i) {
            int tile, last_tile, from, to;
            { const SplPagedItem it = a.items[i]; tile = it.tile_begin; last_tile = it.tile_end; from = seen_first(it); to = seen_last(it); }
            for (; tile < last_tile && ok; ++tile) {
                for (int c = 0; c < VPARTS && ok; ++c, ++n) {
                    if ((n & 1) != (warp - CONVERT) >> 1) continue;
                    const int st = n % NV, sw = n % NW;
                    if (!wait(&full_v[st], n / NV, 71) || !wait(&empty_w[sw], n / NW + 1, 72)) break;
                    const int base = tile * 128 + c * VT;
                    const bool whole = base >= from && base + VT <= to;
#pragma unroll 1
                    for (int e = 0; e < EACH; ++e) {
                        const int group = GROUPS > 1 ? side * EACH + e : 0;
                        const unsigned char *src = v_ring + st * VCHUNK + (HD == 64 ? pair_token * 64 + quarter * 16 : (group >> 1) * vbox * 128 + pair_token * 128 + (((group & 1) * 4 + quarter) ^ pair_token) * 16);
                        unsigned char *dst = w_ring + sw * WCHUNK + group * (VT * 128) + pair_token * 128;
#pragma unroll
                        for (int z0 = 0; z0 < STEPS; z0 += 4) {
                            uint4 codes[4];
#pragma unroll
                            for (int z = 0; z < 4; ++z) {
                                const int token = (eight0 + (z0 + z) * EIGHTS) * 8;
                                codes[z] = *reinterpret_cast<const uint4 *>(src + (token >> vlog) * (vbox * HD) + (token & (vbox - 1)) * ROW);
                                if (!whole && (base + token + pair_token < from || base + token + pair_token >= to)) codes[z] = make_uint4(0u, 0u, 0u, 0u);
                            }
#pragma unroll
                            for (int z = 0; z < 4; ++z) {
                                const uint32_t w[4] = {codes[z].x, codes[z].y, codes[z].z, codes[z].w};
                                uint32_t h[8];
#pragma unroll
                                for (int d = 0; d < 4; ++d) { h[2 * d] = spl_halves_of_e4m3(uint16_t(w[d])); h[2 * d + 1] = spl_halves_of_e4m3(uint16_t(w[d] >> 16)); }
                                unsigned char *row = dst + (eight0 + (z0 + z) * EIGHTS) * 1024;
                                *reinterpret_cast<uint4 *>(row + write_lo) = make_uint4(h[0], h[1], h[2], h[3]);
                                *reinterpret_cast<uint4 *>(row + (write_lo ^ 16)) = make_uint4(h[4], h[5], h[6], h[7]);
                            }
                        }
                    }
                    spl_fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) { spl_mbar_arrive(&full_w[sw]); spl_mbar_arrive(&empty_v[st]); }
                }
            }
        }
    } else {
        // ---- softmax: a warp has 32 rows, and the tokens [32 part, 32 part + 32) of a tile; a lane the rows lane / 4 + 8 i of these, i = 0 ... 3, and eight tokens of each: a token's three numbers then come from
        // shared memory once for four rows. (With a row a lane they came for each: 1,500 of a tile's 6,600 cycles of shared memory's pipe.) What is kept of a row alone (reference, maximum) is lane 4 (row % 8) + row / 8's.
        const int quarter = warp & 3, part = warp >> 2, r = quarter * 32 + lane, own = quarter * 32 + (lane >> 2) + 8 * (lane & 3), of_row = (lane & 7) * 4 + (lane >> 3);
        const uint32_t lanes = uint32_t(quarter * 32) << 16;
        const uint32_t per_group = (65536u + s.group - 1) / s.group;      // x / group = x * per_group >> 16 for x below 192
        int tiles = 0;
        // A piece's queries into the operand tile's two parts: HD / 8 lanes a row, 8 channels each, four pieces on their way a thread. A row's factor turns its scores into log2 of weights; a row that holds
        // what is no finite number has none.
        auto bring_q = [&](const SplPagedItem &it, int parity) {
            const int row0 = it.row0 + it.q0 / s.group, head0 = it.q0 % s.group, pieces = it.q_count * (HD / 8);
#pragma unroll 1
            for (int base = 0; base < pieces; base += 4 * 512) {
                uint4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int idx = base + u * 512 + tid, x = head0 + idx / (HD / 8), row = int(x * per_group >> 16);
                    v[u] = make_uint4(0u, 0u, 0u, 0u);
                    if (idx < pieces) v[u] = *reinterpret_cast<const uint4 *>(a.q + (size_t(row0 + row) * s.heads + it.kv_head * s.group + (x - row * s.group)) * HD + idx % (HD / 8) * 8);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (base + u * 512 >= pieces) break;
                    const int idx = base + u * 512 + tid, piece = idx % (HD / 8), qr = idx / (HD / 8);
                    const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
                    uint32_t most = 0u;
#pragma unroll
                    for (int e = 0; e < 4; ++e) most = max(most, max(w[e] & 0x7fffu, w[e] >> 16 & 0x7fffu));
#pragma unroll
                    for (int o = HD / 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                    // The power of two that takes the largest channel to [128, 256) (exponents as bf16 has them, plus 127).
                    const int up = min(261 - int(most >> 7), 253);
                    const float f = __uint_as_float(uint32_t(up) << 23);
                    uint16_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 x = spl_unpack16<true>(w[e]), y = make_float2(x.x * f, x.y * f);
                        hi[e] = spl_pack_e4m3(y.x, y.y);
                        const uint32_t back = spl_halves_of_e4m3(hi[e]);
                        const float2 z = __half22float2(*reinterpret_cast<const __half2 *>(&back));
                        lo[e] = spl_pack_e4m3(y.x - z.x, y.y - z.y);
                    }
                    if (idx < pieces) {
                        const int place = HD == 64 ? qr * 64 + (((piece >> 1) ^ (qr >> 1 & 3)) * 16) + (piece & 1) * 8 : (piece >> 4) * 16384 + qr * 128 + (((piece >> 1 & 7) ^ (qr & 7)) * 16) + (piece & 1) * 8;
                        *reinterpret_cast<uint2 *>(q_tile + place) = make_uint2(hi[0] | uint32_t(hi[1]) << 16, hi[2] | uint32_t(hi[3]) << 16);
                        *reinterpret_cast<uint2 *>(q_tile + QPART + place) = make_uint2(lo[0] | uint32_t(lo[1]) << 16, lo[2] | uint32_t(lo[3]) << 16);
                        if (piece == 0) factor[parity * 128 + qr] = most >= 0x7f80u ? __int_as_float(0x7fffffff) : s.scale * 1.4426950408889634f * __uint_as_float(uint32_t(254 - up) << 23);
                    }
                }
            }
            spl_fence_proxy_async();
            spl_tc_fence_before();
            __syncwarp();
            if (lane == 0) spl_mbar_arrive(q_full);
        };
        if (item0 < item1) bring_q(first_item, 0);
        for (int i = item0; i < item1; ++i) {
            // (What the tiles do not need of the item is looked up again behind them: the registers are the softmax's.)
            bool busy;                                               // whether this warp's rows hold a query
            int seen_by_all, unseen_by_some, tile, tile_begin, tile_end;
            auto place_of = [&](const SplPagedItem &it, int row) { return it.base + it.q0 / s.group + int((it.q0 % s.group + min(row, it.q_count - 1)) * per_group >> 16); };
            {
                const SplPagedItem it = a.items[i];
                busy = quarter * 32 < it.q_count; seen_by_all = spl_paged_first(s, place_of(it, quarter * 32 + 31)); unseen_by_some = spl_paged_last(s, place_of(it, quarter * 32), it.length);
                tile = tile_begin = it.tile_begin; tile_end = it.tile_end;
            }
            float ref = -INFINITY, c[4], offset[4];
            float2 sum[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) { c[n] = 0.0f; offset[n] = SPL_PAGED8_UNSEEN; sum[n] = make_float2(0.0f, 0.0f); }
            for (; tile < tile_end; ++tile, ++tiles) {
                const int buf = tiles & 1;
                meet(&scaled[tiles % NS], tiles / NS, 73);
                meet(&s_full[buf], tiles >> 1, 66);
                if (busy) {
                    if (tile == tile_begin) {                        // (all of the queries were there before the scores)
#pragma unroll
                        for (int n = 0; n < 4; ++n) c[n] = factor[((i - item0) & 1) * 128 + quarter * 32 + (lane >> 2) + 8 * n];
                    }
                    spl_tc_fence_after();
                    const uint32_t at = tmem + lanes + buf * 128;
                    const float2 *k2 = reinterpret_cast<const float2 *>(scale_ring + (tiles % NS) * 3 * 128 + part * 32) + (lane & 3), *l2 = k2 + 64, *i2 = k2 + 128;
                    uint32_t x[32];                                  // [half of the rows][eight tokens][row of two, token of two]
                    spl_tc_ld_rows(x, at + part * 32);
                    spl_tc_ld_rows(x + 16, at + (16u << 16) + part * 32);
                    spl_tc_ld_done(x);
                    // y = score c ks + log2 vs. (In this order: score c is the row's own size times codes, while score ks could pass fp32's range where y does not.)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 k = k2[4 * j], l = l2[4 * j];
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            uint32_t *z = x + n / 2 * 16 + 4 * j + n % 2 * 2;
                            const float2 y = spl_fma2(spl_mul2(make_float2(__uint_as_float(z[0]), __uint_as_float(z[1])), make_float2(c[n], c[n])), k, l);
                            z[0] = __float_as_uint(y.x); z[1] = __float_as_uint(y.y);
                        }
                    }
                    const int t0 = tile * 128 + part * 32;
                    if (t0 < seen_by_all || t0 + 32 > unseen_by_some) {
                        const SplPagedItem &it = a.items[i];
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const int position = place_of(it, quarter * 32 + (lane >> 2) + 8 * n), first = spl_paged_first(s, position), last = spl_paged_last(s, position, it.length);
#pragma unroll
                            for (int j = 0; j < 4; ++j)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int token = t0 + 8 * j + 2 * (lane & 3) + e;
                                    if (token < first || token >= last) x[n / 2 * 16 + 4 * j + n % 2 * 2 + e] = 0xff800000u;
                                }
                        }
                    }
                    float most[4];
                    bool over = false;
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const uint32_t *z = x + n / 2 * 16 + n % 2 * 2;
                        most[n] = fmaxf(__uint_as_float(z[0]), __uint_as_float(z[1]));
#pragma unroll
                        for (int j = 1; j < 4; ++j) most[n] = fmaxf(most[n], fmaxf(__uint_as_float(z[4 * j]), __uint_as_float(z[4 * j + 1])));
                        over |= most[n] + offset[n] > SPL_PAGED8_MOST;
                    }
                    if (spl_paged8_barrier_or(quarter, over)) {
                        // Some rows' references rise to their maxima: over the four lanes that share a row, then over the four warps.
                        float *others = xmax + buf * 4 * 128 + own;
                        others[part * 128] = spl_paged8_reduce(most, lane, [](float u, float v) { return fmaxf(u, v); });
                        spl_paged8_barrier(quarter);
                        const float m = fmaxf(fmaxf(others[0], others[128]), fmaxf(others[256], others[384]));
                        const bool raise = m > ref + (SPL_PAGED8_MOST - PBIAS);
                        const float old = raise ? exp2f(ref - m) : 1.0f;
                        if (tile > tile_begin) {
                            // The product before has to be done with these sums; the next waits for this warp's probabilities.
                            const float of_mine = __shfl_sync(0xffffffffu, old, of_row);
                            meet(&o_done[(tiles - 1) & 1], (tiles - 1) >> 1, 67);
                            spl_tc_fence_after();
#pragma unroll 1
                            for (int o = 0; o < HD / 4; o += 16) {
                                uint32_t y[16];
                                spl_tc_ld16(y, tmem_o + lanes + part * (HD / 4) + o);
#pragma unroll
                                for (int j = 0; j < 16; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * of_mine);
                                spl_tc_st16(tmem_o + lanes + part * (HD / 4) + o, y);
                            }
                        }
                        if (raise) ref = m;
                        const float now = ref == -INFINITY ? SPL_PAGED8_UNSEEN : PBIAS - ref;
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const float f = __shfl_sync(0xffffffffu, old, (lane & 28) + n);
                            sum[n] = spl_mul2(sum[n], make_float2(f, f));
                            offset[n] = __shfl_sync(0xffffffffu, now, (lane & 28) + n);
                        }
                    }
                    uint32_t p[16];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 inv = i2[4 * j];
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const uint32_t *z = x + n / 2 * 16 + 4 * j + n % 2 * 2;
                            const float2 y = spl_add2(make_float2(__uint_as_float(z[0]), __uint_as_float(z[1])), make_float2(offset[n], offset[n]));
                            const float2 e = n == 3 ? spl_paged_exp2(y) : make_float2(spl_ex2(y.x), spl_ex2(y.y));      // (a quarter of the exponentials on the fp32 pipe)
                            sum[n] = spl_fma2(e, inv, sum[n]);
                            p[n / 2 * 8 + 2 * j + n % 2] = spl_pack16<false>(e.x, e.y);
                        }
                    }
                    spl_tc_st_rows(at + part * 16, p);
                    spl_tc_st_rows(at + (16u << 16) + part * 16, p + 8);
                    spl_tc_st_wait();
                    spl_tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) spl_mbar_arrive(&p_full[buf]);
            }
            // The next piece's queries: all scores of this one have been seen, so its own are no longer read. (O is overwritten by a product that waits for this warp.)
            if (i + 1 < item1) bring_q(a.items[i + 1], (i + 1 - item0) & 1);
            // The piece's sums.
            meet(&o_done[(tiles - 1) & 1], (tiles - 1) >> 1, 68);
            const SplPagedItem it = a.items[i];
            const int row0 = it.row0 + it.q0 / s.group, mine = it.q0 % s.group + min(r, it.q_count - 1), row = int(mine * per_group >> 16), head = it.kv_head * s.group + mine - row * s.group;
            const size_t slot_row = size_t(it.slot) * a.slot_rows + r;
            if (busy) {
                spl_tc_fence_after();
                // (Exchanged where the maxima of the tile before the last were: nobody reads those any more.)
                float *others = xmax + (tiles & 1) * 4 * 128;
                const float sums[4] = {sum[0].x + sum[0].y, sum[1].x + sum[1].y, sum[2].x + sum[2].y, sum[3].x + sum[3].y};
                others[part * 128 + own] = spl_paged8_reduce(sums, lane, [](float u, float v) { return u + v; });
                spl_paged8_barrier(quarter);
                const float all = (others[r] + others[128 + r]) + (others[256 + r] + others[384 + r]), ref_of_mine = __shfl_sync(0xffffffffu, ref, of_row);
                const bool here = r < it.q_count;
                const size_t place = (size_t(row0 + row) * s.heads + head) * HD + part * (HD / 4);
                const float inv = it.slot < 0 ? 1.0f / all : 1.0f;
#pragma unroll 1
                for (int o = 0; o < HD / 4; o += 16) {
                    uint32_t y[16];
                    spl_tc_ld16(y, tmem_o + lanes + part * (HD / 4) + o);
#pragma unroll
                    for (int j = 0; j < 16; ++j) y[j] = __float_as_uint(__uint_as_float(y[j]) * inv);
                    if (!here) {
                    } else if (it.slot >= 0 || a.out_f32) {
                        float *dst = it.slot >= 0 ? a.partial + slot_row * HD + part * (HD / 4) + o : static_cast<float *>(a.out) + place + o;
#pragma unroll
                        for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4 *>(dst + 4 * j) = make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
                    } else {
                        uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + place + o);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int u = 0; u < 4; ++u) w[u] = spl_pack16<true>(__uint_as_float(y[8 * j + 2 * u]), __uint_as_float(y[8 * j + 2 * u + 1]));
                            dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                    __syncwarp();
                }
                if (here && it.slot >= 0 && part == 0) a.partial_ml[slot_row] = make_float2(ref_of_mine, all);
                spl_tc_fence_before();
                spl_paged8_barrier(quarter);              // the sums in shared memory are read before the next piece's
            }
            if (it.merge >= 0) {
                // Whichever block is the last to leave a piece of these rows joins them, in the order of the pieces whoever it is; eight warps do.
                __threadfence();
                spl_named_barrier<6, 32 * SPL_PAGED8_SOFTMAX>();
                if (tid == 0) {
                    const bool all = atomicAdd(&a.arrived[it.merge], 1) == it.pieces - 1;
                    if (all) a.arrived[it.merge] = 0;          // for the next launch
                    *joins = all;
                }
                spl_named_barrier<6, 32 * SPL_PAGED8_SOFTMAX>();
                if (*joins) {
                    __threadfence();
                    if (warp < 8) spl_paged_join<HD, true>(s, a, it, row0, it.q0 % s.group, per_group, xmax + (tiles & 1) * 4 * 128);
                    spl_named_barrier<6, 32 * SPL_PAGED8_SOFTMAX>();      // before the next piece's maxima
                }
            }
        }
    }
    spl_tc_fence_before();
    __syncthreads();
    spl_tc_fence_after();
    if (warp == SCORES) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}

// ---- few rows: the products transposed --------------------------------------------------------------
// A piece of at most 48 packed rows (single tokens, verify blocks) would leave most of the rows above empty, and has no rows to spread a tile's conversion over. Here the cache is the A operand of both products, as it
// lies there, and the rows are columns:
//   S^T[128 tokens x 2 N]       = K [hi; lo]^T            A = K (tokens by channels), B = the N queries' two parts, so that K is read once; a score is the sum of two columns
//   O^T[128 channels x 3 N]    += V^T [P1; P2; P3]        A = V (a block of 128 channels), B = P in three parts: units of sixteen columns of one part, sixteen bytes a token, token after token
// P is a number in fp16 of at most 2^15, of which e5m2 is the upper byte: P1 is P rounded to that (three significant bits), P2 sixteen times what that leaves, rounded likewise, P3 sixteen times what that leaves. What is left
// has either sign and at most an eighth of the part's size, so three parts hold the eleven bits; with the factors of sixteen also of the subnormals, down to fp16's own 2^-24: P1 + P2 / 16 + P3 / 256 is P, exactly, for all of
// them. The parts' sums are columns of their own and are added at the piece's end. (A unit is the operand's layout without a swizzle, its columns the inner dimension: a thread stores its part of a unit at once. With a row of 128 tokens for each column a
// tile's probabilities were 48 one-byte stores a thread and half of the softmax's time.)
// A softmax thread has a token, and 8 or 16 of the columns (groups of four warps share these out): the token's scales, which came with its keys, are its own registers, a row's maximum, where one is wanted, is a reduction over lanes (redux) and
// four warps, its sum stays in the threads until the piece's end. The last four warps copy keys, issue the scores' and the sums' products, copy values.
// A tile of 128 tokens by 256 channels is 64 KB from memory (some 2,700 cycles at an SM's share); the products take 400 cycles of the tensor cores with 16 rows.
__host__ __device__ constexpr int spl_paged8n_groups(int n) { return n == 48 ? 3 : 2; }
__host__ __device__ constexpr int spl_paged8n_threads(int n) { return 128 * spl_paged8n_groups(n) + 128; }
// Chunks of 128 tokens by 128 channels, of keys and of values.
__host__ __device__ constexpr int spl_paged8n_ring_k(int n) { return n == 16 ? 6 : 5; }
__host__ __device__ constexpr int spl_paged8n_ring_v(int n) { return n == 16 ? 6 : n == 32 ? 5 : 4; }
// Tiles of scales. Those of tile j come with its first keys, which waited for the scores of tile j - ring / blocks or a later one, and these for the softmax of the tile two before.
__host__ __device__ constexpr int spl_paged8n_scales(int hd, int n) { return (spl_paged8n_ring_k(n) * 128 + hd - 1) / hd + 2; }
__host__ __device__ constexpr size_t spl_paged8n_smem_bytes(int hd, int n) {
    return size_t(spl_paged8n_ring_k(n) + spl_paged8n_ring_v(n)) * 16384 + size_t(2) * n * hd /* Q */ + size_t(2) * 3 * n * 128 /* P */ + size_t(spl_paged8n_scales(hd, n)) * 1024 + size_t(2 + 8) * n * 4 /* factors, maxima */ + 512 /* barriers */;
}
__device__ __forceinline__ void spl_tc_ld8_later(uint32_t *r, uint32_t taddr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
}
__device__ __forceinline__ void spl_tc_st8_later(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
template <int COUNT> __device__ __forceinline__ void spl_tc_ld_done_of(uint32_t *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < COUNT; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ uint16_t spl_e5m2_of_halves(uint32_t v) {
    uint16_t d;
    asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;\n" : "=h"(d) : "r"(v));
    return d;
}
// Two halves rounded to their upper bytes (a carry raises the exponent, as it should). What is no number becomes -0: what it leaves is none, and so the last part.
__device__ __forceinline__ uint32_t spl_halves_to_e5m2(uint32_t v) { return (v + 0x00800080u) & 0xff00ff00u; }
// Sixteen times what they leave.
__device__ __forceinline__ uint32_t spl_half2_left16(uint32_t a, uint32_t b) {
    const __half2 d = __hmul2(__hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b)), __float2half2_rn(16.0f));
    return *reinterpret_cast<const uint32_t *>(&d);
}

// Columns inner, without a swizzle: sixteen columns (bytes) of a token, eight tokens 128 bytes, the next eight behind them; the next sixteen columns 2,048 bytes on.
__device__ __forceinline__ uint64_t spl_paged8n_p_desc(uint32_t addr) {
    return uint64_t((addr & 0x3FFFFu) >> 4) | uint64_t(128 >> 4) << 16 | uint64_t(2048 >> 4) << 32 | uint64_t(1) << 46;
}

template <int HD, int N>
__global__ void __launch_bounds__(spl_paged8n_threads(N), 1)
spl_paged_attend_e4m3_narrow_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, SplPagedTables t, SplPagedShape s, SplPagedAttend a, SplPagedScaled scales) {
    constexpr int NK = spl_paged8n_ring_k(N), NV = spl_paged8n_ring_v(N), NS = spl_paged8n_scales(HD, N), BLOCKS = HD / 128, GROUPS = spl_paged8n_groups(N), H = N / GROUPS, CHUNK = 16384, PBYTES = 3 * N * 128;      // H: a softmax thread's columns
    constexpr int SOFTMAX = 4 * GROUPS, COPY_K = SOFTMAX, SCORES = COPY_K + 1, SUMS = COPY_K + 2, COPY_V = COPY_K + 3;
    constexpr float PBIAS = 7.0f;
    extern __shared__ __align__(1024) unsigned char spl_paged8n_raw[];
    if (spl_smem_addr(spl_paged8n_raw) % 1024) { if (threadIdx.x == 0) a.error_flag[0] = 299; return; }
    unsigned char *ring = spl_paged8n_raw, *v_ring = ring + NK * CHUNK, *q_tile = v_ring + NV * CHUNK, *p_tile = q_tile + 2 * N * HD;
    float *scale_ring = reinterpret_cast<float *>(p_tile + 2 * PBYTES), *factor = scale_ring + NS * 256, *xmax = factor + 2 * N;      // [tile % NS][keys', values'][token]; [item parity][column]; [tile parity][quarter of the tokens][column]
    uint64_t *bars = reinterpret_cast<uint64_t *>(xmax + 8 * N);
    uint64_t *full_k = bars, *empty_k = full_k + NK, *full_v = empty_k + NK, *empty_v = full_v + NV, *scaled = empty_v + NV, *s_full = scaled + NS, *p_full = s_full + 2, *o_done = p_full + 2, *q_full = o_done + 2, *drained = q_full + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drained + 2);
    volatile int *abort = reinterpret_cast<volatile int *>(tmem_slot + 1), *joins = abort + 1;
    auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < 2 * NK + 2 * NV + NS; ++i) spl_mbar_init(&bars[i], 1);
        for (int i = 0; i < 2; ++i) { spl_mbar_init(&s_full[i], 1); spl_mbar_init(&p_full[i], SOFTMAX); spl_mbar_init(&o_done[i], 1); }
        spl_mbar_init(q_full, SOFTMAX); spl_mbar_init(&drained[0], 1); spl_mbar_init(&drained[1], 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (tid == 32 * COPY_K) { spl_tma_prefetch(&k_map); spl_tma_prefetch(&v_map); }
    if (warp == SCORES) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(spl_smem_addr(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    spl_tc_fence_before();
    __syncthreads();
    spl_tc_fence_after();
    const uint32_t tmem = uint32_t(uniform(int(*tmem_slot))), tmem_o = tmem + 4 * N;      // two buffers of scores, then BLOCKS times 3 N columns of sums
    // What the batch's copies brought is read before the kernel in front is done, and the first tiles are asked for, as in spl_paged_attend_kernel.
    union { SplPagedItem item; int4 four[sizeof(SplPagedItem) / 16]; } first;
#pragma unroll
    for (int i = 0; i < int(sizeof(SplPagedItem) / 16); ++i) first.four[i] = __ldcg(reinterpret_cast<const int4 *>(a.starts + blockIdx.x) + i);
    const SplPagedItem first_item = first.item;
    const int item0 = uniform(__ldcg(a.block_begin + blockIdx.x)), item1 = uniform(__ldcg(a.block_begin + blockIdx.x + 1));
    // A tile's boxes of tokens: a page, or half a page of 256; lane b holds the b-th box's page. A chunk is the boxes of a block of 128 channels.
    const int box = min(s.page_tokens, 128), boxes = 128 / box;
    auto page_of = [&](const SplPagedItem &it, int tile) {
        return tile < it.tile_end && lane < min(boxes, (it.length - tile * 128 + box - 1) / box) ? __ldcg(t.table + size_t(it.sequence) * s.max_pages + (s.page_tokens > 128 ? tile >> 1 : tile * boxes + lane)) : 0;
    };
    auto inside_page = [&](int tile) { return s.page_tokens > 128 ? (tile & 1) * 128 : 0; };
    auto present = [&](const SplPagedItem &it, int tile) { return (min(128, it.length - tile * 128) + box - 1) / box; };
    const bool copies = warp == COPY_K || warp == COPY_V, keys = warp == COPY_K;
    const CUtensorMap *map = keys ? &k_map : &v_map;
    const int first_page = copies && item0 < item1 ? page_of(first_item, first_item.tile_begin) : 0;
    if (copies && item0 < item1) {
        int page = first_page;
        for (int tile = first_item.tile_begin; tile < min(first_item.tile_end, first_item.tile_begin + SPL_PAGED_EARLY); ++tile) {
            const int ahead = page_of(first_item, tile + 1);
            for (int c = 0; c < BLOCKS; ++c) if (lane < present(first_item, tile)) spl_tma_prefetch5(map, 0, inside_page(tile), c, first_item.kv_head, page);
            page = ahead;
        }
    }
    spl_grid_begin();
    int ok = 1;
    auto gave_up = [&](int code) { ok = 0; if (!*abort && lane == 0) { spl_note_wait(a.error_flag, code, 0); a.error_flag[0] = 200 + warp; } *abort = 1; };
    auto wait = [&](uint64_t *bar, int phase, int code) { if (ok && !spl_mbar_wait_warp(bar, phase & 1, const_cast<const int *>(abort))) gave_up(code); return ok != 0; };
    // The softmax's waits: the empty statement keeps the compiler from making a second loop for the case that a wait has run out. With the loop twice as large its instructions came too late: 2,048 rows over
    // 8,192 tokens of 32/8 heads of 128 took 671 us instead of 390. (The products' loops are faster without it.)
    auto meet = [&](uint64_t *bar, int phase, int code) { wait(bar, phase, code); asm volatile("" : "+r"(ok)); };
    // Tokens that some row of a piece sees.
    auto seen_first = [&](const SplPagedItem &it) { return spl_paged_first(s, it.base + it.q0 / s.group); };
    auto seen_last = [&](const SplPagedItem &it) { return spl_paged_last(s, it.base + (it.q0 + it.q_count - 1) / s.group, it.length); };

    if (copies) {
        uint64_t *full = keys ? full_k : full_v, *empty = keys ? empty_k : empty_v;
        unsigned char *to = keys ? ring : v_ring;
        const int slots = keys ? NK : NV;
        int n = 0, st = 0, tiles = 0;
        SplPagedItem it = first_item;
        int page = first_page;
        for (int i = item0; i < item1 && ok; ++i) {
            if (i > item0) { it = a.items[i]; page = page_of(it, it.tile_begin); }
            for (int tile = it.tile_begin; tile < it.tile_end && ok; ++tile, ++tiles) {
                const int ahead = page_of(it, tile + 1), inside = inside_page(tile), there = present(it, tile);
                for (int c = 0; c < BLOCKS && wait(&empty[st], n / slots + 1, 60); ++c) {
                    if (keys && c == 0) {
                        // The tile's scales, as many as there are pages for.
                        const int sl = tiles % NS;
                        if (lane == 0) spl_mbar_expect_tx(&scaled[sl], uint32_t(there) * box * 8);
                        __syncwarp();
                        if (lane < there) {
                            const size_t at = (size_t(page) * s.kv_heads + it.kv_head) * s.page_tokens + inside;
                            spl_bulk_g2s(scale_ring + sl * 256 + lane * box, scales.k + at, box * 4, &scaled[sl]);
                            spl_bulk_g2s(scale_ring + sl * 256 + 128 + lane * box, scales.v + at, box * 4, &scaled[sl]);
                        }
                    }
                    if (lane == 0) spl_mbar_expect_tx(&full[st], uint32_t(there) * box * 128);
                    __syncwarp();
                    if (lane < there) spl_tma_load5(to + st * CHUNK + lane * box * 128, map, 0, inside, c, it.kv_head, page, &full[st]);
                    ++n; st = st + 1 == slots ? 0 : st + 1;
                }
                page = ahead;
            }
        }
        // Nothing may still be on its way into the block's shared memory when it is handed on.
        for (int z = 0; z < slots && z < n; ++z) spl_mbar_wait(&full[z], ((z + (n - 1 - z) / slots * slots) / slots) & 1);
        const int copied = (n + BLOCKS - 1) / BLOCKS;
        if (keys) for (int z = 0; z < NS && z < copied; ++z) spl_mbar_wait(&scaled[z], ((z + (copied - 1 - z) / NS * NS) / NS) & 1);
    } else if (warp == SCORES || warp == SUMS) {
        const uint32_t elected = spl_elect_one() ? 1u : 0u;
        const bool scores = warp == SCORES;
        // Scores: e4m3 by e4m3, both K-major. Sums: A = V, e4m3 with its channels (M) in rows of the tokens, B = P, e5m2 (format 1), its columns (N) in the tokens' sixteen bytes.
        constexpr uint32_t s_idesc = spl_tc_idesc(2 * N), o_idesc = spl_tc_idesc(3 * N) | 1u << 10 | 1u << 15 | 1u << 16;
        const uint64_t k_desc = spl_tc_desc_sw128(spl_smem_addr(ring)), q_desc = spl_tc_desc_sw128(spl_smem_addr(q_tile)), v_desc = spl_tc_desc_mn_sw128(spl_smem_addr(v_ring), CHUNK),
                       p_desc = spl_paged8n_p_desc(spl_smem_addr(p_tile));
        int n = 0, tiles = 0;
        for (int i = item0; i < item1 && ok; ++i) {
            const SplPagedItem it = a.items[i];
            const int tile_begin = uniform(it.tile_begin), count = uniform(it.tile_end) - tile_begin;
            if (scores) {
                if (!wait(q_full, i - item0, 63)) break;
                for (int tile = 0; tile < count && ok; ++tile) {
                    const int at = tiles + tile;
                    if (!wait(&full_k[n % NK], n / NK, 62)) break;
                    if (at >= 2 && !wait(&o_done[at & 1], (at - 2) >> 1, 61)) break;      // tile at - 2's scores have been read, and its P: whoever sees these scores may write over that
#pragma unroll
                    for (int c = 0; c < BLOCKS; ++c, ++n) {
                        const int st = n % NK;
                        if (c > 0 && !wait(&full_k[st], n / NK, 62)) break;
                        spl_tc_fence_after();
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            spl_tc_mma8_ss_if(elected, tmem + (at & 1) * 2 * N, k_desc + uint64_t((st * CHUNK + ks * 32) >> 4), q_desc + uint64_t((c * 2 * N * 128 + ks * 32) >> 4), s_idesc, c + ks > 0 ? 1u : 0u);
                        spl_tc_commit_if(elected, &empty_k[st]);
                        if (c == BLOCKS - 1) spl_tc_commit_if(elected, &s_full[at & 1]);
                    }
                }
            } else {
                const int from_all = uniform(seen_first(it)), to_all = uniform(seen_last(it));
                for (int tile = 0; tile < count && ok; ++tile) {
                    const int at = tiles + tile, token0 = (tile_begin + tile) * 128, from = max(0, from_all - token0), to = min(128, to_all - token0), k0 = from / 32, k1 = (to + 31) / 32;
                    for (int c = 0; c < BLOCKS && ok; ++c, ++n) {
                        const int st = n % NV;
                        if (!wait(&full_v[st], n / NV, 65)) break;
                        if (from % 32 || to % 32) {
                            // Values of unseen tokens in the first and last groups of 32: zero, whatever the cache holds there (0 x NaN is no number).
                            const int before = from % 32, after = (32 - to % 32) % 32;
                            for (int z = lane; z < (before + after) * 8; z += 32) {
                                const int row = z / 8, token = row < before ? k0 * 32 + row : to + row - before;
                                *reinterpret_cast<uint4 *>(v_ring + st * CHUNK + token * 128 + z % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
                            }
                            spl_fence_proxy_async();
                            __syncwarp();
                        }
                        if (c == 0 && !wait(&p_full[at & 1], at >> 1, 64)) break;
                        spl_tc_fence_after();
                        for (int ks = k0; ks < k1; ++ks)      // (the piece's first product overwrites what the sums held)
                            spl_tc_mma8_ss_if(elected, tmem_o + c * 3 * N, v_desc + uint64_t((st * CHUNK + ks * 4096) >> 4), p_desc + uint64_t(((at & 1) * PBYTES + ks * 512) >> 4), o_idesc, tile > 0 || ks > k0 ? 1u : 0u);
                        spl_tc_commit_if(elected, &empty_v[st]);
                        if (c == BLOCKS - 1) spl_tc_commit_if(elected, &o_done[at & 1]);
                    }
                }
            }
            tiles += count;
        }
        // No product may still read shared or write tensor memory when they are handed on.
        spl_tc_commit_if(elected, &drained[scores ? 0 : 1]);
        spl_mbar_wait(&drained[scores ? 0 : 1], 0);
    } else {
        // ---- softmax: token `mine` of a tile, the columns [n0, n0 + H).
        const int quarter = warp & 3, group = warp >> 2, mine = quarter * 32 + lane, n0 = group * H;
        const uint32_t lanes = uint32_t(quarter * 32) << 16;
        const uint32_t per_group = (65536u + s.group - 1) / s.group;      // x / group = x * per_group >> 16 for x below 192
        // A piece's queries: rows n of the operand the upper parts, N + n the rest; columns without a query are zeros.
        constexpr int PIECES = N * (HD / 8), EACH = (PIECES + 32 * SOFTMAX - 1) / (32 * SOFTMAX);      // sixteen bytes of queries; a thread's
        auto load_q = [&](const SplPagedItem &it, uint4 (&v)[EACH]) {
            const int row0 = it.row0 + it.q0 / s.group, head0 = it.q0 % s.group;
#pragma unroll
            for (int u = 0; u < EACH; ++u) {
                const int idx = u * 32 * SOFTMAX + tid, x = head0 + idx / (HD / 8), row = int(x * per_group >> 16);
                v[u] = make_uint4(0u, 0u, 0u, 0u);
                if (idx < it.q_count * (HD / 8)) v[u] = *reinterpret_cast<const uint4 *>(a.q + (size_t(row0 + row) * s.heads + it.kv_head * s.group + (x - row * s.group)) * HD + idx % (HD / 8) * 8);
            }
        };
        // (Held in registers over a tile they would be the softmax's: the next piece's come to L1 while the last tile runs.)
        auto ask_q = [&](const SplPagedItem &it) {
            const int row0 = it.row0 + it.q0 / s.group, head0 = it.q0 % s.group;
#pragma unroll
            for (int u = 0; u < EACH; ++u) {
                const int idx = u * 32 * SOFTMAX + tid, x = head0 + idx / (HD / 8), row = int(x * per_group >> 16);
                if (idx % 8 == 0 && idx < it.q_count * (HD / 8)) asm volatile("prefetch.global.L1 [%0];\n" ::"l"(a.q + (size_t(row0 + row) * s.heads + it.kv_head * s.group + (x - row * s.group)) * HD + idx % (HD / 8) * 8));
            }
        };
        auto place_q = [&](const uint4 (&v)[EACH], int q_count, int parity) {
#pragma unroll
            for (int u = 0; u < EACH; ++u) {
                const int idx = u * 32 * SOFTMAX + tid, piece = idx % (HD / 8), n = idx / (HD / 8);
                const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
                uint32_t most = 0u;
#pragma unroll
                for (int e = 0; e < 4; ++e) most = max(most, max(w[e] & 0x7fffu, w[e] >> 16 & 0x7fffu));
#pragma unroll
                for (int o = HD / 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                const int up = min(261 - int(most >> 7), 253);      // (as above)
                const float f = __uint_as_float(uint32_t(up) << 23);
                uint16_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 x = spl_unpack16<true>(w[e]), y = make_float2(x.x * f, x.y * f);
                    hi[e] = spl_pack_e4m3(y.x, y.y);
                    const uint32_t back = spl_halves_of_e4m3(hi[e]);
                    const float2 z = __half22float2(*reinterpret_cast<const __half2 *>(&back));
                    lo[e] = spl_pack_e4m3(y.x - z.x, y.y - z.y);
                }
                if (PIECES % (32 * SOFTMAX) && n >= N) continue;
                const int place = (piece >> 4) * (2 * N * 128) + n * 128 + (((piece >> 1 & 7) ^ (n & 7)) * 16) + (piece & 1) * 8;
                *reinterpret_cast<uint2 *>(q_tile + place) = make_uint2(hi[0] | uint32_t(hi[1]) << 16, hi[2] | uint32_t(hi[3]) << 16);
                *reinterpret_cast<uint2 *>(q_tile + N * 128 + place) = make_uint2(lo[0] | uint32_t(lo[1]) << 16, lo[2] | uint32_t(lo[3]) << 16);
                if (piece == 0) factor[parity * N + n] = n >= q_count ? 0.0f : most >= 0x7f80u ? __int_as_float(0x7fffffff) : s.scale * 1.4426950408889634f * __uint_as_float(uint32_t(254 - up) << 23);
            }
            spl_fence_proxy_async();
            spl_tc_fence_before();
            __syncwarp();
            if (lane == 0) spl_mbar_arrive(q_full);
        };
        if (item0 < item1) {
            uint4 q[EACH];
            load_q(first_item, q);
            place_q(q, first_item.q_count, 0);
        }
        int tiles = 0;
        for (int i = item0; i < item1; ++i) {
            // (What the tiles do not need of the item is looked up again where it is wanted.)
            int seen_by_all, unseen_by_some, tile, tile_begin, tile_end, from, to, row_at, head_at, last_row;
            {
                const SplPagedItem it = a.items[i];
                row_at = it.base + it.q0 / s.group; head_at = it.q0 % s.group; last_row = it.q_count - 1;
                seen_by_all = spl_paged_first(s, row_at + int(uint32_t(head_at + last_row) * per_group >> 16)); unseen_by_some = spl_paged_last(s, row_at, it.length);
                tile = tile_begin = it.tile_begin; tile_end = it.tile_end; from = seen_first(it); to = seen_last(it);
            }
            float ref = -INFINITY;                                   // of column n0 + lane
            float2 c[H / 2], offset[H / 2], sum[H / 2];              // of two columns
#pragma unroll
            for (int n = 0; n < H / 2; ++n) { c[n] = sum[n] = make_float2(0.0f, 0.0f); offset[n] = make_float2(SPL_PAGED8_UNSEEN, SPL_PAGED8_UNSEEN); }
            for (; tile < tile_end; ++tile, ++tiles) {
                const int buf = tiles & 1;
                if (tile + 1 == tile_end && i + 1 < item1) ask_q(a.items[i + 1]);
                meet(&scaled[tiles % NS], tiles / NS, 70);
                const float *mine_of = scale_ring + tiles % NS * 256 + mine;
                const bool there = tile * 128 + mine >= from && tile * 128 + mine < to;      // (what no row sees is masked)
                const float given = mine_of[128], v = given >= 0.0f && given <= SPL_PAGED8_SCALE_MOST ? fmaxf(given, SPL_PAGED8_SCALE_LEAST) : __int_as_float(0x7fffffff);
                const float k = there ? mine_of[0] : 0.0f, l = there ? spl_lg2(v) : 0.0f, inv = there ? spl_rcp(v) : 0.0f;
                meet(&s_full[buf], tiles >> 1, 66);
                if (tile == tile_begin) {                            // (all of the queries were there before the scores)
#pragma unroll
                    for (int n = 0; n < H / 2; ++n) c[n] = *reinterpret_cast<const float2 *>(factor + ((i - item0) & 1) * N + n0 + 2 * n);
                }
                spl_tc_fence_after();
                uint32_t x[2 * H];
                const uint32_t at = tmem + lanes + buf * 2 * N + n0;
#pragma unroll
                for (int n = 0; n < H; n += 8) { spl_tc_ld8_later(x + n, at + n); spl_tc_ld8_later(x + H + n, at + N + n); }
                spl_tc_ld_done_of<2 * H>(x);
                // y = score c ks + log2 vs (in this order, as above).
                auto two = [](const uint32_t *v) { return make_float2(__uint_as_float(v[0]), __uint_as_float(v[1])); };
                float2 y[H / 2];
#pragma unroll
                for (int n = 0; n < H / 2; ++n) y[n] = spl_fma2(spl_mul2(spl_add2(two(x + 2 * n), two(x + H + 2 * n)), c[n]), make_float2(k, k), make_float2(l, l));
                if (tile * 128 < seen_by_all || tile * 128 + 128 > unseen_by_some) {
                    const int token = tile * 128 + mine, length = a.items[i].length;
                    auto hidden = [&](int n) {
                        const int position = row_at + int(uint32_t(head_at + min(n0 + n, last_row)) * per_group >> 16);
                        return token < spl_paged_first(s, position) || token >= spl_paged_last(s, position, length);
                    };
#pragma unroll
                    for (int n = 0; n < H / 2; ++n) { if (hidden(2 * n)) y[n].x = -INFINITY; if (hidden(2 * n + 1)) y[n].y = -INFINITY; }
                }
                float most = -INFINITY;
#pragma unroll
                for (int n = 0; n < H / 2; ++n) { const float2 z = spl_add2(y[n], offset[n]); most = fmaxf(most, fmaxf(z.x, z.y)); }
                if (spl_paged8_barrier_or(group, most > SPL_PAGED8_MOST)) {
                    // Some columns' references rise to their maxima: over the warp's tokens, then over the four warps'; lane n has column n0 + n's.
                    float m = -INFINITY;
#pragma unroll
                    for (int n = 0; n < H; ++n) { const float all = spl_redux_max(n % 2 ? y[n / 2].y : y[n / 2].x); if (lane == n) m = all; }
                    float *others = xmax + buf * 4 * N + n0 + lane;
                    if (lane < H) others[quarter * N] = m;
                    spl_paged8_barrier(group);
                    if (lane < H) m = fmaxf(fmaxf(others[0], others[N]), fmaxf(others[2 * N], others[3 * N]));
                    const bool raise = lane < H && m > ref + (SPL_PAGED8_MOST - PBIAS);
                    const float old = raise ? exp2f(ref - m) : 1.0f;
                    if (raise) ref = m;
                    const float shift = ref == -INFINITY ? SPL_PAGED8_UNSEEN : PBIAS - ref;
#pragma unroll
                    for (int n = 0; n < H / 2; ++n) {
                        sum[n] = spl_mul2(sum[n], make_float2(__shfl_sync(0xffffffffu, old, 2 * n), __shfl_sync(0xffffffffu, old, 2 * n + 1)));
                        offset[n] = make_float2(__shfl_sync(0xffffffffu, shift, 2 * n), __shfl_sync(0xffffffffu, shift, 2 * n + 1));
                    }
                    if (tile > tile_begin) {
                        // The product before has to be done with these sums; the next waits for this warp's probabilities.
                        meet(&o_done[(tiles - 1) & 1], (tiles - 1) >> 1, 67);
                        spl_tc_fence_after();
#pragma unroll 1
                        for (int n = 0; n < H; n += 8) {
                            float f[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) f[j] = __shfl_sync(0xffffffffu, old, n + j);
#pragma unroll 1
                            for (int b = 0; b < 3 * BLOCKS; ++b) {
                                uint32_t o[8];
                                spl_tc_ld8_later(o, tmem_o + lanes + b * N + n0 + n);
                                spl_tc_ld_done_of<8>(o);
#pragma unroll
                                for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f[j]);
                                spl_tc_st8_later(tmem_o + lanes + b * N + n0 + n, o);
                            }
                        }
                        spl_tc_st_wait();
                    }
                }
                // (P of tile - 2 has been read: its scores' place was free for these.)
                uint32_t part[3][H / 4];
#pragma unroll
                for (int n = 0; n < H / 4; ++n) {
                    uint32_t p[2], rest[2], low[2];      // the parts, the first two in the upper bytes of halves
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float2 z = spl_add2(y[2 * n + e], offset[2 * n + e]), w = make_float2(spl_ex2(z.x), spl_ex2(z.y));
                        sum[2 * n + e] = spl_fma2(w, make_float2(inv, inv), sum[2 * n + e]);
                        const uint32_t whole = spl_pack16<false>(w.x, w.y);
                        p[e] = spl_halves_to_e5m2(whole);
                        const uint32_t left = spl_half2_left16(whole, p[e]);
                        rest[e] = spl_halves_to_e5m2(left);
                        low[e] = spl_e5m2_of_halves(spl_half2_left16(left, rest[e]));
                    }
                    part[0][n] = __byte_perm(p[0], p[1], 0x7531); part[1][n] = __byte_perm(rest[0], rest[1], 0x7531); part[2][n] = low[0] | low[1] << 16;
                }
                unsigned char *to_p = p_tile + buf * PBYTES + n0 / 16 * 2048 + mine * 16 + n0 % 16;
#pragma unroll
                for (int e = 0; e < 3; ++e) {
                    if constexpr (H == 16) *reinterpret_cast<uint4 *>(to_p + e * (N / 16) * 2048) = make_uint4(part[e][0], part[e][1], part[e][2], part[e][3]);
                    else *reinterpret_cast<uint2 *>(to_p + e * (N / 16) * 2048) = make_uint2(part[e][0], part[e][1]);
                }
                spl_fence_proxy_async();
                spl_tc_fence_before();
                __syncwarp();
                if (lane == 0) spl_mbar_arrive(&p_full[buf]);
            }
            // The next piece's queries: all scores of this one have been seen, so its own are no longer read. (The sums are overwritten by a product that waits for this warp.)
            if (i + 1 < item1) {
                uint4 q[EACH];
                load_q(a.items[i + 1], q);
                place_q(q, a.items[i + 1].q_count, (i + 1 - item0) & 1);
            }
            const SplPagedItem it = a.items[i];
            // The piece's sums.
            meet(&o_done[(tiles - 1) & 1], (tiles - 1) >> 1, 68);
            spl_tc_fence_after();
            // Over the lanes: at each step half of the columns stay, and the other half's sums go to the lane that keeps these; lanes that end up with the same column have the same sum.
            int column = 0;
            float sums[H];
#pragma unroll
            for (int n = 0; n < H / 2; ++n) { sums[2 * n] = sum[n].x; sums[2 * n + 1] = sum[n].y; }
#pragma unroll
            for (int o = 16, left = H; o > 0; o >>= 1) {
                if (left > 1) {
                    left /= 2;
                    const bool up = lane & o;
                    if (up) column += left;
#pragma unroll
                    for (int n = 0; n < left; ++n) { const float keep = up ? sums[left + n] : sums[n], give = up ? sums[n] : sums[left + n]; sums[n] = keep + __shfl_xor_sync(0xffffffffu, give, o); }
                } else sums[0] += __shfl_xor_sync(0xffffffffu, sums[0], o);
            }
            float all = 0.0f, *others = xmax + (tiles & 1) * 4 * N + n0 + lane;      // (where the maxima of the tile before the last were: nobody reads those any more)
            others[quarter * N + column - lane] = sums[0];
            spl_paged8_barrier(group);
            if (lane < H) all = (others[0] + others[N]) + (others[2 * N] + others[3 * N]);
            const float inv = it.slot < 0 ? 1.0f / all : 1.0f;
            const int row0 = it.row0 + it.q0 / s.group, head0 = it.q0 % s.group;
            const size_t slot_row = size_t(it.slot) * a.slot_rows + n0;
#pragma unroll 1
            for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                for (int n = 0; n < H; n += 8) {
                    uint32_t o[24];
#pragma unroll
                    for (int part = 0; part < 3; ++part) spl_tc_ld8_later(o + 8 * part, tmem_o + lanes + (b * 3 + part) * N + n0 + n);
                    spl_tc_ld_done_of<24>(o);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float value = fmaf(__uint_as_float(o[16 + j]), 1.0f / 256.0f, fmaf(__uint_as_float(o[8 + j]), 1.0f / 16.0f, __uint_as_float(o[j]))) * __shfl_sync(0xffffffffu, inv, n + j);
                        const int x = head0 + n0 + n + j, row = int(x * per_group >> 16), channel = b * 128 + mine;
                        if (n0 + n + j >= it.q_count) continue;
                        const size_t place = (size_t(row0 + row) * s.heads + it.kv_head * s.group + x - row * s.group) * HD + channel;
                        if (it.slot >= 0) a.partial[(slot_row + n + j) * HD + channel] = value;
                        else if (a.out_f32) static_cast<float *>(a.out)[place] = value;
                        else static_cast<uint16_t *>(a.out)[place] = spl_float_to_bf16(value);
                    }
                }
            if (it.slot >= 0 && quarter == 0 && lane < H && n0 + lane < it.q_count) a.partial_ml[slot_row + lane] = make_float2(ref, all);
            spl_tc_fence_before();
            spl_paged8_barrier(group);                                               // the sums in shared memory are read before the next piece's
            if (N == 16 && it.merge >= 0) {                // (more rows are joined by rows)
                // Whichever block is the last to leave a piece of these rows joins them, in the order of the pieces whoever it is.
                __threadfence();
                spl_named_barrier<6, 32 * SOFTMAX>();
                if (tid == 0) {
                    const bool last = atomicAdd(&a.arrived[it.merge], 1) == it.pieces - 1;
                    if (last) a.arrived[it.merge] = 0;         // for the next launch
                    *joins = last;
                }
                spl_named_barrier<6, 32 * SOFTMAX>();
                if (*joins) {
                    __threadfence();
                    if (warp < 8) spl_paged_join<HD, true>(s, a, it, row0, head0, per_group, reinterpret_cast<float *>(p_tile));      // (the piece's products have read P)
                    spl_named_barrier<6, 32 * SOFTMAX>();
                }
            }
        }
    }
    spl_tc_fence_before();
    __syncthreads();
    spl_tc_fence_after();
    if (warp == SCORES) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}
