// spl_paged_impl.cuh — the entry points of the paged cache (append, attention) and of sampling on the device; included by
// spl_engine.cu, whose engine they belong to.
#pragma once
#include <algorithm>
#include <new>

#include "spl_paged.cuh"
#include "spl_paged_e4m3.cuh"
#include "spl_sample.cuh"

// A call leaves the calling thread's current device as it was.
struct SplDeviceScope {
    int before = -1;
    explicit SplDeviceScope(int device) { cudaGetDevice(&before); if (before != device) cudaSetDevice(device); else before = -1; }
    ~SplDeviceScope() { if (before >= 0) cudaSetDevice(before); }
};

typedef CUresult (*SplEncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct spl_paged {
    spl_engine *e = nullptr;
    int device = 0;                    // the engine's (which may be gone when this object is destroyed)
    spl_paged_config c;
    SplPagedShape shape{};
    int max_pages = 0;
    SplEncodeTiled encode = nullptr;
    // Device tables in one block, filled from one of two pinned blocks (the other's copy may still be on its way): the row count, block_begin, the pieces that have arrived of each merge
    // (none), the blocks' first items, the rows' sequences and positions, the plan's items, the page table. Places do not depend on the batch, so a captured graph finds the next one's.
    size_t words = 0, begin_at = 16, arrived_at = 0, starts_at = 0, batch_at = 0, items_at = 0, table_at = 0;
    SplPagedPlan plan;
    // Partial sums of query rows whose tokens several blocks share.
    int slot_rows = 0;
    float *partial = nullptr;
    float2 *partial_ml = nullptr;
    int *tables_dev = nullptr, *tables_host[2] = {};
    cudaEvent_t copied[2] = {};
    int turn = 0;
    double *turns = nullptr;
    // What a batch is dealt by whose pieces a kernel of its own joins: the count of joining work, the plan's block_begin, starts and items, the records, the work; partial sums by the row.
    struct ByRows {
        size_t words = 0, begin_at = 16, starts_at = 0, items_at = 0, records_at = 0, work_at = 0;
        int *dev = nullptr, *host[2] = {};
        float *partial = nullptr;
        float2 *partial_ml = nullptr;
        SplPagedPlan plan;
        int work = 0;
    };
    // Of batches with groups, made by the first of them, and from then on filled by every batch (a captured graph may hold either form); of batches without that are joined so, which their rows decide.
    ByRows shared, split;
    // The batch that was set last.
    int rows = 0, packed = 0;      // packed: the most packed rows a sequence has
    bool ready = false, shared_write = false, joint = false, by_rows = false;      // joint: some sequences meet a prefix together; by_rows: in `split`
    std::vector<uint8_t> written;      // scratch of the check for pages that two sequences would write

    SplPagedTables tables() const {
        const int *t = tables_dev + batch_at;
        SplPagedTables out;
        out.count = tables_dev;
        out.row_sequence = t; out.row_position = t + c.max_rows;
        out.table = tables_dev + table_at;
        return out;
    }
};

template <int HD> static bool paged_configure_dim() {
    const int bytes = int(spl_paged_smem_bytes(HD));
    return cudaFuncSetAttribute(spl_paged_attend_kernel<HD, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess &&
           cudaFuncSetAttribute(spl_paged_attend_kernel<HD, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}
template <int HD, int N> static bool paged_configure_narrow() {
    return cudaFuncSetAttribute(spl_paged_attend_e4m3_narrow_kernel<HD, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(spl_paged8n_smem_bytes(HD, N))) == cudaSuccess;
}
template <int HD> static bool paged_configure_e4m3() {
    if constexpr (HD >= 128) { if (!paged_configure_narrow<HD, 16>() || !paged_configure_narrow<HD, 32>() || !paged_configure_narrow<HD, 48>()) return false; }
    return cudaFuncSetAttribute(spl_paged_attend_e4m3_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(spl_paged8_smem_bytes(HD))) == cudaSuccess;
}
// (The opt-in is a property of the current device.)
static bool paged_configure(int head_dim, bool e4m3) {
    if (e4m3) return head_dim == 64 ? paged_configure_e4m3<64>() : head_dim == 128 ? paged_configure_e4m3<128>() : paged_configure_e4m3<256>();
    return head_dim == 64 ? paged_configure_dim<64>() : head_dim == 128 ? paged_configure_dim<128>() : paged_configure_dim<256>();
}

// The device and pinned memory of plans of so many items, records, joining work and rows of partial sums.
static spl_status paged_by_rows_create(spl_paged *p, spl_paged::ByRows &t, int64_t items, int64_t records, int64_t work, int64_t partial_rows) {
    spl_engine *e = p->e;
    if (t.dev) return SPL_OK;
    const size_t blocks = size_t(e->sms), item = sizeof(SplPagedItem) / 4;
    t.starts_at = t.begin_at + (blocks + 1 + 3) / 4 * 4;
    t.items_at = t.starts_at + blocks * item;
    t.records_at = t.items_at + size_t(items) * item;
    t.work_at = t.records_at + size_t(records) * (sizeof(SplPagedRecord) / 4);
    t.words = t.work_at + size_t(work) * 2;
    const size_t table_bytes = (t.words * 4 + 255) / 256 * 256;
    int *host = nullptr;
    SPL_CUDA(cudaMallocHost(reinterpret_cast<void **>(&host), t.words * 8));
    unsigned char *block = nullptr;
    const cudaError_t made = cudaMalloc(reinterpret_cast<void **>(&block), table_bytes + size_t(partial_rows) * (size_t(p->c.head_dim) * 4 + sizeof(float2)));
    if (made != cudaSuccess) { cudaFreeHost(host); SPL_CUDA(made); }
    t.host[0] = host; t.host[1] = host + t.words;
    t.partial = reinterpret_cast<float *>(block + table_bytes);
    t.partial_ml = reinterpret_cast<float2 *>(t.partial + size_t(partial_rows) * p->c.head_dim);
    t.dev = reinterpret_cast<int *>(block);
    return SPL_OK;
}

static spl_status paged_create(spl_engine *e, const spl_paged_config *cp, spl_paged *p) {
    const spl_paged_config &c = p->c = *cp;
    if (const char *wrong = spl_paged_config_error(c)) return e->fail(SPL_ERR_INVALID_ARGUMENT, std::string("spl_paged_create: ") + wrong);
    p->max_pages = (c.max_context + c.page_tokens - 1) / c.page_tokens;
    p->shape = SplPagedShape{c.heads, c.kv_heads, c.heads / c.kv_heads, c.head_dim, c.page_tokens, p->max_pages, c.page_stride, c.head_stride, c.token_stride, c.rotary_dim, c.causal != 0, c.window,
                             c.scale > 0.0f ? c.scale : float(1.0 / std::sqrt(double(c.head_dim)))};
    const size_t blocks = size_t(e->sms), items = size_t(spl_paged_items_max(c, e->sms));
    p->arrived_at = p->begin_at + (blocks + 1 + 3) / 4 * 4;
    p->starts_at = p->arrived_at + (blocks + 3) / 4 * 4;
    p->batch_at = p->starts_at + blocks * (sizeof(SplPagedItem) / 4);
    p->items_at = (p->batch_at + size_t(c.max_rows) * 2 + 3) / 4 * 4;
    p->table_at = p->items_at + items * (sizeof(SplPagedItem) / 4);
    p->words = p->table_at + size_t(p->max_pages) * c.max_sequences;
    p->written.assign(size_t(c.pages), 0);
    p->slot_rows = int(std::min<int64_t>(SPL_PAGED_TILE, int64_t(c.max_rows) * p->shape.group));
    // One block of device memory, one pinned one.
    const size_t slot_rows = size_t(spl_paged_slots_max(e->sms)) * p->slot_rows, table_bytes = (p->words * 4 + 255) / 256 * 256, turn_bytes = 1024;
    unsigned char *block = nullptr;
    SPL_CUDA(cudaMalloc(reinterpret_cast<void **>(&block), table_bytes + turn_bytes + slot_rows * (size_t(c.head_dim) * 4 + sizeof(float2))));
    p->tables_dev = reinterpret_cast<int *>(block);
    p->turns = reinterpret_cast<double *>(block + table_bytes);
    p->partial = reinterpret_cast<float *>(block + table_bytes + turn_bytes);
    p->partial_ml = reinterpret_cast<float2 *>(p->partial + slot_rows * c.head_dim);
    SPL_CUDA(cudaMallocHost(reinterpret_cast<void **>(&p->tables_host[0]), p->words * 8));
    p->tables_host[1] = p->tables_host[0] + p->words;
    for (cudaEvent_t &event : p->copied) SPL_CUDA(cudaEventCreateWithFlags(&event, cudaEventDisableTiming));
    cudaDriverEntryPointQueryResult found;
    void *encode = nullptr;
    SPL_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &encode, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !encode) return e->fail(SPL_ERR_UNSUPPORTED_DEVICE, "spl_paged_create: the driver has no tensor maps");
    p->encode = reinterpret_cast<SplEncodeTiled>(encode);
    if (!paged_configure(c.head_dim, c.dtype == SPL_E4M3)) return e->fail(SPL_ERR_UNSUPPORTED_DEVICE, "spl_paged_create: the kernel's shared-memory opt-in failed");
    if (spl_paged_split(c, std::min<int64_t>(int64_t(c.max_rows) * p->shape.group, SPL_PAGED_TILE))) {      // (some batch is joined so)
        const spl_status made = paged_by_rows_create(p, p->split, int64_t(items), int64_t(items), spl_paged_split_combine_max(c, e->sms), spl_paged_split_rows_max(c, e->sms));
        if (made != SPL_OK) return made;
    }
    double turns[128] = {};
    for (int i = 0; i < c.rotary_dim / 2; ++i) turns[i] = std::pow(double(c.rope_theta), -2.0 * i / c.rotary_dim) / 6.283185307179586476925;
    return upload(e, p->turns, turns, sizeof turns);
}

static void paged_release(spl_paged *p) {
    cudaFree(p->tables_dev);
    for (spl_paged::ByRows *t : {&p->shared, &p->split}) { cudaFree(t->dev); if (t->host[0]) cudaFreeHost(t->host[0]); }
    if (p->tables_host[0]) cudaFreeHost(p->tables_host[0]);
    for (cudaEvent_t event : p->copied) if (event) cudaEventDestroy(event);
    delete p;
}

static cudaStream_t paged_stream(const spl_engine *e, void *stream) { return stream ? static_cast<cudaStream_t>(stream) : e->stream; }

// The plan, in the words of pinned block `turn`: how many are used.
static size_t paged_by_rows_fill(const spl_paged *p, spl_paged::ByRows &t, int turn) {
    const SplPagedPlan &plan = t.plan;
    int *w = t.host[turn], work = 0;
    std::memcpy(w + t.begin_at, plan.block_begin.data(), plan.block_begin.size() * 4);
    std::memcpy(w + t.starts_at, plan.starts.data(), plan.starts.size() * sizeof(SplPagedItem));
    std::memcpy(w + t.items_at, plan.items.data(), plan.items.size() * sizeof(SplPagedItem));
    std::memcpy(w + t.records_at, plan.records.data(), plan.records.size() * sizeof(SplPagedRecord));
    const int chunks = (p->c.head_dim + 127) / 128;
    for (size_t r = 0; r < plan.records.size(); ++r)
        for (int job = 0; job < plan.records[r].count * chunks; job += 4, ++work) { w[t.work_at + 2 * work] = int(r); w[t.work_at + 2 * work + 1] = job; }
    std::memset(w, 0, 16 * 4);
    w[0] = work;
    t.work = work;
    return t.work_at + 2 * size_t(work);
}

static spl_status paged_batch(spl_paged *p, int32_t sequences, const int32_t *rows, const int32_t *lengths, const int32_t *table, int32_t table_ld, const SplPagedGroups &groups, cudaStream_t stream) {
    spl_engine *e = p->e;
    const spl_paged_config &c = p->c;
    std::string why;
    bool shared = false;
    const spl_status taken = spl_paged_batch_check(c, sequences, rows, lengths, table, table_ld, p->written, &shared, &why);
    if (taken != SPL_OK) return e->fail(taken, "spl_paged_batch: " + why);
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    SPL_CUDA(cudaStreamIsCapturing(stream, &capture));
    if (capture != cudaStreamCaptureStatusNone) return e->fail(SPL_ERR_INVALID_ARGUMENT, "spl_paged_batch: a batch is set outside a capture");
    if (groups.count) {
        if (!spl_paged_groups_check(c, sequences, rows, lengths, table, table_ld, groups, &why)) return e->fail(SPL_ERR_INVALID_ROWS, "spl_paged_batch_shared: " + why);
        const spl_status made = paged_by_rows_create(p, p->shared, spl_paged_shared_items_max(c, e->sms), spl_paged_records_max(c, e->sms), spl_paged_combine_max(c, e->sms), spl_paged_partial_rows_max(c, e->sms));
        if (made != SPL_OK) { cudaGetLastError(); return made; }
    }
    int64_t total = 0, packed = 0;
    for (int s = 0; s < sequences; ++s) { total += rows[s]; packed = std::max(packed, int64_t(rows[s]) * p->shape.group); }
    // (Only the plan that is launched by has to be right; a graph of these rows takes the same one.)
    const bool by_rows = spl_paged_split(c, packed);
    const SplPagedGroups none{0, nullptr, nullptr};
    if (by_rows) spl_paged_plan(c, e->sms, sequences, rows, lengths, p->split.plan, &none);
    else spl_paged_plan(c, e->sms, sequences, rows, lengths, p->plan);
    if (p->shared.dev) spl_paged_plan(c, e->sms, sequences, rows, lengths, p->shared.plan, &groups);
    const int turn = p->turn;
    SPL_CUDA(cudaEventSynchronize(p->copied[turn]));      // this block's last copy
    int *w = p->tables_host[turn];
    std::memset(w, 0, 16 * 4);
    w[0] = int(total);
    const SplPagedPlan empty, &plan = by_rows ? empty : p->plan;
    std::memcpy(w + p->begin_at, plan.block_begin.data(), plan.block_begin.size() * 4);
    std::memset(w + p->arrived_at, 0, size_t(e->sms) * 4);
    std::memcpy(w + p->starts_at, plan.starts.data(), plan.starts.size() * sizeof(SplPagedItem));
    std::memcpy(w + p->items_at, plan.items.data(), plan.items.size() * sizeof(SplPagedItem));
    int *row_sequence = w + p->batch_at, *row_position = row_sequence + c.max_rows, *pages = w + p->table_at;
    int longest = 1;
    for (int s = 0, r = 0; s < sequences; ++s) {
        for (int i = 0; i < rows[s]; ++i, ++r) { row_sequence[r] = s; row_position[r] = lengths[s] - rows[s] + i; }
        const int used = (lengths[s] + c.page_tokens - 1) / c.page_tokens;
        if (used) std::memcpy(pages + size_t(s) * p->max_pages, table + size_t(s) * table_ld, size_t(used) * 4);
        longest = std::max(longest, used);
    }
    const size_t planned = p->items_at + plan.items.size() * (sizeof(SplPagedItem) / 4), pitch = size_t(p->max_pages) * 4;
    SPL_CUDA(cudaMemcpyAsync(p->tables_dev, w, planned * 4, cudaMemcpyHostToDevice, stream));
    SPL_CUDA(cudaMemcpy2DAsync(p->tables_dev + p->table_at, pitch, pages, pitch, size_t(longest) * 4, size_t(sequences), cudaMemcpyHostToDevice, stream));
    for (spl_paged::ByRows *t : {&p->shared, &p->split}) {
        if (t == &p->shared ? !t->dev : !by_rows) continue;
        const size_t used = paged_by_rows_fill(p, *t, turn);
        SPL_CUDA(cudaMemcpyAsync(t->dev, t->host[turn], used * 4, cudaMemcpyHostToDevice, stream));
    }
    SPL_CUDA(cudaEventRecord(p->copied[turn], stream));
    p->turn ^= 1;
    p->joint = p->shared.dev && p->shared.plan.joint; p->by_rows = by_rows; p->packed = int(std::min<int64_t>(packed, 1 << 30));
    p->rows = int(total); p->shared_write = shared; p->ready = true;
    return SPL_OK;
}

struct SplPagedOut { uint16_t *q; void *k, *v; SplPagedScales scales; };
template <int TYPE, int HD> static void launch_append_dim(const spl_paged *p, const SplPagedRows &in, const uint16_t *q_norm, const uint16_t *k_norm, const SplPagedOut &out, cudaStream_t stream) {
    // A warp a head of a row; few rows are spread over more blocks.
    const int vectors = p->c.heads + 2 * p->c.kv_heads, most = (vectors + 7) / 8;
    const dim3 grid(p->rows, std::max(1, std::min(most, (2 * p->e->sms + p->rows - 1) / p->rows)));
    launch_step(p->c.dtype == SPL_E4M3 ? spl_paged_append_kernel<TYPE, SPL_CACHE_E4M3, HD> : p->c.dtype == SPL_BF16 ? spl_paged_append_kernel<TYPE, SPL_CACHE_BF16, HD> : spl_paged_append_kernel<TYPE, SPL_CACHE_F16, HD>,
                grid, dim3(256), 0, stream, in, q_norm, k_norm, (const double *)p->turns, p->tables(), p->shape, p->e->g.eps, out.q, out.k, out.v, out.scales);
}
template <int TYPE> static void launch_append(const spl_paged *p, const SplPagedRows &in, const uint16_t *q_norm, const uint16_t *k_norm, const SplPagedOut &out, cudaStream_t stream) {
    if (p->c.head_dim == 64) launch_append_dim<TYPE, 64>(p, in, q_norm, k_norm, out, stream);
    else if (p->c.head_dim == 128) launch_append_dim<TYPE, 128>(p, in, q_norm, k_norm, out, stream);
    else launch_append_dim<TYPE, 256>(p, in, q_norm, k_norm, out, stream);
}

// The cache as a tensor (channel in block, token in page, block of 64 channels, kv head, page) for the copies of values, in boxes of all channels by a page's tokens (at most a
// chunk's), or of keys: of a page's tokens (at most a tile's) by 64 channels, or by a chunk's where the box is a tile's tokens.
static bool paged_map(const spl_paged *p, const void *cache, bool values, CUtensorMap *map) {
    const spl_paged_config &c = p->c;
    if (c.dtype == SPL_E4M3) {
        values = values && !spl_paged_narrow(p->c, p->packed);      // (there the values come in the keys' boxes)
        // In bytes, blocks of 128 channels (all of 64): boxes of a block by a page's tokens (at most a tile's) of keys, of all blocks by a page's tokens (at most a chunk's) of values.
        const cuuint64_t row = cuuint64_t(std::min(c.head_dim, 128)), blocks = cuuint64_t(c.head_dim) / row, dims[5] = {row, cuuint64_t(c.page_tokens), blocks, cuuint64_t(c.kv_heads), cuuint64_t(c.pages)};
        const cuuint64_t strides[4] = {cuuint64_t(c.token_stride), row, cuuint64_t(c.head_stride), cuuint64_t(c.page_stride)};
        const cuuint32_t box[5] = {cuuint32_t(row), cuuint32_t(std::min(c.page_tokens, values ? spl_paged8_v_tokens(c.head_dim) : SPL_PAGED_TILE)), values ? cuuint32_t(blocks) : 1u, 1, 1}, steps[5] = {1, 1, 1, 1, 1};
        return p->encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void *>(cache), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : values ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    const cuuint64_t d = cuuint64_t(c.head_dim), dims[5] = {64, cuuint64_t(c.page_tokens), d / 64, cuuint64_t(c.kv_heads), cuuint64_t(c.pages)};
    const cuuint64_t strides[4] = {cuuint64_t(c.token_stride) * 2, 128, cuuint64_t(c.head_stride) * 2, cuuint64_t(c.page_stride) * 2};
    const int chunk = spl_paged_chunk(c.head_dim), tokens = std::min(c.page_tokens, values ? chunk / (2 * c.head_dim) : SPL_PAGED_TILE);
    const cuuint32_t blocks = values ? cuuint32_t(d / 64) : tokens == SPL_PAGED_TILE ? cuuint32_t(chunk / 16384) : 1u;
    const cuuint32_t box[5] = {64, cuuint32_t(tokens), blocks, 1, 1}, steps[5] = {1, 1, 1, 1, 1};
    return p->encode(map, c.dtype == SPL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void *>(cache), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool BF16> static void launch_attend(const spl_paged *p, const CUtensorMap &k_map, const CUtensorMap &v_map, const SplPagedAttend &a, cudaStream_t stream) {
    launch_step(spl_paged_attend_kernel<HD, BF16>, dim3(p->e->sms), dim3(SPL_PAGED_THREADS), spl_paged_smem_bytes(HD), stream, k_map, v_map, p->tables(), p->shape, a);
}

template <int HD> static void launch_attend_e4m3(const spl_paged *p, const CUtensorMap &k_map, const CUtensorMap &v_map, const SplPagedAttend &a, const SplPagedScaled &scales, cudaStream_t stream) {
    if constexpr (HD >= 128) {
        if (spl_paged_narrow(p->c, p->packed)) {
            // (Over a prefix, several sequences' rows: as many as the batch has.)
            const int packed = p->joint ? std::min(p->rows * p->shape.group, SPL_PAGED8_NARROW) : p->packed, n = packed <= 16 ? 16 : packed <= 32 ? 32 : 48;
            launch_step(n == 16 ? spl_paged_attend_e4m3_narrow_kernel<HD, 16> : n == 32 ? spl_paged_attend_e4m3_narrow_kernel<HD, 32> : spl_paged_attend_e4m3_narrow_kernel<HD, 48>, dim3(p->e->sms), dim3(spl_paged8n_threads(n)),
                        spl_paged8n_smem_bytes(HD, n), stream, k_map, v_map, p->tables(), p->shape, a, scales);
            return;
        }
    }
    launch_step(spl_paged_attend_e4m3_kernel<HD>, dim3(p->e->sms), dim3(SPL_PAGED8_THREADS), spl_paged8_smem_bytes(HD), stream, k_map, v_map, p->tables(), p->shape, a, scales);
}

// The blocks of a row's cluster: a wave of clusters costs some 14 us of meetings and sorting whatever a block's share, and 19 us for 32,768 values a block (they fit
// its shared memory; a larger share is read from L2 in every pass, at the same pace). With top-p over 248,077 values, L2 flushed before each call, in blocks of 1, 2, 4
// and 8: 12 rows take 156, 94, 64 and 45 us, 24 rows 162, 98, 70 and 84 (two waves of eights), 64 rows 166, 107, 129 and 193. Over 32,000, 151,936 and 248,077 values
// and 1 to 128 rows, with top-p and with top-k, the rule's choice was the fastest of the four to within 2 us.
static int sample_blocks(const spl_engine *e, int rows, int limit) {
    int best = 1;
    double least = 0.0;
    for (int blocks = 1; blocks <= SPL_SAMPLE_CLUSTER; blocks *= 2) {
        const int resident = e->sample_clusters[blocks];
        if (resident < 1) continue;      // a size the device cannot hold
        const double cost = double((rows + resident - 1) / resident) * (14.0 + 19.0 * ((limit + blocks - 1) / blocks) / SPL_SAMPLE_STRETCH);
        if (blocks == 1 || cost < least) { best = blocks; least = cost; }
    }
    return best;
}

static spl_status launch_sample(spl_engine *e, const SplSampleArgs &args, int rows, cudaStream_t stream, bool verify = false) {
    const int blocks = sample_blocks(e, rows, args.limit);
    const bool held = blocks * SPL_SAMPLE_STRETCH >= args.limit;      // a block's share fits its shared memory
    void (*kernel)(SplSampleArgs) = verify ? (held ? spl_sample_kernel<true, true> : spl_sample_kernel<false, true>) : held ? spl_sample_kernel<true, false> : spl_sample_kernel<false, false>;
    const size_t smem = sizeof(SplSampleShared) + (verify ? spl_verify_bytes() : 0) + (held ? size_t(((args.limit + blocks - 1) / blocks + 31) / 32 * 32) * 4 : 0);      // a block's stretch, as the kernel forms it
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, rows); cfg.blockDim = dim3(1024); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension; attr[1].val.clusterDim.x = blocks; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, kernel, args);
    return check_launch(e, "sampling");
}

// Four warps a block; a graph's replay may have other work than the batch it was captured with, so the blocks go round.
static void launch_combine(const spl_paged *p, int work, const SplPagedCombine &j, cudaStream_t stream) {
    const dim3 grid(std::max(1, std::min(work, 4 * p->e->sms)));
    const int hd = p->c.head_dim;
    const bool bf16 = p->c.dtype != SPL_F16;
    launch_step(hd == 64 ? (bf16 ? spl_paged_combine_kernel<64, true> : spl_paged_combine_kernel<64, false>) : hd == 128 ? (bf16 ? spl_paged_combine_kernel<128, true> : spl_paged_combine_kernel<128, false>) :
                (bf16 ? spl_paged_combine_kernel<256, true> : spl_paged_combine_kernel<256, false>), grid, dim3(128), 0, stream, j, p->shape);
}

static bool misaligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

static spl_status paged_append(spl_paged *p, const char *name, bool scaled, int32_t type, const void *device_q, int64_t q_ld, const void *device_k, int64_t k_ld, const void *device_v, int64_t v_ld,
                               const spl_tensor *q_norm, const spl_tensor *k_norm, const SplPagedOut &out, void *stream) {
    if (!device_q || !device_k || !device_v || !out.q || !out.k || !out.v) return SPL_ERR_INVALID_ARGUMENT;
    spl_engine *e = p->e;
    SPL_NOT_IN_FLIGHT(e);
    const spl_paged_config &c = p->c;
    auto refuse = [&](const char *text) { return e->fail(SPL_ERR_INVALID_ARGUMENT, std::string(name) + text); };
    if (scaled != (c.dtype == SPL_E4M3)) return refuse(scaled ? "the cache has no scales" : "the cache has scales");
    if (!p->ready) return refuse("no batch is set");
    if (p->shared_write) return refuse("two sequences of the batch would write to one page");
    if (type != SPL_F32 && type != SPL_F16 && type != SPL_BF16) return refuse("rows are fp32, fp16 or bf16");
    const int64_t q_width = int64_t(c.heads) * c.head_dim, kv_width = int64_t(c.kv_heads) * c.head_dim;
    if (q_ld < q_width || k_ld < kv_width || v_ld < kv_width || q_ld % 2 || k_ld % 2 || v_ld % 2) return refuse("row strides must be even and hold the heads");
    const size_t pair = type == SPL_F32 ? 8 : 4;
    if (misaligned(device_q, pair) || misaligned(device_k, pair) || misaligned(device_v, pair)) return refuse("rows begin on a boundary of two elements");
    if (misaligned(out.q, 16) || misaligned(out.k, 16) || misaligned(out.v, 16)) return refuse("queries and cache begin on a 16-byte boundary");
    if (misaligned(out.scales.k, 16) || misaligned(out.scales.v, 16)) return refuse("scales begin on a 16-byte boundary");
    if ((q_norm && (!q_norm->vec || q_norm->count != c.head_dim)) || (k_norm && (!k_norm->vec || k_norm->count != c.head_dim))) return refuse("a norm weight is a vector of head_dim elements");
    const SplDeviceScope scope(e->device);
    const SplPagedRows in{device_q, device_k, device_v, q_ld, k_ld, v_ld};
    const uint16_t *qw = q_norm ? q_norm->vec : nullptr, *kw = k_norm ? k_norm->vec : nullptr;
    if (type == SPL_F32) launch_append<0>(p, in, qw, kw, out, paged_stream(e, stream));
    else if (type == SPL_F16) launch_append<1>(p, in, qw, kw, out, paged_stream(e, stream));
    else launch_append<2>(p, in, qw, kw, out, paged_stream(e, stream));
    return check_launch(e, "spl_paged_append");
}

static spl_status paged_attend(spl_paged *p, const char *name, bool scaled, const void *device_q, const void *device_k_cache, const void *device_v_cache, const float *k_scale, const float *v_scale,
                               int32_t out_type, void *device_out, void *stream) {
    if (!device_q || !device_k_cache || !device_v_cache || !device_out) return SPL_ERR_INVALID_ARGUMENT;
    spl_engine *e = p->e;
    SPL_NOT_IN_FLIGHT(e);
    const spl_paged_config &c = p->c;
    auto refuse = [&](const char *text) { return e->fail(SPL_ERR_INVALID_ARGUMENT, std::string(name) + text); };
    if (scaled != (c.dtype == SPL_E4M3)) return refuse(scaled ? "the cache has no scales" : "the cache has scales");
    if (!p->ready) return refuse("no batch is set");
    const int own_type = scaled ? SPL_BF16 : c.dtype;
    if (out_type != SPL_F32 && out_type != own_type) return refuse("outputs are fp32 or of the queries' type");
    if (misaligned(device_q, 16) || misaligned(device_k_cache, 16) || misaligned(device_v_cache, 16) || misaligned(device_out, 16)) return refuse("all buffers begin on a 16-byte boundary");
    if (misaligned(k_scale, 16) || misaligned(v_scale, 16)) return refuse("scales begin on a 16-byte boundary");
    const SplDeviceScope scope(e->device);
    cudaStream_t st = paged_stream(e, stream);
    // Tables, partial sums by the row and a joining kernel of its own, or the attention's own joins.
    const spl_paged::ByRows *const t = p->joint ? &p->shared : p->by_rows ? &p->split : nullptr;
    const int *tables = t ? t->dev : p->tables_dev;
    const SplPagedAttend a{static_cast<const uint16_t *>(device_q), device_out, out_type == SPL_F32, reinterpret_cast<const SplPagedItem *>(tables + (t ? t->starts_at : p->starts_at)),
                           reinterpret_cast<const SplPagedItem *>(tables + (t ? t->items_at : p->items_at)), tables + (t ? t->begin_at : p->begin_at), p->tables_dev + p->arrived_at,
                           t ? t->partial : p->partial, t ? t->partial_ml : p->partial_ml, t ? 1 : p->slot_rows, e->tc_error};
    CUtensorMap k_map, v_map;
    if (!paged_map(p, device_k_cache, false, &k_map) || !paged_map(p, device_v_cache, true, &v_map)) return refuse("the driver takes no tensor map of this cache");
    const bool bf16 = c.dtype == SPL_BF16;
    if (scaled) {
        const SplPagedScaled scales{k_scale, v_scale};
        if (c.head_dim == 64) launch_attend_e4m3<64>(p, k_map, v_map, a, scales, st);
        else if (c.head_dim == 128) launch_attend_e4m3<128>(p, k_map, v_map, a, scales, st);
        else launch_attend_e4m3<256>(p, k_map, v_map, a, scales, st);
    } else if (c.head_dim == 64) { if (bf16) launch_attend<64, true>(p, k_map, v_map, a, st); else launch_attend<64, false>(p, k_map, v_map, a, st); }
    else if (c.head_dim == 128) { if (bf16) launch_attend<128, true>(p, k_map, v_map, a, st); else launch_attend<128, false>(p, k_map, v_map, a, st); }
    else { if (bf16) launch_attend<256, true>(p, k_map, v_map, a, st); else launch_attend<256, false>(p, k_map, v_map, a, st); }
    if (t) {
        const SplPagedCombine j{t->dev, reinterpret_cast<const int2 *>(t->dev + t->work_at), reinterpret_cast<const SplPagedRecord *>(t->dev + t->records_at), t->partial, t->partial_ml, device_out, a.out_f32};
        launch_combine(p, t->work, j, st);
    }
    return check_launch(e, "spl_paged_attend");
}

extern "C" {

spl_status spl_paged_create(spl_engine *e, const spl_paged_config *config, spl_paged **out) {
    if (!e || !config || !out) return SPL_ERR_INVALID_ARGUMENT;
    SPL_NOT_IN_FLIGHT(e);
    const SplDeviceScope scope(e->device);
    spl_paged *p = nullptr;
    try {
        p = new spl_paged;
        p->e = e; p->device = e->device;
        const spl_status s = paged_create(e, config, p);
        if (s != SPL_OK) { cudaGetLastError(); paged_release(p); return s; }
        *out = p;
        return SPL_OK;
    } catch (const std::bad_alloc &) {
        if (p) paged_release(p);
        return SPL_ERR_ALLOCATION_FAILED;
    }
}

void spl_paged_destroy(spl_paged *p) {
    if (!p) return;
    const SplDeviceScope scope(p->device);
    cudaDeviceSynchronize();          // calls may be queued on streams of the caller's
    paged_release(p);
}

spl_status spl_paged_batch(spl_paged *p, int32_t sequences, const int32_t *rows, const int32_t *lengths, const int32_t *page_table, int32_t table_ld, void *stream) {
    return spl_paged_batch_shared(p, sequences, rows, lengths, page_table, table_ld, 0, nullptr, nullptr, stream);
}

spl_status spl_paged_batch_shared(spl_paged *p, int32_t sequences, const int32_t *rows, const int32_t *lengths, const int32_t *page_table, int32_t table_ld, int32_t groups, const int32_t *group_sequences,
                                  const int32_t *group_tokens, void *stream) {
    if (!p || !rows || !lengths || !page_table || table_ld < 0 || groups < 0 || (groups && (!group_sequences || !group_tokens))) return SPL_ERR_INVALID_ARGUMENT;
    spl_engine *e = p->e;
    SPL_NOT_IN_FLIGHT(e);
    const SplDeviceScope scope(e->device);
    try { return paged_batch(p, sequences, rows, lengths, page_table, table_ld, SplPagedGroups{groups, group_sequences, group_tokens}, paged_stream(e, stream)); }
    catch (const std::bad_alloc &) { return SPL_ERR_ALLOCATION_FAILED; }
}

spl_status spl_paged_append(spl_paged *p, int32_t type, const void *device_q, int64_t q_ld, const void *device_k, int64_t k_ld, const void *device_v, int64_t v_ld,
                            const spl_tensor *q_norm, const spl_tensor *k_norm, void *device_q_out, void *device_k_cache, void *device_v_cache, void *stream) {
    if (!p) return SPL_ERR_INVALID_ARGUMENT;
    return paged_append(p, "spl_paged_append: ", false, type, device_q, q_ld, device_k, k_ld, device_v, v_ld, q_norm, k_norm, {static_cast<uint16_t *>(device_q_out), device_k_cache, device_v_cache, {nullptr, nullptr}}, stream);
}

spl_status spl_paged_append_scaled(spl_paged *p, int32_t type, const void *device_q, int64_t q_ld, const void *device_k, int64_t k_ld, const void *device_v, int64_t v_ld, const spl_tensor *q_norm,
                                   const spl_tensor *k_norm, void *device_q_out, void *device_k_cache, void *device_v_cache, float *device_k_scale, float *device_v_scale, void *stream) {
    if (!p || !device_k_scale || !device_v_scale) return SPL_ERR_INVALID_ARGUMENT;
    return paged_append(p, "spl_paged_append_scaled: ", true, type, device_q, q_ld, device_k, k_ld, device_v, v_ld, q_norm, k_norm,
                        {static_cast<uint16_t *>(device_q_out), device_k_cache, device_v_cache, {device_k_scale, device_v_scale}}, stream);
}

spl_status spl_paged_attend(spl_paged *p, const void *device_q, const void *device_k_cache, const void *device_v_cache, int32_t out_type, void *device_out, void *stream) {
    if (!p) return SPL_ERR_INVALID_ARGUMENT;
    return paged_attend(p, "spl_paged_attend: ", false, device_q, device_k_cache, device_v_cache, nullptr, nullptr, out_type, device_out, stream);
}

spl_status spl_paged_attend_scaled(spl_paged *p, const void *device_q, const void *device_k_cache, const void *device_v_cache, const float *device_k_scale, const float *device_v_scale, int32_t out_type,
                                   void *device_out, void *stream) {
    if (!p || !device_k_scale || !device_v_scale) return SPL_ERR_INVALID_ARGUMENT;
    return paged_attend(p, "spl_paged_attend_scaled: ", true, device_q, device_k_cache, device_v_cache, device_k_scale, device_v_scale, out_type, device_out, stream);
}

spl_status spl_pass_sample(spl_engine *e, const float *device_logits, int32_t rows, int64_t ld, int32_t vocab_limit, const float *device_temperature, const int32_t *device_top_k,
                           const float *device_top_p, const float *device_min_p, const float *device_uniform, int32_t *device_ids, void *stream) {
    if (!e || !device_logits || !device_uniform || !device_ids) return SPL_ERR_INVALID_ARGUMENT;
    SPL_NOT_IN_FLIGHT(e);
    if (rows < 1 || rows > 65535) return e->fail(SPL_ERR_INVALID_ROWS, "spl_pass_sample: the number of rows is outside 1 ... 65535");
    if (vocab_limit < 1 || vocab_limit > SPL_SAMPLE_VOCAB || ld < vocab_limit) return e->fail(SPL_ERR_INVALID_ARGUMENT, "spl_pass_sample: vocab_limit must be 1 ... 524288 and at most the rows' stride");
    const SplDeviceScope scope(e->device);
    const SplSampleArgs args{device_logits, ld, vocab_limit, device_temperature, device_top_k, device_top_p, device_min_p, device_uniform, device_ids};
    return launch_sample(e, args, rows, paged_stream(e, stream));
}

spl_status spl_pass_verify(spl_engine *e, const float *device_logits, int32_t sequences, int32_t rows, int64_t ld, int32_t vocab_limit, const int32_t *device_first, const int32_t *device_drafts, int32_t candidates,
                           const int32_t *device_candidates, const float *device_probabilities, const float *device_temperature, const int32_t *device_top_k, const float *device_top_p, const float *device_min_p,
                           const float *device_uniform, int32_t *device_ids, int32_t *device_accepted, int32_t *device_next, void *stream) {
    if (!e || !device_logits || !device_first || !device_drafts || !device_uniform || !device_ids || !device_accepted || !device_next) return SPL_ERR_INVALID_ARGUMENT;
    SPL_NOT_IN_FLIGHT(e);
    if (sequences < 1 || rows < 1 || rows > 65535 || sequences > 65535) return e->fail(SPL_ERR_INVALID_ROWS, "spl_pass_verify: the number of sequences or rows is outside 1 ... 65535");
    if (vocab_limit < 1 || vocab_limit > SPL_SAMPLE_VOCAB || ld < vocab_limit) return e->fail(SPL_ERR_INVALID_ARGUMENT, "spl_pass_verify: vocab_limit must be 1 ... 524288 and at most the rows' stride");
    if (candidates < 0 || candidates > SPL_VERIFY_CANDIDATES || (candidates && (!device_candidates || !device_probabilities)))
        return e->fail(SPL_ERR_INVALID_ARGUMENT, "spl_pass_verify: a token was picked from at most 64 candidates, with their probabilities (0: it was the only choice)");
    const SplDeviceScope scope(e->device);
    cudaStream_t st = paged_stream(e, stream);
    const SplSampleArgs args{device_logits, ld, vocab_limit, device_temperature, device_top_k, device_top_p, device_min_p, device_uniform, device_ids, device_drafts, candidates, device_candidates, device_probabilities};
    const spl_status launched = launch_sample(e, args, rows, st, true);
    if (launched != SPL_OK) return launched;
    launch_step(spl_verify_count_kernel, dim3((sequences + 3) / 4), dim3(128), 0, st, device_first, int(sequences), int(rows), (const int *)device_ids, device_accepted, device_next);
    return check_launch(e, "spl_pass_verify");
}

spl_status spl_sample(spl_engine *e, int32_t vocab_limit, const spl_sampling *settings, const float *uniform, int32_t *ids) {
    if (!e || !settings || !uniform || !ids || vocab_limit <= 0 || vocab_limit > e->g.vocab || vocab_limit > SPL_SAMPLE_VOCAB) return SPL_ERR_INVALID_ARGUMENT;
    SPL_NOT_IN_FLIGHT(e);
    const int rows = e->last_logit_rows;
    if (rows == 0) return SPL_OK;
    const SplDeviceScope scope(e->device);
    // The settings' columns, then the uniform numbers; the ids come back behind them. The device's side lies in `partials`, which no kernel uses between steps
    // and which holds a top-k's 128 words a row.
    if (!e->topk_host) SPL_CUDA(cudaMallocHost(reinterpret_cast<void **>(&e->topk_host), size_t(e->host->config.max_logit_rows) * SPL_TOPK_MAX * 8));
    float *w = reinterpret_cast<float *>(e->topk_host), *d = e->partials;
    for (int r = 0; r < rows; ++r) {
        w[r] = settings[r].temperature; e->topk_host[rows + r] = settings[r].top_k; w[2 * rows + r] = settings[r].top_p; w[3 * rows + r] = settings[r].min_p; w[4 * rows + r] = uniform[r];
    }
    SPL_CUDA(cudaMemcpyAsync(d, w, size_t(rows) * 20, cudaMemcpyHostToDevice, e->stream));
    const SplSampleArgs args{e->logits, e->logits_ld, vocab_limit, d, reinterpret_cast<const int *>(d) + rows, d + 2 * rows, d + 3 * rows, d + 4 * rows, reinterpret_cast<int *>(d) + 5 * rows};
    const spl_status launched = launch_sample(e, args, rows, e->stream);
    if (launched != SPL_OK) return launched;
    SPL_CUDA(cudaMemcpyAsync(e->topk_host + 5 * rows, d + 5 * rows, size_t(rows) * 4, cudaMemcpyDeviceToHost, e->stream));
    SPL_CUDA(cudaStreamSynchronize(e->stream));
    std::memcpy(ids, e->topk_host + 5 * rows, size_t(rows) * 4);
    return SPL_OK;
}

// Host arithmetic, no device needed.
spl_status spl_paged_check(const spl_paged_config *config, int32_t sequences, const int32_t *rows, const int32_t *lengths, const int32_t *page_table, int32_t table_ld, int32_t *shared_write,
                           char *message, size_t message_bytes) {
    return spl_paged_check_shared(config, sequences, rows, lengths, page_table, table_ld, 0, nullptr, nullptr, shared_write, message, message_bytes);
}

spl_status spl_paged_check_shared(const spl_paged_config *config, int32_t sequences, const int32_t *rows, const int32_t *lengths, const int32_t *page_table, int32_t table_ld, int32_t groups,
                                  const int32_t *group_sequences, const int32_t *group_tokens, int32_t *shared_write, char *message, size_t message_bytes) {
    if (!config || (sequences && (!rows || !lengths || !page_table)) || table_ld < 0 || groups < 0 || (groups && (!group_sequences || !group_tokens))) return SPL_ERR_INVALID_ARGUMENT;
    auto say = [&](const std::string &text) { if (message && message_bytes) { const size_t n = std::min(message_bytes - 1, text.size()); std::memcpy(message, text.data(), n); message[n] = 0; } };
    say("");
    try {
        if (const char *wrong = spl_paged_config_error(*config)) { say(wrong); return SPL_ERR_INVALID_ARGUMENT; }
        if (!sequences) return SPL_OK;
        std::vector<uint8_t> written;
        std::string why;
        bool shared = false;
        spl_status s = spl_paged_batch_check(*config, sequences, rows, lengths, page_table, table_ld, written, &shared, &why);
        if (s == SPL_OK && groups && !spl_paged_groups_check(*config, sequences, rows, lengths, page_table, table_ld, SplPagedGroups{groups, group_sequences, group_tokens}, &why)) s = SPL_ERR_INVALID_ROWS;
        say(why);
        if (s == SPL_OK && shared_write) *shared_write = shared;
        return s;
    } catch (const std::bad_alloc &) { return SPL_ERR_ALLOCATION_FAILED; }
}

spl_status spl_debug_paged_plan(const spl_paged_config *config, int32_t blocks, int32_t sequences, const int32_t *rows, const int32_t *lengths, int32_t *block_begin, int32_t *items, int32_t items_capacity,
                                int32_t *item_count, int32_t *merges, int32_t *merge_count) {
    if (!config || !rows || !lengths || !block_begin || !items || !item_count || !merges || !merge_count || blocks < 1 || sequences < 1 || spl_paged_config_error(*config)) return SPL_ERR_INVALID_ARGUMENT;
    try {
        SplPagedPlan plan;
        spl_paged_plan(*config, blocks, sequences, rows, lengths, plan);
        if (plan.items.size() > size_t(std::max(items_capacity, 0)) || plan.merges > blocks) return SPL_ERR_ALLOCATION_FAILED;
        std::memcpy(block_begin, plan.block_begin.data(), plan.block_begin.size() * 4);
        for (size_t i = 0; i < plan.items.size(); ++i) {
            const SplPagedItem &it = plan.items[i];
            std::memcpy(items + 8 * i, &it, 8 * 4);
            const int32_t merge[8] = {it.row0, it.kv_head, it.q0, it.q_count, it.slot0, it.pieces, it.length, it.base};
            if (it.merge >= 0) std::memcpy(merges + 8 * it.merge, merge, sizeof merge);
        }
        *item_count = int32_t(plan.items.size()); *merge_count = plan.merges;
        return SPL_OK;
    } catch (const std::bad_alloc &) { return SPL_ERR_ALLOCATION_FAILED; }
}

spl_status spl_debug_paged_plan_shared(const spl_paged_config *config, int32_t blocks, int32_t sequences, const int32_t *rows, const int32_t *lengths, int32_t groups, const int32_t *group_sequences,
                                       const int32_t *group_tokens, int32_t *block_begin, int32_t *items, int32_t items_capacity, int32_t *item_count, int32_t *records, int32_t records_capacity,
                                       int32_t *record_count, int64_t *partial_rows, int32_t *joint) {
    if (!config || !rows || !lengths || !block_begin || !items || !item_count || !records || !record_count || !partial_rows || !joint || blocks < 1 || sequences < 1 || groups < 0 ||
        (groups && (!group_sequences || !group_tokens)) || spl_paged_config_error(*config)) return SPL_ERR_INVALID_ARGUMENT;
    // (No pages here: of what spl_paged_batch_shared checks, what the plan goes by.)
    for (int i = 0; i < sequences; ++i) if (rows[i] < 0 || lengths[i] < rows[i]) return SPL_ERR_INVALID_ROWS;
    int64_t at = 0;
    for (int g = 0; g < groups; ++g) {
        if (group_sequences[g] < 1 || at + group_sequences[g] > sequences || group_tokens[g] < 0) return SPL_ERR_INVALID_ROWS;
        for (int64_t end = at + group_sequences[g]; at < end; ++at) if (group_tokens[g] > lengths[at] - rows[at]) return SPL_ERR_INVALID_ROWS;
    }
    try {
        SplPagedPlan plan;
        const SplPagedGroups g{groups, group_sequences, group_tokens};
        spl_paged_plan(*config, blocks, sequences, rows, lengths, plan, &g);
        if (plan.items.size() > size_t(std::max(items_capacity, 0)) || plan.records.size() > size_t(std::max(records_capacity, 0))) return SPL_ERR_ALLOCATION_FAILED;
        std::memcpy(block_begin, plan.block_begin.data(), plan.block_begin.size() * 4);
        for (size_t i = 0; i < plan.items.size(); ++i) std::memcpy(items + 8 * i, &plan.items[i], 8 * 4);
        for (size_t i = 0; i < plan.records.size(); ++i) std::memcpy(records + 10 * i, &plan.records[i], 10 * 4);
        *item_count = int32_t(plan.items.size()); *record_count = int32_t(plan.records.size()); *partial_rows = plan.partial_rows; *joint = plan.joint;
        if (plan.items.size() > size_t(spl_paged_shared_items_max(*config, blocks)) || plan.records.size() > size_t(spl_paged_records_max(*config, blocks)) ||
            plan.partial_rows > spl_paged_partial_rows_max(*config, blocks)) return SPL_ERR_DEVICE;      // (what the object sets aside)
        return SPL_OK;
    } catch (const std::bad_alloc &) { return SPL_ERR_ALLOCATION_FAILED; }
}

}  // extern "C"
