// spl_paged_impl.cuh — the entry points of the paged cache (append, attention) and of sampling on the device; included by
// spl_engine.cu, whose engine they belong to.
#pragma once
#include <algorithm>
#include <new>

#include "spl_paged.cuh"
#include "spl_sample.cuh"

// A call leaves the calling thread's current device as it was.
struct SplDeviceScope {
    int before = -1;
    explicit SplDeviceScope(int device) { cudaGetDevice(&before); if (before != device) cudaSetDevice(device); else before = -1; }
    ~SplDeviceScope() { if (before >= 0) cudaSetDevice(before); }
};

struct spl_paged {
    spl_engine *e = nullptr;
    spl_paged_config c;
    SplPagedShape shape{};
    int max_pages = 0;
    // Device tables in one block, filled by one copy from one of two pinned blocks (the other may still be on its way).
    size_t words = 0;
    int *tables_dev = nullptr, *tables_host[2] = {};
    cudaEvent_t copied[2] = {};
    int turn = 0;
    double *turns = nullptr;
    // The batch that was set last.
    int rows = 0, sequences = 0;
    bool ready = false, shared_write = false;
    std::vector<uint8_t> written;      // scratch of the check for pages that two sequences would write

    SplPagedTables tables() const {
        const int *t = tables_dev;
        SplPagedTables out;
        out.counts = t; t += 16;
        out.row_sequence = t; t += c.max_rows; out.row_position = t; t += c.max_rows;
        out.rows = t; t += c.max_sequences; out.lengths = t; t += c.max_sequences;
        out.table = t;
        return out;
    }
};

static spl_status paged_create(spl_engine *e, const spl_paged_config *cp, spl_paged *p) {
    const spl_paged_config &c = p->c = *cp;
    auto refuse = [&](const char *text) { return e->fail(SPL_ERR_INVALID_ARGUMENT, std::string("spl_paged_create: ") + text); };
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return refuse("heads are 64, 128 or 256 channels wide");
    if (c.heads < 1 || c.kv_heads < 1 || c.heads % c.kv_heads || c.heads > 1024 || c.heads / c.kv_heads > 64) return refuse("heads must be a multiple of kv_heads, at most 1024 and 64 a kv head");
    if (c.dtype != SPL_F16 && c.dtype != SPL_BF16) return refuse("the cache holds fp16 or bf16");
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128 && c.page_tokens != 256) return refuse("pages hold 16, 32, 64, 128 or 256 tokens");
    if (c.pages < 1) return refuse("no pages");
    const int64_t d = c.head_dim, ps = c.page_stride, hs = c.head_stride, ts = c.token_stride;
    if (ps % 8 || hs % 8 || ts % 8) return refuse("strides must be multiples of 8 elements");
    const bool token_inside = ts >= d && hs >= ts * c.page_tokens && ps >= hs * c.kv_heads, head_inside = hs >= d && ts >= hs * c.kv_heads && ps >= ts * c.page_tokens;
    if (!token_inside && !head_inside) return refuse("strides must be those of [page][kv head][token][channel] or [page][token][kv head][channel], rows not overlapping");
    if (ps > (int64_t(1) << 38) || ps > (int64_t(1) << 60) / c.pages) return refuse("the cache is too large");
    if (c.rotary_dim < 0 || c.rotary_dim > c.head_dim || c.rotary_dim % 2) return refuse("rotary_dim must be even and at most head_dim");
    if (c.rotary_dim && !(c.rope_theta > 0.0f && std::isfinite(c.rope_theta))) return refuse("rope_theta must be positive");
    if (!(c.scale >= 0.0f) || !std::isfinite(c.scale)) return refuse("scale must be positive, or 0 for 1 / sqrt(head_dim)");
    if (c.window < 0) return refuse("window must be 0 (none) or a number of tokens");
    if (c.max_sequences < 1 || c.max_rows < 1 || c.max_context < 1 || c.max_context > (1 << 30) || c.max_rows > (1 << 20) || c.max_sequences > (1 << 16)) return refuse("max_sequences, max_rows or max_context out of range");
    p->max_pages = (c.max_context + c.page_tokens - 1) / c.page_tokens;
    if (int64_t(p->max_pages) * c.max_sequences > (int64_t(1) << 28)) return refuse("the page table is too large");
    p->e = e;
    p->shape = SplPagedShape{c.heads, c.kv_heads, c.heads / c.kv_heads, c.head_dim, c.page_tokens, p->max_pages, ps, hs, ts, c.rotary_dim, c.causal != 0, c.window,
                             c.scale > 0.0f ? c.scale : float(1.0 / std::sqrt(double(c.head_dim)))};
    p->words = 16 + size_t(c.max_rows) * 2 + size_t(c.max_sequences) * 2 + size_t(p->max_pages) * c.max_sequences;
    p->written.assign(size_t(c.pages), 0);
    SPL_CUDA(cudaMalloc(reinterpret_cast<void **>(&p->tables_dev), p->words * 4));
    for (int i = 0; i < 2; ++i) {
        SPL_CUDA(cudaMallocHost(reinterpret_cast<void **>(&p->tables_host[i]), p->words * 4));
        SPL_CUDA(cudaEventCreateWithFlags(&p->copied[i], cudaEventDisableTiming));
    }
    std::vector<double> turns(size_t(std::max(1, c.rotary_dim / 2)), 0.0);
    for (int i = 0; i < c.rotary_dim / 2; ++i) turns[i] = std::pow(double(c.rope_theta), -2.0 * i / c.rotary_dim) / 6.283185307179586476925;
    SPL_CUDA(cudaMalloc(reinterpret_cast<void **>(&p->turns), turns.size() * 8));
    SPL_CUDA(cudaMemcpy(p->turns, turns.data(), turns.size() * 8, cudaMemcpyHostToDevice));
    return SPL_OK;
}

static void paged_release(spl_paged *p) {
    cudaFree(p->tables_dev); cudaFree(p->turns);
    for (int i = 0; i < 2; ++i) { if (p->tables_host[i]) cudaFreeHost(p->tables_host[i]); if (p->copied[i]) cudaEventDestroy(p->copied[i]); }
    delete p;
}

static cudaStream_t paged_stream(const spl_engine *e, void *stream) { return stream ? static_cast<cudaStream_t>(stream) : e->stream; }

static spl_status paged_batch(spl_paged *p, int32_t sequences, const int32_t *rows, const int32_t *lengths, const int32_t *table, int32_t table_ld, cudaStream_t stream) {
    spl_engine *e = p->e;
    const spl_paged_config &c = p->c;
    auto refuse = [&](spl_status s, const std::string &text) { return e->fail(s, "spl_paged_batch: " + text); };
    if (sequences < 1 || sequences > c.max_sequences) return refuse(SPL_ERR_INVALID_ROWS, "the number of sequences is outside the limit");
    int64_t total = 0;
    for (int s = 0; s < sequences; ++s) {
        if (rows[s] < 0 || lengths[s] < rows[s]) return refuse(SPL_ERR_INVALID_ROWS, "sequence " + std::to_string(s) + " has more new rows than tokens");
        if (lengths[s] > c.max_context) return refuse(SPL_ERR_CONTEXT_EXCEEDED, "sequence " + std::to_string(s) + " is longer than max_context");
        total += rows[s];
        const int used = (lengths[s] + c.page_tokens - 1) / c.page_tokens;
        if (used > table_ld) return refuse(SPL_ERR_INVALID_ROWS, "sequence " + std::to_string(s) + " has more pages than the table's rows");
        for (int i = 0; i < used; ++i) {
            const int page = table[size_t(s) * table_ld + i];
            if (page < 0 || page >= c.pages) return refuse(SPL_ERR_INVALID_ROWS, "page " + std::to_string(i) + " of sequence " + std::to_string(s) + " is not a page of the cache");
        }
    }
    if (total < 1 || total > c.max_rows) return refuse(SPL_ERR_INVALID_ROWS, "the number of rows is outside the limit");
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    SPL_CUDA(cudaStreamIsCapturing(stream, &capture));
    if (capture != cudaStreamCaptureStatusNone) return refuse(SPL_ERR_INVALID_ARGUMENT, "a batch is set outside a capture");
    // Pages that two sequences would write to (or one twice): append refuses such a batch.
    bool shared = false;
    auto each_written = [&](auto &&visit) {
        for (int s = 0; s < sequences; ++s)
            if (rows[s]) for (int i = (lengths[s] - rows[s]) / c.page_tokens; i <= (lengths[s] - 1) / c.page_tokens; ++i) visit(table[size_t(s) * table_ld + i]);
    };
    each_written([&](int page) { shared = shared || p->written[page]; p->written[page] = 1; });
    each_written([&](int page) { p->written[page] = 0; });
    const int turn = p->turn;
    SPL_CUDA(cudaEventSynchronize(p->copied[turn]));      // this block's last copy
    int *w = p->tables_host[turn];
    std::memset(w, 0, 16 * 4);
    w[0] = int(total); w[1] = sequences;
    int *row_sequence = w + 16, *row_position = row_sequence + c.max_rows, *seq_rows = row_position + c.max_rows, *seq_lengths = seq_rows + c.max_sequences, *pages = seq_lengths + c.max_sequences;
    for (int s = 0, r = 0; s < sequences; ++s) {
        for (int i = 0; i < rows[s]; ++i, ++r) { row_sequence[r] = s; row_position[r] = lengths[s] - rows[s] + i; }
        seq_rows[s] = rows[s]; seq_lengths[s] = lengths[s];
        const int used = (lengths[s] + c.page_tokens - 1) / c.page_tokens;
        if (used) std::memcpy(pages + size_t(s) * p->max_pages, table + size_t(s) * table_ld, size_t(used) * 4);
    }
    const size_t used_words = size_t(pages - w) + size_t(sequences) * p->max_pages;
    SPL_CUDA(cudaMemcpyAsync(p->tables_dev, w, used_words * 4, cudaMemcpyHostToDevice, stream));
    SPL_CUDA(cudaEventRecord(p->copied[turn], stream));
    p->turn ^= 1;
    p->rows = int(total); p->sequences = sequences; p->shared_write = shared; p->ready = true;
    return SPL_OK;
}

template <int TYPE> static void launch_append(const spl_paged *p, const SplPagedRows &in, const uint16_t *q_norm, const uint16_t *k_norm, uint16_t *q, uint16_t *k, uint16_t *v, cudaStream_t stream) {
    // A warp a head of a row; few rows are spread over more blocks.
    const int vectors = p->c.heads + 2 * p->c.kv_heads, most = (vectors + 7) / 8;
    const dim3 grid(p->rows, std::max(1, std::min(most, (2 * p->e->sms + p->rows - 1) / p->rows)));
    if (p->c.dtype == SPL_BF16)
        launch_step(spl_paged_append_kernel<TYPE, true>, grid, dim3(256), 0, stream, in, q_norm, k_norm, (const double *)p->turns, p->tables(), p->shape, p->e->g.eps, q, k, v);
    else
        launch_step(spl_paged_append_kernel<TYPE, false>, grid, dim3(256), 0, stream, in, q_norm, k_norm, (const double *)p->turns, p->tables(), p->shape, p->e->g.eps, q, k, v);
}

static bool misaligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

extern "C" {

spl_status spl_paged_create(spl_engine *e, const spl_paged_config *config, spl_paged **out) {
    if (!e || !config || !out) return SPL_ERR_INVALID_ARGUMENT;
    SPL_NOT_IN_FLIGHT(e);
    const SplDeviceScope scope(e->device);
    try {
        spl_paged *p = new spl_paged;
        const spl_status s = paged_create(e, config, p);
        if (s != SPL_OK) { cudaGetLastError(); paged_release(p); return s; }
        *out = p;
        return SPL_OK;
    } catch (const std::bad_alloc &) { return SPL_ERR_ALLOCATION_FAILED; }
}

void spl_paged_destroy(spl_paged *p) {
    if (!p) return;
    const SplDeviceScope scope(p->e->device);
    cudaDeviceSynchronize();          // calls may be queued on streams of the caller's
    paged_release(p);
}

spl_status spl_paged_batch(spl_paged *p, int32_t sequences, const int32_t *rows, const int32_t *lengths, const int32_t *page_table, int32_t table_ld, void *stream) {
    if (!p || !rows || !lengths || !page_table || table_ld < 0) return SPL_ERR_INVALID_ARGUMENT;
    spl_engine *e = p->e;
    SPL_NOT_IN_FLIGHT(e);
    const SplDeviceScope scope(e->device);
    try { return paged_batch(p, sequences, rows, lengths, page_table, table_ld, paged_stream(e, stream)); }
    catch (const std::bad_alloc &) { return SPL_ERR_ALLOCATION_FAILED; }
}

spl_status spl_paged_append(spl_paged *p, int32_t type, const void *device_q, int64_t q_ld, const void *device_k, int64_t k_ld, const void *device_v, int64_t v_ld,
                            const spl_tensor *q_norm, const spl_tensor *k_norm, void *device_q_out, void *device_k_cache, void *device_v_cache, void *stream) {
    if (!p || !device_q || !device_k || !device_v || !device_q_out || !device_k_cache || !device_v_cache) return SPL_ERR_INVALID_ARGUMENT;
    spl_engine *e = p->e;
    SPL_NOT_IN_FLIGHT(e);
    const spl_paged_config &c = p->c;
    auto refuse = [&](const char *text) { return e->fail(SPL_ERR_INVALID_ARGUMENT, std::string("spl_paged_append: ") + text); };
    if (!p->ready) return refuse("no batch is set");
    if (p->shared_write) return refuse("two sequences of the batch would write to one page");
    if (type != SPL_F32 && type != SPL_F16 && type != SPL_BF16) return refuse("rows are fp32, fp16 or bf16");
    const int64_t q_width = int64_t(c.heads) * c.head_dim, kv_width = int64_t(c.kv_heads) * c.head_dim;
    if (q_ld < q_width || k_ld < kv_width || v_ld < kv_width || q_ld % 2 || k_ld % 2 || v_ld % 2) return refuse("row strides must be even and hold the heads");
    const size_t pair = type == SPL_F32 ? 8 : 4;
    if (misaligned(device_q, pair) || misaligned(device_k, pair) || misaligned(device_v, pair)) return refuse("rows begin on a boundary of two elements");
    if (misaligned(device_q_out, 16) || misaligned(device_k_cache, 16) || misaligned(device_v_cache, 16)) return refuse("queries and cache begin on a 16-byte boundary");
    if ((q_norm && (!q_norm->vec || q_norm->count != c.head_dim)) || (k_norm && (!k_norm->vec || k_norm->count != c.head_dim))) return refuse("a norm weight is a vector of head_dim elements");
    const SplDeviceScope scope(e->device);
    const SplPagedRows in{device_q, device_k, device_v, q_ld, k_ld, v_ld};
    const uint16_t *qw = q_norm ? q_norm->vec : nullptr, *kw = k_norm ? k_norm->vec : nullptr;
    uint16_t *q = static_cast<uint16_t *>(device_q_out), *k = static_cast<uint16_t *>(device_k_cache), *v = static_cast<uint16_t *>(device_v_cache);
    if (type == SPL_F32) launch_append<0>(p, in, qw, kw, q, k, v, paged_stream(e, stream));
    else if (type == SPL_F16) launch_append<1>(p, in, qw, kw, q, k, v, paged_stream(e, stream));
    else launch_append<2>(p, in, qw, kw, q, k, v, paged_stream(e, stream));
    return check_launch(e, "spl_paged_append");
}

spl_status spl_paged_attend(spl_paged *p, const void *device_q, const void *device_k_cache, const void *device_v_cache, int32_t out_type, void *device_out, void *stream) {
    if (!p || !device_q || !device_k_cache || !device_v_cache || !device_out) return SPL_ERR_INVALID_ARGUMENT;
    spl_engine *e = p->e;
    SPL_NOT_IN_FLIGHT(e);
    const spl_paged_config &c = p->c;
    auto refuse = [&](const char *text) { return e->fail(SPL_ERR_INVALID_ARGUMENT, std::string("spl_paged_attend: ") + text); };
    if (!p->ready) return refuse("no batch is set");
    if (out_type != SPL_F32 && out_type != c.dtype) return refuse("outputs are fp32 or of the cache's type");
    if (misaligned(device_q, 16) || misaligned(device_k_cache, 16) || misaligned(device_v_cache, 16) || misaligned(device_out, 16)) return refuse("all buffers begin on a 16-byte boundary");
    const SplDeviceScope scope(e->device);
    const dim3 grid((c.heads + 3) / 4, p->rows);
    const uint16_t *q = static_cast<const uint16_t *>(device_q), *k = static_cast<const uint16_t *>(device_k_cache), *v = static_cast<const uint16_t *>(device_v_cache);
    cudaStream_t st = paged_stream(e, stream);
    if (c.dtype == SPL_BF16) {
        if (out_type == SPL_F32) launch_step(spl_paged_attend_kernel<true, true>, grid, dim3(128), 0, st, q, k, v, p->tables(), p->shape, device_out);
        else launch_step(spl_paged_attend_kernel<true, false>, grid, dim3(128), 0, st, q, k, v, p->tables(), p->shape, device_out);
    } else {
        if (out_type == SPL_F32) launch_step(spl_paged_attend_kernel<false, true>, grid, dim3(128), 0, st, q, k, v, p->tables(), p->shape, device_out);
        else launch_step(spl_paged_attend_kernel<false, false>, grid, dim3(128), 0, st, q, k, v, p->tables(), p->shape, device_out);
    }
    return check_launch(e, "spl_paged_attend");
}

spl_status spl_pass_sample(spl_engine *e, const float *device_logits, int32_t rows, int64_t ld, int32_t vocab_limit, const float *device_temperature, const int32_t *device_top_k,
                           const float *device_top_p, const float *device_min_p, const float *device_uniform, int32_t *device_ids, void *stream) {
    if (!e || !device_logits || !device_uniform || !device_ids) return SPL_ERR_INVALID_ARGUMENT;
    SPL_NOT_IN_FLIGHT(e);
    if (rows < 1 || rows > 65535) return e->fail(SPL_ERR_INVALID_ROWS, "spl_pass_sample: the number of rows is outside 1 ... 65535");
    if (vocab_limit < 1 || vocab_limit > SPL_SAMPLE_VOCAB || ld < vocab_limit) return e->fail(SPL_ERR_INVALID_ARGUMENT, "spl_pass_sample: vocab_limit must be 1 ... 524288 and at most the rows' stride");
    const SplDeviceScope scope(e->device);
    const SplSampleArgs args{device_logits, ld, vocab_limit, device_temperature, device_top_k, device_top_p, device_min_p, device_uniform, device_ids};
    launch_step(spl_sample_kernel, dim3(rows), dim3(1024), 0, paged_stream(e, stream), args);
    return check_launch(e, "spl_pass_sample");
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
    launch_step(spl_sample_kernel, dim3(rows), dim3(1024), 0, e->stream, args);
    const spl_status launched = check_launch(e, "spl_sample");
    if (launched != SPL_OK) return launched;
    SPL_CUDA(cudaMemcpyAsync(e->topk_host + 5 * rows, d + 5 * rows, size_t(rows) * 4, cudaMemcpyDeviceToHost, e->stream));
    SPL_CUDA(cudaStreamSynchronize(e->stream));
    std::memcpy(ids, e->topk_host + 5 * rows, size_t(rows) * 4);
    return SPL_OK;
}

}  // extern "C"
