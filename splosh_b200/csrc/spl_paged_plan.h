// spl_paged_plan.h — the host arithmetic of the paged cache: which configurations and batches are taken, and how a batch's attention
// is dealt to the blocks of a launch. No device needed.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <vector>

#include "../../include/splosh_cuda.h"

#define SPL_PAGED_TILE 128            // tokens a tile; packed query rows a block

// A block's piece of work: packed query rows [q0, q0 + q_count) of a sequence (packed row i is the sequence's new token i / group, head i % group of
// the kv head) against the tokens [tile_begin * 128, tile_end * 128). slot >= 0: the piece is one of several of its rows and leaves
// partial sums there; the `pieces` of its rows, merge number `merge`, have the slots from slot0 on. length: the sequence's tokens; base: the position of
// its first new one.
struct alignas(16) SplPagedItem { int32_t sequence, row0, kv_head, q0, q_count, tile_begin, tile_end, slot, length, base, merge, pieces, slot0, reserved[3]; };

struct SplPagedPlan {
    std::vector<SplPagedItem> items;
    std::vector<int32_t> block_begin;         // [blocks + 1]: a block's items
    std::vector<SplPagedItem> starts;         // [blocks]: a block's first item (none: no tiles)
    int merges = 0;
};

// Most items that a configuration's batches come to: a block's boundary cuts at most one tile of query rows.
inline int64_t spl_paged_items_max(const spl_paged_config &c, int blocks) {
    const int64_t group = c.heads / c.kv_heads;
    return c.kv_heads * (int64_t(c.max_rows) * group / SPL_PAGED_TILE + std::min(c.max_sequences, c.max_rows)) + blocks;
}

inline int spl_paged_first_token(const spl_paged_config &c, int position) { return c.window > 0 && position + 1 > c.window ? position + 1 - c.window : 0; }

// Why a configuration is refused, or null.
inline const char *spl_paged_config_error(const spl_paged_config &c) {
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return "heads are 64, 128 or 256 channels wide";
    if (c.heads < 1 || c.kv_heads < 1 || c.heads % c.kv_heads || c.heads > 1024 || c.heads / c.kv_heads > 64) return "heads must be a multiple of kv_heads, at most 1024 and 64 a kv head";
    if (c.dtype != SPL_F16 && c.dtype != SPL_BF16) return "the cache holds fp16 or bf16";
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128 && c.page_tokens != 256) return "pages hold 16, 32, 64, 128 or 256 tokens";
    if (c.pages < 1) return "no pages";
    const int64_t d = c.head_dim, ps = c.page_stride, hs = c.head_stride, ts = c.token_stride, most = int64_t(1) << 38;
    if (ps % 8 || hs % 8 || ts % 8) return "strides must be multiples of 8 elements";
    if (ps <= 0 || hs <= 0 || ts <= 0 || ps > most || hs > most || ts > most || ps > (int64_t(1) << 50) / c.pages) return "strides are out of range";
    const bool token_inside = ts >= d && hs >= ts * c.page_tokens && ps >= hs * c.kv_heads, head_inside = hs >= d && ts >= hs * c.kv_heads && ps >= ts * c.page_tokens;
    if (!token_inside && !head_inside) return "strides must be those of [page][kv head][token][channel] or [page][token][kv head][channel], rows not overlapping";
    if (c.rotary_dim < 0 || c.rotary_dim > c.head_dim || c.rotary_dim % 2) return "rotary_dim must be even and at most head_dim";
    if (c.rotary_dim && !(c.rope_theta > 0.0f && std::isfinite(c.rope_theta))) return "rope_theta must be positive";
    if (!(c.scale >= 0.0f) || !std::isfinite(c.scale)) return "scale must be positive, or 0 for 1 / sqrt(head_dim)";
    if (c.window < 0) return "window must be 0 (none) or a number of tokens";
    if (c.max_sequences < 1 || c.max_rows < 1 || c.max_context < 1 || c.max_context > (1 << 30) || c.max_rows > (1 << 20) || c.max_sequences > (1 << 16))
        return "max_sequences, max_rows or max_context out of range";
    if (int64_t((c.max_context + c.page_tokens - 1) / c.page_tokens) * c.max_sequences > (int64_t(1) << 28)) return "the page table is too large";
    return nullptr;
}

// Whether a batch is taken; `why` says what is wrong with one that is not. `shared_write`: two sequences' new tokens share a page (or a
// sequence's page table holds one twice among those it writes to).
inline spl_status spl_paged_batch_check(const spl_paged_config &c, int32_t sequences, const int32_t *rows, const int32_t *lengths, const int32_t *table, int32_t table_ld,
                                        std::vector<uint8_t> &written, bool *shared_write, std::string *why) {
    auto refuse = [&](spl_status s, const std::string &text) { *why = text; return s; };
    if (sequences < 1 || sequences > c.max_sequences) return refuse(SPL_ERR_INVALID_ROWS, "the number of sequences is outside the limit");
    int64_t total = 0;
    for (int s = 0; s < sequences; ++s) {
        const std::string name = "sequence " + std::to_string(s);
        if (rows[s] < 0 || lengths[s] < rows[s]) return refuse(SPL_ERR_INVALID_ROWS, name + " has more new rows than tokens");
        if (lengths[s] > c.max_context) return refuse(SPL_ERR_CONTEXT_EXCEEDED, name + " is longer than max_context");
        total += rows[s];
        const int used = (lengths[s] + c.page_tokens - 1) / c.page_tokens;
        if (used > table_ld) return refuse(SPL_ERR_INVALID_ROWS, name + " has more pages than the table's rows");
        for (int i = 0; i < used; ++i) {
            const int page = table[size_t(s) * table_ld + i];
            if (page < 0 || page >= c.pages) return refuse(SPL_ERR_INVALID_ROWS, "page " + std::to_string(i) + " of " + name + " is not a page of the cache");
        }
    }
    if (total < 1 || total > c.max_rows) return refuse(SPL_ERR_INVALID_ROWS, "the number of rows is outside the limit");
    bool shared = false;
    auto each_written = [&](auto &&visit) {
        for (int s = 0; s < sequences; ++s)
            if (rows[s]) for (int i = (lengths[s] - rows[s]) / c.page_tokens; i <= (lengths[s] - 1) / c.page_tokens; ++i) visit(table[size_t(s) * table_ld + i]);
    };
    written.resize(size_t(c.pages), 0);
    each_written([&](int page) { shared = shared || written[page]; written[page] = 1; });
    each_written([&](int page) { written[page] = 0; });
    *shared_write = shared;
    return SPL_OK;
}

// The tiles of all (sequence, kv head, 128 packed rows) in a line, cut in one stretch a block of equal cost. In tiles: a piece costs its tiles and
// SPL_PAGED_PIECE_COST more (the first keys' way, the output), and a piece of a cut unit what leaving and joining partial sums takes, which goes by the rows.
// Units of many rows are cut only into pieces that are worth it. (Whole units, longest first, leave the last round of blocks idle for prompts and most of the GPU for
// decode steps of few sequences; stretches that cut everything spent 25 of 47 us on joining 1-tile pieces of 128 rows in a step of six decoding sessions and a
// 301-token prompt.)
#define SPL_PAGED_PIECE_COST 2
inline int spl_paged_cut_cost(int q_count) { return q_count <= 16 ? 0 : q_count <= 64 ? 1 : 2; }
inline int spl_paged_cut_least(int q_count) { return q_count <= 16 ? 1 : q_count <= 64 ? 3 : 5; }      // tiles a piece
// What a block that has `left` of its stretch takes of the `t` tiles left of a unit (cut: some have gone to another block): 0, some, or all; -1: the stretch is too short
// for this unit's pieces.
inline int64_t spl_paged_take(int64_t t, int64_t left, int64_t stretch, int q_count, bool cut) {
    const int64_t piece = SPL_PAGED_PIECE_COST + (cut ? spl_paged_cut_cost(q_count) : 0);
    if (t + piece <= left) return t;
    const int64_t least = spl_paged_cut_least(q_count), some = left - SPL_PAGED_PIECE_COST - spl_paged_cut_cost(q_count);
    if (t >= 2 * least) {
        if (some >= least) return std::min(some, t - least);    // (a rest is a piece, too)
        return left == stretch ? -1 : 0;
    }
    return left == stretch ? t : 0;                             // not worth a cut: whole, in a block of its own at the worst
}
inline void spl_paged_plan(const spl_paged_config &c, int blocks, int32_t sequences, const int32_t *rows, const int32_t *lengths, SplPagedPlan &plan) {
    const int group = c.heads / c.kv_heads, tile = SPL_PAGED_TILE;
    std::vector<SplPagedItem> &units = plan.items;
    std::vector<SplPagedItem> whole;
    int64_t tiles = 0;
    int longest = 0;
    for (int s = 0, row0 = 0; s < sequences; row0 += rows[s], ++s)
        for (int h = 0; h < c.kv_heads; ++h)
            for (int q0 = 0; q0 < rows[s] * group; q0 += tile) {
                const int count = std::min(tile, rows[s] * group - q0), base = lengths[s] - rows[s];
                const int first = spl_paged_first_token(c, base + q0 / group), last = c.causal ? base + (q0 + count - 1) / group + 1 : lengths[s];
                const SplPagedItem u{s, row0, h, q0, count, first / tile, (last + tile - 1) / tile, -1, lengths[s], base, -1, 1, 0, {0, 0, 0}};
                tiles += u.tile_end - u.tile_begin;
                longest = std::max(longest, u.tile_end - u.tile_begin);
                whole.push_back(u);
            }
    // The least stretch that makes do with the blocks there are.
    auto blocks_for = [&](int64_t stretch) {
        int64_t used = 1, left = stretch;
        for (const SplPagedItem &u : whole)
            for (int64_t t = u.tile_end - u.tile_begin, all = t; t > 0;) {
                const int64_t take = spl_paged_take(t, left, stretch, u.q_count, t < all);
                if (take < 0) return int64_t(blocks) + 1;
                if (!take) { if (++used > blocks) return used; left = stretch; continue; }
                left -= take + SPL_PAGED_PIECE_COST + (take < all ? spl_paged_cut_cost(u.q_count) : 0);
                t -= take;
            }
        return used;
    };
    int64_t low = SPL_PAGED_PIECE_COST + 1, high = std::max<int64_t>(low, tiles + int64_t(whole.size()) * (SPL_PAGED_PIECE_COST + 2));
    while (low < high) { const int64_t mid = (low + high) / 2; if (blocks_for(mid) <= blocks) high = mid; else low = mid + 1; }
    units.clear(); plan.merges = 0;
    plan.block_begin.assign(1, 0);
    int64_t left = low;
    int slots = 0;
    for (const SplPagedItem &u : whole) {
        const size_t piece0 = units.size();
        const int all = u.tile_end - u.tile_begin;
        for (int t = u.tile_begin; t < u.tile_end;) {
            const int take = int(spl_paged_take(u.tile_end - t, left, low, u.q_count, t > u.tile_begin));
            if (!take) { plan.block_begin.push_back(int32_t(units.size())); left = low; continue; }
            SplPagedItem piece = u;
            piece.tile_begin = t; piece.tile_end = t + take;
            units.push_back(piece);
            left -= take + SPL_PAGED_PIECE_COST + (take < all ? spl_paged_cut_cost(u.q_count) : 0);
            t += take;
        }
        const int pieces = int(units.size() - piece0);
        if (pieces > 1) {
            for (size_t i = piece0; i < units.size(); ++i) { units[i].slot = slots + int(i - piece0); units[i].slot0 = slots; units[i].pieces = pieces; units[i].merge = plan.merges; }
            slots += pieces; ++plan.merges;
        }
    }
    plan.block_begin.resize(size_t(blocks) + 1, int32_t(units.size()));
    plan.block_begin[blocks] = int32_t(units.size());
    plan.starts.assign(size_t(blocks), SplPagedItem{});
    for (int b = 0; b < blocks; ++b) if (plan.block_begin[b] < plan.block_begin[b + 1]) plan.starts[b] = units[plan.block_begin[b]];
}
// Slots that a plan of `blocks` stretches takes at most: a unit is cut only where a block ends, and each such cut makes two pieces of one.
inline int spl_paged_slots_max(int blocks) { return 2 * blocks; }
