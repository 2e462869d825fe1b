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
#define SPL_PAGED8_NARROW 48          // packed rows at most of attention over a cache of e4m3 in its transposed form

// A block's piece of work: packed query rows [q0, q0 + q_count) of a sequence (packed row i is the sequence's new token i / group, head i % group of
// the kv head) against the tokens [tile_begin * 128, tile_end * 128). slot >= 0: the piece is one of several of its rows and leaves
// partial sums there; the `pieces` of its rows, merge number `merge`, have the slots from slot0 on. length: the sequence's tokens; base: the position of
// its first new one.
struct alignas(16) SplPagedItem { int32_t sequence, row0, kv_head, q0, q_count, tile_begin, tile_end, slot, length, base, merge, pieces, slot0, reserved[3]; };

// Rows of a shared batch whose partial sums a kernel of its own joins: `count` packed rows from q0 on of the sequence whose rows begin at row0. Row i's
// sums of piece n lie at row a_first + n * a_step + i of the partial sums (a_pieces of them), and at b_first + n * b_step + i.
struct alignas(16) SplPagedRecord { int32_t row0, q0, kv_head, count, a_first, a_step, a_pieces, b_first, b_step, b_pieces, reserved[2]; };

struct SplPagedPlan {
    std::vector<SplPagedItem> items;
    std::vector<int32_t> block_begin;         // [blocks + 1]: a block's items
    std::vector<SplPagedItem> starts;         // [blocks]: a block's first item (none: no tiles)
    int merges = 0;
    // Of a batch planned with groups (the items' slots are rows of the partial sums, and no block joins): what is joined behind the attention.
    std::vector<SplPagedRecord> records;
    int64_t partial_rows = 0;
    bool joint = false;                       // some sequences meet a prefix together
};

// Which sequences of a batch share their first pages: group g is the next sequences[g] sequences, tokens[g] tokens each.
struct SplPagedGroups { int32_t count; const int32_t *sequences, *tokens; };

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
    if (c.dtype != SPL_F16 && c.dtype != SPL_BF16 && c.dtype != SPL_E4M3) return "the cache holds fp16, bf16 or e4m3";
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64 && c.page_tokens != 128 && c.page_tokens != 256) return "pages hold 16, 32, 64, 128 or 256 tokens";
    if (c.pages < 1) return "no pages";
    const int64_t d = c.head_dim, ps = c.page_stride, hs = c.head_stride, ts = c.token_stride, most = int64_t(1) << 38;
    const int unit = c.dtype == SPL_E4M3 ? 16 : 8;
    if (ps % unit || hs % unit || ts % unit) return "strides must be multiples of 16 bytes";
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

// Whether a batch's groups are taken: whole pages of tokens that lie in front of every member's new rows, in the same pages.
inline bool spl_paged_groups_check(const spl_paged_config &c, int32_t sequences, const int32_t *rows, const int32_t *lengths, const int32_t *table, int32_t table_ld, const SplPagedGroups &groups, std::string *why) {
    int64_t at = 0;
    for (int g = 0; g < groups.count; ++g) {
        const std::string name = "group " + std::to_string(g);
        const int64_t n = groups.sequences[g], tokens = groups.tokens[g];
        if (n < 1 || at + n > sequences) { *why = name + " has more sequences than are left, or none"; return false; }
        if (tokens < 0 || tokens % c.page_tokens) { *why = name + " does not share whole pages"; return false; }
        for (int64_t s = at; s < at + n; ++s) {
            if (tokens > int64_t(lengths[s]) - rows[s]) { *why = name + " shares more tokens than sequence " + std::to_string(s) + " has in front of its new rows"; return false; }
            for (int64_t i = 0; i < tokens / c.page_tokens; ++i)
                if (table[size_t(s) * table_ld + i] != table[size_t(at) * table_ld + i]) { *why = "page " + std::to_string(i) + " of sequence " + std::to_string(s) + " is not that of its group's first"; return false; }
        }
        at += n;
    }
    return true;
}

// The tiles of all (sequence, kv head, 128 packed rows) in a line, cut in one stretch a block of equal cost. In tiles: a piece costs its tiles and
// SPL_PAGED_PIECE_COST more (the first keys' way, the output), and a piece of a cut unit what leaving and joining partial sums takes, which goes by the rows.
// Units of many rows are cut only into pieces that are worth it. (Whole units, longest first, leave the last round of blocks idle for prompts and most of the GPU for
// decode steps of few sequences; stretches that cut everything spent 25 of 47 us on joining 1-tile pieces of 128 rows in a step of six decoding sessions and a
// 301-token prompt.)
#define SPL_PAGED_PIECE_COST 2
// With groups (by_rows) a kernel of its own joins, and pieces may be smaller: the 72 packed rows of twelve sequences over 8,192 shared tokens 32.9 -> 25.0 us. A piece of 128 rows counts for four tiles more
// there (its partial sums), so that pieces get small only where a block's stretch is short: six verify blocks of 24 rows over 1,024 shared tokens 27.2 -> 17.5 us, sixteen 30.3 -> 22.0, and eight of 48 over
// 20,992 stay at 55.7 (61.5 where such pieces counted for one tile).
inline int spl_paged_cut_cost(int q_count, bool by_rows = false) { return q_count <= 16 ? 0 : by_rows ? (q_count <= 96 ? 1 : 4) : q_count <= 64 ? 1 : 2; }
inline int spl_paged_cut_least(int q_count, bool by_rows = false) { return q_count <= 16 ? 1 : by_rows ? 2 : q_count > 64 ? 5 : 3; }      // tiles a piece
// What a block that has `left` of its stretch takes of the `t` tiles left of a unit (cut: some have gone to another block): 0, some, or all; -1: the stretch is too short
// for this unit's pieces.
inline int64_t spl_paged_take(int64_t t, int64_t left, int64_t stretch, int q_count, bool cut, bool by_rows = false) {
    const int64_t piece = SPL_PAGED_PIECE_COST + (cut ? spl_paged_cut_cost(q_count, by_rows) : 0);
    if (t + piece <= left) return t;
    const int64_t least = spl_paged_cut_least(q_count, by_rows), some = left - SPL_PAGED_PIECE_COST - spl_paged_cut_cost(q_count, by_rows);
    if (t >= 2 * least) {
        if (some >= least) return std::min(some, t - least);    // (a rest is a piece, too)
        return left == stretch ? -1 : 0;
    }
    return left == stretch ? t : 0;                             // not worth a cut: whole, in a block of its own at the worst
}
// With groups, the sequences of a run (consecutive members of a group, none with more packed rows than a block takes) meet the whole tiles of their prefix
// together: their rows lie one behind the other, so they are the rows of one sequence over the prefix, in blocks of 128 packed rows whoever's they are; each sequence's own
// tokens are units of their own, and both leave partial sums (O, m, l) that spl_paged_combine_kernel joins. (Sequences of more packed rows read the prefix once for 128 of them as it is.)
// Over a cache of e4m3 a batch takes the transposed form by the most packed rows that a sequence has (so a prompt's rows, or one block of 54 packed, take it from all: six decode rows over 6,000 tokens of 24/4 heads of 256
// 21.6 us, 301 prompt rows 19.6, in one batch 60.4, where 16 bits take 38.2; nine blocks of eight rows 41.1, with one of nine rows among them 63.2; twelve decode rows and a block of eight rows 45.2, of nine 78.9), also where sequences meet a prefix together (48 rows a block then), so a graph that holds one form is right for
// every batch of its rows. Transposed and wide, before pieces were joined by rows: heads of 256 (24 on 4), eight sequences of about 6,000 tokens with 6, 12, 24, 36 and 48 packed rows 27.7 and 51.4, 31.2 and 54.7, 40.4 and
// 56.1, 48.3 and 65.0, 51.2 and 67.9 us; of 128 (32 on 8), with 8, 16, 32 and 48 21.5 and 35.0, 23.9 and 38.7, 30.6 and 37.0, 37.6 and 47.7. (For 64 rows the sums of three parts
// and two blocks of channels, 384 columns of tensor memory, and two tiles' scores, 256, are more than its 512.)
inline bool spl_paged_narrow(const spl_paged_config &c, int64_t packed) { return c.dtype == SPL_E4M3 && c.head_dim >= 128 && packed <= SPL_PAGED8_NARROW; }
// And over such a cache the pieces of a batch whose sequences have more than 8 packed rows, but at most a block's, are joined by the kernel of its own, groups or not. In and behind the attention: heads of 256
// (24 on 4), two rows over 4,000 tokens 27.7 and 16.5 us, eight of two over 7,200 35.8 and 31.5, one verify block of eight rows over 1,000, 4,000 and 32,000 22.2 and 15.7, 39.2 and 17.0, 82.7 and 31.2, one of sixteen
// over 4,000 66.9 and 22.1, eight of eight over 39,000 135.7 and 123.6; heads of 64 (16 on 2), eight of sixteen over 3,600 45.8 and 18.9; 32 sequences, of which few are cut, the same. With fewer rows a piece's join
// is short and the launch counts: one row over 1,000 tokens 10.0 and 11.5, over 4,000 14.4 and 14.5, twelve over 900 12.8 and 13.2, 32 over 2,700 41.6 and 42.5. Prompts: 300 rows over 300 tokens 19.7 and 22.8,
// 2,048 over 26,624 1,358 and 1,396. (Here and below of three sets of data in turn.)
inline bool spl_paged_split(const spl_paged_config &c, int64_t packed) { return c.dtype == SPL_E4M3 && packed > 8 && packed <= SPL_PAGED_TILE; }
// Meeting together pays where the tiles saved are more than the joining: so many a block for one more launch and the pieces' first keys, and one for so many rows of heads that leave and join sums. Measured with
// heads of 256, 24 of them on 4, together and apart:
//   in 16 bits    six sequences of one row over 1,024 shared tokens 15.2 and 13.7 us, over 4,096 17.7 and 21.8; sixteen of four rows over 512 21.5 and 19.7, over 1,024 22.0 and 23.0;
//                 48 of four over 256 35.7 and 30.3, over 512 35.6 and 36.6;
//   transposed    (apart it is quick where sequences find the same keys in L2) six of one row over 4,096 19.4 and 15.7, sixteen over 2,048 19.2 and 19.3, 48 over 1,024 31.1 and 31.2; two of four rows over
//                 20,992 28.1 and 27.0, four 35.3 and 36.1, eight 46.9 and 59.0; 24 of four over 4,096 47.4 and 50.0, 24 of six 63.2 and 58.5;
//   e4m3, wide    eight of sixteen rows over 4,096 53.7 and 45.5, over 20,992 116 and 126.
// A tile counts the same whatever its channels, though one of 64 is a quarter of the bytes and a join is not. Other heads, together and apart, where the rule deals them together:
//   32 on 8 of 128, 16 bits   six of one row over 1,024 11.8 and 13.1, sixteen over 1,024 14.1 and 20.1, 48 over 1,024 27.1 and 53.6; sixteen of four over 512 18.3 and 15.2, over 2,048 19.8 and 29.8;
//     transposed              two of one row over 16,384 17.4 and 25.1, six over 4,096 14.8 and 19.1, sixteen over 1,024 22.4 and 16.0, over 2,048 23.8 and 23.0; six of four over 4,096 23.6 and 20.2, sixteen over 2,048
//                             32.1 and 25.5;
//   32 on 8 of 64             16 bits sixteen of one row over 1,024 12.8 and 19.2, of four over 512 16.3 and 13.9, over 2,048 18.3 and 27.0; e4m3 15.8 and 29.8, 21.6 and 23.0, 25.6 and 48.1;
//   16 on 2 of 64             16 bits two of one row over 16,384 20.6 and 16.1, sixteen over 2,048 16.2 and 13.8, 48 over 1,024 16.3 and 18.1, two of four over 16,384 20.8 and 25.6; e4m3 sixteen of one over 1,024 20.0
//                             and 15.0, 48 over 1,024 21.1 and 25.8.
// So with eight packed rows a sequence or fewer on two kv heads, and transposed with 128 channels, it takes the slower of the two in places.
inline bool spl_paged_joint_pays(int64_t saved, int blocks, int64_t rows_of_heads, bool narrow) { return saved > int64_t(blocks) * (narrow ? 4 : 1) + rows_of_heads / (narrow ? 3 : 10); }
struct SplPagedUnit { SplPagedItem item; bool joint; int run, prefix; };      // run: its run of sequences or -1; prefix: the first of its run's prefix units of its kv head
inline void spl_paged_plan(const spl_paged_config &c, int blocks, int32_t sequences, const int32_t *rows, const int32_t *lengths, SplPagedPlan &plan, const SplPagedGroups *groups = nullptr) {
    const int group = c.heads / c.kv_heads, tile = SPL_PAGED_TILE;
    std::vector<SplPagedItem> &units = plan.items;
    std::vector<SplPagedUnit> whole;
    int64_t tiles = 0;
    auto add = [&](const SplPagedUnit &u) { tiles += u.item.tile_end - u.item.tile_begin; whole.push_back(u); };
    auto add_sequence = [&](int s, int row0, int skip, int run, int first_prefix, int prefix_step) {
        for (int h = 0; h < c.kv_heads; ++h)
            for (int q0 = 0; q0 < rows[s] * group; q0 += tile) {
                const int count = std::min(tile, rows[s] * group - q0), base = lengths[s] - rows[s];
                const int first = spl_paged_first_token(c, base + q0 / group), last = c.causal ? base + (q0 + count - 1) / group + 1 : lengths[s];
                add({SplPagedItem{s, row0, h, q0, count, std::max(first / tile, skip), (last + tile - 1) / tile, -1, lengths[s], base, -1, 1, 0, {0, 0, 0}}, run >= 0, run, first_prefix + h * prefix_step});
            }
    };
    plan.joint = false;
    int64_t most = 0;
    for (int i = 0; i < sequences; ++i) most = std::max(most, int64_t(rows[i]) * group);
    const int width = spl_paged_narrow(c, most) ? SPL_PAGED8_NARROW : tile;
    std::vector<int> run_row0;
    int s = 0, row0 = 0;
    auto pass_over = [&]() { add_sequence(s, row0, 0, -1, 0, 0); row0 += rows[s]; ++s; };
    for (int g = 0; groups && g < groups->count; ++g) {
        const int end = s + groups->sequences[g], prefix = c.window > 0 ? 0 : groups->tokens[g] / tile;
        while (s < end) {
            // The longest run from here on, and whether it pays.
            int run_end = s, members = 0;
            int64_t packed = 0;
            while (run_end < end && int64_t(rows[run_end]) * group <= tile) { packed += rows[run_end] * group; members += rows[run_end] > 0; ++run_end; }
            const int64_t joint_units = (packed + width - 1) / width;
            if (members < 2 || !spl_paged_joint_pays(int64_t(c.kv_heads) * prefix * (members - joint_units), blocks, packed * c.kv_heads, width < tile)) {
                do pass_over(); while (s < run_end);
                continue;
            }
            const int run = int(run_row0.size()), first_prefix = int(whole.size());
            run_row0.push_back(row0);
            plan.joint = true;
            for (int h = 0; h < c.kv_heads; ++h)
                for (int64_t q0 = 0; q0 < packed; q0 += width)
                    add({SplPagedItem{s, row0, h, int(q0), int(std::min<int64_t>(width, packed - q0)), 0, prefix, -1, prefix * tile, prefix * tile, -1, 1, 0, {0, 0, 0}}, true, -1, 0});
            for (; s < run_end; row0 += rows[s], ++s) add_sequence(s, row0, prefix, run, first_prefix, int(joint_units));
        }
    }
    while (s < sequences) pass_over();
    const bool by_rows = plan.joint || (groups && spl_paged_split(c, most));
    // The least stretch that makes do with the blocks there are.
    auto blocks_for = [&](int64_t stretch) {
        int64_t used = 1, left = stretch;
        for (const SplPagedUnit &u : whole)
            for (int64_t t = u.item.tile_end - u.item.tile_begin, all = t; t > 0;) {
                const int64_t take = spl_paged_take(t, left, stretch, u.item.q_count, t < all || u.joint, by_rows);
                if (take < 0) return int64_t(blocks) + 1;
                if (!take) { if (++used > blocks) return used; left = stretch; continue; }
                left -= take + SPL_PAGED_PIECE_COST + (take < all || u.joint ? spl_paged_cut_cost(u.item.q_count, by_rows) : 0);
                t -= take;
            }
        return used;
    };
    int64_t low = SPL_PAGED_PIECE_COST + 1, high = std::max<int64_t>(low, tiles + int64_t(whole.size()) * (SPL_PAGED_PIECE_COST + 2));
    while (low < high) { const int64_t mid = (low + high) / 2; if (blocks_for(mid) <= blocks) high = mid; else low = mid + 1; }
    units.clear(); plan.merges = 0; plan.records.clear(); plan.partial_rows = 0;
    plan.block_begin.assign(1, 0);
    int64_t left = low;
    int slots = 0;
    std::vector<std::pair<int32_t, int32_t>> left_at;      // with groups: each unit's first row of partial sums, and its pieces
    for (const SplPagedUnit &one : whole) {
        const SplPagedItem &u = one.item;
        const size_t piece0 = units.size();
        const int all = u.tile_end - u.tile_begin;
        for (int t = u.tile_begin; t < u.tile_end;) {
            const int take = int(spl_paged_take(u.tile_end - t, left, low, u.q_count, t > u.tile_begin || one.joint, by_rows));
            if (!take) { plan.block_begin.push_back(int32_t(units.size())); left = low; continue; }
            SplPagedItem piece = u;
            piece.tile_begin = t; piece.tile_end = t + take;
            units.push_back(piece);
            left -= take + SPL_PAGED_PIECE_COST + (take < all || one.joint ? spl_paged_cut_cost(u.q_count, by_rows) : 0);
            t += take;
        }
        const int pieces = int(units.size() - piece0);
        if (groups) {
            left_at.push_back({int32_t(plan.partial_rows), pieces});
            if (pieces > 1 || one.joint)
                for (size_t i = piece0; i < units.size(); ++i) { units[i].slot = int32_t(plan.partial_rows); plan.partial_rows += u.q_count; }
        } else if (pieces > 1) {
            for (size_t i = piece0; i < units.size(); ++i) { units[i].slot = slots + int(i - piece0); units[i].slot0 = slots; units[i].pieces = pieces; units[i].merge = plan.merges; }
            slots += pieces; ++plan.merges;
        }
    }
    for (size_t i = 0; i < left_at.size(); ++i) {
        const SplPagedUnit &one = whole[i];
        const SplPagedItem &u = one.item;
        const auto [first, pieces] = left_at[i];
        if (one.run < 0) {
            if (!one.joint && pieces > 1) plan.records.push_back({u.row0, u.q0, u.kv_head, u.q_count, first, u.q_count, pieces, 0, 0, 0, {0, 0}});
            continue;
        }
        // A sequence's rows may lie in two of the run's blocks of packed rows.
        const int begin = (u.row0 - run_row0[one.run]) * group;
        for (int q = begin; q < begin + u.q_count;) {
            const int end = std::min(begin + u.q_count, (q / width + 1) * width), joint = one.prefix + q / width;
            plan.records.push_back({u.row0, q - begin, u.kv_head, end - q, left_at[joint].first + q % width, whole[joint].item.q_count, left_at[joint].second, first + q - begin, u.q_count, pieces, {0, 0}});
            q = end;
        }
    }
    plan.block_begin.resize(size_t(blocks) + 1, int32_t(units.size()));
    plan.block_begin[blocks] = int32_t(units.size());
    plan.starts.assign(size_t(blocks), SplPagedItem{});
    for (int b = 0; b < blocks; ++b) if (plan.block_begin[b] < plan.block_begin[b + 1]) plan.starts[b] = units[plan.block_begin[b]];
}
// Most items, records and rows of partial sums that a plan with groups comes to: the joint rows once over the prefix and once over their own tokens, and each block's boundary cuts at most one
// unit; a sequence's rows are in one record a kv head and tile, or in two.
inline int64_t spl_paged_joint_rows_max(const spl_paged_config &c) { return std::min(int64_t(c.max_rows) * c.heads, int64_t(c.max_sequences) * SPL_PAGED_TILE * c.kv_heads); }
inline int64_t spl_paged_shared_items_max(const spl_paged_config &c, int blocks) { return 2 * spl_paged_items_max(c, blocks); }
inline int64_t spl_paged_records_max(const spl_paged_config &c, int blocks) { return 2 * spl_paged_items_max(c, blocks); }
inline int64_t spl_paged_partial_rows_max(const spl_paged_config &c, int blocks) { return 2 * spl_paged_joint_rows_max(c) + int64_t(blocks) * 2 * std::min<int64_t>(SPL_PAGED_TILE, int64_t(c.max_rows) * (c.heads / c.kv_heads)); }
inline int64_t spl_paged_combine_max(const spl_paged_config &c, int blocks) {      // of blocks of the joining kernel's work, four (row, channels) each
    return (spl_paged_joint_rows_max(c) + int64_t(blocks) * SPL_PAGED_TILE) * ((c.head_dim + 127) / 128) / 4 + spl_paged_records_max(c, blocks);
}
// The same of a plan without groups whose pieces the kernel of its own joins: a block's boundary cuts at most one unit, and each cut makes two pieces of one.
inline int64_t spl_paged_split_rows_max(const spl_paged_config &c, int blocks) { return int64_t(blocks) * 2 * std::min<int64_t>(SPL_PAGED_TILE, int64_t(c.max_rows) * (c.heads / c.kv_heads)); }
inline int64_t spl_paged_split_combine_max(const spl_paged_config &c, int blocks) { return spl_paged_split_rows_max(c, blocks) / 2 * ((c.head_dim + 127) / 128) / 4 + spl_paged_items_max(c, blocks); }
// Slots that a plan of `blocks` stretches takes at most: a unit is cut only where a block ends, and each such cut makes two pieces of one.
inline int spl_paged_slots_max(int blocks) { return 2 * blocks; }
