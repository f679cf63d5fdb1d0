// Attention of one step over paged caches, cut into pieces for the two kernels: which kernel takes a stretch of positions, how it is cut and dealt to CTAs, and
// who joins what. No CUDA in here.
#pragma once
#include <algorithm>
#include <functional>
#include <utility>
#include <vector>

#include "paged_items.h"

namespace llamd {

struct Plan {
    std::vector<PagedItem> small, large;
    std::vector<int32_t> begin, small_begin;  // large: each CTA's; small: each CTA's of a kv head, of a cache in 8 bits
    std::vector<PagedMerge> merge;
    std::vector<PagedPart> part;
    bool beside = false;  // small and large pieces at the same time, each on SMs of its own
    int small_rows = 0, most = 0;  // rows of a small piece, parts of a token and head
    size_t rows = 0;  // of partial results
};

// A stretch of positions that some tokens attend to: a sequence's own behind the shared prefix, or the prefix itself.
struct Stretch {
    int table, begin, end, token, n_tok, limit, step;
    bool small = false;  // for paged_decode.cu
};

// Positions to a piece of paged_decode.cu. Its CTAs run two to an SM; the longest piece should not outlast an even share of
// the bytes by much, and a piece costs 8 rows of f32 (4 KB at 128 elements) written and read again where a stretch is cut, which 128 positions
// (64 KB) repay.
inline int decode_piece(long long positions, int n_head_kv, int sms) {
    const long long share = (2 * positions * n_head_kv + 3LL * sms - 1) / (3LL * sms);
    return (int)std::min(1LL << 30, std::max(128LL, (share + 15) / 16 * 16));  // (no sequence is longer)
}

// paged_decode8.cu runs kDecode8Ctas CTAs to an SM. A piece costs about as much as kDecode8Piece positions to begin and end (a pipeline's filling and the join of four
// warps), the launch that joins cut pieces as much as kDecode8Join; a CTA's share has room for a piece of kDecode8Least positions at least (one step of each warp). A run that is
// cut leaves pieces of 64 positions and more, its last of 32 and more: at a list's end half the warps may have nothing to do.
constexpr int kDecode8Piece = 64, kDecode8Join = 256, kDecode8Least = 128;

// A stretch's positions for some tokens, and the cuts that deal it out: pieces [first, first + n) of CTA cta.
struct Run {
    int positions;
};
struct RunCut {
    int run, first, n, cta;
};
// Runs dealt out in order, each CTA filled up to `share` and the run cut there, in steps of 32 positions. Returns how many CTAs that takes.
inline int deal_runs(const std::vector<Run> &runs, long long share, std::vector<RunCut> &cuts) {
    cuts.clear();
    int cta = 0;
    long long left = share;
    for (size_t r = 0; r < runs.size(); r++)
        for (int at = 0; at < runs[r].positions;) {
            const int rest = runs[r].positions - at;
            if (left < kDecode8Piece + std::min(rest, kDecode8Piece) && left < share) cta++, left = share;  // (not a piece that is all beginning and end)
            long long n = std::max<long long>(32, (left - kDecode8Piece) / 32 * 32);
            if (n > rest - 32) n = rest;
            cuts.push_back({(int)r, at, (int)n, cta});
            left -= n + kDecode8Piece;
            at += (int)n;
        }
    return runs.empty() ? 0 : cta + 1;
}
// With the least share with which up to `ctas` CTAs do.
inline int deal_runs_evenly(const std::vector<Run> &runs, int ctas, std::vector<RunCut> &cuts, long long &share) {
    long long total = 0, longest = 0;
    for (const Run &r : runs) total += r.positions + kDecode8Piece, longest = std::max<long long>(longest, r.positions);
    long long low = std::max<long long>(kDecode8Least + kDecode8Piece, total / ctas), high = std::max(low, total + longest + kDecode8Piece);
    if (deal_runs(runs, low, cuts) <= ctas) high = low;
    while (high - low > 16 + low / 64) {
        const long long mid = (low + high) / 2;
        (deal_runs(runs, mid, cuts) <= ctas ? high : low) = mid;
    }
    share = high;
    return deal_runs(runs, high, cuts);
}

// When the last of the runs ends where each is a piece, the longest first to the CTA that is free first.
inline long long whole_runs(const std::vector<Run> &runs, int ctas) {
    std::vector<int> longest;
    for (const Run &r : runs) longest.push_back(r.positions);
    std::sort(longest.begin(), longest.end(), std::greater<int>());
    std::vector<long long> load(ctas, 0);  // (a heap, the least in front)
    long long last = 0;
    for (int n : longest) {
        std::pop_heap(load.begin(), load.end(), std::greater<long long>());
        load.back() += n + kDecode8Piece;
        last = std::max(last, load.back());
        std::push_heap(load.begin(), load.end(), std::greater<long long>());
    }
    return last;
}

// paged_prompt.cu runs one CTA to an SM, each with a list of pieces. In blocks of its loop over two tiles, a block over one tile costs kHalfCost (its
// softmax waits for its products), a piece kPieceCost to begin and end, leaving partial results kPartCost more, and the launch that joins
// them kJoinCost (measured with pieces of 1 to 16 blocks, 1 to 4 to a CTA: 1.7 us a block at 64 elements, 2.0 at 128, 3 to 5 us a piece).
constexpr double kHalfCost = 0.85, kPieceCost = 2.0, kPartCost = 2.0, kJoinCost = 4.0;

// Small and large pieces of one batch, one launch after the other, leave first HBM and then the tensor cores waiting; at the same time, each on SMs of its
// own, neither. What they take, in SM-microseconds: an SM draws about 85 GB/s from HBM where all do not draw at once, a block of two tiles
// takes 2 us (1.7 at 64 elements; 2 stands for both). Each has to be worth something (kBesideLeast us on all SMs), or the two kernels run in turn (measured: 100 sequences behind 1024 shared
// positions, 5 query heads to a kv head, 38 us in turn, 33 beside each other; 100 behind 1024, 8 to a kv head, 37 and 28; at worst 200 behind 256, 28 and 29).
constexpr double kSmBytes = 85e3, kBlockMicros = 2.0, kBesideLeast = 0.5;

struct Large {  // a tile of one kv head
    int tile, head, blocks;
};
struct Cut {  // blocks [first, first + n) of a Large, for a CTA
    int which, first, n, cta;
};

struct Dealer {
    int ctas;
    double block;  // what a block costs
    double cost(const Large &x, int blocks) const { return block * blocks + kPieceCost + (blocks < x.blocks ? kPartCost : 0.0); }
    double even(const std::vector<Large> &large, int per, std::vector<Cut> &cuts) const;
    bool filled(const std::vector<Large> &large, double most, std::vector<Cut> &cuts) const;
    double best(const std::vector<Large> &large, std::vector<Cut> &cuts) const;
};

// Tiles in even pieces of up to `per` blocks, the longest of what is left to the CTA with the least so far. Returns when the last CTA ends.
inline double Dealer::even(const std::vector<Large> &large, int per, std::vector<Cut> &cuts) const {
    cuts.clear();
    for (size_t i = 0; i < large.size(); i++) {
        const int n = (large[i].blocks + per - 1) / per, each = (large[i].blocks + n - 1) / n;
        for (int b = 0; b < large[i].blocks; b += each) cuts.push_back({(int)i, b, std::min(each, large[i].blocks - b), 0});
    }
    std::stable_sort(cuts.begin(), cuts.end(), [](const Cut &a, const Cut &b) { return a.n > b.n; });
    std::vector<std::pair<double, int>> load(ctas);
    for (int i = 0; i < ctas; i++) load[i] = {0.0, i};
    double last = 0.0;
    const auto later = std::greater<std::pair<double, int>>();
    for (Cut &c : cuts) {
        std::pop_heap(load.begin(), load.end(), later);
        load.back().first += cost(large[c.which], c.n);
        last = std::max(last, load.back().first);
        c.cta = load.back().second;
        std::push_heap(load.begin(), load.end(), later);
    }
    return last;
}
// One tile after the other, each CTA filled up to `most` and the tile cut there. False where `most` is too little.
inline bool Dealer::filled(const std::vector<Large> &large, double most, std::vector<Cut> &cuts) const {
    cuts.clear();
    int cta = 0;
    double left = most;
    for (size_t i = 0; i < large.size(); i++)
        for (int first = 0; first < large[i].blocks;) {
            const int rest = large[i].blocks - first;
            int n = rest;
            if (first || cost(large[i], rest) > left) n = std::min(rest, (int)((left - kPieceCost - kPartCost) / block));
            if (n < std::min(rest, 2)) {  // (not a piece of one block at a CTA's end)
                if (++cta >= ctas || most < 2 * block + kPieceCost + kPartCost) return false;
                left = most;
                continue;
            }
            cuts.push_back({(int)i, first, n, cta});
            left -= cost(large[i], n);
            first += n;
        }
    return true;
}
// The cut and deal with which all is done soonest, and when. `large`: in falling order of blocks.
inline double Dealer::best(const std::vector<Large> &large, std::vector<Cut> &cuts) const {
    if (large.empty()) return 0.0;
    std::vector<Cut> cut;
    const int longest = large[0].blocks;
    double ends = even(large, longest, cuts), total = 0.0;
    for (int n = 2; n <= longest && (long long)large.size() * n <= 4LL * ctas; n++) {
        const double e = even(large, (longest + n - 1) / n, cut) + kJoinCost;
        if (e < ends) ends = e, cuts = cut;
    }
    for (const Large &x : large) total += block * x.blocks;
    double low = total / ctas, high = ends - kJoinCost;
    while (high - low > 0.02 * high) {
        const double most = 0.5 * (low + high);
        if (filled(large, most, cut)) {
            cuts = cut;
            high = most;
            ends = most + kJoinCost;
        } else {
            low = most;
        }
    }
    return ends;
}

// Is a shared prefix a stretch of its own, read once for all tokens? Every row then leaves two partial results and more (520 bytes each at 128 elements,
// up to a gigabyte for a few long prompts), which another launch joins. A sequence alone shares with nobody, and sequences of two full tiles of
// query rows and more read K and V for so many rows at a time that nothing is saved. Measured, apart against whole, us (32 heads over 4 of 128):
//   behind 256:  64 of 16 tokens (128 rows each) 50.4 / 19.5, 64 of 32 61.8 / 23.2, 256 of 1 22.9 / 21.8, 1 of 2000 behind 1024 102 / 66
//   behind 1024: 256 of 4 62.0 / 110.5, 64 of 8 40.8 / 38.0, 64 of 32 80.6 / 44.9, 32 of 200 303 / 179, 512 beside 100 of 1 42.4 / 55.7, 2000 beside 30 of 1 119 / 78
//   behind 4096: 64 of 1 24.5 / 48.0, 64 of 16 107 / 120, 16 of 32 63.0 / 51.9, 64 of 32 160 / 134, 16 of 2048 2866 / 2327
// From 256 rows a sequence on whole is at worst 1.04 times apart (2 of 512 behind 4096, 8 heads of 64 without groups: 24.5 / 25.5).
inline bool prefix_apart(const PagedView &v, const int32_t *q_len) {
    long long active = 0;
    for (int s = 0; s < v.n_seq; s++) active += q_len[s] > 0;
    return v.n_shared && active > 1 && (long long)v.tokens * v.group < 2LL * kPagedTileRows * active;
}

inline void make_plan(Plan &plan, const PagedView &v, const int32_t *q_len, const int32_t *kv_len, int sms, bool bits8 = false) {
    const int group = v.group, few_tokens = std::max(1, kPagedPieceRows / group);
    std::vector<Stretch> stretch;  // the shared one, where there is one, then the sequences' own
    const bool shared = prefix_apart(v, q_len);
    const int from = shared ? v.n_shared : 0;
    if (shared) {  // (through the table of the first sequence with new tokens)
        int lead = 0;
        while (!q_len[lead]) lead++;
        stretch.push_back({lead * v.table_stride, 0, v.n_shared, 0, v.tokens, v.n_shared, 0});
    }
    for (int s = 0, t = 0; s < v.n_seq; t += q_len[s], s++)
        if (q_len[s]) stretch.push_back({s * v.table_stride, from, kv_len[s], t, q_len[s], kv_len[s] - q_len[s] + 1, 1});
    // Which go to paged_decode.cu: those of one of its pieces' rows, and others while they are little work in all (rows x positions x kv heads): a launch
    // less and no piece to begin weigh more there than reading K and V once for every 16 rows. Measured, that kernel against the other, us: own stretches
    // of 160 rows and 20 positions 4.0 and 7.1, 240 rows and 130 positions 7.2 and 9.0, 4 times 64 and 508 8.3 and 11.5; 16 times 64 and 1000 to 4000
    // 43 and 27, 1 of 128 and 8000 14 and 21; 2000 rows and 250 positions 12.9 and 8.6. A shared stretch, which otherwise makes a third launch: 192 rows and
    // 2048 positions 13.4 and 16.4, 512 and 512 20.5 and 22.9; 1600 and 256 31.8 and 29.3.
    constexpr long long kFewRows = 256, kFewOwnWork = 800000, kFewSharedWork = 1600000;
    long long own_work = 0;
    for (const Stretch &st : stretch)
        if (st.step && st.n_tok * group > kPagedSmallRows) own_work += (long long)st.n_tok * group * (st.end - st.begin) * v.n_head_kv;
    for (Stretch &st : stretch) {
        const long long rows = (long long)st.n_tok * group;
        st.small = group <= kPagedSmallRows && (rows <= kPagedSmallRows || (st.step ? rows <= kFewRows && own_work <= kFewOwnWork : rows * (st.end - st.begin) * v.n_head_kv <= kFewSharedWork));
    }
    // some tokens of a stretch, and where they leave partial results, by kv head
    struct Tile {
        int stretch, token, n_tok, end;
        std::vector<std::vector<PagedPart>> parts;
    };
    // the stretches' tiles in order; the large ones of `tile_tokens`
    auto tiles_of = [&](int tile_tokens, std::vector<Tile> &tiles, std::vector<Large> &large) {
        for (size_t i = 0; i < stretch.size(); i++) {
            const Stretch &st = stretch[i];
            const bool small = st.small;
            const int most = small ? few_tokens : tile_tokens, n_tiles = (st.n_tok + most - 1) / most, per = small ? (st.n_tok + n_tiles - 1) / n_tiles : most;
            for (int x = 0; x < st.n_tok; x += per) {
                const int n = std::min(per, st.n_tok - x), end = std::min(st.end, st.limit + st.step * (x + n - 1));
                tiles.push_back({(int)i, st.token + x, n, end, {}});
                for (int h = 0; !small && h < v.n_head_kv; h++) large.push_back({(int)tiles.size() - 1, h, (end - st.begin + kPagedBlock - 1) / kPagedBlock});
            }
        }
        std::stable_sort(large.begin(), large.end(), [](const Large &a, const Large &b) { return a.blocks > b.blocks; });
    };
    // a large piece is two tiles of query rows, or one where SMs would stand idle
    std::vector<Tile> tiles;
    std::vector<Large> large;
    std::vector<Cut> cuts;
    tiles_of(2 * (kPagedTileRows / group), tiles, large);
    long long small_positions = 0;
    for (const Tile &tile : tiles)
        if (stretch[tile.stretch].small) small_positions += tile.end - stretch[tile.stretch].begin;
    int small_sms = sms, large_sms = sms;
    double blocks = 0.0;
    for (const Large &x : large) blocks += x.blocks + kPieceCost;
    const double small_work = (double)small_positions * v.n_head_kv * v.hd * (bits8 ? 2 : 4) / kSmBytes, large_work = blocks * kBlockMicros;
    if (small_work > kBesideLeast * sms && large_work > kBesideLeast * sms) {
        plan.beside = true;
        large_sms = std::min(sms - 8, std::max(8, (int)(sms * large_work / (small_work + large_work))));
        small_sms = sms - large_sms;
    }
    const double ends = Dealer{large_sms, 1.0}.best(large, cuts);
    if (!large.empty() && (int)large.size() < large_sms) {
        std::vector<Tile> tiles1;
        std::vector<Large> large1;
        std::vector<Cut> cuts1;
        tiles_of(kPagedTileRows / group, tiles1, large1);
        if (Dealer{large_sms, kHalfCost}.best(large1, cuts1) < ends) tiles.swap(tiles1), large.swap(large1), cuts.swap(cuts1);
    }
    for (Tile &tile : tiles) tile.parts.resize(v.n_head_kv);
    auto item_of = [&](const Tile &tile, int begin, int end) {
        const Stretch &st = stretch[tile.stretch];
        return PagedItem{st.table, begin, end, tile.token, tile.n_tok, st.limit + st.step * (tile.token - st.token), st.step, -1, 0, 0, {0, 0}};
    };
    // room for the partial results of a tile's rows, of `heads` kv heads
    auto room = [&](const Tile &tile, int heads) {
        const int32_t at = (int32_t)std::min<size_t>(plan.rows, 0x7fffffff);
        plan.rows += (size_t)tile.n_tok * group * heads;
        return at;
    };

    // the small ones: cut evenly, the kv heads alike
    const int piece = decode_piece(small_positions, v.n_head_kv, small_sms);
    for (Tile &tile : tiles) {
        const Stretch &st = stretch[tile.stretch];
        if (!st.small || bits8) continue;
        const int len = tile.end - st.begin, n = (len + piece - 1) / piece, per = ((len + n - 1) / n + 15) / 16 * 16, rows = tile.n_tok * group;
        for (int b = st.begin; b < tile.end; b += per) {
            PagedItem it = item_of(tile, b, std::min(tile.end, b + per));
            if (shared || len > per) {
                it.part = room(tile, v.n_head_kv), it.part_rows = rows;
                for (int h = 0; h < v.n_head_kv; h++) tile.parts[h].push_back({it.part + h * rows, tile.token});
            }
            plan.small_rows = std::max(plan.small_rows, rows);
            plan.small.push_back(it);
        }
    }
    // (the longest first: what is left at the end is short)
    if (!bits8) std::stable_sort(plan.small.begin(), plan.small.end(), [](const PagedItem &a, const PagedItem &b) { return a.kv_end - a.kv_begin > b.kv_end - b.kv_begin; });

    // Of a cache in 8 bits: each tile a piece, taken up as CTAs become free, or all CTAs' lists of equal length and a launch to join what that cuts; whichever
    // ends first. Measured, us (32 heads over 4 of 128): 64 sequences of 512 positions 9.6 whole and 14 cut, 256 behind 4096 shared positions 59 and 82,
    // 32 of 150 to 8000 positions 46 and 30.
    if (bits8) {
        std::vector<Run> runs;
        std::vector<RunCut> cut;
        std::vector<int> of;
        for (size_t i = 0; i < tiles.size(); i++)
            if (stretch[tiles[i].stretch].small) runs.push_back({tiles[i].end - stretch[tiles[i].stretch].begin}), of.push_back((int)i);
        const int slots = std::max(1, kDecode8Ctas * small_sms / v.n_head_kv);
        long long share = 0;
        int ctas = deal_runs_evenly(runs, slots, cut, share);
        if (whole_runs(runs, slots) <= share + (shared ? 0 : kDecode8Join)) {
            std::stable_sort(of.begin(), of.end(), [&](int a, int b) { return tiles[a].end - stretch[tiles[a].stretch].begin > tiles[b].end - stretch[tiles[b].stretch].begin; });
            cut.clear(), runs.clear();
            for (int i : of) {
                runs.push_back({tiles[i].end - stretch[tiles[i].stretch].begin});
                cut.push_back({(int)runs.size() - 1, 0, runs.back().positions, (int)runs.size() - 1});
            }
            ctas = (int)runs.size();
        }
        if (ctas) plan.small_begin.assign(ctas + 1, 0);
        for (const RunCut &c : cut) {
            Tile &tile = tiles[of[c.run]];
            const int begin = stretch[tile.stretch].begin + c.first, rows = tile.n_tok * group;
            PagedItem it = item_of(tile, begin, begin + c.n);
            if (shared || c.n < runs[c.run].positions) {
                it.part = room(tile, v.n_head_kv), it.part_rows = rows;
                for (int h = 0; h < v.n_head_kv; h++) tile.parts[h].push_back({it.part + h * rows, tile.token});
            }
            plan.small_rows = std::max(plan.small_rows, rows);
            plan.small.push_back(it);
            plan.small_begin[c.cta + 1]++;
        }
        for (int c = 0; c < ctas; c++) plan.small_begin[c + 1] += plan.small_begin[c];
    }

    // the large ones, by CTA
    int ctas = 0;
    for (const Cut &c : cuts) ctas = std::max(ctas, c.cta + 1);
    plan.begin.assign(ctas + 1, 0);
    for (const Cut &c : cuts) plan.begin[c.cta + 1]++;
    for (int c = 0; c < ctas; c++) plan.begin[c + 1] += plan.begin[c];
    plan.large.resize(cuts.size());
    std::vector<int> at(plan.begin.begin(), plan.begin.end());
    for (const Cut &c : cuts) {
        const Large &x = large[c.which];
        Tile &tile = tiles[x.tile];
        const int begin = stretch[tile.stretch].begin + c.first * kPagedBlock;
        PagedItem it = item_of(tile, begin, std::min(tile.end, begin + c.n * kPagedBlock));
        it.head = x.head;
        if (shared || c.n < x.blocks) {
            it.part = room(tile, 1);
            tile.parts[x.head].push_back({it.part, tile.token});
        }
        plan.large[at[c.cta]++] = it;
    }

    // who joins what: the shared stretch's tiles come first and cover all tokens
    size_t prefix = 0, own = 0;
    while (shared && own < tiles.size() && tiles[own].stretch == 0) own++;
    for (; own < tiles.size(); own++) {
        const Tile &tile = tiles[own];
        for (int t = tile.token; t < tile.token + tile.n_tok;) {
            int end = tile.token + tile.n_tok;
            if (shared) {
                while (tiles[prefix].token + tiles[prefix].n_tok <= t) prefix++;
                end = std::min(end, tiles[prefix].token + tiles[prefix].n_tok);
            }
            for (int h = 0; h < v.n_head_kv; h++) {
                const int begin = (int)plan.part.size();
                if (shared) plan.part.insert(plan.part.end(), tiles[prefix].parts[h].begin(), tiles[prefix].parts[h].end());
                plan.part.insert(plan.part.end(), tile.parts[h].begin(), tile.parts[h].end());
                const int count = (int)plan.part.size() - begin;
                plan.most = std::max(plan.most, count);
                for (int x = t; count && x < end; x++) plan.merge.push_back({x, h, begin, count});
            }
            t = end;
        }
    }
}

// What a cache in 8 bits needs of a batch: where its new tokens meet scale blocks.
inline void blocks_of(std::vector<PagedBlock> &block, int n_seq, const int32_t *q_len, const int32_t *kv_len) {
    for (int s = 0, t = 0; s < n_seq; t += q_len[s], s++)
        for (int pos = kv_len[s] - q_len[s]; pos < kv_len[s];) {
            const int n = std::min(kScaleBlock - pos % kScaleBlock, kv_len[s] - pos);
            block.push_back({t + pos - (kv_len[s] - q_len[s]), n});
            pos += n;
        }
}
// The pages that the plan's large pieces read: each once, a shared prefix's for all; and a table of their places in that list beside the batch's own (a
// second [n_seq][table_stride] behind it), which the pieces are pointed to.
inline void wide_pages(std::vector<PagedWide> &wide, std::vector<int32_t> &table, Plan &plan, const PagedView &v, const int32_t *pages, int pages_stride) {
    if (plan.large.empty()) return;
    const int stride = v.table_stride, common = v.n_shared / v.page;
    std::vector<std::pair<int, int>> range(v.n_seq, {0x7fffffff, 0});  // positions that a sequence's pieces read: one stretch, or the prefix and its own behind it
    for (const PagedItem &it : plan.large) {
        auto &r = range[it.table / stride];
        r = {std::min(r.first, it.kv_begin), std::max(r.second, it.kv_end)};
    }
    table.assign((size_t)v.n_seq * stride, 0);
    int prefix = -1;  // where the common pages begin in the list
    for (int s = 0; s < v.n_seq; s++) {
        const int end = range[s].second, n = (end + v.page - 1) / v.page;
        if (!end) continue;
        int i = range[s].first / v.page;
        if (i < common) {  // (a stretch that begins in front of its own positions begins with the prefix)
            if (prefix < 0) {
                prefix = (int)wide.size();
                for (int x = 0; x < common; x++) wide.push_back({pages[(size_t)s * pages_stride + x], v.page});
            }
            for (; i < std::min(n, common); i++) table[(size_t)s * stride + i] = prefix + i;
        }
        for (; i < n; i++) {
            table[(size_t)s * stride + i] = (int32_t)wide.size();
            wide.push_back({pages[(size_t)s * pages_stride + i], std::min(v.page, end - i * v.page)});
        }
    }
    for (PagedItem &it : plan.large) it.table += v.n_seq * stride;
}
// Do two new tokens' places share a page that two sequences list, or one twice?
inline bool writes_shared(int page, int n_seq, const int32_t *q_len, const int32_t *kv_len, const int32_t *pages, int pages_stride) {
    std::vector<int32_t> written;
    for (int s = 0; s < n_seq; s++)
        if (q_len[s])
            for (int i = (kv_len[s] - q_len[s]) / page; i <= (kv_len[s] - 1) / page; i++) written.push_back(pages[(size_t)s * pages_stride + i]);
    std::sort(written.begin(), written.end());
    return std::adjacent_find(written.begin(), written.end()) != written.end();
}

}  // namespace llamd
