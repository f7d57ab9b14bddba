// The work line of kv_tree_line.cuh on the host: every tile is some CTA's exactly once, and the items' counters are zero again
// after a launch in which any of the CTAs gave up anywhere.
#include "kv_tree_line.cuh"

#include <random>
#include <vector>

using namespace axb;

extern "C" int next_error(const int *words, int count)
{
    if (count != ERR_WORDS) return -2;
    int w[ERR_WORDS];
    std::copy(words, words + count, w);
    return next_device_error(w);
}

// what tree_start finds, by a plain walk
static bool start(const KvTreeArgs &a, const TreeLine &ln, int cta, int ctas, TreeCursor &c)
{
    int total = 0;
    std::vector<int> of(a.B);
    for (int b = 0; b < a.B; ++b) total += of[b] = tree_tiles(a, tree_seq(a, ln, b));
    c.per = max((total + ctas - 1) / ctas, ln.min_stretch);
    c.pos = min(c.per * cta, total);
    c.end = min(c.pos + c.per, total);
    c.b = c.base = 0;
    if (c.pos >= c.end) return false;
    while (c.base + of[c.b] <= c.pos) c.base += of[c.b++];
    return true;
}

// 0: good.  *left: what the counters would hold in sum if a CTA that gave up just went.
extern "C" int line_check(int seed, int B, int T, int heads_per, int Hkv, int max_seq, int block_rows, int tile_keys, int min_stretch, int gap, int ctas,
                          int give_up_percent, int *left)
{
    std::mt19937 rng(seed);
    auto draw = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
    std::vector<int32_t> lens(B), n(B);
    for (int b = 0; b < B; ++b) {
        n[b] = draw(0, min(T, max_seq));
        lens[b] = draw(0, max_seq - n[b]);
        if (draw(0, 19) == 0) lens[b] = max_seq + 1;   // refused
    }
    std::vector<int> counters(ctas, 0), plain(ctas, 0);
    KvTreeArgs a = {};
    a.lens = lens.data(); a.n_new = n.data(); a.counters = counters.data();
    a.max_seq = max_seq; a.B = B; a.H = heads_per * Hkv; a.Hkv = Hkv; a.T = T;
    const TreeLine ln = { block_rows, tile_keys, min_stretch, gap };

    std::vector<TreeCursor> from(ctas);
    std::vector<std::vector<TreePiece>> pieces(ctas);
    std::vector<std::vector<uint8_t>> seen;   // [item][tile]
    std::vector<int> item_at;                 // first item of sequence b
    for (int b = 0; b < B; ++b) {
        const TreeSeq s = tree_seq(a, ln, b);
        item_at.push_back((int)seen.size());
        for (int i = 0; i < (s.n ? Hkv * s.blocks : 0); ++i) seen.emplace_back(s.tiles, 0);
    }
    for (int c = 0; c < ctas; ++c) {
        if (!start(a, ln, c, ctas, from[c])) {
            from[c].pos = from[c].end = 0;
            continue;
        }
        TreeCursor cur = from[c];
        TreePiece p;
        int shared = 0;
        while (next_piece(a, ln, cur, p)) {
            pieces[c].push_back(p);
            shared += p.pieces > 1;
            if (p.first > c || p.first + p.pieces <= c || (p.first == c) != (p.t0 == 0 || p.pieces == 1)) return 1;
            for (int t = 0; t < p.count; ++t)
                if (seen[item_at[p.b] + p.hk * p.s.blocks + p.block][p.t0 + t]++) return 2;
        }
        if (shared > 2) return 3;
    }
    for (auto &item : seen)
        for (uint8_t k : item)
            if (k != 1) return 4;

    // arrivals in any order, a CTA's own in its order; some CTAs give up before some piece
    std::vector<uint32_t> at(ctas, 0), stop(ctas);
    std::vector<int> alive;
    for (int c = 0; c < ctas; ++c) {
        stop[c] = draw(1, 100) <= give_up_percent ? draw(0, (int)pieces[c].size()) : 1u << 30;
        alive.push_back(c);
    }
    int lasts = 0, items = 0;
    for (int c = 0; c < ctas; ++c)
        for (auto &p : pieces[c]) items += p.pieces > 1 && p.first == c;
    while (!alive.empty()) {
        const int k = draw(0, (int)alive.size() - 1), c = alive[k];
        if (at[c] >= stop[c] || at[c] >= pieces[c].size()) {
            if (stop[c] <= pieces[c].size()) tree_leave(a, ln, from[c], at[c]);
            alive.erase(alive.begin() + k);
            continue;
        }
        const TreePiece &p = pieces[c][at[c]++];
        if (p.pieces > 1) {
            if (tree_arrive(a, p)) {
                ++lasts;
                tree_clear(a, p);
            }
            if (++plain[p.first] == p.pieces) plain[p.first] = 0;
        }
    }
    *left = 0;
    for (int c = 0; c < ctas; ++c) {
        if (counters[c]) return 5;
        *left += plain[c];
    }
    if (give_up_percent == 0 && lasts != items) return 6;   // each shared item added up once
    return 0;
}
