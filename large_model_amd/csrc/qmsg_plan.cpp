/* qmsg_plan.cpp - checks a batch of sequences and lays it out as work items (qmsg_plan.h). */
#include "qmsg_plan.h"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>

namespace qmsg {

namespace {

std::string text(const char *fmt, ...)
{
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return buf;
}

/* Neighbouring tokens that see the same range of one page table: a sequence's own keys, or a prefix
 * that neighbouring sequences share. */
struct Segment {
    int tok, n_tok;         /* tokens                                        */
    int key0, key1;         /* keys, as far as any of them sees              */
    int table;              /* page table                                    */
    int pos;                /* position of the first token, -1: all see all  */
    int kind;
    int tiles;              /* row tiles                                     */
};

/* A segment's row tile and the items its keys are cut into. */
struct Tile {
    int seg, row, rows;
    int key0, key1, full;
    bool fresh;             /* its first item starts a run                   */
    std::vector<int> cut;   /* where its other items start, each a run       */
};

int kind_of(int rows) { return rows <= attn_rows(kAttnFew, 1) ? kAttnFew : kAttnMany; }

/* Blocks that a CU holds, the fewest keys worth a block, and what an item costs besides its keys, in keys. us by
 * fewest keys: one token over 513 keys 3.9 at 256, 4.1 in one piece of 513 (alone 22 / 24); 8 sequences of 5
 * drafted tokens 14.8 at 256, 13.0 at 384, 12.8 at 512, 14.4 at 768 (alone 40.8, 38.8, 42.6, 46.7); three fp32 prompts
 * to 701 tokens 26.2 at 64 and 128, 27.2 at 256. By an item's cost of 192 / 256 / 320 / 384 keys (alone, the kernels):
 * two prompts to 733 tokens, 64 heads on 4, 34.0 / 32.0 / 28.7 / 26.5 (54 / 57 / 58 / 48), 756 tokens behind 214
 * 42.0 / 40.7 / 37.9 / 39.0 (63 / 62 / 57 / 57), 64 sequences on 8192 shared keys 44.6 / 43.4 / 42.9 / 46.2 (63 / 65
 * / 65 / 69); fp32 prompts 17.9 at 64, 18.2 at 128, 17.3 at 192, 17.5 at 256. */
constexpr int kBlocksPerCu[kAttnKinds] = { 1, 2 };
constexpr int kMinKeys[kAttnKinds] = { 256, 384 }, kMinKeysF32 = 128;
constexpr int kItemCost[kAttnKinds] = { 128, 320 }, kItemCostF32 = 192;
/* Cuts fall on multiples of this many keys from a tile's first. */
constexpr int kCut = 64;

/* The fewest shared keys that are read once for all. */
constexpr int kMinShared = 256;

size_t align16(size_t v) { return (v + 15) & ~(size_t)15; }

size_t most_work(const AttnShape &s)
{
    const size_t G = (size_t)(s.heads / s.kv_heads);
    /* rows in a shared and an own segment, a partial tile for each segment; the cuts, of which each run adds
     * one; and as many empty parts again */
    return 2 * (2 * ((size_t)s.max_tokens * G / 16) + 2 * (size_t)s.max_seq + 16384);
}

}  // namespace

size_t attn_blob_bytes(const AttnShape &s)
{
    const size_t T = (size_t)s.max_tokens;
    return align16(sizeof(AttnHdr)) + T * (sizeof(AttnTok) + sizeof(AttnVTile) + 4) + most_work(s) * sizeof(AttnWork) +
           (size_t)s.max_seq * (size_t)s.max_pages * 4 + 64;
}

std::string attn_plan(const AttnShape &s, int n_cu, int n_seq, const int *q_len, const int *kv_len, const int32_t *pages,
                      int stride, AttnPlan *p, int64_t min_saved)
{
    const int G = s.heads / s.kv_heads, P = s.page;
    if (n_seq < 0 || n_seq > s.max_seq) return text("%d sequences outside [0, max_seq=%d]", n_seq, s.max_seq);
    if (n_seq && (!q_len || !kv_len || !pages)) return "null argument";
    int64_t T = 0;
    for (int i = 0; i < n_seq; i++) {
        const int64_t most = (int64_t)s.max_pages * P;
        if (q_len[i] < 0 || kv_len[i] < q_len[i] || kv_len[i] > most)
            return text("sequence %d: %d new of %d tokens (0 <= new <= all <= %lld)", i, q_len[i], kv_len[i], (long long)most);
        const int need = (int)(((int64_t)kv_len[i] + P - 1) / P);
        if (need > stride) return text("sequence %d: %d tokens need %d pages, a table has %d", i, kv_len[i], need, stride);
        for (int j = 0; j < need; j++) {
            const int32_t id = pages[(size_t)i * (size_t)stride + (size_t)j];
            if (id < 0 || id >= s.n_page) return text("sequence %d: page %d is %d, outside [0, %d)", i, j, id, s.n_page);
        }
        T += q_len[i];
    }
    if (T > s.max_tokens) return text("%lld new tokens, max_tokens is %d", (long long)T, s.max_tokens);
    /* a page takes new tokens of one sequence, at one place of its table */
    if (p->owner.size() != (size_t)s.n_page) p->owner.assign((size_t)s.n_page, 0);
    const int64_t batch = ++p->batches;
    for (int i = 0; i < n_seq; i++) {
        if (q_len[i] == 0) continue;
        for (int j = (kv_len[i] - q_len[i]) / P; j <= (kv_len[i] - 1) / P; j++) {
            const int32_t id = pages[(size_t)i * (size_t)stride + (size_t)j];
            if (p->owner[(size_t)id] == batch) return text("sequence %d: page %d takes new tokens twice", i, id);
            p->owner[(size_t)id] = batch;
        }
    }

    std::vector<AttnTok> tok((size_t)T);
    std::vector<AttnVTile> vt;
    std::vector<int32_t> ids;
    std::vector<int> table((size_t)n_seq), first((size_t)n_seq);
    int t = 0;
    for (int i = 0; i < n_seq; i++) {
        const int32_t *tab = pages + (size_t)i * (size_t)stride;
        table[(size_t)i] = (int)ids.size();
        first[(size_t)i] = t;
        if (q_len[i] == 0) continue;
        ids.insert(ids.end(), tab, tab + (kv_len[i] + P - 1) / P);
        for (int k = 0; k < q_len[i]; k++, t++) {
            const int pos = kv_len[i] - q_len[i] + k, page = tab[pos / P], slot = pos % P;
            tok[(size_t)t] = { pos, page * P + slot, 0, 0 };
            /* tiles start at multiples of kVTile slots where they can, so that their stores are whole */
            if (k && slot % kVTile && slot && vt.back().page == page) vt.back().n++;
            else vt.push_back({ t, 1, page, slot });
        }
    }

    /* neighbouring sequences whose tables start with the same pages, as far as all their new
     * tokens see them and one key at least is left to each */
    auto shared_keys = [&](int a, int b, int most) {
        const int32_t *x = pages + (size_t)a * (size_t)stride, *y = pages + (size_t)b * (size_t)stride;
        int n = 0;
        while ((n + 1) * P <= most && x[n] == y[n]) n++;
        return n * P;
    };
    std::vector<int> used;
    for (int i = 0; i < n_seq; i++)
        if (q_len[i]) used.push_back(i);
    std::vector<Segment> seg;
    auto segments = [&](bool share) -> int64_t {               /* bytes of keys and values that sharing saves */
        int64_t saved = 0;
        seg.clear();
        for (size_t a = 0; a < used.size();) {
            const int i = used[a];
            int keys = kv_len[i] - q_len[i], n_tok = q_len[i];
            size_t b = a + 1;
            while (share && b < used.size()) {
                const int j = used[b], k = shared_keys(i, j, std::min(keys, kv_len[j] - q_len[j]));
                /* joining must not cost the group more keys than the newcomer's prefix saves */
                if (k < kMinShared || (int64_t)k * (int64_t)(b - a) < (int64_t)keys * (int64_t)(b - a - 1)) break;
                keys = k;
                n_tok += q_len[j];
                b++;
            }
            const bool group = b - a > 1;
            if (group) saved += (int64_t)keys * (int64_t)(b - a - 1) * 2 * s.D * (s.type == 1 ? 2 : 4) * s.kv_heads;
            if (group) seg.push_back({ first[(size_t)i], n_tok, 0, keys, table[(size_t)i], -1, kind_of(n_tok * G), 0 });
            for (size_t c = a; c < b; c++) {
                /* a group's own keys in the launch of its shared ones (64 sequences on 8192 shared keys: 44.5 us,
                 * in a launch of their own 51.3), which reads keys for few rows as fast (allotting all
                 * decoding to it: 32 sequences 53.5 us against 54.7) but has more parts to join */
                const int j = used[c], kind = kind_of((group ? n_tok : q_len[j]) * G);
                seg.push_back({ first[(size_t)j], q_len[j], group ? keys : 0, kv_len[j], table[(size_t)j],
                                kv_len[j] - q_len[j], kind, 0 });
            }
            a = b;
        }
        return saved;
    };
    const size_t part_rows = attn_part_rows(s);
    std::vector<Tile> tiles;
    std::vector<int> shared_parts((size_t)T), parts((size_t)T);
    auto make_tiles = [&]() {
        tiles.clear();
        for (size_t i = 0; i < seg.size(); i++) {
            Segment &g = seg[i];
            const int R = attn_rows(g.kind, s.type), rows = g.n_tok * G;
            g.tiles = 0;
            for (int r = 0; r < rows; r += R, g.tiles++) {
                const int n = std::min(R, rows - r);
                /* the tile's last token sees the most keys, its first the fewest */
                const int most = g.pos < 0 ? g.key1 : g.pos + (r + n - 1) / G + 1;
                const int least = g.pos < 0 ? g.key1 : g.pos + r / G + 1;
                tiles.push_back({ (int)i, g.tok * G + r, n, g.key0, most, least, false, {} });
            }
        }
    };
    /* Cut the tiles' keys into runs for the blocks that the card holds. Whole tiles, longest first, where there
     * are enough to even out (parts would cost more). Else each tile in equal pieces, a run each, where that
     * is nearly as even as equal shares of all tiles one after the other, whose runs may span tiles and whose tiles
     * come in more parts. `coarser`: runs that much longer, for fewer parts. */
    auto cut_tiles = [&](int kind, int64_t coarser) {
        const bool f32 = kind == kAttnMany && s.type == 0;
        const int64_t floor = f32 ? kMinKeysF32 : kMinKeys[kind], item = f32 ? kItemCostF32 : kItemCost[kind];
        std::vector<Tile *> of;
        int64_t cost = 0;
        for (Tile &x : tiles)
            if (seg[(size_t)x.seg].kind == kind) {
                of.push_back(&x);
                x.cut.clear();
                x.fresh = true;
                cost += x.key1 - x.key0 + item;
            }
        const int64_t slots = std::max<int64_t>(1, (int64_t)kBlocksPerCu[kind] * n_cu / s.kv_heads);
        if (of.empty() || (int64_t)of.size() >= 2 * slots) return;
        /* the shortest pieces of which there are no more than slots */
        int64_t piece = std::max((cost / slots + kCut - 1) / kCut * kCut, floor) * coarser, n_run = slots + 1;
        for (; (int64_t)of.size() <= slots; piece += piece / 64 / kCut * kCut + kCut) {
            n_run = 0;
            for (const Tile *x : of) n_run += (x->key1 - x->key0 + piece - 1) / piece;
            if (n_run <= slots) break;
        }
        int64_t share = std::max(cost / slots, floor) * coarser + item;
        if (n_run <= slots && piece + item <= share + share / 8) {
            for (Tile *x : of) {
                const int64_t len = x->key1 - x->key0, n = (len + piece - 1) / piece, each = ((len + n - 1) / n + kCut - 1) / kCut * kCut;
                for (int64_t at = each; at < len; at += each) x->cut.push_back(x->key0 + (int)at);
            }
            return;
        }
        for (n_run = slots + 1; n_run > slots; share += share / 64 + kCut) {
            int64_t room = 0;
            n_run = 0;
            for (Tile *x : of) {
                x->cut.clear();
                x->fresh = false;
                for (int at = x->key0;;) {
                    /* no sliver at the end of a run, nor (an eighth over) of a tile */
                    if (room < item + std::min<int64_t>(share / 8, 2 * kCut)) {
                        room = share;
                        n_run++;
                        if (at == x->key0) x->fresh = true;
                        else x->cut.push_back(at);
                    }
                    const int64_t left = x->key1 - at + item, take = (room - item + kCut - 1) / kCut * kCut;
                    if (left <= room + share / 8 || at + take >= x->key1) {
                        room -= left;
                        break;
                    }
                    at += (int)take;
                    room = 0;
                }
            }
        }
    };
    /* Parts of every token: those of the shared segment (as many for all of its tokens), then the most
     * that a tile of the token's own segment is cut into. */
    auto count_parts = [&]() -> bool {
        std::fill(shared_parts.begin(), shared_parts.end(), 0);
        std::fill(parts.begin(), parts.end(), 0);
        size_t x = 0;
        for (const Segment &g : seg) {
            int most = 0;
            for (int k = 0; k < g.tiles; k++) most = std::max(most, (int)tiles[x + (size_t)k].cut.size() + 1);
            for (int k = 0; k < g.tiles; k++, x++) {
                const Tile &y = tiles[x];
                for (int q = y.row / G; q <= (y.row + y.rows - 1) / G; q++) {
                    if (g.pos < 0) shared_parts[(size_t)q] = most;
                    else parts[(size_t)q] = std::max(parts[(size_t)q], (int)y.cut.size() + 1);
                }
            }
        }
        size_t slots = 0;
        for (int k = 0; k < (int)T; k++) {
            tok[(size_t)k].parts = shared_parts[(size_t)k] + parts[(size_t)k];
            tok[(size_t)k].part = (int32_t)slots;
            if (tok[(size_t)k].parts > 1) slots += (size_t)tok[(size_t)k].parts;
        }
        return slots * (size_t)s.heads <= part_rows;
    };
    bool fits = false;
    for (int share = 1; share >= 0 && !fits; share--) {
        if (segments(share != 0) < min_saved && share) continue;
        make_tiles();
        for (int64_t coarser = 1; coarser <= (int64_t)1 << 24 && !fits; coarser *= 2) {
            for (int k = 0; k < kAttnKinds; k++) cut_tiles(k, coarser);
            fits = count_parts();
        }
    }

    std::vector<AttnWork> work[kAttnKinds];
    int n_run[kAttnKinds], counters = 0;
    std::vector<char> apart((size_t)T, 0);                    /* tokens that the join kernel takes */
    for (int kind = 0; kind < kAttnKinds; kind++) {
        std::vector<AttnWork> &first = work[kind], later, empty;
        std::vector<int> run;                                  /* of each later item */
        for (const Tile &x : tiles) {
            const Segment &g = seg[(size_t)x.seg];
            if (g.kind != kind) continue;
            int need = 0;           /* a token in two tiles has the parts of the one that is cut more */
            for (int q = x.row / G; q <= (x.row + x.rows - 1) / G; q++)
                need = std::max(need, g.pos < 0 ? shared_parts[(size_t)q] : parts[(size_t)q]);
            const int base = g.pos < 0 ? 0 : shared_parts[(size_t)(x.row / G)], n = (int)x.cut.size() + 1;
            /* a tile whose rows have no parts but its own items' */
            const bool own = kind == kAttnFew && need > 1 && need <= kAttnJoins && g.pos >= 0 && base == 0 && (counters + 1) * s.kv_heads <= kAttnCounters;
            const int count = own ? counters++ : -1;
            for (int q = x.row / G; q <= (x.row + x.rows - 1) / G; q++) apart[(size_t)q] |= !own;
            for (int k = 0; k < need; k++) {
                AttnWork w{};
                w.row = x.row;
                w.rows = x.rows;
                w.pages = g.table;
                w.key0 = k && k < n ? x.cut[(size_t)k - 1] : x.key0;
                w.key1 = k >= n ? w.key0 : k + 1 < n ? x.cut[(size_t)k] : x.key1;
                w.full = std::min(x.full, w.key1);
                w.part = base + k;
                w.next = -1;
                w.joins = need;
                w.count = count;
                if (k >= n) empty.push_back(w);
                else if (k || x.fresh) first.push_back(w);
                else {
                    later.push_back(w);
                    run.push_back((int)first.size() - 1);
                }
            }
        }
        /* runs of an item each start with the longest: the last ones end soon after another */
        if (later.empty()) std::stable_sort(first.begin(), first.end(), [](const AttnWork &a, const AttnWork &b) { return a.key1 - a.key0 > b.key1 - b.key0; });
        first.insert(first.end(), empty.begin(), empty.end());
        n_run[kind] = (int)first.size();
        for (size_t i = later.size(); i-- > 0;) {              /* a run's items after its first, in their order */
            AttnWork &head = first[(size_t)run[i]];
            later[i].next = head.next;
            head.next = n_run[kind] + (int)i;
        }
        first.insert(first.end(), later.begin(), later.end());
    }

    /* Waves of an item of few rows: the fewest that leave a block for each CU and whose longest item ends with the others.
     * Fewer waves join less and have more steps to overlap; each holds one step's loads in flight whatever their number.
     * us by 8 / 4 / 2 / 1 (one token each; 64 heads on 4, f16): 256 sequences of up to 101 keys 29 / 19 / 15 / 19, of
     * 501 keys 67 / 54 / 50 / 67, 128 of up to 101 15 / 10 / 13 / 18, of up to 1501 41 / 45 / 71 / 115; 16 heads on
     * 16: 256 of up to 101 keys 88 / 55 / 38 / 29. */
    int few_shift = 3;
    if (std::all_of(work[kAttnFew].begin(), work[kAttnFew].end(), [](const AttnWork &w) { return w.joins == 1 && w.next < 0; })) {
        const int step = s.type == 1 ? 32 : 16;                /* keys that a wave takes at a time */
        int64_t steps = 0, most = 0;
        for (const AttnWork &w : work[kAttnFew]) {
            const int64_t n = (w.key1 - w.key0 + step - 1) / step;
            steps += n;
            most = std::max(most, n);
        }
        const double each = (double)(steps * s.kv_heads) / (2.0 * kFewWaves * n_cu);
        const int64_t units = (int64_t)work[kAttnFew].size() * s.kv_heads;
        for (few_shift = 0; few_shift < 3 && ((units << few_shift) < (int64_t)kFewWaves * n_cu || (double)most > (2.0 * each + 1.5) * (1 << few_shift));) few_shift++;
    }

    std::vector<int32_t> comb;
    for (int k = 0; k < (int)T; k++)
        if (tok[(size_t)k].parts > 1 && apart[(size_t)k]) comb.push_back(k);

    AttnHdr h{};
    size_t at = align16(sizeof(AttnHdr));
    auto place = [&](size_t bytes) {
        const size_t o = at;
        at = align16(at + bytes);
        return (int32_t)o;
    };
    h.n_tok = (int)T;
    h.n_vt = (int)vt.size();
    h.n_comb = (int)comb.size();
    h.few_shift = few_shift;
    for (const AttnTok &k : tok) h.max_parts = std::max(h.max_parts, k.parts);
    h.tok = place(tok.size() * sizeof(AttnTok));
    h.vt = place(vt.size() * sizeof(AttnVTile));
    h.comb = place(comb.size() * 4);
    for (int k = 0; k < kAttnKinds; k++) {
        h.n_run[k] = n_run[k];
        h.work[k] = place(work[k].size() * sizeof(AttnWork));
    }
    h.pages = place(ids.size() * 4);
    h.bytes = (int32_t)at;
    if (at > attn_blob_bytes(s)) return text("the batch needs %zu bytes of plan, room for %zu", at, attn_blob_bytes(s));
    p->blob.resize(at);
    uint8_t *o = p->blob.data();
    memcpy(o, &h, sizeof h);
    if (T) memcpy(o + h.tok, tok.data(), tok.size() * sizeof(AttnTok));
    if (!vt.empty()) memcpy(o + h.vt, vt.data(), vt.size() * sizeof(AttnVTile));
    if (!comb.empty()) memcpy(o + h.comb, comb.data(), comb.size() * 4);
    for (int k = 0; k < kAttnKinds; k++)
        if (!work[k].empty()) memcpy(o + h.work[k], work[k].data(), work[k].size() * sizeof(AttnWork));
    if (!ids.empty()) memcpy(o + h.pages, ids.data(), ids.size() * 4);
    p->h = h;
    return "";
}

}  // namespace qmsg
