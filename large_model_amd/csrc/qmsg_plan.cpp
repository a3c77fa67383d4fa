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
    int splits, chunk;      /* items of chunk keys                           */
    int part;               /* first of its splits among its tokens' slots   */
};

int round_up(int v, int m) { return (v + m - 1) / m * m; }

int kind_of(int rows) { return rows <= kAttnRows[kAttnFew] ? kAttnFew : kAttnMany; }

int tiles_of(const Segment &g, int G) { return (g.n_tok * G + kAttnRows[g.kind] - 1) / kAttnRows[g.kind]; }

/* Blocks that fill the card, and the fewest keys worth an item of their own. */
#ifndef FEWB
#define FEWB 2
#endif
#ifndef MANYB
#define MANYB 2
#endif
#ifndef FEWK
#define FEWK 256
#endif
#ifndef MANYK
#define MANYK 256
#endif
constexpr int kBlocksPerCu[kAttnKinds] = { FEWB, MANYB };
constexpr int kMinKeys[kAttnKinds] = { FEWK, MANYK };

/* The fewest shared keys that are read once for all. */
constexpr int kMinShared = 256;

size_t align16(size_t v) { return (v + 15) & ~(size_t)15; }

size_t most_work(const AttnShape &s)
{
    const size_t G = (size_t)(s.heads / s.kv_heads);
    /* rows in a shared and an own segment, a partial tile for each segment, and the items that
     * spreading adds: at most kBlocksPerCu blocks per CU and kind */
    return 2 * ((size_t)s.max_tokens * G / 16) + 2 * (size_t)s.max_seq + 16384;
}

}  // namespace

size_t attn_blob_bytes(const AttnShape &s)
{
    const size_t T = (size_t)s.max_tokens;
    return align16(sizeof(AttnHdr)) + T * (sizeof(AttnTok) + sizeof(AttnVTile) + 4) + most_work(s) * sizeof(AttnWork) +
           (size_t)s.max_seq * (size_t)s.max_pages * 4 + 64;
}

std::string attn_plan(const AttnShape &s, int n_cu, int n_seq, const int *q_len, const int *kv_len, const int32_t *pages,
                      int stride, AttnPlan *p)
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
    auto segments = [&](bool share) {
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
            if (group) {
                if (keys > kv_len[i] - q_len[i]) keys = kv_len[i] - q_len[i];
                keys = keys / P * P;
                seg.push_back({ first[(size_t)i], n_tok, 0, keys, table[(size_t)i], -1, kind_of(n_tok * G), 1, 0, 0 });
            }
            for (size_t c = a; c < b; c++) {
                const int j = used[c];
                seg.push_back({ first[(size_t)j], q_len[j], group ? keys : 0, kv_len[j], table[(size_t)j],
                                kv_len[j] - q_len[j], kind_of(q_len[j] * G), 1, 0, 0 });
            }
            a = b;
        }
    };
    /* Spread each segment's keys over as many items as fill the card. */
    const size_t part_rows = attn_part_rows(s);
    auto spread = [&](int coarser) -> bool {
        int64_t work[kAttnKinds] = { 0, 0 };
        for (const Segment &g : seg) work[g.kind] += (int64_t)tiles_of(g, G) * (g.key1 - g.key0) * s.kv_heads;
        std::vector<int> parts((size_t)T, 0);
        for (Segment &g : seg) {
            const int64_t want = work[g.kind] / ((int64_t)kBlocksPerCu[g.kind] * n_cu) + 1;
            const int64_t chunk = std::max<int64_t>(want, kMinKeys[g.kind]) << coarser;
            const int64_t n = (g.key1 - g.key0 + chunk - 1) / chunk;
            const int64_t k = std::min<int64_t>(n, coarser > 20 ? 1 : kAttnSplits);
            g.chunk = round_up((int)((g.key1 - g.key0 + k - 1) / k), 64);
            g.splits = (g.key1 - g.key0 + g.chunk - 1) / g.chunk;
            g.part = parts[(size_t)g.tok];
            for (int k = 0; k < g.n_tok; k++) parts[(size_t)(g.tok + k)] = g.part + g.splits;
        }
        size_t slots = 0;
        for (int k = 0; k < (int)T; k++) {
            tok[(size_t)k].parts = parts[(size_t)k];
            tok[(size_t)k].part = (int32_t)slots;
            if (parts[(size_t)k] > 1) slots += (size_t)parts[(size_t)k];
        }
        return slots * (size_t)s.heads <= part_rows;
    };
    /* a segment follows the shared one of its tokens, so its slots come after that one's */
    bool fits = false;
    for (int share = 1; share >= 0 && !fits; share--) {
        segments(share != 0);
        for (int coarser = 0; coarser <= 21 && !fits; coarser++) fits = spread(coarser);
    }

    std::vector<AttnWork> work[kAttnKinds];
    for (const Segment &g : seg) {
        const int R = kAttnRows[g.kind], rows = g.n_tok * G;
        for (int r = 0; r < rows; r += R) {
            const int n = std::min(R, rows - r);
            /* the tile's last token sees the most keys, its first the fewest */
            const int most = g.pos < 0 ? g.key1 : g.pos + (r + n - 1) / G + 1;
            const int least = g.pos < 0 ? g.key1 : g.pos + r / G + 1;
            for (int k = 0; k < g.splits; k++) {
                const int64_t k0 = (int64_t)g.key0 + (int64_t)k * g.chunk;
                AttnWork w{};
                w.row = g.tok * G + r;
                w.rows = n;
                w.pages = g.table;
                w.key0 = (int)std::min<int64_t>(k0, g.key1 / 16 * 16);
                w.key1 = (int)std::min<int64_t>(k0 + g.chunk, most);
                if (w.key1 < w.key0 || k0 >= most) w.key1 = w.key0;        /* no keys: an empty part */
                w.full = std::min(least, w.key1);
                w.part = g.part + k;
                work[g.kind].push_back(w);
            }
        }
    }
    /* longest items first: the last ones to start end soon */
    for (auto &w : work)
        std::stable_sort(w.begin(), w.end(), [](const AttnWork &a, const AttnWork &b) { return a.key1 - a.key0 > b.key1 - b.key0; });

    std::vector<int32_t> comb;
    for (int k = 0; k < (int)T; k++)
        if (tok[(size_t)k].parts > 1) comb.push_back(k);

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
    for (const AttnTok &k : tok) h.max_parts = std::max(h.max_parts, k.parts);
    h.tok = place(tok.size() * sizeof(AttnTok));
    h.vt = place(vt.size() * sizeof(AttnVTile));
    h.comb = place(comb.size() * 4);
    for (int k = 0; k < kAttnKinds; k++) {
        h.n_work[k] = (int)work[k].size();
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
