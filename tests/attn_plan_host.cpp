/* The plans of attention batches (csrc/qmsg_plan.cpp) against what the kernels assume: every row sees each
 * of its keys in exactly one item, every page and slot an item touches is the batch's, parts and
 * plan stay inside their buffers.
 *
 *     attn_plan_host SEED N        N random batches; exit 0, or a line on stderr and exit 1 */
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <random>
#include <set>

#include "../large_model_amd/csrc/qmsg_plan.h"

using namespace qmsg;

#define CHECK(c)                                                                                   \
    do {                                                                                           \
        if (!(c)) { fprintf(stderr, "batch %d, line %d: %s\n", batch, __LINE__, #c); exit(1); }    \
    } while (0)

static int batch;

static void check(const AttnShape &s, int n_seq, const std::vector<int> &q, const std::vector<int> &kv, const std::vector<int32_t> &pages,
                  int stride, const AttnPlan &p, bool *shared)
{
    const AttnHdr &h = p.h;
    const int G = s.heads / s.kv_heads, P = s.page;
    CHECK(p.blob.size() == (size_t)h.bytes && p.blob.size() <= attn_blob_bytes(s) && !memcmp(p.blob.data(), &h, sizeof h));
    const AttnTok *tok = (const AttnTok *)(p.blob.data() + h.tok);
    const AttnVTile *vt = (const AttnVTile *)(p.blob.data() + h.vt);
    const int32_t *comb = (const int32_t *)(p.blob.data() + h.comb), *ids = (const int32_t *)(p.blob.data() + h.pages);
    const int n_ids = (h.bytes - h.pages) / 4;
    std::vector<int> seq;
    for (int i = 0; i < n_seq; i++)
        for (int k = 0; k < q[i]; k++) {
            const int t = (int)seq.size(), pos = kv[i] - q[i] + k;
            seq.push_back(i);
            CHECK(tok[t].pos == pos && tok[t].dst == pages[(size_t)i * stride + pos / P] * P + pos % P);
        }
    const int T = (int)seq.size();
    CHECK(h.n_tok == T);
    /* values: each token once, runs in one page */
    std::vector<int> seen((size_t)T, 0);
    for (int i = 0; i < h.n_vt; i++)
        for (int k = 0; k < vt[i].n; k++) {
            CHECK(vt[i].n <= kVTile && vt[i].tok + k < T && vt[i].slot + vt[i].n <= P);
            CHECK(tok[vt[i].tok + k].dst == vt[i].page * P + vt[i].slot + k);
            seen[(size_t)(vt[i].tok + k)]++;
        }
    for (int v : seen) CHECK(v == 1);
    /* parts: ranges of their own, as many as the workspace has */
    size_t slots = 0;
    std::set<int> apart(comb, comb + h.n_comb);
    CHECK((int)apart.size() == h.n_comb);
    for (int t = 0; t < T; t++) {
        CHECK(tok[t].parts >= 1);
        if (tok[t].parts == 1) continue;
        CHECK(tok[t].part == (int)slots);
        slots += (size_t)tok[t].parts;
    }
    CHECK(slots * (size_t)s.heads <= attn_part_rows(s));
    /* rows of several parts are joined: by the join kernel, or by the last of their tile's items, which
     * leaves all of them */
    std::map<int, std::vector<int>> counted;
    std::set<int> joined;
    /* items: (row, part) once; the keys of a row's items are 0 .. pos, each once, on its own pages */
    std::set<std::pair<int, int>> parts;
    std::map<int, std::vector<std::pair<int, int>>> ranges;
    for (int kind = 0; kind < kAttnKinds; kind++) {
        const AttnWork *w = (const AttnWork *)(p.blob.data() + h.work[kind]);
        const int n_item = ((kind + 1 < kAttnKinds ? h.work[kind + 1] : h.pages) - h.work[kind]) / (int)sizeof(AttnWork);
        std::vector<int> reached;
        for (int r = 0; r < h.n_run[kind]; r++)
            for (int i = r; i >= 0; i = w[i].next) {
                CHECK(i < n_item && (i == r) == (i < h.n_run[kind]) && (int)reached.size() < n_item);
                reached.push_back(i);
            }
        CHECK((int)reached.size() == n_item);
        /* fewer waves an item only for items that are a run and a tile each */
        CHECK(h.few_shift >= 0 && 1 << h.few_shift <= kFewWaves);
        if (kind == kAttnFew && 1 << h.few_shift < kFewWaves)
            for (int i : reached) CHECK(w[i].next < 0 && w[i].count < 0 && w[i].joins == 1);
        for (int i : reached) {
            CHECK(w[i].rows > 0 && w[i].rows <= attn_rows(kind, s.type) && w[i].row >= 0 && w[i].row + w[i].rows <= T * G);
            CHECK(w[i].key0 >= 0 && w[i].key0 % 16 == 0 && w[i].key1 >= w[i].key0 && w[i].full <= w[i].key1);
            CHECK(w[i].key1 == w[i].key0 || w[i].pages + (w[i].key1 - 1) / P < n_ids);
            if (w[i].count >= 0) {
                CHECK((w[i].count + 1) * s.kv_heads <= kAttnCounters && w[i].joins <= kAttnJoins);
                auto &v = counted[w[i].count];
                v.push_back(w[i].part);
                if (v.size() == 1) v.push_back(w[i].row);
                CHECK(v[1] == w[i].row && (int)v.size() <= w[i].joins + 1);
                if ((int)v.size() == w[i].joins + 1)
                    for (int r = w[i].row; r < w[i].row + w[i].rows; r++) {
                        CHECK(tok[r / G].parts <= w[i].joins && joined.insert(r).second);
                        std::set<int> all(v.begin() + 2, v.end());
                        all.insert(v[0]);
                        for (int k = 0; k < tok[r / G].parts; k++) CHECK(all.count(k));
                    }
            }
            const int s0 = seq[(size_t)(w[i].row / G)], s1 = seq[(size_t)((w[i].row + w[i].rows - 1) / G)];
            if (s0 != s1) *shared = true;
            for (int r = w[i].row; r < w[i].row + w[i].rows; r++) {
                const int t = r / G, sq = seq[(size_t)t], lim = std::min(tok[t].pos + 1, w[i].key1);
                /* a row of a token that another tile gives fewer parts leaves an empty item's */
                CHECK(w[i].part >= 0 && (w[i].part < tok[t].parts || w[i].key1 == w[i].key0));
                if (w[i].part >= tok[t].parts) continue;
                CHECK(parts.insert({ r, w[i].part }).second);
                CHECK(w[i].full <= tok[t].pos + 1);
                if (lim <= w[i].key0) continue;
                ranges[r].push_back({ w[i].key0, lim });
                for (int k = w[i].key0 / P; k <= (lim - 1) / P; k++) CHECK(ids[w[i].pages + k] == pages[(size_t)sq * stride + k]);
            }
        }
    }
    size_t total = 0;
    for (int r = 0; r < T * G; r++) {
        auto &v = ranges[r];
        std::sort(v.begin(), v.end());
        int at = 0;
        for (auto &x : v) {
            CHECK(x.first == at);
            at = x.second;
        }
        CHECK(at == tok[r / G].pos + 1);
        total += (size_t)tok[r / G].parts;
    }
    CHECK(parts.size() == total);
    for (int r = 0; r < T * G; r++) CHECK(tok[r / G].parts == 1 || joined.count(r) || apart.count(r / G));
}

int main(int argc, char **argv)
{
    std::mt19937 rng((unsigned)atoi(argc > 1 ? argv[1] : "0"));
    auto pick = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    int n_shared = 0, n_waves[4] = { 0, 0, 0, 0 };
    for (batch = 0; batch < atoi(argc > 2 ? argv[2] : "1"); batch++) {
        static const int kHeads[][2] = { { 1, 1 }, { 14, 2 }, { 16, 16 }, { 32, 4 }, { 64, 4 }, { 6, 2 } };
        const int *hd = kHeads[pick(0, 5)];
        AttnShape s{ hd[0], hd[1], 128, pick(0, 1), 16 << pick(0, 4), 0, pick(1, 24), 0, 0 };
        const int n_seq = pick(0, s.max_seq), mode = pick(0, 3), most = pick(0, 1) ? 40 : 5000;
        std::vector<int> q, kv;
        const int shared = mode == 3 ? pick(0, most / s.page) : 0;
        for (int i = 0; i < n_seq; i++) {
            q.push_back(mode == 0 ? 1 : mode == 1 ? pick(0, 6) : mode == 2 ? pick(0, 300) : pick(0, 2));
            kv.push_back(q.back() + shared * s.page + (pick(0, 3) ? pick(0, most) : 0));
        }
        int need = 1, T = 0;
        for (int i = 0; i < n_seq; i++) {
            need = std::max(need, (kv[i] + s.page - 1) / s.page);
            T += q[i];
        }
        s.max_pages = need + pick(0, 2);
        s.max_tokens = std::max(1, T + pick(0, 3));
        const int stride = need + pick(0, 3);
        s.n_page = shared + n_seq * need + 1;
        std::vector<int32_t> deal((size_t)s.n_page), pages((size_t)std::max(1, n_seq) * stride, -1);
        for (int i = 0; i < s.n_page; i++) deal[(size_t)i] = i;
        std::shuffle(deal.begin(), deal.end(), rng);
        int at = shared;
        for (int i = 0; i < n_seq; i++)
            for (int j = 0; j < (kv[i] + s.page - 1) / s.page; j++)
                pages[(size_t)i * stride + j] = j < shared && !(batch % 2 && i > n_seq / 2 && j > shared / 2) ? deal[(size_t)j] : deal[(size_t)at++];
        AttnPlan p;
        const int64_t min_saved = batch % 4 ? 0 : kMinSaved;       /* small batches share too, or few do */
        const std::string err = attn_plan(s, pick(0, 1) ? 256 : 4, n_seq, q.data(), kv.data(), pages.data(), stride, &p, min_saved);
        if (!err.empty()) fprintf(stderr, "%s\n", err.c_str());
        CHECK(err.empty());
        bool sh = false;
        check(s, n_seq, q, kv, pages, stride, p, &sh);
        n_shared += sh;
        if (p.h.n_run[kAttnFew]) n_waves[p.h.few_shift]++;
        /* what is wrong with a batch leaves the plan as it was */
        const std::vector<uint8_t> before = p.blob;
        int seq_bad = -1;
        for (int i = 0; i < n_seq; i++)
            if (q[i]) seq_bad = i;
        if (seq_bad < 0) continue;
        auto bad = [&](std::vector<int> q2, std::vector<int> kv2, std::vector<int32_t> pg2) {
            CHECK(!attn_plan(s, 256, n_seq, q2.data(), kv2.data(), pg2.data(), stride, &p).empty() && p.blob == before);
        };
        auto q2 = q, kv2 = kv;
        auto pg2 = pages;
        kv2[(size_t)seq_bad] = q[(size_t)seq_bad] - 1;
        bad(q, kv2, pages);
        q2[(size_t)seq_bad] = -1;
        bad(q2, kv, pages);
        kv2[(size_t)seq_bad] = s.max_pages * s.page + 1;
        bad(q, kv2, pages);
        q2 = q;
        q2[(size_t)seq_bad] += s.max_tokens;
        kv2[(size_t)seq_bad] = kv[(size_t)seq_bad] + s.max_tokens;
        bad(q2, kv2, pages);
        int32_t &last = pg2[(size_t)seq_bad * stride + (kv[(size_t)seq_bad] - 1) / s.page];
        last = -1;
        bad(q, kv, pg2);
        last = s.n_page;
        bad(q, kv, pg2);
        for (int i = 0; i < seq_bad; i++)
            if (q[(size_t)i]) {
                last = pages[(size_t)i * stride + (kv[(size_t)i] - 1) / s.page];
                bad(q, kv, pg2);
            }
        CHECK(attn_plan(s, 256, n_seq, q.data(), kv.data(), pages.data(), stride, &p).empty());
    }
    printf("%d batches, %d with a shared prefix, %d %d %d %d with items of 1 2 4 8 waves\n", batch, n_shared, n_waves[0], n_waves[1], n_waves[2], n_waves[3]);
    return 0;
}
