/* qmsg_plan.h - a batch of sequences laid out as work for the attention kernels. Host code without
 * the HIP runtime: qmsg_attn_batch checks a batch and plans it here, the kernels read the result.
 *
 * Rows are (token, query head of the kv head's group), token-major: row t * G + g. A work item is a
 * tile of rows against a range of keys of one page table, for every kv head; a run is the items
 * that one block works through. Rows whose keys are spread over several items leave partial
 * results (reference maximum, sum, weighted values) in slots of their own, which the join kernel
 * takes together in slot order. */
#ifndef QMSG_PLAN_H
#define QMSG_PLAN_H

#include <stddef.h>
#include <stdint.h>

#include <string>
#include <vector>

namespace qmsg {

/* A token of the batch. */
struct AttnTok {
    int32_t pos;      /* position in its sequence: it sees keys 0 .. pos */
    int32_t dst;      /* page * page_tokens + slot of its key and value   */
    int32_t part;     /* first partial slot, where parts > 1              */
    int32_t parts;    /* items its keys are spread over (a tile's: at most) */
};

/* Up to kVTile tokens whose values go to neighbouring slots of one page. */
struct AttnVTile {
    int32_t tok, n, page, slot;
};
constexpr int kVTile = 32;

struct AttnWork {
    int32_t row, rows;      /* first row and rows of the tile                             */
    int32_t pages;          /* the page table, as an index into the batch's page ids     */
    int32_t key0, key1;     /* keys of this item (key0 a multiple of 16)                  */
    int32_t full;           /* every row sees the keys below this one                     */
    int32_t part;           /* which of its rows' partial slots it fills                  */
    int32_t next;           /* the run's next item, or -1                                 */
    int32_t joins, count;   /* items of the tile, and the counter of those that are done (the
                             * last one joins the tile's parts), or -1: the join kernel does  */
    int32_t pad[2];
};

/* Row tiles of the kernels: waves that split the keys, waves that split the rows and share the keys
 * through LDS. */
enum { kAttnFew = 0, kAttnMany = 1, kAttnKinds = 2 };
constexpr int attn_rows(int kind, int type) { return kind == kAttnFew ? 16 : type == 0 ? 64 : 128; }
constexpr int kFewWaves = 8;              /* waves of a few-row block */
/* Where the parts of a batch sit in its blob (byte offsets) and how many there are. */
struct AttnHdr {
    int32_t n_tok, n_vt, n_comb, max_parts, few_shift, n_run[kAttnKinds];      /* 1 << few_shift: waves of an item of few rows */
    int32_t tok, vt, comb, work[kAttnKinds], pages, bytes;
    /* run r of a kind starts with item r */
};

struct AttnShape {
    int heads, kv_heads, D, type, page, n_page;
    int max_seq, max_tokens, max_pages;
};

/* Partial rows (one query head of one token and slot) of a context's workspace. */
constexpr size_t kAttnPartRows = (size_t)1 << 18;
inline size_t attn_part_rows(const AttnShape &s)
{
    const size_t most = (size_t)s.max_tokens * (size_t)s.heads * 128;
    return most < kAttnPartRows ? most : kAttnPartRows;
}
/* Few rows' tiles of up to this many items are joined by the last of them, which saves a launch (us of a token
 * over 513 keys in three items 4.1 / 7.3, alone 22 / 27); its block reads what the join kernel spreads over
 * the card, which took 64 / 42 us alone for tiles of 80 rows in 16 items (kAttnMany, left to that kernel). */
constexpr int kAttnJoins = 16;
/* Counters of done items (a tile's, for each kv head). */
constexpr int kAttnCounters = 1 << 14;
/* Bytes that hold any batch of this shape. */
size_t attn_blob_bytes(const AttnShape &s);

struct AttnPlan {
    AttnHdr h{};
    std::vector<uint8_t> blob;            /* header, then the parts */
    std::vector<int64_t> owner;           /* per page: the last batch that writes it */
    int64_t batches = 0;
};

/* Sharing that saves fewer bytes than this is left: its parts need a launch of their own to be joined. us (alone,
 * host round trip included) by the MB saved, shared / not: 4.3 6.2 / 3.9 (25 / 22), 15.6 6.3 / 6.5 (26 / 23), 24.8 8.8 /
 * 10.0 (34 / 25), 33.6 6.6 / 10.1 (26 / 27), 62.9 10.0 / 14.9 (35 / 29), 66.1 10.8 / 21.5 (32 / 36). */
constexpr int64_t kMinSaved = 24 << 20;

/* Plan n_seq sequences: q_len[i] new tokens, the last of kv_len[i] tokens, on pages
 * [i * stride ..]. Returns an empty string, or what is wrong with the batch (p keeps its last). */
std::string attn_plan(const AttnShape &s, int n_cu, int n_seq, const int *q_len, const int *kv_len, const int32_t *pages,
                      int stride, AttnPlan *p, int64_t min_saved = kMinSaved);

}  // namespace qmsg

#endif /* QMSG_PLAN_H */
