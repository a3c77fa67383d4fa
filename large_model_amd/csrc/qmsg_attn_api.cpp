/* qmsg_attn_api.cpp - the C ABI of the attention: caches, batches, the append and the attention itself. */
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>

#include "qmsg_ctx.h"
#include "qmsg_gguf.h"

using namespace qmsg;

namespace {

/* Bytes of a cache's keys that are taken: more than a card has, and layers of any page fit 64 bits below it. */
constexpr uint64_t kMostBytes = 1ull << 48;

uint64_t page_bytes_of(const qmsg_attn_cfg &f)
{
    return (uint64_t)f.n_head_kv * (uint64_t)f.page_tokens * (uint64_t)f.head_dim * (f.type == QMSG_T_F16 ? 2 : 4);
}

/* The scores' scale for exponents of two. */
float log2_scale(const qmsg_attn_cfg &f)
{
    return (float)((f.scale > 0.0f ? (double)f.scale : 1.0 / std::sqrt((double)f.head_dim)) * 1.4426950408889634);
}

/* Whether the kernels take this configuration; 0 and the reason otherwise. */
int check_cfg(const qmsg_attn_cfg &f, const char **why)
{
    *why = nullptr;
    if (f.n_head <= 0 || f.n_head_kv <= 0 || f.n_head % f.n_head_kv || f.n_page <= 0 || f.n_layer <= 0 || f.max_seq <= 0 ||
        f.max_tokens <= 0 || f.max_pages <= 0 || (f.qk_norm != 0 && f.qk_norm != 1)) {
        *why = "bad shape";
        return QMSG_E_INVALID;
    }
    if (!(f.rope_base > 0.0f) || !std::isfinite(f.rope_base) || !(f.scale >= 0.0f) || (f.scale > 0.0f && !std::isfinite(log2_scale(f)))) {
        *why = "rope_base must be positive and scale not negative, both finite";
        return QMSG_E_INVALID;
    }
    if (f.type != QMSG_T_F16 && f.type != QMSG_T_F32) *why = "cache types are F16 and F32";
    else if (f.head_dim != 64 && f.head_dim != 128) *why = "head_dim is 64 or 128";
    else if (f.page_tokens < 16 || f.page_tokens > 256 || (f.page_tokens & (f.page_tokens - 1))) *why = "page_tokens is a power of two from 16 to 256";
    else if (f.n_head > 1024) *why = "more than 1024 heads";
    else if ((int64_t)f.n_page * f.page_tokens > INT32_MAX || (int64_t)f.max_pages * f.page_tokens > INT32_MAX ||
             (int64_t)f.max_tokens * f.n_head > INT32_MAX)
        *why = "tokens of the pool, tokens of a sequence and rows of a batch are 32-bit";
    else if ((int64_t)f.max_seq * f.max_pages > 1 << 28) *why = "page tables above 2^28 pages";
    else if (f.n_layer > 1 << 16) *why = "more than 65536 layers";
    else if ((uint64_t)f.n_page * page_bytes_of(f) > kMostBytes / (uint64_t)f.n_layer) *why = "keys above 2^48 bytes";
    return *why ? QMSG_E_UNSUPPORTED : QMSG_OK;
}

AttnShape shape_of(const qmsg_attn_cfg &f)
{
    return { f.n_head, f.n_head_kv, f.head_dim, f.type, f.page_tokens, f.n_page, f.max_seq, f.max_tokens, f.max_pages };
}

AttnStore *find_attn(qmsg_ctx *c, int id, int layer, const char *what, int *rc)
{
    if (id < 0 || id >= (int)c->attns.size()) {
        *rc = fail(c, QMSG_E_INVALID, "%s: attention id %d unknown", what, id);
        return nullptr;
    }
    AttnStore *a = c->attns[(size_t)id].get();
    if (layer < 0 || layer >= a->cfg.n_layer) {
        *rc = fail(c, QMSG_E_RANGE, "%s: layer %d outside [0, %d)", what, layer, a->cfg.n_layer);
        return nullptr;
    }
    return a;
}

bool overlap(const float *a, size_t na, const float *b, size_t nb) { return a < b + nb && b < a + na; }

/* The device's copy of the batch: pinned plan, copied in stream order. */
int send_plan(qmsg_ctx *c, AttnStore &a, const AttnPlan &plan)
{
    const int k = a.next;
    HIP_TRY(c, hipEventSynchronize(a.copied[k]));
    memcpy(a.pin[k], plan.blob.data(), plan.blob.size());
    HIP_TRY(c, hipMemcpyAsync(a.blob, a.pin[k], plan.blob.size(), hipMemcpyHostToDevice, c->stream));
    HIP_TRY(c, hipEventRecord(a.copied[k], c->stream));
    a.next ^= 1;
    return QMSG_OK;
}

/* Fill what every kernel of a call on the batch needs. A captured call reads the batch's header when
 * it runs. */
int make_call(qmsg_ctx *c, const AttnStore &a, int layer, AttnCall *o)
{
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    HIP_TRY(c, hipStreamIsCapturing(c->stream, &cap));
    AttnCall k{};
    k.h = a.plan.h;
    k.live = cap != hipStreamCaptureStatusNone;
    k.blob = a.blob;
    k.k = a.k + (uint64_t)layer * a.layer_bytes;
    k.v = a.v + (uint64_t)layer * a.layer_bytes;
    k.page_bytes = a.page_bytes;
    k.shift = __builtin_ctz((unsigned)a.cfg.page_tokens);
    k.heads = a.cfg.n_head;
    k.kv_heads = a.cfg.n_head_kv;
    k.group = a.cfg.n_head / a.cfg.n_head_kv;
    k.scale_log2 = log2_scale(a.cfg);
    k.done = a.done;
    k.part_o = a.part_o;
    k.part_ml = a.part_ml;
    *o = k;
    return QMSG_OK;
}

/* Blocks of a captured launch: its kernels loop over what the batch then holds. */
int live_grid(const qmsg_ctx *c) { return 4 * c->n_cu; }

}  // namespace

void qmsg::attn_release(AttnStore &a)
{
    for (int k = 0; k < 2; k++) {
        if (a.copied[k]) hipEventDestroy(a.copied[k]);
        if (a.pin[k]) hipHostFree(a.pin[k]);
        a.copied[k] = nullptr;
        a.pin[k] = nullptr;
    }
    for (AttnLayer &l : a.layers) {
        hipFree(l.qw);
        hipFree(l.kw);
        hipFree(l.norm);
    }
    a.layers.clear();
    for (void *p : a.allocs) hipFree(p);
    a.allocs.clear();
}

/* No exception leaves a C entry point: those of the host containers are reported as memory. */
#define NO_THROW(c, what, ...)                                                              \
    try {                                                                                   \
        __VA_ARGS__                                                                         \
    } catch (...) {                                                                         \
        return fail((c), QMSG_E_NOMEM, "%s: out of host memory", (what));                   \
    }

extern "C" {

uint64_t qmsg_attn_cache_bytes(const qmsg_attn_cfg *f)
{
    const char *why;
    if (!f || check_cfg(*f, &why) != QMSG_OK) return 0;
    return (uint64_t)f->n_layer * (uint64_t)f->n_page * page_bytes_of(*f);
}

static int attn_new(qmsg_ctx *c, const qmsg_attn_cfg &f, void *d_k, void *d_v, AttnStore &a)
{
    a.cfg = f;
    a.shape = shape_of(f);
    a.page_bytes = (uint32_t)page_bytes_of(f);
    a.layer_bytes = (uint64_t)f.n_page * a.page_bytes;
    a.layers.resize((size_t)f.n_layer);
    const size_t bytes = (size_t)f.n_layer * a.layer_bytes, blob = attn_blob_bytes(a.shape), rows = attn_part_rows(a.shape);
    int rc;
    a.k = (uint8_t *)d_k;
    a.v = (uint8_t *)d_v;
    if (!d_k && ((rc = dev_alloc(c, (void **)&a.k, bytes, a.allocs)) || (rc = dev_alloc(c, (void **)&a.v, bytes, a.allocs)))) return rc;
    const int n = f.head_dim / 2;
    if ((rc = dev_alloc(c, (void **)&a.freq, (size_t)n * 8, a.allocs)) || (rc = dev_alloc(c, (void **)&a.blob, blob, a.allocs)) ||
        (rc = dev_alloc(c, (void **)&a.part_o, rows * (size_t)f.head_dim * 4, a.allocs)) ||
        (rc = dev_alloc(c, (void **)&a.part_ml, rows * 8, a.allocs)) ||
        (rc = dev_alloc(c, (void **)&a.done, kAttnCounters * 4, a.allocs)))
        return rc;
    HIP_TRY(c, hipMemset(a.done, 0, kAttnCounters * 4));
    double freq[64];
    for (int i = 0; i < n; i++) freq[i] = std::pow((double)f.rope_base, -(double)i / n) / 6.283185307179586476925;
    HIP_TRY(c, hipMemcpy(a.freq, freq, (size_t)n * 8, hipMemcpyHostToDevice));
    for (int k = 0; k < 2; k++) {
        if (hipHostMalloc((void **)&a.pin[k], blob, hipHostMallocDefault) != hipSuccess) {
            a.pin[k] = nullptr;
            (void)hipGetLastError();
            return fail(c, QMSG_E_NOMEM, "qmsg_attn_create: pinned buffer of %zu bytes", blob);
        }
        HIP_TRY(c, hipEventCreateWithFlags(&a.copied[k], hipEventDisableTiming));
    }
    /* an empty batch, so that a call before the first one has nothing to do */
    const std::string err = attn_plan(a.shape, c->n_cu, 0, nullptr, nullptr, nullptr, 0, &a.plan);
    if (!err.empty()) return fail(c, QMSG_E_INVALID, "qmsg_attn_create: %s", err.c_str());
    HIP_TRY(c, hipMemcpy(a.blob, a.plan.blob.data(), a.plan.blob.size(), hipMemcpyHostToDevice));
    return QMSG_OK;
}

int qmsg_attn_create(qmsg_ctx *c, const qmsg_attn_cfg *f, void *d_k, void *d_v, int *id)
{
    if (!c || !f || !id) return QMSG_E_INVALID;
    const char *why;
    const int bad = check_cfg(*f, &why);
    if (bad) return fail(c, bad, "qmsg_attn_create: %s", why);
    if (attn_blob_bytes(shape_of(*f)) > INT32_MAX) return fail(c, QMSG_E_UNSUPPORTED, "qmsg_attn_create: batches above 2 GiB of plan");
    if (!d_k != !d_v) return fail(c, QMSG_E_INVALID, "qmsg_attn_create: give both of d_k and d_v, or neither");
    if (((uintptr_t)d_k | (uintptr_t)d_v) & 15) return fail(c, QMSG_E_INVALID, "qmsg_attn_create: d_k and d_v must be 16-byte aligned");
    const uint64_t bytes = qmsg_attn_cache_bytes(f);
    if (d_k && (uintptr_t)d_k < (uintptr_t)d_v + bytes && (uintptr_t)d_v < (uintptr_t)d_k + bytes)
        return fail(c, QMSG_E_INVALID, "qmsg_attn_create: d_k and d_v overlap");
    HIP_TRY(c, hipSetDevice(c->device));
    NO_THROW(c, "qmsg_attn_create", {
        auto a = std::make_unique<AttnStore>();
        c->attns.reserve(c->attns.size() + 1);
        const int rc = attn_new(c, *f, d_k, d_v, *a);
        if (rc) {
            attn_release(*a);
            return rc;
        }
        c->attns.push_back(std::move(a));
    })
    *id = (int)c->attns.size() - 1;
    return QMSG_OK;
}

int qmsg_attn_cache(qmsg_ctx *c, int id, void **d_k, void **d_v)
{
    if (!c || !d_k || !d_v) return QMSG_E_INVALID;
    int rc = QMSG_OK;
    AttnStore *a = find_attn(c, id, 0, "qmsg_attn_cache", &rc);
    if (!a) return rc;
    *d_k = a->k;
    *d_v = a->v;
    return QMSG_OK;
}

/* n host floats to a device vector made on first use. NULL: ones, where there is one (a captured call may hold
 * it, so it stays). */
static int set_vector(qmsg_ctx *c, float **d, const float *w, size_t n)
{
    if (!w && !*d) return QMSG_OK;
    std::vector<float> ones;
    if (!w) {
        ones.assign(n, 1.0f);
        w = ones.data();
    }
    if (!*d) {
        std::vector<void *> tmp;
        const int rc = dev_alloc(c, (void **)d, n * 4, tmp);
        if (rc) return rc;
    }
    HIP_TRY(c, hipMemcpy(*d, w, n * 4, hipMemcpyHostToDevice));
    return QMSG_OK;
}

int qmsg_attn_norms(qmsg_ctx *c, int id, int layer, const float *q_norm, const float *k_norm)
{
    if (!c) return QMSG_E_INVALID;
    int rc = QMSG_OK;
    AttnStore *a = find_attn(c, id, layer, "qmsg_attn_norms", &rc);
    if (!a) return rc;
    if (!a->cfg.qk_norm) return fail(c, QMSG_E_INVALID, "qmsg_attn_norms: created without head norms (qk_norm)");
    HIP_TRY(c, hipSetDevice(c->device));
    HIP_TRY(c, hipStreamSynchronize(c->stream));
    AttnLayer &l = a->layers[(size_t)layer];
    NO_THROW(c, "qmsg_attn_norms", {
        if ((rc = set_vector(c, &l.qw, q_norm, (size_t)a->cfg.head_dim))) return rc;
        rc = set_vector(c, &l.kw, k_norm, (size_t)a->cfg.head_dim);
    })
    return rc;
}

int qmsg_attn_batch(qmsg_ctx *c, int id, int n_seq, const int *q_len, const int *kv_len, const int32_t *pages, int stride)
{
    if (!c) return QMSG_E_INVALID;
    int rc = QMSG_OK;
    AttnStore *a = find_attn(c, id, 0, "qmsg_attn_batch", &rc);
    if (!a) return rc;
    HIP_TRY(c, hipSetDevice(c->device));
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    HIP_TRY(c, hipStreamIsCapturing(c->stream, &cap));
    if (cap != hipStreamCaptureStatusNone) return fail(c, QMSG_E_INVALID, "qmsg_attn_batch: the stream is capturing (set the batch before, or between replays)");
    NO_THROW(c, "qmsg_attn_batch", {
        const std::string err = attn_plan(a->shape, c->n_cu, n_seq, q_len, kv_len, pages, stride, &a->plan);
        if (!err.empty()) return fail(c, QMSG_E_INVALID, "qmsg_attn_batch: %s", err.c_str());
        rc = send_plan(c, *a, a->plan);
        if (rc) a->plan.h = AttnHdr{};              /* no batch, rather than another than the device's */
    })
    return rc;
}

int qmsg_attn_append_device(qmsg_ctx *c, int id, int layer, float *d_qr, const float *d_q, const float *d_k, const float *d_v, float eps)
{
    if (!c) return QMSG_E_INVALID;
    int rc = QMSG_OK;
    AttnStore *a = find_attn(c, id, layer, "qmsg_attn_append_device", &rc);
    if (!a) return rc;
    if (!d_k || !d_v || !d_q != !d_qr) return fail(c, QMSG_E_INVALID, "qmsg_attn_append_device: null buffer");
    if (((uintptr_t)d_qr | (uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_v) & 15)
        return fail(c, QMSG_E_INVALID, "qmsg_attn_append_device: buffers must be 16-byte aligned");
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(c, QMSG_E_INVALID, "qmsg_attn_append_device: eps %g", (double)eps);
    const size_t T = (size_t)a->plan.h.n_tok, nq = T * (size_t)a->cfg.n_head * (size_t)a->cfg.head_dim, nk = T * (size_t)a->cfg.n_head_kv * (size_t)a->cfg.head_dim;
    if (d_q && ((d_qr != d_q && overlap(d_qr, nq, d_q, nq)) || overlap(d_qr, nq, d_k, nk) || overlap(d_qr, nq, d_v, nk)))
        return fail(c, QMSG_E_INVALID, "qmsg_attn_append_device: d_qr overlaps an input (it may only be d_q itself)");
    HIP_TRY(c, hipSetDevice(c->device));
    AttnAppend b{};
    if ((rc = make_call(c, *a, layer, &b.c))) return rc;
    if (T == 0 && !b.c.live) return QMSG_OK;
    const AttnLayer &l = a->layers[(size_t)layer];
    b.q = d_q;
    b.k = d_k;
    b.v = d_v;
    b.qr = d_qr;
    b.qw = l.qw;
    b.kw = l.kw;
    b.freq = a->freq;
    b.eps = eps;
    b.norm = a->cfg.qk_norm;
    LAUNCH(c, "append", launch_attn_append(b, a->cfg.type, a->cfg.head_dim, live_grid(c), c->stream));
    return QMSG_OK;
}

int qmsg_attn_device(qmsg_ctx *c, int id, int layer, const float *d_q, float *d_out)
{
    if (!c) return QMSG_E_INVALID;
    int rc = QMSG_OK;
    AttnStore *a = find_attn(c, id, layer, "qmsg_attn_device", &rc);
    if (!a) return rc;
    if (!d_q || !d_out) return fail(c, QMSG_E_INVALID, "qmsg_attn_device: null buffer");
    if (((uintptr_t)d_q | (uintptr_t)d_out) & 15) return fail(c, QMSG_E_INVALID, "qmsg_attn_device: buffers must be 16-byte aligned");
    const size_t n = (size_t)a->plan.h.n_tok * (size_t)a->cfg.n_head * (size_t)a->cfg.head_dim;
    if (overlap(d_out, n, d_q, n) || d_out == d_q) return fail(c, QMSG_E_INVALID, "qmsg_attn_device: d_out overlaps d_q");
    HIP_TRY(c, hipSetDevice(c->device));
    AttnCall k;
    if ((rc = make_call(c, *a, layer, &k))) return rc;
    if (n == 0 && !k.live) return QMSG_OK;
    k.q = d_q;
    k.out = d_out;
    LAUNCH(c, "attend", launch_attend(k, a->cfg.type, a->cfg.head_dim, live_grid(c), c->stream));
    return QMSG_OK;
}

/* The dense matrices of a layer's q, k, v and output products, checked against the attention's heads. */
static int check_mats(qmsg_ctx *c, const AttnStore &a, const int *ids, const char *what)
{
    const int64_t E = c->cfg.n_embd, Q = (int64_t)a.cfg.n_head * a.cfg.head_dim, KV = (int64_t)a.cfg.n_head_kv * a.cfg.head_dim;
    const struct { int64_t rows, cols; const char *name; } want[4] = { { Q, E, "q" }, { KV, E, "k" }, { KV, E, "v" }, { E, Q, "output" } };
    for (int i = 0; i < 4; i++) {
        if (ids[i] < 0 || ids[i] >= (int)c->mats.size()) return fail(c, QMSG_E_INVALID, "%s: matrix id %d unknown", what, ids[i]);
        const DenseStore &m = c->mats[(size_t)ids[i]];
        if (m.rows != want[i].rows || m.cols != want[i].cols)
            return fail(c, QMSG_E_INVALID, "%s: %s matrix is %lld x %lld, expected %lld x %lld", what, want[i].name, (long long)m.rows,
                        (long long)m.cols, (long long)want[i].rows, (long long)want[i].cols);
    }
    return QMSG_OK;
}

int qmsg_attn_mats(qmsg_ctx *c, int id, int layer, const int *ids, const float *attn_norm)
{
    if (!c || !ids) return QMSG_E_INVALID;
    int rc = QMSG_OK;
    AttnStore *a = find_attn(c, id, layer, "qmsg_attn_mats", &rc);
    if (!a) return rc;
    if ((rc = check_mats(c, *a, ids, "qmsg_attn_mats"))) return rc;
    if (rmsnorm_lds_bytes(c->cfg.n_embd) > 160 * 1024)
        return fail(c, QMSG_E_UNSUPPORTED, "qmsg_attn_mats: rows of %d floats exceed the norm's LDS", c->cfg.n_embd);
    HIP_TRY(c, hipSetDevice(c->device));
    HIP_TRY(c, hipStreamSynchronize(c->stream));
    AttnLayer &l = a->layers[(size_t)layer];
    NO_THROW(c, "qmsg_attn_mats", {
        if (!a->rows) {
            const size_t T = (size_t)a->cfg.max_tokens, Q = (size_t)a->cfg.n_head * (size_t)a->cfg.head_dim, KV = (size_t)a->cfg.n_head_kv * (size_t)a->cfg.head_dim;
            if ((rc = dev_alloc(c, (void **)&a->rows, T * (2 * (size_t)c->cfg.n_embd + 2 * Q + 2 * KV) * 4, a->allocs))) return rc;
        }
        if ((rc = set_vector(c, &l.norm, attn_norm, (size_t)c->cfg.n_embd))) return rc;
    })
    memcpy(l.mats, ids, sizeof l.mats);
    return QMSG_OK;
}

int qmsg_attn_layer(qmsg_ctx *c, int id, int layer, float *d_h, float eps)
{
    if (!c) return QMSG_E_INVALID;
    int rc = QMSG_OK;
    AttnStore *a = find_attn(c, id, layer, "qmsg_attn_layer", &rc);
    if (!a) return rc;
    const AttnLayer &l = a->layers[(size_t)layer];
    if (l.mats[0] < 0) return fail(c, QMSG_E_INVALID, "qmsg_attn_layer: layer %d has no matrices", layer);
    if (!d_h || ((uintptr_t)d_h & 15)) return fail(c, QMSG_E_INVALID, "qmsg_attn_layer: d_h must be 16-byte aligned");
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(c, QMSG_E_INVALID, "qmsg_attn_layer: eps %g", (double)eps);
    const int T = a->plan.h.n_tok, E = c->cfg.n_embd;
    if (T == 0) return QMSG_OK;
    HIP_TRY(c, hipSetDevice(c->device));
    const size_t t = (size_t)T, Q = (size_t)a->cfg.n_head * (size_t)a->cfg.head_dim, KV = (size_t)a->cfg.n_head_kv * (size_t)a->cfg.head_dim;
    float *x = a->rows, *q = x + t * (size_t)E, *k = q + t * Q, *v = k + t * KV, *out = v + t * KV, *o = out + t * Q;
    LAUNCH(c, "rmsnorm", launch_rmsnorm(d_h, nullptr, l.norm, x, T, E, eps, c->norm_walk, c->d_walked, c->stream));
    float *const ys[3] = { q, k, v };
    float *const yo[1] = { o };
    NO_THROW(c, "qmsg_attn_layer", {
        if ((rc = qmsg_matmul_n_device(c, l.mats, 3, x, T, ys))) return rc;
        if ((rc = qmsg_attn_append_device(c, id, layer, q, q, k, v, eps))) return rc;
        if ((rc = qmsg_attn_device(c, id, layer, q, out))) return rc;
        if ((rc = qmsg_matmul_n_device(c, l.mats + 3, 1, out, T, yo))) return rc;
    })
    LAUNCH(c, "add", launch_add_rows(d_h, o, t * (size_t)E, c->stream));
    return QMSG_OK;
}

int qmsg_gguf_attn_cfg(const qmsg_gguf *g, qmsg_attn_cfg *f)
{
    if (!g || !f) return QMSG_E_INVALID;
    qmsg_cfg moe;
    int n_layer = 0;
    int rc = qmsg_gguf_moe_cfg(g, &moe, &n_layer, nullptr);
    if (rc) return rc;
    int64_t v[2];
    const char *names[2] = { "qwen3moe.attention.head_count", "qwen3moe.attention.head_count_kv" };
    for (int i = 0; i < 2; i++) {
        if ((rc = qmsg_gguf_get_int(g, names[i], &v[i]))) return rc;
        if (v[i] <= 0 || v[i] > 1 << 20) return fail(nullptr, QMSG_E_INVALID, "qmsg_gguf_attn_cfg: %s = %lld", names[i], (long long)v[i]);
    }
    int64_t dk = moe.n_embd / v[0], dv;
    if (g->scalar("qwen3moe.attention.key_length") && (rc = qmsg_gguf_get_int(g, "qwen3moe.attention.key_length", &dk))) return rc;
    dv = dk;
    if (g->scalar("qwen3moe.attention.value_length") && (rc = qmsg_gguf_get_int(g, "qwen3moe.attention.value_length", &dv))) return rc;
    if (dk != dv || dk <= 0 || dk > 1 << 20)
        return fail(nullptr, QMSG_E_UNSUPPORTED, "qmsg_gguf_attn_cfg: key_length %lld, value_length %lld", (long long)dk, (long long)dv);
    /* rotations that the kernels do not have: of a part of the head, at stretched positions */
    int64_t n_rot = dk;
    if (g->scalar("qwen3moe.rope.dimension_count") && (rc = qmsg_gguf_get_int(g, "qwen3moe.rope.dimension_count", &n_rot))) return rc;
    if (n_rot != dk) return fail(nullptr, QMSG_E_UNSUPPORTED, "qmsg_gguf_attn_cfg: rope.dimension_count %lld of heads of %lld", (long long)n_rot, (long long)dk);
    char how[16] = "none";
    if (g->scalar("qwen3moe.rope.scaling.type") && (rc = qmsg_gguf_get_str(g, "qwen3moe.rope.scaling.type", how, sizeof how))) return rc;
    if (strcmp(how, "none")) return fail(nullptr, QMSG_E_UNSUPPORTED, "qmsg_gguf_attn_cfg: rope.scaling.type %s", how);
    double base = 10000.0;
    if (g->scalar("qwen3moe.rope.freq_base") && (rc = qmsg_gguf_get_float(g, "qwen3moe.rope.freq_base", &base))) return rc;
    f->n_head = (int)v[0];
    f->n_head_kv = (int)v[1];
    f->head_dim = (int)dk;
    f->n_layer = n_layer;
    f->qk_norm = 1;
    f->rope_base = (float)base;
    return QMSG_OK;
}

int qmsg_gguf_attn_upload(qmsg_ctx *c, const qmsg_gguf *g, int id, int first, int n)
{
    if (!c || !g || n < 0) return QMSG_E_INVALID;
    int rc = QMSG_OK;
    AttnStore *a = find_attn(c, id, 0, "qmsg_gguf_attn_upload", &rc);
    if (!a) return rc;
    if (first < 0 || first > a->cfg.n_layer - n)
        return fail(c, QMSG_E_RANGE, "layers %d .. %d outside [0, %d)", first, first + n - 1, a->cfg.n_layer);
    const int64_t E = c->cfg.n_embd, D = a->cfg.head_dim, Q = a->cfg.n_head * D, KV = a->cfg.n_head_kv * D;
    const struct { const char *name; int64_t ne0, ne1; } want[7] = {
        { "attn_q", E, Q }, { "attn_k", E, KV }, { "attn_v", E, KV }, { "attn_output", Q, E }, { "attn_norm", E, 1 }, { "attn_q_norm", D, 1 }, { "attn_k_norm", D, 1 } };
    const int n_vec = a->cfg.qk_norm ? 3 : 1;
    NO_THROW(c, "qmsg_gguf_attn_upload", {
        /* every layer's tensors are checked before any device memory changes */
        std::vector<const qmsg_tensor *> t((size_t)n * 7, nullptr);
        for (int l = 0; l < n; l++)
            for (int k = 0; k < 4 + n_vec; k++) {
                char name[96];
                snprintf(name, sizeof name, "blk.%d.%s.weight", first + l, want[k].name);
                const int i = gguf_find(g, name);
                if (i < 0) return fail(c, QMSG_E_INVALID, "model: missing tensor %s", name);
                const qmsg_tensor &x = g->tensors[(size_t)i];
                if (x.ne[0] != want[k].ne0 || x.ne[1] != want[k].ne1 || x.ne[2] != 1 || x.ne[3] != 1)
                    return fail(c, QMSG_E_INVALID, "model: %s expected [%lld x %lld], got ne=[%lld,%lld,%lld]", name, (long long)want[k].ne0,
                                (long long)want[k].ne1, (long long)x.ne[0], (long long)x.ne[1], (long long)x.ne[2]);
                if (k >= 4 && x.type != QMSG_T_F32) return fail(c, QMSG_E_UNSUPPORTED, "%s: norms are F32 (got type %d)", name, x.type);
                t[(size_t)l * 7 + (size_t)k] = &x;
            }
        std::vector<float> vec[3];
        for (int l = 0; l < n; l++) {
            int ids[4];
            for (int k = 0; k < 4; k++)
                if ((rc = qmsg_gguf_upload_mat(c, g, t[(size_t)l * 7 + (size_t)k]->name, &ids[k]))) return rc;
            for (int k = 0; k < n_vec; k++) {
                const qmsg_tensor &x = *t[(size_t)l * 7 + 4 + (size_t)k];
                vec[k].resize((size_t)x.ne[0]);
                if (gguf_pread(g, x.shard, x.off, (uint64_t)x.ne[0] * 4, vec[k].data()))
                    return fail(c, QMSG_E_INVALID, "gguf upload: read failed for %s", x.name);
            }
            if ((rc = qmsg_attn_mats(c, id, first + l, ids, vec[0].data()))) return rc;
            if (n_vec == 3 && (rc = qmsg_attn_norms(c, id, first + l, vec[1].data(), vec[2].data()))) return rc;
        }
    })
    return QMSG_OK;
}

}  // extern "C"
