/* qmsg_attn_api.cpp - the C ABI of the attention: caches, batches, the append and the attention itself. */
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>

#include "qmsg_ctx.h"

using namespace qmsg;

namespace {

uint64_t page_bytes_of(const qmsg_attn_cfg &f)
{
    return (uint64_t)f.n_head_kv * (uint64_t)f.page_tokens * (uint64_t)f.head_dim * (f.type == QMSG_T_F16 ? 2 : 4);
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
    if (!(f.rope_base > 0.0f) || !std::isfinite(f.rope_base) || !(f.scale >= 0.0f) || !std::isfinite(f.scale)) {
        *why = "rope_base must be positive and scale not negative";
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
    k.scale_log2 = (float)((a.cfg.scale > 0.0f ? (double)a.cfg.scale : 1.0 / std::sqrt((double)a.cfg.head_dim)) * 1.4426950408889634);
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

/* n host floats to a device vector made on first use; NULL frees it (unit weights). */
static int set_vector(qmsg_ctx *c, float **d, const float *w, size_t n)
{
    if (!w) {
        hipFree(*d);
        *d = nullptr;
        return QMSG_OK;
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

}  // extern "C"
