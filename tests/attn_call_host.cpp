/* Host side of the attention's calls (csrc/qmsg_attn_api.cpp) against a small stand-in for the HIP runtime and the
 * launchers: what is refused and with which status, that a refusal changes nothing and launches nothing, memory that
 * runs out, and what a captured call is given.
 *
 *     attn_call_host SCENARIO        exit 0, or a line on stderr and exit 1 */
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>
#include <string>
#include <vector>

#include "../include/qmsg.h"
#include "../large_model_amd/csrc/qmsg_ctx.h"

namespace {

std::set<void *> live;                 /* device and pinned memory, events */
int fail_at = -1, allocs = 0, set_devices = 0;
hipError_t last = hipSuccess;
bool capturing = false, copy_fails = false;
std::vector<qmsg::AttnCall> attends;
std::vector<qmsg::AttnAppend> appends;
struct Step {
    const char *name;
    const float *in;
    float *out;
    int n;
    const float *w;
};
std::vector<Step> steps;

hipError_t ret(hipError_t e)
{
    if (e != hipSuccess) last = e;
    return e;
}
hipError_t take(void **p, size_t n)
{
    if (allocs++ == fail_at) return ret(hipErrorOutOfMemory);
    *p = calloc(1, n < 65536 ? 65536 : n < (1u << 24) ? n : 64);
    live.insert(*p);
    return hipSuccess;
}
void drop(void *p)
{
    if (!p) return;
    if (!live.erase(p)) { fprintf(stderr, "freed twice\n"); exit(1); }
    free(p);
}

}  // namespace

extern "C" {
hipError_t hipMalloc(void **p, size_t n) { return take(p, n); }
hipError_t hipFree(void *p) { drop(p); return hipSuccess; }
hipError_t hipHostMalloc(void **p, size_t n, unsigned) { return take(p, n); }
hipError_t hipHostFree(void *p) { drop(p); return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t *e, unsigned) { return take((void **)e, 64); }
hipError_t hipEventDestroy(hipEvent_t e) { drop(e); return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipGetLastError() { const hipError_t e = last; last = hipSuccess; return e; }
const char *hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipGetDeviceCount(int *n) { *n = 1; return hipSuccess; }
hipError_t hipSetDevice(int) { set_devices++; return hipSuccess; }
hipError_t hipDeviceGetAttribute(int *v, hipDeviceAttribute_t, int) { *v = 256; return hipSuccess; }
hipError_t hipGetSymbolAddress(void **p, const void *s) { *p = (void *)s; return hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t *s, unsigned) { *s = (hipStream_t)8; return hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return capturing ? ret(hipErrorStreamCaptureUnsupported) : hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s)
{
    *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipMemset(void *, int, size_t) { return hipSuccess; }
hipError_t hipMemcpy(void *, const void *, size_t, hipMemcpyKind) { return hipSuccess; }
hipError_t hipMemcpyAsync(void *d, const void *s, size_t n, hipMemcpyKind, hipStream_t)
{
    if (copy_fails) return ret(hipErrorInvalidValue);
    memcpy(d, s, n);
    return hipSuccess;
}
}

namespace qmsg {
thread_local const LaunchTimer *g_launch_timer = nullptr;
hipError_t launch_attend(const AttnCall &a, int, int, int, hipStream_t) { attends.push_back(a); return hipGetLastError(); }
hipError_t launch_rmsnorm(float *x, const float *, const float *w, float *y, int T, int E, float, int, unsigned long long *, hipStream_t)
{
    steps.push_back({ "rmsnorm", x, y, T * E, w });
    return hipGetLastError();
}
hipError_t launch_add_rows(float *h, const float *d, size_t n, hipStream_t)
{
    steps.push_back({ "add", d, h, (int)n, nullptr });
    return hipGetLastError();
}
hipError_t launch_dense(const DenseArgs &a, int, uint8_t *, uint64_t, bool *, hipStream_t)
{
    for (int i = 0; i < a.nm; i++) steps.push_back({ "dense", a.x, a.m[i].y, a.T * a.m[i].rows, nullptr });
    return hipGetLastError();
}
hipError_t launch_attn_append(const AttnAppend &b, int, int, int, hipStream_t) { appends.push_back(b); return hipGetLastError(); }
}  // namespace qmsg

#define CHECK(c)                                                                     \
    do {                                                                             \
        if (!(c)) { fprintf(stderr, "line %d: %s (%s)\n", __LINE__, #c, qmsg_last_error(ctx)); exit(1); } \
    } while (0)

static qmsg_ctx *ctx;

static qmsg_attn_cfg config()
{
    qmsg_attn_cfg f{};
    f.n_head = 8;
    f.n_head_kv = 2;
    f.head_dim = 64;
    f.type = QMSG_T_F16;
    f.page_tokens = 16;
    f.n_page = 32;
    f.n_layer = 2;
    f.max_seq = 3;
    f.max_tokens = 20;
    f.max_pages = 8;
    f.qk_norm = 1;
    f.rope_base = 1e4f;
    return f;
}

static float *const kQ = (float *)(1ull << 20), *const kQr = (float *)(2ull << 20), *const kK = (float *)(3ull << 20), *const kV = (float *)(4ull << 20);

static void configs()
{
    int id = -1;
    auto expect = [&](int rc, auto change) {
        qmsg_attn_cfg f = config();
        change(f);
        const size_t before = live.size();
        CHECK(qmsg_attn_create(ctx, &f, nullptr, nullptr, &id) == rc && live.size() == before);
        CHECK(qmsg_attn_cache_bytes(&f) == 0);
    };
    const int kInts[] = { 0, -1 };
    for (int v : kInts) {
        expect(QMSG_E_INVALID, [&](qmsg_attn_cfg &f) { f.n_head = v; });
        expect(QMSG_E_INVALID, [&](qmsg_attn_cfg &f) { f.n_head_kv = v; });
        expect(QMSG_E_INVALID, [&](qmsg_attn_cfg &f) { f.n_page = v; });
        expect(QMSG_E_INVALID, [&](qmsg_attn_cfg &f) { f.n_layer = v; });
        expect(QMSG_E_INVALID, [&](qmsg_attn_cfg &f) { f.max_seq = v; });
        expect(QMSG_E_INVALID, [&](qmsg_attn_cfg &f) { f.max_tokens = v; });
        expect(QMSG_E_INVALID, [&](qmsg_attn_cfg &f) { f.max_pages = v; });
    }
    expect(QMSG_E_INVALID, [](qmsg_attn_cfg &f) { f.n_head = 9; });
    expect(QMSG_E_INVALID, [](qmsg_attn_cfg &f) { f.qk_norm = 2; });
    expect(QMSG_E_INVALID, [](qmsg_attn_cfg &f) { f.rope_base = 0.0f; });
    expect(QMSG_E_INVALID, [](qmsg_attn_cfg &f) { f.rope_base = NAN; });
    expect(QMSG_E_INVALID, [](qmsg_attn_cfg &f) { f.rope_base = INFINITY; });
    expect(QMSG_E_INVALID, [](qmsg_attn_cfg &f) { f.scale = -1.0f; });
    expect(QMSG_E_INVALID, [](qmsg_attn_cfg &f) { f.scale = NAN; });
    expect(QMSG_E_INVALID, [](qmsg_attn_cfg &f) { f.scale = 3e38f; });          /* infinite in powers of two */
    expect(QMSG_E_UNSUPPORTED, [](qmsg_attn_cfg &f) { f.type = QMSG_T_Q8_0; });
    for (int d : { 0, 32, 96, 256 }) expect(QMSG_E_UNSUPPORTED, [&](qmsg_attn_cfg &f) { f.head_dim = d; });
    for (int p : { 0, 8, 24, 512, -16 }) expect(QMSG_E_UNSUPPORTED, [&](qmsg_attn_cfg &f) { f.page_tokens = p; });
    expect(QMSG_E_UNSUPPORTED, [](qmsg_attn_cfg &f) { f.n_head = f.n_head_kv = 1025; });
    expect(QMSG_E_UNSUPPORTED, [](qmsg_attn_cfg &f) { f.n_page = INT32_MAX; });
    expect(QMSG_E_UNSUPPORTED, [](qmsg_attn_cfg &f) { f.max_pages = INT32_MAX; });
    expect(QMSG_E_UNSUPPORTED, [](qmsg_attn_cfg &f) { f.max_tokens = INT32_MAX; });
    expect(QMSG_E_UNSUPPORTED, [](qmsg_attn_cfg &f) { f.max_seq = f.max_pages = 1 << 26; });
    expect(QMSG_E_UNSUPPORTED, [](qmsg_attn_cfg &f) { f.n_layer = (1 << 16) + 1; });
    expect(QMSG_E_UNSUPPORTED, [](qmsg_attn_cfg &f) { f.n_layer = INT32_MAX; });
    /* bytes that would wrap in 64 bits: 2^19 pages of 2^27 bytes, 2^16 layers and more */
    expect(QMSG_E_UNSUPPORTED, [](qmsg_attn_cfg &f) {
        f.n_head = f.n_head_kv = 1024;
        f.type = QMSG_T_F32;
        f.head_dim = 128;
        f.page_tokens = 256;
        f.n_page = 1 << 22;
        f.n_layer = 1 << 16;
    });
    qmsg_attn_cfg f = config();
    CHECK(qmsg_attn_create(ctx, &f, kK, kK, &id) == QMSG_E_INVALID && qmsg_attn_create(ctx, &f, kK, (char *)kK + qmsg_attn_cache_bytes(&f) - 16, &id) == QMSG_E_INVALID);
    CHECK(qmsg_attn_create(ctx, &f, (char *)kK + qmsg_attn_cache_bytes(&f) - 16, kK, &id) == QMSG_E_INVALID);
    CHECK(qmsg_attn_create(nullptr, &f, nullptr, nullptr, &id) == QMSG_E_INVALID && qmsg_attn_create(ctx, nullptr, nullptr, nullptr, &id) == QMSG_E_INVALID);
    CHECK(qmsg_attn_create(ctx, &f, kK, nullptr, &id) == QMSG_E_INVALID && qmsg_attn_create(ctx, &f, nullptr, kV, &id) == QMSG_E_INVALID);
    CHECK(qmsg_attn_create(ctx, &f, (char *)kK + 8, kV, &id) == QMSG_E_INVALID);
    CHECK(qmsg_attn_cache_bytes(&f) == 2ull * 32 * 2 * 16 * 64 * 2 && qmsg_attn_cache_bytes(nullptr) == 0);
    CHECK(qmsg_attn_create(ctx, &f, kK, (char *)kK + qmsg_attn_cache_bytes(&f), &id) == QMSG_OK);
}

static void memory()
{
    qmsg_attn_cfg f = config();
    int id = -1, failed = 0;
    const size_t before = live.size();
    for (int k = 0;; k++) {                      /* the k-th allocation fails */
        fail_at = allocs + k;
        const int rc = qmsg_attn_create(ctx, &f, nullptr, nullptr, &id);
        fail_at = -1;
        if (rc == QMSG_OK) break;
        CHECK((rc == QMSG_E_NOMEM || rc == QMSG_E_DEVICE) && live.size() == before && last == hipSuccess && id == -1);
        failed++;
    }
    CHECK(failed >= 8 && id == 0);
}

static int make()
{
    qmsg_attn_cfg f = config();
    int id = -1;
    CHECK(qmsg_attn_create(ctx, &f, nullptr, nullptr, &id) == QMSG_OK);
    return id;
}

static void batches()
{
    const int id = make();
    const int q[3] = { 1, 2, 0 }, kv[3] = { 20, 2, 5 };
    const int32_t pages[3][8] = { { 3, 4 }, { 5 }, { 6 } };
    CHECK(qmsg_attn_batch(ctx, id, 3, q, kv, &pages[0][0], 8) == QMSG_OK);
    const auto *h = &ctx->attns[(size_t)id]->plan.h;
    CHECK(h->n_tok == 3);
    auto expect = [&](int rc, int n, const int *a, const int *b, const int32_t *pg, int stride) {
        CHECK(qmsg_attn_batch(ctx, id, n, a, b, pg, stride) == rc && h->n_tok == 3);
    };
    expect(QMSG_E_INVALID, 4, q, kv, &pages[0][0], 8);
    expect(QMSG_E_INVALID, -1, q, kv, &pages[0][0], 8);
    expect(QMSG_E_INVALID, 3, nullptr, kv, &pages[0][0], 8);
    expect(QMSG_E_INVALID, 3, q, nullptr, &pages[0][0], 8);
    expect(QMSG_E_INVALID, 3, q, kv, nullptr, 8);
    expect(QMSG_E_INVALID, 3, q, kv, &pages[0][0], 1);               /* tables too short */
    const int long_kv[3] = { 129, 2, 5 }, neg[3] = { -1, 2, 0 }, more[3] = { 1, 3, 0 }, many[3] = { 19, 2, 0 };
    expect(QMSG_E_INVALID, 3, q, long_kv, &pages[0][0], 8);
    expect(QMSG_E_INVALID, 3, neg, kv, &pages[0][0], 8);
    expect(QMSG_E_INVALID, 3, more, kv, &pages[0][0], 8);
    expect(QMSG_E_INVALID, 3, many, kv, &pages[0][0], 8);
    for (int32_t bad : { -1, 32, INT32_MAX, INT32_MIN }) {
        int32_t p2[3][8];
        memcpy(p2, pages, sizeof p2);
        p2[0][0] = bad;
        expect(QMSG_E_INVALID, 3, q, kv, &p2[0][0], 8);
        memcpy(p2, pages, sizeof p2);
        p2[2][0] = bad;                                               /* a sequence without new tokens too */
        expect(QMSG_E_INVALID, 3, q, kv, &p2[0][0], 8);
    }
    const int32_t twice[3][8] = { { 3, 5 }, { 5 }, { 6 } };
    expect(QMSG_E_INVALID, 3, q, kv, &twice[0][0], 8);
    const int32_t own[1][8] = { { 7, 7 } };
    const int q1[1] = { 17 }, kv1[1] = { 17 };
    expect(QMSG_E_INVALID, 1, q1, kv1, &own[0][0], 8);
    capturing = true;
    expect(QMSG_E_INVALID, 3, q, kv, &pages[0][0], 8);
    capturing = false;
    CHECK(qmsg_attn_batch(ctx, id + 1, 0, q, kv, &pages[0][0], 8) == QMSG_E_INVALID && qmsg_attn_batch(nullptr, id, 0, q, kv, &pages[0][0], 8) == QMSG_E_INVALID);
    /* a batch that does not reach the device leaves none */
    copy_fails = true;
    CHECK(qmsg_attn_batch(ctx, id, 3, q, kv, &pages[0][0], 8) == QMSG_E_DEVICE && h->n_tok == 0 && last == hipSuccess);
    copy_fails = false;
    CHECK(qmsg_attn_device(ctx, id, 0, kQ, kQr) == QMSG_OK && attends.empty());
    CHECK(qmsg_attn_batch(ctx, id, 3, q, kv, &pages[0][0], 8) == QMSG_OK && h->n_tok == 3);
    CHECK(qmsg_attn_batch(ctx, id, 0, nullptr, nullptr, nullptr, 0) == QMSG_OK && h->n_tok == 0);
}

static void calls()
{
    const int id = make();
    const int q[1] = { 3 }, kv[1] = { 20 };
    const int32_t pages[2] = { 1, 2 };
    const size_t n = 3 * 8 * 64;
    /* nothing to do before a batch, or for one without tokens */
    CHECK(qmsg_attn_device(ctx, id, 0, kQ, kQr) == QMSG_OK && qmsg_attn_append_device(ctx, id, 0, kQr, kQ, kK, kV, 1e-6f) == QMSG_OK);
    CHECK(attends.empty() && appends.empty());
    CHECK(qmsg_attn_batch(ctx, id, 1, q, kv, pages, 2) == QMSG_OK);
    auto attend = [&](int rc, int i, int layer, const float *a, float *o) { CHECK(qmsg_attn_device(ctx, i, layer, a, o) == rc && attends.empty()); };
    attend(QMSG_E_INVALID, -1, 0, kQ, kQr);
    attend(QMSG_E_INVALID, id + 1, 0, kQ, kQr);
    attend(QMSG_E_RANGE, id, -1, kQ, kQr);
    attend(QMSG_E_RANGE, id, 2, kQ, kQr);
    attend(QMSG_E_INVALID, id, 0, nullptr, kQr);
    attend(QMSG_E_INVALID, id, 0, kQ, nullptr);
    attend(QMSG_E_INVALID, id, 0, kQ + 1, kQr);
    attend(QMSG_E_INVALID, id, 0, kQ, kQr + 2);
    attend(QMSG_E_INVALID, id, 0, kQ, kQ);
    attend(QMSG_E_INVALID, id, 0, kQ, kQ + n - 4);
    attend(QMSG_E_INVALID, id, 0, kQ + n - 4, kQ);
    CHECK(qmsg_attn_device(nullptr, id, 0, kQ, kQr) == QMSG_E_INVALID);
    CHECK(qmsg_attn_device(ctx, id, 1, kQ, kQ + n) == QMSG_OK && attends.size() == 1 && !attends[0].live);
    CHECK(attends[0].k == ctx->attns[(size_t)id]->k + ctx->attns[(size_t)id]->layer_bytes && attends[0].group == 4 && attends[0].shift == 4);
    auto append = [&](int rc, int i, int layer, float *o, const float *a, const float *k, const float *v, float eps) {
        CHECK(qmsg_attn_append_device(ctx, i, layer, o, a, k, v, eps) == rc && appends.empty());
    };
    append(QMSG_E_INVALID, id + 1, 0, kQr, kQ, kK, kV, 1e-6f);
    append(QMSG_E_RANGE, id, 2, kQr, kQ, kK, kV, 1e-6f);
    append(QMSG_E_INVALID, id, 0, kQr, kQ, nullptr, kV, 1e-6f);
    append(QMSG_E_INVALID, id, 0, kQr, kQ, kK, nullptr, 1e-6f);
    append(QMSG_E_INVALID, id, 0, nullptr, kQ, kK, kV, 1e-6f);
    append(QMSG_E_INVALID, id, 0, kQr, nullptr, kK, kV, 1e-6f);
    append(QMSG_E_INVALID, id, 0, kQr, kQ, kK + 1, kV, 1e-6f);
    append(QMSG_E_INVALID, id, 0, kQr, kQ, kK, kV + 3, 1e-6f);
    append(QMSG_E_INVALID, id, 0, kQr, kQ, kK, kV, -1.0f);
    append(QMSG_E_INVALID, id, 0, kQr, kQ, kK, kV, NAN);
    append(QMSG_E_INVALID, id, 0, kQ + 4, kQ, kK, kV, 1e-6f);
    append(QMSG_E_INVALID, id, 0, const_cast<float *>(kK) - 4, kQ, kK, kV, 1e-6f);
    append(QMSG_E_INVALID, id, 0, const_cast<float *>(kV), kQ, kK, kV, 1e-6f);
    CHECK(qmsg_attn_append_device(ctx, id, 0, kQ, kQ, kK, kV, 1e-6f) == QMSG_OK && qmsg_attn_append_device(ctx, id, 0, nullptr, nullptr, kK, kV, 0.0f) == QMSG_OK);
    CHECK(appends.size() == 2 && appends[0].norm == 1 && !appends[1].q);
    /* captured calls read the batch when they run, and are launched for one without tokens too */
    capturing = true;
    CHECK(qmsg_attn_device(ctx, id, 0, kQ, kQr) == QMSG_OK && attends.size() == 2 && attends[1].live);
    capturing = false;
    CHECK(qmsg_attn_batch(ctx, id, 0, nullptr, nullptr, nullptr, 0) == QMSG_OK);
    capturing = true;
    CHECK(qmsg_attn_device(ctx, id, 0, kQ, kQr) == QMSG_OK && qmsg_attn_append_device(ctx, id, 0, kQr, kQ, kK, kV, 1e-6f) == QMSG_OK);
    CHECK(attends.size() == 3 && appends.size() == 3 && appends[2].c.live && attends[2].blob == attends[1].blob);
    capturing = false;
    float w[64] = { 1 };
    void *k = nullptr, *v = nullptr;
    CHECK(qmsg_attn_norms(ctx, id, 2, w, w) == QMSG_E_RANGE && qmsg_attn_norms(ctx, id + 1, 0, w, w) == QMSG_E_INVALID);
    CHECK(qmsg_attn_norms(ctx, id, 1, w, nullptr) == QMSG_OK && qmsg_attn_norms(ctx, id, 1, nullptr, w) == QMSG_OK);
    /* the vector stays where a captured call may read it */
    CHECK(ctx->attns[(size_t)id]->layers[1].qw && live.count(ctx->attns[(size_t)id]->layers[1].qw));
    CHECK(qmsg_attn_cache(ctx, id, &k, nullptr) == QMSG_E_INVALID && qmsg_attn_cache(ctx, -1, &k, &v) == QMSG_E_INVALID && qmsg_attn_cache(ctx, id, &k, &v) == QMSG_OK && k && v);
    qmsg_attn_cfg f = config();
    f.qk_norm = 0;
    int plain = -1;
    CHECK(qmsg_attn_create(ctx, &f, kK, kV, &plain) == QMSG_OK && qmsg_attn_norms(ctx, plain, 0, w, w) == QMSG_E_INVALID);
    CHECK(qmsg_attn_cache(ctx, plain, &k, &v) == QMSG_OK && k == kK && v == kV);
}

static int mat(int64_t rows, int64_t cols)
{
    static uint8_t data[16];
    const qmsg_mat m = { QMSG_T_Q4_0, rows, cols, (uint64_t)cols / 32 * 18, data };
    int id = -1;
    CHECK(qmsg_mat_upload(ctx, &m, &id) == QMSG_OK);
    return id;
}

static void layers()
{
    const int id = make();
    const int q[1] = { 3 }, kv[1] = { 20 };
    const int32_t pages[2] = { 1, 2 };
    const int good[4] = { mat(512, 256), mat(128, 256), mat(128, 256), mat(256, 512) };
    float norm[256] = { 1 };
    float *const h = (float *)(8ull << 20);
    CHECK(qmsg_attn_batch(ctx, id, 1, q, kv, pages, 2) == QMSG_OK);
    CHECK(qmsg_attn_layer(ctx, id, 0, h, 1e-6f) == QMSG_E_INVALID);           /* no matrices yet */
    for (int k = 0; k < 4; k++)
        for (int bad : { -1, 99, good[(k + 1) % 4 == 2 ? 3 : (k + 1) % 4] }) {
            int ids[4] = { good[0], good[1], good[2], good[3] };
            ids[k] = bad;
            CHECK(qmsg_attn_mats(ctx, id, 0, ids, norm) == QMSG_E_INVALID);
        }
    CHECK(qmsg_attn_mats(ctx, id, 2, good, norm) == QMSG_E_RANGE && qmsg_attn_mats(ctx, id + 1, 0, good, norm) == QMSG_E_INVALID);
    CHECK(qmsg_attn_mats(ctx, id, 0, nullptr, norm) == QMSG_E_INVALID && qmsg_attn_mats(nullptr, id, 0, good, norm) == QMSG_E_INVALID);
    CHECK(qmsg_attn_mats(ctx, id, 1, good, norm) == QMSG_OK && qmsg_attn_mats(ctx, id, 0, good, nullptr) == QMSG_OK);
    CHECK(qmsg_attn_layer(ctx, id, 2, h, 1e-6f) == QMSG_E_RANGE && qmsg_attn_layer(ctx, id + 1, 0, h, 1e-6f) == QMSG_E_INVALID);
    CHECK(qmsg_attn_layer(ctx, id, 1, nullptr, 1e-6f) == QMSG_E_INVALID && qmsg_attn_layer(ctx, id, 1, h + 1, 1e-6f) == QMSG_E_INVALID);
    CHECK(qmsg_attn_layer(ctx, id, 1, h, NAN) == QMSG_E_INVALID && qmsg_attn_layer(nullptr, id, 1, h, 1e-6f) == QMSG_E_INVALID && steps.empty());
    CHECK(qmsg_attn_layer(ctx, id, 1, h, 1e-6f) == QMSG_OK);
    /* norm, q, k, v, append, attention, output, residual: each on what the one before left */
    CHECK(steps.size() == 6 && appends.size() == 1 && attends.size() == 1);
    const float *x = steps[0].out;
    CHECK(steps[0].in == h && steps[0].n == 3 * 256 && steps[0].w && steps[1].in == x && steps[2].in == x && steps[3].in == x);
    CHECK(steps[1].n == 3 * 512 && steps[2].n == 3 * 128 && steps[1].out + steps[1].n <= steps[2].out && steps[2].out + steps[2].n <= steps[3].out);
    CHECK(appends[0].q == steps[1].out && appends[0].qr == steps[1].out && appends[0].k == steps[2].out && appends[0].v == steps[3].out);
    CHECK(attends[0].q == steps[1].out && steps[4].in == attends[0].out && steps[5].in == steps[4].out && steps[5].out == h && steps[5].n == 3 * 256);
    CHECK(attends[0].out >= steps[3].out + steps[3].n && steps[4].out == attends[0].out + 3 * 512);
    CHECK(appends[0].c.k == ctx->attns[(size_t)id]->k + ctx->attns[(size_t)id]->layer_bytes);
    CHECK(qmsg_attn_batch(ctx, id, 0, nullptr, nullptr, nullptr, 0) == QMSG_OK && qmsg_attn_layer(ctx, id, 1, h, 1e-6f) == QMSG_OK && steps.size() == 6);
}

int main(int argc, char **argv)
{
    const std::string s = argc > 1 ? argv[1] : "";
    const qmsg_cfg cfg = { 256, 16, 4, 128 };
    CHECK(qmsg_create(&ctx, 0, &cfg, 1, 1) == QMSG_OK);
    if (s == "configs") configs();
    else if (s == "memory") memory();
    else if (s == "batches") batches();
    else if (s == "calls") calls();
    else if (s == "layers") layers();
    else return 2;
    qmsg_destroy(ctx);
    ctx = nullptr;
    if (!live.empty()) { fprintf(stderr, "%zu allocations left\n", live.size()); return 1; }
    return 0;
}
