/* qmsg_ctx.h - the context behind the C ABI and what its entry points share (host code). */
#ifndef QMSG_CTX_H
#define QMSG_CTX_H

#include <hip/hip_runtime.h>

#include <memory>
#include <string>
#include <vector>

#include "../../include/qmsg.h"
#include "qmsg_attn.h"
#include "qmsg_internal.h"

namespace qmsg {

struct LayerStore {
    float *router = nullptr;
    float *norm = nullptr;        /* ffn_norm [E], nullptr: unit weights */
    uint8_t *gate = nullptr, *up = nullptr, *down = nullptr;
    int gate_type = -1, up_type = -1, down_type = -1;
    bool ready = false;
};

/* A dense (trunk) matrix resident in HBM, QmsMat (src/quant.h:11-16) with device data. */
struct DenseStore {
    uint8_t *w = nullptr;
    int type = -1;
    int64_t rows = 0, cols = 0;
    uint64_t rb = 0;
};

struct ProfRec {
    std::string name;
    hipEvent_t a, b;
};

/* One layer's part of an attention: head norms, and the matrices of qmsg_attn_chain. */
struct AttnLayer {
    float *qw = nullptr, *kw = nullptr;     /* head norms [D], nullptr: unit weights   */
    float *norm = nullptr;                  /* attn_norm [E], nullptr: unit weights    */
    int mats[4] = { -1, -1, -1, -1 };       /* q, k, v, output: ids of dense matrices  */
};

/* An attention over a paged cache (qmsg_attn_create). */
struct AttnStore {
    qmsg_attn_cfg cfg{};
    AttnShape shape{};
    uint8_t *k = nullptr, *v = nullptr;     /* [layer][page][kv head][...]             */
    uint64_t layer_bytes = 0;
    uint32_t page_bytes = 0;
    double *freq = nullptr;                 /* [D/2] turns per position                */
    uint8_t *blob = nullptr;                /* the batch's plan on the device          */
    float *part_o = nullptr, *part_ml = nullptr;
    int32_t *done = nullptr;                /* counters of the tiles' done items       */
    AttnPlan plan;
    /* two pinned plans: one is filled while the copy of the other may still run */
    uint8_t *pin[2] = { nullptr, nullptr };
    hipEvent_t copied[2] = { nullptr, nullptr };
    int next = 0;
    /* rows of qmsg_attn_chain, on its first call: layer input, q, k, v, rotated q, attention, output */
    float *rows = nullptr;
    std::vector<AttnLayer> layers;
    std::vector<void *> allocs;
};

}  // namespace qmsg

struct qmsg_ctx {
    int device = 0;
    qmsg_cfg cfg{};
    int n_layer = 0, max_tokens = 0, path = QMSG_PATH_AUTO;
    int norm_walk = 0;                      /* rmsnorm: form every row's sum in order */
    unsigned long long *d_walked = nullptr; /* rmsnorm: rows that formed it in order */
    float *d_hb = nullptr;                  /* the one-token chain's second row of h */
    int n_cu = 256;
    hipStream_t stream = nullptr;
    std::vector<qmsg::LayerStore> layers;
    qmsg::Scratch S{};
    std::vector<void *> scratch_allocs, user_allocs;
    float *d_x = nullptr, *d_out = nullptr;
    std::vector<qmsg::DenseStore> mats;
    std::vector<std::unique_ptr<qmsg::AttnStore>> attns;
    /* grow-on-demand buffers of the dense products: input records, host-call staging */
    void *dense_xqk = nullptr;
    size_t dense_xqk_bytes = 0;
    bool dense_xqk_held = false;            /* by a captured call: never freed before the context */
    void *dense_io = nullptr;
    size_t dense_io_bytes = 0;
    /* pinned rows of the host-buffer layer call (kHostStage bytes in, as many out), on first use */
    uint8_t *pin = nullptr;
    std::string err;
    bool prof = false;
    std::vector<qmsg::ProfRec> prof_recs, prof_free;
    struct Tot { std::string name; int64_t n; double ms; };
    std::vector<Tot> prof_tot;
};

namespace qmsg {

/* Record the reason of a failure and return its code (c may be NULL: qmsg_last_error(NULL)). */
int fail(qmsg_ctx *c, int code, const char *fmt, ...);
/* hipMalloc with 256 bytes of tail padding; the pointer is added to `list`. */
int dev_alloc(qmsg_ctx *c, void **p, size_t bytes, std::vector<void *> &list);
/* Timing hook: hands out an event pair per kernel dispatch while profiling is on. */
void prof_events(void *vc, const char *kernel, hipEvent_t *start, hipEvent_t *stop);
/* What an attention holds besides its entries of `allocs`. */
void attn_release(AttnStore &a);

}  // namespace qmsg

/* A failed runtime call's error also stays the thread's last error, which the next launch would
 * report as its own: it is cleared where the failure is returned or absorbed. */
#define HIP_TRY(c, call)                                                                               \
    do {                                                                                               \
        hipError_t e_ = (call);                                                                        \
        if (e_ != hipSuccess) {                                                                        \
            (void)hipGetLastError();                                                                   \
            return fail((c), QMSG_E_DEVICE, "%s: %s", #call, hipGetErrorString(e_));                   \
        }                                                                                              \
    } while (0)

#define LAUNCH(c, name, expr)                                                                             \
    do {                                                                                                  \
        const LaunchTimer timer_{ (c), prof_events };                                                     \
        g_launch_timer = (c)->prof ? &timer_ : nullptr;                                                   \
        hipError_t e_ = (expr);                                                                           \
        g_launch_timer = nullptr;                                                                         \
        if (e_ != hipSuccess) return fail((c), QMSG_E_DEVICE, "%s launch: %s", (name), hipGetErrorString(e_)); \
    } while (0)

#endif /* QMSG_CTX_H */
