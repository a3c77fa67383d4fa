/* qmsg_attn.h - arguments and launchers of the attention kernels (qmsg_attn.hip). */
#ifndef QMSG_ATTN_H
#define QMSG_ATTN_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmsg_plan.h"

namespace qmsg {

/* A call on the batch in `blob` (a plan, header first). live: read the header there when the kernel
 * runs (a captured call, replayed on later batches), else h is it. */
struct AttnCall {
    AttnHdr h;
    int live;
    const uint8_t *blob;
    const uint8_t *k, *v;       /* the layer's pages: keys [kv head][slot][D], values [kv head][D][slot] */
    uint32_t page_bytes;        /* of a page's keys, or its values */
    int shift;                  /* page tokens = 1 << shift        */
    int heads, kv_heads, group;
    float scale_log2;           /* scale * log2(e)                 */
    const float *q;             /* [T][heads][D]                   */
    float *out;                 /* [T][heads][D]                   */
    int32_t *done;              /* counters, 0 between calls       */
    float *part_o, *part_ml;    /* partial rows [slot][heads][D], their reference and sum [slot][heads][2] */
};

struct AttnAppend {
    AttnCall c;
    const float *q, *k, *v;     /* [T][heads][D] (q may be NULL), [T][kv heads][D] */
    float *qr;
    const float *qw, *kw;       /* norm weights [D]                */
    const double *freq;         /* [D/2] turns per position        */
    float eps;
    int norm;
};

/* grid: blocks of a live call, whose kernels loop over what the batch holds. */
hipError_t launch_attend(const AttnCall &a, int type, int D, int grid, hipStream_t st);
hipError_t launch_attn_append(const AttnAppend &b, int type, int D, int grid, hipStream_t st);

}  // namespace qmsg

#endif /* QMSG_ATTN_H */
