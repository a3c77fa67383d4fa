/* qmsg_attn.hip - head norms, rotation and the append to the paged cache; attention over the cache.
 *
 * Cache pages: keys [kv head][slot][D], values [kv head][D][slot], so that both products read their
 * matrix operand in 16-byte pieces along the axis they sum over, without a transpose:
 *
 *   S^T = K q^T     (keys x rows),  A operand 16 keys x D,      B operand the rows' queries
 *   O^T += V^T P^T  (D x rows),     A operand 16 d x the keys,  B operand P^T
 *
 * A 16x16 result leaves lane (col = lane % 16, g = lane / 16) the four keys 4g .. 4g+3 of row col,
 * and the B operand wants from it one 16-byte piece of consecutive keys. The order in which keys
 * are dealt to the rows of the first product is free, so key (m / 4) * CE + 4 tl + m % 4 of a step goes
 * to row m of its tile tl: then lane (col, g) holds exactly the keys g * CE .. of its row, and P needs
 * neither a shuffle nor LDS on its way into the second product (CE elements in 16 bytes: 8 f16 in
 * two tiles a step of 32 keys, 4 f32 in one tile of 16).
 *
 * Activations are fp32. With an f16 cache q and p are split into two f16, x = hi + lo to 22 bits, and each product is two f16 MFMAs
 * into fp32: twice the f16 work, against the sixteenth of the rate that fp32 MFMAs would have. An fp32
 * cache takes the fp32 MFMAs as it is.
 *
 * Softmax in one pass: p = 2^(s - ref) with s in powers of two (q is scaled) and ref a row's running reference, set 6 below the row's
 * largest score so far and raised only when a score passes it by 14, so that p stays below 2^14 (f16's
 * range) and the usual step needs no reduction across lanes. The products' accumulators start at -ref, so
 * that s - ref costs no instruction. Sums, references and O are fp32. */
#include <cmath>
#include <type_traits>

#include "qmsg_attn.h"
#include "qmsg_device.h"

namespace qmsg {

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLowest = -INFINITY;

/* A cache of one type and head width. */
template <int TYPE, int D>
struct Att {
    static constexpr int ES = TYPE == 1 ? 2 : 4;        /* bytes of an element                    */
    static constexpr int CE = 16 / ES;                  /* elements of a piece                    */
    static constexpr int TL = CE / 4;                   /* key tiles of a step                    */
    static constexpr int KS = 16 * TL;                  /* keys of a step                         */
    static constexpr int NCH = D / (4 * CE);            /* pieces per lane of a key tile          */
    static constexpr int NK = TL * NCH, NV = D / 16;    /* 16-byte loads per lane and step        */
};

/* The row's query as B operand: lane (col, g) holds d = 4 CE c + CE g .. of piece c. */
template <int TYPE, int D>
struct AttQ {
    h8 hi[Att<TYPE, D>::NCH], lo[Att<TYPE, D>::NCH];
};
template <int D>
struct AttQ<0, D> {
    f32x4 v[Att<0, D>::NCH];
};

/* Running softmax of a lane's row: reference, this lane's part of the sum, O^T (d = 16 i + 4 g + r). What its
 * scores are summed from (less the reference, in the units of the row's query) stands apart. */
template <int D>
struct AttRow {
    float ref = kLowest, l = 0.0f;
    f32x4 o[D / 16] = {};
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

/* The larger of the four lanes of a row (g = 0..3), in all of them. */
__device__ __forceinline__ float row_max(float v)
{
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
    u = __builtin_bit_cast(uint32_t, v);
    r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float row_sum(float v)
{
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    u = __builtin_bit_cast(uint32_t, v);
    r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

/* A row's query as it lies in memory, 16 bytes a load. */
template <int TYPE, int D>
struct AttRaw {
    f32x4 x[D / 16];
};
template <int TYPE, int D>
__device__ __forceinline__ void load_q(const float *row, int g, AttRaw<TYPE, D> &raw)
{
    constexpr int CE = Att<TYPE, D>::CE;
#pragma unroll
    for (int i = 0; i < D / 16; i++) raw.x[i] = *(const f32x4 *)(row + i / (CE / 4) * 4 * CE + CE * g + i % (CE / 4) * 4);
}

/* x - (float)half I of h, in one instruction. */
template <int I>
__device__ __forceinline__ float less_half(float x, uint32_t h)
{
    float r;
    if constexpr (I == 0) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}

/* x and y as two f16 each: what hi's 11 bits leave out is in lo, to 11 more. */
__device__ __forceinline__ void split(float x, float y, uint32_t &hi, uint32_t &lo)
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    hi = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{ x, y }), h2));
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{ less_half<0>(x, hi), less_half<1>(y, hi) }), h2));
}

/* A query times `scale` as B operand; returns the power of two that its scores come out multiplied with: 1
 * but for fp16 rows whose largest element is outside [2^-4, 2^14) (a row of zeros is inside). Those are
 * scaled to [2^8, 2^9), so that neither half leaves f16's range. */
template <int TYPE, int D>
__device__ __forceinline__ float make_q(AttRaw<TYPE, D> &raw, float scale, AttQ<TYPE, D> &q)
{
    using A = Att<TYPE, D>;
    if constexpr (TYPE == 0) {
#pragma unroll
        for (int c = 0; c < A::NCH; c++) q.v[c] = raw.x[c] * scale;
        return 1.0f;
    } else {
        float top = 0.0f, up = 1.0f;
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            raw.x[i] *= scale;
#pragma unroll
            for (int e = 0; e < 4; e += 2) top = fmaxf(top, fmaxf(fabsf(raw.x[i][e]), fabsf(raw.x[i][e + 1])));
        }
        top = row_max(top);
        const bool far = top != 0.0f && (top < 0.0625f || top >= 16384.0f);
        if (__ballot(far)) {
            /* subnormal rows and rows with an infinity keep a factor inside fp32's range */
            const int ex = min(max((int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127, -110), 127);
            if (far) up = __builtin_bit_cast(float, (uint32_t)(127 + 8 - ex) << 23);
#pragma unroll
            for (int i = 0; i < D / 16; i++) raw.x[i] *= up;
        }
#pragma unroll
        for (int c = 0; c < A::NCH; c++) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; k++) split(raw.x[2 * c + k / 2][2 * (k % 2)], raw.x[2 * c + k / 2][2 * (k % 2) + 1], hi[k], lo[k]);
            q.hi[c] = __builtin_bit_cast(h8, u32x4{ hi[0], hi[1], hi[2], hi[3] });
            q.lo[c] = __builtin_bit_cast(h8, u32x4{ lo[0], lo[1], lo[2], lo[3] });
        }
        return up;
    }
}

/* A piece of keys (piece c of tile t) times the first NA of a wave's NT row tiles, into their scores. */
template <int TYPE, int D, int NT, int NA>
__device__ __forceinline__ void score(u32x4 k, int c, int t, const AttQ<TYPE, D> (&q)[NT], f32x4 (&s)[NA][Att<TYPE, D>::TL])
{
    if constexpr (TYPE == 0) {
        const f32x4 x = __builtin_bit_cast(f32x4, k);
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int n = 0; n < NA; n++) s[n][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], q[n].v[c][e], s[n][t], 0, 0, 0);
    } else {
        const h8 x = __builtin_bit_cast(h8, k);
#pragma unroll
        for (int n = 0; n < NA; n++) s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[n].lo[c], s[n][t], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NA; n++) s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[n].hi[c], s[n][t], 0, 0, 0);
    }
}

/* A step's scores s[n][t][r] of key g * CE + 4 t + r start at `from`: they come out off their references. */
template <int NT, int NA, int TL>
__device__ __forceinline__ void score_from(const float (&from)[NT], f32x4 (&s)[NA][TL])
{
#pragma unroll
    for (int n = 0; n < NA; n++)
#pragma unroll
        for (int t = 0; t < TL; t++) s[n][t] = f32x4{ from[n], from[n], from[n], from[n] };
}

/* P as B operand: two f16 of each weight, or the weights. */
template <int TYPE>
struct AttP {
    uint32_t hi[4], lo[4];
};
template <>
struct AttP<0> {
    float v[4];
};

/* Scores of rows whose query was scaled up, taken back down. */
template <int NT, int NA, int NS, int TL>
__device__ __forceinline__ void unscale(const float (&up)[NT], f32x4 (&s)[NS][NA][TL])
{
#pragma unroll
    for (int n = 0; n < NA; n++) {
        const float down = 1.0f / up[n];                     /* powers of two */
#pragma unroll
        for (int k = 0; k < NS; k++)
#pragma unroll
            for (int t = 0; t < TL; t++) s[k][n][t] *= down;
    }
}

/* A step's scores of keys that the row does not see (left: its limit less the lane's first key). */
template <int TL>
__device__ __forceinline__ void hide(int left, f32x4 (&s)[TL])
{
#pragma unroll
    for (int t = 0; t < TL; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[t][r] = 4 * t + r < left ? s[t][r] : kLowest;
}

/* Raise the references of NA row tiles for NS steps of scores (off their references) where one is too far
 * above its row's. */
template <int D, int NT, int NA, int NS, int TL>
__device__ __forceinline__ void raise(const float (&up)[NT], f32x4 (&s)[NS][NA][TL], float (&from)[NT], AttRow<D> (&row)[NT])
{
    float top[NA];
    bool far = false;
#pragma unroll
    for (int n = 0; n < NA; n++) {
        top[n] = s[0][n][0][0];
#pragma unroll
        for (int k = 0; k < NS; k++)
#pragma unroll
            for (int t = 0; t < TL; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) top[n] = fmaxf(top[n], s[k][n][t][r]);
        /* a row without a reference has its scores as they are */
        far = far || top[n] > (row[n].ref == kLowest ? kLowest : 14.0f);
    }
    if (__builtin_expect(__ballot(far) != 0, 0)) {
#pragma unroll
        for (int n = 0; n < NA; n++) {
            const float base = row[n].ref == kLowest ? 0.0f : row[n].ref;
            const float ref = fmaxf(row[n].ref, base + row_max(top[n]) - 6.0f);
            const float a = ref == row[n].ref ? 1.0f : exp2_fast(row[n].ref - ref);
            const float off = ref == kLowest ? 0.0f : base - ref;
            row[n].ref = ref;
            from[n] = ref == kLowest ? 0.0f : -ref * up[n];
            row[n].l *= a;
#pragma unroll
            for (int i = 0; i < D / 16; i++) row[n].o[i] *= a;
#pragma unroll
            for (int k = 0; k < NS; k++)
#pragma unroll
                for (int t = 0; t < TL; t++) s[k][n][t] += off;
        }
    }
}

/* The weights of key tile t of a row's step, from its scores. */
template <int TYPE, int D>
__device__ __forceinline__ void soften(int t, f32x4 s, AttRow<D> &row, AttP<TYPE> &p)
{
    float x[4];
#pragma unroll
    for (int r = 0; r < 4; r++) x[r] = exp2_fast(s[r]);
    row.l += (x[0] + x[1]) + (x[2] + x[3]);
    if constexpr (TYPE == 0) {
#pragma unroll
        for (int r = 0; r < 4; r++) p.v[r] = x[r];
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) split(x[2 * i], x[2 * i + 1], p.hi[2 * t + i], p.lo[2 * t + i]);
    }
}

/* Masks over the lane's piece of values: keys the item has (of n_key from the piece's first on), and of
 * those the ones that not every row sees (from n_full on). */
struct AttMask {
    uint32_t has[4], some[4];
};
template <int TYPE>
__device__ __forceinline__ AttMask piece_mask(int n_full, int n_key)
{
    AttMask m;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if constexpr (TYPE == 0) {
            m.has[w] = w < n_key ? ~0u : 0u;
            m.some[w] = w >= n_full ? m.has[w] : 0u;
        } else {
            m.has[w] = (2 * w < n_key ? 0xffffu : 0u) | (2 * w + 1 < n_key ? 0xffff0000u : 0u);
            m.some[w] = m.has[w] & ((2 * w >= n_full ? 0xffffu : 0u) | (2 * w + 1 >= n_full ? 0xffff0000u : 0u));
        }
    }
    return m;
}

/* The piece with zeros for keys past the item's end (what a page holds there may be anything), and for
 * infinities and NaN of keys that some rows do not see: 0 * infinity would reach these. The rows that do
 * see them get them in the end (add_wild). */
template <int TYPE>
__device__ __forceinline__ u32x4 clean(u32x4 v, const AttMask &m, uint32_t &bad)
{
#pragma unroll
    for (int w = 0; w < 4; w++) {
        uint32_t wild;                                  /* all ones where the exponent is */
        if constexpr (TYPE == 0) {
            wild = (uint32_t)((int32_t)((v[w] & 0x7f800000u) + 0x00800000u) >> 31);
        } else {
            const uint32_t b = ((v[w] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
            wild = (b - (b >> 15)) | b;
        }
        wild &= m.some[w];
        bad |= wild;
        v[w] &= m.has[w] & ~wild;
    }
    return v;
}

/* O^T += V^T P^T of NA row tiles for the piece v of values d = 16 i + col. */
template <int TYPE, int D, int NT, int NA>
__device__ __forceinline__ void weigh(u32x4 v, int i, const AttP<TYPE> (&p)[NA], AttRow<D> (&row)[NT])
{
    if constexpr (TYPE == 0) {
        const f32x4 x = __builtin_bit_cast(f32x4, v);
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int n = 0; n < NA; n++) row[n].o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], p[n].v[e], row[n].o[i], 0, 0, 0);
    } else {
        const h8 x = __builtin_bit_cast(h8, v);
#pragma unroll
        for (int n = 0; n < NA; n++)
            row[n].o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(h8, u32x4{ p[n].hi[0], p[n].hi[1], p[n].hi[2], p[n].hi[3] }), row[n].o[i], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NA; n++)
            row[n].o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, __builtin_bit_cast(h8, u32x4{ p[n].lo[0], p[n].lo[1], p[n].lo[2], p[n].lo[3] }), row[n].o[i], 0, 0, 0);
    }
}

/* Byte address of a page's keys or values of one kv head. */
__device__ __forceinline__ const uint8_t *page_at(const uint8_t *pool, int page, uint32_t page_bytes, uint32_t head_off)
{
    return pool + (size_t)(uint32_t)page * page_bytes + head_off;
}

/* What clean() left out of the keys [from, to) of values d .. d+3, summed. */
template <int TYPE, int D>
__device__ __forceinline__ f32x4 wild_sum(const uint8_t *pool, const int32_t *tab, uint32_t page_bytes, uint32_t head_off, int shift, int from,
                                          int to, int d)
{
    constexpr int ES = Att<TYPE, D>::ES;
    f32x4 sum = { 0, 0, 0, 0 };
#pragma unroll 1
    for (int k = from; k < to; k++) {
        const uint8_t *base = page_at(pool, tab[k >> shift], page_bytes, head_off);
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint32_t off = ((uint32_t)(d + r) << shift) + (uint32_t)(k & ((1 << shift) - 1));
            float v;
            if constexpr (TYPE == 0) v = *(const float *)(base + off * ES);
            else v = (float)*(const _Float16 *)(base + off * ES);
            if (!(fabsf(v) < INFINITY)) sum[r] += v;
        }
    }
    return sum;
}

/* The part of a call's header that is in use: the launch's own, or the blob's for a captured call. */
__device__ __forceinline__ const AttnHdr &header(const AttnCall &a) { return a.live ? *(const AttnHdr *)a.blob : a.h; }

/* Parts that a block joins go past its die's L2 (and are read past it): it may run on another than theirs. A
 * release and an acquire of the whole L2 instead took 262 us where this takes 55 (32 decoded sequences). */
__device__ __forceinline__ void put_far(float *p, f32x4 v)
{
    const uint64_t x = __builtin_bit_cast(uint64_t, (f32x2){ v.x, v.y }), y = __builtin_bit_cast(uint64_t, (f32x2){ v.z, v.w });
    __hip_atomic_store((uint64_t *)p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store((uint64_t *)p + 1, y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put_far(float *p, float a, float b)
{
    __hip_atomic_store((uint64_t *)p, __builtin_bit_cast(uint64_t, (f32x2){ a, b }), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 get_far(const float *p)
{
    return __builtin_bit_cast(f32x2, __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

/* Where a row's results go: the output where the token has no other part, else its part. */
__device__ __forceinline__ float *row_out(const AttnCall &a, const AttnTok &tk, int part, int t, int head, int D)
{
    return tk.parts == 1 ? a.out + ((size_t)t * a.heads + head) * D : a.part_o + ((size_t)(tk.part + part) * a.heads + head) * D;
}
/* A part's reference is +infinity where its sum is NaN, so that joining keeps it. An empty item's parts may be
 * more than a token has. */
__device__ __forceinline__ void put_row(const AttnCall &a, const AttnTok &tk, const AttnWork &w, int t, int head, int d, int D, float ref,
                                        float l, f32x4 o, bool stats)
{
    const bool whole = tk.parts == 1;
    if (w.part >= tk.parts) return;
    float *to = row_out(a, tk, w.part, t, head, D) + d, *ml = a.part_ml + 2 * ((size_t)(tk.part + w.part) * a.heads + head);
    ref = l != l ? INFINITY : ref;
    if (whole) {
        *(f32x4 *)to = o * (1.0f / l);
    } else if (w.count >= 0) {
        put_far(to, o);
        if (stats) put_far(ml, ref, l);
    } else {
        *(f32x4 *)to = o;
        if (stats) *(f32x2 *)ml = f32x2{ ref, l };
    }
}

/* Parts of four values taken together: o = sum_p 2^(m_p - m) o_p, l likewise. */
struct AttJoin {
    float m = kLowest, l = 0.0f;
    f32x4 o = { 0, 0, 0, 0 };
    __device__ __forceinline__ void add(float mp, float lp, f32x4 op)
    {
        if (mp == kLowest) return;                                  /* saw no key */
        const float top = fmaxf(m, mp), f0 = m == kLowest ? 0.0f : exp2_fast(m - top), f1 = exp2_fast(mp - top);
        m = top;
        l = l * f0 + lp * f1;
        o = o * f0 + op * f1;
    }
};

/* After an item of a tile whose parts its last item joins: count it, and join if it is the last. Each wave waits
 * until its parts have arrived before the block counts. */
template <int D, int THREADS>
__device__ __forceinline__ void join_tile(const AttnCall &a, const AttnTok *toks, const AttnWork &w, int kvh, int &s_last)
{
    if (w.count < 0) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        int32_t *c = a.done + w.count * a.kv_heads + kvh;
        s_last = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == w.joins - 1;
        if (s_last) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!s_last) return;
    for (int e = threadIdx.x; e < w.rows * (D / 4); e += THREADS) {
        const int r = w.row + e / (D / 4), d = e % (D / 4) * 4, t = r / a.group, head = kvh * a.group + r % a.group;
        const AttnTok tk = toks[t];
        if (tk.parts == 1) continue;                                /* is in the output */
        const size_t r0 = (size_t)tk.part * a.heads + head;
        AttJoin j;
        for (int p = 0; p < tk.parts; p += 4) {                     /* four parts' loads at a time */
            f32x2 ml[4], lo[4], hi[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const size_t at = r0 + (size_t)min(p + k, tk.parts - 1) * a.heads;
                ml[k] = get_far(a.part_ml + 2 * at);
                lo[k] = get_far(a.part_o + at * D + d);
                hi[k] = get_far(a.part_o + at * D + d + 2);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (p + k < tk.parts) j.add(ml[k].x, ml[k].y, f32x4{ lo[k].x, lo[k].y, hi[k].x, hi[k].y });
        }
        *(f32x4 *)(a.out + ((size_t)t * a.heads + head) * D + d) = j.o * (1.0f / j.l);
    }
}

/* Few rows (16): eight waves (of many short items: one, two or four) take turns at the steps of the item's keys, each
 * from memory straight into the operands' registers with the next step's loads in flight, and join in LDS.
 *
 * Bound: the cache's bytes, read once; no byte is used twice in a block, so LDS would only add a step, and a
 * wave's 16 loads of 16 bytes a lane in flight (one block of eight waves a CU) reach the rate of a large copy: 32
 * sequences of 4096 to 8191 keys (64 heads on 4, f16) 54 us, 5.1 TB/s; one of 131071 keys 43 us, 6.2 TB/s,
 * and 4 to join. Short calls are latency: a token over 513 keys 9 us, of which 3 pass until the first
 * keys' loads are issued, 2 until the products are done and 3 in joining waves and items; 2 sequences of 33 keys 6. Waves
 * without a step load and join nothing (those 2 sequences 11 us otherwise). 256 sequences of up to 101 keys: 14 us. */
template <int D>
struct FewLds {
    __align__(16) float o[kFewWaves][16][D + 4];
    float m[kFewWaves][16], l[kFewWaves][16], top[kFewWaves][16];
    int last;
};

/* The launch's items with W waves each: a block's waves are groups of W with an item of their own. */
template <int TYPE, int D, int W>
__device__ __forceinline__ void few_items(const AttnCall &a, const AttnHdr &h, FewLds<D> &lds)
{
    using A = Att<TYPE, D>;
    constexpr int NT = 1, groups = kFewWaves / W, o_rows = 64 * W / (D / 4);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, g = lane >> 4, P1 = (1 << a.shift) - 1;
    const int n_unit = h.n_run[kAttnFew] * a.kv_heads;
    const int group = wave / W, sub = wave % W;
    const int o_row = threadIdx.x % (64 * W) / (D / 4), o_d = threadIdx.x % (D / 4) * 4;
    const AttnWork *work = (const AttnWork *)(a.blob + h.work[kAttnFew]);
    const AttnTok *toks = (const AttnTok *)(a.blob + h.tok);
    for (int u0 = blockIdx.x * groups, next = -1; next >= 0 || u0 < n_unit;) {
        const int u = min(u0 + group, n_unit - 1);
        const AttnWork w = work[next >= 0 ? next : u / a.kv_heads];
        const int kvh = u % a.kv_heads, n_row = u0 + group < n_unit ? min(w.rows, 16) : 0;      /* 0: no item for the group */
        next = w.next;
        if (next < 0) u0 += gridDim.x * groups;
        const int32_t *tab = (const int32_t *)(a.blob + h.pages) + w.pages;
        const uint32_t head_off = (uint32_t)kvh * ((uint32_t)(D * A::ES) << a.shift);
        const int n_step = n_row ? (w.key1 - w.key0 + A::KS - 1) / A::KS : 0, busy = min(W, n_step);     /* waves with a step */
        const int o_r = w.row + min(o_row, w.rows - 1);
        int o_tok = o_r / a.group, o_head = kvh * a.group + o_r % a.group;
        AttnTok o_tk = toks[o_tok];
        AttRow<D> row[NT];
        uint32_t bad = 0;
        if (sub < busy) {
            /* a row behind the last one takes the last one's query: its results are not stored */
            const int qr = w.row + min(col, w.rows - 1), qt = qr / a.group;
            AttRaw<TYPE, D> raw;
            load_q<TYPE, D>(a.q + ((size_t)qt * a.heads + (size_t)(kvh * a.group + qr % a.group)) * D, g, raw);
            const int limit[NT] = { min(toks[qt].pos + 1, w.key1) };
            const int last = w.key1 - 1;
            const int k_off = (col >> 2) * A::CE + (col & 3), v_off = g * A::CE;
            u32x4 kf[A::NK], vf[A::NV];
            int kp = 0, vp = 0;
            auto pages = [&](int s) {
                const int k = w.key0 + s * A::KS;
                kp = tab[min(k + k_off, last) >> a.shift];
                vp = tab[min(k + v_off, last) >> a.shift];
            };
            auto load_k = [&](int s) {
                const int slot = (w.key0 + s * A::KS + k_off) & P1;
                const uint8_t *p = page_at(a.k, kp, a.page_bytes, head_off) + (uint32_t)(slot * D + g * A::CE) * A::ES;
#pragma unroll
                for (int t = 0; t < A::TL; t++)
#pragma unroll
                    for (int i = 0; i < A::NCH; i++) kf[t * A::NCH + i] = *(const u32x4 *)(p + (4 * t * D + 4 * i * A::CE) * A::ES);
            };
            auto load_v = [&](int s) {
                const int slot = (w.key0 + s * A::KS + v_off) & P1;
                const uint8_t *p = page_at(a.v, vp, a.page_bytes, head_off) + (uint32_t)((col << a.shift) + slot) * A::ES;
                const uint32_t step = (uint32_t)(16 * A::ES) << a.shift;
#pragma unroll
                for (int i = 0; i < A::NV; i++) vf[i] = *(const u32x4 *)(p + i * step);
            };
            pages(sub);
            load_k(sub);
            load_v(sub);
            if (sub + W < n_step) pages(sub + W);
            AttQ<TYPE, D> q[NT];
            float up[NT] = { make_q<TYPE, D>(raw, a.scale_log2, q[0]) }, from[NT] = {};
            const bool unit = __ballot(up[0] != 1.0f) == 0;
            for (int s = sub; s < n_step; s += W) {
                const int key = w.key0 + s * A::KS;
                const bool more = s + W < n_step, mask = key + A::KS > w.full;
                f32x4 sc[1][NT][A::TL];
                score_from(from, sc[0]);
#pragma unroll
                for (int i = 0; i < A::NCH; i++)
#pragma unroll
                    for (int t = 0; t < A::TL; t++) score<TYPE, D>(kf[t * A::NCH + i], i, t, q, sc[0]);
                if (!unit) unscale(up, sc);
                if (more) load_k(s + W);
                if (mask) {
                    hide(limit[0] - key - v_off, sc[0][0]);
                    const AttMask m = piece_mask<TYPE>(w.full - key - v_off, w.key1 - key - v_off);
#pragma unroll
                    for (int i = 0; i < A::NV; i++) vf[i] = clean<TYPE>(vf[i], m, bad);
                }
                raise(up, sc, from, row);
                AttP<TYPE> p[NT];
#pragma unroll
                for (int t = 0; t < A::TL; t++) soften<TYPE, D>(t, sc[0][0][t], row[0], p[0]);
#pragma unroll
                for (int i = 0; i < A::NV; i++) weigh<TYPE, D>(vf[i], i, p, row);
                if (more) {
                    load_v(s + W);
                    if (s + 2 * W < n_step) pages(s + 2 * W);
                }
            }
        }
        /* the group's results on the largest of its references, then summed: four values of a row a thread */
        const float l = row_sum(row[0].l), mine = l != l ? INFINITY : row[0].ref;
        if (g == 0 && sub < busy) lds.m[wave][col] = mine;
        const bool wild = __syncthreads_or(bad != 0);
        const int first = group * W;
        float m = kLowest;
#pragma unroll
        for (int i = 0; i < W; i++)
            if (i < busy) m = fmaxf(m, lds.m[first + i][col]);
        if (sub < busy) {
            const float f = mine == kLowest ? 0.0f : exp2_fast(mine - m);
            if (g == 0) lds.l[wave][col] = l * f;
#pragma unroll
            for (int i = 0; i < D / 16; i++) *(f32x4 *)&lds.o[wave][col][16 * i + 4 * g] = row[0].o[i] * f;
        }
        if (sub == 0 && g == 0) lds.top[group][col] = m;
        __syncthreads();
        for (int rr = o_row; rr < n_row; rr += o_rows) {
            if (rr != o_row) {
                const int r = w.row + rr;
                o_tok = r / a.group;
                o_head = kvh * a.group + r % a.group;
                o_tk = toks[o_tok];
            }
            float ll = 0.0f;
            f32x4 o = { 0, 0, 0, 0 };
#pragma unroll
            for (int i = 0; i < W; i++) {
                if (i >= busy) continue;
                ll += lds.l[first + i][rr];
                o += *(const f32x4 *)&lds.o[first + i][rr][o_d];
            }
            if (__builtin_expect(wild, 0))
                o += wild_sum<TYPE, D>(a.v, tab, a.page_bytes, head_off, a.shift, w.full, min(o_tk.pos + 1, w.key1), o_d);
            put_row(a, o_tk, w, o_tok, o_head, o_d, D, lds.top[group][rr], ll, o, o_d == 0);
        }
        __syncthreads();
        join_tile<D, 64 * kFewWaves>(a, toks, w, kvh, lds.last);
    }
}

/* W 0: a captured call's, which reads how many when it runs. */
template <int TYPE, int D, int W>
__global__ __launch_bounds__(64 * kFewWaves, 2) void attn_few_kernel(AttnCall a)
{
    __shared__ FewLds<D> lds;
    const AttnHdr &h = header(a);
    if constexpr (W > 0) few_items<TYPE, D, W>(a, h, lds);
    else if (h.few_shift == 3) few_items<TYPE, D, 8>(a, h, lds);
    else if (h.few_shift == 2) few_items<TYPE, D, 4>(a, h, lds);
    else if (h.few_shift == 1) few_items<TYPE, D, 2>(a, h, lds);
    else few_items<TYPE, D, 1>(a, h, lds);
}

/* Many rows (128, fp32 64): four waves of one or two row tiles of 16 share tiles of keys and values, copied to
 * LDS by the LDS DMA, the next tile's copy in flight while one is worked on. Pieces are stored with their index in
 * the row xored by the row, so that the 16 rows a wave instruction reads lie in all banks (no conflicts).
 *
 * Bound: the matrix cores. Two row tiles a wave halve its LDS reads per product; the two blocks that a CU
 * holds have one wave each on a SIMD, one's softmax under the other's products. 2047 prompt tokens (64 heads on 4,
 * f16): 119 us, 575 TFLOP/s of the formula, 1150 on the f16 pipe with both halves (a large library product: 1072);
 * 509 tokens behind 16000: 202 us, 672 and 1344. The pipe is busy for two thirds of the cycles, at a clock that falls
 * to 1.9 GHz under this load. 32x32 instructions are slower on data than these (a loop of nothing else: 1680
 * against 1850 TFLOP/s). Up to 64 rows a wave has one row tile, since two waves with two leave two idle: 32
 * sequences of 4 drafted tokens (64 rows) over 4007 keys 29 / 37 us. */
constexpr int kManyThreads = 256;

template <int TYPE, int D>
struct ManyLds {
    static constexpr int KT = 2 * Att<TYPE, D>::KS;                 /* keys of a tile             */
    static constexpr int BYTES = KT * D * Att<TYPE, D>::ES;         /* of its keys, or its values */
};

template <int TYPE, int D>
__global__ __launch_bounds__(kManyThreads, 2) void attn_many_kernel(AttnCall a)
{
    using A = Att<TYPE, D>;
    using L = ManyLds<TYPE, D>;
    constexpr int NT = attn_rows(kAttnMany, TYPE) / 64, RC = D / A::CE, VC = L::KT / A::CE, NG = L::KT / 16;
    constexpr int NL = L::BYTES / 16 / kManyThreads;                /* pieces per thread          */
    constexpr int RP = D * A::ES >= 256 ? 1 : 256 / (D * A::ES);    /* key rows per 256 bytes     */
    static_assert(VC == 8, "a row of values is 128 bytes");
    __shared__ __align__(16) uint8_t lds[2][2][L::BYTES];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), P1 = (1 << a.shift) - 1;
    /* the wave's row tiles are tile + 4 n; the first tile's place turns with the block, since the blocks 256 apart share a CU */
    const int tile0 = (wave + (blockIdx.x >> 8) * 2) & 3;
    const AttnHdr &h = header(a);
    const int n_unit = h.n_run[kAttnMany] * a.kv_heads;
    const AttnWork *work = (const AttnWork *)(a.blob + h.work[kAttnMany]);
    const AttnTok *toks = (const AttnTok *)(a.blob + h.tok);
    for (int u = blockIdx.x, next = -1; next >= 0 || u < n_unit;) {
        const AttnWork w = work[next >= 0 ? next : u / a.kv_heads];
        const int kvh = u % a.kv_heads;
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));                               /* an item's addresses are not kept for the next one */
        const int lane = tid & 63, col = lane & 15, g = lane >> 4;
        next = w.next;
        if (next < 0) u += gridDim.x;
        const int32_t *tab = (const int32_t *)(a.blob + h.pages) + w.pages;
        const uint32_t head_off = (uint32_t)kvh * ((uint32_t)(D * A::ES) << a.shift);
        AttRaw<TYPE, D> raw[NT];
        int limit[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {                              /* rows behind the last one: its query, not stored */
            const int r = w.row + min(16 * (tile0 + 4 * n) + col, w.rows - 1), t = r / a.group;
            load_q<TYPE, D>(a.q + ((size_t)t * a.heads + (size_t)(kvh * a.group + r % a.group)) * D, g, raw[n]);
            limit[n] = min(toks[t].pos + 1, w.key1);
        }
        const int n_tile = (w.key1 - w.key0 + L::KT - 1) / L::KT, last = w.key1 - 1;
        /* the next tile's pages, loaded a tile ahead of their use: in lane i the page of keys 16 (i % NG) ..,
         * and the one of the values that the thread copies */
        const int v_piece = (tid & 7) ^ ((tid >> 4) & 7);
        int k_page = 0, v_page = 0;
        auto pages = [&](int tile) {
            const int key = w.key0 + tile * L::KT;
            k_page = tab[min(key + 16 * (lane % NG), last) >> a.shift];
            v_page = tab[min(key + v_piece * A::CE, last) >> a.shift];
        };
        auto copy = [&](int tile) {
            const int key = w.key0 + tile * L::KT;
            uint8_t *kd = lds[tile & 1][0], *vd = lds[tile & 1][1];
            constexpr int RI = kManyThreads / RC;                   /* key rows of one pass       */
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int r = i * RI + tid / RC;                     /* key row, and its 16 keys   */
                const int pg = __builtin_amdgcn_readlane(k_page, (i * RI + wave * (64 / RC)) / 16);
                const int m = TYPE == 1 ? (((r >> 3) & 3) << 2 | (r & 3)) : (r & 15);
                const int piece = (tid % RC) ^ (m / RP);
                const int slot = (key + r) & P1;
                dma_to_lds<16>(page_at(a.k, pg, a.page_bytes, head_off) + (uint32_t)(slot * D + piece * A::CE) * A::ES,
                               kd + (i * kManyThreads + wave * 64) * 16);
            }
            const int slot = (key + v_piece * A::CE) & P1;
            const uint8_t *p = page_at(a.v, v_page, a.page_bytes, head_off) + (uint32_t)(((tid >> 3) << a.shift) + slot) * A::ES;
            const uint32_t step = (uint32_t)(kManyThreads / 8 * A::ES) << a.shift;
#pragma unroll
            for (int i = 0; i < NL; i++) dma_to_lds<16>(p + i * step, vd + (i * kManyThreads + wave * 64) * 16);
        };
        if (n_tile > 0) {
            pages(0);
            copy(0);
            if (n_tile > 1) pages(1);
        }
        uint32_t bad = 0;
        const int n_own = (w.rows - 16 * tile0 + 63) / 64;          /* row tiles that hold rows */
        AttQ<TYPE, D> q[NT];
        AttRow<D> row[NT];
        float up[NT], from[NT] = {};
#pragma unroll
        for (int n = 0; n < NT; n++) up[n] = make_q<TYPE, D>(raw[n], a.scale_log2, q[n]);
        bool scaled = false;
#pragma unroll
        for (int n = 0; n < NT; n++) scaled = scaled || up[n] != 1.0f;
        const bool unit = __ballot(scaled) == 0;
        auto turn = [&](int tile) {                                 /* tile's copy is there, the next one starts */
            mx_wait_barrier();
            if (tile + 1 < n_tile) {
                copy(tile + 1);
                if (tile + 2 < n_tile) pages(tile + 2);
            }
        };
        /* Steps of a tile, from st0 on: all their scores first, so that one branch serves them. LDS reads run two
         * pieces of keys and four of values ahead of their products, and a step's softmax between the
         * products of the one before; the barriers keep the compiler from undoing that. */
        auto work_on = [&](auto masked, auto steps, auto own, int tile, int st0) {
            constexpr bool MASK = decltype(masked)::value;
            constexpr int NS = decltype(steps)::value, NA = decltype(own)::value, GK = NS * A::NCH, GV = NS * A::NV, KB = 3, VB = 4;
            const uint8_t *kr = lds[tile & 1][0] + (st0 * A::KS + (col >> 2) * A::CE + (col & 3)) * D * A::ES;
            const uint8_t *vr = lds[tile & 1][1] + col * 128;
            const int at = w.key0 + tile * L::KT + st0 * A::KS + g * A::CE;
            f32x4 sc[NS][NA][A::TL];
            u32x4 kb[KB][A::TL], vb[VB];
            auto read_k = [&](int j) {
#pragma unroll
                for (int t = 0; t < A::TL; t++)
                    kb[j % KB][t] = *(const u32x4 *)(kr + (j / A::NCH * A::KS + 4 * t) * D * A::ES + (((4 * (j % A::NCH) + g) ^ (col / RP)) * 16));
            };
            auto read_v = [&](int j) { vb[j % VB] = *(const u32x4 *)(vr + 2048 * (j % A::NV) + (((4 * (st0 + j / A::NV) + g) ^ ((col >> 1) & 7)) * 16)); };
            AttP<TYPE> p[2][NA];
            constexpr int PARTS = NA * A::TL;                       /* of a step's softmax */
            auto soft = [&](int st, int k) { soften<TYPE, D>(k % A::TL, sc[st][k / A::TL][k % A::TL], row[k / A::TL], p[st % 2][k / A::TL]); };
            __builtin_amdgcn_s_setprio(1);                          /* over the SIMD's other wave where that has its softmax */
#pragma unroll
            for (int st = 0; st < NS; st++) score_from(from, sc[st]);
#pragma unroll
            for (int j = 0; j < KB - 1; j++) read_k(j);
#pragma unroll
            for (int j = 0; j < GK; j++) {
                if (j + KB - 1 < GK) read_k(j + KB - 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < A::TL; t++) score<TYPE, D>(kb[j % KB][t], j % A::NCH, t, q, sc[j / A::NCH]);
            }
#pragma unroll
            for (int j = 0; j < VB; j++) read_v(j);
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(0);
            if (!unit) unscale(up, sc);
            if constexpr (MASK) {
#pragma unroll
                for (int st = 0; st < NS; st++)
#pragma unroll
                    for (int n = 0; n < NA; n++) hide(limit[n] - at - st * A::KS, sc[st][n]);
            }
            raise(up, sc, from, row);
#pragma unroll
            for (int k = 0; k < PARTS; k++) soft(0, k);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = 0; j < GV; j++) {
                const int st = j / A::NV, i = j % A::NV;
                u32x4 v = vb[j % VB];
                if constexpr (MASK) v = clean<TYPE>(v, piece_mask<TYPE>(w.full - at - st * A::KS, w.key1 - at - st * A::KS), bad);
                weigh<TYPE, D>(v, i, p[st % 2], row);
                if (j + VB < GV) read_v(j + VB);
                if (st + 1 < NS && i % (A::NV / PARTS) == 0) soft(st + 1, i / (A::NV / PARTS));
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
        };
        const int n_clear = max(0, w.full - w.key0) / L::KT;        /* tiles that every row sees whole */
        /* each wave runs the loop of its own row tiles: the barriers in it are as many */
        auto work_all = [&](auto own) {
            for (int tile = 0; tile < n_clear; tile++) {
                turn(tile);
                if (n_own > 0) work_on(std::false_type{}, std::integral_constant<int, 2>{}, own, tile, 0);
            }
#pragma unroll 1
            for (int tile = n_clear; tile < n_tile; tile++) {
                turn(tile);
                if (n_own <= 0) continue;
#pragma unroll 1
                for (int st = 0; st < 2; st++)
                    if (w.key0 + tile * L::KT + st * A::KS < w.key1) work_on(std::true_type{}, std::integral_constant<int, 1>{}, own, tile, st);
            }
        };
        if (NT == 1 || n_own >= NT) work_all(std::integral_constant<int, NT>{});
        else work_all(std::integral_constant<int, 1>{});
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float l = row_sum(row[n].l);
            const int i = 16 * (tile0 + 4 * n) + col, r = w.row + i, t = r / a.group, head = kvh * a.group + r % a.group;
            if (i >= w.rows) continue;
            const AttnTok tk = toks[t];
#pragma unroll
            for (int k = 0; k < D / 16; k++)
                put_row(a, tk, w, t, head, 16 * k + 4 * g, D, row[n].ref, l, row[n].o[k], k == 0 && g == 0);
            if (__builtin_expect(__ballot(bad) != 0, 0)) {
                float *o = row_out(a, tk, w.part, t, head, D);
#pragma unroll 1
                for (int d = 4 * g; d < D; d += 16) {
                    const f32x4 e = wild_sum<TYPE, D>(a.v, tab, a.page_bytes, head_off, a.shift, w.full, limit[n], d);
                    *(f32x4 *)(o + d) += e;
                }
            }
        }
        __syncthreads();                                            /* the buffers, before the next item */
    }
}

/* Parts of a row joined: out = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p. PL lanes of D / 4 threads take
 * every PL-th part in slot order, then lane 0 takes the lanes' results in theirs.
 *
 * Bound: latency, then the parts' bytes (16384 rows of 4 or 5 parts 7.8 us). */
template <int D, int PL>
__device__ __forceinline__ void join_rows(const AttnCall &a, const AttnHdr &h, f32x4 (*s_o)[D / 4], float (*s_ml)[2])
{
    constexpr int TPR = D / 4, RPB = 256 / (TPR * PL);
    const int n = h.n_comb * a.heads, d = threadIdx.x % TPR, pl = threadIdx.x / TPR % PL, rb = threadIdx.x / (TPR * PL);
    const int32_t *comb = (const int32_t *)(a.blob + h.comb);
    const AttnTok *toks = (const AttnTok *)(a.blob + h.tok);
    for (int i0 = blockIdx.x * RPB; i0 < n; i0 += gridDim.x * RPB) {
        const int i = min(i0 + rb, n - 1), t = comb[i / a.heads], head = i % a.heads;
        const AttnTok tk = toks[t];
        const size_t r0 = (size_t)tk.part * a.heads + head;
        AttJoin j;
        for (int p = pl; p < tk.parts; p += 4 * PL) {               /* four parts' loads at a time */
            f32x2 ml[4];
            f32x4 o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const size_t r = r0 + (size_t)min(p + k * PL, tk.parts - 1) * a.heads;
                ml[k] = *(const f32x2 *)(a.part_ml + 2 * r);
                o[k] = *(const f32x4 *)(a.part_o + r * D + 4 * d);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (p + k * PL < tk.parts) j.add(ml[k].x, ml[k].y, o[k]);
        }
        if constexpr (PL > 1) {
            s_o[rb * PL + pl][d] = j.o;
            if (d == 0) {
                s_ml[rb * PL + pl][0] = j.m;
                s_ml[rb * PL + pl][1] = j.l;
            }
            __syncthreads();
            if (pl == 0)
                for (int k = 1; k < PL; k++) j.add(s_ml[rb * PL + k][0], s_ml[rb * PL + k][1], s_o[rb * PL + k][d]);
            __syncthreads();
        }
        if (pl == 0 && i0 + rb < n) *(f32x4 *)(a.out + ((size_t)t * a.heads + head) * D + 4 * d) = j.o * (1.0f / j.l);
    }
}

/* One lane up to 16 parts (four rounds of loads), else eight. us by one / eight lanes: 2560 rows of up to 11 parts 4.7 /
 * 6.7; 64 rows of 63 parts 15.5 / 4.2, 256 of 79 19.0 / 5.2. */
constexpr int kJoinLanes = 8;
__host__ __device__ inline int join_lanes(const AttnHdr &h) { return h.max_parts > 16 ? kJoinLanes : 1; }

template <int D>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnCall a)
{
    __shared__ __align__(16) f32x4 s_o[256 / (D / 4)][D / 4];
    __shared__ float s_ml[256 / (D / 4)][2];
    const AttnHdr &h = header(a);
    if (join_lanes(h) > 1) join_rows<D, kJoinLanes>(a, h, s_o, s_ml);
    else join_rows<D, 1>(a, h, s_o, s_ml);
}

/* Head norms, rotation and the append. Units of 16 (D 128) or 32 (D 64) heads of one token: D / 8 lanes a
 * head, each with four elements and their four partners half a head away, so that the norm's sum and
 * the rotation stay in the lanes. Values go through LDS in tiles of up to 32 tokens of one page, so that
 * their transposed rows are stored in runs.
 *
 * Bound: bytes for many tokens (2047 of 64 + 2 x 4 heads: 28 us, 5.2 TB/s, a large copy's rate), the launch for
 * few (one token 2.8 us, 64 tokens 4.1). One launch for q, k and v: three would cost more than the work. */
template <int TYPE, int D>
__global__ __launch_bounds__(256) void attn_append_kernel(AttnAppend b)
{
    constexpr int LPH = D / 8, HPB = 256 / LPH;
    constexpr int ES = Att<TYPE, D>::ES;
    __shared__ float s_v[kVTile][D + 1];
    const AttnCall &a = b.c;
    const AttnHdr &h = header(a);
    const AttnTok *toks = (const AttnTok *)(a.blob + h.tok);
    const int n_head = (b.q ? a.heads : 0) + a.kv_heads, passes = (n_head + HPB - 1) / HPB;
    const int n_qk = h.n_tok * passes, n_unit = n_qk + h.n_vt * a.kv_heads;
    const int P1 = (1 << a.shift) - 1;
    for (int u = blockIdx.x; u < n_unit; u += gridDim.x) {
        if (u < n_qk) {
            const int t = u / passes, hd = u % passes * HPB + threadIdx.x / LPH, i0 = threadIdx.x % LPH * 4;
            if (hd >= n_head) continue;
            const AttnTok tk = toks[t];
            const bool is_k = hd >= n_head - a.kv_heads;
            const int kvh = hd - (n_head - a.kv_heads);
            const float *x = is_k ? b.k + ((size_t)t * a.kv_heads + kvh) * D : b.q + ((size_t)t * a.heads + hd) * D;
            f32x4 lo = *(const f32x4 *)(x + i0), hi = *(const f32x4 *)(x + D / 2 + i0);
            if (b.norm) {
                const float *wt = is_k ? b.kw : b.qw;
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; e++) ss = __builtin_fmaf(lo[e], lo[e], __builtin_fmaf(hi[e], hi[e], ss));
#pragma unroll
                for (int o = 1; o < LPH; o *= 2) ss += __shfl_xor(ss, o);
                const float inv = 1.0f / sqrtf(ss / D + b.eps);
                lo *= inv;
                hi *= inv;
                if (wt) {
                    lo *= *(const f32x4 *)(wt + i0);
                    hi *= *(const f32x4 *)(wt + D / 2 + i0);
                }
            }
            f32x4 y0, y1;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                /* the angle in turns, in double: far positions keep their fraction of a turn */
                const double turns = (double)tk.pos * b.freq[i0 + e];
                float sn, cs;
                sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
                y0[e] = lo[e] * cs - hi[e] * sn;
                y1[e] = hi[e] * cs + lo[e] * sn;
            }
            if (!is_k) {
                float *y = b.qr + ((size_t)t * a.heads + hd) * D;
                *(f32x4 *)(y + i0) = y0;
                *(f32x4 *)(y + D / 2 + i0) = y1;
            } else {
                uint8_t *y = const_cast<uint8_t *>(page_at(a.k, tk.dst >> a.shift, a.page_bytes, (uint32_t)kvh * ((uint32_t)(D * ES) << a.shift))) +
                             (uint32_t)((tk.dst & P1) * D + i0) * ES;
                if constexpr (TYPE == 0) {
                    *(f32x4 *)y = y0;
                    *(f32x4 *)(y + D / 2 * ES) = y1;
                } else {
                    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
                    *(h4 *)y = __builtin_convertvector(y0, h4);
                    *(h4 *)(y + D / 2 * ES) = __builtin_convertvector(y1, h4);
                }
            }
        } else {
            const int kvh = (u - n_qk) % a.kv_heads;
            const AttnVTile vt = ((const AttnVTile *)(a.blob + h.vt))[(u - n_qk) / a.kv_heads];
            uint8_t *y = const_cast<uint8_t *>(page_at(a.v, vt.page, a.page_bytes, (uint32_t)kvh * ((uint32_t)(D * ES) << a.shift)));
            auto put = [&](int d, int slot, float v) {
                const uint32_t off = ((uint32_t)d << a.shift) + (uint32_t)slot;
                if constexpr (TYPE == 0) *(float *)(y + off * ES) = v;
                else *(_Float16 *)(y + off * ES) = (_Float16)v;
            };
            const float *x = b.v + ((size_t)vt.tok * a.kv_heads + kvh) * D;
            if (vt.n == 1) {
                if (threadIdx.x < D) put(threadIdx.x, vt.slot, x[threadIdx.x]);
                continue;
            }
            for (int e = threadIdx.x; e < vt.n * (D / 4); e += 256) {
                const f32x4 v = *(const f32x4 *)(x + (size_t)(e / (D / 4)) * a.kv_heads * D + e % (D / 4) * 4);
#pragma unroll
                for (int j = 0; j < 4; j++) s_v[e / (D / 4)][e % (D / 4) * 4 + j] = v[j];
            }
            __syncthreads();
            for (int e = threadIdx.x; e < kVTile * D; e += 256)
                if (e % kVTile < vt.n) put(e / kVTile, vt.slot + e % kVTile, s_v[e % kVTile][e / kVTile]);
            __syncthreads();
        }
    }
}

template <int TYPE, int D>
hipError_t attend(const AttnCall &a, int grid, hipStream_t st)
{
    const int groups = kFewWaves >> a.h.few_shift;
    const int nb[kAttnKinds] = { a.live ? grid : (a.h.n_run[0] * a.kv_heads + groups - 1) / groups, a.live ? grid : a.h.n_run[1] * a.kv_heads };
    if (nb[kAttnMany]) QLAUNCH("attend", (attn_many_kernel<TYPE, D>), dim3((unsigned)nb[kAttnMany]), dim3(kManyThreads), 0, st, a);
    if (nb[kAttnFew]) {
        auto few = [&](auto waves) {
            QLAUNCH("attend", (attn_few_kernel<TYPE, D, decltype(waves)::value>), dim3((unsigned)nb[kAttnFew]), dim3(64 * kFewWaves), 0, st, a);
        };
        if (a.live) few(std::integral_constant<int, 0>{});
        else if (a.h.few_shift == 3) few(std::integral_constant<int, 8>{});
        else if (a.h.few_shift == 2) few(std::integral_constant<int, 4>{});
        else if (a.h.few_shift == 1) few(std::integral_constant<int, 2>{});
        else few(std::integral_constant<int, 1>{});
    }
    const int rpb = 256 / (D / 4 * join_lanes(a.h)), nj = a.live ? grid : (a.h.n_comb * a.heads + rpb - 1) / rpb;
    if (nj) QLAUNCH("join", (attn_join_kernel<D>), dim3((unsigned)nj), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attend(const AttnCall &a, int type, int D, int grid, hipStream_t st)
{
    if (type == 1) return D == 128 ? attend<1, 128>(a, grid, st) : attend<1, 64>(a, grid, st);
    return D == 128 ? attend<0, 128>(a, grid, st) : attend<0, 64>(a, grid, st);
}

hipError_t launch_attn_append(const AttnAppend &b, int type, int D, int grid, hipStream_t st)
{
    const int hpb = 256 / (D / 8), n_head = (b.q ? b.c.heads : 0) + b.c.kv_heads;
    const int units = b.c.h.n_tok * ((n_head + hpb - 1) / hpb) + b.c.h.n_vt * b.c.kv_heads;
    const dim3 nb((unsigned)(b.c.live ? grid : units));
    if (type == 1 && D == 128) QLAUNCH("append", (attn_append_kernel<1, 128>), nb, dim3(256), 0, st, b);
    else if (type == 1) QLAUNCH("append", (attn_append_kernel<1, 64>), nb, dim3(256), 0, st, b);
    else if (D == 128) QLAUNCH("append", (attn_append_kernel<0, 128>), nb, dim3(256), 0, st, b);
    else QLAUNCH("append", (attn_append_kernel<0, 64>), nb, dim3(256), 0, st, b);
    return hipGetLastError();
}

}  // namespace qmsg
