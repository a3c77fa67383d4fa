"""Attention batches for the tests: page tables, the cache's layout, and everything in float64 from the formulas."""
import numpy as np

F16, F32 = 1, 0
EPS32 = 2.0 ** -24          # half a step of fp32, relative


def dtype_of(type_):
    return np.float16 if type_ == F16 else np.float32


class Batch:
    """Sequences of (new tokens, all tokens) on dealt pages; the first ``shared`` tokens on common pages for the
    sequences of each run of ``runs`` (all of them by default)."""

    def __init__(self, lens, page, shared=0, runs=None, seed=0, spare=2):
        rng = np.random.default_rng(seed)
        self.q, self.kv, self.page = [a for a, _ in lens], [b for _, b in lens], page
        n = len(lens)
        runs = [n] if runs is None else runs
        ns = shared // page
        need = [-(-b // page) for b in self.kv]
        self.n_page = sum(need) + ns * len(runs) + spare
        deal = list(rng.permutation(self.n_page))
        self.max_pages = max(need + [1])
        self.pages = np.full((n, self.max_pages), -1, np.int32)
        i = 0
        for run in runs:
            common = [deal.pop() for _ in range(ns)]
            for _ in range(run):
                for j in range(need[i]):
                    self.pages[i, j] = common[j] if j < ns else deal.pop()
                i += 1
        self.free = deal                                  # pages of no sequence
        self.T = sum(self.q)
        self.seq = np.concatenate([np.full(a, s) for s, a in enumerate(self.q)] + [np.zeros(0)]).astype(int)
        self.pos = np.concatenate([np.arange(b - a, b) for a, b in lens] + [np.zeros(0)]).astype(int)


def pack(batch, k, v, heads, D, type_, fill=np.nan):
    """Pools holding k, v (per sequence [kv][heads][D]); every other slot holds `fill`."""
    P, dt = batch.page, dtype_of(type_)
    kp = np.full((batch.n_page, heads, P, D), fill, dt)
    vp = np.full((batch.n_page, heads, D, P), fill, dt)
    for s, n in enumerate(batch.kv):
        for j in range(n):
            kp[batch.pages[s, j // P], :, j % P] = k[s][j]
            vp[batch.pages[s, j // P], :, :, j % P] = v[s][j]
    return kp, vp


def values(batch, heads, D, type_, seed, shared=0, runs=None, scale=1.0):
    """Random k, v per sequence, as the cache's type holds them; shared tokens equal within a run."""
    rng = np.random.default_rng(seed)
    dt = dtype_of(type_)
    k = [(scale * rng.standard_normal((n, heads, D))).astype(dt) for n in batch.kv]
    v = [rng.standard_normal((n, heads, D)).astype(dt) for n in batch.kv]
    i = 0
    for run in ([len(batch.kv)] if runs is None else runs):
        for s in range(i + 1, i + run):
            k[s][:shared], v[s][:shared] = k[i][:shared], v[i][:shared]
        i += run
    return k, v


def attend64(batch, q, k, v, scale):
    """The attention in float64 and, per output element, how far fp32 arithmetic may be from it.

    With e = 2^-24, n keys, u_j = scale * sum_i |q_i k_ji|: a score's D products and its D + 8 roundings (the two halves of
    a split q included) move it by at most (D + 8) e u_j, taking it to powers of two and off the reference by 4 e (|s_j| +
    max |s|) more; exp2 gives 2 steps, a p split into two f16, each rounded to nearest, leaves 2^-22 of it (2^-20 allowed), and n sums in each of numerator
    and denominator 2 n e, a few more in joining parts. Relative to sum p |v| / sum p, first order, doubled for
    what products of these errors add."""
    T, H, D = q.shape
    out, tol = np.zeros((T, H, D)), np.zeros((T, H, D))
    for t in range(T):
        s, n = batch.seq[t], batch.pos[t] + 1
        heads = k[s].shape[1]
        G = H // heads
        for g in range(heads):
            K, V = k[s][:n, g].astype(np.float64), v[s][:n, g].astype(np.float64)
            x = q[t, g * G:(g + 1) * G].astype(np.float64)
            with np.errstate(all="ignore"):
                sc = scale * (x @ K.T)
                u = scale * (np.abs(x) @ np.abs(K).T)
                p = np.exp(sc - sc.max(-1, keepdims=True))
                l = p.sum(-1, keepdims=True)
                out[t, g * G:(g + 1) * G] = (p @ V) / l
                ds = (D + 8) * EPS32 * u + 4 * EPS32 * (np.abs(sc) + np.abs(sc).max(-1, keepdims=True))
                rel = ds + 2.0 ** -20 + 2.0 ** -22 + (n + 64) * EPS32
                a = ((p * rel) @ np.abs(V)) / l + (p @ np.abs(V)) / l * ((p * rel).sum(-1, keepdims=True) / l)
                tol[t, g * G:(g + 1) * G] = 2 * a
    return out, tol


def rotate64(x, w, pos, base, eps, norm=True):
    """Normed and rotated heads x [T][H][D] in float64."""
    x = x.astype(np.float64)
    D = x.shape[-1]
    if norm:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if w is not None:
            x = x * w.astype(np.float64)
    a = np.asarray(pos, np.float64)[:, None] * np.float64(np.float32(base)) ** (-2.0 * np.arange(D // 2) / D)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)


def rotate_tol(x, w, pos, base, eps, D, norm=True):
    """How far an element's fp32 norm and rotation may be off: the norm's sum and root (D/2 + 8 roundings, halved by the root,
    then 3), sine and cosine to 2 steps of an angle kept to 2^-24 of a turn in [-1/2, 1/2] (an angle error of 2 pi 2^-26), the
    products' 3, on |lo| + |hi| of the pair."""
    y = np.abs(rotate64(x, w, np.zeros(len(pos)), base, eps, norm))
    pair = y[..., :D // 2] + y[..., D // 2:]
    return np.concatenate([pair, pair], -1) * ((D / 4 + 4 + 3 + 4 + 3 + 2 * np.pi / 4) * EPS32) + 1e-37
