"""Head norms, rotation and the append to the cache on the GPU against float64, and whole steps: append, attend, graphs."""
import ctypes

import numpy as np
import pytest

from attn_cases import EPS32, F16, F32, Batch, attend64, dtype_of, pack, rotate64, rotate_tol, values
from test_gpu_attn import TINY, Pool, check
from test_gpu_dense_capture import hip_lib

pytestmark = pytest.mark.gpu
BASE, EPS = 1e6, 1e-6


@pytest.fixture(scope="module")
def ctx():
    from large_model_amd import qmsg
    with qmsg.Context(*TINY, n_layer=1, max_tokens=1) as c:
        yield c


class Rows:
    """Random q, k, v rows of a batch on the device."""

    def __init__(self, ctx, T, H, kv, D, seed):
        rng = np.random.default_rng(seed)
        self.q, self.k, self.v = (rng.standard_normal((T, n, D)).astype(np.float32) for n in (H, kv, kv))
        self.k *= 3
        self.d = [ctx.device_alloc(a.nbytes + 16) for a in (self.q, self.k, self.v)]
        for p, a in zip(self.d, (self.q, self.k, self.v)):
            ctx.h2d(p, a)


def half_step(type_, x):
    """What rounding to the cache's type may move x by (subnormals of f16: 2^-25)."""
    return np.maximum(np.abs(x) * 2.0 ** -11, 2.0 ** -25) if type_ == F16 else np.zeros_like(x)


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads", [(14, 2, 64), (16, 16, 128), (64, 4, 128), (5, 5, 64), (40, 8, 64)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("lens,page", [([(1, 1)], 16), ([(1, 4321), (1, 64), (0, 30), (1, 65)], 64), ([(77, 77), (1, 9), (150, 1000)], 128),
                                       ([(5, 20), (33, 100), (2, 16), (64, 64)], 16), ([(70, 70 + 250)], 256)])
def test_append(ctx, lens, page, heads, type_):
    H, kv, D = heads
    print(f"[case] append {lens} pages of {page} {heads} type {type_}", flush=True)
    b = Batch(lens, page, seed=1)
    pool = Pool(ctx, H, kv, D, type_, b, n_layer=2, rope_base=BASE)
    rng = np.random.default_rng(2)
    qw, kw = (1 + 0.3 * rng.standard_normal((2, D))).astype(np.float32)
    ctx.attn_norms(pool.id, 1, qw, kw)
    r = Rows(ctx, b.T, H, kv, D, 3)
    shape = (2, b.n_page, kv, page, D), (2, b.n_page, kv, D, page)
    before = [rng.standard_normal(s).astype(dtype_of(type_)) for s in shape]
    ctx.h2d(pool.k, before[0])
    ctx.h2d(pool.v, before[1])
    d_qr = ctx.device_alloc(r.q.nbytes + 4096)
    ctx.h2d(d_qr, np.full(r.q.size + 1024, 7.0, np.float32))
    ctx.attn_batch(pool.id, b.q, b.kv, b.pages)
    ctx.attn_append_device(pool.id, 1, d_qr, *r.d, EPS)
    ctx.sync()
    qr = ctx.d2h(d_qr, r.q.size + 1024)
    assert np.all(qr[r.q.size:] == 7.0)
    check(qr[:r.q.size].reshape(r.q.shape), rotate64(r.q, qw, b.pos, BASE, EPS), rotate_tol(r.q, qw, b.pos, BASE, EPS, D))
    kp, vp = ctx.d2h(pool.k, shape[0], dtype_of(type_)), ctx.d2h(pool.v, shape[1], dtype_of(type_))
    pg, sl = b.pages[b.seq, b.pos // page], b.pos % page
    k64 = rotate64(r.k, kw, b.pos, BASE, EPS)
    check(kp[1][pg, :, sl].astype(np.float64), k64, (rotate_tol(r.k, kw, b.pos, BASE, EPS, D) + half_step(type_, k64)) * 1.001)
    assert np.array_equal(vp[1][pg, :, :, sl], r.v.astype(dtype_of(type_)))
    kp[1][pg, :, sl], vp[1][pg, :, :, sl] = before[0][1][pg, :, sl], before[1][1][pg, :, :, sl]
    assert np.array_equal(kp, before[0]) and np.array_equal(vp, before[1]), "other slots were written"


@pytest.mark.parametrize("base", [1e4, 1e6])
def test_far_positions(ctx, base):
    H, kv, D, page = 4, 2, 128, 256
    b = Batch([(3, 3)], page, seed=4)
    n_page, far = 8192, 8192 * 256 - 5                     # two million tokens
    pool_pages = np.zeros((1, n_page), np.int32)
    pool_pages[0] = np.arange(n_page)
    print(f"[case] position {far}, base {base}", flush=True)
    from large_model_amd import qmsg
    with qmsg.Context(*TINY, n_layer=1, max_tokens=1) as c:
        i = c.attn_create(H, kv, D, page=page, n_page=n_page, max_pages=n_page, max_tokens=3, rope_base=base, qk_norm=False)
        r = Rows(c, 3, H, kv, D, 5)
        c.attn_batch(i, [3], [far + 3], pool_pages)
        c.attn_append_device(i, 0, r.d[0], r.d[0], r.d[1], r.d[2], EPS)          # in place
        c.sync()
        pos = far + np.arange(3)
        check(c.d2h(r.d[0], r.q.shape), rotate64(r.q, None, pos, base, EPS, False), rotate_tol(r.q, None, pos, base, EPS, D, False))


def test_keys_and_values_only_and_unit_weights(ctx):
    H, kv, D = 8, 2, 64
    b = Batch([(9, 30)], 16, seed=6)
    pool = Pool(ctx, H, kv, D, F32, b, rope_base=1e4)
    r = Rows(ctx, b.T, H, kv, D, 7)
    print("[case] no queries, unit weights", flush=True)
    ctx.attn_batch(pool.id, b.q, b.kv, b.pages)
    ctx.attn_append_device(pool.id, 0, None, None, r.d[1], r.d[2], EPS)
    ctx.sync()
    kp = ctx.d2h(pool.k, (b.n_page, kv, 16, D))
    got = kp[b.pages[b.seq, b.pos // 16], :, b.pos % 16]
    check(got, rotate64(r.k, None, b.pos, 1e4, EPS), rotate_tol(r.k, None, b.pos, 1e4, EPS, D))


def test_norm_of_odd_rows(ctx):
    """Zero, tiny and large heads."""
    H, kv, D = 8, 2, 128
    b = Batch([(4, 4)], 16, seed=8)
    pool = Pool(ctx, H, kv, D, F32, b, rope_base=1e4)
    r = Rows(ctx, b.T, H, kv, D, 9)
    r.q[0] = 0
    r.q[1] *= 1e-15
    r.q[2] *= 1e15
    ctx.h2d(r.d[0], r.q)
    print("[case] odd heads", flush=True)
    ctx.attn_batch(pool.id, b.q, b.kv, b.pages)
    ctx.attn_append_device(pool.id, 0, r.d[0], r.d[0], r.d[1], r.d[2], EPS)
    ctx.sync()
    check(ctx.d2h(r.d[0], r.q.shape), rotate64(r.q, None, b.pos, 1e4, EPS), rotate_tol(r.q, None, b.pos, 1e4, EPS, D))


@pytest.mark.parametrize("type_", [F16, F32])
def test_steps_of_a_batch(ctx, type_):
    """A prompt each, then tokens one, two and three at a time: every step against the whole history in float64 (keys and
    values as the cache holds them, so that only the attention's own arithmetic is judged)."""
    H, kv, D, page = 14, 2, 64, 16
    steps = [[40, 0, 17], [1, 33, 1], [3, 1, 2], [1, 1, 0], [2, 1, 1]]
    total = [sum(s[i] for s in steps) for i in range(3)]
    b = Batch([(1, n) for n in total], page, seed=10)
    b.T = 64
    pool = Pool(ctx, H, kv, D, type_, b, rope_base=1e4)
    ctx.h2d(pool.k, np.full((b.n_page, kv, page, D), np.nan, dtype_of(type_)))
    ctx.h2d(pool.v, np.full((b.n_page, kv, page, D), np.nan, dtype_of(type_)))
    at = [0, 0, 0]
    for n, new in enumerate(steps):
        print(f"[case] step {n}: {new}, type {type_}", flush=True)
        at = [a + x for a, x in zip(at, new)]
        now = Batch([(x, a) for x, a in zip(new, at)], page)
        now.pages = b.pages
        r = Rows(ctx, now.T, H, kv, D, 100 + n)
        d_o = ctx.device_alloc(r.q.nbytes)
        ctx.attn_batch(pool.id, now.q, now.kv, b.pages)
        ctx.attn_append_device(pool.id, 0, r.d[0], *r.d, EPS)
        ctx.attn_device(pool.id, 0, r.d[0], d_o)
        ctx.sync()
        kp, vp = ctx.d2h(pool.k, (b.n_page, kv, page, D), dtype_of(type_)), ctx.d2h(pool.v, (b.n_page, kv, D, page), dtype_of(type_))
        k = [np.stack([kp[b.pages[s, j // page], :, j % page] for j in range(a)]) if a else np.zeros((0, kv, D)) for s, a in enumerate(at)]
        v = [np.stack([vp[b.pages[s, j // page], :, :, j % page] for j in range(a)]) if a else np.zeros((0, kv, D)) for s, a in enumerate(at)]
        q = ctx.d2h(r.d[0], r.q.shape)
        check(ctx.d2h(d_o, r.q.shape), *attend64(now, q, k, v, D ** -0.5))


@pytest.mark.parametrize("type_", [F16, F32])
def test_graph_follows_the_batch(ctx, type_):
    """Append and attention captured once, replayed on other batches: eager calls' bits each time."""
    hip, vp = hip_lib(), ctypes.c_void_p
    H, kv, D, page = 32, 4, 128, 16
    shared = Batch([(1, 6500), (1, 6600), (1, 6470)], page, 6416, seed=11)        # 26 MB of keys and values saved
    batches = [Batch([(1, 300), (1, 17), (1, 600)], page, seed=12), Batch([(1, 301), (1, 18), (1, 601)], page, seed=12), shared,
               Batch([(20, 50), (1, 3), (0, 9)], page, seed=13), Batch([(0, 0), (0, 4)], page, seed=14), Batch([(2, 2000)], page, seed=15)]
    top = Batch([(1, 1)], page)
    top.n_page, top.T, top.max_pages, top.q = max(b.n_page for b in batches), 32, 420, [0] * 3
    pool = Pool(ctx, H, kv, D, type_, top, rope_base=1e4)
    rng = np.random.default_rng(16)
    pools = [rng.standard_normal((top.n_page, kv, page, D)).astype(dtype_of(type_)) for _ in range(2)]
    r = Rows(ctx, 32, H, kv, D, 17)
    d_qr, d_o = ctx.device_alloc(r.q.nbytes), ctx.device_alloc(r.q.nbytes)
    st = vp(ctx_stream(ctx))

    def both():
        ctx.attn_append_device(pool.id, 0, d_qr, *r.d, EPS)
        ctx.attn_device(pool.id, 0, d_qr, d_o)

    def result(run):
        ctx.h2d(pool.k, pools[0])
        ctx.h2d(pool.v, pools[1])
        for d in (d_qr, d_o):
            ctx.h2d(d, np.full(r.q.shape, 5.0, np.float32))
        run()
        ctx.sync()
        return [ctx.d2h(d, r.q.shape) for d in (d_qr, d_o)] + [ctx.d2h(p, pools[0].shape, dtype_of(type_)) for p in (pool.k, pool.v)]

    graph, exe = vp(), vp()
    ctx.attn_batch(pool.id, batches[0].q, batches[0].kv, batches[0].pages)
    print("[case] capture", flush=True)
    assert hip.hipStreamBeginCapture(st, 2) == 0
    both()
    from large_model_amd import qmsg
    with pytest.raises(qmsg.QmsgError, match="capturing"):
        ctx.attn_batch(pool.id, batches[1].q, batches[1].kv, batches[1].pages)
    assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
    try:
        for n, b in enumerate(batches + batches[:2]):
            print(f"[case] batch {n}", flush=True)
            ctx.attn_batch(pool.id, b.q, b.kv, b.pages)
            want = result(both)
            for _ in range(2):
                got = result(lambda: hip.hipGraphLaunch(exe, st))
                assert all(np.array_equal(x, y) for x, y in zip(got, want)), n
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


@pytest.mark.parametrize("type_", [F16, F32])
def test_graph_of_few_and_many_sequences(ctx, type_):
    """An attention captured once: batches whose items have one to eight waves, joined or not, long after short."""
    hip, vp = hip_lib(), ctypes.c_void_p
    H, kv, D, page = 16, 16, 128, 16
    batches = [Batch([(1, 700), (1, 33)], page, seed=31), Batch([(1, 20)] * 260, page, seed=32), Batch([(1, 1 + i % 90) for i in range(259)], page, seed=33),
               Batch([(1, 130)] * 40, page, seed=34), Batch([(1, 3000)], page, seed=35), Batch([(1, 5)] * 3, page, seed=36)]
    top = Batch([(1, 1)] * 260, page)
    top.n_page, top.max_pages = max(b.n_page for b in batches), 190
    pool = Pool(ctx, H, kv, D, type_, top)
    rng = np.random.default_rng(37)
    for d in (pool.k, pool.v):
        ctx.h2d(d, rng.standard_normal((top.n_page, kv, page, D)).astype(dtype_of(type_)))
    r = Rows(ctx, 260, H, kv, D, 38)
    d_o = ctx.device_alloc(r.q.nbytes)
    st, graph, exe = vp(ctx_stream(ctx)), vp(), vp()

    def result(run):
        ctx.h2d(d_o, np.full(r.q.shape, 5.0, np.float32))
        run()
        ctx.sync()
        return ctx.d2h(d_o, r.q.shape)

    attend = lambda: ctx.attn_device(pool.id, 0, r.d[0], d_o)
    ctx.attn_batch(pool.id, batches[0].q, batches[0].kv, batches[0].pages)
    assert hip.hipStreamBeginCapture(st, 2) == 0
    attend()
    assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
    try:
        for n, b in enumerate(batches + batches[::-1]):
            print(f"[case] batch {n}", flush=True)
            ctx.attn_batch(pool.id, b.q, b.kv, b.pages)
            want = result(attend)
            assert np.all(want[b.T:] == 5.0)
            for _ in range(2):
                assert np.array_equal(result(lambda: hip.hipGraphLaunch(exe, st)), want), n
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


def ctx_stream(ctx):
    from large_model_amd import qmsg
    return qmsg.lib.qmsg_stream(ctx._h)


def test_two_attentions_on_one_cache(ctx):
    """Two batches in flight on a shared pool, two contexts (streams), the second's own plan and workspace."""
    from large_model_amd import qmsg
    H, kv, D, page = 32, 4, 128, 64
    b = Batch([(1, 900), (1, 1200)], page, seed=18)
    k, v = values(b, kv, D, F16, 19)
    kp, vp = pack(b, k, v, kv, D, F16)
    one = Pool(ctx, H, kv, D, F16, b)
    ctx.h2d(one.k, kp)
    ctx.h2d(one.v, vp)
    q = np.random.default_rng(20).standard_normal((2, 2, H, D)).astype(np.float32)
    want, tol = zip(*(attend64(b, q[i], k, v, D ** -0.5) for i in range(2)))
    print("[case] two contexts", flush=True)
    with qmsg.Context(*TINY, n_layer=1, max_tokens=1) as other:
        i = other.attn_create(H, kv, D, page=page, n_page=b.n_page, max_seq=2, max_tokens=2, max_pages=b.max_pages, d_k=one.k, d_v=one.v)
        assert other.attn_cache(i) == (one.k, one.v)
        pairs = [(ctx, one.id), (other, i)]
        d = [(c.device_alloc(q[0].nbytes), c.device_alloc(q[0].nbytes)) for c, _ in pairs]
        for n, (c, a) in enumerate(pairs):
            c.h2d(d[n][0], q[n])
            c.attn_batch(a, b.q, b.kv, b.pages)
            c.sync()
        for _ in range(10):
            for n, (c, a) in enumerate(pairs):
                c.attn_device(a, 0, *d[n])
        for n, (c, a) in enumerate(pairs):
            c.sync()
            check(c.d2h(d[n][1], q[n].shape), want[n], tol[n])
