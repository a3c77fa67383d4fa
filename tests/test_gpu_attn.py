"""Attention over the paged cache on the GPU against float64: head layouts, lengths, pages, masks, shared prefixes."""
import numpy as np
import pytest

from attn_cases import EPS32, F16, F32, Batch, attend64, dtype_of, pack, values

pytestmark = pytest.mark.gpu

TINY = (256, 16, 4, 128)


@pytest.fixture(scope="module")
def ctx():
    from large_model_amd import qmsg
    with qmsg.Context(*TINY, n_layer=1, max_tokens=1) as c:
        yield c


class Pool:
    """An attention and its pools in the context, device rows for a batch."""

    def __init__(self, ctx, heads, kv_heads, D, type_, batch, n_layer=1, **kw):
        self.ctx, self.H, self.D, self.b = ctx, heads, D, batch
        self.id = ctx.attn_create(heads, kv_heads, D, type_=type_, page=batch.page, n_page=batch.n_page, n_layer=n_layer,
                                  max_seq=max(1, len(batch.q)), max_tokens=max(1, batch.T), max_pages=batch.max_pages, **kw)
        self.k, self.v = ctx.attn_cache(self.id)

    def run(self, q, kp, vp, layer=0):
        """out [T][H][D] with rows of a canary behind it, which have to stay."""
        ctx, b = self.ctx, self.b
        ctx.h2d(self.k + layer * kp.nbytes, kp)
        ctx.h2d(self.v + layer * vp.nbytes, vp)
        d_q, d_o = ctx.device_alloc(q.nbytes + 16), ctx.device_alloc(q.nbytes + 4096)
        ctx.h2d(d_q, q)
        ctx.h2d(d_o, np.full(q.size + 1024, 7.0, np.float32))
        ctx.attn_batch(self.id, b.q, b.kv, b.pages)
        ctx.attn_device(self.id, layer, d_q, d_o)
        ctx.sync()
        o = ctx.d2h(d_o, q.size + 1024)
        assert np.all(o[q.size:] == 7.0), "rows behind the batch were written"
        return o[:q.size].reshape(q.shape)


def check(got, want, tol):
    assert np.array_equal(np.isnan(got), np.isnan(want)) or np.all(np.isfinite(got)), "not finite"
    off = np.abs(got - want)
    i = np.unravel_index(np.argmax(off - tol), off.shape)
    assert np.all(off <= tol), f"at {i}: {got[i]} for {want[i]}, {off[i]:.3g} off, {tol[i]:.3g} allowed"


HEADS = [(14, 2, 64), (16, 16, 128), (32, 4, 128), (64, 4, 128), (6, 2, 64), (8, 8, 64), (64, 1, 128)]
LENS = {
    "one": [(1, 1)],
    "ends": [(1, 15), (1, 16), (1, 17), (1, 31), (1, 32), (1, 33), (1, 63), (1, 64), (1, 65)],
    "ragged": [(1, 300), (0, 40), (1, 1), (1, 777), (0, 0), (1, 129)],
    "draft": [(5, 5), (3, 260), (8, 515)],
    "prompt": [(33, 33), (130, 130), (1, 90), (65, 301)],
    "chunk": [(20, 2000), (1, 1200), (37, 1500)],
}


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads", HEADS, ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("lens", list(LENS))
def test_attention(ctx, lens, heads, type_):
    H, kv, D = heads
    page = {"one": 16, "ends": 16, "ragged": 64, "draft": 32, "prompt": 128, "chunk": 64}[lens]
    print(f"[case] {lens} {heads} type {type_}", flush=True)
    b = Batch(LENS[lens], page, seed=H + D)
    k, v = values(b, kv, D, type_, 1)
    q = (2 * np.random.default_rng(2).standard_normal((b.T, H, D))).astype(np.float32)
    got = Pool(ctx, H, kv, D, type_, b).run(q, *pack(b, k, v, kv, D, type_))      # NaN in every other slot
    check(got, *attend64(b, q, k, v, D ** -0.5))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("type_", [F16, F32])
def test_every_key_counts_once(ctx, page, type_):
    """Equal scores and whole values: sums are exact, so that one key more or less shows."""
    b = Batch([(1, 1000), (40, 777), (1, 5), (3, 3), (1, 2049), (7, 391)], page, seed=page)
    kv, D, H = 2, 128, 16
    k, v = values(b, kv, D, type_, 3)
    v = [np.round(a * 3).astype(dtype_of(type_)) for a in v]
    q = np.zeros((b.T, H, D), np.float32)
    print(f"[case] equal scores, pages of {page}, type {type_}", flush=True)
    got = Pool(ctx, H, kv, D, type_, b).run(q, *pack(b, k, v, kv, D, type_))
    want = np.stack([np.repeat(v[s][:p + 1].astype(np.float64).mean(0), H // kv, 0) for s, p in zip(b.seq, b.pos)])
    assert np.all(np.abs(got - want) <= 4 * EPS32 * np.abs(want))          # the reciprocal, its product, the output


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("what", ["one", "two_runs", "tokens", "wide", "idle"])
def test_shared_prefix(ctx, what, type_):
    H, kv, D, page = (64, 4, 128, 32) if what == "wide" else (32, 16, 128, 32)     # enough bytes to be worth sharing
    shared, runs, lens = {
        "one": (1024, None, [(1, 1025), (1, 1200), (1, 1400), (1, 1030)]),
        "two_runs": (1056, [3, 1, 2], [(1, 1057), (1, 1180), (1, 1058), (1, 333 + 1056), (1, 1300), (1, 1090)]),
        "tokens": (1024, None, [(3, 1100), (1, 1025), (2, 1026), (6, 1150)]),
        "wide": (1024, None, [(1, 1025 + 37 * i) for i in range(24)]),
        "idle": (1536, None, [(1, 1600), (0, 1600), (1, 1800), (2, 1601)]),
    }[what]
    print(f"[case] shared prefix {what} type {type_}", flush=True)
    b = Batch(lens, page, shared, runs, seed=5)
    k, v = values(b, kv, D, type_, 4, shared, runs)
    q = (2 * np.random.default_rng(6).standard_normal((b.T, H, D))).astype(np.float32)
    ctx.profile(True)
    got = Pool(ctx, H, kv, D, type_, b).run(q, *pack(b, k, v, kv, D, type_))
    joins, _ = ctx.profile_read("join")
    ctx.profile(False)
    assert joins == 1, "the prefix was not shared"             # shared and own keys are two parts at least
    check(got, *attend64(b, q, k, v, D ** -0.5))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("n", [3, 6, 150])
def test_what_a_row_does_not_see(ctx, type_, bad, n):
    """Infinities and NaN in later tokens' keys and values do not reach earlier rows; those that see them get them."""
    H, kv, D = 8, 2, 64
    b = Batch([(n, 200), (1, 77)], 16, seed=8)
    k, v = values(b, kv, D, type_, 9)
    p_v, p_k = 200 - n + n // 3, 200 - n + 2 * n // 3
    v[0][p_v, 1, 5] = bad
    k[0][p_k, 0, 3] = np.nan
    print(f"[case] {bad} from position {p_v}, type {type_}, {n} rows", flush=True)
    q = np.random.default_rng(10).standard_normal((b.T, H, D)).astype(np.float32)
    got = Pool(ctx, H, kv, D, type_, b).run(q, *pack(b, k, v, kv, D, type_))
    want, tol = attend64(b, q, k, v, D ** -0.5)
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine)
    assert not fine[:n, 4:, 5][p_v - 200 + n:].any() and not fine[:n, :4][p_k - 200 + n:].any() and fine[n:].all()
    check(got[fine], want[fine], tol[fine])


@pytest.mark.parametrize("type_", [F16, F32])
def test_score_and_query_ranges(ctx, type_):
    """Scores of thousands, rows of zeros, of tiny and of large queries."""
    H, kv, D = 16, 2, 64
    b = Batch([(1, 700), (20, 333)], 64, seed=11)
    k, v = values(b, kv, D, type_, 12)
    q = np.random.default_rng(13).standard_normal((b.T, H, D)).astype(np.float32)
    q[0, 0] *= 3000
    q[0, 1] = 0
    q[1, 2] *= 1e-30
    q[2, 3] *= 1e-42                       # subnormal
    q[3, 4] *= 500
    q[4] *= np.float32(2.0) ** np.arange(-20, 12, 2)[:, None].astype(np.float32)
    print(f"[case] ranges, type {type_}", flush=True)
    got = Pool(ctx, H, kv, D, type_, b).run(q, *pack(b, k, v, kv, D, type_))
    check(got, *attend64(b, q, k, v, D ** -0.5))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("what", ["long", "long_group", "many", "more_tiles_than_blocks"])
def test_batch_sizes(ctx, what, type_):
    """Parts for the join kernel, more sequences than blocks, more tiles than the card holds blocks."""
    H, kv, D = 8, 1, 64
    lens, shared = {"long": ([(1, 20011)], 0), "long_group": ([(1, 33800), (1, 34100), (1, 33801), (1, 33900)], 33792), "many": ([(1, 1 + 7 * i % 61) for i in range(300)], 0),
                    "more_tiles_than_blocks": ([(150, 150 + i % 5) for i in range(110)], 0)}[what]
    print(f"[case] {what}, type {type_}", flush=True)
    b = Batch(lens, 64, shared, seed=24)
    k, v = values(b, kv, D, type_, 25, shared)
    q = (2 * np.random.default_rng(26).standard_normal((b.T, H, D))).astype(np.float32)
    got = Pool(ctx, H, kv, D, type_, b).run(q, *pack(b, k, v, kv, D, type_))
    check(got, *attend64(b, q, k, v, D ** -0.5))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("group", [1, 16])
def test_every_number_of_row_tiles(ctx, group, type_, D):
    """Tiles of 17 to 128 rows in steps of a row (group 1) or a row tile (group 16), whose waves have none, one or two of
    them, and more blocks than a card's CUs; a value that only a tile's last rows see is infinite."""
    print(f"[case] group {group} type {type_} D {D}", flush=True)
    kv = 8
    rows = range(17, 129, 3) if group == 1 else [2, 3, 4, 5, 6, 7, 8] * 5
    b = Batch([(n, n + 50 + 7 * i) for i, n in enumerate(rows)], 32, seed=group + D)
    k, v = values(b, kv, D, type_, 5)
    v[3][-1, 2, 5] = np.inf
    q = np.random.default_rng(6).standard_normal((b.T, group * kv, D)).astype(np.float32)
    got = Pool(ctx, group * kv, kv, D, type_, b).run(q, *pack(b, k, v, kv, D, type_))
    with np.errstate(invalid="ignore"):
        want, tol = attend64(b, q, k, v, D ** -0.5)
    last = sum(b.q[:4]) - 1                                   # the only token that sees it
    hit = np.zeros(want.shape, bool)
    hit[last, 2 * group:3 * group, 5] = True
    assert np.all(np.isposinf(want[hit])) and not np.any(np.isfinite(got[hit]))
    check(np.where(hit, 0, got), np.where(hit, 0, want), np.where(hit, 0, tol))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads", [(16, 16, 128), (32, 4, 128), (14, 2, 64), (10, 2, 128)], ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("lens", ["ones", "steps", "ragged", "one_long", "odd"])
def test_many_short_sequences(ctx, lens, heads, type_):
    """Batches whose items have a wave or two each: as many as fill the card, an odd one at the end, some
    sequences without new tokens, values that a draft's first token does not see."""
    H, kv, D = heads
    print(f"[case] {lens} {heads} type {type_}", flush=True)
    n = [(1, 1)] * 150 if lens == "ones" else [(1, 1 + i % 70) for i in range(257)] if lens == "steps" else \
        [(1 - (i % 9 == 4), 1 + 37 * i % 230) for i in range(300)] if lens == "ragged" else \
        [(1, 60)] * 200 + [(1, 1500)] if lens == "one_long" else [(1 + (i % 3 == 0), 2 + 11 * i % 95) for i in range(131)]
    b = Batch(n, 16, seed=len(n) + D)
    k, v = values(b, kv, D, type_, 7)
    for i in range(0, len(n), 7):
        if b.q[i] == 2: v[i][-1, 0, 1] = -np.inf                  # its first token does not see this one
    q = np.random.default_rng(8).standard_normal((b.T, H, D)).astype(np.float32)
    got = Pool(ctx, H, kv, D, type_, b).run(q, *pack(b, k, v, kv, D, type_))
    with np.errstate(invalid="ignore"):
        want, tol = attend64(b, q, k, v, D ** -0.5)
    hit = ~np.isfinite(want)
    assert not np.any(np.isfinite(got[hit])) and (lens != "odd" or np.any(hit))
    check(np.where(hit, 0, got), np.where(hit, 0, want), np.where(hit, 0, tol))


@pytest.mark.parametrize("type_", [F16, F32])
def test_many_groups_of_few_rows(ctx, type_):
    """Pairs of sequences on prefixes of their own: shared and own items of few rows, several of them a block."""
    H = kv = 16
    runs = [2] * 60
    b = Batch([(1, 257 + 13 * i % 60) for i in range(120)], 32, shared=256, runs=runs, seed=9)
    k, v = values(b, kv, 128, type_, 10, shared=256, runs=runs)
    q = np.random.default_rng(11).standard_normal((b.T, H, 128)).astype(np.float32)
    print("[case] pairs", flush=True)
    got = Pool(ctx, H, kv, 128, type_, b).run(q, *pack(b, k, v, kv, 128, type_))
    check(got, *attend64(b, q, k, v, 128 ** -0.5))


def test_scale_and_layers(ctx):
    H, kv, D = 8, 2, 128
    b = Batch([(1, 100), (4, 60)], 32, seed=14)
    q = np.random.default_rng(15).standard_normal((b.T, H, D)).astype(np.float32)
    pool = Pool(ctx, H, kv, D, F16, b, n_layer=3, scale=0.25)
    print("[case] scale, layers", flush=True)
    for layer in (2, 0, 1):
        k, v = values(b, kv, D, F16, 20 + layer)
        check(pool.run(q, *pack(b, k, v, kv, D, F16), layer=layer), *attend64(b, q, k, v, 0.25))


def test_offsets_past_32_bits(ctx):
    """Pages that start beyond 2^32 bytes and 2^31 elements of a pool."""
    H, kv, D, page, n_page = 16, 16, 128, 256, 4300
    b = Batch([(1, 700), (3, 515)], page, seed=16)
    b.pages = np.where(b.pages >= 0, b.pages + n_page - b.n_page, b.pages).astype(np.int32)
    k, v = values(b, kv, D, F32, 17)
    q = np.random.default_rng(18).standard_normal((b.T, H, D)).astype(np.float32)
    shift = n_page - b.n_page
    print("[case] far pages", flush=True)
    from large_model_amd import qmsg
    with qmsg.Context(*TINY, n_layer=1, max_tokens=1) as c:      # the pools go with it
        small = b.n_page
        b.n_page = n_page
        pool = Pool(c, H, kv, D, F32, b)
        b.n_page, b.pages = small, b.pages - shift
        kp, vp = pack(b, k, v, kv, D, F32)
        b.pages = b.pages + shift
        off = shift * kv * page * D * 4
        assert off > 2 ** 33
        pool.k, pool.v = pool.k + off, pool.v + off
        check(pool.run(q, kp, vp), *attend64(b, q, k, v, D ** -0.5))


def test_empty_batches(ctx):
    b = Batch([(0, 5), (0, 0)], 16, seed=19)
    pool = Pool(ctx, 8, 2, 64, F16, b)
    d = ctx.device_alloc(4096)
    print("[case] no new tokens", flush=True)
    ctx.h2d(d, np.full(1024, 3.0, np.float32))
    ctx.attn_device(pool.id, 0, d, d + 2048)                     # before any batch
    ctx.attn_batch(pool.id, b.q, b.kv, b.pages)
    ctx.attn_device(pool.id, 0, d, d + 2048)
    ctx.attn_append_device(pool.id, 0, d, d, d + 1024, d + 2048)
    ctx.attn_batch(pool.id, [], [], np.zeros((0, 1), np.int32))
    ctx.attn_device(pool.id, 0, d, d + 2048)
    ctx.sync()
    assert np.all(ctx.d2h(d, 1024) == 3.0)


def test_same_call_same_bits(ctx):
    H, kv, D = 64, 4, 128
    b = Batch([(1, 3000), (5, 900), (100, 100)], 64, seed=21)
    k, v = values(b, kv, D, F16, 22)
    q = np.random.default_rng(23).standard_normal((b.T, H, D)).astype(np.float32)
    kp, vp = pack(b, k, v, kv, D, F16)
    pool = Pool(ctx, H, kv, D, F16, b)
    print("[case] the same call again", flush=True)
    first = pool.run(q, kp, vp)
    for _ in range(3):
        assert np.array_equal(pool.run(q, kp, vp), first)
