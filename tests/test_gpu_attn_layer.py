"""The attention half of the layer loop on the GPU: qmsg_attn_layer against its steps through the public calls, bit for bit;
a model file's layers; decoder steps with the MoE half."""
import ctypes

import numpy as np
import pytest

import gguf_file as gf
import oracle as orc
from attn_cases import F16, F32, Batch
from test_gpu_dense_capture import hip_lib

pytestmark = pytest.mark.gpu
E, X, K, F = 256, 16, 4, 128
EPS = 1e-6


def steps(ctx, attn, layer, mats, norm, h, heads, kv_heads, D):
    """h + output(attention(...)) with a call for each step and the sum on the host."""
    T = h.shape[0]
    d = {n: ctx.device_alloc(T * w * 4) for n, w in (("x", E), ("q", heads * D), ("k", kv_heads * D), ("v", kv_heads * D), ("o", heads * D), ("y", E))}
    d_w = ctx.device_alloc(E * 4)
    ctx.h2d(d_w, norm)
    ctx.h2d(d["x"], h)
    ctx.rmsnorm_device(d["x"], d["x"], d_w, T, E, EPS)
    ctx.matmul_n_device(mats[:3], d["x"], T, [d["q"], d["k"], d["v"]])
    ctx.attn_append_device(attn, layer, d["q"], d["q"], d["k"], d["v"], EPS)
    ctx.attn_device(attn, layer, d["q"], d["o"])
    ctx.matmul_n_device(mats[3:], d["o"], T, [d["y"]])
    ctx.sync()
    return h + ctx.d2h(d["y"], (T, E))


def same(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("heads", [(8, 2, 64), (4, 1, 128)])
def test_layer_equals_its_steps(heads, type_):
    from large_model_amd import qmsg
    H, kv, D = heads
    b = Batch([(1, 70), (9, 9), (0, 4), (2, 33)], 16, seed=1)
    rng = np.random.default_rng(2)
    print(f"[case] layer {heads} type {type_}", flush=True)
    with qmsg.Context(E, X, K, F, n_layer=1, max_tokens=16) as ctx:
        attn = ctx.attn_create(H, kv, D, type_=type_, page=16, n_page=b.n_page, n_layer=2, max_seq=4, max_tokens=16, max_pages=b.max_pages)
        shapes = [(H * D, E), (kv * D, E), (kv * D, E), (E, H * D)]
        types = [orc.T_Q4_0, orc.T_Q4_0, orc.T_Q4_1, orc.T_Q4_0]
        mats = [ctx.mat_upload(t, orc.synth_mat(t, r, c, 30 + i), r, c) for i, (t, (r, c)) in enumerate(zip(types, shapes))]
        norm = (1 + 0.1 * rng.standard_normal(E)).astype(np.float32)
        for layer in range(2):
            ctx.attn_mats(attn, layer, mats, norm)
            ctx.attn_norms(attn, layer, *(1 + 0.2 * rng.standard_normal((2, D))).astype(np.float32))
        k, v = ctx.attn_cache(attn)
        n = 2 * b.n_page * kv * 16 * D
        cache = rng.standard_normal((2, n)).astype(np.float16 if type_ == F16 else np.float32)
        ctx.attn_batch(attn, b.q, b.kv, b.pages)
        h = rng.standard_normal((b.T, E)).astype(np.float32)
        d_h = ctx.device_alloc(h.nbytes)
        for layer in range(2):
            got = []
            for run in range(2):
                ctx.h2d(k, cache[0])
                ctx.h2d(v, cache[1])
                if run:
                    ctx.h2d(d_h, h)
                    ctx.attn_layer(attn, layer, d_h, EPS)
                    ctx.sync()
                    got.append(ctx.d2h(d_h, h.shape))
                else:
                    got.append(steps(ctx, attn, layer, mats, norm, h, H, kv, D))
                got += [ctx.d2h(k, n, cache.dtype), ctx.d2h(v, n, cache.dtype)]
            assert same(got[0], got[3]) and np.array_equal(got[1], got[4]) and np.array_equal(got[2], got[5])
            assert not np.array_equal(got[1], cache[0]) and not same(got[0], h)


def test_model_file_and_decoder_steps(tmp_path):
    """Two layers of a file, attention half and MoE half in turn: a prompt, then a token at a time, eager and from a captured
    graph, against the steps through the public calls."""
    from large_model_amd import qmsg
    hip, vp = hip_lib(), ctypes.c_void_p
    H, kv, D = 4, 2, 64
    lays = [orc.Layer(E, X, K, F, 60 + l, layer=l) for l in range(2)]
    path, norms = gf.moe_model(str(tmp_path / "m.gguf"), lays, n_head=H, n_head_kv=kv, head_dim=D)
    rng = np.random.default_rng(3)
    prompt = rng.standard_normal((21, E)).astype(np.float32)
    print("[case] model file", flush=True)
    with qmsg.Gguf(path) as g, qmsg.Context.from_gguf(g, max_tokens=32) as ctx:
        attn = ctx.attn_from_gguf(g, page=16, n_page=8, max_seq=2, max_tokens=32, max_pages=4)
        other = ctx.attn_create(H, kv, D, page=16, n_page=8, n_layer=2, rope_base=5000000.0, max_seq=2, max_tokens=32, max_pages=4)
        mats = [[ctx.gguf_upload_mat(g, f"blk.{l}.attn_{n}.weight") for n in ("q", "k", "v", "output")] for l in range(2)]
        pages = np.array([[5, 2, 7, 0], [1, 3, 4, 6]], np.int32)
        d_h = ctx.device_alloc(32 * E * 4)

        def batch(q, n):
            for a in (attn, other):
                ctx.attn_batch(a, q, n, pages)

        def device():
            for l in range(2):
                ctx.attn_layer(attn, l, d_h, EPS)
                ctx.moe_chain(l, 1, d_h, T, EPS)

        def by_steps(h):
            for l in range(2):
                h = steps(ctx, other, l, mats[l], np.ones(E, np.float32), h, H, kv, D)
                h = h + lays[l].moe(orc.rmsnorm(h, norms[l], eps=EPS))
            return h

        T = 21
        batch([13, 8], [13, 8])
        ctx.h2d(d_h, prompt)
        device()
        ctx.sync()
        assert same(ctx.d2h(d_h, (T, E)), by_steps(prompt))
        T, graph, exe = 2, vp(), vp()
        st = vp(qmsg.lib.qmsg_stream(ctx._h))
        try:
            for n in range(6):
                print(f"[case] token {n}", flush=True)
                batch([1, 1], [14 + n, 9 + n])
                h = rng.standard_normal((2, E)).astype(np.float32)
                want = by_steps(h)
                for replay in range(2 if n > 2 else 1):
                    ctx.h2d(d_h, h)
                    if replay:
                        assert hip.hipGraphLaunch(exe, st) == 0
                    else:
                        device()
                    ctx.sync()
                    assert same(ctx.d2h(d_h, (2, E)), want), (n, replay)
                if n == 2:                                 # later steps run from a graph too
                    assert hip.hipStreamBeginCapture(st, 2) == 0
                    device()
                    assert hip.hipStreamEndCapture(st, ctypes.byref(graph)) == 0
                    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        finally:
            if exe:
                hip.hipGraphExecDestroy(exe)
                hip.hipGraphDestroy(graph)


def test_upload_checks_the_file(tmp_path):
    from large_model_amd import qmsg
    lays = [orc.Layer(E, X, K, F, 1)]
    path, _ = gf.moe_model(str(tmp_path / "m.gguf"), lays, n_head=4, n_head_kv=2, head_dim=64)
    print("[case] refused uploads", flush=True)
    with qmsg.Gguf(path) as g, qmsg.Context.from_gguf(g, max_tokens=4) as ctx:
        sizes = dict(page=16, n_page=4, max_seq=1, max_tokens=4, max_pages=4)
        for args, n_layer, status in (((8, 2, 64), 1, -1), ((4, 1, 64), 1, -1), ((4, 2, 128), 1, -1), ((4, 2, 64), 2, -1)):
            i = ctx.attn_create(*args, n_layer=n_layer, **sizes)
            st = qmsg.lib.qmsg_gguf_attn_upload(ctx._h, g._h, i, 0, n_layer)
            assert st == status, args
        assert qmsg.lib.qmsg_gguf_attn_upload(ctx._h, g._h, i, 1, 2) == -5 and qmsg.lib.qmsg_gguf_attn_upload(ctx._h, g._h, 99, 0, 1) == -1
        assert ctx.attn_from_gguf(g, **sizes) == i + 1
