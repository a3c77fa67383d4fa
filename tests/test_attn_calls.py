"""The attention's entry points on a stand-in for the HIP runtime (tests/attn_call_host.cpp, CPU): refusals and their
status, memory that runs out, what a captured call is given."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIP_INC = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "include")
CSRC = os.path.join(ROOT, "large_model_amd", "csrc")


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    if shutil.which("g++") is None or not os.path.exists(os.path.join(HIP_INC, "hip", "hip_runtime_api.h")):
        pytest.skip("no g++ or HIP headers")
    out = str(tmp_path_factory.mktemp("attn_call") / "attn_call_host")
    cmd = ["g++", "-std=c++17", "-O1", "-w", "-D__HIP_PLATFORM_AMD__", "-D__align__(n)=__attribute__((aligned(n)))",
           "-DHIP_SYMBOL(s)=&s", "-I", HIP_INC] + [os.path.join(CSRC, f) for f in ("qmsg_api.cpp", "qmsg_attn_api.cpp", "qmsg_plan.cpp")] + \
          [os.path.join(ROOT, "tests", "attn_call_host.cpp"), "-no-pie", "-pthread", "-Wl,--unresolved-symbols=ignore-all", "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return out


@pytest.mark.parametrize("scenario", ["configs", "memory", "batches", "calls", "layers"])
def test_calls(exe, scenario):
    r = subprocess.run([exe, scenario], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr[-2000:]


def test_binding_checks_shapes():
    import numpy as np
    from large_model_amd import qmsg
    c = qmsg.Context.__new__(qmsg.Context)
    c._h = None
    for q, kv, pages in (([1], [1], np.zeros(1, np.int32)), ([1, 1], [1], np.zeros((1, 1), np.int32)), ([1], [1, 2], np.zeros((1, 1), np.int32))):
        with pytest.raises(ValueError):
            c.attn_batch(0, q, kv, pages)
    assert qmsg.lib.qmsg_attn_create(None, None, None, None, None) == -1
    assert qmsg.lib.qmsg_attn_device(None, 0, 0, None, None) == -1


def test_gguf_attention_keys(tmp_path):
    """The attention keys of a qwen3moe file, and what is refused."""
    import gguf_file as gf
    import oracle as orc
    from large_model_amd import qmsg
    from large_model_amd.gguf_writer import F32, STR, U32, write_gguf
    path, _ = gf.moe_model(str(tmp_path / "m.gguf"), [orc.Layer(256, 16, 4, 128, 1), orc.Layer(256, 16, 4, 128, 2, layer=1)],
                           n_head=8, n_head_kv=2, head_dim=128)
    with qmsg.Gguf(path) as g:
        assert g.attn_cfg() == {"n_head": 8, "n_head_kv": 2, "head_dim": 128, "n_layer": 2, "rope_base": 5000000.0}
    keys = {"general.architecture": (STR, "qwen3moe"), "qwen3moe.block_count": (U32, 3), "qwen3moe.embedding_length": (U32, 512),
            "qwen3moe.expert_count": (U32, 16), "qwen3moe.expert_used_count": (U32, 4), "qwen3moe.expert_feed_forward_length": (U32, 128),
            "qwen3moe.attention.layer_norm_rms_epsilon": (F32, 1e-6), "qwen3moe.attention.head_count": (U32, 8),
            "qwen3moe.attention.head_count_kv": (U32, 4)}

    def cfg(**change):
        k = {**keys, **{f"qwen3moe.{n.replace('__', '.')}": v for n, v in change.items()}}
        write_gguf(str(tmp_path / "k.gguf"), [(n, *v) for n, v in k.items() if v is not None], [])
        with qmsg.Gguf(str(tmp_path / "k.gguf")) as g:
            return g.attn_cfg()

    assert cfg() == {"n_head": 8, "n_head_kv": 4, "head_dim": 64, "n_layer": 3, "rope_base": 10000.0}
    same = {"rope__dimension_count": (U32, 64), "rope__scaling__type": (STR, "none")}
    assert cfg(**same) == cfg()
    for change, status in (({"attention__head_count": None}, -1), ({"attention__head_count_kv": None}, -1), ({"attention__head_count": (U32, 0)}, -1),
                           ({"attention__key_length": (U32, 64), "attention__value_length": (U32, 128)}, -2), ({"attention__key_length": (STR, "x")}, -1),
                           ({"rope__dimension_count": (U32, 32)}, -2), ({"rope__scaling__type": (STR, "yarn")}, -2)):
        with pytest.raises(qmsg.QmsgError) as e:
            cfg(**change)
        assert e.value.status == status, change
