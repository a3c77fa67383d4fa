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


@pytest.mark.parametrize("scenario", ["configs", "memory", "batches", "calls"])
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
