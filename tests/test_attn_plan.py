"""Plans of attention batches (csrc/qmsg_plan.cpp) on the CPU: coverage of every row's keys, bounds, refusals."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    out = str(tmp_path_factory.mktemp("attn_plan") / "attn_plan_host")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-fsanitize=address,undefined", os.path.join(ROOT, "tests", "attn_plan_host.cpp"),
                        os.path.join(ROOT, "large_model_amd", "csrc", "qmsg_plan.cpp"), "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return out


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_random_batches(exe, seed):
    r = subprocess.run([exe, str(seed), "300"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    n = [int(x) for x in r.stdout.replace(",", "").split() if x.isdigit()]
    assert n[1] > 0, "no batch shared a prefix"
    assert all(n[2:6]), "no batch with items of some number of waves"
