"""The decode-step operators through include/vortx_b200.hpp: compiled with g++ against the shared library."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def binary(tmp_path_factory):
    import vortx_b200
    vortx_b200.load()                                   # fails loudly if the library has not been built
    lib_dir = ROOT / "vortx_b200"
    out = tmp_path_factory.mktemp("cpp") / "decode_test"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(ROOT / "tests" / "cpp" / "decode_test.cpp"),
           "-o", str(out), f"-L{lib_dir}", "-lvortx_b200", f"-Wl,-rpath,{lib_dir}"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    return out


def test_tree_mask_on_cpu(binary):
    res = subprocess.run([str(binary), "host"], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and res.stdout.strip().endswith("ok"), res.stdout + res.stderr


@pytest.mark.gpu
def test_operators_on_gpu(binary):
    res = subprocess.run([str(binary), "gpu"], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip().endswith("ok"), res.stdout + res.stderr
