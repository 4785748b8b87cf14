"""The norm and block-FP8 functions run the library that _lib.lib() loaded, also
where NFLOW_QUANT_LIB names another build, and there is one in the process."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from neuroflow_amd import _lib

ROOT = Path(__file__).resolve().parents[1]

CODE = """
from neuroflow_amd import _lib, block_fp8
ops = block_fp8._ops()
print(_lib.lib()._name)
print(ops.library())
for path in sorted({line.split()[-1] for line in open("/proc/self/maps") if "libnflow_quant" in line}):
    print("mapped", path)
"""


def run(**env):
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env={**os.environ, **env}, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr
    return r.stdout.splitlines()


@pytest.mark.parametrize("name", ["libnflow_quant.so", "other_build_libnflow_quant.so"])
def test_another_build(tmp_path, name):
    """In a folder of its own, under the same name or another."""
    other = tmp_path / name
    shutil.copy(ROOT / "neuroflow_amd" / "lib" / "libnflow_quant.so", other)
    assert run(NFLOW_QUANT_LIB=str(other)) == [str(other), str(other), f"mapped {other}"]


def test_the_build_in_the_tree():
    lib = str(ROOT / "neuroflow_amd" / "lib" / "libnflow_quant.so")
    env = {k: v for k, v in os.environ.items() if k != "NFLOW_QUANT_LIB"}
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.splitlines() == [lib, lib, f"mapped {lib}"], r.stdout + r.stderr


def test_every_entry_point_is_bound():
    """The module's own list holds every function of nflow_block.h that is no query for tests."""
    from neuroflow_amd import block_fp8
    names = set(block_fp8._ops().entry_points())
    assert names - {"nflow_last_error"} == {n for n in _lib.SIGNATURES if "layer_norm" in n or "fp8_block" in n} - {
        n for n in _lib.SIGNATURES if "debug" in n}
