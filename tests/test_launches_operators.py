"""What the device operators and the models' 8-bit cache launch, without a GPU.

tests/launch/operator_checks.cpp, as tests/test_launches.py runs its program:
refused launches and allocations, the arguments of launches.
"""
import os
import shutil
import subprocess

import pytest

from test_launches import CSRC, HERE, OBJECTS, ROCM

pytestmark = pytest.mark.skipif(shutil.which("g++") is None or not os.path.isdir(os.path.join(ROCM, "include", "hip")),
                                reason="no host compiler or no HIP headers")


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    subprocess.run(["make", "-s", "-j", "8", "-C", CSRC], check=True)
    objects = [os.path.join(OBJECTS, f) for f in sorted(os.listdir(OBJECTS))
               if f.endswith(".o") and f not in ("capi.o", "mesh_gpt_cli.o", "mesh_gpt_bench.o")]
    exe = str(tmp_path_factory.mktemp("launch") / "operator_checks")
    built = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-pthread", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROCM, "include"),
                            "-I", CSRC, os.path.join(HERE, "operator_checks.cpp"), os.path.join(HERE, "fake_hip.cpp"),
                            *objects, "-o", exe], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    return exe


@pytest.mark.parametrize("name", ["refused_launches", "foreign_errors", "scores_without_memory", "cache_without_memory",
                                  "many_sequences"])
def test_launches(checks, name):
    run = subprocess.run([checks, name], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout == "ok\n", run.stdout + run.stderr
