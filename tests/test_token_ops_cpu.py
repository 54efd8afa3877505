"""The token operators' kernels compiled for the CPU (tests/cpu_kernels: a block's threads as
fibers, waves and barriers between them) with address checks on every buffer and on
static shared memory, memory filled with junk, and the GPU tests run on them: what they
read and write lies within their operands, nothing they use is left uninitialised, and
the results hold whatever order the threads run in.  What a CPU cannot show stays with
the GPU: streams, graphs, rounding of the device's own exponential."""
import glob
import os
import re
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pytest

from conftest import ROOT

HERE = os.path.join(ROOT, "tests", "cpu_kernels")
OUT = os.path.join(ROOT, "build", "cpu_kernels" + os.environ.get("PYTEST_XDIST_WORKER", ""))
CLANG = "/opt/rocm/llvm/bin/clang++"
ASAN = sorted(glob.glob("/opt/rocm/llvm/lib/clang/*/lib/*/libclang_rt.asan-x86_64.so"))
FLAGS = ["-std=c++17", "-O1", "-gline-tables-only", "-fPIC", "-Wno-everything", "-Xarch_host", "-fsanitize=address", "-shared-libasan"]
SOURCES = ("ghm_score", "ghm_distill", "ghm_embed")

pytestmark = pytest.mark.skipif(not (os.path.exists(CLANG) and ASAN), reason="no clang++ with its address sanitizer")


def _build():
    """The three sources; shared memory of a launch's size taken from the fibers' buffer, and the threads
    that a grid's x holds from the environment ($GRID_THREADS), so that small launches can be made to go
    over both dimensions."""
    work = OUT
    shutil.rmtree(work, ignore_errors=True)
    for d in ("a/csrc", "include", "a/csrc/hip"):
        os.makedirs(os.path.join(work, d))
    csrc = os.path.join(ROOT, "multimodal-ghm_amd", "csrc")
    shutil.copy(os.path.join(ROOT, "include", "ghm_hip.h"), os.path.join(work, "include"))
    shutil.copy(os.path.join(HERE, "hip", "hip_runtime.h"), os.path.join(work, "a", "csrc", "hip"))
    shutil.copy(os.path.join(HERE, "block.cpp"), os.path.join(work, "a", "csrc"))
    shutil.copy(os.path.join(csrc, "ghm_launch.h"), os.path.join(work, "a", "csrc"))

    def put(name, text):
        with open(os.path.join(work, "a", "csrc", name), "w") as f:
            f.write(text)
    put("ghm_common.h", "#pragma once\n#include <hip/hip_runtime.h>\n")
    token = open(os.path.join(csrc, "ghm_token.h")).read()
    token, n = re.subn(r"\(int64_t\(1\) << 32\) - 1\)", "grid_threads())", token)
    assert n == 1
    put("ghm_token.h", token)
    for s in SOURCES:
        text = open(os.path.join(csrc, s + ".hip")).read()
        text = re.sub(r"^( +)extern __shared__ float (\w+)\[\];", r"\1float* \2 = reinterpret_cast<float*>(dynamic_lds);",
                      text, flags=re.M)
        text = re.sub(r"^extern __shared__ float (\w+)\[\];", r"#define \1 reinterpret_cast<float*>(dynamic_lds)", text,
                      flags=re.M)
        assert "extern __shared__" not in text
        put(s + ".cpp", text)
    src = os.path.join(work, "a", "csrc")

    def one(name):
        subprocess.run([CLANG, *FLAGS, f"-I{src}", "-c", os.path.join(src, name + ".cpp"), "-o",
                        os.path.join(work, name + ".o")], check=True)
    with ThreadPoolExecutor(4) as pool:
        list(pool.map(one, (*SOURCES, "block")))
    lib = os.path.join(work, "libtoken_cpu.so")
    subprocess.run([CLANG, *FLAGS, "-shared", "-fuse-ld=lld", *[os.path.join(work, n + ".o") for n in (*SOURCES, "block")],
                    "-o", lib], check=True)
    return lib


def _run(lib, select, order, fill, **more):
    env = {k: v for k, v in os.environ.items() if not k.startswith("PYTEST_")}
    env = dict(env, **more, CPU_KERNELS=lib, PYTHONPATH=HERE, LANE_ORDER=str(order), LD_PRELOAD=ASAN[-1],
               ASAN_OPTIONS="detect_leaks=0:detect_stack_use_after_return=0:allocator_may_return_null=1:"
                            f"max_malloc_fill_size=2147483647:malloc_fill_byte={fill}")
    r = subprocess.run([sys.executable, "-m", "pytest", "-p", "cpu_device", "-p", "no:cacheprovider", "-q", "-x", "-n", "4",
                        os.path.join(ROOT, "tests", "test_token_ops_gpu.py"), "-k", select], env=env, cwd=ROOT,
                       capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-6000:] + r.stderr[-3000:]
    passed = int(re.search(r"(\d+) passed", r.stdout).group(1))
    assert "skipped" not in r.stdout
    return passed


@pytest.fixture(scope="module")
def lib():
    return _build()


# not on the CPU: graphs, streams, the model's own kernels, the wrappers' device checks; sizes of minutes
ELSEWHERE = "not captured and not streams and not vlm and not refusals and not large_outputs and not 2_31 and not 32_bits"
LONG = "not 140001 and not 300001 and not 200003 and not 600000 and not 270001 and not 262144 and not 262145"


@pytest.mark.parametrize("order,fill,select,least", [
    (0, 255, f"(test_score or test_distill) and dtype1 and {ELSEWHERE} and {LONG} and not far_apart", 80),
    (1, 90, f"test_embedding and (dtype0 or every_row) and {ELSEWHERE} and {LONG}", 60),
    (2, 255, f"(masks_and_special or special_values or without) and dtype0 and {ELSEWHERE} and {LONG} and not 70001", 15),
], ids=["rows", "tables", "any order"])
def test_on_the_cpu(lib, order, fill, select, least):
    assert _run(lib, select, order, fill) >= least


def test_grids_of_two_dimensions_on_the_cpu(lib):
    few = {"GRID_THREADS": "2047"}
    assert _run(lib, f"(test_score_gradient or test_distill) and dtype2 and {ELSEWHERE} and {LONG} and not far_apart and "
                     "not 70001 and not 40000 and not 32771 and not 9000 and not 8193 and not 20000", 0, 255, **few) >= 40
    assert _run(lib, f"test_embedding and dtype1 and not every_row and {ELSEWHERE} and {LONG} and not 70000 and not 20000", 0,
                255, **few) >= 20
