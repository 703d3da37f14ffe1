"""The kernels of the packed key / value cache executed on the CPU: their HIP sources compiled for the host behind
tests/cpp/emu/hip/hip_runtime.h (see test_kernels_on_host.py, whose source rewriting is used here), and the GPU-marked
tests run against that library.  Bad slots, pages and lengths meet the kernels here first."""
import os
import re
import shutil
import subprocess
import sys

import pytest

from helpers import ROOT_DIR
from test_kernels_on_host import rewrite_launches

UNITS = ("mxq_capi_kv.hip", "mxq_capi_kv_decode.hip", "mxq_capi_kv_prompt.hip")
# what fits: streams, graphs and large caches are the GPU's; the larger shapes take minutes here
SKIP = "not stream and not captured and not 32_bits and not 290 and not workgroup_scans and not 600 and not fp16_rows"
FEW = ("(append_then_read and (96 or 31)) or consecutive or layout or block_tables_of or (block_tables and (300 or 40)) or "
       "(single_tokens and (lens1 or lens7) and dtype0) or (single_tokens and lens5 and dtype1) or "
       "(some_tokens and lens3) or (prompt_chunks and lens5) or missing_pages or (shared_by and lens0) or refusals or in_an_array or no_request or (not_in_order and starts0 and 60000) or "
       "(wide_tables and lens3 and dtype0) or (wide_tables and lens6 and dtype1)")


@pytest.fixture(scope="module")
def host_build(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("kv_on_host")
    csrc, emu = os.path.join(ROOT_DIR, "microxcaling_amd", "csrc"), os.path.join(ROOT_DIR, "tests", "cpp", "emu")
    clang = ["/opt/rocm/lib/llvm/bin/clang++", "-std=c++20", "-fPIC", "-ffp-contract=off", "-pthread", "-msse4.1", "-O1"]
    jobs, objects = [], [str(tmp / "emu_math.o")]
    jobs.append(subprocess.Popen([*clang, "-c", os.path.join(emu, "emu_math.cpp"), "-o", objects[0]]))
    with open(os.path.join(csrc, "mxq_kv_attention.h")) as f:
        text, pins = re.subn(r'asm volatile\(""\s*:[^;]*\);', ";", f.read())       # a register pin
    assert pins == 1 and "asm volatile" not in text
    with open(str(tmp / "mxq_kv_attention.h"), "w") as f:                            # found before the original
        f.write(text)
    shutil.copy(os.path.join(csrc, "mxq_capi_kv.h"), str(tmp))                        # (includes it from beside itself)
    for unit in UNITS:
        with open(os.path.join(csrc, unit)) as f:
            text = rewrite_launches(f.read())
        assert "<<<" not in text
        source = str(tmp / (unit[:-4] + "_on_host.cpp"))
        with open(source, "w") as f:
            f.write(text)
        objects.append(source[:-4] + ".o")
        jobs.append(subprocess.Popen([*clang, "-I" + str(tmp), "-I" + emu, "-I" + os.path.join(ROOT_DIR, "include"), "-I" + csrc, "-c", source,
                                      "-o", objects[-1]], stderr=subprocess.PIPE))
    with open(str(tmp / "last_error.cpp"), "w") as f:              # exported by another unit of the library
        f.write('#include "mxq_params.h"\nextern "C" const char* mxq_last_error(void) { return mxq_detail::last_error().c_str(); }\n')
    objects.append(str(tmp / "last_error.cpp"))
    for job in jobs:
        err = job.communicate(timeout=1800)[1]
        assert job.returncode == 0, err
    lib = str(tmp / "libmxq_kv_on_host.so")
    subprocess.run([*clang, "-I" + os.path.join(ROOT_DIR, "include"), "-I" + csrc, "-shared", "-o", lib, *objects], check=True, capture_output=True, timeout=600)
    return lib


def test_gpu_tests_pass_on_the_kernels_compiled_for_the_host(host_build):
    if os.environ.get("MXQ_KERNELS_ON_HOST") == "none":
        pytest.skip("MXQ_KERNELS_ON_HOST=none")
    everything = os.environ.get("MXQ_KERNELS_ON_HOST") == "all"
    select = SKIP if everything else "(%s) and %s" % (FEW, SKIP)
    env = dict(os.environ, MXQ_HIP_ON_HOST_LIB=host_build,
               PYTHONPATH=os.path.join(ROOT_DIR, "tests") + os.pathsep + os.environ.get("PYTHONPATH", ""))
    res = subprocess.run([sys.executable, "-m", "pytest", "-p", "hip_on_host_plugin", "-p", "no:cacheprovider", "-q", "-x",
                          "-m", "gpu", "-k", select, "--durations=8", "tests/test_zy_kv_cache.py"],
                         cwd=ROOT_DIR, env=env, capture_output=True, text=True, timeout=2 * 3600)
    tail = res.stdout[-6000:] + res.stderr[-2000:]
    assert res.returncode == 0, tail
    assert " passed" in res.stdout and "failed" not in res.stdout, tail
    print(tail)


# of the edges, what takes a minute or two; behind the skipped ones are prompts of thousands of rows
EDGES = ("(several_items_in_a_stretch and lens0 and dtype0) or (many_rows_of_no_request and 400) or (overflows and 64 and dtype0) or "
         "rows_overlap or too_large")
EDGES_SKIP = "not long_prompts and not more_rows_than and not captured and not streams"


def test_edges_pass_on_the_kernels_compiled_for_the_host(host_build):
    if os.environ.get("MXQ_KERNELS_ON_HOST") == "none":
        pytest.skip("MXQ_KERNELS_ON_HOST=none")
    select = EDGES_SKIP if os.environ.get("MXQ_KERNELS_ON_HOST") == "all" else "(%s) and %s" % (EDGES, EDGES_SKIP)
    env = dict(os.environ, MXQ_HIP_ON_HOST_LIB=host_build,
               PYTHONPATH=os.path.join(ROOT_DIR, "tests") + os.pathsep + os.environ.get("PYTHONPATH", ""))
    res = subprocess.run([sys.executable, "-m", "pytest", "-p", "hip_on_host_plugin", "-p", "no:cacheprovider", "-q", "-x",
                          "-m", "gpu", "-k", select, "--durations=8", "tests/test_zy_kv_cache_edges.py"],
                         cwd=ROOT_DIR, env=env, capture_output=True, text=True, timeout=2 * 3600)
    tail = res.stdout[-6000:] + res.stderr[-2000:]
    assert res.returncode == 0, tail
    assert " passed" in res.stdout and "failed" not in res.stdout, tail
    print(tail)
