"""Host code of the attention backward and of the rotary positions under AddressSanitizer + UndefinedBehaviorSanitizer (no GPU needed), as
``test_host_sanitizers.py`` has it for the other entries."""
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from alto_amd import build as B
from tests.test_host_sanitizers import HERE, OUT, SAN, _rocm_llvm_clang

SOURCES = ["capi.hip", "rotary.hip"] + [f for f in B.SOURCES if f.startswith("attention_backward")]


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_entries_with_argument_structs_under_asan_and_ubsan():
    clang = _rocm_llvm_clang()
    if clang is None:
        pytest.skip("ROCm's clang++ not found next to hipcc")
    out = os.path.join(OUT, "training")
    os.makedirs(out, exist_ok=True)
    host = [f for s in SAN for f in ("-Xarch_host", s)]
    flags = [f for f in B.HIPCC_FLAGS if f != "-O3"] + ["-O1", "-g"] + host

    def comp(src):
        obj = os.path.join(out, os.path.splitext(src)[0] + ".o")
        r = subprocess.run([B._hipcc(), *flags, "-c", os.path.join(B.CSRC, src), "-o", obj], capture_output=True, text=True)
        assert r.returncode == 0, f"{src}:\n{r.stderr[-3000:]}"
        return obj

    with ThreadPoolExecutor(max_workers=4) as pool:
        objs = list(pool.map(comp, SOURCES))
    exe = os.path.join(out, "driver")
    rocm_lib = os.path.join(os.path.dirname(os.path.realpath(B._hipcc())), "..", "lib")
    r = subprocess.run([clang, "-std=c++17", "-O1", "-g", *SAN, "-I", os.path.join(HERE, "..", "include"), os.path.join(HERE, "host_sanitizers", "driver_training.cpp"), *objs, "-o", exe,
                        "-L", rocm_lib, "-lamdhip64", f"-Wl,-rpath,{rocm_lib}"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=0", UBSAN_OPTIONS="print_stacktrace=1", HIP_VISIBLE_DEVICES="", ROCR_VISIBLE_DEVICES="")
    r = subprocess.run([exe, "4000"], capture_output=True, text=True, env=env, timeout=600)
    tail = r.stdout[-2500:] + "\n" + r.stderr[-4000:]
    assert r.returncode == 0, tail
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr, tail
    assert "attention_bwd calls 4000" in r.stdout, tail
