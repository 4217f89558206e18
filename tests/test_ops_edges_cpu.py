"""How an attention is shared out, against what the compiled kernels let a CU hold; which tensors are no cache."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "qwen3-tts_amd", "csrc")


def waves_per_simd(tmp_path):
    """{(kernel, template arguments): waves of it that a SIMD holds}, as the compiler reports them for the flags of the build."""
    flags = re.search(r"^HIPFLAGS = (.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1).split()
    r = subprocess.run([HIPCC, "--offload-arch=gfx950", "--offload-device-only", "-O3", "-std=c++17", "-fPIC", *flags, "-Rpass-analysis=kernel-resource-usage",
                        "-c", os.path.join(CSRC, "kernels_attn.hip"), "-o", str(tmp_path / "a.o")], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    found, name = {}, None
    for line in r.stderr.splitlines():
        m = re.search(r"Function Name: _ZN6hipvoc\d+(\w+?_kernel)I((?:Li\d+E)+)E", line)
        if m:
            name = (m.group(1), tuple(int(v) for v in re.findall(r"Li(\d+)E", m.group(2))))
        m = re.search(r"Occupancy \[waves/SIMD\]: (\d+)", line)
        if m and name:
            found[name], name = int(m.group(1)), None
        m = re.search(r"ScratchSize \[bytes/lane\]: (\d+)", line)
        if m and name:
            assert m.group(1) == "0", (name, line)
    return found


HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def test_the_card_holds_the_workers_of_a_call_at_a_time(tmp_path):
    """More workers than that are two rounds of equal shares: twice the time of the last one."""
    if not os.path.exists(HIPCC) or not shutil.which("g++"):
        pytest.skip("no compiler")
    held = waves_per_simd(tmp_path)
    src = tmp_path / "plan.cpp"
    src.write_text('#include <stdio.h>\n#include "ops_index.hpp"\nint main() { for (int dtype = 0; dtype < 3; dtype++) for (int coded = 0; coded < 2; coded++)\n'
                   'for (int hd = 64; hd <= 128; hd += 64) for (int group = 1; group <= 20; group++)\n'
                   'printf("%d %d %d %d %d\\n", dtype, coded, hd, group, hipvoc::attention_plan(dtype, coded, hd, 8, 8 * group, 64, 100000, 0).workers); }\n')
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, "-o", exe, str(src)], check=True)
    seen = 0
    for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines():
        dtype, coded, hd, group, workers = (int(v) for v in line.split())
        if dtype == 0 and not coded:                                    # a worker is a workgroup of four waves, one on each SIMD
            assert workers <= 256 * held["attn_rows_kernel", (hd, group if group < 3 else 4)], line
            seen += 1
        else:                                                           # a worker is a wave
            for store in ((3, 4) if coded else (dtype,)):
                assert workers <= 256 * 4 * held["attn_stream_kernel", (dtype, store, hd)], line
                seen += 1
    assert seen == 2 * 20 * (1 + 2 + 2 * 3)


def test_a_cache_is_memory_alone(pkg):
    """A cache's tensors carry no gradient and are no views of a negative."""
    import torch
    ok, s = torch.zeros((3, 2, 16, 64)), torch.zeros((3, 2, 16))
    q = torch.zeros((3, 2, 16, 64), dtype=torch.int8)
    pkg.KvCache(ok, ok.clone())
    for bad in [lambda: pkg.KvCache(ok.clone().requires_grad_(), ok), lambda: pkg.KvCache(ok, ok.clone().requires_grad_() * 2), lambda: pkg.KvCache(torch._neg_view(ok), ok),
                lambda: pkg.KvCache(q, q, s.clone().requires_grad_(), s), lambda: pkg.KvCache(q, q, s, torch._neg_view(s))]:
        with pytest.raises(pkg.HipVocError):
            bad()
