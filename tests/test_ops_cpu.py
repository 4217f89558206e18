"""CPU-side tests of the token-step operators: exports, what is refused before a launch, index arithmetic of the kernels."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_the_operators(pkg):
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "hipvoc_ops.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(hipvoc_[a-z0-9_]+)\s*\(", hdr))
    lib = pkg.load_library()
    for sym in sorted(declared):
        assert hasattr(lib, sym), f"{sym} declared in include/hipvoc_ops.h but not exported"
    assert declared == set(pkg.ops.OPS_EXPORTS)


def test_header_is_plain_c(tmp_path):
    src = tmp_path / "t.c"
    src.write_text('#include "hipvoc_ops.h"\nint main(void) { hipvoc_kv_cache c; hipvoc_kv_rows r; (void)c; (void)r; return sizeof(c) == 60 || sizeof(c) == 64 ? 0 : 1; }\n')
    exe = str(tmp_path / "t")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), "-o", exe, str(src)], check=True)
    assert subprocess.run([exe]).returncode == 0


def test_python_mirror_has_the_header_layout(pkg, tmp_path):
    """sizeof and offsets of the two structs as C sees them, against the ctypes mirror."""
    fields = {"hipvoc_kv_cache": (pkg.ops._Cache, [f[0] for f in pkg.ops._Cache._fields_]), "hipvoc_kv_rows": (pkg.ops._Rows, [f[0] for f in pkg.ops._Rows._fields_])}
    lines = ['#include <stdio.h>\n#include "hipvoc_ops.h"\nint main(void) {']
    for name, (_, fs) in fields.items():
        lines.append(f'printf("%zu", sizeof({name}));')
        lines += [f'printf(" %zu", offsetof({name}, {f}));' for f in fs]
        lines.append('printf("\\n");')
    src = tmp_path / "o.c"
    src.write_text("\n".join(lines) + "return 0; }\n")
    exe = str(tmp_path / "o")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", exe, str(src)], check=True)
    got = subprocess.run([exe], capture_output=True, text=True, check=True).stdout.strip().split("\n")
    import ctypes
    for line, (_, (cls, fs)) in zip(got, fields.items()):
        assert [int(v) for v in line.split()] == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fs]


def test_no_cpu_fallback_for_the_operators(pkg):
    if pkg.load_library().hipvoc_device_count() > 0:
        pytest.skip("a GPU is present")
    with pytest.raises(pkg.HipVocError):
        pkg.HipOps.open(0)
    lib = pkg.ops._lib()
    assert lib.hipvoc_ops_sync(None, None) == -1                       # no handle: an error code, not a crash
    assert lib.hipvoc_attention_workspace(None, 4, 4, 100, 0) == 0


def test_workspace_of_any_sizes(pkg):
    """A size function answers whatever it is asked: heads that do not divide, nothing to do, extreme lengths."""
    import torch
    lib = pkg.ops._lib()
    k = torch.zeros((2, 8, 16, 64), dtype=torch.bfloat16)
    c = pkg.KvCache(k, k.clone())
    for heads in (0, -8, 4, 12, 1):                                     # fewer than, or no multiple of, the eight key heads
        assert lib.hipvoc_attention_workspace(c._p, heads, 4, 5000, 0) == 0
    assert lib.hipvoc_attention_workspace(c._p, 16, 4, 768, 0) == 0 and lib.hipvoc_attention_workspace(c._p, 16, 4, 5000, 700) == 0
    assert 0 < lib.hipvoc_attention_workspace(c._p, 16, 4, 5000, 0) < 1 << 24
    assert lib.hipvoc_attention_workspace(c._p, 16, 0, 5000, 0) == 0 and lib.hipvoc_attention_workspace(c._p, 16, 4, 0, 0) == 0
    assert lib.hipvoc_attention_workspace(c._p, 16, 2000, 5000, 0) == 0
    assert lib.hipvoc_attention_workspace(c._p, 16384, 1024, 2 ** 31 - 1, 0) > 1 << 32


def test_what_is_refused_and_where_the_kernels_read(tmp_path):
    """tests/native/fuzz_ops.cpp under the host sanitizers: chunks of a sequence cover what its token sees and nothing else, for sound,
    extreme and malformed lengths; positions and pages out of range are never followed; every refusal of the C entry points."""
    if not shutil.which("g++"):
        pytest.skip("no g++")
    exe = str(tmp_path / "fuzz_ops")
    r = subprocess.run(["g++", "-O1", "-g", "-std=c++17", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-o", exe,
                        os.path.join(ROOT, "tests", "native", "fuzz_ops.cpp")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fuzz_ops OK" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


def test_cache_descriptor_refusals(pkg):
    """KvCache looks at its tensors before any handle is involved."""
    import torch
    ok = torch.zeros((3, 2, 16, 64), dtype=torch.bfloat16)
    pkg.KvCache(ok, ok.clone())
    both = torch.zeros((3, 2, 2, 16, 64), dtype=torch.float16)          # K and V as halves of one allocation
    assert pkg.KvCache(both[:, 0], both[:, 1])._c.page_stride == 2 * 2 * 16 * 64
    q = torch.zeros((3, 2, 16, 64), dtype=torch.int8)
    s = torch.zeros((3, 2, 16))
    pkg.KvCache(q, q.clone(), s, s.clone())
    for bad in [lambda: pkg.KvCache(ok, ok[:2]), lambda: pkg.KvCache(ok, ok.float()), lambda: pkg.KvCache(ok[0], ok[0]), lambda: pkg.KvCache(q, q),
                lambda: pkg.KvCache(ok, ok, s, s), lambda: pkg.KvCache(q, q, s, None), lambda: pkg.KvCache(q, q, s, s[:, :1]),
                lambda: pkg.KvCache(q, q, s.double(), s.double()), lambda: pkg.KvCache(ok.transpose(1, 2), ok.transpose(1, 2)),
                lambda: pkg.KvCache(ok.long(), ok.long()), lambda: pkg.KvCache(both[:, 0], ok.half())]:
        with pytest.raises(pkg.HipVocError):
            bad()
