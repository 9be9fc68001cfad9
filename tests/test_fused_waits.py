"""Guards on the compiled gfx950 code of the products whose results go straight into what follows (fused_tiles.hip, fused_rows.hip,
fused_logits.hip), whose LDS copies are written out and so not waited for by the compiler: m0 is set by the copies alone, right
before each, and on every path the copies that others read have landed at a barrier. A tile kernel's barrier comes before even and
odd tiles in turn: at most the next piece's words and scales may be in flight there, never a row of a; the kernel of few rows has
none in flight at any of its barriers. Registers that a kernel spills are few: it needs the waves a SIMD that it asks for."""
import os
import re
import subprocess

import pytest
from test_tile_waits import CSRC, HIPCC, ROOT, blocks_of, copies_at_barriers

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc is missing")
FILES = ("fused_tiles.hip", "fused_rows.hip", "fused_logits.hip")


@pytest.fixture(scope="module")
def compiled(tmp_path_factory):
    """The files' assembly, compiled side by side."""
    d = tmp_path_factory.mktemp("s")
    runs = {f: subprocess.Popen([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                                 "-mllvm", "-amdgpu-mfma-vgpr-form", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC, "-x", "hip", "-S",
                                 "--cuda-device-only", os.path.join(CSRC, f), "-o", str(d / (f + ".s"))], stderr=open(str(d / (f + ".err")), "w"))
            for f in FILES}
    for f, r in runs.items():
        r.wait(timeout=900)
        assert r.returncode == 0, (d / (f + ".err")).read_text()
    out = {}
    for f in FILES:
        text = (d / (f + ".s")).read_text()
        out[f] = f, text, [(m.group(1), m.group(0)) for m in re.finditer(r"^(_Z\w*fused_\w*kernel\w*):.*?^\.Lfunc_end", text, re.M | re.S)]
    return out


@pytest.fixture(params=FILES)
def code(request, compiled):
    return compiled[request.param]


def test_m0_is_written_only_by_the_copies(code):
    name, _, kernels = code
    seen = 0
    for kernel, body in kernels:
        lines = [l for l in (l.strip() for l in body.splitlines()) if l and not l.startswith((";", "."))]
        refs = [i for i, l in enumerate(lines) if re.search(r"\bm0\b", l.split(";")[0])]
        seen += len(refs)
        for i in refs:
            assert lines[i].startswith("s_mov_b32 m0,"), (kernel, lines[i])
            assert lines[i + 1].startswith("global_load_lds_dword"), (kernel, lines[i], lines[i + 1])
        assert len(refs) == sum(l.startswith("global_load_lds") for l in lines), kernel
    assert seen


def test_copies_have_landed_at_every_barrier(code):
    name, _, kernels = code
    checked = 0
    for kernel, body in kernels:
        if "fused_tiles_kernel" in kernel:
            bits, asym, epi, rt, ct = (int(x) for x in re.search(r"kernelI" + r"L[ib](\d+)E" * 5, kernel).groups())
            allowed = (2 * ct if bits == 4 else 2 * ct * bits) + (4 if asym else 2)  # a piece's words, its two of the scales
        elif "fused_rows_kernel" in kernel:
            allowed = 0
        else:
            continue
        worst, barriers = copies_at_barriers(blocks_of(body.splitlines()[1:]))
        assert barriers
        assert worst <= allowed, (kernel, "copies in flight at a barrier: %d of %d" % (worst, allowed))
        checked += 1
    assert checked


def test_spills_are_few(code):
    _, text, kernels = code
    assert len(kernels) >= 15
    spills = re.findall(r"\.name:\s+(_Z\w*fused_\w*kernel\w*).*?\.vgpr_spill_count:\s+(\d+)", text, re.S)
    assert len(spills) == len(kernels)
    assert [(k, n) for k, n in spills if int(n) > 8] == []  # (128 rows x 64 columns of 3 bits: 5, of a loop of 1800 instructions)
