"""The code-generation checks of tests/test_latent_isa.py and tests/test_latent_isa_waits.py, for the attention kernels'
forms over a part of the context: waits around written-out products on every path, no scratch, no flat accesses."""

from __future__ import annotations

import re
import subprocess

import pytest

from fused_cpp_amd.build import CSRC, HIP_FLAGS, ROCM
from tests import test_latent_isa as near
from tests import test_latent_isa_waits as waits

PRODUCTS = {"fcmoe_absorbed_masked": 1, "fcmoe_expanded_window": 352}


@pytest.fixture(scope="module", params=sorted(PRODUCTS))
def kernels(request, tmp_path_factory):
    hipcc = ROCM / "bin" / "hipcc"
    if not hipcc.exists():
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("isa") / (request.param + ".s")
    proc = subprocess.run([str(hipcc), *HIP_FLAGS, "--cuda-device-only", "-S", str(CSRC / (request.param + ".hip")), "-o",
                           str(out)], capture_output=True, text=True)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    asm = out.read_text()
    found = {m.group(1): asm[m.end():asm.index(".Lfunc_end", m.end())].splitlines() for m in near._KERNEL.finditer(asm)}
    assert len(found) >= 10, sorted(found)
    return request.param, found


def test_products_have_their_waits(kernels):
    source, found = kernels
    seen = 0
    for name, body in found.items():
        for check in (near, waits):
            bad, n = check._faults(body)
            assert not bad, (name, bad[:4])
        seen += n
    assert seen >= PRODUCTS[source]


def test_no_scratch_and_no_flat_accesses(kernels):
    for name, body in kernels[1].items():
        bad = [x.strip() for x in body if re.match(r"\s*(flat_|scratch_)", x)]
        assert not bad, (name, bad[:4])


def test_wide_loop_waits_by_its_own_count(kernels):
    wide = {n: b for n, b in kernels[1].items() if "wide" in n}
    if not wide:
        pytest.skip("no 256-row kernel in this source")
    assert len(wide) == 4
    for name, body in wide.items():
        first = max(i for i, x in enumerate(body) if "Inner Loop Header" in x)
        last = max(i for i, x in enumerate(body) if "in Loop:" in x)
        counts = {m.group(1) for x in body[first:last] if (m := re.search(r"vmcnt\((\d+)\)", x))}
        assert len(counts) == 1 and counts <= {"10", "8", "6", "4"}, (name, counts)
