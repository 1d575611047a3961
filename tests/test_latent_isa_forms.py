"""Code generation of the attention kernels, checked in the device assembly beside what tests/test_latent_isa.py and
tests/test_latent_masked_isa.py check:

* every instance of a kernel is there, with as many written-out products as its sizes ask for, so that the checks of the
  waits around those look at all of them;
* no region of lanes is empty. Where one of a vector's values is replaced under `a || b`, the block that does it is reached
  by two branches; the compiler then forms the new vector ahead of the first branch only, in the registers that the
  lanes which come by the second one have filled with the old vector again, and leaves the block empty: those lanes keep
  the old value. Scores are masked without branches for that reason, or under a condition that becomes a select.
"""

from __future__ import annotations

import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from fused_cpp_amd.build import CSRC, HIP_FLAGS, ROCM
from tests.test_latent_isa import _KERNEL, _instructions

SOURCES = ("fcmoe_absorbed", "fcmoe_absorbed_masked", "fcmoe_expanded", "fcmoe_expanded_window")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    hipcc = ROCM / "bin" / "hipcc"
    if not hipcc.exists():
        pytest.skip("hipcc not available")
    to = tmp_path_factory.mktemp("isa")

    def compiled(source):
        out = to / (source + ".s")
        proc = subprocess.run([str(hipcc), *HIP_FLAGS, "--cuda-device-only", "-S", str(CSRC / (source + ".hip")), "-o", str(out)],
                              capture_output=True, text=True)
        assert proc.returncode == 0, proc.stdout + proc.stderr
        asm = out.read_text()
        return {m.group(1): asm[m.end():asm.index(".Lfunc_end", m.end())].splitlines() for m in _KERNEL.finditer(asm)}

    with ThreadPoolExecutor(len(SOURCES)) as pool:
        return dict(zip(SOURCES, pool.map(compiled, SOURCES)))


def _empty_regions(body):
    """Instructions that narrow the lanes to some for which nothing follows before the others are back."""
    found, narrowed = [], None
    for item in _instructions(body):
        if item is None:
            continue
        if narrowed and re.match(r"s_or_b64\s+exec, exec", item[0]):
            found.append(narrowed)
        narrowed = item[0] if item[0].startswith("s_and_saveexec") else None
    return found


def test_the_check_sees_an_empty_region():
    body = ["\ts_and_saveexec_b64 s[0:1], s[2:3]", ".LBB0_1:", "; %bb.46:", "\ts_or_b64 exec, exec, s[0:1]"]
    assert len(_empty_regions(body)) == 1
    assert not _empty_regions(body[:1] + ["\tv_mov_b32_e32 v50, s2"] + body[1:])
    assert not _empty_regions(["\ts_andn2_saveexec_b64 s[0:1], s[0:1]"] + body[1:])  # an else part whose value is there


@pytest.mark.parametrize("source", SOURCES)
def test_no_region_of_lanes_is_empty(kernels, source):
    for name, body in kernels[source].items():
        found = _empty_regions(body)
        assert not found, (name, len(found), found[:4])


def _products(name):
    """Written-out products of an instance by its template arguments, or None for a kernel without any."""
    kernel = re.search(r"(absorbed_tall|absorbed|expanded_wide)_kernelI", name)
    if not kernel:
        return None
    args = [int(v) for v in re.findall(r"L[ib](\d+)E", name[kernel.end() - 1:])]
    if kernel.group(1) == "absorbed_tall":
        R, P = args[:2]  # S of a tile's first half with and without whole pages, of its second; P V and zeros
        return 3 * (R + P) // 16 + 5 * R // 32
    if kernel.group(1) == "absorbed":
        R, P, _, MT = args[:4]  # 16 rows leave S to the compiler
        return 3 * (R + P) // 32 * MT if MT > 1 else 0
    N, P, V = args[:3]  # S before the loop and in it, P V
    return 8 * (N + P) // 16 + 8 * V // 32


@pytest.mark.parametrize("source,count", [("fcmoe_absorbed", 32), ("fcmoe_absorbed_masked", 32), ("fcmoe_expanded", 4),
                                          ("fcmoe_expanded_window", 4)])
def test_every_instance_has_its_products(kernels, source, count):
    seen = 0
    for name, body in kernels[source].items():
        want = _products(name)
        if want is not None:
            seen += 1
            got = sum(written and text.startswith("v_mfma") for text, written in filter(None, _instructions(body)))
            assert got == want, (name, got, want)
    assert seen == count
    if source == "fcmoe_absorbed_masked":
        assert sum("absorbed_tall" in name for name in kernels[source]) == 8
