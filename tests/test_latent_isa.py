"""Code-generation invariants of the attention kernels whose matrix products are written out.

The compiler does not know those for MFMAs and puts none of its waits around them, so the device assembly is checked:

* no vector instruction writes an operand of one within two states before it (a copy that register allocation put
  between a fragment's read and its product would do that);
* nothing but another product touches an accumulator until the last product into it has left the pipe: 7 states for a
  16x16x32 product, 11 for a 32x32x16 one;
* the 256-row loop waits for vector memory only by its own count of loads, and no kernel has scratch or flat accesses.
"""

from __future__ import annotations

import re
import subprocess

import pytest

from fused_cpp_amd.build import CSRC, HIP_FLAGS, ROCM

_KERNEL = re.compile(r"^(_Z\w*(?:absorbed|expanded)\w*kernel\w*):", re.M)
_REG = re.compile(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)")


@pytest.fixture(scope="module", params=["fcmoe_absorbed", "fcmoe_expanded"])
def kernels(request, tmp_path_factory):
    hipcc = ROCM / "bin" / "hipcc"
    if not hipcc.exists():
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("isa") / (request.param + ".s")
    proc = subprocess.run([str(hipcc), *HIP_FLAGS, "--cuda-device-only", "-S", str(CSRC / (request.param + ".hip")), "-o",
                           str(out)], capture_output=True, text=True)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    asm = out.read_text()
    found = {}
    for m in _KERNEL.finditer(asm):
        found[m.group(1)] = asm[m.end():asm.index(".Lfunc_end", m.end())].splitlines()
    assert len(found) >= 6, sorted(found)
    return found


def _instructions(body):
    """(text, written out) of each instruction; labels as None."""
    inside = False
    for line in body:
        if "#ASMSTART" in line:
            inside = True
        elif "#ASMEND" in line:
            inside = False
        s = line.split(";")[0].strip()
        if s.endswith(":"):
            yield None
        elif s and not s.startswith("."):
            yield s, inside


def _registers(text):
    out = set()
    for kind, low, high, one in _REG.findall(text):
        out |= {(kind, i) for i in range(int(low or one), int(high or one) + 1)}
    return out


def _operands(text):
    return [_registers(o) for o in text.split(None, 1)[1].split(", ")] if " " in text or "\t" in text else []


def _states(text):
    if text.startswith("s_nop"):
        return int(text.split()[1]) + 1
    if text.startswith("v_mfma"):
        return 8 if "32x32" in text else 4
    return 1


def _vector(text):
    return text.startswith("v_") and not text.startswith("v_mfma")


def _faults(body):
    ins = list(_instructions(body))
    bad, seen = [], 0
    for k, item in enumerate(ins):
        if item is None or not item[1] or not item[0].startswith("v_mfma"):
            continue
        seen += 1
        ops = _operands(item[0])
        dst, src = ops[0], set().union(*ops[1:])
        left = 2
        for prev in reversed(ins[max(0, k - 4):k]):
            if left <= 0 or prev is None:
                break
            if _vector(prev[0]) and _operands(prev[0])[0] & src:
                bad.append(f"{prev[0]}  ->  {item[0]}")
            left -= _states(prev[0])
        left = 11 if "32x32" in item[0] else 7
        for after in ins[k + 1:k + 16]:
            if left <= 0:
                break
            if after is None:
                continue
            if _vector(after[0]) and set().union(set(), *_operands(after[0])) & dst:
                bad.append(f"{item[0]}  ->  {after[0]}")
            left -= _states(after[0])
            if after[0].startswith(("s_branch", "s_endpgm")):
                break
    return bad, seen


def test_the_check_sees_faults():
    ok = ["\t;;#ASMSTART", "\tv_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], a[0:3], 0", "\t;;#ASMEND", "\ts_nop 15", "\tv_add_f32_e32 v30, v0, v1"]
    assert _faults(ok) == ([], 1)
    assert len(_faults(["\tv_mov_b32_e32 v21, v9", "\ts_nop 0"] + ok)[0]) == 1
    assert not _faults(["\tv_mov_b32_e32 v21, v9", "\ts_nop 1"] + ok)[0]
    assert len(_faults(ok[:3] + ["\ts_nop 7", "\tv_add_f32_e32 v30, v0, v1"])[0]) == 1


def test_written_out_products_have_their_waits(kernels):
    seen = 0
    for name, body in kernels.items():
        bad, n = _faults(body)
        assert not bad, (name, bad[:4])
        seen += n
    assert seen >= 352  # the 256-row kernels': S before and in the loop, P V, over the four head sizes


def test_no_scratch_and_no_flat_accesses(kernels):
    for name, body in kernels.items():
        found = [x.strip() for x in body if re.match(r"\s*(flat_|scratch_)", x)]
        assert not found, (name, found[:4])


def test_wide_loop_waits_by_its_own_count(kernels):
    wide = {n: b for n, b in kernels.items() if "wide" in n}
    if not wide:
        pytest.skip("no 256-row kernel in this source")
    assert len(wide) == 4
    for name, body in wide.items():
        first = max(i for i, x in enumerate(body) if "Inner Loop Header" in x)
        last = max(i for i, x in enumerate(body) if "in Loop:" in x)
        waits = {m.group(1) for x in body[first:last] if (m := re.search(r"vmcnt\((\d+)\)", x))}
        assert len(waits) == 1 and waits <= {"10", "8", "6", "4"}, (name, waits)
