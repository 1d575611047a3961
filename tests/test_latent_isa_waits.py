"""Waits around the matrix products of the attention kernels, followed through labels and branches.

The compiler puts waits between a product and other instructions that touch its result or its accumulator operand, and
ahead of a product that reads what a vector instruction has just written; around instructions that are written out it
puts none. For gfx950 those are 8 states behind a 16x16x32 product, 12 behind a 32x32x16 one, and two ahead (its own
output for the same products is compared below). Where one of the two is written out they are checked here: on every
path, for vector, LDS and memory instructions alike, and for products that take the result as a factor or as part of
another accumulator.
"""

from __future__ import annotations

import re
import subprocess

import pytest

from fused_cpp_amd.build import HIP_FLAGS, ROCM
from tests.test_latent_isa import _operands, _registers, _states, _vector, kernels  # noqa: F401

READ_AFTER = {"16x16": 8, "32x32": 12}
WRITE_BEFORE = 2


def _parse(body):
    """Instructions as (text, written out), and the index that each label stands before."""
    ins, labels, inside = [], {}, False
    for line in body:
        if "#ASMSTART" in line:
            inside = True
        elif "#ASMEND" in line:
            inside = False
        s = line.split(";")[0].strip()
        if s.endswith(":"):
            labels[s[:-1]] = len(ins)
        elif s and not s.startswith("."):
            ins.append((s, inside))
    return ins, labels


def _target(text):
    return text.split()[-1] if text.startswith(("s_branch", "s_cbranch")) else None


def _edges(ins, labels):
    after = [[] for _ in ins]
    for k, (text, _) in enumerate(ins):
        to = _target(text)
        if to in labels and labels[to] < len(ins):
            after[k].append(labels[to])
        if not text.startswith(("s_branch", "s_endpgm", "s_setpc")) and k + 1 < len(ins):
            after[k].append(k + 1)
    before = [[] for _ in ins]
    for k, to in enumerate(after):
        for t in to:
            before[t].append(k)
    return after, before


def _walk(start, edges, left, ins):
    """Indices that lie fewer than `left` states from `start` on some path."""
    best, todo = {}, [(k, left) for k in edges[start]]
    while todo:
        k, left = todo.pop()
        if left <= 0 or best.get(k, 0) >= left:
            continue
        best[k] = left
        todo += [(n, left - _states(ins[k][0])) for n in edges[k]]
    return best


def _touches(text, dst, acc):
    """Whether an instruction depends on a product that still runs, or overwrites the accumulator that it still reads:
    products add to the very same accumulator in turn."""
    ops = _operands(text)
    if text.startswith("v_") and ops and ops[0] & acc and not (text.startswith("v_mfma") and ops[0] == acc):
        return True
    if text.startswith("v_mfma"):
        if (ops[1] | ops[2]) & dst:
            return True
        return any(o & dst and o != dst for o in (ops[0], ops[3] if len(ops) > 3 else set()))
    return bool(set().union(set(), *ops) & dst)


def _faults(body):
    ins, labels = _parse(body)
    after, before = _edges(ins, labels)
    bad, seen = [], 0
    for k, (text, written) in enumerate(ins):
        if not text.startswith("v_mfma"):
            continue
        seen += written
        ops = _operands(text)
        dst, src = ops[0], set().union(*ops[1:])
        for n in _walk(k, after, READ_AFTER["32x32" if "32x32" in text else "16x16"], ins):
            if not (written or ins[n][1]) or ins[n][0].startswith("s_") or n == k:
                continue
            if _touches(ins[n][0], dst, ops[3]):
                bad.append(f"{text}  ->  {ins[n][0]}")
        if written:
            for n in _walk(k, before, WRITE_BEFORE, ins):
                if _vector(ins[n][0]) and _operands(ins[n][0])[0] & src:
                    bad.append(f"{ins[n][0]}  ->  {text}")
    return bad, seen


SMALL = ["\t;;#ASMSTART", "\tv_mfma_f32_16x16x32_bf16 v[0:3], v[20:23], a[0:3], v[0:3]", "\t;;#ASMEND"]
LARGE = ["\t;;#ASMSTART", "\tv_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], a[0:3], 0", "\t;;#ASMEND"]
USES = ["\tv_add_f32_e32 v30, v0, v1", "\tglobal_store_dwordx4 v40, v[0:3], s[2:3]", "\tds_write_b64 v40, v[2:3]",
        "\tbuffer_store_dword v3, v40, s[0:3], 0 offen", "\tv_mfma_f32_16x16x32_bf16 v[40:43], v[0:3], v[50:53], 0",
        "\tv_mfma_f32_16x16x32_bf16 v[2:5], v[40:43], v[50:53], 0", "\tv_mov_b32_e32 v1, 0"]


@pytest.mark.parametrize("use", USES)
@pytest.mark.parametrize("product,states", [(SMALL, 8), (LARGE, 12)])
def test_the_check_sees_a_result_used_one_state_early(product, states, use):
    assert _faults(product + [f"\ts_nop {states - 1}", use]) == ([], 1)
    short = product + [f"\ts_nop {states - 2}"]
    assert len(_faults(short + [use])[0]) == 1
    assert len(_faults(short + [".LBB0_1:", use])[0]) == 1  # past a label
    # behind a branch, taken or not
    away = ["\ts_cbranch_scc1 .LBB0_2", "\ts_nop 15", "\ts_endpgm", ".LBB0_2:", use]
    assert len(_faults(product + [f"\ts_nop {states - 3}"] + away)[0]) == 1
    assert not _faults(product + [f"\ts_nop {states - 2}"] + away)[0]
    assert not _faults(product + ["\ts_branch .LBB0_2", use, ".LBB0_2:", "\ts_endpgm"])[0]


def test_the_check_sees_written_out_vector_instructions():
    """Of the compiler's own products only what is written out behind them has to be looked at."""
    mine = ["\tv_mfma_f32_16x16x32_bf16 v[60:63], v[40:43], v[44:47], v[86:89]"]
    for to in ("v86", "v61"):  # the accumulator it reads, the one it writes
        lane = ["\t;;#ASMSTART", f"\tv_mbcnt_lo_u32_b32 {to}, -1, 0", "\t;;#ASMEND"]
        assert len(_faults(mine + lane)[0]) == 1
        assert len(_faults(mine + ["\ts_nop 6"] + lane)[0]) == 1
        assert not _faults(mine + ["\ts_nop 7"] + lane)[0]
        assert not _faults(mine + lane[1:2])[0]


def test_the_check_sees_an_operand_written_too_late():
    for product in (SMALL, LARGE):
        for write in ("\tv_mov_b32_e32 v21, v9", "\tv_accvgpr_write_b32 a2, v9"):
            assert len(_faults([write] + product)[0]) == 1
            assert len(_faults([write, "\ts_nop 0"] + product)[0]) == 1
            assert len(_faults([write, ".LBB0_1:"] + product)[0]) == 1  # the end of a block before the product's
            assert len(_faults([write, "\ts_branch .LBB0_1", "\tv_mov_b32_e32 v60, v9", ".LBB0_1:"] + product)[0]) == 1
            assert not _faults([write, "\ts_nop 1"] + product)[0]
    assert not _faults(SMALL + SMALL)[0]


def test_the_compilers_own_waits(tmp_path):
    """What the compiler puts behind these products itself is what is asked for here."""
    hipcc = ROCM / "bin" / "hipcc"
    if not hipcc.exists():
        pytest.skip("hipcc not available")
    src = tmp_path / "products.hip"
    src.write_text("#include <hip/hip_runtime.h>\ntypedef __bf16 v8bf __attribute__((ext_vector_type(8)));\n" + "".join(
        f"typedef float acc{n} __attribute__((ext_vector_type({n})));\n"
        f"__global__ void product_{shape}(v8bf* x, acc{n}* o) {{ acc{n} s = {{}}; "
        f"s = __builtin_amdgcn_mfma_f32_{shape}_bf16(x[threadIdx.x], x[threadIdx.x + 64], s, 0, 0, 0); s[0] += 1.0f; "
        f"o[threadIdx.x] = s; }}\n" for shape, n in (("16x16x32", 4), ("32x32x16", 16))))
    out = tmp_path / "products.s"
    subprocess.run([str(hipcc), *HIP_FLAGS, "--cuda-device-only", "-S", str(src), "-o", str(out)], check=True, capture_output=True)
    body = out.read_text().splitlines()
    waits = [int(b.split()[1]) + 1 for a, b in zip(body, body[1:]) if "v_mfma" in a and "s_nop" in b]
    assert waits == [READ_AFTER["16x16"], READ_AFTER["32x32"]]


def test_products_have_their_waits_on_every_path(kernels):  # noqa: F811
    seen = 0
    for name, body in kernels.items():
        bad, n = _faults(body)
        assert not bad, (name, bad[:4])
        seen += n
    assert seen >= 352
