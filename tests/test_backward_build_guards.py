"""Guards on the compiled attention backward kernels (CPU; needs hipcc).

Their copies to LDS are inline ``global_load_lds_dwordx4`` with M0 as the LDS
base, hidden from the compiler's memory counters and ordered by explicit waits
and barriers in the source.  That rests on facts of the toolchain: nothing else
touches M0, every copy follows its own ``s_mov_b32 m0``, the compiler's own
waits inside the loops over units do not wait for the copies in flight, and no
packed fp32 instruction is formed.
"""
from __future__ import annotations

import re

import pytest

from test_build_guards import HIPCC, PKG, _device_asm, _kernels

pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc is not installed")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    out = tmp_path_factory.mktemp("backward_asm") / "attention_backward.s"
    return _kernels(_device_asm(PKG / "csrc" / "attention_backward.hip", out))


def test_only_the_copies_use_m0(kernels):
    copies = 0
    for name, body in kernels.items():
        for i, instr in enumerate(body):
            if re.search(r"\bm0\b", instr):
                assert re.fullmatch(r"s_mov_b32 m0, s\d+", instr), f"{name}: M0 used by '{instr}'"
                assert body[i + 1] == "s_nop 0" and body[i + 2].startswith("global_load_lds_dwordx4"), \
                    f"{name}: 's_mov_b32 m0' is not followed by its copy: {body[i:i + 3]}"
            if instr.startswith("global_load_lds_dwordx4"):
                copies += 1
                assert body[i - 2].startswith("s_mov_b32 m0"), f"{name}: a copy without its own 's_mov_b32 m0'"
    assert copies > 0


def test_waits_for_the_copies_come_with_a_barrier(kernels):
    """Between the first copy and the last barrier a full wait for loads stands before an s_barrier only."""
    mains = {n: b for n, b in kernels.items() if "attention_backward_kernel" in n}
    assert len(mains) == 12
    for name, body in mains.items():
        waits = [i for i, x in enumerate(body) if x.startswith("s_waitcnt") and "vmcnt(0)" in x and "lgkmcnt(0)" in x
                 and body[i + 1] == "s_barrier"]
        assert len(waits) >= 4, f"{name}: the waits that order the copies are missing"


def test_no_packed_fp32(kernels):
    for name, body in kernels.items():
        bad = [x for x in body if re.match(r"v_pk_(add|mul|fma)_f32", x)]
        assert not bad, f"{name}: {bad[:3]}"
