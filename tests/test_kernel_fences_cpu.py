"""Rows that lanes hand each other through LDS: what the compiler is given has to order the stores
before the loads.  Read from the unoptimised IR of this repository's own source, where every device
function is still one of its own."""

from __future__ import annotations

import re
import subprocess

import pytest

from qwendopamine_amd import build


def _functions(source: str, tmp_path) -> dict[str, str]:
    """Name to body of every device function of ``source``."""
    try:
        hipcc = build._hipcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    out = tmp_path / "device.ll"
    flags = [f for f in build.HIPCC_FLAGS if f != "-O3"]
    subprocess.run([hipcc, *flags, "-O1", "-Xclang", "-disable-llvm-passes", "--cuda-device-only", "-S", "-emit-llvm",
                    str(build.CSRC / source), "-o", str(out)], check=True, capture_output=True)
    return {m[1]: m[2] for m in re.finditer(r"^define [^@\n]*@([\w.$]+)\([^\n]*\{\n(.*?)^\}", out.read_text(), re.M | re.S)}


def test_rows_exchanged_through_lds_are_fenced(tmp_path):
    """``put_rows`` stores a lane's channels of its row, ``write_rows`` loads whole rows that other
    lanes stored, and the next ``put_rows`` overwrites them: each ends with the fence."""
    fn = _functions("gdn2_attn_train.hip", tmp_path)
    fence = [b for n, b in fn.items() if "wave_fence" in n]
    assert fence and all('fence syncscope("wavefront") acq_rel' in b and "llvm.amdgcn.wave.barrier" in b for b in fence)
    both = {n: b for n, b in fn.items() if "put_rows" in n or "write_rows" in n}
    # Two types x two head sizes x two forms of the forward, dq and dk / dv, and both sides of each.
    assert len(both) >= 2 * 2 * 2 * 3 * 2
    for name, body in both.items():
        at = body.rfind("wave_fence")
        assert at >= 0, f"{name} has no fence"
        assert not re.search(r"^\s*(%\S+ = load|store) ", body[at:], re.M), f"{name} touches memory after its fence"
