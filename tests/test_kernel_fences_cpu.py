"""What the attention kernels hand the compiler, where a wrong result would depend on sizes or on
luck: rows that lanes exchange through LDS are fenced, and offsets of 32 bits do not wrap.  Read from
the unoptimised IR of this repository's own source, where every device function is still one of its own."""

from __future__ import annotations

import ctypes
import re
import subprocess

import pytest

from qwendopamine_amd import _native as nat
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


def test_staged_tiles_fit_their_offsets(tmp_path):
    """A tile's rows are addressed from its first by 32 bits of bytes: ``stage<D, waves, rows>`` at the
    largest token stride that the entry points take."""
    tiles = {tuple(map(int, m)) for n in _functions("gdn2_attn_train.hip", tmp_path)
             for m in re.findall(r"5stageILi(\d+)ELi(\d+)ELi(\d+)EE", n)}
    assert {d for d, _, _ in tiles} == {64, 128}
    for d, _, rows in tiles:
        assert (rows - 1) * 2 * 2 ** 25 + 2 * d <= 2 ** 32 - 1, f"{rows} rows of 2^26 bytes"


@pytest.mark.parametrize("over,want", [(0, nat.ERR_WORKSPACE), (8, nat.ERR_UNSUPPORTED)])
@pytest.mark.parametrize("i", [1, 4, 7])
def test_largest_token_stride(i, over, want):
    """2^25 elements are taken (the call then ends for its missing workspace, before any launch)."""
    st = [256, 256, 64] * 3
    st[i] = 2 ** 25 + over
    st = (ctypes.c_int64 * 9)(*st)
    got = nat.load().gdn2_attn_fwd(4096, 4096, 4096, ctypes.addressof(st), 4096, None, 4096,
                                   nat.DTYPE_BF16, None, None, None, 0, 1, 4, 100000, 4, 2, 64, 1.0, 1, None, 0, None)
    assert got == want
