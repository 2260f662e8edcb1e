"""Refusals of the softmax operators that need no GPU: shapes, dtypes, options, CPU tensors, and the
C entry points' own argument checks."""

from __future__ import annotations

import ctypes

import pytest
import torch

from qwendopamine_amd import _native as nat
from qwendopamine_amd import ops

BF = torch.bfloat16


def _qkv(B=2, Tq=5, Tk=5, H=4, G=2, D=64, dt=BF):
    return torch.zeros(B, Tq, H, D, dtype=dt), torch.zeros(B, Tk, G, D, dtype=dt), torch.zeros(B, Tk, G, D, dtype=dt)


@pytest.mark.parametrize("err,args,kw", [
    (ValueError, lambda: (_qkv()[0][0], *_qkv()[1:]), {}),
    (ValueError, lambda: _qkv(H=3, G=2), {}),
    (ValueError, lambda: (*_qkv()[:2], _qkv(Tk=6)[2]), {}),
    (ValueError, lambda: (_qkv()[0], *_qkv(B=3)[1:]), {}),
    (ValueError, lambda: (_qkv()[0], *_qkv(D=128)[1:]), {}),
    (ValueError, lambda: (_qkv()[0], *_qkv(dt=torch.float16)[1:]), {}),
    (NotImplementedError, lambda: _qkv(dt=torch.float32), {}),
    (NotImplementedError, lambda: _qkv(D=96), {}),
    (NotImplementedError, lambda: _qkv(), dict(scale=0.0)),
    (NotImplementedError, lambda: _qkv(), dict(scale=-1.0)),
    (NotImplementedError, lambda: _qkv(), dict(scale=float("nan"))),
    (ValueError, lambda: _qkv(), dict(kv_lengths=torch.zeros(3, dtype=torch.int64))),
    (ValueError, lambda: _qkv(), dict(kv_lengths=torch.zeros(2))),
    (ValueError, lambda: _qkv(), dict(cu_seqlens=torch.tensor([0, 5]))),
    (ValueError, lambda: _qkv(B=1, Tk=6), dict(cu_seqlens=torch.tensor([0, 5]))),
    (ValueError, lambda: _qkv(B=1), dict(cu_seqlens=torch.tensor([0, 5]), kv_lengths=torch.tensor([5]))),
    (RuntimeError, lambda: _qkv(), {}),  # CPU tensors
])
def test_attention_refuses(err, args, kw):
    with pytest.raises(err):
        ops.attention(*args(), **kw)


@pytest.fixture(scope="module")
def lib():
    return nat.load()


def _attn_call(lib, **over):
    """gdn2_attn_fwd with pointers that are never dereferenced: every call here must be refused
    (or be empty) before a launch."""
    a = dict(ptr=4096, strides=(256, 256, 64) * 3, o=4096, lse=4096, dt=nat.DTYPE_BF16, kv=None, cu=None, cu_host=None,
             n=0, B=1, Tq=4, Tk=4, H=4, G=2, D=64, scale=1.0)
    a.update(over)
    st = (ctypes.c_int64 * 9)(*a["strides"]) if a["strides"] else None
    host = None if a["cu_host"] is None else (ctypes.c_int64 * len(a["cu_host"]))(*a["cu_host"])
    return lib.gdn2_attn_fwd(a["ptr"], a["ptr"], a["ptr"], st and ctypes.addressof(st), a["o"], None, a["lse"],
                             a["dt"], a["kv"],
                             a["cu"], host and ctypes.addressof(host), a["n"], a["B"], a["Tq"], a["Tk"], a["H"], a["G"],
                             a["D"], a["scale"], 1, None)


@pytest.mark.parametrize("want,over", [
    (nat.ERR_INVALID, dict(dt=9)),
    (nat.ERR_INVALID, dict(H=3)),
    (nat.ERR_INVALID, dict(B=-1)),
    (nat.ERR_INVALID, dict(strides=None)),
    (nat.ERR_INVALID, dict(strides=(256, 260, 64) * 3)),
    (nat.ERR_INVALID, dict(ptr=4104)),
    (nat.ERR_INVALID, dict(ptr=None)),
    (nat.ERR_INVALID, dict(o=None)),
    (nat.ERR_INVALID, dict(cu=4096)),
    (nat.ERR_INVALID, dict(cu=4096, cu_host=(0, 3), n=1)),
    (nat.ERR_INVALID, dict(cu=4096, cu_host=(0, 3, 1, 4), n=3)),
    (nat.ERR_INVALID, dict(cu=4096, cu_host=(0, 9, 4), n=2)),
    (nat.ERR_INVALID, dict(cu=4096, cu_host=(0, 4), n=1, kv=4096)),
    (nat.ERR_UNSUPPORTED, dict(dt=nat.DTYPE_F32)),
    (nat.ERR_UNSUPPORTED, dict(D=96)),
    (nat.ERR_UNSUPPORTED, dict(scale=0.0)),
    (nat.ERR_UNSUPPORTED, dict(scale=float("nan"))),
    (nat.ERR_UNSUPPORTED, dict(B=1 << 30, Tq=1 << 20)),
    (nat.OK, dict(B=0)),
    (nat.OK, dict(Tq=0)),
])
def test_attention_entry_point_checks(lib, want, over):
    assert _attn_call(lib, **over) == want


@pytest.mark.parametrize("err,x,t,kw", [
    (ValueError, torch.zeros(3, 0), torch.zeros(3, dtype=torch.int64), {}),
    (ValueError, torch.zeros(3, 5), torch.zeros(4, dtype=torch.int64), {}),
    (ValueError, torch.zeros(3, 5), torch.zeros(3, dtype=torch.int32), {}),
    (ValueError, torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), dict(top_k=6)),
    (ValueError, torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64), dict(top_k=-1)),
    (NotImplementedError, torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64), dict(top_k=33)),
    (NotImplementedError, torch.zeros(3, 50, dtype=torch.float64), torch.zeros(3, dtype=torch.int64), {}),
    (RuntimeError, torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64), {}),
])
def test_token_logprobs_refuses(err, x, t, kw):
    with pytest.raises(err):
        ops.token_logprobs(x, t, **kw)


@pytest.mark.parametrize("want,over", [
    (nat.ERR_INVALID, dict(dt=nat.DTYPE_I32)),
    (nat.ERR_INVALID, dict(n=0)),
    (nat.ERR_INVALID, dict(inner=0)),
    (nat.ERR_INVALID, dict(sr=-1)),
    (nat.ERR_INVALID, dict(x=4097)),
    (nat.ERR_INVALID, dict(x=None)),
    (nat.ERR_INVALID, dict(t=None)),
    (nat.ERR_INVALID, dict(logp=None)),
    (nat.ERR_INVALID, dict(top=101)),
    (nat.ERR_INVALID, dict(top=5)),  # without outputs for them
    (nat.ERR_UNSUPPORTED, dict(top=33)),
    (nat.ERR_UNSUPPORTED, dict(n=1 << 31)),
    (nat.ERR_UNSUPPORTED, dict(rows=1 << 28)),
    (nat.ERR_WORKSPACE, dict(n=100000)),
    (nat.OK, dict(rows=0)),
])
def test_token_logprobs_entry_point_checks(lib, want, over):
    a = dict(x=4096, inner=4, so=0, sr=100, dt=nat.DTYPE_BF16, rows=4, n=100, t=4096, logp=4096, top=0)
    a.update(over)
    assert lib.gdn2_token_logprobs_fwd(a["x"], a["inner"], a["so"], a["sr"], a["dt"], a["rows"], a["n"], a["t"], -100,
                                       a["logp"], 4096, None, a["top"], None, None, None, 0, None) == want
