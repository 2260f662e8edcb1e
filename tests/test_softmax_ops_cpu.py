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
                             a["D"], a["scale"], 1, None, 0, None)


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
    (nat.ERR_UNSUPPORTED, dict(Tq=1 << 24, H=128, G=1)),  # 2^31 rows of one group
    (nat.ERR_WORKSPACE, dict(Tk=100000)),
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


def _cache(B=2, G=2, L=10, D=64):
    return ops.kv_cache_q4(B, G, L, D)


def test_kv_cache_q4_shapes():
    c = ops.kv_cache_q4(2, 3, 5, 128)
    assert c.k.shape == (2, 3, 5, 64) and c.k_meta.shape == (2, 3, 5, 2, 2) and c.v.dtype == torch.uint8
    with pytest.raises(NotImplementedError):
        ops.kv_cache_q4(1, 1, 1, 80)


@pytest.mark.parametrize("err,cache,kv,start", [
    (ValueError, _cache(), torch.zeros(3, 4, 2, 64), None),
    (ValueError, _cache(), torch.zeros(2, 4, 2, 128), None),
    (ValueError, _cache()._replace(k=torch.zeros(2, 2, 9, 32, dtype=torch.uint8)), torch.zeros(2, 4, 2, 64), None),
    (ValueError, _cache()._replace(k=torch.zeros(2, 2, 10, 32)), torch.zeros(2, 4, 2, 64), None),
    (ValueError, _cache()._replace(v_meta=torch.zeros(2, 2, 10, 1, 2)), torch.zeros(2, 4, 2, 64), None),
    (ValueError, ops.KVCacheQ4(*(t.transpose(0, 1) for t in _cache())), torch.zeros(2, 4, 2, 64), None),
    (NotImplementedError, _cache(), torch.zeros(2, 4, 2, 64, dtype=torch.float64), None),
    (RuntimeError, _cache(), torch.zeros(2, 4, 2, 64), None),
])
def test_kv_cache_q4_store_refuses(err, cache, kv, start):
    with pytest.raises(err):
        ops.kv_cache_q4_store(cache, kv, kv, start)


@pytest.mark.parametrize("err,over", [
    (ValueError, dict(n_head=3)),
    (ValueError, dict(n_head=0)),
    (ValueError, dict(qkv=torch.zeros(2, 1, 100, dtype=BF))),
    (ValueError, dict(pos=None)),
    (NotImplementedError, dict(qkv=torch.zeros(2, 1, 8 * 64))),
    (NotImplementedError, dict(qkv=torch.zeros(2, 1, 38 * 64, dtype=BF), n_head=34)),
    (RuntimeError, dict()),
])
def test_attention_decode_q4_refuses(err, over):
    a = dict(qkv=torch.zeros(2, 1, 8 * 64, dtype=BF), cos=torch.zeros(10, 32), pos=torch.tensor([1]), n_head=4)
    a.update(over)
    with pytest.raises(err):
        ops.attention_decode_q4(a["qkv"], a["cos"], a["cos"], a["pos"], _cache(), a["n_head"])


def test_positions_are_checked():
    for bad in (torch.zeros(3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.int64)):
        with pytest.raises(ValueError):
            ops._positions("x", "start", bad, 2, torch.device("cpu"))
    with pytest.raises(RuntimeError):
        ops._positions("x", "start", torch.zeros(2, dtype=torch.int64), 2, torch.device("cpu"))


@pytest.mark.parametrize("want,over", [
    (nat.ERR_INVALID, dict(dt=9)),
    (nat.ERR_INVALID, dict(qpk=0)),
    (nat.ERR_INVALID, dict(L=0)),
    (nat.ERR_INVALID, dict(pairs=33)),
    (nat.ERR_INVALID, dict(cos=None)),
    (nat.ERR_INVALID, dict(rs=8)),
    (nat.ERR_INVALID, dict(kc=4104)),
    (nat.ERR_INVALID, dict(km=4098)),
    (nat.ERR_INVALID, dict(pos=None)),
    (nat.ERR_UNSUPPORTED, dict(dt=nat.DTYPE_F32)),
    (nat.ERR_UNSUPPORTED, dict(qpk=17)),
    (nat.ERR_UNSUPPORTED, dict(D=192)),
    (nat.ERR_UNSUPPORTED, dict(D=96)),
    (nat.ERR_UNSUPPORTED, dict(L=1 << 31)),
    (nat.ERR_WORKSPACE, dict(L=100000)),
    (nat.OK, dict(B=0)),
])
def test_attention_decode_q4_entry_point_checks(lib, want, over):
    a = dict(cos=4096, pairs=32, rs=32, pos=4096, kc=4096, km=4096, dt=nat.DTYPE_BF16, B=1, G=1, qpk=1, D=64, L=10)
    a.update(over)
    assert lib.gdn2_attn_decode_q4(4096, a["cos"], a["cos"], a["pairs"], a["rs"], a["pos"], 0, a["kc"], a["km"], a["kc"],
                                   a["km"], 4096, a["dt"], a["B"], a["G"], a["qpk"], a["D"], a["L"], 1.0, None, 0,
                                   None) == want


def test_hybrid_options_are_checked():
    from qwendopamine_amd.hybrid import HybridConfig, HybridDecoder

    with pytest.raises(ValueError):
        HybridConfig(attention="other")
    cfg = HybridConfig(n_layer=1, n_embd=64, n_head=1, n_query_groups=1, intermediate_size=64, vocab_size=10,
                       gdn2_layers=[], block_size=16, attention="hip")
    m = HybridDecoder(cfg).eval()
    with pytest.raises(ValueError):
        m.setup_caches(1, 8, kv_bits=8)
    with pytest.raises(NotImplementedError):
        m.setup_caches(1, 8, kv_bits=4)  # on the CPU
    idx = torch.zeros(1, 5, dtype=torch.int64)
    assert m(idx).shape == (1, 5, 10)  # on the CPU "hip" is torch's attention
    with pytest.raises(RuntimeError):
        m.loss(idx)


@pytest.mark.parametrize("make", [
    lambda: torch.tensor([0, 5, 70, 400]),
    lambda: torch.tensor([0, 5, 70, 400], dtype=torch.int32),
    lambda: torch.tensor([[0, 1], [5, 1], [70, 1], [400, 1]])[:, 0],
])
def test_packed_offsets_are_copied(make):
    """A backward pass takes its sizes from the host's offsets: they may not change with the
    caller's buffer, which a data loader writes again before the backward."""
    cu = make()
    dev, host = ops._cu(cu, torch.device("cpu"), 400)
    cu[1], cu[2] = 399, 399
    assert host.tolist() == [0, 5, 70, 400] and dev.tolist() == [0, 5, 70, 400]
    assert host.dtype == torch.int64 and host.is_contiguous()


# A launch holds fewer than 2^32 threads: sizes beyond are refused before any (or take several).

@pytest.mark.parametrize("over", [
    dict(B=1 << 20, Tq=1, Tk=1, H=32, G=32),                                   # a workgroup per row and head
    dict(B=1 << 24, Tq=1, Tk=1, H=1, G=1),
    dict(cu=4096, cu_host=tuple(range((1 << 20) + 1)), n=1 << 20, Tq=1 << 20, Tk=1 << 20, H=32, G=32),
])
def test_attention_refuses_more_than_a_launch(lib, over):
    assert _attn_call(lib, **over) == nat.ERR_UNSUPPORTED


def test_attention_forward_for_a_gradient_is_refused_with_it(lib):
    """Few queries over the long keys of very many rows: their forward is one launch, the gradient of
    the keys is not.  A forward that keeps what the gradient reads is refused as it is (the calls end
    for what they lack, before any launch)."""
    B, Tk, st = 1 << 23, 257, (ctypes.c_int64 * 9)(*(256, 256, 64) * 3)

    def call(o, o_lo):
        return lib.gdn2_attn_fwd(4096, 4096, 4096, ctypes.addressof(st), o, o_lo, 4096, nat.DTYPE_BF16, None, None, None,
                                 0, B, 1, Tk, 1, 1, 64, 1.0, 1, None, 0, None)

    assert call(None, None) == nat.ERR_INVALID  # sizes accepted, no output given
    assert call(None, 4096) == nat.ERR_UNSUPPORTED
    size = lib.gdn2_attn_bwd_workspace_size
    assert size(None, 0, B, 1, Tk, 1, 1, 64, 1) == 0 and size(None, 0, 1 << 10, 1, Tk, 1, 1, 64, 1) > 0


def test_four_bit_cache_refuses_more_than_a_launch(lib):
    def decode(B, G, qpk=1, L=10):
        return lib.gdn2_attn_decode_q4(4096, 4096, 4096, 32, 32, 4096, 0, 4096, 4096, 4096, 4096, 4096, nat.DTYPE_BF16, B,
                                       G, qpk, 64, L, 1.0, None, 0, None)

    assert decode(1 << 20, 32) == nat.ERR_UNSUPPORTED
    assert decode(1 << 16, 32, 16, 5000) == nat.ERR_UNSUPPORTED  # shares: a merge per query head
    st = (ctypes.c_int64 * 6)(*(256, 256, 64) * 2)
    store = (4096, 4096, ctypes.addressof(st), nat.DTYPE_BF16, None, 0, 4096, 4096, 4096, 4096)
    load = (4096, 4096, 4096, 4096, None, 0, 4096, 4096, nat.DTYPE_BF16)
    for f, head in ((lib.gdn2_kv_cache_q4_store, store), (lib.gdn2_kv_cache_q4_load, load)):
        assert f(*head, 1 << 19, 1, 32, 64, 10, None) == nat.ERR_UNSUPPORTED
        assert f(*head, 4, 1 << 29, 1, 64, 10, None) == nat.ERR_UNSUPPORTED


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(monkeypatch, grad):
    """A tangent on any input, with and without gradients, never yields a result without one.  The
    launches are stood in for."""
    from torch.autograd import forward_ad

    monkeypatch.setattr(ops, "_require_gpu", lambda *a: None)
    monkeypatch.setattr(ops, "_attention_fwd", lambda q, *a: (torch.zeros_like(q),) * 3)
    monkeypatch.setattr(ops, "_token_logprobs_fwd",
                        lambda x, t, *a: (torch.zeros(t.shape), torch.zeros(t.shape), None, None, x, None))
    logits, targets = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for i in range(3):
            x = list(_qkv())
            x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises(NotImplementedError):
                ops.attention(*x)
        with pytest.raises(NotImplementedError):
            ops.token_logprobs(forward_ad.make_dual(logits, torch.ones_like(logits)), targets)
        # Without a tangent nothing changes within the level.
        assert ops.attention(*_qkv()).shape == (2, 5, 4, 64) and ops.token_logprobs(logits, targets).logprobs.shape == (3,)
