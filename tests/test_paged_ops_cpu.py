"""Refusals of the norm-and-rotation pass, the paged cache, its attention and the sampling that need no
GPU: shapes, dtypes, settings, CPU tensors, and the C entry points' own argument checks (page tables
and sizes that no kernel may index by)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from qwendopamine_amd import _native as nat
from qwendopamine_amd import ops

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _rope(B=2, T=5, H=4, G=2, D=64, dt=BF, rows=9, pairs=32, wdt=BF, **over):
    a = dict(qkv=torch.zeros(B, T, (H + 2 * G) * D, dtype=dt), cos=torch.zeros(rows, pairs), sin=torch.zeros(rows, pairs),
             n_head=H, n_query_groups=G, q_weight=torch.ones(D, dtype=wdt), k_weight=torch.ones(D, dtype=wdt))
    a.update(over)
    return a


@pytest.mark.parametrize("err,over", [
    (ValueError, dict(qkv=torch.zeros(5, 512, dtype=BF))),
    (ValueError, dict(qkv=torch.zeros(2, 5, 500, dtype=BF))),
    (ValueError, dict(n_head=3)),
    (ValueError, dict(n_query_groups=0)),
    (NotImplementedError, dict(D=12, pairs=4)),
    (NotImplementedError, dict(D=264)),
    (NotImplementedError, dict(dt=torch.float64, wdt=torch.float64)),
    (ValueError, dict(k_weight=None)),
    (ValueError, dict(q_weight=torch.ones(32, dtype=BF))),
    (ValueError, dict(wdt=FP)),
    (ValueError, dict(q_weight=torch.ones(64))),
    (ValueError, dict(pairs=33)),
    (ValueError, dict(cos=torch.zeros(9, 16))),
    (ValueError, dict(cos=torch.zeros(9, 32, dtype=BF), sin=torch.zeros(9, 32, dtype=BF))),
    (ValueError, dict(cos=torch.zeros(32, 9).T)),
    (ValueError, dict(cos=torch.zeros(9, 32, requires_grad=True))),
    (ValueError, dict(rows=4)),
    (ValueError, dict(input_pos=torch.zeros(5, dtype=torch.int32))),
    (ValueError, dict(input_pos=torch.zeros(1, dtype=torch.int64))),
    (ValueError, dict(input_pos=torch.zeros(2, 4, dtype=torch.int64))),
    (RuntimeError, {}),  # CPU tensors
])
def test_qkv_norm_rope_refuses(err, over):
    with pytest.raises(err):
        ops.qkv_norm_rope(**_rope(**over))


def _cache(P=6, G=2, S=16, D=64, B=2, N=3, dt=BF):
    return ops.KVCachePaged(torch.zeros(P, G, S, D, dtype=dt), torch.zeros(P, G, S, D, dtype=dt),
                            torch.zeros(B, N, dtype=torch.int32))


BAD_CACHES = [
    (ValueError, _cache()._replace(v=torch.zeros(6, 2, 16, 32, dtype=BF))),
    (ValueError, _cache()._replace(v=torch.zeros(6, 2, 16, 64, dtype=FP))),
    (ValueError, _cache()._replace(k=torch.zeros(6, 16, 2, 64, dtype=BF).transpose(1, 2))),
    (ValueError, _cache()._replace(k=torch.zeros(0, 2, 16, 64, dtype=BF), v=torch.zeros(0, 2, 16, 64, dtype=BF))),
    (NotImplementedError, _cache(S=8)),
    (NotImplementedError, _cache(S=24)),
    (ValueError, _cache()._replace(table=torch.zeros(2, 3, dtype=torch.int64))),
    (ValueError, _cache()._replace(table=torch.zeros(2, 0, dtype=torch.int32))),
    (ValueError, _cache()._replace(table=torch.zeros(6, dtype=torch.int32))),
    (ValueError, _cache()._replace(table=torch.zeros(3, 2, dtype=torch.int32).T)),
]


def _append(cache=None, **over):
    a = _rope(**{k: v for k, v in over.items() if k not in ("input_pos", "lengths")})
    a.pop("n_query_groups")
    a.update(cache=cache or _cache(), input_pos=torch.zeros(2, dtype=torch.int64))
    a.update({k: v for k, v in over.items() if k in ("input_pos", "lengths")})
    return a


@pytest.mark.parametrize("err,cache", BAD_CACHES)
def test_bad_caches_are_refused(err, cache):
    with pytest.raises(err):
        ops.kv_cache_paged_append(**_append(cache))
    with pytest.raises(err):
        ops.attention_paged(torch.zeros(2, 1, 4, 64, dtype=BF), cache, torch.zeros(1, dtype=torch.int64))


@pytest.mark.parametrize("err,over", [
    (ValueError, dict(B=3)),
    (ValueError, dict(D=128)),
    (ValueError, dict(dt=FP, wdt=FP)),
    (ValueError, dict(H=6, G=2, n_head=4)),
    (ValueError, dict(input_pos=None)),
    (RuntimeError, dict(input_pos=torch.zeros(3, dtype=torch.int64))),  # refused as a CPU tensor first
    (ValueError, dict(lengths=torch.zeros(3, dtype=torch.int64))),
    (ValueError, dict(lengths=torch.zeros(2))),
    (ValueError, dict(k_weight=None)),
    (RuntimeError, {}),
])
def test_append_refuses(err, over):
    with pytest.raises(err):
        ops.kv_cache_paged_append(**_append(**over))


def _q(B=2, T=1, H=4, D=64, dt=BF):
    return torch.zeros(B, T, H, D, dtype=dt)


@pytest.mark.parametrize("err,args,kw", [
    (ValueError, (_q()[0], _cache()), {}),
    (ValueError, (_q(B=3), _cache()), {}),
    (ValueError, (_q(D=128), _cache()), {}),
    (ValueError, (_q(H=3), _cache()), {}),
    (ValueError, (_q(dt=FP), _cache()), {}),
    (NotImplementedError, (_q(dt=F32), _cache(dt=F32)), {}),
    (NotImplementedError, (_q(D=96), _cache(D=96)), {}),
    (NotImplementedError, (_q(), _cache()), dict(scale=0.0)),
    (NotImplementedError, (_q(), _cache()), dict(scale=float("inf"))),
    (ValueError, (_q(), _cache()), dict(input_pos=None)),
    (ValueError, (_q(), _cache()), dict(lengths=torch.zeros(2))),
    (RuntimeError, (_q(), _cache()), {}),
])
def test_attention_paged_refuses(err, args, kw):
    with pytest.raises(err):
        ops.attention_paged(*args, **{"input_pos": torch.zeros(1, dtype=torch.int64), **kw})


@pytest.mark.parametrize("what", ["qkv", "q_weight", "k_weight", "k", "v"])
@pytest.mark.parametrize("how", ["gradient", "tangent"])
def test_append_refuses_derivatives(what, how):
    """Instead of passing for constant; the check of devices, which CPU tensors do not pass, comes after it."""
    def call(mark):
        a = _append()
        a["cache"] = a["cache"]._replace(**{what: mark(getattr(a["cache"], what))}) if what in "kv" else a["cache"]
        a.update({} if what in "kv" else {what: mark(a[what])})
        return ops.kv_cache_paged_append(**a)
    _derivative(call, how)


@pytest.mark.parametrize("what", ["q", "k", "v"])
@pytest.mark.parametrize("how", ["gradient", "tangent"])
def test_attention_paged_refuses_derivatives(what, how):
    def call(mark):
        q, cache = _q(), _cache()
        if what == "q":
            q = mark(q)
        else:
            cache = cache._replace(**{what: mark(getattr(cache, what))})
        return ops.attention_paged(q, cache, torch.zeros(1, dtype=torch.int64))
    _derivative(call, how)


def _derivative(call, how):
    if how == "gradient":
        with pytest.raises(NotImplementedError):
            call(lambda x: x.requires_grad_(True))
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
            call(lambda x: x.requires_grad_(True))
    else:
        with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
            call(lambda x: torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


def test_tangents_of_rotation_tables_are_refused():
    with torch.autograd.forward_ad.dual_level():
        cos = torch.autograd.forward_ad.make_dual(torch.zeros(9, 32), torch.ones(9, 32))
        with pytest.raises(ValueError):
            ops.qkv_norm_rope(**_rope(cos=cos))


def test_paged_cache_constructor():
    c = ops.kv_cache_paged(3, 2, 100, 64, page_size=32)
    assert c.k.shape == (12, 2, 32, 64) and c.table.shape == (3, 4) and c.table.unique().numel() == 12
    c = ops.kv_cache_paged(3, 2, 100, 64, page_size=32, pages=5)
    assert c.k.shape == (5, 2, 32, 64) and (c.table == -1).all()
    with pytest.raises(NotImplementedError):
        ops.kv_cache_paged(1, 1, 10, 64, page_size=8)


@pytest.mark.parametrize("err,over", [
    (ValueError, dict(logits=torch.zeros(()))),
    (ValueError, dict(logits=torch.zeros(3, 0))),
    (NotImplementedError, dict(logits=torch.zeros(1, 1).expand(3, (1 << 20) + 1))),
    (NotImplementedError, dict(logits=torch.zeros(3, 4, dtype=torch.float64))),
    (ValueError, dict(uniforms=torch.zeros(4))),
    (ValueError, dict(uniforms=torch.zeros(3, dtype=torch.float64))),
    (ValueError, dict(temperature=-0.1)),
    (ValueError, dict(temperature=float("nan"))),
    (ValueError, dict(temperature=float("inf"))),
    (ValueError, dict(top_k=-1)),
    (ValueError, dict(top_k=1.5)),
    (ValueError, dict(top_p=0.0)),
    (ValueError, dict(top_p=1.1)),
    (ValueError, dict(top_p=float("nan"))),
    (ValueError, dict(min_p=-0.1)),
    (ValueError, dict(min_p=1.1)),
    (RuntimeError, {}),
])
def test_sample_tokens_refuses(err, over):
    a = dict(logits=torch.zeros(3, 4), uniforms=torch.zeros(3))
    a.update(over)
    with pytest.raises(err):
        ops.sample_tokens(**a)


# ---- the C entry points; pointers are never dereferenced: every call is refused (or empty) before a launch ----

@pytest.fixture(scope="module")
def lib():
    return nat.load()


def _append_call(lib, **over):
    a = dict(qkv=4096, sb=512, st=512, dt=nat.DTYPE_BF16, wq=4096, wk=4096, wdt=nat.DTYPE_BF16, cos=4096, sin=4096, pairs=32,
             rows=9, pos=4096, ps=1, lengths=None, q=4096, k=4096, v=4096, pages=6, S=16, table=4096, ts=3, N=3, B=2, T=1,
             G=2, R=2, D=64)
    a.update(over)
    return lib.gdn2_kv_cache_paged_append(
        a["qkv"], a["sb"], a["st"], a["dt"], a["wq"], a["wk"], a["wdt"], 1e-5, a["cos"], a["sin"], a["pairs"], a["rows"],
        a["pos"], a["ps"], a["lengths"], a["q"], a["k"], a["v"], a["pages"], a["S"], a["table"], a["ts"], a["N"], a["B"],
        a["T"], a["G"], a["R"], a["D"], None)


def _paged_call(lib, **over):
    a = dict(q=4096, strides=(256, 256, 64), dt=nat.DTYPE_BF16, k=4096, v=4096, pages=6, S=16, table=4096, ts=3, N=3,
             pos=4096, ps=1, lengths=None, out=4096, B=2, T=1, G=2, R=2, D=64, scale=1.0, ws=None, nbytes=0)
    a.update(over)
    st = (ctypes.c_int64 * 3)(*a["strides"]) if a["strides"] else None
    return lib.gdn2_attn_paged(
        a["q"], st and ctypes.addressof(st), a["dt"], a["k"], a["v"], a["pages"], a["S"], a["table"], a["ts"], a["N"],
        a["pos"], a["ps"], a["lengths"], a["out"], a["B"], a["T"], a["G"], a["R"], a["D"], a["scale"], a["ws"],
        a["nbytes"], None)


PAGED_CACHE = [
    (nat.ERR_INVALID, dict(pages=0)),
    (nat.ERR_INVALID, dict(S=0)),
    (nat.ERR_UNSUPPORTED, dict(S=24)),
    (nat.ERR_INVALID, dict(N=0)),
    (nat.ERR_INVALID, dict(ts=-1)),
    (nat.ERR_INVALID, dict(k=None)),
    (nat.ERR_INVALID, dict(v=4104)),
    (nat.ERR_INVALID, dict(table=None)),
    (nat.ERR_INVALID, dict(table=4098)),
    (nat.ERR_UNSUPPORTED, dict(S=1 << 20, N=1 << 11)),        # positions in 31 bits
    (nat.ERR_UNSUPPORTED, dict(pages=1 << 30, G=2, S=16)),    # rows in 32 bits
    (nat.ERR_INVALID, dict(B=-1)),
    (nat.ERR_INVALID, dict(G=0)),
    (nat.ERR_INVALID, dict(dt=7)),
    (nat.ERR_INVALID, dict(pos=None)),
    (nat.ERR_INVALID, dict(ps=-1)),
    (nat.OK, dict(B=0)),
    (nat.OK, dict(T=0)),
]


@pytest.mark.parametrize("want,over", PAGED_CACHE + [
    (nat.ERR_INVALID, dict(q=None)),
    (nat.ERR_INVALID, dict(q=4104)),
    (nat.ERR_INVALID, dict(qkv=4104)),
    (nat.ERR_INVALID, dict(sb=516)),
    (nat.ERR_INVALID, dict(wk=None)),
    (nat.ERR_INVALID, dict(wdt=nat.DTYPE_F16)),
    (nat.ERR_INVALID, dict(pairs=33)),
    (nat.ERR_INVALID, dict(cos=None)),
    (nat.ERR_INVALID, dict(rows=1 << 31)),
    (nat.ERR_UNSUPPORTED, dict(D=12)),
    (nat.ERR_UNSUPPORTED, dict(D=264)),
    (nat.ERR_UNSUPPORTED, dict(G=20000)),
    (nat.ERR_UNSUPPORTED, dict(B=1 << 20, T=1 << 20)),
])
def test_append_entry(lib, want, over):
    assert _append_call(lib, **over) == want


@pytest.mark.parametrize("want,over", PAGED_CACHE + [
    (nat.ERR_INVALID, dict(strides=None)),
    (nat.ERR_INVALID, dict(strides=(256, 256, 60))),
    (nat.ERR_INVALID, dict(strides=(-256, 256, 64))),
    (nat.ERR_INVALID, dict(out=None)),
    (nat.ERR_INVALID, dict(out=4104)),
    (nat.ERR_INVALID, dict(R=0)),
    (nat.ERR_UNSUPPORTED, dict(dt=nat.DTYPE_F32)),
    (nat.ERR_UNSUPPORTED, dict(D=96)),
    (nat.ERR_UNSUPPORTED, dict(scale=0.0)),
    (nat.ERR_UNSUPPORTED, dict(T=1 << 30, R=4)),
    (nat.ERR_WORKSPACE, dict(N=2000)),                         # shares of the keys need one
    (nat.ERR_WORKSPACE, dict(N=2000, ws=4104, nbytes=1 << 30)),
    (nat.ERR_WORKSPACE, dict(N=2000, ws=4096, nbytes=64)),
])
def test_attn_paged_entry(lib, want, over):
    assert _paged_call(lib, **over) == want


@pytest.mark.parametrize("fits,over", [
    (True, dict(B=32, T=16384, G=8, R=4, D=128)),             # more rows than HIP's workgroups, in tiles of 128
    (True, dict(B=32, T=65535 * 128, G=8, R=1)),
    (False, dict(B=32, T=65536 * 128, G=8, R=1)),
    (True, dict(B=(1 << 24) - 1, T=1, G=1, R=32)),            # few rows: a workgroup for each group
    (False, dict(B=1 << 24, T=1, G=1, R=32)),
    (True, dict(B=1, T=(1 << 30) // 4, G=1, R=4)),
    (False, dict(B=1, T=(1 << 30) // 4 + 1, G=1, R=4)),
])
def test_attn_paged_sizes(lib, fits, over):
    """What is launched decides, not the rows; a call that fits goes on to its missing queries."""
    assert _paged_call(lib, q=None, **over) == (nat.ERR_INVALID if fits else nat.ERR_UNSUPPORTED)


@pytest.mark.parametrize("runs,B,G,L", [
    (True, 2, 8, 32768),
    (False, 2, 8, 1024),
    (True, 100, 1, 1 << 30),
    (True, 1, 600, 1 << 30),
    (False, 2, 2000, 1 << 30),   # one run over both sequences would end at 2^31
    (False, 7, 512, 1 << 30),
    (False, 4000, 1, 1 << 30),
])
def test_attn_paged_runs_end_within_31_bits(lib, runs, B, G, L):
    """One token over the longest contexts: a run of several sequences' positions is counted from its first sequence's."""
    assert (lib.gdn2_attn_paged_workspace_size(B, 1, G, 1, 64, L) > 0) == runs


@pytest.mark.parametrize("want,over", [
    (nat.ERR_INVALID, dict(dt=5)),
    (nat.ERR_INVALID, dict(rows=-1)),
    (nat.ERR_INVALID, dict(n=0)),
    (nat.ERR_INVALID, dict(inner=0)),
    (nat.ERR_UNSUPPORTED, dict(n=(1 << 20) + 1)),
    (nat.ERR_INVALID, dict(t=-1.0)),
    (nat.ERR_INVALID, dict(t=float("nan"))),
    (nat.ERR_INVALID, dict(p=0.0)),
    (nat.ERR_INVALID, dict(p=1.5)),
    (nat.ERR_INVALID, dict(m=-0.5)),
    (nat.ERR_INVALID, dict(k=-1)),
    (nat.ERR_INVALID, dict(x=None)),
    (nat.ERR_INVALID, dict(x=4097)),
    (nat.ERR_INVALID, dict(u=None)),
    (nat.ERR_INVALID, dict(out=None)),
    (nat.ERR_WORKSPACE, dict(ws=None)),
    (nat.ERR_WORKSPACE, dict(ws=4104)),
    (nat.ERR_WORKSPACE, dict(nbytes=100)),
    (nat.ERR_UNSUPPORTED, dict(rows=1 << 32)),
    (nat.ERR_UNSUPPORTED, dict(rows=1 << 22)),
    (nat.ERR_WORKSPACE, dict(rows=(1 << 22) - 1, ws=None)),
    (nat.ERR_WORKSPACE, dict(rows=300000, n=1 << 20, ws=None)),
    (nat.OK, dict(rows=0)),
])
def test_sample_entry(lib, want, over):
    a = dict(x=4096, inner=3, so=0, sr=50, dt=nat.DTYPE_BF16, rows=3, n=50, u=4096, t=1.0, k=0, p=1.0, m=0.0, out=4096, ws=4096,
             nbytes=1 << 40)
    a.update(over)
    assert lib.gdn2_sample_tokens(a["x"], a["inner"], a["so"], a["sr"], a["dt"], a["rows"], a["n"], a["u"], None, a["t"], None,
                                  a["k"], None, a["p"], None, a["m"], a["out"], a["ws"], a["nbytes"], None) == want


@pytest.mark.parametrize("want,over", [
    (nat.ERR_INVALID, dict(dq=None)),
    (nat.ERR_INVALID, dict(dv=4104)),
    (nat.ERR_INVALID, dict(dqkv=None)),
    (nat.ERR_INVALID, dict(dwq=None)),
    (nat.ERR_WORKSPACE, dict(ws=None)),
    (nat.ERR_WORKSPACE, dict(nbytes=16)),
    (nat.OK, dict(T=0)),
])
def test_rope_backward_entry(lib, want, over):
    a = dict(dq=4096, dk=4096, dv=4096, dqkv=4096, dwq=4096, dwk=4096, ws=4096, nbytes=1 << 30, T=3)
    a.update(over)
    assert lib.gdn2_qkv_norm_rope_bwd(4096, 512, 512, nat.DTYPE_BF16, 4096, 4096, nat.DTYPE_BF16, 1e-5, 4096, 4096, 32, 9,
                                      None, 0, 0, a["dq"], a["dk"], a["dv"], a["dqkv"], a["dwq"], a["dwk"], 2, a["T"], 2, 2,
                                      64, a["ws"], a["nbytes"], None) == want


# ---- the decoder host ----

def test_hybrid_qk_norm_parameters():
    from qwendopamine_amd.hybrid import HybridConfig, HybridDecoder, count_parameters

    cfg = HybridConfig(n_layer=2, n_embd=64, n_head=2, head_size=32, n_query_groups=1, intermediate_size=64, vocab_size=50,
                       gdn2_layers=[], qk_norm=True)
    m = HybridDecoder(cfg)
    assert sum(p.numel() for p in m.parameters()) == count_parameters(cfg)
    assert {n.split(".", 2)[2] for n, _ in m.named_parameters() if "attn.q_norm" in n or "attn.k_norm" in n} == {
        "attn.q_norm.weight", "attn.k_norm.weight"}
    idx = torch.randint(0, 50, (2, 9), generator=torch.Generator().manual_seed(0))
    scaled = HybridDecoder(cfg)
    scaled.load_state_dict(m.state_dict())
    with torch.no_grad():
        for blk in scaled.h:  # normalised: the scale of queries and keys does not matter
            at = blk.attn
            rows = at.attn.weight.view(at.n_query_groups, at.n_head // at.n_query_groups + 2, at.head_size, -1)
            rows[:, :-1] *= 8.0
        assert torch.allclose(m(idx), scaled(idx), rtol=1e-3, atol=1e-3)


def test_hybrid_paged_needs_the_gpu():
    from qwendopamine_amd.hybrid import HybridConfig, HybridDecoder

    m = HybridDecoder(HybridConfig(n_layer=1, n_embd=64, n_head=1, head_size=64, n_query_groups=1, intermediate_size=64,
                                   vocab_size=50, gdn2_layers=[]))
    with pytest.raises(NotImplementedError):
        m.setup_caches(1, 32, page_size=16)
    with pytest.raises(NotImplementedError):
        m.setup_caches(1, 32, kv_bits=4, page_size=16)


def _cpu_decoder(monkeypatch, gdn2_layers):
    """A decoder of two layers whose caches are set up as on the GPU and whose blocks pass their input on."""
    from qwendopamine_amd import hybrid

    m = hybrid.HybridDecoder(hybrid.HybridConfig(
        n_layer=2, n_embd=64, n_head=1, head_size=64, n_query_groups=1, intermediate_size=64, vocab_size=50, block_size=32,
        gdn2_layers=gdn2_layers)).to(BF)
    monkeypatch.setattr(ops, "attention_paged_supported", lambda q, head_dim: True)
    monkeypatch.setattr(hybrid.Block, "forward", lambda self, x, *args: x)
    return m


def test_hybrid_pages_without_attention_layers(monkeypatch):
    """No layer reads the mask, yet its rows are selected: they have to be there."""
    m = _cpu_decoder(monkeypatch, [0, 1])
    idx = torch.arange(5)[None]
    for page_size in (None, 16):
        m.setup_caches(1, 20, page_size=page_size)
        assert m(idx, input_pos=torch.arange(5)).shape == (1, 5, 50)
        assert m(idx, input_pos=torch.arange(15, 20)).shape == (1, 5, 50)


def test_hybrid_refused_pages_leave_the_caches(monkeypatch):
    m = _cpu_decoder(monkeypatch, [0])
    m.setup_caches(1, 20)
    before = m.mask_cache, m.max_seq_length, m.h[1].attn.kv_cache
    m.h[0].gdn2_cache = state = {}
    for page_size in (8, 24, 0, -16):
        with pytest.raises(NotImplementedError):
            m.setup_caches(2, 40, page_size=page_size)
    assert (m.mask_cache, m.max_seq_length, m.h[1].attn.kv_cache) == before and m.h[0].gdn2_cache is state


def test_hybrid_prompt_longer_than_its_pages():
    """Refused, as over the other caches: its last tokens would have no place and count as padding."""
    from qwendopamine_amd.hybrid import CausalSelfAttention, HybridConfig

    at = CausalSelfAttention(HybridConfig(n_layer=1, n_embd=64, n_head=1, head_size=64, n_query_groups=1, vocab_size=50), 0)
    at.kv_cache = ops.kv_cache_paged(1, 1, 40, 64, page_size=16)
    cos, sin = torch.zeros(64, 32), torch.zeros(64, 32)
    for t, err in ((49, ValueError), (48, NotImplementedError)):  # (48 fit, and need the GPU)
        with torch.no_grad(), pytest.raises(err):
            at.forward_qkv(torch.zeros(1, t, 192), cos, sin, torch.arange(t))
