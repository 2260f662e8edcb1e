"""``ops.token_logprobs`` and its gradient against float64: types, row lengths and alignments,
alternatives with ties, ignored and unknown targets, rows with infinities and NaN, layouts, graphs.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _ref(x, t, dlogp, dent, ignore=-100):
    """float64: logp, entropy, dlogits, and (sorted) values and indices by (value, lower index)."""
    x = x.detach().cpu().double()
    t = t.cpu()
    V = x.shape[-1]
    lse = torch.logsumexp(x, -1, keepdim=True)
    lp = x - lse
    p = lp.exp()
    plp = torch.where(p == 0, 0.0, p * lp)
    h = -plp.sum(-1)
    known = (t >= 0) & (t < V) & (t != ignore)
    one = torch.nn.functional.one_hot(t.clamp(0, V - 1), V).double() * known[..., None]
    logp = torch.where(known, (one * torch.where(one > 0, lp, 0.0)).sum(-1), torch.where(t == ignore, 0.0, float("nan")))
    gl = torch.where(known, dlogp.cpu().double(), 0.0)[..., None]
    ge = dent.cpu().double()[..., None]
    d = one * gl - torch.where(p == 0, 0.0, p * (gl + ge * (lp + h[..., None])))
    return logp, h, d, lp


def _order(x):
    """Indices by (value descending, NaN first, lower index)."""
    x = x.detach().cpu().double()
    key = torch.where(torch.isnan(x), torch.inf, x)
    nan_first = torch.isnan(x).double()
    i = torch.argsort(key, dim=-1, descending=True, stable=True)
    j = torch.argsort(nan_first.gather(-1, i), dim=-1, descending=True, stable=True)
    return i.gather(-1, j)


def _run(x, t, top_k=0, dlogp=None, dent=None, **kw):
    from qwendopamine_amd import ops

    r = ops.token_logprobs(x, t, top_k=top_k, **kw)
    outs = [o for o, g in ((r.logprobs, dlogp), (r.entropy, dent)) if g is not None]
    (dx,) = torch.autograd.grad(outs, x, [g for g in (dlogp, dent) if g is not None]) if outs else (None,)
    torch.cuda.synchronize()
    return r, dx


def _check(x, t, r, dx, dlogp, dent, ignore=-100):
    """Float32 results: the sum of V exponentials loses at most about V / 64 roundings of a lane's
    running sum and its exponent error 2^-23 |x - m| each; 2e-6 (1 + |lse|) covers both at these
    sizes.  The gradient is rounded once to its type (half a step) after float32 terms."""
    logp, h, d, lp = _ref(x, t, dlogp, dent, ignore)
    scale = 1 + torch.logsumexp(x.detach().cpu().double(), -1).abs()
    assert ((r.logprobs.cpu().double() - logp).abs() <= 2e-6 * scale).logical_or(logp.isnan() & r.logprobs.cpu().isnan()).all()
    assert ((r.entropy.cpu().double() - h).abs() <= 4e-6 * (scale + h)).all()
    if r.top_ids is not None:
        ids = _order(x)[..., : r.top_ids.shape[-1]]
        assert torch.equal(r.top_ids.cpu(), ids)
        have, want = r.top_logprobs.cpu().double(), lp.gather(-1, ids)
        assert ((have == want) | ((have - want).abs() <= 2e-6 * scale[..., None])).all()  # -inf equals -inf
    if dx is not None:
        u = torch.finfo(x.dtype).eps / 2
        tiny = torch.finfo(x.dtype).smallest_normal * 2 * u
        gl = dlogp.cpu().double().abs()[..., None]
        ge = dent.cpu().double().abs()[..., None]
        p = lp.exp()
        terms = p * (gl + ge * (torch.where(p == 0, 0.0, lp.abs()) + h[..., None].abs()))
        bound = u * d.abs() + 4e-6 * scale[..., None] * (terms + 2 * p * ge) + 2 ** -22 * d.abs() + tiny + 2e-38
        e = (dx.cpu().double() - d).abs()
        assert (e <= bound).all(), f"gradient {float((e / bound).max()):.2f} times its bound"


def _case(dev, rows, V, dt, seed=0, spread=2.0, grad=True):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=gen) * spread).to(dt).to(dev).requires_grad_(grad)
    t = torch.randint(0, V, (rows,), generator=gen).to(dev)
    return x, t, torch.randn(rows, generator=gen).to(dev), torch.randn(rows, generator=gen).to(dev) * 0.1


@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("rows,V,top", [
    (1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 64, 32), (1, 513, 5), (4, 1000, 20), (3, 4096, 1), (2, 4097, 32),
    (7, 8191, 8), (2, 50257, 20), (600, 333, 4), (1, 151936, 20),
])
def test_logprobs_match_float64(gpu_device, rows, V, top, dt):
    print(f"[case] logprobs {rows}x{V} top {top} {dt}", flush=True)
    x, t, gl, ge = _case(gpu_device, rows, V, dt, seed=V + rows)
    if rows > 2:
        t[1] = -100
    r, dx = _run(x, t, top, gl, ge)
    _check(x, t, r, dx, gl, ge)


def test_logprobs_without_alternatives_are_the_same(gpu_device):
    x, t, gl, ge = _case(gpu_device, 9, 3001, BF)
    a, da = _run(x, t, 5, gl, ge)
    b, db = _run(x, t, 0, gl, ge)
    assert torch.equal(a.logprobs, b.logprobs) and torch.equal(a.entropy, b.entropy) and torch.equal(da, db)
    assert b.top_ids is None and b.top_logprobs is None


@pytest.mark.parametrize("dt", [BF, F32])
def test_alternatives_with_ties(gpu_device, dt):
    """Equal logits go by the lower index: a constant row, few distinct values, signed zeros, a
    falling and a rising row, -inf almost everywhere, the ragged ends of a row."""
    V = 20011
    gen = torch.Generator().manual_seed(3)
    rows = [torch.zeros(V), torch.randint(-2, 3, (V,), generator=gen).float(),
            torch.where(torch.rand(V, generator=gen) < 0.5, 0.0, -0.0), -torch.arange(V).float(), torch.arange(V).float(),
            torch.full((V,), float("-inf")), torch.full((V,), -3.0), torch.full((V,), torch.finfo(dt).min)]
    rows[5][torch.tensor([7, 9000, V - 1])] = torch.tensor([1.0, 2.0, 1.0])
    rows[6][V - 3:] = 5.0
    rows[6][:2] = 5.0
    x = torch.stack(rows).to(dt).to(gpu_device)
    t = torch.zeros(len(rows), dtype=torch.int64, device=gpu_device)
    for lo in (0, 1, 3):  # other alignments of a row's start
        y = x[:, lo:]
        r, _ = _run(y, t, 20)
        assert torch.equal(r.top_ids.cpu(), _order(y)[:, :20]), lo


@pytest.mark.parametrize("dt", [BF, FP, F32])
def test_logprobs_nonfinite_rows(gpu_device, dt):
    V = 5000
    x, t, gl, ge = _case(gpu_device, 6, V, dt, seed=8)
    with torch.no_grad():
        x[0, 123] = float("nan")
        x[1, 4999] = float("inf")
        x[2] = float("-inf")
        x[3, :2500] = float("-inf")
        x[4, 1:] = float("-inf")
        t[3], t[4] = 10, 0
    r, dx = _run(x, t, 3, gl, ge)
    assert r.logprobs[:3].isnan().all() and r.entropy[:3].isnan().all() and dx[0].isnan().any() and dx[1].isnan().any()
    assert r.top_ids[0, 0] == 123 and r.top_ids[1, 0] == 4999
    assert r.logprobs[3] == float("-inf") and r.logprobs[4] == 0 and abs(float(r.entropy[4].detach())) < 1e-6
    assert (dx[3, :10] == 0).all() and dx[3].isfinite().all() and (dx[4] == 0).all()
    keep = torch.tensor([4, 5], device=gpu_device)
    _check(x[keep], t[keep], type(r)(*(o[keep] for o in r)), dx[keep], gl[keep], ge[keep])


def test_logprobs_targets(gpu_device):
    """Ignored targets give 0 and no gradient; others out of range NaN; the choice of ignore_index."""
    x, t, gl, ge = _case(gpu_device, 5, 777, BF)
    t[:] = torch.tensor([-100, -1, 777, 776, 0])
    r, dx = _run(x, t, 0, gl, torch.zeros_like(ge))
    assert r.logprobs[0] == 0 and r.logprobs[1].isnan() and r.logprobs[2].isnan() and (dx[0] == 0).all()
    assert dx[1].isnan().any() and dx[2].isnan().any()
    r, dx = _run(x, t, 0, gl, ge, ignore_index=-1)
    assert r.logprobs[0].isnan() and r.logprobs[1] == 0
    keep = torch.tensor([1, 3, 4], device=gpu_device)
    _check(x[keep], t[keep], type(r)(r.logprobs[keep], r.entropy[keep], None, None), dx[keep], gl[keep], ge[keep], -1)
    with torch.no_grad():  # nothing of an ignored row without gradient is read
        x[0] = float("nan")
    r, dx = _run(x, t, 0, gl, torch.zeros_like(ge))
    assert (dx[0] == 0).all()


@pytest.mark.parametrize("V", [777, 40000])  # rows of one part, and of several
def test_logprobs_ignored_token_of_the_vocabulary(gpu_device, V):
    """``ignore_index`` may be a token, as a padding id is."""
    x, t, gl, ge = _case(gpu_device, 6, V, BF)
    t[:] = torch.tensor([0, 5, 0, V - 1, 1, 0])
    r, dx = _run(x, t, 3, gl, ge, ignore_index=0)
    assert (r.logprobs[t == 0] == 0).all() and (r.logprobs[t != 0] < 0).all()
    _check(x, t, r, dx, gl, ge, 0)
    _, dx = _run(x, t, 0, gl, ignore_index=0)
    assert (dx[t == 0] == 0).all() and (dx[t != 0] != 0).any(-1).all()


def test_logprobs_one_gradient_or_none(gpu_device):
    x, t, gl, ge = _case(gpu_device, 4, 999, F32)
    z = torch.zeros_like(gl)
    assert torch.equal(_run(x, t, 0, gl)[1], _run(x, t, 0, gl, z)[1])
    assert torch.equal(_run(x, t, 0, None, ge)[1], _run(x, t, 0, z, ge)[1])


@pytest.mark.parametrize("layout", ["shifted", "sliced", "vocab sliced", "expanded", "four axes", "channels strided", "one row"])
def test_logprobs_layouts(gpu_device, layout):
    B, T, V = 3, 6, 1003
    gen = torch.Generator().manual_seed(4)
    full = torch.randn(B, T, V + 5, generator=gen).to(BF).to(gpu_device)
    t = torch.randint(0, V, (B, T), generator=gen).to(gpu_device)
    gl, ge = torch.randn(B, T, generator=gen).to(gpu_device), torch.randn(B, T, generator=gen).to(gpu_device)
    if layout == "shifted":  # a model's logits against the next tokens
        x, t, gl, ge = full[:, :-1], t[:, 1:], gl[:, 1:], ge[:, 1:]
    elif layout == "sliced":
        x, t, gl, ge = full[:, ::2], t[:, ::2], gl[:, ::2], ge[:, ::2]
    elif layout == "vocab sliced":
        x = full[..., 3:V + 3]
    elif layout == "expanded":
        x = full[:, :1].expand(B, T, V + 5)
    elif layout == "four axes":
        x, t, gl, ge = full[None].expand(2, B, T, V + 5), t[None].expand(2, B, T), gl[None].expand(2, B, T), ge[None].expand(2, B, T)
    elif layout == "channels strided":
        x = full.transpose(0, 2).contiguous().transpose(0, 2)
    else:
        x, t, gl, ge = full[0, 0], t[0, 0], gl[0, 0], ge[0, 0]
    x = x.detach().requires_grad_(True)
    r, dx = _run(x, t, 4, gl, ge)
    assert r.logprobs.shape == t.shape and r.top_ids.shape == (*t.shape, 4) and dx.shape == x.shape
    _check(x, t, r, dx, gl, ge)


def test_logprobs_no_rows(gpu_device):
    x = torch.zeros(0, 10, device=gpu_device, requires_grad=True)
    r, dx = _run(x, torch.zeros(0, dtype=torch.int64, device=gpu_device), 2, torch.zeros(0, device=gpu_device))
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 2) and dx.shape == (0, 10)


def test_logprobs_gradient_against_differences(gpu_device):
    x, t, gl, ge = _case(gpu_device, 3, 50, F32, seed=2)
    _, dx = _run(x, t, 0, gl, ge)
    X = x.detach().cpu().double()

    def loss(X):
        lp = X.log_softmax(-1)
        return (lp.gather(1, t.cpu()[:, None])[:, 0] * gl.cpu().double()).sum() - ((lp.exp() * lp).sum(-1) * ge.cpu().double()).sum()

    gen = torch.Generator().manual_seed(6)
    d = torch.randn(X.shape, generator=gen, dtype=torch.float64)
    want = (loss(X + 1e-5 * d) - loss(X - 1e-5 * d)) / 2e-5
    have = (dx.cpu().double() * d).sum()
    assert abs(float(have - want)) <= 1e-6 * float((dx.cpu().double() * d).abs().sum()) + 1e-8


def test_logprobs_captured_and_repeated(gpu_device):
    """Captured forward and backward, replayed on new logits beside eager work: eager bits."""
    from qwendopamine_amd import ops

    x, t, gl, ge = _case(gpu_device, 4, 30011, BF, seed=1)
    _run(x, t, 20, gl, ge)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = ops.token_logprobs(x, t, top_k=20)
        (dx,) = torch.autograd.grad((r.logprobs, r.entropy), x, (gl, ge))
    for seed in (2, 3, 4):
        new = _case(gpu_device, 4, 30011, BF, seed=seed)
        with torch.no_grad():
            x.copy_(new[0])
            t.copy_(new[1])
        g.replay()
        want, dwant = _run(new[0], new[1], 20, gl, ge)
        assert all(torch.equal(a, b) for a, b in zip(r, want)) and torch.equal(dx, dwant)


@pytest.mark.parametrize("rows,V,top", [(2 ** 24 + 5, 4, 0), (2 ** 26 + 3, 2, 1)])
def test_logprobs_more_rows_than_a_launch(gpu_device, rows, V, top):
    """Past 2^24 rows the backward, past 2^26 the forward takes more than one launch.  Logits of 0, 1, 2
    and 3, so that float32 results of few values are known for all rows at once."""
    from qwendopamine_amd import ops

    print(f"[case] logprobs {rows}x{V}", flush=True)
    r = torch.arange(rows, device=gpu_device)
    hot = (r * 7 + r // 1000) % V
    x = torch.nn.functional.one_hot(hot, V).to(BF) * ((r % 4)[:, None]).to(BF)
    x.requires_grad_(True)
    t = (r // 3) % V
    out = ops.token_logprobs(x, t, top_k=top)
    gl = ((r % 5) - 2).float()
    (dx,) = torch.autograd.grad(out.logprobs, x, gl)
    for lo in range(0, rows, 2 ** 24):
        s = slice(lo, min(rows, lo + 2 ** 24))
        lp = x[s].detach().double().log_softmax(-1)
        one = torch.nn.functional.one_hot(t[s], V).double()
        want = (one - lp.exp()) * gl[s, None].double()
        assert float((out.logprobs[s].detach().double() - (lp * one).sum(-1)).abs().max()) <= 2e-6 * 5
        # Rounded once to bf16, whose half step is 2^-9 of a value's power of two.
        assert bool(((dx[s].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all())
        if top:
            first = torch.where((r[s] % 4) == 0, 0, hot[s])
            assert torch.equal(out.top_ids[s, 0], first)


@pytest.mark.parametrize("V", [777, 40000])
def test_logprobs_unknown_target_that_nothing_asks_for(gpu_device, V):
    """A target outside the vocabulary whose log probability is selected away (padding of -1): no
    gradient arrives at its row, and none passes; the entropy's still does."""
    from qwendopamine_amd import ops

    x, t, gl, ge = _case(gpu_device, 5, V, BF, seed=12)
    t[1], t[3] = -1, V
    wanted = (t >= 0) & (t < V)
    r = ops.token_logprobs(x, t)
    (dx,) = torch.autograd.grad((torch.where(wanted, r.logprobs, 0.0) * gl).sum(), x)
    want = _run(x, torch.where(wanted, t, -100), 0, torch.where(wanted, gl, 0.0))[1]
    assert torch.equal(dx, want) and not dx[~wanted].any() and dx[wanted].any(-1).all()
    z = torch.where(wanted, gl, 0.0)
    dx = _run(x, t, 0, z, ge)[1]
    assert torch.equal(dx, _run(x, torch.where(wanted, t, -100), 0, z, ge)[1]) and dx.isfinite().all()
