"""``ops.attention`` and its gradients against the float64 formulas, elementwise within bounds that
count the roundings (``tests/_attention_ref.py``): lengths from one token on, odd sizes, grouped
heads, causal offsets, padded and packed rows, strides, streams, graphs.
"""

from __future__ import annotations

import pytest
import torch

from tests._attention_ref import reference, worst

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _inputs(dev, B, Tq, Tk, H, G, D, dt, seed=0, mag=1.0, do_mag=1.0):
    gen = torch.Generator().manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=gen)

    q, k, v = ((randn(B, T, h, D) * mag).to(dt).to(dev).requires_grad_(True)
               for T, h in ((Tq, H), (Tk, G), (Tk, G)))
    return q, k, v, (randn(B, Tq, H, D) * do_mag).to(dt).to(dev)


def _run(q, k, v, do, **kw):
    from qwendopamine_amd import ops

    o = ops.attention(q, k, v, **kw)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    torch.cuda.synchronize()
    assert o.dtype == q.dtype and o.shape == q.shape and dk.shape == k.shape
    return dict(o=o, dq=dq, dk=dk, dv=dv)


def _check(got, q, k, v, do, scale=None, causal=True, kv_lengths=None, cu=None):
    val, bnd = reference(q, k, v, do, q.shape[-1] ** -0.5 if scale is None else scale, causal, kv_lengths, cu)
    w = worst(got, val, bnd)
    print("  error / bound " + " ".join(f"{n}={x:.2f}" for n, x in w.items()), flush=True)
    for n, x in w.items():
        if x > 1.0:
            d = (got[n].detach().cpu().double() - val[n]).abs()
            i = (d / bnd[n]).argmax()
            print(f"  {n}: value {val[n].flatten()[i]:.3e}, off {d.flatten()[i]:.3e}, bound {bnd[n].flatten()[i]:.3e}")
    assert all(x <= 1.0 for x in w.values()), w


@pytest.mark.parametrize("B,Tq,Tk,H,G,D,dt,causal", [
    (1, 1, 1, 1, 1, 64, BF, True),
    (1, 1, 1, 4, 2, 128, FP, False),
    (2, 33, 33, 4, 4, 64, BF, True),
    (1, 64, 64, 2, 1, 128, BF, True),
    (1, 65, 65, 2, 2, 128, FP, True),
    (2, 31, 97, 4, 2, 64, FP, True),       # the queries are the last 31 positions
    (1, 1, 300, 8, 1, 128, BF, True),      # a single token over a context
    (1, 130, 70, 4, 2, 64, BF, True),      # 60 queries see nothing
    (1, 257, 257, 3, 3, 64, FP, False),
    (2, 300, 511, 8, 2, 128, BF, False),
    (1, 1023, 1023, 4, 1, 64, BF, True),
    (1, 777, 1200, 6, 3, 128, FP, True),
    (1, 1, 2100, 4, 2, 64, FP, True),      # few queries over many keys: the keys are shared out
    (2, 5, 1500, 8, 2, 128, BF, True),
    (1, 150, 1111, 2, 1, 64, BF, False),
])
def test_attention_matches_float64(gpu_device, B, Tq, Tk, H, G, D, dt, causal):
    print(f"[case] attention B{B} Tq{Tq} Tk{Tk} H{H} G{G} D{D} {dt} causal={causal}", flush=True)
    x = _inputs(gpu_device, B, Tq, Tk, H, G, D, dt, seed=Tq + Tk)
    _check(_run(*x, causal=causal), *x, causal=causal)


@pytest.mark.parametrize("scale", [0.01, 1.0])
def test_attention_scale(gpu_device, scale):
    x = _inputs(gpu_device, 1, 100, 100, 2, 2, 64, BF, seed=3)
    _check(_run(*x, scale=scale), *x, scale=scale)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dt,D", [(BF, 128), (FP, 64)])
def test_attention_padded_rows(gpu_device, dt, D, causal):
    """Lengths from none to all; the padding holds NaN and infinities, which nothing may read."""
    lens = [0, 1, 63, 64, 65, 140]
    print(f"[case] attention padded {dt} D{D} causal={causal}", flush=True)
    q, k, v, do = _inputs(gpu_device, len(lens), 140, 140, 4, 2, D, dt, seed=5)
    with torch.no_grad():
        for b, n in enumerate(lens):
            k[b, n:], v[b, n:] = float("nan"), float("inf")
    for it in (torch.int64, torch.int32):
        kv = torch.tensor(lens, device=gpu_device, dtype=it)
        got = _run(q, k, v, do, causal=causal, kv_lengths=kv)
        _check(got, q, k, v, do, causal=causal, kv_lengths=lens)
    assert (got["o"][0] == 0).all() and (got["dq"][0] == 0).all() and (got["dk"][0] == 0).all()


@pytest.mark.parametrize("D,dt", [(64, FP), (128, BF), (128, FP)])
@pytest.mark.parametrize("rows", ["whole", "padded", "packed"])
def test_attention_shares_of_many_heads(gpu_device, rows, D, dt):
    """Eight query heads per group over few key tiles: dK and dV are summed in shares."""
    print(f"[case] attention shares {rows} {dt} D{D}", flush=True)
    T = 400
    x = _inputs(gpu_device, 2 if rows == "padded" else 1, T, T, 8, 1, D, dt, seed=17)
    if rows == "padded":
        _check(_run(*x, causal=False, kv_lengths=torch.tensor([130, 400], device=gpu_device)), *x, causal=False,
               kv_lengths=[130, 400])
    elif rows == "packed":
        cu = [0, 3, 70, 71, 400]
        _check(_run(*x, cu_seqlens=torch.tensor(cu)), *x, cu=cu)
    else:
        _check(_run(*x), *x)


def test_attention_lengths_are_clamped(gpu_device):
    x = _inputs(gpu_device, 2, 50, 50, 2, 2, 64, BF, seed=6)
    a = _run(*x, causal=False, kv_lengths=torch.tensor([-7, 10 ** 12], device=gpu_device))
    b = _run(*x, causal=False, kv_lengths=torch.tensor([0, 50], device=gpu_device))
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("cu", [[0, 1, 1, 66, 130, 131, 400], [0, 0, 257], [0, 64, 128, 192]])
def test_attention_packed(gpu_device, cu, causal):
    print(f"[case] attention packed {cu} causal={causal}", flush=True)
    T = cu[-1]
    x = _inputs(gpu_device, 1, T, T, 4, 2, 64, BF, seed=T)
    got = _run(*x, causal=causal, cu_seqlens=torch.tensor(cu))
    _check(got, *x, causal=causal, cu=cu)
    on_device = _run(*x, causal=causal, cu_seqlens=torch.tensor(cu, device=gpu_device, dtype=torch.int32))
    assert all(torch.equal(got[n], on_device[n]) for n in got)


@pytest.mark.parametrize("n,longest", [(70, 1500), (256, 300), (256, 2000), (257, 2000), (4200, 2600)])
def test_attention_many_packed_sequences(gpu_device, n, longest):
    """Empty, single-token and short sequences around one long one: each tile is found once."""
    print(f"[case] attention {n} packed sequences", flush=True)
    lens = [(i * 7) % 3 if n > 1000 else (i * i * 13) % 140 if i % 4 else 0 for i in range(n)]
    lens[n // 2] = longest
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    x = _inputs(gpu_device, 1, cu[-1], cu[-1], 2, 1, 64, BF, seed=n)
    _check(_run(*x, cu_seqlens=torch.tensor(cu)), *x, cu=cu)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("T,packed", [(2, False), (5, False), (64, False), (128, False), (128, True)])
def test_attention_short_sequences_are_as_exact_as_their_rounding(gpu_device, T, packed, dt):
    """Up to 128 tokens P and dS are multiplied in two parts: 2 x 8 (bf16) significant bits leave
    2^-17 of a term, against the 2^-9 of the result's rounding, whose root mean square is thus
    all but the whole error; 1.05 leaves room for results that round the other way."""
    print(f"[case] attention short T{T} packed={packed} {dt}", flush=True)
    n = 3
    shape = (1, n * T) if packed else (n, T)
    x = _inputs(gpu_device, shape[0], shape[1], shape[1], 4, 2, 64, dt, seed=T)
    cu = [T * i for i in range(n + 1)] if packed else None
    got = _run(*x, **(dict(cu_seqlens=torch.tensor(cu)) if packed else {}))
    for name, e in reference(*x, 0.125, True, cu=cu)[0].items():
        off, rounding = (got[name].detach().double().cpu() - e).norm(), (e.to(dt).double() - e).norm()
        assert off <= 1.05 * rounding, (name, float(off / rounding))


@pytest.mark.parametrize("lens,H,G", [
    ([(7 * i) % 60 + 1 for i in range(700)] + [140], 6, 3),          # groups not a multiple of the eight XCDs
    ([(5 * i) % 20 for i in range(600)] + [2000], 8, 8),             # and tiles looked up
])
def test_attention_many_rounds_of_packed_sequences(gpu_device, lens, H, G):
    """Over 4096 workgroups: groups are dealt out, the last deal short."""
    print(f"[case] attention {len(lens)} packed sequences, H{H} G{G}", flush=True)
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    x = _inputs(gpu_device, 1, cu[-1], cu[-1], H, G, 64, BF, seed=H)
    _check(_run(*x, cu_seqlens=torch.tensor(cu)), *x, cu=cu)


@pytest.mark.parametrize("B,Tq,Tk,H,G,D,causal", [
    (130, 33, 33, 32, 32, 64, True),     # many rounds
    (70, 20, 50, 120, 60, 64, False),    # more keys than queries
    (3, 5, 700, 32, 2, 128, True),       # sixteen heads of a query in a tile, the keys shared out
    (2, 77, 77, 21, 3, 128, True),       # seven heads: queries across tiles
])
def test_attention_rows_of_a_group(gpu_device, B, Tq, Tk, H, G, D, causal):
    print(f"[case] attention rows B{B} Tq{Tq} Tk{Tk} H{H} G{G} D{D}", flush=True)
    x = _inputs(gpu_device, B, Tq, Tk, H, G, D, BF, seed=B)
    _check(_run(*x, causal=causal), *x, causal=causal)


def test_attention_shared_keys_of_padded_rows(gpu_device):
    """Key shares past a row's length hold nothing; a row of no keys gives zeros."""
    lens = [0, 1, 700, 1600]
    x = _inputs(gpu_device, 4, 3, 1600, 2, 2, 64, BF, seed=19)
    got = _run(*x, causal=False, kv_lengths=torch.tensor(lens, device=gpu_device))
    _check(got, *x, causal=False, kv_lengths=lens)
    assert (got["o"][0] == 0).all() and (got["dq"][0] == 0).all()


def test_attention_nothing_to_see(gpu_device):
    """No keys at all, no queries at all, no rows at all."""
    from qwendopamine_amd import ops

    q, k, v, do = _inputs(gpu_device, 2, 5, 5, 2, 2, 64, BF)
    got = _run(q, k[:, :0].detach().requires_grad_(True), v[:, :0].detach().requires_grad_(True), do)
    assert (got["o"] == 0).all() and (got["dq"] == 0).all() and got["dk"].numel() == 0
    got = _run(q[:, :0].detach().requires_grad_(True), k, v, do[:, :0])
    assert got["o"].numel() == 0 and (got["dk"] == 0).all() and (got["dv"] == 0).all()
    assert ops.attention(q[:0], k[:0], v[:0]).shape == (0, 5, 2, 64)
    e = _run(*(x[:1, :0].detach().requires_grad_(True) for x in (q, k, v)), do[:1, :0], cu_seqlens=torch.tensor([0]))
    assert e["dq"].numel() == 0


@pytest.mark.parametrize("layout", ["fused", "heads first", "misaligned", "channels strided", "expanded"])
def test_attention_strides(gpu_device, layout):
    """The same values through other layouts give the same bits, gradients included."""
    B, T, H, G, D = 2, 70, 4, 2, 64
    q, k, v, do = (x.detach() for x in _inputs(gpu_device, B, T, T, H, G, D, BF, seed=9))
    if layout == "expanded":  # one row of k and v for the whole batch
        k, v = k[:1].expand(B, -1, -1, -1), v[:1].expand(B, -1, -1, -1)
    base = _run(*(x.contiguous().requires_grad_(True) for x in (q, k, v)), do)

    def other(x):
        if layout == "fused":
            return torch.cat((x.flatten(2), x.flatten(2)), -1).split(x.shape[2] * D, dim=-1)[1].view(x.shape)
        if layout == "heads first":
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "misaligned":
            return torch.cat((x.new_zeros(1), x.flatten()))[1:].view(x.shape)
        if layout == "channels strided":
            return torch.stack((x, x), -1)[..., 0]
        return x

    got = _run(*(other(x).requires_grad_(True) for x in (q, k, v)), other(do))
    assert all(torch.equal(base[n], got[n]) for n in base)
    if layout == "expanded":  # the leaf behind the broadcast gets the sum of its rows' gradients
        from qwendopamine_amd import ops

        leaf = k[:1].clone().requires_grad_(True)
        o = ops.attention(q, leaf.expand(B, -1, -1, -1), v)
        (dk,) = torch.autograd.grad(o, leaf, do)
        assert torch.equal(dk, base["dk"].sum(0, keepdim=True))


def test_attention_float16_gradients_keep_their_range(gpu_device):
    """Upstream gradients of 1e-5 and of 1e3, values of 30: fp16 dS would underflow or overflow
    unscaled; and one row of infinite gradient leaves the other heads alone."""
    for mag, do_mag in ((1.0, 1e-5), (30.0, 1e3)):
        print(f"[case] attention fp16 mag {mag} do {do_mag}", flush=True)
        x = _inputs(gpu_device, 1, 200, 200, 2, 2, 64, FP, seed=11, mag=mag, do_mag=do_mag)
        sc = 64 ** -0.5 / mag ** 2
        _check(_run(*x, scale=sc), *x, scale=sc)
    q, k, v, do = _inputs(gpu_device, 1, 40, 40, 2, 2, 64, FP, seed=12)
    base = _run(q, k, v, do)
    do = do.clone()
    do[0, 3, 0, 5] = float("inf")
    got = _run(q, k, v, do)
    assert all(torch.equal(base[n][:, :, 1], got[n][:, :, 1]) for n in ("dq", "dk", "dv"))
    assert torch.equal(base["dq"][0, 4:, 0], got["dq"][0, 4:, 0])


def test_attention_large_scores(gpu_device):
    """Scores of several hundred: the softmax is one-hot almost everywhere, the statistics hold."""
    x = _inputs(gpu_device, 1, 150, 150, 2, 1, 64, BF, seed=13, mag=8.0)
    _check(_run(*x), *x)


def test_attention_nonfinite_spreads_as_the_formula_says(gpu_device):
    from qwendopamine_amd import ops

    q, k, v, _ = (x.detach() for x in _inputs(gpu_device, 1, 80, 80, 2, 2, 64, BF, seed=14))
    q[0, 10, 0, 0] = float("nan")
    k[0, 70, 1, 0] = float("inf")
    o = ops.attention(q, k, v)
    assert torch.isnan(o[0, 10, 0]).all() and torch.isfinite(o[0, :10, 0]).all() and torch.isfinite(o[0, 11:, 0]).all()
    assert torch.isfinite(o[0, :70, 1]).all()  # a hidden infinite key leaves the queries before it alone


@pytest.mark.parametrize("D,dt", [(64, BF), (128, FP)])
def test_attention_single_key_rows_have_no_score_gradient(gpu_device, D, dt):
    """Where a query sees one key, P = 1 whatever the score: o is that key's v and dq exactly zero."""
    x = _inputs(gpu_device, 3, 300, 300, 4, 2, D, dt, seed=18, mag=3.0)
    got = _run(*x, causal=False, kv_lengths=torch.tensor([1, 1, 1], device=gpu_device))
    assert torch.equal(got["o"], x[2][:, :1].repeat_interleave(2, 2).expand(3, 300, 4, D))
    assert (got["dq"] == 0).all() and (got["dk"] == 0).all()
    got = _run(*x)
    assert (got["dq"][:, 0] == 0).all() and (got["dq"][:, 1] != 0).any()


def test_attention_gradient_against_differences(gpu_device):
    """<gradient, d> against central differences of the float64 loss along random directions."""
    q, k, v, do = _inputs(gpu_device, 1, 45, 45, 2, 1, 64, FP, seed=15)
    got = _run(q, k, v, do)
    X = [x.detach().cpu().double() for x in (q, k, v)]
    W = do.cpu().double()

    def loss(Q, K, V):
        S = torch.einsum("bihd,bjd->bhij", Q, K[:, :, 0]) / 8
        S = S.masked_fill(torch.ones(45, 45, dtype=torch.bool).triu(1), float("-inf"))
        return (torch.einsum("bhij,bjd->bihd", S.softmax(-1), V[:, :, 0]) * W).sum()

    gen = torch.Generator().manual_seed(1)
    for n, i in (("dq", 0), ("dk", 1), ("dv", 2)):
        d = torch.randn(X[i].shape, generator=gen, dtype=torch.float64)
        up, dn = ([x + (s * 1e-4 * d if j == i else 0) for j, x in enumerate(X)] for s in (1, -1))
        want = (loss(*up) - loss(*dn)) / 2e-4
        have = (got[n].cpu().double() * d).sum()
        # Each of the gradient's elements is off by about 2 u of its own size, at random.
        tol = 6 * 2.0 ** -11 * float((got[n].cpu().double() * d).norm()) + 1e-6 * abs(float(want))
        print(f"  {n}: {float(have):.6f} against {float(want):.6f} (tolerance {tol:.2e})", flush=True)
        assert abs(float(have - want)) <= tol


def test_attention_same_bits_twice_and_under_a_busy_device(gpu_device):
    x = _inputs(gpu_device, 2, 500, 500, 8, 2, 128, BF, seed=16)
    a = _run(*x)
    side = torch.cuda.Stream()
    noise = torch.randn(2048, 2048, device=gpu_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(5):
            noise = noise @ noise * 1e-3
        b = _run(*_inputs(gpu_device, 2, 500, 500, 8, 2, 128, BF, seed=16))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_attention_captured_training_replays(gpu_device):
    """Forward and backward captured together, replayed on new inputs: eager bits every time, and
    two graphs do not disturb each other."""
    from qwendopamine_amd import ops

    def capture(shape, dt):
        stat = [x.detach().clone() for x in _inputs(gpu_device, *shape, dt, seed=20)]
        leaves = [x.requires_grad_(True) for x in stat[:3]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(ops.attention(*leaves), leaves, stat[3])
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = ops.attention(*leaves)
            grads = torch.autograd.grad(o, leaves, stat[3])
        return g, stat, [o.detach(), *grads]

    graphs = [(capture((1, 96, 96, 4, 2, 64), FP), (1, 96, 96, 4, 2, 64), FP),
              (capture((2, 70, 70, 2, 2, 128), BF), (2, 70, 70, 2, 2, 128), BF)]
    for seed in (21, 22, 23):
        for (g, stat, out), shape, dt in graphs:
            new = _inputs(gpu_device, *shape, dt, seed=seed)
            with torch.no_grad():
                for s, x in zip(stat, new):
                    s.copy_(x)
            g.replay()
        for (g, stat, out), shape, dt in graphs:
            want = _run(*_inputs(gpu_device, *shape, dt, seed=seed))
            assert all(torch.equal(a, b) for a, b in zip(out, want.values()))


def test_attention_captured_with_lengths(gpu_device):
    """Padded rows replayed with other lengths (int32), key shares included."""
    from qwendopamine_amd import ops

    q, k, v, _ = (x.detach() for x in _inputs(gpu_device, 2, 4, 2000, 2, 1, 64, BF, seed=25))
    kv = torch.tensor([2000, 10], device=gpu_device, dtype=torch.int32)
    ops.attention(q, k, v, causal=False, kv_lengths=kv)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ops.attention(q, k, v, causal=False, kv_lengths=kv)
    for lens in ([5, 1999], [0, 700], [2000, 2000]):
        kv.copy_(torch.tensor(lens, device=gpu_device, dtype=torch.int32))
        g.replay()
        assert torch.equal(o, ops.attention(q, k, v, causal=False, kv_lengths=kv))


def test_attention_on_a_side_stream(gpu_device):
    """Inputs made on another stream, after it has been waited for; results used there."""
    x = _inputs(gpu_device, 1, 90, 90, 2, 2, 64, FP, seed=26)
    want = _run(*x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(*(t.detach().clone().requires_grad_(i < 3) for i, t in enumerate(x)))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(want[n], got[n]) for n in want)


def test_attention_refuses_a_second_derivative(gpu_device):
    from qwendopamine_amd import ops

    q, k, v, do = _inputs(gpu_device, 1, 8, 8, 1, 1, 64, BF)
    (dq,) = torch.autograd.grad(ops.attention(q, k, v), q, do, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()


@pytest.mark.parametrize("first,then", [([0, 400, 400, 400, 400], [0, 100, 200, 300, 400]),
                                        ([0, 3, 70, 400], [0, 400, 400, 400])])
def test_attention_packed_offsets_written_again_before_the_backward(gpu_device, first, then):
    """The caller's offsets buffer holds another partition by the time of the backward: gradients of
    the one that the forward took."""
    from qwendopamine_amd import ops

    x = _inputs(gpu_device, 1, 400, 400, 4, 2, 64, BF, seed=31)
    want = _run(*x, cu_seqlens=torch.tensor(first))
    cu = torch.tensor(first)
    o = ops.attention(*x[:3], cu_seqlens=cu)
    cu.copy_(torch.tensor(then))
    got = torch.autograd.grad(o, x[:3], x[3])
    assert torch.equal(o, want["o"]) and all(torch.equal(a, want[n]) for a, n in zip(got, ("dq", "dk", "dv")))


@pytest.mark.parametrize("T,D", [(128, 128), (150, 128), (200, 128), (150, 64)])
def test_attention_tokens_at_the_largest_stride(gpu_device, T, D):
    """q, k and v as columns of rows of 2^25 elements: offsets within a tile reach 2^32 bytes.  The
    same bits as contiguous ones."""
    print(f"[case] attention token stride 2^25, T{T} D{D}", flush=True)
    x = _inputs(gpu_device, 1, T, T, 4, 2, D, BF, seed=T)
    want = _run(*x)
    rows = torch.empty((T - 1) * 2 ** 25 + 8 * D, dtype=BF, device=gpu_device)
    at, far = 0, []
    for z in x[:3]:
        h = z.shape[2]
        y = rows.as_strided((1, T, h, D), (T * 2 ** 25, 2 ** 25, D, 1), at)
        y.copy_(z.detach())
        far.append(y.requires_grad_(True))
        at += h * D
    got = _run(*far, x[3])
    assert all(torch.equal(want[n], got[n]) for n in want)


def test_attention_float16_gradients_of_many_rows(gpu_device):
    """65536 rows of one token, 32 heads: the norms that scale fp16's dS take more than one launch.  A
    query that sees one key: o is its v, dv its dout, dq and dk zero."""
    print("[case] attention fp16 B65536 T1 H32 D64", flush=True)
    B, H, D = 65536, 32, 64
    gen = torch.Generator(gpu_device).manual_seed(3)
    q, k, v, do = (torch.randn(B, 1, H, D, generator=gen, device=gpu_device, dtype=FP) for _ in range(4))
    x = [z.requires_grad_(True) for z in (q, k, v)]
    got = _run(*x, do)
    assert torch.equal(got["o"], v) and torch.equal(got["dv"], do)
    assert not got["dq"].any() and not got["dk"].any()


@pytest.mark.parametrize("dt", [FP, BF])
@pytest.mark.parametrize("bits", [20.0, 25.5, 30.0])
@pytest.mark.parametrize("D,at", [(64, 0), (64, 9000), (128, 0)])
def test_attention_faint_keys_count_together(gpu_device, D, at, bits, dt):
    """One key of value 0 with all but the whole weight, 16383 others of 2^-bits of it each and values
    about 1000: the output is what the others add up to.  A probability is rounded by half a step ``u``
    of itself; fp16 holds it normal down to 2^-27 of the row's largest and to 2^-38 of that
    below; ``slack`` as in the reference, scores of up to 21."""
    from qwendopamine_amd import ops

    Tq, Tk, H = 2048, 16384, 16  # enough queries that the keys are not shared out
    print(f"[case] attention faint keys 2^-{bits} D{D} strong key {at} {dt}", flush=True)
    gen = torch.Generator(gpu_device).manual_seed(40)
    q, k = torch.zeros(1, 1, 1, D, device=gpu_device), torch.zeros(1, Tk, 1, D, device=gpu_device)
    q[..., 3], k[0, at, 0, 3] = 4.0, bits * 0.6931472 / 4
    v = 1000 * (0.5 + torch.rand(1, Tk, 1, D, generator=gen, device=gpu_device))
    v[0, at] = 0
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    o = ops.attention(q.expand(1, Tq, H, D), k.expand(1, Tk, H, D), v.expand(1, Tk, H, D), scale=1.0, causal=False)
    S = k[0, :, 0].double() @ q[0, 0, 0].double()
    P = torch.softmax(S, 0)
    want = P @ v[0, :, 0].double()
    u = torch.finfo(dt).eps / 2
    slack = 4 * D * 2.0 ** -24 * float(S.max()) + 2.0 ** -20
    bound = (2 * u + slack) * want * 1.01 + (Tk * 2.0 ** -38 * 1500 if dt == FP else 0.0)
    e = (o[0].double() - want).abs()
    print(f"  value {float(want[0]):.3e}, error / bound {float((e / bound).max()):.2f}", flush=True)
    assert bool((e <= bound).all())
