"""``ops.qkv_norm_rope`` against float64: both directions, types, head layouts, partial rotations, positions
inside and outside the tables, strides, graphs and streams.

Bounds, with u = 2^-24.  1 / rms: the mean of D <= 256 squares is 8 additions in a lane, up to 5 between lanes, a
division and the sum with eps, 15 u, halved by the root, and 2 u of the root itself; two products with it: n is
within 12 u.  A rotated value adds a product and a sum: within 14 u of |n_1 c| + |n_2 s| <= 1.42 |(n_1, n_2)|, 20 u
of the pair's norm.  The result is rounded once: half a step of its type, which is eps / 2 of the value and, under the
smallest normal number (fp16: 2^-14), eps / 2 of that (2^-25), as the steps there are all alike."""

from __future__ import annotations

import pytest
import torch

from qwendopamine_amd import ops
from qwendopamine_amd.hybrid import apply_rotary_emb

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
EPS = 1e-5


def tables(rows, pairs, dev):
    th = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
    a = torch.outer(torch.arange(rows, dtype=torch.float64), th)
    return a.cos().float().to(dev), a.sin().float().to(dev)


def rounding(y, dt):
    f = torch.finfo(dt)
    return f.eps / 2 * y.abs().clamp_min(f.tiny)


def turned(x, cos, sin, back=False):
    """``x [B, T, G, R, D]`` rotated by ``cos, sin [B, T, pairs]``; and the norms of the pairs."""
    r = 2 * cos.shape[-1]
    c, s = cos.double()[:, :, None, None], sin.double()[:, :, None, None]
    s = -s if back else s
    x1, x2 = x[..., :r:2], x[..., 1:r:2]
    y = torch.cat((torch.stack((x1 * c - x2 * s, x1 * s + x2 * c), -1).flatten(-2), x[..., r:]), -1)
    size = torch.cat(((x1 ** 2 + x2 ** 2).sqrt().repeat_interleave(2, -1), x[..., r:].abs()), -1)
    return y, size


def reference(qkv, cos, sin, H, G, wq, wk, pos, dq=None, dk=None, dv=None):
    """float64 values and bounds: ``{name: (value, bound)}``."""
    B, T, _ = qkv.shape
    R = H // G
    D = qkv.shape[-1] // (H + 2 * G)
    dt = qkv.dtype
    x = qkv.detach().double().view(B, T, G, R + 2, D)[..., :-1, :]
    at = torch.arange(T, device=qkv.device).expand(B, T) if pos is None else pos.expand(B, T)
    ok = (at >= 0) & (at < cos.shape[0])
    at = torch.where(ok, at, 0)
    ok = ok[:, :, None, None, None]
    c, s = cos[at], sin[at]
    if wq is not None:
        w = torch.cat((wq.detach().double().expand(R, D), wk.detach().double()[None]))
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        n = x * r * w
    else:
        n = x
    y, size = turned(n, c, s)
    y, size = torch.where(ok, y, 0.0), torch.where(ok, size, 0.0)
    tol = rounding(y, dt) + 20 * U * size + 1e-30
    out = dict(q=(y[..., :-1, :].flatten(2, 3), tol[..., :-1, :].flatten(2, 3)), k=(y[..., -1, :], tol[..., -1, :]))
    if dq is None:
        return out
    dy = torch.cat((dq.double().view(B, T, G, R, D), dk.double()[..., None, :]), -2)
    dn, dsize = turned(dy, c, s, back=True)
    dn, dsize = torch.where(ok, dn, 0.0), torch.where(ok, dsize, 0.0)
    if wq is not None:
        xr = x * r
        term = dn * xr
        dw = term.sum((0, 1, 2))
        # dn is within 3 u of its pair, xr within 11 u; a sum of N terms in lanes, waves and workgroups has
        # at most N / 8 + 80 additions in a chain (one lane alone takes every eighth row at most).
        count = B * T * G * R
        slack = (14 + count / 8 + 80) * U * (dsize * xr.abs()).sum((0, 1, 2))
        for name, a, b in (("dwq", dw[:-1].sum(0), slack[:-1].sum(0)), ("dwk", dw[-1], slack[-1])):
            out[name] = (a, rounding(a, wq.dtype) + b + 1e-30)
        m = (dn * w * xr).mean(-1, keepdim=True)
        mabs = (dsize * w.abs() * xr.abs()).mean(-1, keepdim=True)
        dx = (dn * w - xr * m) * r
        # Three products and a difference on top of dn (3 u), r (9 u), and of m: 13 additions, 16 u in its factors.
        slack = 40 * U * r * (dsize * w.abs() + xr.abs() * mabs)
    else:
        dx, slack = dn, 3 * U * dsize
    g = torch.cat((dx, dv.double()[..., None, :]), -2).flatten(2)
    b = torch.cat((rounding(dx, dt) + slack, torch.zeros_like(dv.double()[..., None, :])), -2).flatten(2) + 1e-30
    out["dqkv"] = (g, b)
    return out


def check(got, ref):
    for name, (want, tol) in ref.items():
        err = (got[name].detach().double() - want).abs()
        worst = (err - tol).max().item() if err.numel() else 0.0
        assert worst <= 0, f"{name}: {worst:.3e} past its bound (at {int((err - tol).argmax())})"


def inputs(B, T, H, G, D, dt, dev, seed=0, norm=True, wdt=None, scale=1.0):
    g = torch.Generator().manual_seed(seed)

    def r(*shape):
        return torch.randn(*shape, generator=g, dtype=F32)
    qkv = (r(B, T, (H + 2 * G) * D) * scale).to(dt).to(dev)
    wq = wk = None
    if norm:
        wq, wk = ((1 + 0.3 * r(D)).to(wdt or dt).to(dev) for _ in range(2))
    return qkv, wq, wk, [r(B, T, n, D).to(dt).to(dev) for n in (H, G, G)]


SHAPES = [  # B, T, H, G, D, pairs
    (1, 1, 1, 1, 8, 4),
    (2, 3, 2, 1, 16, 3),
    (3, 5, 4, 2, 32, 16),
    (1, 33, 6, 3, 40, 10),
    (2, 17, 16, 16, 64, 32),
    (2, 9, 7, 1, 64, 16),
    (1, 7, 12, 4, 96, 48),
    (2, 130, 8, 2, 128, 64),
    (1, 5, 32, 8, 128, 32),
    (1, 40, 3, 3, 256, 128),
    (2, 6, 4, 4, 248, 1),
    (1, 3, 64, 1, 64, 0),
]


@pytest.mark.parametrize("dt", [BF, FP, F32], ids=str)
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_both_directions(gpu_device, shape, norm, dt):
    B, T, H, G, D, pairs = shape
    qkv, wq, wk, d = inputs(B, T, H, G, D, dt, gpu_device, 1, norm)
    cos, sin = tables(T + 3, pairs, gpu_device)
    leaves = [x.requires_grad_(True) for x in (qkv, wq, wk) if x is not None]
    q, k, v = ops.qkv_norm_rope(qkv, cos, sin, H, G, wq, wk, EPS)
    grads = torch.autograd.grad((q, k, v), leaves, d)
    got = dict(q=q, k=k, dqkv=grads[0])
    if norm:
        got.update(dwq=grads[1], dwk=grads[2])
    check(got, reference(qkv, cos, sin, H, G, wq, wk, None, *d))
    assert torch.equal(v, qkv.view(B, T, G, H // G + 2, D)[..., -1, :])
    assert v.data_ptr() == qkv.data_ptr() + (H // G + 1) * D * qkv.element_size()  # in place


@pytest.mark.parametrize("dt", [BF, FP, F32], ids=str)
def test_rotation_has_the_bits_of_the_hosts(gpu_device, dt):
    H, G, D = 8, 4, 64
    qkv, _, _, d = inputs(2, 50, H, G, D, dt, gpu_device, 2, False)
    cos, sin = tables(50, 24, gpu_device)
    a, b = qkv.clone().requires_grad_(True), qkv.clone().requires_grad_(True)
    q, k, v = ops.qkv_norm_rope(a, cos, sin, H, G)
    xq, xk, xv = b.view(2, 50, G, 4, D).split((2, 1, 1), dim=-2)
    want = (apply_rotary_emb(xq.reshape(2, 50, H, D), cos, sin), apply_rotary_emb(xk.reshape(2, 50, G, D), cos, sin),
            xv.reshape(2, 50, G, D))
    for x, y in zip((q, k, v), want):
        assert torch.equal(x, y)
    assert torch.equal(*(torch.autograd.grad(o, (x,), d)[0] for o, x in (((q, k, v), a), (want, b))))


@pytest.mark.parametrize("each", [True, False])
def test_positions(gpu_device, each):
    """Positions of every order, and outside the tables: zeros, and no gradient but the values'."""
    B, T, H, G, D = 3, 6, 4, 2, 64
    qkv, wq, wk, d = inputs(B, T, H, G, D, BF, gpu_device, 3)
    cos, sin = tables(20, 32, gpu_device)
    pos = torch.tensor([[5, 19, 0, -1, 20, 7], [3, 3, 3, 2 ** 40, 1, 18], [-2 ** 60, 4, 11, 12, 13, 0]], device=gpu_device)
    pos = pos if each else pos[0]
    leaves = [x.requires_grad_(True) for x in (qkv, wq, wk)]
    q, k, v = ops.qkv_norm_rope(qkv, cos, sin, H, G, wq, wk, EPS, pos)
    grads = torch.autograd.grad((q, k, v), leaves, d)
    check(dict(q=q, k=k, dqkv=grads[0], dwq=grads[1], dwk=grads[2]), reference(qkv, cos, sin, H, G, wq, wk, pos, *d))
    strided = torch.empty(B, T, 2, dtype=torch.int64, device=gpu_device)
    strided[..., 0] = pos
    p2 = strided[..., 0] if each else strided[0, :, 0]
    q2, k2, _ = ops.qkv_norm_rope(qkv.detach(), cos, sin, H, G, wq.detach(), wk.detach(), EPS, p2)
    assert torch.equal(q, q2) and torch.equal(k, k2)


def test_no_position_passes_nothing_of_nan(gpu_device):
    """A padded token may hold anything: its NaN reaches neither other tokens nor the weights."""
    qkv, wq, wk, d = inputs(1, 4, 2, 1, 64, BF, gpu_device, 4)
    qkv[0, 2] = float("nan")
    d[0][0, 2] = float("nan")
    d[1][0, 2] = float("inf")
    cos, sin = tables(9, 32, gpu_device)
    leaves = [x.requires_grad_(True) for x in (qkv, wq, wk)]
    outs = ops.qkv_norm_rope(qkv, cos, sin, 2, 1, wq, wk, EPS, torch.tensor([1, 2, -1, 3], device=gpu_device))
    grads = torch.autograd.grad(outs, leaves, d)
    assert (outs[0][0, 2] == 0).all() and (outs[1][0, 2] == 0).all()
    assert (grads[0][0, 2, :192] == 0).all() and torch.equal(grads[0][0, 2, 192:], d[2][0, 2, 0])
    assert all(g.isfinite().all() for g in grads[1:])


@pytest.mark.parametrize("how", ["columns", "unaligned", "transposed", "batch"])
def test_strides(gpu_device, how):
    B, T, H, G, D = 2, 12, 4, 2, 64
    W = (H + 2 * G) * D
    qkv, wq, wk, d = inputs(B, T, H, G, D, FP, gpu_device, 5)
    cos, sin = tables(T, 32, gpu_device)
    if how == "columns":
        x = torch.zeros(B, T, W + 64, dtype=FP, device=gpu_device)[..., 32:32 + W]
    elif how == "unaligned":
        x = torch.zeros(B, T, W + 64, dtype=FP, device=gpu_device)[..., 3:3 + W]
    elif how == "transposed":
        x = torch.zeros(T, B, W, dtype=FP, device=gpu_device).transpose(0, 1)
    else:
        x = torch.zeros(1, T, W, dtype=FP, device=gpu_device).expand(B, T, W)
        qkv = qkv[:1].expand(B, T, W)
    if how != "batch":
        x.copy_(qkv)
    else:
        x = qkv
    x = x.detach().requires_grad_(True)
    w = [t.requires_grad_(True) for t in (wq, wk)]
    # Weights of any alignment, too.
    w = [torch.zeros(D + 3, dtype=FP, device=gpu_device)[3:].copy_(t).requires_grad_(True) for t in w]
    outs = ops.qkv_norm_rope(x, cos, sin, H, G, *w)
    grads = torch.autograd.grad(outs, (x, *w), [torch.empty_like(t.transpose(1, 2)).transpose(1, 2).copy_(t) for t in d])
    check(dict(q=outs[0], k=outs[1], dqkv=grads[0], dwq=grads[1], dwk=grads[2]),
          reference(qkv.contiguous(), cos, sin, H, G, wq, wk, None, *d))


def test_float32_weights_of_a_16_bit_layer(gpu_device):
    qkv, wq, wk, d = inputs(2, 30, 4, 4, 64, BF, gpu_device, 6, wdt=F32)
    cos, sin = tables(30, 32, gpu_device)
    leaves = [x.requires_grad_(True) for x in (qkv, wq, wk)]
    outs = ops.qkv_norm_rope(qkv, cos, sin, 4, 4, wq, wk)
    grads = torch.autograd.grad(outs, leaves, d)
    assert grads[1].dtype == F32
    check(dict(q=outs[0], k=outs[1], dqkv=grads[0], dwq=grads[1], dwk=grads[2]),
          reference(qkv, cos, sin, 4, 4, wq, wk, None, *d))


def test_gradient_against_differences(gpu_device):
    """Central differences along random directions of a float32 layer.  The loss is a sum of about 3000 products of
    size 1, each value within 20 u: its error is under 3000 * 20 u sqrt-free = 4e-3 at worst and 1e-5 in the mean
    square; over a step of 2 * 0.01 that is 1e-3 of a directional derivative of size about 50; the third
    derivative adds 0.01^2 of it."""
    B, T, H, G, D = 2, 4, 2, 1, 96
    qkv, wq, wk, d = inputs(B, T, H, G, D, F32, gpu_device, 7)
    cos, sin = tables(T, 40, gpu_device)

    def loss(x, a, b):
        return sum((o.double() * g.double()).sum() for o, g in zip(ops.qkv_norm_rope(x, cos, sin, H, G, a, b), d))
    leaves = [x.clone().requires_grad_(True) for x in (qkv, wq, wk)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    gen = torch.Generator().manual_seed(8)
    for i, (x, g) in enumerate(zip((qkv, wq, wk), grads)):
        v = torch.randn(x.shape, generator=gen).to(gpu_device)
        v = v / v.square().mean().sqrt()
        h = 0.01
        args = [[qkv, wq, wk], [qkv, wq, wk]]
        args[0][i], args[1][i] = x + h * v, x - h * v
        with torch.no_grad():
            diff = (loss(*args[0]) - loss(*args[1])) / (2 * h)
        along = (g.double() * v.double()).sum()
        size = (g.double().square().sum() * v.double().square().sum()).sqrt()  # of the scalar product's factors
        assert abs(diff - along) <= 2e-3 * size, (i, float(diff), float(along))


def test_partial_gradients(gpu_device):
    """Outputs that get no gradient, and inputs that want none."""
    qkv, wq, wk, d = inputs(1, 8, 2, 2, 64, BF, gpu_device, 9)
    cos, sin = tables(8, 32, gpu_device)
    x = qkv.clone().requires_grad_(True)
    q, k, v = ops.qkv_norm_rope(x, cos, sin, 2, 2, wq, wk)
    (g,) = torch.autograd.grad(q, x, d[0])
    zero = torch.zeros_like(d[1])
    check(dict(dqkv=g), {"dqkv": reference(qkv, cos, sin, 2, 2, wq, wk, None, d[0], zero, zero)["dqkv"]})
    w = wq.clone().requires_grad_(True)
    q, k, v = ops.qkv_norm_rope(qkv, cos, sin, 2, 2, w, wk)
    (g,) = torch.autograd.grad(q, w, d[0])
    check(dict(dwq=g), {"dwq": reference(qkv, cos, sin, 2, 2, wq, wk, None, d[0], zero, zero)["dwq"]})
    x = qkv.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.qkv_norm_rope(x, cos, sin, 2, 2, wq, wk)[2], x, d[2])
    assert torch.equal(g.view(1, 8, 2, 3, 64)[..., 2, :], d[2]) and (g.view(1, 8, 2, 3, 64)[..., :2, :] == 0).all()


def test_second_derivatives_and_tangents_are_refused(gpu_device):
    qkv, wq, wk, _ = inputs(1, 2, 2, 2, 64, F32, gpu_device, 10)
    cos, sin = tables(2, 32, gpu_device)
    x = qkv.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.qkv_norm_rope(x, cos, sin, 2, 2, wq, wk)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        ops.qkv_norm_rope(torch.autograd.forward_ad.make_dual(qkv, qkv), cos, sin, 2, 2, wq, wk)


def test_empty(gpu_device):
    cos, sin = tables(4, 32, gpu_device)
    for shape in ((0, 3, 256), (2, 0, 256)):
        x = torch.zeros(shape, dtype=BF, device=gpu_device, requires_grad=True)
        w = [torch.ones(64, dtype=BF, device=gpu_device, requires_grad=True) for _ in range(2)]
        q, k, v = ops.qkv_norm_rope(x, cos, sin, 2, 1, *w)
        assert q.shape == (*shape[:2], 2, 64)
        grads = torch.autograd.grad((q.sum() + k.sum() + v.sum()), (x, *w))
        assert grads[0].shape == shape and all((g == 0).all() for g in grads[1:])


def test_large(gpu_device):
    """Many rounds of workgroups in the backward; the same bits in every run."""
    B, T, H, G, D = 2, 3001, 16, 4, 64
    qkv, wq, wk, d = inputs(B, T, H, G, D, BF, gpu_device, 11)
    cos, sin = tables(T, 32, gpu_device)
    leaves = [x.requires_grad_(True) for x in (qkv, wq, wk)]
    runs = []
    for _ in range(2):
        outs = ops.qkv_norm_rope(qkv, cos, sin, H, G, wq, wk)
        runs.append(torch.autograd.grad(outs, leaves, d))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    check(dict(q=outs[0], k=outs[1], dqkv=runs[0][0], dwq=runs[0][1], dwk=runs[0][2]),
          reference(qkv, cos, sin, H, G, wq, wk, None, *d))


def test_graph_and_stream(gpu_device):
    """Forward and backward captured together, replayed on new inputs with eager work between; a side stream."""
    H, G, D, T = 4, 2, 64, 70
    cos, sin = tables(T, 32, gpu_device)
    new = [inputs(2, T, H, G, D, BF, gpu_device, 20 + i) for i in range(4)]
    static = [x.clone().requires_grad_(True) for x in new[0][:3]]
    d = [x.clone() for x in new[0][3]]

    def step(leaves, d):
        outs = ops.qkv_norm_rope(leaves[0], cos, sin, H, G, leaves[1], leaves[2])
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, d)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [step([x.clone().requires_grad_(True) for x in n[:3]], n[3]) for n in new]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static, d)
    for n, want in zip(new, eager):
        with torch.no_grad():
            for dst, src in zip((*static, *d), (*n[:3], *n[3])):
                dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        torch.randn(1000, device=gpu_device).sum()


@pytest.mark.parametrize("norm", [True, False])
def test_tables_without_rows(gpu_device, norm):
    """No token has a position: q and k are zeros, and no gradient passes but the values'."""
    B, T, H, G, D = 2, 5, 4, 2, 64
    qkv, wq, wk, d = inputs(B, T, H, G, D, BF, gpu_device, 30, norm)
    cos = sin = torch.empty(0, 32, device=gpu_device)
    pos = torch.tensor([0, 1, -1, 2 ** 40, 4], device=gpu_device)
    leaves = [x.requires_grad_(True) for x in (qkv, wq, wk) if x is not None]
    q, k, v = ops.qkv_norm_rope(qkv, cos, sin, H, G, wq, wk, EPS, pos)
    grads = torch.autograd.grad((q, k, v), leaves, d)
    rows = grads[0].view(B, T, G, H // G + 2, D)
    assert (q == 0).all() and (k == 0).all() and torch.equal(v, qkv.view(rows.shape)[..., -1, :])
    assert (rows[..., :-1, :] == 0).all() and torch.equal(rows[..., -1, :], d[2])
    assert all((g == 0).all() for g in grads[1:])


@pytest.mark.parametrize("how,copies", [("readable", 0), ("unaligned", 1), ("spread", 1)])
def test_projection_is_copied_once(gpu_device, how, copies):
    """In training, where it cannot be read in place; its gradient has its layout all the same."""
    from torch.utils._python_dispatch import TorchDispatchMode

    B, T, H, G, D = 2, 12, 4, 2, 64
    W = (H + 2 * G) * D
    qkv, wq, wk, d = inputs(B, T, H, G, D, BF, gpu_device, 31)
    cos, sin = tables(T, 32, gpu_device)
    base = torch.zeros(B, T, 2 * W, dtype=BF, device=gpu_device)
    x = {"readable": base[..., :W], "unaligned": base[..., 3:3 + W], "spread": base[..., ::2]}[how]
    x = x.copy_(qkv).detach().requires_grad_(True)
    made = []

    class Count(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if func in (torch.ops.aten.clone.default, torch.ops.aten._to_copy.default, torch.ops.aten.copy_.default):
                made.append(out.numel())
            return out
    with Count():
        outs = ops.qkv_norm_rope(x, cos, sin, H, G, wq, wk)
    assert made == [B * T * W] * copies
    (g,) = torch.autograd.grad(outs, x, d)
    check(dict(q=outs[0], k=outs[1], dqkv=g),
          {n: r for n, r in reference(qkv, cos, sin, H, G, wq, wk, None, *d).items() if n in ("q", "k", "dqkv")})
