"""``ops.sample_tokens`` against the definition in float64, token for token: settings alone and together, equal
logits, masked and infinite ones, lengths from one on, lists that overflow, layouts, graphs and streams.

A token differs from the definition's only if the random number (or a border of a filter) lies within about
2^-42 of a running sum's relative place: none of these inputs does but with a chance of 1e-6."""

from __future__ import annotations

import pytest
import torch

from qwendopamine_amd import ops

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def f32(x):
    return torch.tensor(float(x), dtype=F32).double().item()


def pick(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """One row, on the CPU in float64."""
    x = x.double().cpu()
    T, p, m, u = f32(T), f32(p), f32(m), f32(u)
    top = x.max()
    if T <= 0 or not torch.isfinite(top):
        nan = x.isnan().nonzero()
        return int(nan[0]) if len(nan) else int((x == top).nonzero()[0])
    order = torch.sort(x, descending=True, stable=True).indices
    w = ((x - top) / T).exp()[order]
    n = len(x)
    if m > 0:
        n = min(n, int((w >= m).sum()))
    if k > 0:
        n = min(n, k)
    if p < 1:
        before = w[:n].cumsum(0) - w[:n]
        n = max(1, int((before < p * w[:n].sum()).sum()))
    kept = order[:n].sort().values
    run = ((x[kept] - top) / T).exp().cumsum(0)
    return int(kept[min(int((run <= u * run[-1]).sum()), n - 1)])


def logits(rows, V, dt, seed=0, spread=2.2):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, V, generator=g) * spread
    x.scatter_add_(1, torch.randint(0, V, (rows, 20), generator=g), 8 * torch.rand(rows, 20, generator=g))
    return x.to(dt), torch.rand(rows, generator=g)


def check(x, u, dev, **kw):
    got = ops.sample_tokens(x.to(dev), u.to(dev), **kw)
    assert got.dtype == torch.int64 and got.shape == u.shape
    names = dict(temperature="T", top_k="k", top_p="p", min_p="m")

    def at(v, i):
        return v.flatten()[i].item() if isinstance(v, torch.Tensor) else v
    rows, us = x.reshape(-1, x.shape[-1]), u.flatten()
    want = [pick(rows[i], us[i], **{names[n]: at(v, i) for n, v in kw.items()}) for i in range(len(us))]
    assert got.flatten().tolist() == want


SETTINGS = [
    {}, dict(temperature=0.0), dict(temperature=0.3), dict(temperature=2.5), dict(top_k=1), dict(top_k=5), dict(top_k=40),
    dict(top_p=0.9), dict(top_p=0.3), dict(top_p=1e-6), dict(min_p=0.1), dict(min_p=1.0), dict(min_p=1e-9),
    dict(temperature=0.8, top_k=50, top_p=0.95), dict(temperature=1.4, top_k=300, top_p=0.7, min_p=0.01),
    dict(top_p=0.99, min_p=0.02), dict(top_k=7, min_p=0.2), dict(temperature=1.5, top_k=20, top_p=0.9),
]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("dt", [BF, FP, F32], ids=str)
@pytest.mark.parametrize("rows,V", [(40, 1), (40, 2), (60, 7), (50, 300), (21, 4099), (5, 40007)])
def test_settings(gpu_device, rows, V, dt, kw):
    check(*logits(rows, V, dt, V), gpu_device, **kw)


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("dt", [BF, F32], ids=str)
def test_equal_logits(gpu_device, kw, dt):
    """Few distinct values, so that every border falls among equals: the lower index first."""
    g = torch.Generator().manual_seed(3)
    for V in (6, 250, 3001):
        x = torch.randint(-2, 3, (24, V), generator=g).to(dt)
        check(x, torch.rand(24, generator=g), gpu_device, **kw)


@pytest.mark.parametrize("kw", [{}, dict(top_k=9000), dict(top_k=3), dict(top_p=0.55), dict(top_k=15000, top_p=0.5),
                                dict(top_k=5, top_p=0.5, min_p=0.3), dict(top_p=0.999)], ids=str)
@pytest.mark.parametrize("dt", [BF, FP, F32], ids=str)
def test_more_equals_than_are_listed(gpu_device, kw, dt):
    """Border bins of more elements than the list holds: the row itself is searched."""
    g = torch.Generator().manual_seed(4)
    V = 20011
    x = torch.zeros(4, V)
    x[1] = torch.randint(0, 2, (V,), generator=g) * 2.0 - 1.0
    x[2] = -7.5
    x[2, 19000:] = -7.0
    x[3] = torch.randint(0, 3, (V,), generator=g) * 0.5
    x[3, 777] = 3.0
    u = torch.tensor([0.37, 0.81, 0.93, 0.52])
    check(x.to(dt), u, gpu_device, **kw)


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_masked_and_infinite(gpu_device, kw):
    x, u = logits(12, 700, BF, 5)
    low = torch.finfo(BF).min
    x[0, 1:] = -float("inf")         # a single token left, the first
    x[1, :-1] = -float("inf")        # the last
    x[2] = -float("inf")             # none
    x[3] = low                       # all at the type's lowest value
    x[4, ::2] = low
    x[5, 100:] = -float("inf")
    x[6, 33] = float("inf")
    x[6, 40] = float("inf")
    x[7, 44] = float("nan")
    x[7, 20] = float("inf")
    x[8] = float("nan")
    x[9] = float("inf")
    x[10, ::3] = -float("inf")
    x[11, :350] = float("-0.0")
    x[11, 350:] = 0.0
    check(x, u, gpu_device, **kw)


def test_random_numbers(gpu_device):
    """Every share of [0, 1) to its token; 0, the last number under 1, and what is outside."""
    x, _ = logits(1, 9, F32, 6, 1.0)
    u = torch.arange(4001) / 4001
    check(x.expand(4001, 9), u, gpu_device)
    check(x.expand(4001, 9), u, gpu_device, top_k=4, temperature=0.7)
    edge = torch.tensor([0.0, 1.0 - 2.0 ** -24, 2.0 ** -149])
    check(x.expand(3, 9), edge, gpu_device)
    check(x.expand(3, 9), edge, gpu_device, top_p=0.6)
    out = ops.sample_tokens(x.expand(4, 9).to(gpu_device),
                            torch.tensor([-1.0, 1.0, 7.0, float("nan")], device=gpu_device), top_k=3)
    three = x[0].topk(3).indices.sort().values
    assert out.tolist() == [int(three[0]), int(three[2]), int(three[2]), int(three[0])]


def test_settings_of_each_row(gpu_device):
    x, u = logits(14, 5000, BF, 7)
    kw = dict(temperature=torch.tensor([0.0, 0.5, 1.0, 1.3, 2.0, 0.8, 1.0] * 2), top_k=torch.tensor([0, 1, 50, 0, 4999, 5000, 9000] * 2),
              top_p=torch.tensor([1.0, 0.9, 0.5, 0.95, 1.0, 0.2, 1.0] * 2), min_p=torch.tensor([0.0, 0.0, 0.01, 0.0, 0.0, 0.3, 0.02] * 2))
    dev = {n: v.to(gpu_device) for n, v in kw.items()}
    got = ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), **dev).tolist()
    assert got == [pick(x[i], u[i], *(kw[n][i].item() for n in ("temperature", "top_k", "top_p", "min_p"))) for i in range(14)]
    dev["top_k"] = dev["top_k"].int()
    dev["top_p"] = dev["top_p"].double()
    assert ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), **dev).tolist() == got
    one = dict(temperature=0.9, top_k=dev["top_k"], top_p=0.95)
    check(x, u, gpu_device, **one)
    # Outside their ranges: as documented.
    odd = ops.sample_tokens(x[:6].to(gpu_device), u[:6].to(gpu_device),
                            temperature=torch.tensor([-1.0, float("nan"), 1.0, 1.0, 1.0, 1.0], device=gpu_device),
                            top_k=torch.tensor([0, 0, -5, 0, 0, 0], device=gpu_device),
                            top_p=torch.tensor([1.0, 1.0, 1.0, 2.0, -1.0, float("nan")], device=gpu_device),
                            min_p=torch.tensor([0.0, 0.0, float("nan"), -1.0, 0.0, 2.0], device=gpu_device))
    want = [pick(x[0], u[0], 0.0), pick(x[1], u[1], 0.0), pick(x[2], u[2]), pick(x[3], u[3]), pick(x[4], u[4], k=1),
            pick(x[5], u[5], m=1.0)]
    assert odd.tolist() == want


def test_layouts(gpu_device):
    """Rows of any alignment and stride, two leading axes, one row without any."""
    for dt in (BF, F32):
        x, u = logits(12, 1003, dt, 8)
        kw = dict(top_k=30, top_p=0.9)
        want = ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), **kw)
        check(x, u, gpu_device, **kw)
        for off in (0, 1, 3, 5, 8):
            wide = torch.full((12, 1003 + 21), 50.0, dtype=dt, device=gpu_device)  # what lies outside must not count
            wide[:, off:off + 1003] = x.to(gpu_device)
            assert torch.equal(ops.sample_tokens(wide[:, off:off + 1003], u.to(gpu_device), **kw), want)
        y = torch.zeros(3, 5, 1003, dtype=dt, device=gpu_device)
        y[:, 1:] = x.view(3, 4, 1003).to(gpu_device)
        assert torch.equal(ops.sample_tokens(y[:, 1:], u.view(3, 4).to(gpu_device), **kw), want.view(3, 4))
        assert torch.equal(ops.sample_tokens(x.t().contiguous().to(gpu_device).t(), u.to(gpu_device), **kw), want)
        assert int(ops.sample_tokens(x[2].to(gpu_device), u[2].to(gpu_device), **kw)) == int(want[2])
        assert ops.sample_tokens(x[:0].to(gpu_device), u[:0].to(gpu_device)).shape == (0,)


def test_many_rows(gpu_device):
    """More rows than a round of workgroups holds, and no dependence on how a row is divided."""
    x, u = logits(700, 2600, BF, 9)
    kw = dict(temperature=0.9, top_k=100, top_p=0.9)
    many = ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), **kw)
    few = torch.cat([ops.sample_tokens(x[i:i + 1].to(gpu_device), u[i:i + 1].to(gpu_device), **kw) for i in range(0, 700, 70)])
    assert torch.equal(many[::70], few)
    check(x[:50], u[:50], gpu_device, **kw)


@pytest.mark.parametrize("kw", [{}, dict(temperature=0.7, top_p=0.95), dict(top_k=60, top_p=0.8), dict(min_p=0.02), dict(top_k=3000)],
                         ids=str)
def test_long_parts(gpu_device, kw):
    """So many rows that each is a part of its own, long enough for bf16 values to be counted first: the tokens of
    the same rows a hundred at a time, whose parts are shorter; and the definition's of the odd rows."""
    rows, V = 2100, 9001
    x, u = logits(rows, V, BF, 12)
    x[0] = 0.0
    x[1, ::2] = -float("inf")
    x[2, 5:] = torch.finfo(BF).min
    x[3] = x[3] + 300.0
    x[4] = x[4] * 1e-4
    x[5] = x[5] * 1e-30
    x[6, 17] = float("nan")
    x[7] = x[7] * 3000.0
    x[8, 4500:] = -1e4
    x[9] = -x[9].abs() - 50.0
    x[10] = -float("inf")
    got = ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), **kw)
    few = torch.cat([ops.sample_tokens(x[i:i + 100].to(gpu_device), u[i:i + 100].to(gpu_device), **kw)
                     for i in range(0, rows, 100)])
    assert torch.equal(got, few)
    check(x[:12], u[:12], gpu_device, **kw)


def test_largest_row(gpu_device):
    V = 1 << 20
    g = torch.Generator().manual_seed(10)
    x = torch.randn(2, V, generator=g)
    u = torch.tensor([0.2, 0.9])
    check(x.to(BF), u, gpu_device, top_p=0.8)
    check(x, u, gpu_device)
    check(x * 0, u, gpu_device)


def test_greedy_is_argmax_rows(gpu_device):
    x, u = logits(30, 2000, BF, 11)
    x = (x * 2).round().to(gpu_device)
    assert torch.equal(ops.sample_tokens(x, u.to(gpu_device), temperature=0.0), ops.argmax_rows(x)[:, 0])


def test_graph_and_streams(gpu_device):
    """Captured once, replayed on new logits and numbers; two graphs in turn; calls on two streams at once."""
    kw = dict(temperature=0.9, top_k=200, top_p=0.95)
    data = [tuple(t.to(gpu_device) for t in logits(8, 30000, BF, 50 + i)) for i in range(4)]
    want = [ops.sample_tokens(x, u, **kw) for x, u in data]
    x, u = (t.clone() for t in data[0])
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.sample_tokens(x, u, **kw)
        graphs.append((graph, out))
    for i, (a, b) in enumerate(data):
        x.copy_(a)
        u.copy_(b)
        graphs[i % 2][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[i % 2][1], want[i])
        torch.randn(100, device=gpu_device).sum()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.sample_tokens(*data[i], **kw))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_refusals_on_the_device(gpu_device):
    x, u = logits(2, 10, F32, 1)
    with pytest.raises(RuntimeError):
        ops.sample_tokens(x.to(gpu_device), u)
    with pytest.raises(RuntimeError):
        ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), top_p=torch.ones(2))
    with pytest.raises(ValueError):
        ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), top_p=torch.ones(1, device=gpu_device))
    with pytest.raises(ValueError):
        ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), top_k=torch.ones(2, device=gpu_device))


def test_rows_past_a_quarter_million(gpu_device):
    """More rows than the largest number of parts would leave workgroups for: as in smaller calls."""
    g = torch.Generator().manual_seed(90)
    x, u = torch.randn(300001, 7, generator=g), torch.rand(300001, generator=g)
    xd, ud = x.to(gpu_device), u.to(gpu_device)
    got = ops.sample_tokens(xd, ud, temperature=0.9, top_k=4, top_p=0.95)
    parts = [ops.sample_tokens(xd[i:i + 100000], ud[i:i + 100000], temperature=0.9, top_k=4, top_p=0.95)
             for i in range(0, 300001, 100000)]
    assert torch.equal(got, torch.cat(parts))
    assert got[-300:].tolist() == [pick(x[i], u[i], T=0.9, k=4, p=0.95) for i in range(-300, 0)]


@pytest.mark.parametrize("p", [1e-30, 1e-40, 1e-46, 5e-324])
def test_shares_under_float32(gpu_device, p):
    """A share that is 0 in float32 keeps one token, given as a number or for each row."""
    x, u = logits(9, 300, BF, 91)
    want = [int((row == row.max()).nonzero()[0]) for row in x]
    assert ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), top_p=p).tolist() == want
    each = torch.full((9,), p, device=gpu_device)
    assert ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), top_p=each).tolist() == want


@pytest.mark.parametrize("kw", [{}, dict(top_p=0.7), dict(top_k=9), dict(top_k=1500, top_p=0.5), dict(min_p=1.0), dict(min_p=0.3)],
                         ids=str)
@pytest.mark.parametrize("dt", [BF, FP, F32], ids=str)
def test_largest_temperatures(gpu_device, kw, dt):
    """All weights are 1, in the order of the logits; an infinite temperature of a row counts as the largest."""
    x, u = logits(8, 4000, dt, 92)
    x[1, ::3] = -float("inf")
    x[2] = -float("inf")
    x[3, 1:] = -float("inf")
    x[4] = torch.finfo(dt).min
    x[4, 77] = torch.finfo(dt).max / 2
    want = [pick(x[i], u[i], T=3e38, **{dict(top_k="k", top_p="p", min_p="m")[n]: v for n, v in kw.items()}) for i in range(8)]
    for t in (3e38, torch.full((8,), 3e38, device=gpu_device), torch.full((8,), float("inf"), device=gpu_device)):
        got = ops.sample_tokens(x.to(gpu_device), u.to(gpu_device), temperature=t, **kw).tolist()
        for i in range(8):
            if i != 4 or not isinstance(t, torch.Tensor) or bool(t[4].isfinite()):  # (there a span of the type's counts)
                assert got[i] == want[i], i
