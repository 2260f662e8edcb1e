"""The 4-bit key / value cache: ``ops.kv_cache_q4_store`` / ``kv_cache_q4_load`` code for code against
the definition, ``ops.attention_decode_q4`` against float64 attention over what the cache stands for:
lengths from one position on, ragged and outside positions, heads per group, partial rotations,
graphs, and a whole prompt in pieces.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def quantise(x):
    """The definition, in CPU float32: codes ``[..., D]`` and (scale, minimum) ``[..., D / 64, 2]``."""
    g = x.cpu().float().unflatten(-1, (-1, 64))
    ok = g.isfinite().all(-1, keepdim=True)
    lo = g.amin(-1, keepdim=True).bfloat16()
    fifteenth = torch.tensor(1.0 / 15.0, dtype=F32)
    sc = ((g.amax(-1, keepdim=True) - lo.float()) * fifteenth).clamp_min(0).bfloat16()
    inv = torch.where(sc.float() > 0, 1.0 / sc.float(), 0.0)
    n = torch.where(ok, ((g - lo.float()) * inv).round().clamp(0, 15), 0.0)
    nan = torch.tensor(float("nan"), dtype=BF)
    return n.flatten(-2).to(torch.uint8), torch.cat((torch.where(ok, sc, nan), torch.where(ok, lo, nan)), -1)


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


def values(codes, meta, dtype=torch.float64):
    n = unpack(codes.cpu()).to(dtype).unflatten(-1, (-1, 64))
    m = meta.cpu().to(dtype)
    return (n * m[..., :1] + m[..., 1:]).flatten(-2)


def same(a, b):
    return torch.equal(a.nan_to_num(nan=1e30), b.nan_to_num(nan=1e30))


def tables(L, D, pairs, dev):
    th = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) * 2 / D)
    a = torch.outer(torch.arange(L, dtype=torch.float64), th)
    return a.cos().float().to(dev), a.sin().float().to(dev)


def rope(x, cos, sin):
    """Pair rotation in float32, each operation rounded, result in ``x``'s dtype; ``cos`` ``[B, pairs]``."""
    r = 2 * cos.shape[-1]
    f = x.cpu().float()
    c, s = (t.cpu()[:, None, None] for t in (cos, sin))
    x1, x2 = f[..., :r:2], f[..., 1:r:2]
    return torch.cat((torch.stack((x1 * c - x2 * s, x1 * s + x2 * c), -1).flatten(-2), f[..., r:]), -1).to(x.dtype)


def random_cache(B, G, L, D, dev, seed=0, mag=1.0):
    from qwendopamine_amd import ops

    gen = torch.Generator().manual_seed(seed)
    c = ops.kv_cache_q4(B, G, L, D, dev)
    for codes, meta in ((c.k, c.k_meta), (c.v, c.v_meta)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=gen, dtype=torch.uint8))
        m = torch.rand(meta.shape, generator=gen)
        m[..., 0] = (0.25 + 0.2 * m[..., 0]) * mag
        m[..., 1] = -7.5 * m[..., 0] + (m[..., 1] - 0.5) * mag
        meta.copy_(m.bfloat16())
    return c


def decode_check(qkv, cos, sin, pos, cache, n_head, out, before):
    """``out`` and the updated ``cache`` against the definition from the cache ``before``."""
    B, G, L, half = cache.k.shape
    D, qpk, dt = 2 * half, n_head // G, qkv.dtype
    P = pos.cpu().expand(B).tolist()
    x = qkv.cpu().view(B, G, qpk + 2, D)
    u = torch.finfo(dt).eps / 2
    worst = 0.0
    for b, p in enumerate(P):
        if not 0 <= p < L:
            assert (out[b] == 0).all()
            assert all(same(a[b].float(), z[b].float()) for a, z in zip(cache, before))
            continue
        qk = rope(x[b:b + 1, :, :-1], cos[p][None] if cos.shape[0] > 1 else cos, sin[p][None] if sin.shape[0] > 1 else sin)[0]
        for codes, meta, old_c, old_m, new in ((cache.k, cache.k_meta, before[0], before[1], qk[:, -1]),
                                               (cache.v, cache.v_meta, before[2], before[3], x[b, :, -1])):
            n, m = quantise(new)
            assert torch.equal(unpack(codes[b, :, p].cpu()), n) and same(meta[b, :, p].cpu().float(), m.float())
            rest = torch.arange(L) != p
            assert torch.equal(codes[b].cpu()[:, rest], old_c[b].cpu()[:, rest])
            assert same(meta[b].cpu()[:, rest].float(), old_m[b].cpu()[:, rest].float())
        K, V = (values(c[b, :, :p + 1], m[b, :, :p + 1]) for c, m in (cache[:2], cache[2:]))
        q = qk[:, :-1].double()
        S = q @ K.transpose(1, 2) / math.sqrt(D)
        W = torch.softmax(S, -1)
        O = W @ V
        # Rounding of the output; P in 16 bits against values held as 1 + n / 16 (at most 32 scale
        # and the minimum); scores as float32 sums of q times at most 32 scale.
        big = [(32 * m[b, :, :p + 1, :, 0].double() + m[b, :, :p + 1, :, 1].double().abs()).cpu().amax(-1) for m in
               (cache.k_meta, cache.v_meta)]
        slack = 4 * D * 2.0 ** -24 * float((q.abs().sum(-1)[:, :, None] * big[0][:, None, :]).max()) / math.sqrt(D) + 2.0 ** -20
        bound = u * O.abs() + (2.0 ** -16 + slack) * (W * big[1][:, None, :]).sum(-1, keepdim=True) + torch.finfo(dt).smallest_normal * u
        e = (out[b].view(G, qpk, D).cpu().double() - O).abs()
        assert e.isfinite().all()
        worst = max(worst, float((e / bound).max()))
    print(f"  error / bound {worst:.2f}", flush=True)
    assert worst <= 1.0


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("B,G,qpk,D,L,P", [
    (1, 1, 1, 64, 1, [0]),
    (1, 2, 1, 128, 5, [4]),
    (2, 2, 4, 64, 40, [0, 39]),
    (3, 1, 16, 128, 300, [31, 32, 127]),
    (2, 4, 3, 64, 1000, [128, 999]),
    (4, 2, 2, 128, 513, [512, 0, 255, 256]),
    (1, 3, 7, 64, 4099, [4098]),
    (1, 1, 8, 128, 20000, [19990]),
    (5, 2, 4, 64, 77, [-1, 5, 77, 10 ** 10, -10 ** 10]),   # outside: zeros, the cache left alone
    (4, 1, 2, 128, 3000, [2999, -5, 3000, 700]),           # the same, with shares
    (2, 1, 12, 64, 5000, [4999, 1]),                       # more than eight heads, ragged shares
])
def test_decode_matches_float64(gpu_device, B, G, qpk, D, L, P, dt):
    from qwendopamine_amd import ops

    print(f"[case] q4 decode B{B} G{G} qpk{qpk} D{D} L{L} at {P} {dt}", flush=True)
    H = G * qpk
    cache = random_cache(B, G, L, D, gpu_device, seed=L)
    before = [t.clone() for t in cache]
    gen = torch.Generator().manual_seed(1)
    qkv = torch.randn(B, 1, (H + 2 * G) * D, generator=gen).to(dt).to(gpu_device)
    cos, sin = tables(max(L, 2), D, D // 2, gpu_device)
    pos = torch.tensor(P, device=gpu_device)
    out = ops.attention_decode_q4(qkv, cos, sin, pos, cache, H)
    torch.cuda.synchronize()
    decode_check(qkv, cos, sin, pos, cache, H, out, before)


@pytest.mark.parametrize("pairs", [0, 8, 32])
def test_decode_partial_rotation_and_single_row(gpu_device, pairs):
    """Fewer rotated channels; the token's own row of the tables; one position for all sequences."""
    from qwendopamine_amd import ops

    B, G, qpk, D, L = 3, 2, 2, 64, 90
    cache = random_cache(B, G, L, D, gpu_device, seed=7)
    before = [t.clone() for t in cache]
    qkv = torch.randn(B, 1, (qpk + 2) * G * D, generator=torch.Generator().manual_seed(2)).to(BF).to(gpu_device)
    cos, sin = tables(L, D, pairs, gpu_device)
    pos = torch.tensor([70], device=gpu_device)
    one = [t.clone() for t in cache]
    a = ops.attention_decode_q4(qkv, cos, sin, pos, cache, G * qpk)
    b = ops.attention_decode_q4(qkv, cos[70:71], sin[70:71], pos, ops.KVCacheQ4(*one), G * qpk)
    torch.cuda.synchronize()
    decode_check(qkv, cos, sin, pos, cache, G * qpk, a, before)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(one, cache))


def test_decode_strided_positions_and_wide_values(gpu_device):
    """Positions as a column of a wider tensor; scales of 200 and scores of several hundred."""
    from qwendopamine_amd import ops

    B, G, qpk, D, L = 2, 2, 2, 128, 600
    cache = random_cache(B, G, L, D, gpu_device, seed=9, mag=40.0)
    before = [t.clone() for t in cache]
    qkv = torch.randn(B, 1, (qpk + 2) * G * D, generator=torch.Generator().manual_seed(3)).to(BF).to(gpu_device)
    cos, sin = tables(L, D, D // 2, gpu_device)
    pos = torch.tensor([[599, 1], [17, 2]], device=gpu_device)[:, 0]
    out = ops.attention_decode_q4(qkv, cos, sin, pos, cache, G * qpk)
    torch.cuda.synchronize()
    decode_check(qkv, cos, sin, pos, cache, G * qpk, out, before)


def test_decode_garbage_past_the_position_is_not_seen(gpu_device):
    """NaN scales after the position (never written rows) leave the result alone; one before makes it NaN."""
    from qwendopamine_amd import ops

    B, G, qpk, D, L = 1, 2, 1, 64, 200
    for p in (31, 64, 100):
        a, b = (random_cache(B, G, L, D, gpu_device, seed=4) for _ in range(2))
        b.k_meta[:, :, p + 1:], b.v_meta[:, :, p + 1:] = float("nan"), float("inf")
        qkv = torch.randn(B, 1, (qpk + 2) * G * D, generator=torch.Generator().manual_seed(5)).to(FP).to(gpu_device)
        cos, sin = tables(L, D, 32, gpu_device)
        pos = torch.tensor([p], device=gpu_device)
        o = ops.attention_decode_q4(qkv, cos, sin, pos, b, G * qpk)
        assert torch.equal(ops.attention_decode_q4(qkv, cos, sin, pos, a, G * qpk), o)
    a.k_meta[0, 0, 3] = float("nan")
    o = ops.attention_decode_q4(qkv, cos, sin, pos, a, G * qpk)
    assert o[0, 0].isnan().all() and o[0, 1].isfinite().all()


def test_decode_token_that_is_not_finite(gpu_device):
    from qwendopamine_amd import ops

    G, D, L = 2, 64, 50
    cache = random_cache(1, G, L, D, gpu_device)
    before = [t.clone() for t in cache]
    qkv = torch.ones(1, 1, 3 * G * D, dtype=BF, device=gpu_device)
    qkv[0, 0, 2 * D + 5] = float("inf")  # v of group 0
    cos, sin = tables(L, D, 32, gpu_device)
    o = ops.attention_decode_q4(qkv, cos, sin, torch.tensor([9], device=gpu_device), cache, G)
    assert o[0, 0].isnan().all() and o[0, 1].isfinite().all() and cache.v_meta[0, 0, 9].isnan().all()
    assert torch.equal(before[2][0, 1, :9], cache.v[0, 1, :9]) and not cache.v_meta[0, 1].isnan().any()


@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("B,T,G,D,L,start", [
    (1, 1, 1, 64, 1, None), (2, 7, 3, 128, 20, None), (2, 33, 2, 64, 40, [5, 0]), (3, 9, 1, 192, 12, [-4, 3, 11]),
    (1, 100, 2, 64, 30, [10 ** 10]), (2, 64, 2, 128, 64, [0]),
])
def test_store_and_load_code_for_code(gpu_device, B, T, G, D, L, start, dt):
    from qwendopamine_amd import ops

    print(f"[case] q4 store B{B} T{T} G{G} D{D} L{L} from {start} {dt}", flush=True)
    gen = torch.Generator().manual_seed(T)
    k, v = (torch.randn(B, T, G, D, generator=gen) * 3 for _ in range(2))
    k[0, 0, 0, :64] = 0.7          # a constant group
    v[0, 0, 0, 3] = 1000.0         # an outlier
    v[0, T // 2, 0, :64] = 0.0
    if T > 5:
        k[0, 5, G - 1, 1] = float("nan")
        v[0, 5, G - 1, 2] = float("-inf")
    k, v = k.to(dt).to(gpu_device), v.to(dt).to(gpu_device)
    cache = random_cache(B, G, L, D, gpu_device, seed=1) if D != 192 else ops.kv_cache_q4(B, G, L, D, gpu_device)
    before = [t.clone() for t in cache]
    st = None if start is None else torch.tensor(start, device=gpu_device)
    ops.kv_cache_q4_store(cache, k, v, st)
    torch.cuda.synchronize()
    first = [0] * B if start is None else (start * B if len(start) == 1 else start)
    want = [t.cpu().clone() for t in before]
    for x, c, m in ((k, 0, 1), (v, 2, 3)):
        n, meta = quantise(x.transpose(1, 2))
        n = n[..., 0::2] | (n[..., 1::2] << 4)
        for b in range(B):
            for t in range(T):
                if 0 <= first[b] + t < L:
                    want[c][b, :, first[b] + t], want[m][b, :, first[b] + t] = n[b, :, t], meta[b, :, t]
    for a, z in zip(cache, want):
        assert same(a.cpu().float(), z.float())
    for out_dt in (F32, dt):
        lk, lv = ops.kv_cache_q4_load(cache, st, T, out_dt)
        for y, c, m in ((lk, 0, 1), (lv, 2, 3)):
            z = values(want[c], want[m], F32)
            for b in range(B):
                for t in range(T):
                    w = z[b, :, first[b] + t] if 0 <= first[b] + t < L else torch.zeros(G, D)
                    assert same(y[b, t].cpu().float(), w.to(out_dt).float())


def test_store_strides(gpu_device):
    from qwendopamine_amd import ops

    B, T, G, D = 2, 11, 3, 64
    x = torch.randn(B, T, 2 * G * D, generator=torch.Generator().manual_seed(8)).to(BF).to(gpu_device)
    k, v = (z.view(B, T, G, D) for z in x.split(G * D, -1))
    a, b = ops.kv_cache_q4(B, G, T, D, gpu_device), ops.kv_cache_q4(B, G, T, D, gpu_device)
    ops.kv_cache_q4_store(a, k, v)
    ops.kv_cache_q4_store(b, k.transpose(1, 2).contiguous().transpose(1, 2), torch.stack((v, v), -1)[..., 0])
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_prompt_in_pieces_then_decode(gpu_device):
    """Prompt pieces stored, read back and attended with ``attention``, then tokens with
    ``attention_decode_q4``: the same as attention over the values the whole cache stands for."""
    from qwendopamine_amd import ops

    B, G, qpk, D, L, dt = 2, 2, 2, 64, 140, BF
    H = G * qpk
    gen = torch.Generator().manual_seed(6)
    cos, sin = tables(L, D, D // 2, gpu_device)
    cache = ops.kv_cache_q4(B, G, L, D, gpu_device)
    at = 0
    for T in (64, 37, 1, 30):
        q, k, v = (torch.randn(B, T, h, D, generator=gen).to(dt).to(gpu_device) for h in (H, G, G))
        ops.kv_cache_q4_store(cache, k, v, torch.tensor([at], device=gpu_device))
        at += T
        K, V = ops.kv_cache_q4_load(cache, None, at, dt)
        o = ops.attention(q, K, V)
        S = torch.einsum("bigrd,bjgd->bgrij", q.double().cpu().view(B, T, G, qpk, D), K.double().cpu()) / 8
        S = S.masked_fill(torch.arange(at) > torch.arange(T)[:, None] + at - T, float("-inf"))
        want = torch.einsum("bgrij,bjgd->bigrd", S.softmax(-1), V.double().cpu()).reshape(B, T, H, D)
        # P and the output rounded to bf16, against values of up to about 4.
        assert float((o.cpu().double() - want).abs().max()) <= 2.0 ** -8 * 2 * float(V.double().abs().max())
    for step in range(3):
        before = [t.clone() for t in cache]
        qkv = torch.randn(B, 1, (H + 2 * G) * D, generator=gen).to(dt).to(gpu_device)
        pos = torch.full((B,), at + step, device=gpu_device)
        out = ops.attention_decode_q4(qkv, cos, sin, pos, cache, H)
        torch.cuda.synchronize()
        decode_check(qkv, cos, sin, pos, cache, H, out, before)


def test_decode_captured_graphs_do_not_share_state(gpu_device):
    """Two captured decode steps of different shapes, replayed in turn with moving positions and eager
    steps between: the same caches and outputs as eager steps alone."""
    from qwendopamine_amd import ops

    def make(B, G, qpk, D, L, seed):
        cache = random_cache(B, G, L, D, gpu_device, seed=seed)
        twin = ops.KVCacheQ4(*(t.clone() for t in cache))
        qkv = torch.randn(B, 1, (qpk + 2) * G * D, generator=torch.Generator().manual_seed(seed)).to(BF).to(gpu_device)
        cos, sin = tables(L, D, D // 2, gpu_device)
        pos = torch.arange(B, device=gpu_device) + 40
        args = (qkv, cos, sin, pos)
        ops.attention_decode_q4(*args, ops.KVCacheQ4(*(t.clone() for t in cache)), G * qpk)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.attention_decode_q4(*args, cache, G * qpk)
        return g, args, cache, twin, out, G * qpk

    sets = [make(2, 2, 2, 64, 3000, 1), make(3, 1, 8, 128, 2000, 2)]
    for step in range(4):
        for g, args, cache, twin, out, H in sets:
            g.replay()
        for g, args, cache, twin, out, H in sets:
            want = ops.attention_decode_q4(*args, twin, H)
            assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(cache, twin))
            args[0].mul_(-0.9)
            args[3].add_(300)
        torch.cuda.synchronize()
