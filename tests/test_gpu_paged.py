"""The paged cache: ``ops.kv_cache_paged_append`` against the pass over plain rows, ``ops.attention_paged`` against
float64 attention: pages in any order, shared, missing and ending inside a tile, every sequence at its own
position, pieces from one token to several tiles, padding, shares of long contexts, graphs and streams."""

from __future__ import annotations

import math

import pytest
import torch

from qwendopamine_amd import ops

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def tables(rows, pairs, dev):
    th = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))
    a = torch.outer(torch.arange(rows, dtype=torch.float64), th)
    return a.cos().float().to(dev), a.sin().float().to(dev)


def make_cache(B, G, S, D, N, dt, dev, seed=0, spare=3, fill=True):
    """Pages in random order, some in nobody's table."""
    g = torch.Generator().manual_seed(seed)
    P = B * N + spare
    table = torch.randperm(P, generator=g)[:B * N].view(B, N).to(torch.int32).to(dev)
    k, v = (torch.randn(P, G, S, D, generator=g).to(dt).to(dev) if fill else
            torch.full((P, G, S, D), float("nan"), dtype=dt, device=dev) for _ in range(2))
    return ops.KVCachePaged(k, v, table)


def page_of(cache, b, j):
    """The page of position ``j`` of sequence ``b``, or None."""
    S, P, N = cache.k.shape[2], cache.k.shape[0], cache.table.shape[1]
    if not 0 <= j < N * S:
        return None
    p = int(cache.table[b, j // S])
    return p if 0 <= p < P else None


# ---- append ----

def expected_append(qkv, cos, sin, pos, cache, H, wq, wk, lengths):
    """By the pass over rows at each token's position (its own test holds it to float64), and a copy."""
    B, T, _ = qkv.shape
    P, G, S, D = cache.k.shape
    at = pos.expand(B)[:, None] + torch.arange(T, device=qkv.device)
    n = torch.full((B,), T) if lengths is None else lengths.cpu()
    t = torch.arange(T)[None]
    cap = cache.table.shape[1] * S
    there = (t < n[:, None]).to(qkv.device) & (pos.expand(B)[:, None] >= 0) & (at < min(cap, cos.shape[0]))
    q, k, v = ops.qkv_norm_rope(qkv, cos, sin, H, G, wq, wk, 1e-5, torch.where(there, at, -1))
    kp, vp = cache.k.clone(), cache.v.clone()
    for b in range(B):
        for i in range(T):
            p = page_of(cache, b, int(at[b, i])) if there[b, i] else None
            if p is not None:
                kp[p, :, int(at[b, i]) % S], vp[p, :, int(at[b, i]) % S] = k[b, i], v[b, i]
    return q, kp, vp


APPENDS = [  # B, T, H, G, D, S, N, pairs, norm, dt
    (1, 1, 1, 1, 64, 16, 1, 32, False, BF),
    (3, 1, 8, 2, 128, 16, 9, 64, True, BF),
    (4, 7, 4, 4, 64, 48, 4, 32, True, FP),
    (2, 65, 7, 1, 64, 32, 5, 8, True, BF),
    (2, 33, 6, 2, 96, 64, 2, 48, False, F32),
    (2, 20, 2, 2, 256, 16, 7, 128, True, F32),
    (5, 3, 64, 8, 128, 256, 1, 64, True, FP),
]


@pytest.mark.parametrize("case", APPENDS, ids=str)
@pytest.mark.parametrize("padded", [False, True])
def test_append(gpu_device, case, padded):
    B, T, H, G, D, S, N, pairs, norm, dt = case
    g = torch.Generator().manual_seed(5)
    cache = make_cache(B, G, S, D, N, dt, gpu_device, 6)
    cap = N * S
    qkv = torch.randn(B, T, (H + 2 * G) * D, generator=g).to(dt).to(gpu_device)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(dt).to(gpu_device) if norm else None for _ in range(2))
    cos, sin = tables(cap + 2, pairs, gpu_device)
    pos = torch.tensor([(cap - T + 2 + 5 * b) % (cap + 3) - (b == 3) * 1000 for b in range(B)], device=gpu_device)
    lengths = torch.tensor([(T * (b + 1)) // B - (b == 0) for b in range(B)], device=gpu_device) if padded else None
    want = expected_append(qkv, cos, sin, pos, cache, H, wq, wk, lengths)
    q = ops.kv_cache_paged_append(qkv, cos, sin, pos, cache, H, wq, wk, 1e-5, lengths)
    for name, a, b in zip("qkv", (q, cache.k, cache.v), want):
        assert torch.equal(a, b), name


def test_append_missing_pages_and_tables(gpu_device):
    """No page: q is given, nothing stored.  Tables shorter than the cache: no rotation, no token."""
    B, T, H, G, D, S, N = 3, 40, 4, 2, 64, 16, 4
    cache = make_cache(B, G, S, D, N, BF, gpu_device, 7)
    cache.table[0, 1] = -1
    cache.table[1, 0] = cache.k.shape[0]
    cache.table[2, 2] = 2 ** 31 - 1
    cache.table[1, 3] = -2 ** 31
    qkv = torch.randn(B, T, (H + 2 * G) * D, generator=torch.Generator().manual_seed(8)).to(BF).to(gpu_device)
    cos, sin = tables(50, 32, gpu_device)
    pos = torch.tensor([0, 20, 12], device=gpu_device)
    want = expected_append(qkv, cos, sin, pos, cache, H, None, None, None)
    assert (want[0][1, 30:] == 0).all() and (want[0][0] != 0).any(-1).all()
    q = ops.kv_cache_paged_append(qkv, cos, sin, pos, cache, H)
    for name, a, b in zip("qkv", (q, cache.k, cache.v), want):
        assert torch.equal(a, b), name


def test_append_lengths_past_32_bits(gpu_device):
    B, T, H, G, D, S, N = 4, 3, 2, 2, 64, 16, 2
    cache = make_cache(B, G, S, D, N, BF, gpu_device, 24)
    qkv = torch.randn(B, T, (H + 2 * G) * D, generator=torch.Generator().manual_seed(25)).to(BF).to(gpu_device)
    cos, sin = tables(N * S, 32, gpu_device)
    lengths = torch.tensor([-2 ** 40 + 2, 2 ** 40, 2, -2 ** 62 + 3], device=gpu_device)
    pos = torch.tensor([0, 5, 2 ** 33 + 1, 2], device=gpu_device)
    want = expected_append(qkv, cos, sin, pos, cache, H, None, None, lengths.clamp(0, T))
    q = ops.kv_cache_paged_append(qkv, cos, sin, pos, cache, H, lengths=lengths)
    for name, a, b in zip("qkv", (q, cache.k, cache.v), want):
        assert torch.equal(a, b), name


def test_append_layouts(gpu_device):
    """Column ranges, one position for all, a table that is a column range, int32 lengths."""
    B, T, H, G, D, S, N = 2, 5, 4, 2, 64, 16, 3
    cache = make_cache(B, G, S, D, N, BF, gpu_device, 9)
    wide = torch.full((B, N + 4), -7, dtype=torch.int32, device=gpu_device)
    wide[:, 2:2 + N] = cache.table
    cache = cache._replace(table=wide[:, 2:2 + N])
    W = (H + 2 * G) * D
    qkv = torch.randn(B, T, W + 128, generator=torch.Generator().manual_seed(10)).to(BF).to(gpu_device)[..., 64:64 + W]
    cos, sin = tables(N * S, 32, gpu_device)
    pos = torch.tensor([17], device=gpu_device)
    lengths = torch.tensor([5, 2], dtype=torch.int32, device=gpu_device)
    want = expected_append(qkv, cos, sin, pos, cache, H, None, None, lengths)
    q = ops.kv_cache_paged_append(qkv, cos, sin, pos, cache, H, lengths=lengths)
    for name, a, b in zip("qkv", (q, cache.k, cache.v), want):
        assert torch.equal(a, b), name


# ---- attention ----

def expected_attention(q, cache, pos, lengths=None, scale=None):
    """float64 value and bound.  Scores: D products and sums, within (D + 4) u of sum |q k| scale; a probability is
    off by that, by two roundings (two parts: 2^-17 of it in bf16) and by its sums, L / 32 + 64 additions in a
    chain; the result is rounded once.  The exponential is the hardware's, 2 u and u of its argument (at most
    the scores' spread, 150 octaves where a probability still counts).  Half a step of fp16 is 2^-25 under 2^-14.
    Groups of more than 16 rows (heads of 64 channels: 32): probabilities are rounded once, each is off by half a
    step of itself."""
    B, T, H, D = q.shape
    G, S = cache.k.shape[1], cache.k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    f = torch.finfo(q.dtype)
    u = 2.0 ** -24
    pos = pos.expand(B).tolist()
    n = [T] * B if lengths is None else lengths.tolist()
    cap = cache.table.shape[1] * S
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.full(q.shape, 1e-30, dtype=torch.float64)
    kc, vc, qc = cache.k.cpu().double(), cache.v.cpu().double(), q.cpu().double()
    for b in range(B):
        for t in range(T):
            last = pos[b] + t
            if t >= n[b] or pos[b] < 0 or last >= cap:
                continue
            at = [(page_of(cache, b, j), j) for j in range(0, last + 1, 16)]
            rows = [(p, (j + i) % S) for p, j in at if p is not None for i in range(16) if j + i <= last]
            if not rows:
                continue
            p, r = (torch.tensor(x) for x in zip(*rows))
            k, v = kc[p, :, r], vc[p, :, r]  # [keys, G, D]
            x = qc[b, t].view(G, H // G, D)
            s = torch.einsum("grd,jgd->grj", x, k) * scale
            w = torch.softmax(s, -1)
            o = torch.einsum("grj,jgd->grd", w, v)
            off = (D + 4) * u * (torch.einsum("grd,jgd->grj", x.abs(), k.abs()) * scale).amax(-1, keepdim=True)
            rel = 2 * off + (f.eps / 2 if T * (H // G) > (32 if D == 64 else 16) else 2.0 ** -16) + (len(rows) / 32 + 64 + 4 + 150) * u
            out[b, t] = o.reshape(H, D)
            tol[b, t] = (f.eps / 2 * o.abs().clamp_min(f.tiny) + rel * torch.einsum("grj,jgd->grd", w, v.abs())).reshape(H, D) + 1e-30
    return out.to(q.device), tol.to(q.device)


def check(o, want):
    ref, tol = want
    err = (o.double() - ref).abs()
    assert (err <= tol).all(), f"{float((err / tol).max()):.3f} of the bound"


def queries(B, T, H, D, dt, dev, seed=1, scale=1.0):
    return (torch.randn(B, T, H, D, generator=torch.Generator().manual_seed(seed)) * scale).to(dt).to(dev)


ATTN = [  # B, T, H, G, D, S, N
    (1, 1, 1, 1, 64, 16, 1),
    (3, 1, 2, 2, 64, 16, 7),
    (2, 1, 8, 2, 128, 48, 5),
    (2, 1, 16, 1, 64, 64, 4),
    (2, 1, 20, 1, 128, 32, 6),
    (2, 1, 40, 1, 64, 16, 9),
    (2, 3, 4, 4, 128, 16, 12),
    (2, 5, 14, 2, 64, 32, 8),
    (1, 17, 2, 2, 64, 16, 11),
    (2, 33, 4, 2, 128, 64, 3),
    (1, 130, 7, 1, 64, 16, 17),
    (1, 70, 3, 3, 128, 256, 1),
]


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("case", ATTN, ids=str)
def test_attention(gpu_device, case, dt):
    """From the first positions to the last, those outside among them; what lies past a sequence's last token in its
    pages, and in pages of nobody, is NaN."""
    B, T, H, G, D, S, N = case
    cap = N * S
    q = queries(B, T, H, D, dt, gpu_device)
    for first in sorted({0, 1, 15, 16, 31, 32, max(0, cap - T), cap - 1, cap, -1}):
        cache = make_cache(B, G, S, D, N, dt, gpu_device, 11)
        pos = torch.tensor([max(-1, first - 7 * b) if first >= 0 else first for b in range(B)], device=gpu_device)
        used = torch.zeros(cache.k.shape[0], S, dtype=torch.bool)
        for b in range(B):
            for j in range(min(cap, int(pos[b]) + T) if 0 <= int(pos[b]) < cap else 0):
                used[page_of(cache, b, j), j % S] = True
        for x in (cache.k, cache.v):
            x.transpose(1, 2)[~used.to(gpu_device)] = float("nan")
        o = ops.attention_paged(q, cache, pos)
        check(o, expected_attention(q, cache, pos))


@pytest.mark.parametrize("T,H,G,D", [(1, 4, 2, 64), (9, 4, 1, 128), (40, 4, 2, 64)])
def test_padded_batch(gpu_device, T, H, G, D):
    B, S, N = 5, 16, 8
    cache = make_cache(B, G, S, D, N, BF, gpu_device, 12)
    q = queries(B, T, H, D, BF, gpu_device, 2)
    pos = torch.tensor([60, 0, 33, 5, 100], device=gpu_device)
    lengths = torch.tensor([T, 0, max(1, T // 2), -3, T + 9], device=gpu_device)
    q[2, max(1, T // 2):] = float("nan")
    o = ops.attention_paged(q, cache, pos, lengths)
    check(o, expected_attention(q, cache, pos, lengths))
    assert (o[1] == 0).all() and (o[3] == 0).all()


@pytest.mark.parametrize("T", [1, 20])
def test_missing_pages(gpu_device, T):
    """Positions without a page are not seen, whatever lies in page 0; a sequence without any page gives zeros."""
    B, H, G, D, S, N = 4, 4, 2, 64, 32, 6
    cache = make_cache(B, G, S, D, N, BF, gpu_device, 13)
    cache.table[cache.table == 0] = 1  # page 0 is nobody's
    cache.k[0] = float("nan")
    cache.v[0] = float("inf")
    P = cache.k.shape[0]
    cache.table[0, 0] = -1
    cache.table[1, 2] = P
    cache.table[1, 4] = -2 ** 31
    cache.table[2, 5] = 2 ** 31 - 1
    cache.table[3] = -1
    q = queries(B, T, H, D, BF, gpu_device, 3)
    pos = torch.tensor([150, 163, 170, 100], device=gpu_device)
    o = ops.attention_paged(q, cache, pos)
    check(o, expected_attention(q, cache, pos))
    assert (o[3] == 0).all()
    cache.table[0, :] = -1
    cache.table[0, 5] = 3
    o = ops.attention_paged(q, cache, torch.tensor([3, 160, 170, 190], device=gpu_device))
    assert (o[0] == 0).all() and o.isfinite().all()


def test_shared_pages(gpu_device):
    """Sequences that read a prefix in common, and a page twice in one sequence."""
    B, T, H, G, D, S, N = 3, 2, 8, 2, 64, 16, 6
    cache = make_cache(B, G, S, D, N, FP, gpu_device, 14)
    cache.table[1, :3] = cache.table[0, :3]
    cache.table[2, 1] = cache.table[2, 0]
    q = queries(B, T, H, D, FP, gpu_device, 4)
    pos = torch.tensor([80, 50, 94], device=gpu_device)
    check(ops.attention_paged(q, cache, pos), expected_attention(q, cache, pos))


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("B,T,H,G,D,S,L", [(1, 1, 4, 1, 64, 16, 9000), (2, 1, 6, 2, 128, 48, 5000), (1, 3, 8, 1, 128, 64, 3000),
                                           (1, 50, 2, 1, 64, 32, 2500)])
def test_long_contexts(gpu_device, B, T, H, G, D, S, L, dt):
    """Shares of the positions that a second launch joins, of sequences of very unequal lengths."""
    N = (L + S - 1) // S
    cache = make_cache(B, G, S, D, N, dt, gpu_device, 15)
    q = queries(B, T, H, D, dt, gpu_device, 5)
    assert ops.nat.load().gdn2_attn_paged_workspace_size(B, T, G, H // G, D, N * S) > 0
    for pos in ([L - T] * B, [0] * B, [700 + 3000 * b for b in range(B)]):
        pos = torch.tensor(pos, device=gpu_device)
        o = ops.attention_paged(q, cache, pos)
        check(o, expected_attention(q, cache, pos))
        assert torch.equal(o, ops.attention_paged(q, cache, pos))


@pytest.mark.parametrize("T,H,G,D", [(1, 2, 1, 64), (4, 8, 4, 128), (5, 6, 1, 64)])
def test_many_sequences(gpu_device, T, H, G, D):
    """More sequences than a wave has lanes, in runs that begin and end within them: empty ones, padding, positions
    outside, from one position to over a thousand."""
    B, S, N = 150, 16, 70
    g = torch.Generator().manual_seed(18)
    P = 400
    cache = make_cache(1, G, S, D, P - 3, BF, gpu_device, 19)._replace(
        table=torch.randint(0, P, (B, N), generator=g).to(torch.int32).to(gpu_device))  # pages in common
    assert ops.nat.load().gdn2_attn_paged_workspace_size(B, T, G, H // G, D, N * S) > 0
    q = queries(B, T, H, D, BF, gpu_device, 8)
    pos = torch.randint(-40, N * S + 40, (B,), generator=g)
    pos[:9] = torch.tensor([0, N * S - 1, N * S - T, -1, N * S, 127, 128, 255, 1])
    lengths = torch.randint(-1, T + 2, (B,), generator=g)
    lengths[70:80] = 0
    lengths[5], lengths[100], lengths[101] = -2 ** 40 + 3, 2 ** 40 + 1, -2 ** 62 + 1  # past 32 bits
    pos, lengths = pos.to(gpu_device), lengths.to(gpu_device)
    check(ops.attention_paged(q, cache, pos, lengths), expected_attention(q, cache, pos, lengths))
    none = ops.attention_paged(q, cache, torch.full_like(pos, -1), lengths)
    assert (none == 0).all()


def test_very_many_sequences(gpu_device):
    """One workgroup for each where there are many times more than the card holds."""
    B, T, H, G, D, S, N = 4200, 1, 2, 1, 64, 16, 70
    g = torch.Generator().manual_seed(20)
    cache = make_cache(1, G, S, D, 97, BF, gpu_device, 23)._replace(
        table=torch.randint(0, 100, (B, N), generator=g).to(torch.int32).to(gpu_device))
    assert ops.nat.load().gdn2_attn_paged_workspace_size(B, T, G, H // G, D, N * S) == 0
    q = queries(B, T, H, D, BF, gpu_device, 9)
    pos = torch.randint(0, N * S, (B,), generator=g).to(gpu_device)
    o = ops.attention_paged(q, cache, pos)
    for at in (0, 2000, 4180):
        part = slice(at, at + 20)
        check(o[part], expected_attention(q[part], cache._replace(table=cache.table[part]), pos[part]))


def test_sharp_scores(gpu_device):
    """Scores far apart and far from zero: one key carries nearly all, references move late in the walk; and
    probabilities that underflow."""
    B, T, H, G, D, S, N = 2, 3, 4, 2, 64, 16, 40
    for dt in (BF, FP):
        cache = make_cache(B, G, S, D, N, dt, gpu_device, 16)
        ramp = torch.linspace(-4, 4, N * S, device=gpu_device)
        for b in range(B):
            for i in range(N):
                cache.k[int(cache.table[b, i])] += ramp[i * S:i * S + S, None].to(dt)
        q = queries(B, T, H, D, dt, gpu_device, 6, 2.0)
        pos = torch.tensor([N * S - 3, 333], device=gpu_device)
        for scale in (None, 1e-6, 3.0):
            check(ops.attention_paged(q, cache, pos, scale=scale), expected_attention(q, cache, pos, scale=scale))


def test_query_layouts(gpu_device):
    B, T, H, G, D, S, N = 2, 4, 4, 2, 64, 16, 5
    cache = make_cache(B, G, S, D, N, BF, gpu_device, 17)
    pos = torch.tensor([9, 70], device=gpu_device)
    q = queries(B, T, H, D, BF, gpu_device, 7)
    want = ops.attention_paged(q, cache, pos)
    wide = torch.zeros(B, T, H * D + 64, dtype=BF, device=gpu_device)
    for x in (wide[..., 8:8 + H * D].view(B, T, H, D), wide[..., 3:3 + H * D].view(B, T, H, D),
              torch.zeros(B, H, T, D, dtype=BF, device=gpu_device).transpose(1, 2)):
        x.copy_(q)
        assert torch.equal(ops.attention_paged(x, cache, pos), want)
    one = ops.attention_paged(q, cache, torch.tensor([9], device=gpu_device))
    assert torch.equal(one[0], want[0])
    spread = torch.tensor([[9, 1], [70, 2]], device=gpu_device)[:, 0]
    assert torch.equal(ops.attention_paged(q, cache, spread), want)
    assert ops.attention_paged(q[:, :0], cache, pos).shape == (B, 0, H, D)


def test_offsets_past_32_bits(gpu_device):
    """Pages that begin past 2^32 bytes of the cache."""
    G, S, D = 8, 256, 128
    P = (9 << 30) // (2 * G * S * D) // 2  # 4.5 GiB of keys, and of values
    k = torch.zeros(P, G, S, D, dtype=BF, device=gpu_device)
    v = torch.zeros_like(k)
    table = torch.tensor([[P - 1, 0, P - 2], [1, P - 3, 2]], dtype=torch.int32, device=gpu_device)
    cache = ops.KVCachePaged(k, v, table)
    B, H, n = 2, 8, 600
    cos, sin = tables(3 * S, 64, gpu_device)
    qkv = torch.randn(B, n, (H + 2 * G) * D, generator=torch.Generator().manual_seed(3)).to(BF).to(gpu_device)
    zero = torch.tensor([0], device=gpu_device)
    q = ops.kv_cache_paged_append(qkv, cos, sin, zero, cache, H)
    small = ops.KVCachePaged(torch.zeros(6, G, S, D, dtype=BF, device=gpu_device),
                             torch.zeros(6, G, S, D, dtype=BF, device=gpu_device),
                             torch.arange(6, dtype=torch.int32, device=gpu_device).view(2, 3))
    q2 = ops.kv_cache_paged_append(qkv, cos, sin, zero, small, H)
    assert torch.equal(q, q2)
    assert torch.equal(ops.attention_paged(q, cache, zero), ops.attention_paged(q2, small, zero))


def test_prompt_in_pieces_and_steps(gpu_device):
    """As they are used together: prompts of unequal lengths appended in pieces, then single tokens, against
    ``ops.attention`` over the whole sequences."""
    B, H, G, D, S = 3, 8, 2, 64, 16
    total = [200, 77, 131]
    N = 13
    g = torch.Generator().manual_seed(21)
    cache = make_cache(B, G, S, D, N, BF, gpu_device, 22, fill=False)
    qkv = torch.randn(B, 200, (H + 2 * G) * D, generator=g).to(BF).to(gpu_device)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(BF).to(gpu_device) for _ in range(2)]
    cos, sin = tables(N * S, 32, gpu_device)
    q, k, v = ops.qkv_norm_rope(qkv, cos, sin, H, G, *w)
    whole = ops.attention(q, k, v)
    got = torch.zeros_like(whole)
    done = [0] * B
    for piece in (64, 1, 50, 1, 1, 90):
        n = [min(piece, t - d) for t, d in zip(total, done)]
        part = torch.zeros(B, piece, qkv.shape[2], dtype=BF, device=gpu_device)
        for b in range(B):
            part[b, :n[b]] = qkv[b, done[b]:done[b] + n[b]]
        pos, lengths = torch.tensor(done, device=gpu_device), torch.tensor(n, device=gpu_device)
        pq = ops.kv_cache_paged_append(part, cos, sin, pos, cache, H, *w, lengths=lengths)
        o = ops.attention_paged(pq, cache, pos, lengths)
        for b in range(B):
            got[b, done[b]:done[b] + n[b]] = o[b, :n[b]]
            assert (o[b, n[b]:] == 0).all()
        done = [d + x for d, x in zip(done, n)]
    assert done == total
    # Both are float32 softmax; ops.attention rounds each probability to bf16 once (sequences past 128 tokens: half a
    # step of every term, 2^-8 of sum p |v|), and both round the result.
    p_abs = ops.attention(q, k, v.abs())
    for b in range(B):
        n = total[b]
        err = (got[b, :n].double() - whole[b, :n].double()).abs()
        bound = 2.0 ** -8 * (whole[b, :n].double().abs() * 2 + p_abs[b, :n].double() * 1.02) + 1e-6
        assert (err <= bound).all()


def test_graph_and_streams(gpu_device):
    """A step of append and attention captured once and replayed as positions advance; two captured steps of one
    cache in turn; the same on a side stream."""
    B, H, G, D, S, N = 2, 8, 2, 64, 16, 200
    g = torch.Generator().manual_seed(31)
    cos, sin = tables(N * S, 32, gpu_device)
    xs = [torch.randn(B, 1, (H + 2 * G) * D, generator=g).to(BF).to(gpu_device) for _ in range(6)]
    start = torch.tensor([5, 3000], device=gpu_device)

    def run(cache, x, pos):
        q = ops.kv_cache_paged_append(x, cos, sin, pos, cache, H)
        return ops.attention_paged(q, cache, pos)
    side = torch.cuda.Stream()
    a = make_cache(B, G, S, D, N, BF, gpu_device, 32)
    want, pos = [], start.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            want.append(run(a, x, pos))
            pos = pos + 1
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    b = make_cache(B, G, S, D, N, BF, gpu_device, 32)
    x, pos = xs[0].clone(), start.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(b, x, pos)
            pos.add_(1)
        graphs.append((graph, out))
    assert torch.equal(pos, start)
    for i in range(6):
        x.copy_(xs[i])
        graphs[i % 2][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[i % 2][1], want[i])
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_two_streams_at_once(gpu_device):
    caches = [make_cache(2, 2, 16, 128, 300, BF, gpu_device, 40 + i) for i in range(2)]
    q = [queries(2, 1, 8, 128, BF, gpu_device, 41 + i) for i in range(2)]
    pos = torch.tensor([4000, 4700], device=gpu_device)
    want = [ops.attention_paged(a, c, pos) for a, c in zip(q, caches)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.attention_paged(q[i], caches[i], pos))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
    assert math.isfinite(float(want[0].float().sum()))


@pytest.mark.parametrize("B,T,H,N", [(512, 520, 64, 34), (1 << 20, 1, 17, 1)])
def test_calls_of_many_rows(gpu_device, B, T, H, N):
    """More rows than one launch holds workgroups, in tiles and of few rows a sequence: as in smaller calls, which give
    every sequence its workgroups by the same rule."""
    G, D, S = 1, 64, 16
    assert B * T * H > 2 ** 24
    g = torch.Generator().manual_seed(70)
    cache = make_cache(1, G, S, D, 97, BF, gpu_device, 71)._replace(
        table=torch.randint(0, 100, (B, N), generator=g).to(torch.int32).to(gpu_device))
    q = queries(1, T, H, D, BF, gpu_device, 72).expand(B, T, H, D)
    pos = torch.randint(0, N * S - T + 1, (B,), generator=g).to(gpu_device)
    o = ops.attention_paged(q, cache, pos)
    for at in range(0, B, B // 4):
        part = slice(at, at + B // 4)
        assert torch.equal(o[part], ops.attention_paged(q[part], cache._replace(table=cache.table[part]), pos[part]))
    part = slice(B - 1, B)
    check(o[part], expected_attention(q[part], cache._replace(table=cache.table[part]), pos[part]))


def check_groups(o, q, cache, pos, groups):
    """Some groups' heads of every sequence against float64."""
    R = q.shape[2] // cache.k.shape[1]
    for g in groups:
        heads = slice(g * R, (g + 1) * R)
        check(o[:, :, heads], expected_attention(q[:, :, heads], cache._replace(k=cache.k[:, g:g + 1], v=cache.v[:, g:g + 1]),
                                                 pos))


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("G,D,S,T,shares", [(32, 64, 16, 40, 1), (32, 128, 64, 23, 1), (20, 64, 32, 40, 2)])
def test_tiles_look_pages_up_again(gpu_device, G, D, S, T, shares, dt):
    """A workgroup's walk over more than the 16 tiles whose pages are looked up at once: pages that are missing on either
    side of each look-up, or all of one, and last positions there.  Queries are near keys on either side, so that each
    of these carries a row."""
    B, L, P = 16, 2560, 200
    g = torch.Generator().manual_seed(50)
    cache = make_cache(1, G, S, D, P - 3, dt, gpu_device, 51)._replace(
        table=torch.randint(0, P, (B, L // S), generator=g).to(torch.int32).to(gpu_device))
    nbytes = ops.nat.load().gdn2_attn_paged_workspace_size(B, T, G, 1, D, L)
    assert nbytes == (0 if shares == 1 else 4 * shares * B * T * G * (D + 2))
    table = cache.table
    table[0, 1040 // S] = -1
    table[1, 2100 // S] = P
    table[2, 1008 // S] = table[2, 1024 // S] = -5
    table[3, 1024 // S:2048 // S] = -1
    table[4, :2304 // S] = -1
    q = queries(B, T, G, D, dt, gpu_device, 52)
    near = [(996, 1020, 1028, 1044, 1060, 2040, 2056, 2104, 2312)[t % 9] + t // 9 for t in range(T)]
    some = slice(0, 9)
    for b in range(9):
        for t, j in enumerate(near):
            p = page_of(cache, b, j)
            if p is not None:
                q[b, t] = 2 * cache.k[p, :, j % S]
    pos = torch.full((B,), L - T, device=gpu_device)
    pos[5], pos[6], pos[7], pos[8] = 1024 - T, 1025 - T, 1024, 2048 + 64 - T
    o = ops.attention_paged(q, cache, pos)
    check_groups(o[some], q[some], cache._replace(table=table[some]), pos[some], (0, G - 1))


@pytest.mark.parametrize("dt", [BF, FP], ids=str)
@pytest.mark.parametrize("R,D,T", [(2, 64, 1), (10, 64, 2), (4, 128, 2)])
def test_runs_look_pages_up_again(gpu_device, R, D, T, dt):
    """Runs of more than the 32 rounds of 128 positions whose pages are looked up at once, some over two sequences."""
    B, G, S, L, P = 4, 64, 32, 20000, 80
    N = L // S
    g = torch.Generator().manual_seed(60)
    cache = make_cache(1, G, S, D, P - 3, dt, gpu_device, 61)._replace(
        table=torch.randint(0, P, (B, N), generator=g).to(torch.int32).to(gpu_device))
    # 8 workgroups a group for all four sequences' 600 rounds.
    assert ops.nat.load().gdn2_attn_paged_workspace_size(B, T, G, R, D, N * S) == 4 * (8 + B) * G * T * R * (D + 2)
    table = cache.table
    table[0, 4100 // S] = -1
    table[0, 8192 // S] = P
    table[1, 4090 // S] = table[1, 9000 // S] = -1
    table[2, 4096 // S:12000 // S] = -1
    q = queries(B, T, G * R, D, dt, gpu_device, 62)
    pos = torch.tensor([N * S - T, 18000, N * S - T - 5, 19111], device=gpu_device)
    check_groups(ops.attention_paged(q, cache, pos), q, cache, pos, (0, G - 1))


@pytest.mark.parametrize("T,H,G,D", [(40, 4, 2, 64), (150, 8, 1, 128), (3, 8, 2, 128)])
def test_captured_pieces(gpu_device, T, H, G, D):
    """A padded piece of every sequence captured once (in tiles and their shares, or few rows in runs) and replayed as
    positions, lengths and page numbers change, with eager work between the replays."""
    B, S, N = 3, 16, 150
    g = torch.Generator().manual_seed(80)
    cos, sin = tables(N * S, D // 2, gpu_device)
    a, b = (make_cache(B, G, S, D, N, BF, gpu_device, 81) for _ in range(2))
    assert ops.nat.load().gdn2_attn_paged_workspace_size(B, T, G, H // G, D, N * S) > 0
    steps = []
    for i in range(4):
        n = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
        pos = torch.randint(0, N * S - T, (B,), generator=g)
        table = a.table.clone()
        if i == 2:
            table[0, 3], table[1] = -1, table[1].flip(0)
        steps.append((torch.randn(B, T, (H + 2 * G) * D, generator=g).to(BF).to(gpu_device), pos.to(gpu_device),
                      n.to(gpu_device), table))

    def run(cache, x, pos, n):
        q = ops.kv_cache_paged_append(x, cos, sin, pos, cache, H, lengths=n)
        return ops.attention_paged(q, cache, pos, n)
    want = [run(a._replace(table=t), x, pos, n).clone() for x, pos, n, t in steps]
    torch.cuda.synchronize()
    static = [x.clone() for x in steps[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(b._replace(table=static[3]), *static[:3])
    for w, step in zip(want, steps):
        for to, x in zip(static, step):
            to.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
        torch.randn(1000, device=gpu_device).sum()
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_append_float32_weights_and_tables_of_any_alignment(gpu_device):
    B, T, H, G, D, S, N = 2, 9, 4, 2, 64, 16, 2
    g = torch.Generator().manual_seed(85)
    qkv = torch.randn(B, T, (H + 2 * G) * D, generator=g).to(FP).to(gpu_device)
    wq, wk = ((1 + 0.2 * torch.randn(D + 1, generator=g)).to(gpu_device)[1:] for _ in range(2))
    cos, sin = tables(N * S, 32, gpu_device)
    pos = torch.tensor([20, 3], device=gpu_device)
    cache = make_cache(B, G, S, D, N, FP, gpu_device, 86)
    want = expected_append(qkv, cos, sin, pos, cache, H, wq, wk, None)
    odd = [torch.zeros(N * S * 32 + 1, device=gpu_device)[1:].view(N * S, 32).copy_(x) for x in (cos, sin)]
    assert odd[0].data_ptr() % 16 != 0
    q = ops.kv_cache_paged_append(qkv, *odd, pos, cache, H, wq, wk)
    for name, a, b in zip("qkv", (q, cache.k, cache.v), want):
        assert torch.equal(a, b), name


def test_no_sequences_no_tokens_and_inference_mode(gpu_device):
    H, G, D, S, N = 4, 2, 64, 16, 3
    cos, sin = tables(N * S, 32, gpu_device)
    for B, T in ((0, 3), (2, 0)):
        cache = make_cache(2, G, S, D, N, BF, gpu_device, 87)
        cache = cache._replace(table=cache.table[:B])
        before = cache.k.clone(), cache.v.clone()
        pos = torch.zeros(1, dtype=torch.int64, device=gpu_device)
        q = ops.kv_cache_paged_append(torch.zeros(B, T, (H + 2 * G) * D, dtype=BF, device=gpu_device), cos, sin, pos, cache, H)
        assert q.shape == (B, T, H, D) and ops.attention_paged(q, cache, pos).shape == (B, T, H, D)
        assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])
    cache, pos = make_cache(2, G, S, D, N, BF, gpu_device, 88), torch.tensor([5, 40], device=gpu_device)
    qkv = torch.randn(2, 3, (H + 2 * G) * D, generator=torch.Generator().manual_seed(89)).to(BF).to(gpu_device)
    want = expected_append(qkv, cos, sin, pos, cache, H, None, None, None)
    with torch.inference_mode():
        q = ops.kv_cache_paged_append(qkv, cos, sin, pos, cache, H)
        o = ops.attention_paged(q, cache, pos)
    assert torch.equal(q, want[0]) and torch.equal(cache.k, want[1]) and torch.equal(cache.v, want[2])
    check(o, expected_attention(q, cache, pos))


def test_sequences_of_one_table_row(gpu_device):
    """Every sequence over the same pages: a table whose rows are one row."""
    B, T, H, G, D, S, N = 4, 2, 4, 2, 64, 16, 9
    cache = make_cache(1, G, S, D, N, BF, gpu_device, 90)
    q, pos = queries(B, T, H, D, BF, gpu_device, 91), torch.tensor([3, 140, 77, 16], device=gpu_device)
    o = ops.attention_paged(q, cache._replace(table=cache.table.expand(B, N)), pos)
    assert torch.equal(o, ops.attention_paged(q, cache._replace(table=cache.table.repeat(B, 1)), pos))
    check(o, expected_attention(q, cache._replace(table=cache.table.repeat(B, 1)), pos))
