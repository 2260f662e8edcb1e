"""Performance cases of the hybrid decoder's softmax operators: attention with its gradient, token
log probabilities with their gradient, and decode attention over a key / value cache held in 4 bits.

``run`` computes every case in plain float32 torch, or, with ``own`` set, through the framework's
entry points (``ops.attention``, ``ops.token_logprobs``, ``ops.attention_decode_q4``,
``ops.kv_cache_q4_store``, ``ops.kv_cache_q4_load``).  ``exact`` restates each of them in float64.
"""

from __future__ import annotations

import math
from typing import Any

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 64  # channels that share one scale and minimum in the 4-bit cache


def listed() -> list[dict]:
    return [
        # A short prompt of one sequence, no gradient, q / k / v as column ranges of one projection: the
        # smallest call, bound by launches and latency.
        dict(name="attn-b1-t33-d64", kind="attn", B=1, Tq=33, Tk=33, H=4, G=4, D=64, dtype="bf16",
             causal=True, mask="none", seqs=0, grad=False, fused=True),
        # A right-padded batch of short texts read in both directions (scoring, embedding), training.
        dict(name="attn-train-padded-b8-t509", kind="attn", B=8, Tq=509, Tk=509, H=8, G=8, D=64, dtype="fp16",
             causal=False, mask="lengths", seqs=0, grad=True, fused=False),
        # The hybrid decoder's attention layer in a training step.
        dict(name="attn-train-b4-t2048-d64", kind="attn", B=4, Tq=2048, Tk=2048, H=16, G=16, D=64, dtype="bf16",
             causal=True, mask="none", seqs=0, grad=True, fused=False),
        # Documents of unequal lengths packed into one row, grouped heads, training.
        dict(name="attn-train-packed-n9-d128", kind="attn", B=1, Tq=7013, Tk=7013, H=16, G=4, D=128, dtype="bf16",
             causal=True, mask="packed", seqs=9, grad=True, fused=False),
        # A long-context training step, grouped heads: the largest product work.
        dict(name="attn-train-b2-t8192-d128", kind="attn", B=2, Tq=8192, Tk=8192, H=16, G=4, D=128, dtype="bf16",
             causal=True, mask="none", seqs=0, grad=True, fused=False),
        # One piece of a long prompt, prefilled over the context before it.
        dict(name="attn-prefill-1537-of-16384", kind="attn", B=1, Tq=1537, Tk=16384, H=32, G=8, D=128, dtype="bf16",
             causal=True, mask="none", seqs=0, grad=False, fused=False),
        # The log probabilities of one generated token of a small batch, with twenty alternatives.
        dict(name="logp-step-b4-v151936", kind="logp", rows=4, V=151936, dtype="bf16", top=20, grad=False),
        # The loss of a training batch over the 32000-word head, and its gradient.
        dict(name="logp-train-8192x32000", kind="logp", rows=8192, V=32000, dtype="bf16", top=0, grad=True),
        # Scoring with entropies, alternatives and a gradient over the full head in float32; some rows ignored.
        dict(name="logp-train-1000x151936-fp32", kind="logp", rows=1000, V=151936, dtype="fp32", top=5, grad=True),
        # One token of a small served batch, one attention layer of the hybrid decoder.
        dict(name="q4-decode-b4-l2304-d64", kind="decode", B=4, L=2304, H=16, G=16, D=64, dtype="bf16", ragged=False),
        # One token of a large served batch at unequal positions of long caches, grouped heads.
        dict(name="q4-decode-b32-l32768-d128", kind="decode", B=32, L=32768, H=32, G=8, D=128, dtype="bf16",
             ragged=True),
        # Prompts stored into the 4-bit cache and read back for the prompt's next piece.
        dict(name="q4-store-b4-t2048-d64", kind="store", B=4, L=2304, T=2048, G=16, D=64, dtype="bf16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["attn", "attn", "attn", "logp", "logp", "decode", "decode", "store"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    D = rng.choice([64, 128])
    if kind == "attn":
        mask = rng.choice(["none", "none", "lengths", "packed"])
        G = rng.choice([1, 2, 4, 8])
        H = G * rng.choice([1, 1, 2, 4, 8])
        Tq = min(_log_int(rng, 1, 6000), int(math.sqrt(1.0e9 / H)))
        Tk = Tq
        if mask == "none" and rng.random() < 0.4:
            Tk = max(Tq, min(Tq + _log_int(rng, 1, 16000), int(1.0e9 / (Tq * H))))
        B = 1 if mask == "packed" else max(1, min(_log_int(rng, 1, 16), int(1.0e9 / (Tq * Tk * H))))
        return dict(kind=kind, B=B, Tq=Tq, Tk=Tk, H=H, G=G, D=D, dtype=dtype,
                    causal=mask == "packed" or rng.random() < 0.75, mask=mask,
                    seqs=rng.randint(1, 12) if mask == "packed" else 0, grad=rng.random() < 0.7, fused=rng.random() < 0.3)
    if kind == "logp":
        V = _log_int(rng, 50, 160000)
        return dict(kind=kind, rows=max(1, _log_int(rng, 1, max(2, int(1.5e8 / V)))), V=V,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    top=rng.choice([0, 0, 1, 5, 20, 32]) if V >= 64 else 0, grad=rng.random() < 0.5)
    G = rng.choice([1, 2, 4, 8, 16])
    L = _log_int(rng, 1, 32768)
    B = max(1, min(_log_int(rng, 1, 64), int(8.0e6 / (L * G))))
    if kind == "decode":
        return dict(kind=kind, B=B, L=L, H=G * rng.choice([1, 2, 4, 8]), G=G, D=D, dtype=dtype, ragged=rng.random() < 0.6)
    return dict(kind=kind, B=B, L=L, T=max(1, min(L, _log_int(rng, 1, 8192))), G=G, D=D, dtype=dtype)


# ---- inputs ----

def _lengths(case: dict) -> list[int]:
    """Visible keys of each row of a padded batch: from none at all to all of them."""
    B, Tk = case["B"], case["Tk"]
    return [Tk if B == 1 else (Tk * i * i) // ((B - 1) * (B - 1)) for i in range(B)]


def _offsets(case: dict) -> list[int]:
    """Offsets of the packed sequences: unequal lengths."""
    n, total = case["seqs"], case["Tq"]
    w = [1 + (7 * i) % 5 for i in range(n)]
    cu = [0]
    for x in w:
        cu.append(cu[-1] + (total * x) // sum(w))
    cu[-1] = total
    return cu


def _positions(case: dict) -> list[int]:
    """The position of each sequence's token: near the end of the caches, or spread over them."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L - 1 - L // 10] * B
    return [min(L - 1, (L * (2 * i + 1)) // (2 * B)) for i in range(B)]


def _rope(L: int, D: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    theta = 10000.0 ** (-torch.arange(0, D, 2, device=device, dtype=torch.float64) / D)
    ang = torch.outer(torch.arange(L, device=device, dtype=torch.float64), theta)
    return ang.cos().float(), ang.sin().float()


def prepare(case: dict, seed: int) -> dict[str, Any]:
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)

    s: dict[str, Any] = dict(case=case)
    if case["kind"] == "attn":
        B, Tq, Tk, H, G, D = (case[n] for n in ("B", "Tq", "Tk", "H", "G", "D"))
        if case["fused"] and Tq == Tk:
            q, k, v = randn(B, Tq, (H + 2 * G) * D).split((H * D, G * D, G * D), dim=-1)
            q, k, v = q.view(B, Tq, H, D), k.view(B, Tk, G, D), v.view(B, Tk, G, D)
        else:
            q, k, v = randn(B, Tq, H, D), randn(B, Tk, G, D), randn(B, Tk, G, D)
        lengths = torch.tensor(_lengths(case), device=dev) if case["mask"] == "lengths" else None
        cu = torch.tensor(_offsets(case)) if case["mask"] == "packed" else None
        seg = None
        if cu is not None:
            seg = torch.bucketize(torch.arange(Tq, device=dev), cu.to(dev)[1:], right=True)
        if case["grad"]:
            q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
            s.update(do=randn(B, Tq, H, D))
        s.update(q=q, k=k, v=v, lengths=lengths, cu=cu, seg=seg)
    elif case["kind"] == "logp":
        n, V = case["rows"], case["V"]
        logits = randn(n, V, dtype=torch.float32) * 2
        targets = torch.randint(0, V, (n,), generator=gen, device=dev)
        logits[torch.arange(n, device=dev), targets] += 6  # a model that has learned something
        if n >= 1000:
            targets[::50] = -100
        s.update(logits=logits.to(dt).requires_grad_(case["grad"]), targets=targets)
        if case["grad"]:
            s.update(dlogp=-torch.rand(n, generator=gen, device=dev) / n,
                     dent=torch.rand(n, generator=gen, device=dev) * (0.01 / n))
    else:
        B, L, G, D = (case[n] for n in ("B", "L", "G", "D"))

        def codes():
            return torch.randint(0, 256, (B, G, L, D // 2), generator=gen, device=dev, dtype=torch.uint8)

        def meta():
            m = torch.rand(B, G, L, D // GROUP, 2, generator=gen, device=dev)
            m[..., 0] = 0.25 + 0.2 * m[..., 0]             # scale
            m[..., 1] = -7.5 * m[..., 0] + m[..., 1] - 0.5  # minimum
            return m.bfloat16()

        s.update(cache=(codes(), meta(), codes(), meta()))
        if case["kind"] == "decode":
            H = case["H"]
            cos, sin = _rope(L, D, dev)
            s.update(qkv=randn(B, 1, (H + 2 * G) * D), cos=cos, sin=sin,
                     pos=torch.tensor(_positions(case), device=dev))
        else:
            s.update(k=randn(B, case["T"], G, D), v=randn(B, case["T"], G, D))
    return s


# ---- the plain forms: float32, rounded once at the end ----

def _visible(s: dict[str, Any]) -> torch.Tensor | None:
    """Which key a query may see, [B or 1, 1, 1, Tq, Tk]; None where it may see all."""
    c, dev = s["case"], s["q"].device
    i, j = torch.arange(c["Tq"], device=dev)[:, None], torch.arange(c["Tk"], device=dev)[None, :]
    m = None
    if c["causal"]:
        m = (j <= i + (c["Tk"] - c["Tq"]))[None]
    if s["lengths"] is not None:
        inside = j[None] < s["lengths"][:, None, None]
        m = inside if m is None else m & inside
    if s["seg"] is not None:
        same = (s["seg"][:, None] == s["seg"][None, :])[None]
        m = same if m is None else m & same
    return None if m is None else m[:, None, None]


def _attention(s: dict[str, Any]) -> Any:
    c = s["case"]
    B, Tq, Tk, H, G, D = (c[n] for n in ("B", "Tq", "Tk", "H", "G", "D"))
    dt, scale = s["q"].dtype, D ** -0.5
    q = s["q"].detach().float().view(B, Tq, G, H // G, D).permute(0, 2, 3, 1, 4)          # [B, G, R, Tq, D]
    k, v = (s[n].detach().float().permute(0, 2, 1, 3)[:, :, None] for n in ("k", "v"))    # [B, G, 1, Tk, D]

    def heads(x):  # back to [B, T, heads, D]
        return x.permute(0, 3, 1, 2, 4).reshape(B, x.shape[3], -1, D)

    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    visible = _visible(s)
    if visible is not None:
        p.masked_fill_(~visible, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = torch.matmul(p, v)
    if not c["grad"]:
        return dict(o=heads(o).to(dt))
    do = s["do"].float().view(B, Tq, G, H // G, D).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2, keepdim=True)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True)
    return dict(o=heads(o).to(dt), dq=heads(dq).to(dt), dk=heads(dk).to(dt), dv=heads(dv).to(dt))


def _logprobs(s: dict[str, Any]) -> Any:
    c = s["case"]
    x = s["logits"].detach().float()
    t, top = s["targets"], c["top"]
    known = t >= 0
    col = t.clamp_min(0)[:, None]
    m = x.amax(-1, keepdim=True)
    lse = (x - m).exp_().sum(-1, keepdim=True).log_() + m
    lp = x - lse
    p = lp.exp()
    h = -(p * lp).sum(-1)
    out = dict(logp=torch.where(known, lp.gather(1, col)[:, 0], 0.0), entropy=h)
    if top:
        # The largest logits, of equal ones the lowest index first: one ordered whole number holds both.
        bits = x.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = order * (1 << 20) - torch.arange(c["V"], device=x.device)
        ids = ((1 << 20) - key.topk(top, dim=-1).values % (1 << 20)) % (1 << 20)
        out.update(top_logp=lp.gather(1, ids), top_ids=ids)
    if c["grad"]:
        gl, ge = torch.where(known, s["dlogp"], 0.0)[:, None], s["dent"][:, None]
        d = -p * (gl + ge * (lp + h[:, None]))
        d.scatter_add_(1, col, gl)
        out.update(dlogits=d.to(s["logits"].dtype))
    return out


def _quantised(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes 0..15 and (scale, minimum) of groups of channels, ``x [..., D]`` -> ``[..., D], [..., D / 64, 2]``."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo = g.amin(-1, keepdim=True).bfloat16()
    scale = ((g.amax(-1, keepdim=True) - lo.float()) / 15).clamp_min(0).bfloat16()
    inv = torch.where(scale == 0, 0.0, 1.0 / scale.float())
    n = ((g - lo.float()) * inv).round_().clamp_(0, 15)
    return n.flatten(-2).to(torch.uint8), torch.cat((scale, lo), dim=-1)


def _values(codes: torch.Tensor, meta: torch.Tensor) -> torch.Tensor:
    """What packed codes ``[..., D / 2]`` (even channels in the low bits) stand for, in float32 ``[..., D]``."""
    n = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).float().unflatten(-1, (-1, GROUP))
    m = meta.float()
    return (n * m[..., :1] + m[..., 1:]).flatten(-2)


def _put(s: dict[str, Any], k: torch.Tensor, v: torch.Tensor, start: torch.Tensor) -> None:
    """Stores ``k, v [B, T, G, D]`` at positions ``start ..`` of the cache."""
    B, T, G, _ = k.shape
    dev = k.device
    at = (torch.arange(B, device=dev)[:, None, None], torch.arange(G, device=dev)[None, :, None],
          (start[:, None] + torch.arange(T, device=dev))[:, None, :])
    for x, codes, meta in ((k, *s["cache"][:2]), (v, *s["cache"][2:])):
        n, m = _quantised(x.transpose(1, 2))
        codes[at] = n[..., 0::2] | (n[..., 1::2] << 4)
        meta[at] = m


def _got(s: dict[str, Any], start: torch.Tensor, T: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The values of positions ``start .. start + T - 1``, ``[B, T, G, D]``."""
    ck, mk, cv, mv = s["cache"]
    B, G = ck.shape[:2]
    dev = ck.device
    at = (torch.arange(B, device=dev)[:, None, None], torch.arange(G, device=dev)[None, None, :],
          (start[:, None] + torch.arange(T, device=dev))[:, :, None])
    return _values(ck[at], mk[at]), _values(cv[at], mv[at])


def _decode(s: dict[str, Any]) -> Any:
    c = s["case"]
    B, L, H, G, D = (c[n] for n in ("B", "L", "H", "G", "D"))
    dt = s["qkv"].dtype
    x = s["qkv"].view(B, 1, G, H // G + 2, D)
    cos, sin = s["cos"][s["pos"]].view(B, 1, 1, 1, D // 2), s["sin"][s["pos"]].view(B, 1, 1, 1, D // 2)
    qk = x[..., :-1, :].float()
    x1, x2 = qk[..., 0::2], qk[..., 1::2]
    qk = torch.stack((x1 * cos - x2 * sin, x1 * sin + x2 * cos), dim=-1).flatten(-2).to(dt)
    _put(s, qk[..., -1, :], x[..., -1, :], s["pos"])
    q = qk[:, 0, :, :-1].float()                                                        # [B, G, R, D]
    k, v = _values(*s["cache"][:2]), _values(*s["cache"][2:])                           # [B, G, L, D]
    p = torch.matmul(q, k.transpose(-1, -2)) * D ** -0.5
    p.masked_fill_(torch.arange(L, device=q.device) > s["pos"][:, None, None, None], float("-inf"))
    p = (p - p.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    kn, vn = _got(s, s["pos"], 1)
    return dict(o=o.reshape(B, H, D).to(dt), k=kn, v=vn)


def _store(s: dict[str, Any]) -> Any:
    start = torch.zeros(s["case"]["B"], dtype=torch.int64, device=s["k"].device)
    _put(s, s["k"], s["v"], start)
    k, v = _got(s, start, s["case"]["T"])
    return dict(k=k.to(s["k"].dtype), v=v.to(s["v"].dtype))


# ---- the framework's kernels ----

def _own(s: dict[str, Any]) -> Any:
    from qwendopamine_amd import ops

    c = s["case"]
    if c["kind"] == "attn":
        o = ops.attention(s["q"], s["k"], s["v"], causal=c["causal"], kv_lengths=s["lengths"], cu_seqlens=s["cu"])
        if not c["grad"]:
            return dict(o=o)
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return dict(o=o.detach(), dq=dq, dk=dk, dv=dv)
    if c["kind"] == "logp":
        r = ops.token_logprobs(s["logits"], s["targets"], top_k=c["top"])
        out = dict(logp=r.logprobs.detach(), entropy=r.entropy.detach())
        if c["top"]:
            out.update(top_logp=r.top_logprobs, top_ids=r.top_ids)
        if c["grad"]:
            (out["dlogits"],) = torch.autograd.grad((r.logprobs, r.entropy), (s["logits"],), (s["dlogp"], s["dent"]))
        return out
    cache = ops.KVCacheQ4(*s["cache"])
    if c["kind"] == "decode":
        o = ops.attention_decode_q4(s["qkv"], s["cos"], s["sin"], s["pos"], cache, c["H"])
        k, v = ops.kv_cache_q4_load(cache, s["pos"], 1, torch.float32)
        return dict(o=o, k=k, v=v)
    ops.kv_cache_q4_store(cache, s["k"], s["v"])
    k, v = ops.kv_cache_q4_load(cache, None, c["T"], s["k"].dtype)
    return dict(k=k, v=v)


def run(s: dict[str, Any]) -> Any:
    if own:
        return _own(s)
    with torch.no_grad():
        return {"attn": _attention, "logp": _logprobs, "decode": _decode, "store": _store}[s["case"]["kind"]](s)


# ---- what a pass cannot do without ----

def _pairs(case: dict) -> int:
    """Query / key pairs of one head over the batch that the masks leave."""
    def tri(Tq, Tk, n):  # keys visible below n, causal from the end
        first = Tk - Tq  # query i sees keys 0 .. i + first
        lo = min(Tq, max(0, -first))              # queries before this see none
        hi = min(Tq, max(lo, n - 1 - first))      # queries from this on see n
        seen = (hi - lo) * (lo + first + 1) + (hi - lo) * (hi - lo - 1) // 2
        return seen + (Tq - hi) * max(0, n)

    Tq, Tk = case["Tq"], case["Tk"]
    if case["mask"] == "packed":
        cu = _offsets(case)
        return sum(tri(b - a, b - a, b - a) if case["causal"] else (b - a) ** 2 for a, b in zip(cu, cu[1:]))
    lens = _lengths(case) if case["mask"] == "lengths" else [Tk] * case["B"]
    return sum(tri(Tq, Tk, n) if case["causal"] else Tq * n for n in lens)


def work(case: dict) -> dict[str, float]:
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "attn":
        B, Tq, Tk, H, G, D = (case[n] for n in ("B", "Tq", "Tk", "H", "G", "D"))
        q, kv = B * Tq * H * D * es, 2 * B * Tk * G * D * es
        products = 2 + (5 if case["grad"] else 0)  # s, o; s again, dv, dp, dq, dk
        nbytes = 2 * q + kv + ((2 * q + kv) if case["grad"] else 0)
        return dict(bytes=nbytes, flops=2.0 * products * H * D * _pairs(case))
    if case["kind"] == "logp":
        n = case["rows"] * case["V"]
        return dict(bytes=n * es * (2 if case["grad"] else 1) + case["rows"] * (16 + 12 * case["top"]),
                    flops=(10.0 if case["grad"] else 5.0) * n)
    G, D = case["G"], case["D"]
    row = G * 2 * (D // 2 + 4 * (D // GROUP))  # a position's codes, scales and minima, k and v
    if case["kind"] == "decode":
        B, H = case["B"], case["H"]
        n = sum(p + 1 for p in _positions(case))
        return dict(bytes=n * row + B * ((2 * H + 2 * G) * D * es + 2 * G * D * 4), flops=4.0 * n * H * D)
    n = case["B"] * case["T"]
    return dict(bytes=n * (2 * row + 2 * 2 * G * D * es), flops=10.0 * n * G * D)


# ---- the definitions in 64 bits ----

def _exact_attention(s: dict[str, Any]) -> Any:
    c = s["case"]
    Tq, Tk, H, G, D = (c[n] for n in ("Tq", "Tk", "H", "G", "D"))
    dev = s["q"].device
    q, k, v = (s[n].detach() for n in ("q", "k", "v"))
    out = {"o": torch.zeros(q.shape, dtype=torch.float64, device=dev)}
    if c["grad"]:
        out.update({"d" + n: torch.zeros(x.shape, dtype=torch.float64, device=dev) for n, x in zip("qkv", (q, k, v))})
    if c["mask"] == "packed":
        cu = _offsets(c)
        spans = [(0, slice(a, b), slice(a, b)) for a, b in zip(cu, cu[1:])]
    else:
        lens = _lengths(c) if c["mask"] == "lengths" else [Tk] * c["B"]
        spans = [(b, slice(0, Tq), slice(0, n)) for b, n in enumerate(lens)]
    for b, rows, cols in spans:
        nq, nk = rows.stop - rows.start, cols.stop - cols.start
        if nq == 0 or nk == 0:
            continue
        shift = 0 if c["mask"] == "packed" else Tk - Tq
        hidden = None
        if c["causal"]:
            hidden = torch.ones(nq, nk, dtype=torch.bool, device=dev).triu(1 + shift)
        for h in range(H):
            g = h // (H // G)
            Q, K, V = q[b, rows, h].double(), k[b, cols, g].double(), v[b, cols, g].double()
            S = Q @ K.T / math.sqrt(D)
            if hidden is not None:
                S[hidden] = -math.inf
            P = torch.softmax(S, dim=1).nan_to_num_(nan=0.0)  # a query that sees nothing: zeros
            del S
            O = P @ V
            out["o"][b, rows, h] = O
            if c["grad"]:
                dO = s["do"][b, rows, h].double()
                out["dv"][b, cols, g] += P.T @ dO
                dS = P * (dO @ V.T - (dO * O).sum(1, keepdim=True)) / math.sqrt(D)
                out["dq"][b, rows, h] = dS @ K
                out["dk"][b, cols, g] += dS.T @ Q
    return out


def _exact_logprobs(s: dict[str, Any]) -> Any:
    c = s["case"]
    logits = s["logits"].detach()
    parts = []
    for lo in range(0, c["rows"], 256):
        x = logits[lo:lo + 256].double()
        t = s["targets"][lo:lo + 256]
        lp = torch.log_softmax(x, dim=-1)
        h = -(lp.exp() * lp).sum(-1)
        col = t.clamp_min(0)[:, None]
        one = dict(logp=lp.gather(1, col)[:, 0].masked_fill(t < 0, 0.0), entropy=h)
        if c["top"]:
            one["top_logp"] = lp.sort(dim=-1, descending=True).values[:, : c["top"]]
        if c["grad"]:
            gl = s["dlogp"][lo:lo + 256].double().masked_fill(t < 0, 0.0)[:, None]
            ge = s["dent"][lo:lo + 256].double()[:, None]
            p = lp.exp()
            d = torch.zeros_like(p).scatter_(1, col, gl) - p * gl
            one["dlogits"] = (d - ge * p * (lp + h[:, None])).to(torch.float64)
        parts.append(one)
    out = {n: torch.cat([x[n] for x in parts]) for n in parts[0]}
    if c["top"]:
        out["top_ids"] = None
    return out


def _exact_decode(s: dict[str, Any]) -> Any:
    """Attention over what the cache stands for after the token's store.  The token's own codes
    follow from float32 values by definition, so that k and v have no value apart from it."""
    c = s["case"]
    B, H, G, D = (c[n] for n in ("B", "H", "G", "D"))
    dt = s["qkv"].dtype
    o = torch.empty(B, H, D, dtype=torch.float64, device=s["qkv"].device)

    def values(codes, meta):
        n = torch.empty(*codes.shape[:-1], D, dtype=torch.float64, device=codes.device)
        n[..., 0::2], n[..., 1::2] = (codes % 16).double(), (codes // 16).double()
        m = meta.double().repeat_interleave(GROUP, dim=-2)
        return n * m[..., 0] + m[..., 1]

    def held(x):  # [..., D] in the token's type -> what four bits keep of it
        y = x.float().reshape(*x.shape[:-1], D // GROUP, GROUP)
        lo = y.min(-1, keepdim=True).values.bfloat16().float()
        sc = torch.relu((y.max(-1, keepdim=True).values - lo) / 15.0).bfloat16().float()
        n = torch.clamp(torch.round((y - lo) * torch.where(sc > 0, sc.reciprocal(), sc)), 0, 15)
        return (n.double() * sc.double() + lo.double()).reshape(x.shape)

    for b, p in enumerate(_positions(c)):
        x = s["qkv"][b, 0].view(G, H // G + 2, D)
        z = torch.complex(x[:, :-1, 0::2].double(), x[:, :-1, 1::2].double())
        z = z * torch.complex(s["cos"][p].double(), s["sin"][p].double())
        qk = torch.view_as_real(z).flatten(-2).to(dt)
        ck, mk, cv, mv = (y[b, :, : p + 1] for y in s["cache"])
        K, V = values(ck, mk), values(cv, mv)
        K[:, p], V[:, p] = held(qk[:, -1]), held(x[:, -1])
        P = torch.softmax(qk[:, :-1].double() @ K.transpose(1, 2) / math.sqrt(D), dim=-1)
        o[b] = (P @ V).reshape(H, D)
    return dict(o=o, k=None, v=None)


def exact(case: dict, seed: int) -> Any:
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "attn":
            return _exact_attention(s)
        if case["kind"] == "logp":
            return _exact_logprobs(s)
        if case["kind"] == "decode":
            return _exact_decode(s)
    return None  # whole codes by definition: what they stand for follows from float32 arithmetic
