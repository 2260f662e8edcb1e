"""Performance cases of the serving side of the hybrid decoder's attention layers and of its answers:
norms of queries and keys with the rotation of positions (with their gradient), the append of rotated
keys and of values to a paged cache, attention over that cache, and sampling of tokens.

``run`` computes every case in plain torch (float32; sampling in float64), or, with ``own`` set, through
the framework's entry points (``ops.qkv_norm_rope``, ``ops.kv_cache_paged_append``,
``ops.attention_paged``, ``ops.sample_tokens``).  ``exact`` restates each of them in float64.
"""

from __future__ import annotations

import math
from typing import Any

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


def listed() -> list[dict]:
    return [
        # One token of a small served batch at unequal positions, q and k normalised: the smallest call.
        dict(name="rope-step-b8-d64", kind="rope", B=8, T=1, H=16, G=16, D=64, rot=64, dtype="bf16", norm=True,
             grad=False, each=True),
        # The hybrid decoder's attention layer in a training step, q and k normalised.
        dict(name="rope-train-b4-t2048-d64", kind="rope", B=4, T=2048, H=16, G=16, D=64, rot=64, dtype="bf16",
             norm=True, grad=True, each=False),
        # A long text of odd length, grouped heads, half of the channels rotated, training.
        dict(name="rope-train-t7013-g4-d128", kind="rope", B=1, T=7013, H=16, G=4, D=128, rot=64, dtype="fp16",
             norm=True, grad=True, each=False),
        # The rotation alone of a long prompt.
        dict(name="rope-prompt-t16384-d128", kind="rope", B=1, T=16384, H=32, G=8, D=128, rot=128, dtype="bf16",
             norm=False, grad=False, each=False),
        # One token of each sequence of a served batch into its pages.
        dict(name="append-step-b32-d128", kind="append", B=32, T=1, H=32, G=8, D=128, rot=128, S=16, L=1024,
             dtype="bf16", norm=True),
        # Padded prompts of unequal lengths into their pages.
        dict(name="append-prompts-b4-t2048-d64", kind="append", B=4, T=2048, H=16, G=16, D=64, rot=64, S=64, L=2304,
             dtype="bf16", norm=True),
        # One token of a small served batch, one attention layer of the hybrid decoder.
        dict(name="paged-step-b4-l2304-d64", kind="paged", B=4, T=1, L=2304, H=16, G=16, D=64, S=64, dtype="bf16",
             ragged=False),
        # One token of a large served batch at unequal positions of long contexts, small pages.
        dict(name="paged-step-b32-l32768-d128", kind="paged", B=32, T=1, L=32768, H=32, G=8, D=128, S=16,
             dtype="bf16", ragged=True),
        # Pieces of three prompts, unequal in length and in what lies before them.
        dict(name="paged-piece-b3-t517-l9000", kind="paged", B=3, T=517, L=9000, H=16, G=4, D=128, S=32, dtype="fp16",
             ragged=True),
        # The next token of a small batch over the full head.
        dict(name="sample-b4-v151936", kind="sample", rows=4, V=151936, dtype="bf16", mix=False, T=0.8, k=50, p=0.95,
             m=0.0),
        # A large batch in which every sequence has settings of its own.
        dict(name="sample-b256-v151936", kind="sample", rows=256, V=151936, dtype="bf16", mix=True, T=1.0, k=0, p=1.0,
             m=0.0),
        # A nucleus of float32 logits over the 32000-word head.
        dict(name="sample-b64-v32000-fp32", kind="sample", rows=64, V=32000, dtype="fp32", mix=False, T=1.2, k=0,
             p=0.9, m=0.0),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["rope", "rope", "append", "paged", "paged", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    G = rng.choice([1, 2, 4, 8, 16])
    R = rng.choice([1, 1, 2, 4, 7, 8])
    if kind == "sample":
        V = _log_int(rng, 50, 160000)
        return dict(kind=kind, rows=_log_int(rng, 1, min(512, max(2, int(3.8e7 / V)))), V=V,
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), mix=rng.random() < 0.4,
                    T=rng.choice([0.0, 0.6, 0.8, 1.0, 1.0, 1.5]), k=rng.choice([0, 0, 1, 20, 50, 1000]),
                    p=rng.choice([1.0, 0.95, 0.9, 0.5]), m=rng.choice([0.0, 0.0, 0.05]))
    if kind == "rope":
        D = rng.choice([32, 64, 64, 96, 128, 128, 256])
        tokens = _log_int(rng, 1, max(2, int(6.0e7 / ((R + 2) * G * D))))
        B = 1 if rng.random() < 0.4 else max(1, min(tokens, _log_int(rng, 1, 64)))
        return dict(kind=kind, B=B, T=max(1, tokens // B), H=G * R, G=G, D=D, rot=rng.choice([D, D, D // 2]),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), norm=rng.random() < 0.7, grad=rng.random() < 0.6,
                    each=rng.random() < 0.4)
    D = rng.choice([64, 128])
    S = rng.choice([16, 16, 32, 64, 128, 256])
    if kind == "append":
        tokens = _log_int(rng, 1, max(2, int(4.0e7 / ((R + 2) * G * D))))
        B = max(1, min(tokens, _log_int(rng, 1, 64)))
        T = max(1, tokens // B)
        return dict(kind=kind, B=B, T=T, H=G * R, G=G, D=D, rot=rng.choice([D, D, D // 2]), S=S,
                    L=T + _log_int(rng, 1, 1000), dtype=dtype, norm=rng.random() < 0.6)
    T = rng.choice([1, 1, 1, rng.randint(2, 8), _log_int(rng, 9, 600)])
    L = max(T, _log_int(rng, 1, 32768))
    B = max(1, min(_log_int(rng, 1, 64), int(8.0e6 / (L * G)), int(5.0e8 / (T * L * G * R))))
    return dict(kind=kind, B=B, T=T, L=L, H=G * R, G=G, D=D, S=S, dtype=dtype, ragged=rng.random() < 0.6)


# ---- inputs ----

def _tables(R: int, case: dict, device) -> tuple[torch.Tensor, torch.Tensor]:
    """float32 cos / sin of positions 0 .. R - 1, ``[R, rot / 2]``; the angles in float64."""
    rot = case["rot"]
    theta = 10000.0 ** (-torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
    ang = torch.outer(torch.arange(R, device=device, dtype=torch.float64), theta)
    return ang.cos().float(), ang.sin().float()


def _lengths(case: dict) -> list[int]:
    """Tokens of each sequence's piece: all of them, but for the padded batches' shorter ones."""
    B, T = case["B"], case["T"]
    uneven = case["kind"] == "append" or case.get("ragged")
    return [T if T == 1 or not uneven else max(1, T - (T * b) // (2 * B)) for b in range(B)]


def _starts(case: dict) -> list[int]:
    """The position of each sequence's first new token: near the end of the caches, or spread over them."""
    B, T, L = case["B"], case["T"], case["L"]
    free = L - T
    if case["kind"] == "append":
        return [0 if T > 1 else (free * (b + 1)) // B for b in range(B)]
    if not case["ragged"]:
        return [free - free // 10] * B
    return [(free * (2 * b + 1)) // (2 * B) for b in range(B)]


def _pages(case: dict, lengths: list[int], starts: list[int], gen, dev) -> tuple[int, torch.Tensor]:
    """The pages that the sequences need, in no order: their number, and the table ``[B, N]`` (-1: none)."""
    S, B = case["S"], case["B"]
    need = [(s + n + S - 1) // S for s, n in zip(starts, lengths)]
    order = torch.randperm(sum(need), generator=gen, device=dev).to(torch.int32)
    table = torch.full((B, (case["L"] + S - 1) // S), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return sum(need), table


def prepare(case: dict, seed: int) -> dict[str, Any]:
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)

    s: dict[str, Any] = dict(case=case)
    if case["kind"] == "sample":
        n, V = case["rows"], case["V"]
        logits = randn(n, V, dtype=torch.float32) * 2.2
        # What the model thinks likely: some tokens well above the others.
        likely = torch.randint(0, V, (n, 40), generator=gen, device=dev)
        logits.scatter_add_(1, likely, torch.rand(n, 40, generator=gen, device=dev) ** 2 * 10)
        s.update(logits=logits.to(dt), u=torch.rand(n, generator=gen, device=dev))
        if case["mix"]:  # every row with settings of its own
            def rows(*values, dtype=torch.float32):
                return torch.tensor([values[i % len(values)] for i in range(n)], dtype=dtype, device=dev)
            s.update(T=rows(0.7, 1.0, 1.3, 0.0, 0.9, 1.0, 1.0), k=rows(0, 50, 0, 0, 200, 0, 0, dtype=torch.int32),
                     p=rows(0.95, 1.0, 0.9, 1.0, 0.8, 1.0, 0.5), m=rows(0.0, 0.0, 0.0, 0.0, 0.0, 0.05, 0.0))
        else:
            s.update(T=case["T"], k=case["k"], p=case["p"], m=case["m"])
        return s
    B, T, H, G, D = (case[n] for n in ("B", "T", "H", "G", "D"))
    if case["kind"] == "paged":
        s.update(q=randn(B, T, H, D))
    else:
        s.update(qkv=randn(B, T, (H + 2 * G) * D), wq=None, wk=None)
        if case["norm"]:
            s.update(wq=randn(D, dtype=torch.float32).mul(0.2).add(1).to(dt),
                     wk=randn(D, dtype=torch.float32).mul(0.2).add(1).to(dt))
    if case["kind"] == "rope":
        pos = None
        if case["each"]:  # every sequence at a position of its own
            first = torch.randint(0, 4000, (B, 1), generator=gen, device=dev)
            pos = first + torch.arange(T, device=dev)
        s["cos"], s["sin"] = _tables(T + 4000 if case["each"] else T, case, dev)
        s["pos"] = pos
        if case["grad"]:
            for n in ("qkv", "wq", "wk"):
                s[n] = None if s[n] is None else s[n].requires_grad_(True)
            s.update(dq=randn(B, T, H, D), dk=randn(B, T, G, D), dv=randn(B, T, G, D))
        return s
    lengths, starts = _lengths(case), _starts(case)
    n, table = _pages(case, lengths, starts, gen, dev)
    kp, vp = (torch.randn(n, G, case["S"], D, generator=gen, device=dev, dtype=dt) for _ in range(2))
    s.update(cache=(kp, vp, table), start=torch.tensor(starts, device=dev),
             lengths=torch.tensor(lengths, device=dev) if min(lengths) < T else None)
    if case["kind"] == "append":
        s["cos"], s["sin"] = _tables(case["L"], case, dev)
    return s


# ---- the plain forms: float32, rounded once at the end ----

def _positions(s: dict[str, Any]) -> torch.Tensor:
    """``[B, T]``"""
    c = s["case"]
    dev = s["cache"][0].device
    return s["start"][:, None] + torch.arange(c["T"], device=dev)


def _there(s: dict[str, Any]) -> torch.Tensor:
    """Which tokens of the padded batch exist, ``[B, T]``."""
    c = s["case"]
    t = torch.arange(c["T"], device=s["cache"][0].device)[None].expand(c["B"], -1)
    return t >= 0 if s["lengths"] is None else t < s["lengths"][:, None]


def _rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """``x [B, T, G, R, D]`` with ``cos, sin [B or 1, T, rot / 2]``."""
    rot = 2 * cos.shape[-1]
    c, n = cos[:, :, None, None], sin[:, :, None, None]
    x1, x2 = x[..., :rot:2], x[..., 1:rot:2]
    y = torch.stack((x1 * c - x2 * n, x1 * n + x2 * c), dim=-1).flatten(-2)
    return torch.cat((y, x[..., rot:]), dim=-1)


def _split(s: dict[str, Any]) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(q and k, their weights, 1 / rms, v)`` in float32, ``[B, T, G, R + 1, D]`` (the key last)."""
    c = s["case"]
    B, T, H, G, D = (c[n] for n in ("B", "T", "H", "G", "D"))
    x = s["qkv"].detach().float().view(B, T, G, H // G + 2, D)
    qk, v = x[..., :-1, :], x[..., -1, :]
    if not c["norm"]:
        return qk, None, None, v
    w = torch.cat((s["wq"].detach().float().expand(H // G, D), s["wk"].detach().float()[None]))
    r = torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS)
    return qk, w, r, v


def _rope(s: dict[str, Any]) -> Any:
    c = s["case"]
    B, T, H, G, D = (c[n] for n in ("B", "T", "H", "G", "D"))
    dt = s["qkv"].dtype
    cos, sin = (s[n][None, :T] if s["pos"] is None else s[n][s["pos"]] for n in ("cos", "sin"))
    x, w, r, v = _split(s)
    y = _rotated(x if w is None else x * r * w, cos, sin)
    out = dict(q=y[..., :-1, :].reshape(B, T, H, D).to(dt), k=y[..., -1, :].to(dt), v=v.to(dt))
    if not c["grad"]:
        return out
    dy = torch.cat((s["dq"].float().view(B, T, G, H // G, D), s["dk"].float()[..., None, :]), dim=-2)
    dn = _rotated(dy, cos, -sin)
    if w is not None:
        xr = x * r
        dw = (dn * xr).sum((0, 1, 2))
        dn = dn * w
        dn = (dn - xr * (dn * xr).mean(-1, keepdim=True)) * r
        out.update(dwq=dw[:-1].sum(0).to(dt), dwk=dw[-1].to(dt))
    out.update(dqkv=torch.cat((dn, s["dv"].float()[..., None, :]), dim=-2).reshape(B, T, -1).to(dt))
    return out


def _append(s: dict[str, Any]) -> Any:
    c = s["case"]
    B, T, H, G, D, S = (c[n] for n in ("B", "T", "H", "G", "D", "S"))
    dt = s["qkv"].dtype
    kp, vp, table = s["cache"]
    pos, there = _positions(s), _there(s)
    safe = torch.where(there, pos, 0)
    x, w, r, v = _split(s)
    y = _rotated(x if w is None else x * r * w, s["cos"][safe], s["sin"][safe]).to(dt)
    page = table.long().gather(1, safe // S)
    at = page[there], slice(None), (pos % S)[there]
    kp[at] = y[..., -1, :][there]
    vp[at] = v.to(dt)[there]
    q = torch.where(there[:, :, None, None, None], y[..., :-1, :], 0)
    return dict(q=q.reshape(B, T, H, D), k=kp, v=vp)


def _paged(s: dict[str, Any]) -> Any:
    c = s["case"]
    B, T, H, G, D, S, L = (c[n] for n in ("B", "T", "H", "G", "D", "S", "L"))
    kp, vp, table = s["cache"]
    pages = table.long().clamp_min(0)
    k, v = (x[pages].transpose(1, 2).reshape(B, G, -1, D).float() for x in (kp, vp))        # [B, G, N S, D]
    q = s["q"].float().view(B, T, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)  # [B, G, R T, D]
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(D ** -0.5).view(B, G, H // G, T, -1)
    hidden = torch.arange(k.shape[2], device=q.device) > _positions(s)[:, :, None]
    p.masked_fill_(hidden[:, None, None], float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, G, -1, k.shape[2]), v).view(B, G, H // G, T, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, H, D)
    return dict(o=torch.where(_there(s)[:, :, None, None], o, 0).to(s["q"].dtype))


def _setting(s: dict[str, Any], name: str) -> torch.Tensor:
    """A row's setting as the float32 (top-k: whole) number that it is, in float64 ``[rows or 1, 1]``."""
    v = s[name]
    if not isinstance(v, torch.Tensor):
        v = torch.tensor([v], dtype=torch.float32, device=s["logits"].device)
    return v.double()[:, None]


def _sample(s: dict[str, Any]) -> Any:
    x = s["logits"].double()
    V = x.shape[1]
    T, k, p, m = (_setting(s, n) for n in ("T", "k", "p", "m"))
    # The largest logits first, of equal ones the lowest index.
    ordered, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    w = ((ordered - ordered[:, :1]) / torch.where(T > 0, T, 1.0)).exp()
    rank = torch.arange(V, device=x.device)
    kept = torch.where((w >= m) & ((k < 1) | (rank < k)), w, 0.0)
    before = kept.cumsum(-1) - kept
    kept = torch.where((p >= 1) | (before < p * kept.sum(-1, keepdim=True)), kept, 0.0)
    # Back to the order of the tokens, and the first whose running sum exceeds the random share.
    cum = torch.zeros_like(x).scatter_(1, ids, kept).cumsum(-1)
    drawn = (cum <= s["u"].double()[:, None] * cum[:, -1:]).sum(-1)
    return torch.where(T[:, 0] > 0, drawn, ids[:, 0])


# ---- the framework's kernels ----

def _own(s: dict[str, Any]) -> Any:
    from qwendopamine_amd import ops

    c = s["case"]
    if c["kind"] == "rope":
        q, k, v = ops.qkv_norm_rope(s["qkv"], s["cos"], s["sin"], c["H"], c["G"], s["wq"], s["wk"], EPS, s["pos"])
        out = dict(q=q.detach(), k=k.detach(), v=v.detach())
        if c["grad"]:
            leaves = [s[n] for n in ("qkv", "wq", "wk") if s[n] is not None]
            grads = torch.autograd.grad((q, k, v), leaves, (s["dq"], s["dk"], s["dv"]))
            if c["norm"]:
                out.update(dwq=grads[1], dwk=grads[2])
            out.update(dqkv=grads[0])
        return out
    if c["kind"] == "append":
        cache = ops.KVCachePaged(*s["cache"])
        q = ops.kv_cache_paged_append(s["qkv"], s["cos"], s["sin"], s["start"], cache, c["H"], s["wq"], s["wk"], EPS,
                                      s["lengths"])
        return dict(q=q, k=cache.k, v=cache.v)
    if c["kind"] == "paged":
        return dict(o=ops.attention_paged(s["q"], ops.KVCachePaged(*s["cache"]), s["start"], s["lengths"]))
    return ops.sample_tokens(s["logits"], s["u"], temperature=s["T"], top_k=s["k"], top_p=s["p"], min_p=s["m"])


def run(s: dict[str, Any]) -> Any:
    if own:
        return _own(s)
    with torch.no_grad():
        return {"rope": _rope, "append": _append, "paged": _paged, "sample": _sample}[s["case"]["kind"]](s)


# ---- what a pass cannot do without ----

def work(case: dict) -> dict:
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "sample":
        # The logits once; an exponential and a sum an element.
        n = case["rows"] * case["V"]
        return dict(bytes=n * size, flops=8 * n)
    B, T, H, G, D = (case[n] for n in ("B", "T", "H", "G", "D"))
    if case["kind"] == "rope":
        # q and k in and out, (cos, sin); backward: three gradients in, q and k again for the norm, one out.
        qk, v = B * T * (H + G) * D * size, B * T * G * D * size
        nbytes = 2 * qk + T * case["rot"] * 4
        if case["grad"]:
            nbytes += 2 * (qk + v) + (qk if case["norm"] else 0)
        return dict(bytes=nbytes, flops=(20 if case["grad"] else 8) * B * T * (H + G) * D)
    if case["kind"] == "append":
        tokens = sum(_lengths(case))
        return dict(bytes=2 * tokens * (H + 2 * G) * D * size + tokens * case["rot"] * 4,
                    flops=8 * tokens * (H + G) * D)
    pairs = keys = 0
    for s, n in zip(_starts(case), _lengths(case)):
        pairs += n * s + n * (n + 1) // 2
        keys += s + n
    return dict(bytes=2 * keys * G * D * size + 2 * B * T * H * D * size, flops=4 * D * H * pairs)


# ---- the definition in float64 ----

def _exact_rows(s: dict[str, Any], cos: torch.Tensor, sin: torch.Tensor, leaves=None):
    """q, k, v of ``qkv`` by the complex form of the rotation; ``cos, sin [B, T, rot / 2]``."""
    c = s["case"]
    B, T, H, G, D = (c[n] for n in ("B", "T", "H", "G", "D"))
    qkv, wq, wk = leaves if leaves else (None if s[n] is None else s[n].detach().double() for n in ("qkv", "wq", "wk"))
    rows = qkv.unflatten(-1, (G, H // G + 2, D))
    turn = torch.complex(cos.double(), sin.double())[:, :, None]
    out = []
    for x, w in ((rows[:, :, :, :-2].flatten(2, 3), wq), (rows[:, :, :, -2], wk)):
        if w is not None:
            x = x / (x.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w
        z = torch.view_as_complex(x[..., :c["rot"]].unflatten(-1, (-1, 2)).contiguous()) * turn
        out.append(torch.cat((torch.view_as_real(z).flatten(-2), x[..., c["rot"]:]), dim=-1))
    return *out, rows[:, :, :, -1]


def _exact_token(x: torch.Tensor, T: float, k: float, p: float, m: float, u: float) -> torch.Tensor:
    order = torch.argsort(-x, stable=True)
    if T <= 0:
        return order[0]
    logp = torch.log_softmax(x[order] / T, dim=0)
    n = x.numel() if m <= 0 else int((logp - logp[0] >= math.log(m)).sum())
    if k >= 1:
        n = min(n, int(k))
    if p < 1:
        prob = torch.softmax(x[order[:n]] / T, dim=0)
        n = max(1, int((prob.cumsum(0) - prob < p).sum()))
    chosen = order[:n].sort().values
    run = torch.softmax(x[chosen] / T, dim=0).cumsum(0)
    return chosen[min(int((run <= u).sum()), n - 1)]


def exact(case: dict, seed: int) -> Any:
    s = prepare(case, seed)
    if case["kind"] == "rope":
        B, T = case["B"], case["T"]
        at = torch.arange(T, device=s["qkv"].device).expand(B, T) if s["pos"] is None else s["pos"]
        cos, sin = s["cos"][at], s["sin"][at]
        if not case["grad"]:
            q, k, v = _exact_rows(s, cos, sin)
            return dict(q=q, k=k, v=v)
        leaves = [None if s[n] is None else s[n].detach().double().requires_grad_(True) for n in ("qkv", "wq", "wk")]
        outs = _exact_rows(s, cos, sin, leaves)
        grads = torch.autograd.grad(outs, [x for x in leaves if x is not None],
                                    [s[n].double() for n in ("dq", "dk", "dv")])
        res = dict(q=outs[0].detach(), k=outs[1].detach(), v=outs[2].detach())
        if case["norm"]:
            res.update(dwq=grads[1], dwk=grads[2])
        res.update(dqkv=grads[0])
        return res
    if case["kind"] == "append":
        S = case["S"]
        kp, vp, table = s["cache"]
        kp, vp = kp.double(), vp.double()
        table = table.tolist()
        dev = kp.device
        at = (s["start"][:, None] + torch.arange(case["T"], device=dev)).clamp_max(case["L"] - 1)
        q, k, v = _exact_rows(s, s["cos"][at], s["sin"][at])
        for b, (first, n) in enumerate(zip(_starts(case), _lengths(case))):
            q[b, n:] = 0
            slots = torch.tensor([table[b][j // S] * S + j % S for j in range(first, first + n)], device=dev)
            for pages, x in ((kp, k), (vp, v)):
                pages[slots // S, :, slots % S] = x[b, :n]
        return dict(q=q, k=kp, v=vp)
    if case["kind"] == "paged":
        H, G, D, S = (case[n] for n in ("H", "G", "D", "S"))
        kp, vp, table = s["cache"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=kp.device)
        for b, (first, n) in enumerate(zip(_starts(case), _lengths(case))):
            mine = table[b, :(first + n + S - 1) // S].long()
            k, v = (x[mine].double().transpose(0, 1).flatten(1, 2)[:, :first + n] for x in (kp, vp))  # [G, keys, D]
            after = torch.ones(n, first + n, dtype=torch.bool, device=kp.device).triu(first + 1)
            for h in range(H):
                a = s["q"][b, :n, h].double() @ k[h // (H // G)].T / math.sqrt(D)
                out[b, :n, h] = torch.softmax(a.masked_fill(after, -math.inf), dim=-1) @ v[h // (H // G)]
        return dict(o=out)
    settings = [_setting(s, n).expand(case["rows"], 1)[:, 0].tolist() for n in ("T", "k", "p", "m")]
    rows = zip(s["logits"], *settings, s["u"].tolist())
    return torch.stack([_exact_token(x.double(), *setting) for x, *setting in rows])
