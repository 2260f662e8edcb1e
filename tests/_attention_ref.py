"""Float64 reference of softmax attention with its gradients, and how far a result may be from it.

The bounds follow from the roundings of a computation that keeps scores, statistics and sums in
float32 and rounds four things to the io dtype (half a step ``u = eps / 2`` each): the
probabilities ``P`` before ``P V`` and ``P^T dO``, the gradients ``dS`` before ``dS K`` and ``dS^T Q``, the
output (from which ``D = dO . O`` is formed) and every gradient.  ``slack`` covers the float32
parts: a score is a sum of D exact products, off by at most about ``D 2^-24 sum |q k|``, which
moves P by as much relative to itself.  A probability below 2^-126 is flushed to zero by the
hardware exponential, and an operand below that by the products: ``FLUSH`` absolute for P, and
relative to dP's terms for dS.
"""

from __future__ import annotations

import torch

FLUSH = 2.0 ** -125


def visible(Tq: int, Tk: int, causal: bool, n: int) -> torch.Tensor:
    i, j = torch.arange(Tq)[:, None], torch.arange(Tk)[None, :]
    m = (j < n).expand(Tq, Tk)
    return m & (j <= i + Tk - Tq) if causal else m


def spans(B, Tq, Tk, kv_lengths, cu):
    """(batch row, query slice, key slice, visible keys) of every independent block."""
    if cu is not None:
        return [(0, slice(a, b), slice(a, b), b - a) for a, b in zip(cu, cu[1:])]
    return [(b, slice(0, Tq), slice(0, Tk), Tk if kv_lengths is None else max(0, min(Tk, int(kv_lengths[b]))))
            for b in range(B)]


def reference(q, k, v, do, scale, causal, kv_lengths=None, cu=None):
    """dict of float64 values and dict of elementwise bounds, for o, dq, dk, dv."""
    u = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * u * 2  # a subnormal result's absolute half step
    q, k, v, do = (x.detach().cpu().double() for x in (q, k, v, do))
    B, Tq, H, D = q.shape
    G = k.shape[2]
    val = {"o": torch.zeros_like(q), "dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    bnd = {n: torch.zeros_like(x) for n, x in val.items()}
    for b, rq, rk, n in spans(B, Tq, k.shape[1], kv_lengths, cu):
        nq, nk = rq.stop - rq.start, rk.stop - rk.start
        if nq == 0 or nk == 0:
            continue
        see = visible(nq, nk, causal, n)
        for h in range(H):
            g = h // (H // G)
            Q, dO = q[b, rq, h], do[b, rq, h]
            # Keys past the length are not read: whatever they hold, they count for nothing.
            K, V = (torch.where((torch.arange(nk) < n)[:, None], x[b, rk, g], 0.0) for x in (k, v))
            S = (scale * Q @ K.T).masked_fill(~see, float("-inf"))
            P = torch.where(see.any(1, keepdim=True), torch.softmax(S, 1), 0.0).nan_to_num(0.0)
            O = P @ V
            dP = dO @ V.T
            Dl = (dO * O).sum(1, keepdim=True)
            dS = P * (dP - Dl)
            slack = 4 * D * 2.0 ** -24 * scale * (Q.abs() @ K.abs().T).max() + 2.0 ** -20
            A = P @ V.abs()
            e_o = (u + slack) * A + FLUSH * V.abs().sum(0)
            e_O = e_o + u * O.abs()
            e_D = (dO.abs() * e_O).sum(1, keepdim=True) + slack * (dO.abs() @ V.abs().T).amax(1, keepdim=True)
            e_S = (u + slack) * dS.abs() + P * e_D + slack * P * (dO.abs() @ V.abs().T)
            e_S = e_S + FLUSH * (1 + (dP - Dl).abs())
            val["o"][b, rq, h], bnd["o"][b, rq, h] = O, e_O
            val["dq"][b, rq, h] = scale * dS @ K
            bnd["dq"][b, rq, h] = scale * e_S @ K.abs()
            val["dk"][b, rk, g] += scale * dS.T @ Q
            bnd["dk"][b, rk, g] += scale * e_S.T @ Q.abs()
            val["dv"][b, rk, g] += P.T @ dO
            bnd["dv"][b, rk, g] += (u + slack) * P.T @ dO.abs() + FLUSH * dO.abs().sum(0)
    for n in ("dq", "dk", "dv"):
        bnd[n] += u * val[n].abs()
    for n in bnd:
        bnd[n] = bnd[n] * 1.01 + tiny
    return val, bnd


def worst(got: dict, val: dict, bnd: dict) -> dict:
    """Largest error over its bound, per output."""
    out = {}
    for n, x in got.items():
        d = (x.detach().cpu().double() - val[n]).abs()
        assert torch.isfinite(d).all(), f"{n} is not finite"
        out[n] = float((d / bnd[n]).max()) if d.numel() else 0.0
    return out
