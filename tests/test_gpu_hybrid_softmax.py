"""The hybrid decoder on the softmax operators together: a training step on ``ops.attention`` and
``ops.token_logprobs``, scoring, and greedy decoding from a 4-bit KV cache with log probabilities."""

from __future__ import annotations

import pytest
import torch

from tests._helpers import rel_l2

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _model(dtype, dev, attention="hip", layers=(0, 1), n_layer=4, **kw):
    from qwendopamine_amd.hybrid import HybridConfig, HybridDecoder

    torch.manual_seed(0)
    cfg = dict(n_layer=n_layer, n_embd=256, n_head=4, head_size=64, n_query_groups=2, intermediate_size=512,
               vocab_size=1000, gdn2_layers=list(layers), block_size=512, attention=attention)
    return HybridDecoder(HybridConfig(**{**cfg, **kw})).to(dev, dtype).eval()


def _grads(m, idx, loss):
    m.zero_grad(set_to_none=True)
    value = loss(m, idx)
    value.backward()
    torch.cuda.synchronize()
    return float(value.detach()), {n: p.grad.detach().double() for n, p in m.named_parameters()}


def test_training_step(gpu_device):
    """Loss and every parameter's gradient in bf16 against the same weights in float32 on torch's
    attention and log-softmax: as near as the bf16 model on torch's own attention and loss is,
    whose roundings are of the same kind and number (a quarter more for their chance)."""
    print("[case] hybrid training step, hip attention and loss", flush=True)
    idx = torch.randint(0, 1000, (3, 130), device=gpu_device, generator=torch.Generator(gpu_device).manual_seed(1))

    def torch_loss(m, idx):
        return torch.nn.functional.cross_entropy(m(idx)[:, :-1].float().flatten(0, 1), idx[:, 1:].flatten())

    hip = _model(BF, gpu_device)
    sdpa = _model(BF, gpu_device, attention="sdpa")
    sdpa.load_state_dict(hip.state_dict())
    full = _model(torch.float32, gpu_device, attention="sdpa")
    full.load_state_dict(hip.state_dict())
    want, gw = _grads(full, idx, torch_loss)
    have, gh = _grads(hip, idx, lambda m, i: m.loss(i))
    base, gb = _grads(sdpa, idx, torch_loss)
    print(f"  loss {have:.6f}, torch bf16 {base:.6f}, float32 {want:.6f}", flush=True)
    assert abs(have - want) <= 1.25 * abs(base - want) + 2.0 ** -8 * abs(want)

    def err(g):
        num = sum(float((g[n] - gw[n]).square().sum()) for n in gw)
        return (num / sum(float(x.square().sum()) for x in gw.values())) ** 0.5

    print(f"  gradients {err(gh):.3e}, torch bf16 {err(gb):.3e}", flush=True)
    assert err(gh) <= 1.25 * err(gb) + 2.0 ** -9
    for n in gw:
        if ".attn.attn." in n or ".attn.proj." in n:
            assert rel_l2(gh[n], gw[n]) <= 1.25 * rel_l2(gb[n], gw[n]) + 2.0 ** -8, n


def test_loss_ignores_targets_and_repeats(gpu_device):
    m = _model(BF, gpu_device)
    idx = torch.randint(0, 1000, (2, 40), device=gpu_device)
    targets = torch.randint(0, 1000, (2, 40), device=gpu_device)
    targets[0, 5:] = -100
    a, ga = _grads(m, idx, lambda m, i: m.loss(i, targets))
    b, gb = _grads(m, idx, lambda m, i: m.loss(i, targets))
    r = m.token_logprobs(idx, targets)
    assert a == pytest.approx(-float(r.logprobs.sum().detach()) / 45, rel=1e-6)
    attn = [n for n in ga if n.startswith(("h.2.attn", "h.3.attn", "lm_head"))]
    assert a == b and attn and all(torch.equal(ga[n], gb[n]) for n in attn)
    targets[:] = -100
    v, g = _grads(m, idx, lambda m, i: m.loss(i, targets))
    assert v == 0 and all((x == 0).all() for x in g.values())
    targets.random_(0, 3)
    with torch.no_grad():
        v, r = m.loss(idx, targets, ignore_index=1), m.token_logprobs(idx, targets).logprobs
    assert float(v) == pytest.approx(-float(r[targets != 1].mean()), rel=1e-5)


def test_scoring(gpu_device):
    """``token_logprobs`` of the next tokens against a float64 log-softmax of the model's logits."""
    m = _model(BF, gpu_device)
    idx = torch.randint(0, 1000, (2, 61), device=gpu_device)
    with torch.no_grad():
        r = m.token_logprobs(idx, top_k=5)
        lp = m(idx).double().log_softmax(-1)[:, :-1]
    assert r.logprobs.shape == (2, 60) and r.top_ids.shape == (2, 60, 5)
    assert float((r.logprobs.double() - lp.gather(-1, idx[:, 1:, None])[..., 0]).abs().max()) <= 2e-5
    assert float((r.entropy.double() + (lp.exp() * lp).sum(-1)).abs().max()) <= 2e-5
    assert torch.equal(lp.gather(-1, r.top_ids), lp.topk(5, -1).values)


@pytest.mark.parametrize("kv_bits", [16, 4])
@pytest.mark.parametrize("attention", ["sdpa", "hip"])
def test_greedy_decoder_graph_equals_eager(gpu_device, kv_bits, attention):
    """Tokens, logits and log probabilities of the captured step are the eager step's."""
    from qwendopamine_amd.hybrid import GreedyDecoder

    print(f"[case] greedy decoding kv_bits {kv_bits} attention {attention}", flush=True)
    m = _model(BF, gpu_device, attention=attention)
    prompt = torch.randint(0, 1000, (2, 70), device=gpu_device, generator=torch.Generator(gpu_device).manual_seed(2))
    runs = []
    for use_graph in (False, True):
        dec = GreedyDecoder(m, use_graph=use_graph, keep_logits=True, kv_bits=kv_bits, keep_logprobs=4)
        toks = dec.generate(prompt, 12)
        torch.cuda.synchronize()
        runs.append((toks, dec.logits.clone(), dec.sequence_logprobs))
    (t0, l0, s0), (t1, l1, s1) = runs
    assert torch.equal(t0, t1) and torch.equal(l0, l1) and all(torch.equal(a, b) for a, b in zip(s0, s1))
    assert s0.logprobs.shape == (2, 12) and s0.top_ids.shape == (2, 12, 4)
    assert torch.equal(s0.top_ids[..., 0], t0) and torch.equal(s0.top_logprobs[..., 0], s0.logprobs)
    want = l0.double().log_softmax(-1).gather(-1, t0[:, -1:])[:, 0]
    assert float((s0.logprobs[:, -1].double() - want).abs().max()) <= 2e-5


def test_decoder_without_alternatives_or_logprobs(gpu_device):
    from qwendopamine_amd.hybrid import GreedyDecoder

    m = _model(BF, gpu_device)
    prompt = torch.randint(0, 1000, (1, 9), device=gpu_device)
    a = GreedyDecoder(m, keep_logprobs=0)
    ta = a.generate(prompt, 5)
    b = GreedyDecoder(m)
    assert torch.equal(ta, b.generate(prompt, 5)) and b.sequence_logprobs is None
    assert a.sequence_logprobs.logprobs.shape == (1, 5) and a.sequence_logprobs.top_ids is None
    # The prompt gives a token whatever the number asked for.
    assert torch.equal(a.generate(prompt, 0), ta[:, :1]) and a.sequence_logprobs.logprobs.shape == (1, 1)


def test_four_bit_layer_is_the_operator(gpu_device):
    """The model's cached prefill stores its rotated keys and values, and its decode step is the
    operator over them; a prompt of a single token as well."""
    from qwendopamine_amd import ops
    from qwendopamine_amd.hybrid import apply_rotary_emb

    m = _model(BF, gpu_device, layers=(), n_layer=1)
    at = m.h[0].attn
    x = torch.randn(2, 33, 256, device=gpu_device).to(BF)
    with torch.no_grad():
        for t in (33, 1):
            m.setup_caches(2, 50, kv_bits=4)
            assert isinstance(at.kv_cache, ops.KVCacheQ4)
            cos, sin = m._rope_tables(50, x.device)
            pos = torch.arange(t, device=gpu_device)
            at(x[:, :t], cos[:t], sin[:t], pos)
            want = ops.kv_cache_q4(2, 2, 50, 64, gpu_device)
            qkv = ops.linear(x[:, :t], at.attn.weight).view(2, t, 2, 4, 64)
            k = apply_rotary_emb(qkv[..., 2, :], cos[:t], sin[:t]) if t > 1 else qkv[..., 2, :]  # position 0: identity
            ops.kv_cache_q4_store(want, k, qkv[..., 3, :])
            assert all(torch.equal(a, b) for a, b in zip(at.kv_cache, want))
            y = torch.randn(2, 1, 256, device=gpu_device).to(BF)
            pos = torch.tensor([t], device=gpu_device)
            got = at(y, cos[t:t + 1], sin[t:t + 1], pos)
            o = ops.attention_decode_q4(ops.linear(y, at.attn.weight), cos, sin, pos, want, 4)
            assert torch.equal(got, ops.linear(o.reshape(2, 1, 256), at.proj.weight))
            assert all(torch.equal(a, b) for a, b in zip(at.kv_cache, want))
    m.setup_caches(2, 20, kv_bits=4)
    with torch.no_grad(), pytest.raises(ValueError):
        at(x, cos[:33], sin[:33], torch.arange(33, device=gpu_device))  # a prompt longer than the cache
    m.setup_caches(2, 50, kv_bits=4)
    with pytest.raises(NotImplementedError):
        at(x[:, :1], cos[:1], sin[:1], torch.tensor([0], device=gpu_device))  # gradients through a 4-bit step


def test_head_size_128_and_float32_fall_back_or_run(gpu_device):
    """``attention='hip'`` runs heads of 128 channels; a float32 model keeps torch's attention, and
    refuses a 4-bit cache."""
    idx = torch.randint(0, 1000, (2, 50), device=gpu_device)
    for kw in (dict(head_size=128, n_head=2, n_query_groups=1), dict(head_size=64)):
        a = _model(BF, gpu_device, layers=(), n_layer=2, **kw)
        b = _model(BF, gpu_device, attention="sdpa", layers=(), n_layer=2, **kw)
        b.load_state_dict(a.state_dict())
        with torch.no_grad():
            # Two bf16 attentions, each output half a step from the exact one, through two layers.
            assert rel_l2(a(idx).float(), b(idx).float()) <= 2e-2
    a, b = _model(torch.float32, gpu_device, layers=()), _model(torch.float32, gpu_device, attention="sdpa", layers=())
    b.load_state_dict(a.state_dict())
    with torch.no_grad():
        assert torch.equal(a(idx), b(idx))
    with pytest.raises(NotImplementedError):
        a.setup_caches(1, 10, kv_bits=4)
