"""The hybrid decoder with query and key norms, paged key / value caches and drawn tokens."""

from __future__ import annotations

import pytest
import torch

from qwendopamine_amd import ops
from qwendopamine_amd.hybrid import GreedyDecoder, HybridConfig, HybridDecoder, SamplingDecoder
from qwendopamine_amd.hybrid import apply_rotary_emb, build_rope_cache
from tests._helpers import REL_TOL, rel_l2

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def _model(dtype, dev, layers=(0, 2), **kw):
    torch.manual_seed(0)
    cfg = dict(n_layer=4, n_embd=256, n_head=4, head_size=64, n_query_groups=2, intermediate_size=512, vocab_size=1000,
               gdn2_layers=list(layers), block_size=512, attention="hip")
    m = HybridDecoder(HybridConfig(**{**cfg, **kw}))
    for n, p in m.named_parameters():
        if "q_norm" in n or "k_norm" in n:
            torch.nn.init.normal_(p, 1.0, 0.3)
    return m.to(dev, dtype).eval()


def _ids(dev, B=3, T=70, seed=1):
    return torch.randint(0, 1000, (B, T), generator=torch.Generator().manual_seed(seed)).to(dev)


def test_query_and_key_norms_train_as_on_the_cpu(gpu_device):
    """Attention layers alone, float32 on the GPU against float64 torch operations on the CPU: the loss, and every
    gradient, the norms' weights among them."""
    m = _model(F32, gpu_device, layers=(), qk_norm=True, attention="sdpa")
    ref = _model(torch.float64, "cpu", layers=(), qk_norm=True, attention="sdpa")
    ref.load_state_dict(m.state_dict())
    idx = _ids("cpu", 2, 33)
    out, want = m(idx.to(gpu_device)), ref(idx)
    assert rel_l2(out, want) <= REL_TOL[F32]
    w = torch.randn(want.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    (out.double() * w.to(gpu_device)).sum().backward()
    (want * w).sum().backward()
    for (n, p), (_, q) in zip(m.named_parameters(), ref.named_parameters()):
        assert rel_l2(p.grad, q.grad) <= REL_TOL[F32], n


@pytest.mark.parametrize("qk_norm", [False, True])
def test_paged_cache_decodes_as_the_whole_sequence(gpu_device, qk_norm):
    """Prefill and single tokens, over pages and over the contiguous cache: as near the same weights in float32 as one
    bf16 forward over the whole sequence is, whose roundings are of the same kind and number (a quarter more for
    their chance)."""
    m = _model(BF, gpu_device, qk_norm=qk_norm)
    full = _model(F32, gpu_device, qk_norm=qk_norm)
    full.load_state_dict(m.state_dict())
    idx = _ids(gpu_device)
    with torch.no_grad():
        whole = full(idx)
        base = rel_l2(m(idx), whole)
        runs = []
        for page_size in (16, 64, None):
            m.setup_caches(3, 80, page_size=page_size)
            out = [m(idx[:, :50], input_pos=torch.arange(50, device=gpu_device))]
            out += [m(idx[:, i:i + 1], input_pos=torch.tensor([i], device=gpu_device)) for i in range(50, 70)]
            runs.append(torch.cat(out, 1))
    for r in runs:
        assert rel_l2(r, whole) <= 1.25 * base
    assert torch.equal(runs[0], runs[1])  # whatever the pages' size


def test_greedy_and_drawn_tokens(gpu_device):
    """Captured and eager steps give the same tokens; a generator's seed decides them; temperature 0 and a single
    candidate are greedy."""
    m = _model(BF, gpu_device, qk_norm=True)
    prompt = _ids(gpu_device, 3, 20)
    greedy = GreedyDecoder(m, page_size=16).generate(prompt, 12)
    assert torch.equal(greedy, GreedyDecoder(m, use_graph=False, page_size=16).generate(prompt, 12))
    # The contiguous cache, whose decode step has no norms of its own: torch operations around the pass.
    assert torch.equal(GreedyDecoder(m).generate(prompt, 12), GreedyDecoder(m, use_graph=False).generate(prompt, 12))

    def drawn(seed, **kw):
        g = torch.Generator(gpu_device).manual_seed(seed)
        return SamplingDecoder(m, generator=g, **{"page_size": 16, **kw}).generate(prompt, 12)
    assert torch.equal(drawn(1, temperature=0.0), greedy)
    assert torch.equal(drawn(1, top_k=1), greedy)
    a = drawn(2, temperature=1.5, top_p=0.95)
    assert torch.equal(a, drawn(2, temperature=1.5, top_p=0.95, use_graph=False))
    assert not torch.equal(a, drawn(3, temperature=1.5, top_p=0.95))
    each = drawn(2, temperature=torch.tensor([0.0, 1.5, 1.5], device=gpu_device), top_p=0.95)
    assert torch.equal(each[0], greedy[0]) and torch.equal(each[1:], a[1:])
    assert a.shape == greedy.shape == (3, 12) and a.min() >= 0 and a.max() < 1000


def test_drawn_tokens_are_the_definitions(gpu_device):
    """Each drawn token is ``ops.sample_tokens`` of the step's logits at the step's numbers; with log probabilities kept."""
    m = _model(BF, gpu_device)
    prompt = _ids(gpu_device, 2, 9)
    kw = dict(temperature=1.2, top_k=40, top_p=0.9, min_p=0.01)
    dec = SamplingDecoder(m, generator=torch.Generator(gpu_device).manual_seed(5), keep_logits=True, keep_logprobs=3, **kw)
    tok = dec.prefill(prompt, 8)
    for i in range(7):
        want = ops.sample_tokens(dec.logits.to(BF), dec.uniforms, **kw)
        assert torch.equal(tok[:, 0], want)
        assert dec.logprobs.logprobs.isfinite().all()
        tok = dec.step().clone()


def test_refusals(gpu_device):
    m = _model(BF, gpu_device, qk_norm=True)
    with pytest.raises(NotImplementedError):
        m.setup_caches(1, 32, kv_bits=4)
    with pytest.raises(NotImplementedError):
        m.setup_caches(1, 32, kv_bits=4, page_size=16)
    with pytest.raises(NotImplementedError):
        m.setup_caches(1, 32, page_size=8)
    with pytest.raises(NotImplementedError):
        _model(F32, gpu_device).setup_caches(1, 32, page_size=16)
    m.setup_caches(1, 32, page_size=16)
    with pytest.raises(NotImplementedError):  # gradients
        m(_ids(gpu_device, 1, 5), input_pos=torch.arange(5, device=gpu_device))


def test_norms_that_train_are_refused_over_pages(gpu_device):
    """Over a frozen projection, too: a step through the pages would take their gradients for nothing."""
    m = _model(BF, gpu_device, layers=(), qk_norm=True).requires_grad_(False)
    m.setup_caches(1, 32, page_size=16)
    idx, pos = _ids(gpu_device, 1, 5), torch.arange(5, device=gpu_device)
    assert m(idx, input_pos=pos).shape == (1, 5, 1000)
    m.h[1].attn.k_norm.weight.requires_grad_(True)
    with pytest.raises(NotImplementedError):
        m(idx, input_pos=pos)
    with torch.no_grad():
        assert m(idx, input_pos=pos).shape == (1, 5, 1000)


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("how", ["float32", "bfloat16", "float64", "strided", "trained", "one row"])
def test_attention_layer_takes_tables_of_any_kind(gpu_device, how, qk_norm):
    """By itself, with a caller's own rotation tables: queries and keys are the torch operations' on those tables."""
    at = _model(BF, gpu_device, layers=(), qk_norm=qk_norm).h[0].attn
    T, H, G, D = 9, at.n_head, at.n_query_groups, at.head_size
    cos, sin = build_rope_cache(T, D, gpu_device)
    if how in ("bfloat16", "float64"):
        cos, sin = (x.to(getattr(torch, how)) for x in (cos, sin))
    elif how == "strided":
        cos, sin = (x.T.contiguous().T for x in (cos, sin))
    elif how == "one row":
        cos, sin = cos[3:4], sin[3:4]
    elif how == "trained":
        cos.requires_grad_(True)
    x = torch.randn(2, T, 256, generator=torch.Generator().manual_seed(3)).to(BF).to(gpu_device)
    qkv = at.attn(x)
    q, k, v = at._heads(qkv, cos, sin)
    wq, wk, wv = qkv.view(2, T, G, H // G + 2, D).split((H // G, 1, 1), dim=-2)
    wq, wk = wq.reshape(2, T, H, D), wk.reshape(2, T, G, D)
    if qk_norm:
        wq, wk = at.q_norm(wq), at.k_norm(wk)
    assert torch.equal(v, wv.reshape(2, T, G, D))
    for got, want in ((q, apply_rotary_emb(wq, cos, sin)), (k, apply_rotary_emb(wk, cos, sin))):
        if how == "float32" and qk_norm:
            assert rel_l2(got, want) <= REL_TOL[BF]  # torch's norm rounds every operation
        else:
            assert torch.equal(got, want)
    o = at(x, cos, sin)
    assert o.shape == x.shape and o.isfinite().all()
    if how == "trained":
        (g,) = torch.autograd.grad(o.float().sum(), cos)
        assert g.shape == cos.shape and g.isfinite().all() and (g != 0).any()


def test_prompt_in_pieces(gpu_device):
    """A prompt in pieces and then single tokens through attention layers over pages (gdn2 layers begin their short
    convolutions anew in every call of several tokens, as the reference's do): as near the weights in float32 as one
    bf16 forward over the whole sequence (a quarter more for the roundings' chance)."""
    m = _model(BF, gpu_device, layers=(), qk_norm=True)
    full = _model(F32, gpu_device, layers=(), qk_norm=True)
    full.load_state_dict(m.state_dict())
    idx = _ids(gpu_device, 2, 70)
    with torch.no_grad():
        whole = full(idx)
        base = rel_l2(m(idx), whole)
        m.setup_caches(2, 80, page_size=16)
        out, at = [], 0
        for n in (30, 1, 25, 13, 1):
            out.append(m(idx[:, at:at + n], input_pos=torch.arange(at, at + n, device=gpu_device)))
            at += n
    assert rel_l2(torch.cat(out, 1), whole) <= 1.25 * base
