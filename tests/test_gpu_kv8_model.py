"""The 8-bit cache and the log-probabilities where they are used: the decode harness
(`llama_decode.DecodeModel`, attention="kv8") and its prompt scoring.

Tolerances: a cached value is off by at most half a step, max |x| / 254 of its page: for Gaussian
pages of 1024 values (max ~ 3.5 sigma) an error of 0.4% of sigma rms in k and v each, which the
attention's mean over 17 or more positions does not enlarge; two random-init layers and bf16
activations (2^-8) bring the logits to within 3%.
"""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from llm_serving_engine_b200 import _lib, ops
from llm_serving_engine_b200.llama_decode import DecodeModel, LlamaShape, decode_bytes_per_step

pytestmark = pytest.mark.gpu

TINY = LlamaShape(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, intermediate=512, vocab=1000)


def _models(batch, context, quantize=True):
    paged = DecodeModel(TINY, batch=batch, context=context, device="cuda", seed=5, quantize=quantize)
    kv8 = DecodeModel(TINY, batch=batch, context=context, device="cuda", seed=5, quantize=quantize, weights=paged.weights,
                      attention="kv8")
    return paged, kv8


@pytest.mark.parametrize("batch,context", [(4, 16), (24, 70)])
def test_step_matches_the_bf16_cache(batch, context):
    paged, kv8 = _models(batch, context)
    tokens = (torch.arange(batch, device="cuda") * 37) % TINY.vocab
    a, b = kv8.logits(tokens), paged.logits(tokens)
    assert float((a - b).norm() / b.norm()) < 3e-2
    assert torch.equal(a, kv8.logits(tokens))  # the caches were left alone
    assert ops.device_status() == _lib.LSE_OK


def test_step_appends_to_the_cache_and_answers_with_logprobs():
    _, kv8 = _models(4, 40)
    tokens = torch.tensor([3, 1, 4, 1], device="cuda")
    logits = kv8.logits(tokens)
    page = kv8.kv["block_table"][:, 40 // 16].long()
    before = kv8.kv["cache"][1].k[page, :, 40 % 16].clone()
    chosen, lp = kv8.step_logprobs(tokens, top_k=3)
    assert not torch.equal(before, kv8.kv["cache"][1].k[page, :, 40 % 16])
    ref = torch.log_softmax(logits.double(), -1)
    assert torch.equal(chosen, logits.argmax(-1)) and torch.equal(lp.top_ids[:, 0], chosen)
    assert torch.allclose(lp.logprob.double(), ref.gather(1, chosen[:, None])[:, 0], atol=1e-5)
    assert torch.allclose(lp.entropy.double(), torch.special.entr(ref.exp()).sum(-1), atol=1e-4)
    assert torch.equal(kv8.step(tokens), chosen)


def test_step_in_a_cuda_graph():
    _, kv8 = _models(8, 33)
    tokens = torch.arange(8, device="cuda") * 11
    want = kv8.step_logprobs(tokens, 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        kv8.step_logprobs(tokens, 2)
        with torch.cuda.graph(graph, stream=stream):
            held = kv8.step_logprobs(tokens, 2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want[0], held[0])
    for a, b in zip(want[1], held[1]):
        assert torch.equal(a, b)


def _plain_logits(model, weights, prompt):
    """The network in fp32 on one prompt, with torch's own attention."""
    s, hd, T = TINY, TINY.head_dim, prompt.shape[0]
    inv = 1.0 / (s.rope_theta ** (torch.arange(0, hd, 2, device="cuda").float() / hd))
    ang = torch.arange(T, device="cuda").float()[:, None] * inv
    cos, sin = torch.cat([ang, ang], 1).cos(), torch.cat([ang, ang], 1).sin()
    norm = lambda x: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s.eps)
    turn = lambda x: x * cos + torch.cat([-x[..., hd // 2:], x[..., :hd // 2]], -1) * sin
    h = model.embed[prompt].float()
    for wqkv, wo, wgu, wd in weights:
        q, k, v = (norm(h) @ wqkv.float().T).view(T, -1, hd).transpose(0, 1).split([s.heads, s.kv_heads, s.kv_heads])
        o = F.scaled_dot_product_attention(turn(q)[None], turn(k)[None], v[None], is_causal=True, enable_gqa=True)[0]
        h = h + o.transpose(0, 1).reshape(T, -1) @ wo.float().T
        gu = norm(h) @ wgu.float().T
        h = h + (F.silu(gu[:, :s.intermediate]) * gu[:, s.intermediate:]) @ wd.float().T
    return norm(h) @ model.lm_head.float().T


@pytest.mark.parametrize("lens", [[1], [200], [5, 130, 1, 64, 17]])
def test_score_of_packed_prompts(lens):
    """Every position's log-probability, entropy and likeliest token against the network in fp32; logits
    agree to 3% of their norm (see above), and log-probabilities by twice the largest difference."""
    _, kv8 = _models(2, 16, quantize=False)
    gen = torch.Generator().manual_seed(len(lens))
    prompts = [torch.randint(0, TINY.vocab, (n,), generator=gen) for n in lens]
    out = kv8.score(prompts, top_k=1)
    assert out.logprob.shape == (sum(lens),) and out.top_ids.shape == (sum(lens), 1)
    row = 0
    for p in prompts:
        n = p.shape[0]
        logits = _plain_logits(kv8, kv8.weights, p.cuda())
        ref = torch.log_softmax(logits, -1)
        spread = float(logits.std(-1).mean())
        # 3% of the norm is 0.03 spread rms a logit; the largest of 1000 within 5 of those
        tol = 2 * 5 * 0.03 * spread
        got = out.logprob[row:row + n - 1]
        if n > 1:
            assert float((got - ref[:-1].gather(1, p.cuda()[1:, None])[:, 0]).abs().max()) < tol
        assert torch.isnan(out.logprob[row + n - 1])
        assert float((out.entropy[row:row + n] - torch.special.entr(ref.exp()).sum(-1)).abs().max()) < tol
        top = out.top_logprobs[row:row + n, 0]
        assert float((top - ref.amax(-1)).abs().max()) < tol
        row += n
    with pytest.raises(ValueError):
        kv8.score([])


def test_bytes_of_a_step_with_an_8_bit_cache():
    full = decode_bytes_per_step(TINY, 8, 1023, True)
    half = decode_bytes_per_step(TINY, 8, 1023, True, kv8=True)
    kv = 2 * TINY.layers * 8 * TINY.kv_heads * 1024 * TINY.head_dim
    assert full - half == kv - 2 * 4 * TINY.layers * 8 * TINY.kv_heads * 64
