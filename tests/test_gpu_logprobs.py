"""`ops.token_logprobs` against the float64 oracle.

Tolerances, by derivation: each exp has a relative error of a few 2^-24 and so has their fp32 sum,
its logarithm at most 2^-20 absolute; x - max is rounded once (2^-24 |x - max|).  logprob:
2^-19 + 2^-22 |ref|.  The entropy adds the mean of |x - max| with the same relative errors: at most
log Z + H of it, 2^-19 + 2^-20 (H + log V).  Ids are exact.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from llm_serving_engine_b200 import _lib, ops
from oracle.ref_kv8 import ref_logprobs

pytestmark = pytest.mark.gpu


def _check(x, tokens, k):
    got = ops.token_logprobs(x, tokens, k)
    V = x.shape[-1]
    lp, ent, top, ids = ref_logprobs(x.reshape(-1, V).float().cpu().numpy(),
                                     None if tokens is None else tokens.reshape(-1).cpu().numpy(), k)
    close = lambda a, b, tol: np.all((a == b) | (np.isnan(a) & np.isnan(b)) | (np.abs(a - b) <= tol))
    f = lambda t: t.cpu().numpy().astype(np.float64)
    with np.errstate(invalid="ignore"):
        if tokens is None:
            assert got.logprob.numel() == 0
        else:
            assert got.logprob.shape == x.shape[:-1] and close(f(got.logprob).ravel(), lp, 2.0 ** -19 + 2.0 ** -22 * np.abs(lp))
        assert close(f(got.entropy).ravel(), ent, 2.0 ** -19 + 2.0 ** -20 * (np.abs(ent) + np.log(V)))
        assert got.top_logprobs.shape == (*x.shape[:-1], k)
        assert close(f(got.top_logprobs).reshape(len(lp), k), top, 2.0 ** -19 + 2.0 ** -22 * np.abs(top))
    assert np.array_equal(got.top_ids.cpu().numpy().reshape(len(lp), k), ids)
    return got


def _logits(M, V, dtype, seed, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(M, V, generator=gen) * spread).to(dtype).cuda(), torch.randint(0, V, (M,), generator=gen).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,V,k", [(1, 1, 1), (2, 7, 3), (3, 33, 33), (5, 511, 20), (2, 513, 0), (4, 4096, 1), (3, 50257, 20),
                                   (1, 128256, 5), (2, 128256, 128), (40, 8191, 8), (300, 1003, 4)])
def test_against_the_oracle(M, V, k, dtype):
    x, tokens = _logits(M, V, dtype, seed=V + k)
    got = _check(x, tokens, k)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.token_logprobs(x, tokens, k)))
    assert ops.device_status() == _lib.LSE_OK


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,V,k", [(3, 8192, 20), (70, 9001, 33), (2, 32000, 128), (1, 37001, 128), (2, 50257, 128), (2, 66000, 128)])
def test_more_alternatives_than_groups(M, V, k, dtype):
    x, tokens = _logits(M, V, dtype, seed=11 * V + k)
    _check(x, tokens, k)


def test_leading_shape_and_no_tokens():
    x, tokens = _logits(6, 1000, torch.bfloat16, seed=1)
    _check(x.view(2, 3, 1000), tokens.view(2, 3), 4)
    _check(x, None, 4)
    _check(x[0], tokens[0], 2)
    empty = ops.token_logprobs(x[:0], tokens[:0], 3)
    assert empty.entropy.shape == (0,) and empty.top_ids.shape == (0, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_odd_starts(dtype):
    wide, tokens = _logits(9, 3001, dtype, seed=2)
    _check(wide[:, 1:2990], tokens.clamp(max=2988), 7)  # rows that start at any element
    _check(wide[::2, 3:], tokens[::2].clamp(max=2997), 7)
    _check(wide.t().contiguous().t()[:, :50], tokens.clamp(max=49), 3)  # column-major: copied


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_ties_go_to_the_lowest_index(dtype):
    """Constant rows, rows of two values, and runs of equal values across the row."""
    V = 20011
    x = torch.zeros(5, V, dtype=dtype, device="cuda")
    x[1] = -3.0
    x[2, V // 2:] = 1.0
    x[3, ::97] = 2.0
    x[4] = torch.arange(V, device="cuda").remainder(5).to(dtype)
    x[0, ::2] = -0.0  # equal to 0
    tokens = torch.tensor([0, V - 1, V // 2, 97, 4], device="cuda")
    for k in (1, 20, 128):
        _check(x, tokens, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masks(dtype):
    """-inf and the type's lowest value as masks, one live token, none at all."""
    x, tokens = _logits(7, 5000, dtype, seed=3)
    low = torch.finfo(dtype).min
    x[0, torch.arange(5000, device="cuda") % 3 != 0] = -float("inf")
    x[1, 100:] = low
    x[2] = -float("inf")
    x[2, 4321] = 1.5
    x[3] = -float("inf")
    x[4] = low
    x[5] = -float("inf")
    x[5, 10:20] = low
    tokens[:6] = torch.tensor([3, 50, 4321, 17, 9, 15], device="cuda")
    _check(x, tokens, 20)
    tokens[:6] = torch.tensor([1, 200, 0, 4999, 4999, 0], device="cuda")
    _check(x, tokens, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_nan_and_infinity(dtype):
    x, tokens = _logits(5, 3000, dtype, seed=4)
    x[0, 2999] = float("nan")
    x[1, 0] = float("inf")
    x[2, [5, 7]] = float("nan")
    x[3, 100] = -float("nan")
    got = _check(x, tokens, 6)
    assert torch.isnan(got.entropy[:4]).all() and torch.isfinite(got.entropy[4])


@pytest.mark.parametrize("shift", [0.0, 3.0e4, -3.0e4])
def test_large_offsets_and_peaks(shift):
    x, tokens = _logits(4, 9001, torch.float32, seed=5, spread=30.0)
    _check(x + shift, tokens, 9)
    x[:, 77] = 1.0e4 + shift
    _check(x, tokens, 9)


def test_tokens_out_of_range_are_reported():
    x, tokens = _logits(3, 100, torch.bfloat16, seed=6)
    ops.device_status()
    tokens[0], tokens[2] = -1, 100
    got = ops.token_logprobs(x, tokens, 2)
    assert ops.device_status() == _lib.LSE_ERR_INVALID_ARG
    assert torch.isnan(got.logprob[[0, 2]]).all() and torch.isfinite(got.logprob[1]) and torch.isfinite(got.entropy).all()


def test_streams_and_graphs():
    x, tokens = _logits(3, 128256, torch.bfloat16, seed=7)
    want = ops.token_logprobs(x, tokens, 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        other = ops.token_logprobs(x, tokens, 20)
        with torch.cuda.graph(graph, stream=side):
            held = ops.token_logprobs(x, tokens, 20)
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, other, held):
        assert torch.equal(a, b) and torch.equal(a, c)
