"""The 8-bit paged K/V cache (`ops.kv8_rope_append`, `kv8_read`, `kv8_decode_attention`,
`kv8_paged_attention`) against the float64 oracle.

Tolerances, by derivation: with u the unit roundoff of the element type (2^-8 bf16, 2^-11 fp16),
* q and read values carry one rounding, u |x|, on top of fp32 arithmetic (2^-22 of the operands);
* a page's scale is an fp32 maximum of fp32 values: 2^-21 of max |x| sqrt(2) / 127;
* a code is rint(x / s) with x and s off by 2^-21: within 1/2 + 127 * 2^-20 of the exact quotient;
* attention rounds its output once (u |o|) and its weights to 11 bits or better before they meet V;
  2^-10 of sum_p w_p |v_p| covers that and the fp32 softmax.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from llm_serving_engine_b200 import _lib, ops
from oracle.ref_kv8 import ref_append, ref_attention, ref_rotate

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _i32(a):
    return torch.as_tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _np(t):
    return t.detach().float().cpu().numpy().astype(np.float64) if t.is_floating_point() else t.cpu().numpy()


def _table(lens, bs, gen, spare=2, extra_cols=0):
    pages = [-(-int(n) // bs) for n in lens]
    nb = sum(pages) + spare
    ids = torch.randperm(nb, generator=gen)[: sum(pages)].to(torch.int32)
    table = torch.full((len(lens), max(pages + [1]) + extra_cols), -1, dtype=torch.int32)
    at = 0
    for e, n in enumerate(pages):
        table[e, :n] = ids[at:at + n]
        at += n
    return table, nb


def _random_cache(nb, H_kv, bs, D, gen):
    k = torch.randint(-127, 128, (nb, H_kv, bs, D), generator=gen, dtype=torch.int8)
    v = torch.randint(-127, 128, (nb, H_kv, bs, D), generator=gen, dtype=torch.int8)
    sk = torch.rand(nb, H_kv, generator=gen) * 0.02 + 1e-3
    sv = torch.exp(torch.randn(nb, H_kv, generator=gen) * 2) * 0.01  # pages of very different sizes
    return ops.Kv8Cache(k.cuda(), v.cuda(), sk.cuda(), sv.cuda())


# ------------------------------------------------------------------------------------ append
def _append_case(H, H_kv, D, bs, q_len, offset, dtype, R, interleaved, cs_dtype, seed, pad=0, gap=1):
    gen = torch.Generator().manual_seed(seed)
    q_len, offset = np.asarray(q_len), np.asarray(offset)
    start, row = np.zeros_like(q_len), 0
    for e, n in enumerate(q_len):
        row += gap
        start[e] = row
        row += n
    M = row + gap
    table, nb = _table(np.maximum(offset + q_len, 1), bs, gen)
    cache = _random_cache(nb, H_kv, bs, D, gen)
    wide = torch.randn(M, (H + 2 * H_kv) * D + pad, generator=gen) * 3
    qkv = wide.to(dtype).cuda()[:, : (H + 2 * H_kv) * D]
    cos = sin = None
    if R:
        ang = torch.rand(M, R // 2, generator=gen) * 6.3
        ang = ang.repeat_interleave(2, 1) if interleaved else torch.cat([ang, ang], 1)
        cos, sin = ang.cos().to(cs_dtype).cuda(), ang.sin().to(cs_dtype).cuda()
    return dict(qkv=qkv, H=H, cache=cache, table=table.cuda(), offset=offset, start=start, q_len=q_len, cos=cos, sin=sin,
                interleaved=interleaved, bs=bs)


def _run_append(c):
    return ops.kv8_rope_append(c["qkv"], c["H"], c["cache"], c["table"], _i32(c["offset"]), _i32(c["start"]),
                               _i32(c["q_len"]), c["cos"], c["sin"], c["interleaved"])


def _check_append(c, q, before):
    cache, H = c["cache"], c["H"]
    H_kv, D = cache.k.shape[1], cache.k.shape[3]
    M, dt = c["qkv"].shape[0], c["qkv"].dtype
    x = _np(c["qkv"]).reshape(M, H + 2 * H_kv, D)
    turned = x.copy()
    if c["cos"] is not None:
        turned[:, : H + H_kv] = ref_rotate(x[:, : H + H_kv], _np(c["cos"]), _np(c["sin"]), c["interleaved"])
    ref_q = turned[:, :H].transpose(1, 0, 2)
    size = np.abs(x).max()
    assert np.all(np.abs(_np(q) - ref_q) <= UNIT[dt] * np.abs(ref_q) + 2.0 ** -22 * 2 * size + 2.0 ** -25)
    for which, (codes0, scale0, codes, scale) in enumerate(
            [(before.k, before.k_scale, cache.k, cache.k_scale), (before.v, before.v_scale, cache.v, cache.v_scale)]):
        new = turned[:, H + which * H_kv:H + (which + 1) * H_kv]
        ref_c, ref_s, exact = ref_append(_np(codes0), _np(scale0), new, _np(c["table"]), c["offset"], c["start"],
                                         c["q_len"], c["bs"])
        got_s, got_c = _np(scale), _np(codes).astype(np.float64)
        assert np.all(np.abs(got_s - ref_s) <= 2.0 ** -21 * (np.abs(ref_s) + 1.5 * size / 127))
        # within half a step of the exact quotient (a tie may fall either way), and never past 127
        assert np.all(np.abs(got_c - np.clip(exact, -127, 127)) <= 0.5 + 127 * 2.0 ** -20 * (1 + 1.5 * size / (127 * np.maximum(ref_s, 1e-30)))[:, :, None, None])
        assert np.abs(got_c).max() <= 127
        assert np.mean(got_c != ref_c) < 1e-3
        same = exact == _np(codes0)  # slots that the call leaves alone
        assert np.array_equal(got_c[same], _np(codes0).astype(np.float64)[same])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,H_kv,D,bs,R,interleaved", [
    (8, 2, 128, 16, 128, False), (8, 8, 64, 16, 64, True), (8, 1, 128, 7, 64, False), (4, 2, 64, 32, 16, True),
    (2, 2, 128, 1, 6, False), (2, 1, 128, 5, 10, True), (8, 4, 64, 128, 0, False), (16, 2, 128, 48, 2, True)])
def test_append_mixed_batch(H, H_kv, D, bs, R, interleaved, dtype):
    """Fresh prompts, chunks that start inside a page, single tokens and an empty entry."""
    c = _append_case(H, H_kv, D, bs, [1, 37, 0, 1, 150, 1, 16], [40, 0, 9, 0, 13, 31, 16], dtype, R, interleaved,
                     torch.float32, seed=D + bs + R)
    before = ops.Kv8Cache(*[t.clone() for t in c["cache"]])
    q = _run_append(c)
    _check_append(c, q, before)
    assert ops.device_status() == _lib.LSE_OK


@pytest.mark.parametrize("cs_dtype", [torch.bfloat16, torch.float16])
def test_append_strided_rows_and_16_bit_tables(cs_dtype):
    c = _append_case(8, 2, 128, 16, [21, 1], [3, 15], torch.bfloat16, 128, False, cs_dtype, seed=3, pad=24)
    assert not c["qkv"].is_contiguous()
    before = ops.Kv8Cache(*[t.clone() for t in c["cache"]])
    _check_append(c, _run_append(c), before)
    odd = _append_case(8, 2, 128, 16, [21, 1], [3, 15], torch.bfloat16, 128, False, cs_dtype, seed=3, pad=3)
    before = ops.Kv8Cache(*[t.clone() for t in odd["cache"]])
    _check_append(odd, _run_append(odd), before)  # a row stride that 16-byte loads cannot take


def test_append_many_entries():
    n = 700
    c = _append_case(2, 1, 64, 16, [1] * n, [(7 * e) % 50 for e in range(n)], torch.float16, 64, False, torch.float32,
                     seed=5, gap=0)
    before = ops.Kv8Cache(*[t.clone() for t in c["cache"]])
    _check_append(c, _run_append(c), before)


def test_append_token_by_token_follows_the_growth_of_the_page():
    """16 tokens one call each into one page: every scale and code equals the oracle's, whose scale
    grows with the largest value so far and rescales the earlier codes."""
    H_kv, D, bs = 2, 64, 16
    gen = torch.Generator().manual_seed(11)
    cache = ops.kv8_cache(3, bs, H_kv, D)
    cache.k_scale.fill_(5.0)  # stale: a page whose first slot is written starts over
    x = torch.randn(bs, (2 + 2 * H_kv) * D, generator=gen) * torch.linspace(0.1, 4.0, bs)[:, None]
    x = x.to(torch.float16).cuda()
    table = _i32([[1]])
    for t in range(bs):
        before = ops.Kv8Cache(*[a.clone() for a in cache])
        c = dict(qkv=x[t:t + 1], H=2, cache=cache, table=table, offset=np.array([t]), start=np.array([0]),
                 q_len=np.array([1]), cos=None, sin=None, interleaved=False, bs=bs)
        _check_append(c, _run_append(c), before)
    k, v = ops.kv8_read(cache, torch.tensor([1], device="cuda"), torch.float16)
    want = x.view(bs, 2 + 2 * H_kv, D)[:, 2:2 + H_kv].transpose(0, 1).float()
    step = cache.k_scale[1][:, None, None]
    # half a step for the token's own rounding and at most half a step for each of its rescalings
    assert ((k[0].float() - want).abs() <= step * (bs / 2 + 1)).all()
    assert float((k[0].float() - want).norm() / want.norm()) < 0.02


def test_append_zero_page_and_values_after_it():
    cache = ops.kv8_cache(2, 16, 1, 64)
    args = (_i32([[1]]), _i32([0]), _i32([0]), _i32([3]))
    ops.kv8_rope_append(torch.zeros(3, 3 * 64, dtype=torch.bfloat16, device="cuda"), 1, cache, *args)
    assert cache.k_scale[1, 0] == 0 and not cache.k.any()
    one = torch.full((1, 3 * 64), 2.0 ** -20, dtype=torch.bfloat16, device="cuda")
    ops.kv8_rope_append(one, 1, cache, _i32([[1]]), _i32([3]), _i32([0]), _i32([1]))
    k, _ = ops.kv8_read(cache, torch.tensor([1], device="cuda"))
    assert (k[0, 0, 3] == 2.0 ** -20).all() and not k[0, 0, :3].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_append_nan_and_infinity_stay_in_their_page_and_head(bad):
    cache = ops.kv8_cache(4, 16, 2, 64)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(40, (2 + 4) * 64, generator=gen).to(torch.bfloat16).cuda()
    x[20, (2 + 1) * 64 + 5] = bad  # k head 1, position 20: the second page
    ops.kv8_rope_append(x, 2, cache, _i32([[2, 0, 3]]), _i32([0]), _i32([0]), _i32([40]))
    k, v = ops.kv8_read(cache, torch.tensor([2, 0, 3], device="cuda"))
    assert torch.isnan(k[1, 1]).all()
    assert torch.isfinite(k[1, 0]).all() and torch.isfinite(k[[0, 2]]).all() and torch.isfinite(v).all()
    # a later token does not heal the page; writing its first slot does
    ops.kv8_rope_append(x[:1], 2, cache, _i32([[2, 0, 3]]), _i32([25]), _i32([0]), _i32([1]))
    assert torch.isnan(cache.k_scale[0, 1])
    ops.kv8_rope_append(x[:1], 2, cache, _i32([[2, 0, 3]]), _i32([16]), _i32([0]), _i32([1]))
    assert torch.isfinite(cache.k_scale).all()


def test_append_bad_pages_and_rows_are_skipped_and_reported():
    cache = ops.kv8_cache(4, 16, 1, 64)
    x = torch.ones(5, 3 * 64, dtype=torch.bfloat16, device="cuda")
    ops.device_status()
    for table, off, start, n in (([[4]], 0, 0, 5), ([[-1]], 0, 0, 5), ([[1]], 16, 0, 5), ([[1]], 0, 3, 5), ([[1]], 0, -1, 3)):
        ops.kv8_rope_append(x, 1, cache, _i32(table), _i32([off]), _i32([start]), _i32([n]))
        assert ops.device_status() == _lib.LSE_ERR_INVALID_ARG
        assert not cache.k.any() and not cache.k_scale.any()
    for n in (0, -3):
        ops.kv8_rope_append(x, 1, cache, _i32([[1]]), _i32([0]), _i32([0]), _i32([n]))
        assert ops.device_status() == _lib.LSE_OK and not cache.k.any()


def test_read_values_and_bad_ids():
    gen = torch.Generator().manual_seed(2)
    cache = _random_cache(5, 2, 3, 64, gen)
    ids = torch.tensor([4, 0, 0], device="cuda")
    for dt in (torch.bfloat16, torch.float16):
        k, v = ops.kv8_read(cache, ids, dt)
        assert torch.equal(k, (cache.k[ids].float() * cache.k_scale[ids][..., None, None]).to(dt))
        assert torch.equal(v, (cache.v[ids].float() * cache.v_scale[ids][..., None, None]).to(dt))
    assert ops.kv8_read(cache, ids[:0])[0].shape == (0, 2, 3, 64)
    ops.device_status()
    k, _ = ops.kv8_read(cache, torch.tensor([5], device="cuda"))
    assert not k.any() and ops.device_status() == _lib.LSE_ERR_INVALID_ARG


# ------------------------------------------------------------------------------------ attention
def _check_attention(o, ref, size, dt):
    got = _np(o)
    assert np.all(np.isfinite(got))
    err, tol = np.abs(got - ref), UNIT[dt] * np.abs(ref) + 2.0 ** -10 * size + 2.0 ** -24
    assert np.all(err <= tol), float((err / tol).max())


def _decode(context, H, H_kv, D, bs, dtype, seed, extra_cols=0):
    gen = torch.Generator().manual_seed(seed)
    table, nb = _table(context, bs, gen, extra_cols=extra_cols)
    cache = _random_cache(nb, H_kv, bs, D, gen)
    q = (torch.randn(len(context), H, D, generator=gen) * 2).to(dtype).cuda()
    return q, cache, table.cuda()


def _ref(q, cache, table, context, **kw):
    return ref_attention(_np(q), _np(cache.k), _np(cache.v), _np(cache.k_scale), _np(cache.v_scale), _np(table), context, **kw)


CONTEXTS = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 257, 500, 1025]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,H_kv,D,bs", [(8, 2, 128, 16), (8, 8, 64, 16), (8, 1, 128, 7), (4, 2, 64, 32), (2, 2, 128, 1),
                                         (16, 2, 128, 48), (8, 1, 64, 128), (4, 1, 128, 64)])
def test_decode_attention(H, H_kv, D, bs, dtype):
    q, cache, table = _decode(CONTEXTS, H, H_kv, D, bs, dtype, seed=D + bs)
    o = ops.kv8_decode_attention(q, cache, table, _i32(CONTEXTS))
    ref, size, _ = _ref(q, cache, table, CONTEXTS)
    _check_attention(o, ref, size, dtype)
    assert torch.equal(o, ops.kv8_decode_attention(q, cache, table, _i32(CONTEXTS)))
    assert ops.device_status() == _lib.LSE_OK


@pytest.mark.parametrize("context", [[1], [40], [9000], [0, 0, 0], [5] * 300, [1, 4000] * 20, [70000, 3]])
def test_decode_attention_batches(context):
    """One sequence, long ones split over the whole GPU, many short ones, empty ones."""
    q, cache, table = _decode(context, 8, 2, 128, 16, torch.bfloat16, seed=len(context) + context[0])
    o = ops.kv8_decode_attention(q, cache, table, _i32(context))
    ref, size, _ = _ref(q, cache, table, context)
    _check_attention(o, ref, size, torch.bfloat16)


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
def test_decode_attention_scales_and_strides(scale):
    context = [33, 130]
    q, cache, table = _decode(context, 8, 2, 128, 16, torch.float16, seed=4, extra_cols=3)
    ref, size, _ = _ref(q, cache, table, context, scale=scale)
    _check_attention(ops.kv8_decode_attention(q, cache, table, _i32(context), scale), ref, size, torch.float16)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    _check_attention(ops.kv8_decode_attention(turned, cache, table, _i32(context), scale), ref, size, torch.float16)
    odd = torch.empty(2, 8, 131, dtype=q.dtype, device="cuda")[..., 1:129].copy_(q)
    _check_attention(ops.kv8_decode_attention(odd, cache, table, _i32(context), scale), ref, size, torch.float16)


def test_decode_attention_large_scores_and_extreme_pages():
    """Scores of many hundreds (one position takes everything), pages of zeros, pages of very small
    and very large values."""
    context = [400, 400]
    q, cache, table = _decode(context, 8, 2, 128, 16, torch.bfloat16, seed=8)
    cache.k_scale.mul_(40.0)
    cache.v_scale[::3] = 0.0
    cache.v_scale[1::3] *= 2.0 ** -30
    ref, size, _ = _ref(q, cache, table, context)
    _check_attention(ops.kv8_decode_attention(q, cache, table, _i32(context)), ref, size, torch.bfloat16)
    cache.v_scale.zero_()
    assert not ops.kv8_decode_attention(q, cache, table, _i32(context)).any()


def test_decode_attention_bad_blocks_and_long_contexts():
    context = [64, 64]
    q, cache, table = _decode(context, 4, 1, 64, 16, torch.bfloat16, seed=9)
    table[0, 1] = -1
    table[1, :] = cache.k.shape[0]
    ops.device_status()
    o = ops.kv8_decode_attention(q, cache, table, _i32(context))
    assert ops.device_status() == _lib.LSE_ERR_INVALID_ARG
    ref, size, _ = _ref(q, cache, table, context)
    _check_attention(o, ref, size, torch.bfloat16)
    assert not o[1].any()  # nothing to attend to
    q, cache, table = _decode(context, 4, 1, 64, 16, torch.bfloat16, seed=10)
    o = ops.kv8_decode_attention(q, cache, table, _i32([70, -5]))  # past the table: cut to 64
    assert ops.device_status() == _lib.LSE_ERR_INVALID_ARG
    ref, size, _ = _ref(q, cache, table, [64, 0])
    _check_attention(o, ref, size, torch.bfloat16)


def test_nan_reaches_only_those_who_attend_to_it():
    context = [40, 40]
    q, cache, table = _decode(context, 4, 2, 64, 16, torch.bfloat16, seed=12)
    cache.k_scale[int(table[0, 1]), 0] = float("nan")
    cache.v_scale[int(table[1, 2]), 1] = float("nan")
    o = ops.kv8_decode_attention(q, cache, table, _i32(context))
    assert torch.isnan(o[0, :2]).all() and torch.isfinite(o[0, 2:]).all()
    assert torch.isnan(o[1, 2:]).all() and torch.isfinite(o[1, :2]).all()
    # a causal prompt: rows before the page never see it
    q = torch.randn(4, 40, 64, device="cuda").to(torch.bfloat16)
    o = ops.kv8_paged_attention(q, cache, table[1:].contiguous(), _i32([40]), _i32([0]), _i32([0]), _i32([40]))
    assert torch.isfinite(o[:, :32]).all() and torch.isnan(o[2:, 32:]).all() and torch.isfinite(o[:2]).all()


def _prompt(q_len, offset, H, H_kv, D, bs, dtype, seed, gap=1):
    gen = torch.Generator().manual_seed(seed)
    q_len, offset = np.asarray(q_len), np.asarray(offset)
    start, row = np.zeros_like(q_len), 0
    for e, n in enumerate(q_len):
        row += gap
        start[e] = row
        row += n
    table, nb = _table(np.maximum(offset + q_len, 1), bs, gen)
    cache = _random_cache(nb, H_kv, bs, D, gen)
    q = (torch.randn(H, row + gap, D, generator=gen) * 2).to(dtype).cuda()
    return q, cache, table.cuda(), offset + q_len, offset, start, q_len


def _check_prompt(q, cache, table, context, offset, start, q_len, dtype, **kw):
    o = ops.kv8_paged_attention(q, cache, table, _i32(context), _i32(offset), _i32(start), _i32(q_len), **kw)
    ref, size, written = _ref(q.transpose(0, 1), cache, table, context, offset=offset, start=start, length=q_len, **kw)
    _check_attention(o.transpose(0, 1)[torch.as_tensor(written).cuda()], ref[written], size[written], dtype)
    return o


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,H_kv,D,bs", [(8, 2, 128, 16), (4, 4, 64, 16), (8, 1, 128, 7), (4, 2, 64, 32), (2, 2, 128, 1),
                                         (16, 2, 128, 48), (8, 1, 64, 128), (4, 1, 128, 64)])
def test_paged_attention_mixed_batch(H, H_kv, D, bs, dtype):
    case = _prompt([1, 37, 0, 129, 1, 70, 5], [200, 0, 9, 0, 0, 131, 300], H, H_kv, D, bs, dtype, seed=D + bs)
    o = _check_prompt(*case, dtype)
    again = ops.kv8_paged_attention(case[0], case[1], case[2], *[_i32(a) for a in case[3:]])
    rows = np.concatenate([np.arange(s, s + n) for s, n in zip(case[5], case[6])])
    assert torch.equal(o[:, rows], again[:, rows])
    assert ops.device_status() == _lib.LSE_OK


@pytest.mark.parametrize("q_len,offset", [([1], [0]), ([300], [0]), ([3], [2500]), ([64, 64], [63, 64]), ([1] * 40, list(range(40)))])
def test_paged_attention_shapes(q_len, offset):
    _check_prompt(*_prompt(q_len, offset, 4, 2, 128, 16, torch.bfloat16, seed=len(q_len)), torch.bfloat16)


def test_paged_attention_context_shorter_than_the_queries_see():
    """context_len cuts the causal range; an entry whose context is 0 gets zeros."""
    q, cache, table, context, offset, start, q_len = _prompt([20, 20, 4], [10, 0, 0], 4, 2, 64, 16, torch.float16, seed=3)
    context = np.array([15, 20, 0])
    o = _check_prompt(q, cache, table, context, offset, start, q_len, torch.float16)
    assert not o[:, start[2]:start[2] + 4].any()


@pytest.mark.parametrize("scale", [-0.2, 0.5])
def test_paged_attention_scale_and_strides(scale):
    q, *rest = _prompt([50, 9], [5, 30], 8, 2, 128, 16, torch.bfloat16, seed=7)
    _check_prompt(q, *rest, torch.bfloat16, scale=scale)
    _check_prompt(q.transpose(0, 1).contiguous().transpose(0, 1), *rest, torch.bfloat16, scale=scale)


def test_paged_attention_leaves_rows_of_no_entry_alone():
    """Through the C entry, on an output that holds something else; rows outside q are skipped and
    reported."""
    q, cache, table, context, offset, start, q_len = _prompt([5, 40], [0, 20], 4, 2, 128, 16, torch.bfloat16, seed=5, gap=3)
    lib = _lib.load()
    ws = torch.zeros(int(lib.lse_kv8_paged_attention_workspace(4, 2, 128)) + 16, dtype=torch.uint8, device="cuda")

    def call(start):
        o = torch.full_like(q, 7.0)
        t = [_i32(a) for a in (context, offset, start, q_len)]
        rc = lib.lse_kv8_paged_attention(
            q.data_ptr(), _lib.DT_BF16, q.shape[1], 4, 128, q.stride(0), q.stride(1), cache.k.data_ptr(), cache.v.data_ptr(),
            cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), cache.k.shape[0], 16, 2, table.data_ptr(), table.stride(0),
            table.shape[1], t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), t[3].data_ptr(), 2, 128 ** -0.5, o.data_ptr(),
            o.stride(0), o.stride(1), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        _lib.check(rc, "lse_kv8_paged_attention")
        torch.cuda.synchronize()
        return o

    o = call(start)
    free = np.ones(q.shape[1], dtype=bool)
    for s, n in zip(start, q_len):
        free[s:s + n] = False
    assert (o[:, torch.as_tensor(free).cuda()] == 7.0).all() and ops.device_status() == _lib.LSE_OK
    for shift in (-start[0] - 2, q.shape[1] - start[1] - 10):
        bad = start.copy()
        bad[0 if shift < 0 else 1] += shift
        call(bad)
        assert ops.device_status() == _lib.LSE_ERR_INVALID_ARG


def test_offsets_past_32_bits():
    """Pools of more than 2^32 bytes: pages at their far end."""
    H_kv, D, bs = 8, 128, 16
    nb = (1 << 32) // (H_kv * D * bs) + 40
    cache = ops.Kv8Cache(*[torch.empty(nb, H_kv, bs, D, dtype=torch.int8, device="cuda") for _ in range(2)],
                         *[torch.zeros(nb, H_kv, device="cuda") for _ in range(2)])
    gen = torch.Generator().manual_seed(6)
    n = 37
    x = torch.randn(n, (8 + 2 * H_kv) * D, generator=gen).to(torch.bfloat16).cuda()
    table = _i32([[nb - 1, nb - 7, nb - 3]])
    q = ops.kv8_rope_append(x, 8, cache, table, _i32([0]), _i32([0]), _i32([n]))
    small = ops.Kv8Cache(*[t[[nb - 1, nb - 7, nb - 3]].contiguous() for t in cache])
    k, v = ops.kv8_read(cache, table[0].long())
    want = x.view(n, 8 + 2 * H_kv, D)[:, 8:8 + H_kv].transpose(0, 1).float()
    assert float((k.transpose(0, 1).reshape(H_kv, -1, D)[:, :n].float() - want).norm() / want.norm()) < 0.02
    ref, size, _ = _ref(q.transpose(0, 1), small, _i32([[0, 1, 2]]), [n], offset=[0], start=[0], length=[n])
    o = ops.kv8_paged_attention(q, cache, table, _i32([n]), _i32([0]), _i32([0]), _i32([n]))
    _check_attention(o.transpose(0, 1), ref, size, torch.bfloat16)
    last = ops.kv8_decode_attention(q[:, -1][None].contiguous(), cache, table, _i32([n]))
    _check_attention(last[0], ref[-1], size[-1], torch.bfloat16)


def test_streams_and_graphs():
    """A captured step (append, decode and prompt attention) replays on new inputs, and a side
    stream gives the same bits."""
    context = [600, 33, 1]
    q, cache, table = _decode(context, 8, 2, 128, 16, torch.bfloat16, seed=20)
    gen = torch.Generator().manual_seed(21)
    qkv = torch.randn(3, 12 * 128, generator=gen).to(torch.bfloat16).cuda()
    off, start, one, ctx = _i32([c - 1 for c in context]), _i32([0, 1, 2]), _i32([1, 1, 1]), _i32(context)

    def step():
        qh = ops.kv8_rope_append(qkv, 8, cache, table, off, start, one)
        return (ops.kv8_decode_attention(qh.transpose(0, 1), cache, table, ctx),
                ops.kv8_paged_attention(qh, cache, table, ctx, off, start, one))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.synchronize()
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    ref = [a.clone() for a in first]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(ref, held):
            assert torch.equal(a, b)
    qkv.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    eager = step()
    for a, b in zip(eager, held):
        assert torch.equal(a, b)


@pytest.mark.parametrize("q_len,offset", [([300, 5], [0, 900]), ([2000], [1000])])
def test_paged_attention_timeout_reports_and_next_call_is_clean(q_len, offset):
    """A wait limit of one cycle makes the kernel's waits give up: the status says so, and with the
    limit back the same call on the same stream is right (its tensor memory was freed, its
    workspace zeroed anew)."""
    q, cache, table, context, off, start, n = _prompt(q_len, offset, 8, 2, 128, 16, torch.bfloat16, seed=31)
    args = (q, cache, table, *[_i32(a) for a in (context, off, start, n)])
    want = ops.kv8_paged_attention(*args)
    assert ops.device_status() == _lib.LSE_OK
    ops.set_wait_limit(1)
    try:
        ops.kv8_paged_attention(*args)  # the launch itself succeeds
        assert ops.device_status() == _lib.LSE_ERR_DEVICE_TIMEOUT
    finally:
        ops.set_wait_limit(0)
    got = ops.kv8_paged_attention(*args)
    assert ops.device_status() == _lib.LSE_OK
    rows = np.concatenate([np.arange(s, s + k) for s, k in zip(start, n)])
    assert torch.equal(got[:, rows], want[:, rows])
