"""The 8-bit cache and log-probability entries refuse bad arguments on the host, before any
device call, and the torch-facing calls refuse CPU tensors (no GPU here)."""

from __future__ import annotations

import pytest
import torch

from llm_serving_engine_b200 import _lib, ops

P = 256  # an aligned non-null address that these paths never read


def _append(lib, dtype=_lib.DT_BF16, M=4, ld=1536, H=8, H_kv=2, D=128, cos=P, ld_cs=128, cs=_lib.DT_F32, R=128, q=P, k=P,
            ks=P, nb=10, bs=16, bt=P, bts=4, cols=4, off=P, E=2, qkv=P):
    return lib.lse_kv8_rope_append(qkv, dtype, M, ld, H, H_kv, D, cos, P, ld_cs, cs, R, 0, q, k, P, ks, P, nb, bs, bt, bts,
                                   cols, off, P, P, E, None)


def test_append_refusals():
    lib = _lib.load()
    bad, off, no = _lib.LSE_ERR_INVALID_ARG, _lib.LSE_ERR_ALIGNMENT, _lib.LSE_ERR_UNSUPPORTED
    assert _append(lib, M=0) == _lib.LSE_OK
    for kw in (dict(M=-1), dict(E=-1), dict(R=3), dict(R=130), dict(R=-2), dict(ld=1535), dict(cos=None), dict(ld_cs=64),
               dict(cs=9), dict(q=None), dict(k=None), dict(ks=None), dict(nb=0), dict(bs=0), dict(H=9), dict(bt=None),
               dict(off=None), dict(bts=3), dict(qkv=None), dict(H_kv=0), dict(cols=-1)):
        assert _append(lib, **kw) == bad, kw
    for kw in (dict(dtype=_lib.DT_F32), dict(D=96, ld=1152, R=96), dict(H=6, ld=1280), dict(H=32, ld=4608), dict(bs=70000),
               dict(nb=1 << 30), dict(E=1 << 21), dict(M=1 << 31)):
        assert _append(lib, **kw) == no, kw
    for kw in (dict(ld=1540), dict(qkv=P + 2), dict(q=P + 8), dict(k=P + 8), dict(ks=P + 2), dict(cos=P + 2), dict(bt=P + 2)):
        assert _append(lib, **kw) == off, kw


def _decode(lib, q=P, dtype=_lib.DT_BF16, E=2, H=8, D=128, sq=1024, k=P, nb=10, bs=16, H_kv=2, bt=P, bts=4, cols=4, ctx=P,
            o=P, so=1024):
    return lib.lse_kv8_decode_attention(q, dtype, E, H, D, sq, 128, k, P, P, P, nb, bs, H_kv, bt, bts, cols, ctx, 0.1, o, so,
                                        128, P, 0, None)


def _paged(lib, q=P, dtype=_lib.DT_BF16, T=5, H=8, D=128, sq=1024, k=P, nb=10, bs=16, H_kv=2, bt=P, bts=4, cols=4, ctx=P,
           off=P, E=2, o=P, so=1024):
    return lib.lse_kv8_paged_attention(q, dtype, T, H, D, sq, 128, k, P, P, P, nb, bs, H_kv, bt, bts, cols, ctx, off, P, P, E,
                                       0.1, o, so, 128, P, 0, None)


@pytest.mark.parametrize("call", [_decode, _paged])
def test_attention_refusals(call):
    lib = _lib.load()
    assert call(lib, E=0) == _lib.LSE_OK
    for kw in (dict(E=-1), dict(q=None), dict(o=None), dict(ctx=None), dict(k=None), dict(nb=0), dict(bs=0), dict(H=9),
               dict(bt=None), dict(bts=3), dict(cols=-1)):
        assert call(lib, **kw) == _lib.LSE_ERR_INVALID_ARG, kw
    for kw in (dict(dtype=_lib.DT_F32), dict(D=96), dict(H=6), dict(H=32), dict(nb=1 << 30), dict(cols=1 << 30, bts=1 << 30)):
        assert call(lib, **kw) == _lib.LSE_ERR_UNSUPPORTED, kw
    for kw in (dict(q=P + 8), dict(o=P + 2), dict(k=P + 8), dict(sq=1028), dict(so=1023), dict(ctx=P + 2), dict(bt=P + 1)):
        assert call(lib, **kw) == _lib.LSE_ERR_ALIGNMENT, kw


def test_read_and_logprobs_refusals():
    lib = _lib.load()
    bad, off, no = _lib.LSE_ERR_INVALID_ARG, _lib.LSE_ERR_ALIGNMENT, _lib.LSE_ERR_UNSUPPORTED
    read = lambda pool=P, scale=P, nb=4, bs=16, hk=2, D=64, ids=P, n=3, out=P, dt=0: lib.lse_kv8_read(  # noqa: E731
        pool, P, scale, P, nb, bs, hk, D, ids, n, out, P, dt, None)
    assert read(n=0) == _lib.LSE_OK
    for kw in (dict(pool=None), dict(scale=None), dict(ids=None), dict(out=None), dict(nb=0), dict(bs=0), dict(n=-1)):
        assert read(**kw) == bad, kw
    assert read(dt=_lib.DT_F32) == no and read(D=24) == no
    assert read(pool=P + 8) == off and read(out=P + 2) == off and read(ids=P + 4) == off
    lp = lambda x=P, dt=0, M=3, V=100, ld=100, t=P, k=5, a=P, b=P, c=P, d=P: lib.lse_token_logprobs(  # noqa: E731
        x, dt, M, V, ld, t, k, a, b, c, d, None)
    assert lp(M=0) == _lib.LSE_OK
    for kw in (dict(M=-1), dict(V=0), dict(ld=99), dict(k=-1), dict(k=101), dict(x=None), dict(a=None), dict(b=None),
               dict(c=None), dict(d=None)):
        assert lp(**kw) == bad, kw
    assert lp(dt=7) == no and lp(V=1000, ld=1000, k=_lib.LOGPROBS_MAX_TOP + 1) == no
    for kw in (dict(x=P + 1), dict(x=P + 2, dt=_lib.DT_F32), dict(t=P + 4), dict(b=P + 2), dict(d=P + 4)):
        assert lp(**kw) == off, kw


def test_torch_calls_refuse_cpu_tensors():
    cache = ops.kv8_cache(2, 16, 1, 64, device="cpu")
    one = torch.ones(1, dtype=torch.int32)
    table = torch.zeros(1, 1, dtype=torch.int32)
    x = torch.zeros(1, 192, dtype=torch.bfloat16)
    for call in (lambda: ops.kv8_rope_append(x, 1, cache, table, one, one, one),
                 lambda: ops.kv8_read(cache, torch.zeros(1, dtype=torch.long)),
                 lambda: ops.kv8_decode_attention(x.view(1, 3, 64), cache, table, one),
                 lambda: ops.kv8_paged_attention(x.view(3, 1, 64), cache, table, one, one, one, one),
                 lambda: ops.token_logprobs(x)):
        with pytest.raises(RuntimeError, match="CUDA only"):
            call()


def test_header_limit_matches_binding():
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "lse_int8.h")).read()
    assert int(re.search(r"#define LSE_LOGPROBS_MAX_TOP (\d+)", text).group(1)) == _lib.LOGPROBS_MAX_TOP
