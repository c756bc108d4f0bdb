"""The 8-bit K/V cache operators and the token log-probabilities as measured workloads.

Four kinds of case:

* ``append``   -- rotate q and k of a fused QKV output and quantise k and v into the pages of an
  8-bit paged cache (one fp32 scale per page and KV head), returning rotated q, the scales, and
  the values that the touched pages now hold;
* ``decode``   -- attention of one query token per sequence over that cache;
* ``prompt``   -- causal attention of packed prompts or prompt chunks over that cache;
* ``logprobs`` -- log-probability of given tokens, entropy and the top alternatives of logits.

``run`` computes a case in its plain form (elementary torch operations in fp32) or, with ``own``
set, through ``llm_serving_engine_b200.ops``.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one chat request in decode: the call where only latency counts
        dict(name="append-1", kind="append", E=1, q_max=1, past_max=1024, ragged=False, H=32, H_kv=8, D=128, bs=16,
             R=128, interleaved=False, dtype="bf16", lens=1),
        # a decode batch of 64 sequences at different lengths, pages of 32, half of each head rotated in
        # interleaved pairs
        dict(name="append-64", kind="append", E=64, q_max=1, past_max=4096, ragged=True, H=32, H_kv=8, D=64, bs=32,
             R=32, interleaved=True, dtype="fp16", lens=2),
        # five prompt chunks packed into one batch, their first pages partly filled by earlier chunks
        dict(name="append-prompts", kind="append", E=5, q_max=2048, past_max=1000, ragged=True, H=64, H_kv=8, D=128,
             bs=16, R=128, interleaved=False, dtype="bf16", lens=3),
        # one chat request in decode
        dict(name="decode-1", kind="decode", E=1, ctx_max=1025, ragged=False, H=32, H_kv=8, D=128, bs=16, dtype="bf16",
             lens=4),
        # a decode batch of 64 sequences at different lengths
        dict(name="decode-64", kind="decode", E=64, ctx_max=4096, ragged=True, H=32, H_kv=8, D=128, bs=16, dtype="fp16",
             lens=5),
        # few long documents, eight query heads per KV head
        dict(name="decode-long", kind="decode", E=8, ctx_max=65536, ragged=True, H=64, H_kv=8, D=128, bs=16,
             dtype="bf16", lens=6),
        # a first prompt of ordinary length
        dict(name="prompt-512", kind="prompt", E=1, q_max=512, past_max=0, ragged=False, singles=0, H=32, H_kv=8, D=128,
             bs=16, dtype="bf16", lens=7),
        # one long prompt in a single chunk
        dict(name="prompt-8192", kind="prompt", E=1, q_max=8192, past_max=0, ragged=False, singles=0, H=32, H_kv=8,
             D=128, bs=16, dtype="bf16", lens=8),
        # a mixed batch: decode entries beside ragged chunks of longer documents
        dict(name="prompt-mixed", kind="prompt", E=12, q_max=700, past_max=5000, ragged=True, singles=8, H=32, H_kv=4,
             D=64, bs=64, dtype="fp16", lens=9),
        # the answer of one request, five alternatives
        dict(name="logprobs-1", kind="logprobs", M=1, V=128256, k=5, dtype="bf16", masked=False),
        # the answers of a decode batch under a grammar mask, twenty alternatives
        dict(name="logprobs-64", kind="logprobs", M=64, V=128256, k=20, dtype="fp16", masked=True),
        # scoring the tokens of prompts
        dict(name="logprobs-2048", kind="logprobs", M=2048, V=128256, k=1, dtype="bf16", masked=False),
    ]


def _log_int(rng, lo, hi):
    """An integer whose logarithm is spread evenly over [lo, hi]; as often odd as even."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "prompt", "logprobs"))
    if kind == "logprobs":
        M = _log_int(rng, 1, 2048)
        V = min(_log_int(rng, 1000, 200000), 2048 * 128256 // M)
        return dict(kind=kind, M=M, V=V, k=rng.randint(0, 20), dtype=rng.choice(("bf16", "fp16", "fp32") if M * V < 10 ** 8
                                                                               else ("bf16", "fp16")),
                    masked=rng.random() < 0.3)
    H_kv = rng.choice((1, 2, 4, 8))
    G = rng.choice((1, 2, 4, 8))
    D = rng.choice((64, 128))
    base = dict(kind=kind, H=H_kv * G, H_kv=H_kv, D=D, bs=rng.choice((8, 16, 32, 64, 128)),
                dtype=rng.choice(("bf16", "fp16")), ragged=rng.random() < 0.7, lens=rng.randrange(1 << 30))
    if kind == "decode":
        E = _log_int(rng, 1, 128)
        return dict(base, E=E, ctx_max=_log_int(rng, 16, min(65536, 8 * 65536 // E)))
    E = _log_int(rng, 1, 16)
    q_max = rng.choice((1, _log_int(rng, 2, 4096 // E)))
    past = rng.choice((0, _log_int(rng, 1, 8192 if kind == "append" or E * q_max <= 512 else 2048)))
    if kind == "append":
        return dict(base, E=E, q_max=q_max, past_max=past, R=rng.choice((D, D // 2, D // 4)),
                    interleaved=rng.random() < 0.5)
    return dict(base, E=E, q_max=q_max, past_max=past, singles=rng.randint(0, E - 1))


def _lens(case):
    """The lengths of a case's entries, the same for every seed: (tokens before the call, new tokens) each."""
    r = random.Random(case["lens"])
    out = []
    for e in range(case["E"]):
        if case["kind"] == "decode":
            n = r.randint(max(1, case["ctx_max"] // 8), case["ctx_max"]) if case["ragged"] and e else case["ctx_max"]
            out.append((n - 1, 1))
            continue
        past = r.randint(0, case["past_max"]) if case["ragged"] else case["past_max"]
        q = r.randint((case["q_max"] + 3) // 4, case["q_max"]) if case["ragged"] and e else case["q_max"]
        out.append((past, 1 if e >= case["E"] - case.get("singles", 0) else q))
    return out


def work(case):
    """Bytes that have to be read and written once, and the floating-point operations, of one pass."""
    if case["kind"] == "logprobs":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["M"] * (case["V"] * size + 8 + 8 + case["k"] * 12), "flops": 5.0 * case["M"] * case["V"]}
    lens, H, H_kv, D, bs = _lens(case), case["H"], case["H_kv"], case["D"], case["bs"]
    M = sum(n for _, n in lens)
    if case["kind"] == "append":
        pages = sum((p + n - 1) // bs - p // bs + 1 for p, n in lens)
        rows = M * (H + 2 * H_kv) * D * 2 + M * case["R"] * 8  # qkv, cos and sin
        # rotated q, new codes and scales, and the values of the touched pages (their codes read, values written)
        return {"bytes": rows + M * H * D * 2 + 2 * M * H_kv * D + 2 * pages * H_kv * 4 + 2 * pages * H_kv * bs * D * 3,
                "flops": 3.0 * M * (H + H_kv) * case["R"] + 4.0 * M * H_kv * D}
    kv = sum((p + n) * H_kv * 2 * D + 2 * 4 * H_kv * -(-(p + n) // bs) for p, n in lens)
    pairs = sum(n * p + n * (n + 1) // 2 for p, n in lens)  # visible (query, key) pairs of one head
    return {"bytes": kv + 2 * M * H * D * 2, "flops": 4.0 * D * H * pairs}


# ------------------------------------------------------------------------------------ inputs
def _cache(case, lens, new, g):
    """A paged 8-bit cache holding each entry's tokens (``new``: those of the call too) in shuffled pages.
    Keys have a few channels larger than the rest, as rotated keys do."""
    E, H_kv, D, bs = case["E"], case["H_kv"], case["D"], case["bs"]
    pages = [-(-(p + n) // bs) for p, n in lens]
    nb = sum(pages) + 1
    cols = max(pages)
    ids = torch.randperm(nb, generator=g, device="cuda")[: nb - 1].to(torch.int32)
    table = torch.zeros(E, cols, dtype=torch.int32, device="cuda")
    cut = torch.tensor(pages, device="cuda")
    at = torch.arange(cols, device="cuda")[None] < cut[:, None]
    table[at] = ids
    gain = 0.5 + 2.5 * torch.rand(H_kv, 1, D, generator=g, device="cuda") ** 8
    out = []
    for which in range(2):
        codes = torch.empty(nb, H_kv, bs, D, dtype=torch.int8, device="cuda")
        scale = torch.empty(nb, H_kv, dtype=torch.float32, device="cuda")
        step = max(1, (1 << 26) // (H_kv * bs * D))
        for b in range(0, nb, step):
            x = torch.randn(min(step, nb - b), H_kv, bs, D, generator=g, device="cuda")
            if which == 0:
                x = x * gain
            s = x.abs().amax((2, 3)) / 127.0
            codes[b:b + step] = torch.round(x / s[:, :, None, None]).clamp(-127, 127).to(torch.int8)
            scale[b:b + step] = s
        out += [codes, scale]
    return dict(k=out[0], k_scale=out[1], v=out[2], v_scale=out[3], table=table)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "logprobs":
        M, V = case["M"], case["V"]
        x = torch.empty(M, V, dtype=dt, device="cuda")
        step = max(1, (1 << 26) // V)
        for m in range(0, M, step):
            y = torch.randn(min(step, M - m), V, generator=g, device="cuda") * 2.5 - 4.0
            y += 9.0 * torch.rand(y.shape, generator=g, device="cuda") ** 64  # few likely tokens
            if case["masked"]:
                y[torch.rand(y.shape, generator=g, device="cuda") < 0.7] = -math.inf
            x[m:m + step] = y.to(dt)
        tokens = torch.randint(0, V, (M,), generator=g, device="cuda")
        tokens[::2] = x[::2].argmax(-1)  # every other token is the likeliest one
        return dict(case=case, x=x, tokens=tokens)
    lens = _lens(case)
    H, H_kv, D = case["H"], case["H_kv"], case["D"]
    M = sum(n for _, n in lens)
    i32 = dict(dtype=torch.int32, device="cuda")
    st = dict(case=case, **_cache(case, lens, case["kind"] != "append", g))
    starts, pos, row = [], [], 0
    for p, n in lens:
        starts.append(row)
        pos.append(torch.arange(p, p + n, device="cuda"))
        row += n
    st["pos"] = torch.cat(pos)
    st["entry"] = torch.repeat_interleave(torch.arange(case["E"], device="cuda"),
                                          torch.tensor([n for _, n in lens], device="cuda"))
    st["q_start"] = torch.tensor(starts, **i32)
    st["q_len"] = torch.tensor([n for _, n in lens], **i32)
    st["offset"] = torch.tensor([p for p, _ in lens], **i32)
    st["context"] = torch.tensor([p + n for p, n in lens], **i32)
    if case["kind"] == "append":
        st["qkv"] = torch.randn(M, (H + 2 * H_kv) * D, generator=g, device="cuda").to(dt)
        R = case["R"]
        inv = 500000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float32) / R)
        ang = st["pos"].float()[:, None] * inv
        ang = ang.repeat_interleave(2, 1) if case["interleaved"] else torch.cat([ang, ang], 1)
        st["cos"], st["sin"] = ang.cos(), ang.sin()
        bs = case["bs"]
        st["touched"] = torch.unique(st["table"].long()[st["entry"], st["pos"] // bs])
    elif case["kind"] == "decode":
        st["q"] = torch.randn(case["E"], H, D, generator=g, device="cuda").to(dt)
    else:
        st["q"] = torch.randn(H, M, D, generator=g, device="cuda").to(dt)
    return st


# ------------------------------------------------------------------------------------ plain forms
def _turned(x, interleaved):
    """The partner of each element of the rotated part, with its sign."""
    if interleaved:
        return torch.stack([-x[..., 1::2], x[..., 0::2]], -1).flatten(-2)
    h = x.shape[-1] // 2
    return torch.cat([-x[..., h:], x[..., :h]], -1)


def _plain_append(st):
    c = st["case"]
    H, H_kv, D, bs, R = c["H"], c["H_kv"], c["D"], c["bs"], c["R"]
    M = st["qkv"].shape[0]
    x = st["qkv"].float().view(M, H + 2 * H_kv, D)
    qk, v = x[:, : H + H_kv], x[:, H + H_kv:]
    cos, sin = st["cos"][:, None], st["sin"][:, None]
    rot = qk[..., :R]
    qk = torch.cat([rot * cos + _turned(rot, c["interleaved"]) * sin, qk[..., R:]], -1)
    q = qk[:, :H].transpose(0, 1).to(st["qkv"].dtype).contiguous()
    page = st["table"].long()[st["entry"], st["pos"] // bs]
    slot = st["pos"] % bs
    t = st["touched"]
    nb = st["k"].shape[0]
    # tokens that a touched page held before: all slots below the call's first one in it
    kept = torch.full((nb,), bs, device=x.device, dtype=torch.long).index_reduce_(0, page, slot, "amin")[t]
    old = torch.arange(bs, device=x.device)[None] < kept[:, None]
    out = [q]
    for new, codes, scale in ((qk[:, H:], st["k"], st["k_scale"]), (v, st["v"], st["v_scale"])):
        top = torch.zeros(nb, H_kv, device=x.device).index_reduce_(0, page, new.abs().amax(-1), "amax")[t] / 127.0
        before = torch.where(kept[:, None] > 0, scale[t], torch.zeros_like(top))
        s = torch.maximum(before, top)
        grown = torch.where(s > before, before / s, torch.ones_like(s))
        held = torch.where(old[:, None, :, None], torch.round(codes[t].float() * grown[..., None, None]), codes[t].float())
        codes[t] = held.to(torch.int8)
        scale[t] = s
        sn = scale[page][..., None]
        codes[page, :, slot] = torch.where(sn > 0, torch.round(new / sn).clamp(-127, 127), torch.zeros_like(new)).to(torch.int8)
        out += [scale, (codes[t].float() * s[..., None, None]).to(st["qkv"].dtype)]
    return tuple(out)


def _values(codes, scale, table):
    """fp32 [E, H_kv, positions, D] of the pages in a block table."""
    x = codes[table.long()].float() * scale[table.long()][..., None, None]
    E, n, H_kv, bs, D = x.shape
    return x.transpose(1, 2).reshape(E, H_kv, n * bs, D)


def _plain_attention(q, st, limit):
    """softmax(q k^T / sqrt(D)) v in fp32; q [E, H, T, D], limit [E, T]: positions below it are seen."""
    c = st["case"]
    E, H, T, D = q.shape
    k = _values(st["k"], st["k_scale"], st["table"])
    s = torch.matmul(q.reshape(E, c["H_kv"], -1, D), k.transpose(-1, -2)).view(E, H, T, -1)
    s.mul_(D ** -0.5)
    s.masked_fill_((torch.arange(s.shape[-1], device=q.device) >= limit[..., None])[:, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    v = _values(st["v"], st["v_scale"], st["table"])
    return torch.matmul(s.view(E, c["H_kv"], -1, v.shape[2]), v).view(E, H, T, D) / total


def _plain_decode(st):
    q = st["q"].float()[:, :, None]
    return _plain_attention(q, st, st["context"][:, None])[:, :, 0].to(st["q"].dtype)


def _plain_prompt(st):
    c = st["case"]
    q = st["q"].float().transpose(0, 1)  # [tokens, H, D]
    within = st["pos"] - st["offset"].long()[st["entry"]]
    most = max(n for _, n in _lens(c))
    grid = torch.zeros(c["E"], most, c["H"], c["D"], device=q.device)
    grid[st["entry"], within] = q
    limit = st["offset"][:, None] + torch.arange(1, most + 1, device=q.device)[None]
    o = _plain_attention(grid.transpose(1, 2), st, torch.minimum(limit, st["context"][:, None]))
    return o.transpose(1, 2)[st["entry"], within].transpose(0, 1).to(st["q"].dtype).contiguous()


def _plain_logprobs(st):
    x, k = st["x"].float(), st["case"]["k"]
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1)
    entropy = total.log() - torch.where(e > 0, d * e, torch.zeros_like(d)).sum(-1) / total
    log_z = (total.log() + x.amax(-1))
    logprob = x.gather(1, st["tokens"][:, None])[:, 0] - log_z
    # an integer that orders values first and, among equal ones, lower indices first
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = order * (1 << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device=x.device))
    ids = (1 << 20) - 1 - (torch.topk(key, k, -1).values & ((1 << 20) - 1))
    return logprob, entropy, x.gather(1, ids) - log_z[:, None], ids


def run(state):
    c = state["case"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt,
                "logprobs": _plain_logprobs}[c["kind"]](state)
    from llm_serving_engine_b200 import ops

    st = state
    if c["kind"] == "logprobs":
        return tuple(ops.token_logprobs(st["x"], st["tokens"], c["k"]))
    cache = ops.Kv8Cache(st["k"], st["v"], st["k_scale"], st["v_scale"])
    if c["kind"] == "append":
        q = ops.kv8_rope_append(st["qkv"], c["H"], cache, st["table"], st["offset"], st["q_start"], st["q_len"],
                                st["cos"], st["sin"], c["interleaved"])
        k, v = ops.kv8_read(cache, st["touched"], st["qkv"].dtype)
        return q, st["k_scale"], k, st["v_scale"], v
    if c["kind"] == "decode":
        return ops.kv8_decode_attention(st["q"], cache, st["table"], st["context"])
    return ops.kv8_paged_attention(st["q"], cache, st["table"], st["context"], st["offset"], st["q_start"], st["q_len"])


# ------------------------------------------------------------------------------------ exact values
def _exact_append(st):
    c = st["case"]
    H, H_kv, D, bs, R = c["H"], c["H_kv"], c["D"], c["bs"], c["R"]
    x = st["qkv"].double().view(-1, H + 2 * H_kv, D)
    cos, sin = st["cos"].double()[:, None], st["sin"].double()[:, None]
    rotated = x.clone()
    heads = slice(0, H + H_kv)
    first = torch.arange(0, R, 2, device=x.device) if c["interleaved"] else torch.arange(R // 2, device=x.device)
    second = first + (1 if c["interleaved"] else R // 2)
    a, b = x[:, heads][..., first], x[:, heads][..., second]
    rotated[:, :H + H_kv, first] = a * cos[..., first] - b * sin[..., first]
    rotated[:, :H + H_kv, second] = b * cos[..., second] + a * sin[..., second]
    out = [rotated[:, :H].transpose(0, 1)]
    lens = _lens(c)
    for new, codes, scale in ((rotated[:, H:H + H_kv], st["k"], st["k_scale"]), (x[:, H + H_kv:], st["v"], st["v_scale"])):
        scale, held = scale.double(), codes.double()
        row = 0
        for e, (past, n) in enumerate(lens):
            table = st["table"][e].tolist()
            for p in range(past // bs, (past + n - 1) // bs + 1):
                lo, hi = max(past, p * bs), min(past + n, (p + 1) * bs)
                b, rows = table[p], new[row + lo - past: row + hi - past].transpose(0, 1)  # [H_kv, tokens, D]
                before = scale[b].clone() if lo > p * bs else torch.zeros_like(scale[b])
                s = torch.maximum(before, rows.abs().amax((1, 2)) / 127)
                f = torch.where(s > before, before / s, torch.ones_like(s))
                held[b, :, : lo - p * bs] = torch.round(held[b, :, : lo - p * bs] * f[:, None, None])
                held[b, :, lo - p * bs: hi - p * bs] = torch.round(rows / s[:, None, None]).clamp(-127, 127)
                scale[b] = s
            row += n
        out += [scale, held[st["touched"]] * scale[st["touched"]][..., None, None]]
    return tuple(out)


def _exact_rows(q, k, v, limit):
    """One KV head in fp64, query rows a few at a time: q [rows, D], k and v [positions, D], limit [rows]."""
    out = []
    step = max(1, (1 << 26) // k.shape[0])
    for r in range(0, q.shape[0], step):
        s = q[r:r + step] @ k.T / math.sqrt(q.shape[1])
        s = s.masked_fill(torch.arange(k.shape[0], device=q.device)[None] >= limit[r:r + step, None], -math.inf)
        out.append(torch.softmax(s, -1) @ v)
    return torch.cat(out)


def _exact_attention(st):
    c = st["case"]
    H, H_kv, D, bs = c["H"], c["H_kv"], c["D"], c["bs"]
    G = H // H_kv
    decode = c["kind"] == "decode"
    q = st["q"].double() if not decode else st["q"].double().transpose(0, 1)  # [H, tokens, D]
    o = torch.empty_like(q)
    row = 0
    for e, (past, n) in enumerate(_lens(c)):
        ids = st["table"][e, : -(-(past + n) // bs)].long()
        limit = past + 1 + torch.arange(n, device=q.device)
        for h in range(H_kv):
            k = (st["k"][ids, h].double() * st["k_scale"][ids, h].double()[:, None, None]).reshape(-1, D)[: past + n]
            v = (st["v"][ids, h].double() * st["v_scale"][ids, h].double()[:, None, None]).reshape(-1, D)[: past + n]
            rows = q[h * G:(h + 1) * G, row:row + n].reshape(-1, D)
            o[h * G:(h + 1) * G, row:row + n] = _exact_rows(rows, k, v, limit.repeat(G)).view(G, n, D)
        row += n
    return o.transpose(0, 1) if decode else o


def _exact_logprobs(st):
    lp, entropy, tops = [], [], []
    step = max(1, (1 << 25) // st["x"].shape[1])
    for m in range(0, st["x"].shape[0], step):
        p = torch.log_softmax(st["x"][m:m + step].double(), -1)
        lp.append(p.gather(1, st["tokens"][m:m + step, None])[:, 0])
        entropy.append(torch.special.entr(p.exp()).sum(-1))
        tops.append(torch.sort(p, dim=-1, descending=True, stable=True).values[:, : st["case"]["k"]])
    return torch.cat(lp), torch.cat(entropy), torch.cat(tops), None


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_attention, "prompt": _exact_attention,
            "logprobs": _exact_logprobs}[case["kind"]](st)
