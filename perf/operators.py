"""Paged KV cache operators as measurable cases: appending rotated keys and values, and attention over the pages.

Two kinds of case:

* ``append``  ``kernels.paged_rope_append``: the q and k heads of a ragged batch's fused-QKV rows rotated, keys and
              values written to the sequences' pages, in fp16, bf16 or 4 bits.
* ``attend``  ``kernels.paged_attend``: softmax attention of a ragged batch's queries (one token a sequence, a few
              drafted ones, or a prompt's) over the pages, with the scores optionally capped by a tanh or biased by
              distance, and a sliding window or a prefix beside the causal mask.

A sequence of ``kv_lens[b]`` keys has its last ``q_start[b + 1] - q_start[b]`` tokens in the call; position p of it is
row p % page of page ``block_table[b, p // page]``.  Sizes are the head layouts of the 3B-shaped decoder (24 query / 8
KV heads of 128) and generic ones; ``own`` picks the framework's calls instead of the plain form.
"""
import math
import random

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "4bit": torch.float16}


def _case(op, kind="fp16", batch=1, heads=24, kv_heads=8, head_dim=128, page=16, q=(1, 1), ctx=(0, 0), cap=0.0, window=0,
          slopes=False, prefix=0.0, shape=0, name=None):
    """``q``: tokens of a sequence in the call, ``ctx``: keys before them, both from .. to; the first sequence has the
    most of both, the others are spread by ``shape``.  ``prefix``: share of a sequence that every token sees."""
    c = dict(op=op, kind=kind, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, q_lo=q[0],
             q_hi=q[1], ctx_lo=ctx[0], ctx_hi=ctx[1], cap=cap, window=window, slopes=slopes, prefix=prefix, shape=shape)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # the smallest call: one token of batch-1 generation enters the cache
        _case("append", name="append_token", ctx=(640, 640)),
        # prompts of several users enter a bf16 cache together, ragged
        _case("append", name="append_prompts_bf16", kind="bf16", batch=5, heads=32, page=64, q=(3, 1801), ctx=(0, 700),
              shape=1),
        # prompts stored in 4 bits, quantised on the way (the values that the pages stand for are read back)
        _case("append", name="append_prompts_4bit", kind="4bit", batch=3, page=32, q=(600, 1500), shape=2),
        # one token of batch-1 generation over a short cache: latency
        _case("attend", name="decode_one_short", ctx=(96, 96)),
        # a served batch of 64 users at all stages of their answers, one token each
        _case("attend", name="decode_b64", batch=64, page=32, ctx=(0, 8191), shape=3),
        # one user with a very long document: the key axis has to be split
        _case("attend", name="decode_long_bf16", kind="bf16", page=64, ctx=(131070, 131070)),
        # a served batch whose long caches are held in 4 bits
        _case("attend", name="decode_b48_4bit", kind="4bit", batch=48, heads=32, page=64, ctx=(100, 16000), shape=4),
        # five drafted tokens a sequence verified at once: capped scores, sliding window, small heads
        _case("attend", name="verify_cap_window", kind="bf16", batch=16, heads=32, head_dim=64, q=(5, 5), ctx=(300, 6000),
              cap=30.0, window=1024, shape=5),
        # a prompt of ragged length, as the decoder's prefill runs
        _case("attend", name="prompt_777", q=(777, 777)),
        # a long prompt at once
        _case("attend", name="prompt_8192", page=64, q=(8192, 8192)),
        # chunks of several prompts on their contexts, capped scores, sliding window
        _case("attend", name="chunks_cap_bf16", kind="bf16", batch=6, heads=32, page=32, q=(120, 1000), ctx=(0, 5500),
              cap=50.0, window=4096, shape=6),
        # prompts read back from 4 bits: distance bias, a prefix that every token sees, no shared heads
        _case("attend", name="prompts_4bit_bias", kind="4bit", batch=3, heads=16, kv_heads=16, head_dim=64, page=16,
              q=(200, 2100), slopes=True, prefix=0.3, shape=7),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["fp16", "fp16", "bf16", "4bit"])
    heads, kv = rng.choice([(24, 8), (24, 8), (32, 8), (32, 4), (16, 16), (14, 2), (8, 1)])
    d, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128])
    c = dict(kind=kind, heads=heads, kv_heads=kv, head_dim=d, page=page, shape=rng.randrange(1 << 20))
    stage = rng.choices(["append", "decode", "verify", "prompt"], [3, 4, 1, 3])[0]
    if stage == "append":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 6000 // batch))
        return _case("append", batch=batch, q=(max(1, hi // 4), hi), ctx=(0, _log(rng, 1, max(1, 4000 // batch))), **c)
    if rng.random() < 0.3:
        c["cap"] = rng.choice([20.0, 30.0, 50.0])
    if rng.random() < 0.3:
        c["window"] = _log(rng, 16, 4096)
    if rng.random() < 0.25:
        c["slopes"] = True
    if stage == "decode":
        batch = _log(rng, 1, 128)
        return _case("attend", batch=batch, ctx=(0, _log(rng, 1, 260000 // batch)), **c)
    if stage == "verify":
        batch = _log(rng, 1, 64)
        q = rng.randint(2, 16)
        return _case("attend", batch=batch, q=(max(1, q // 2), q), ctx=(0, _log(rng, 16, 130000 // batch)), **c)
    batch = rng.randint(1, 6)
    if rng.random() < 0.3:
        c["prefix"] = rng.choice([0.1, 0.5, 0.9])
    hi = _log(rng, 17, 4096 // batch)
    return _case("attend", batch=batch, q=(max(1, hi // 3), hi), ctx=(0, _log(rng, 1, 8192 // batch)), **c)


def _lengths(case):
    """Tokens in the call and keys after it, per sequence."""
    r = random.Random(case["shape"])
    nq = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    nq[0], ctx[0] = case["q_hi"], case["ctx_hi"]
    return nq, [a + b for a, b in zip(nq, ctx)]


# -- inputs --------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1 + int(seed))
    nq, lens = _lengths(case)
    b, h, kv, d, page, kind = (case[k] for k in ("batch", "heads", "kv_heads", "head_dim", "page", "kind"))
    dt = _DT[kind]

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dt)

    # the sequences' pages lie scattered in the pool, two of which nobody uses; unused table entries hold -1
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((b, max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at: at + n]
        at += n
    starts = [0]
    for n in nq:
        starts.append(starts[-1] + n)
    s = dict(op=case["op"], kind=kind, heads=h, kv_heads=kv, head_dim=d, page=page, max_q=max(nq),
             cap=case["cap"], window=case["window"], table=table,
             kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    if kind == "4bit":  # codes, scales and zero points as the quantiser leaves them for values of deviation 1

        def pool():
            codes = torch.randint(0, 256, (pages, kv, page, d // 2), generator=gen, device="cuda", dtype=torch.uint8)
            scales = torch.rand(pages, kv, page, d // 32, generator=gen, device="cuda").mul_(0.15).add_(0.2).half()
            zeros = torch.randint(5, 11, scales.shape, generator=gen, device="cuda", dtype=torch.uint8)
            return codes, scales, zeros

        s["k"], s["v"] = pool(), pool()
    else:
        s["k"], s["v"] = rand(pages, kv, page, d), rand(pages, kv, page, d)
    if case["op"] == "append":
        s["qkv"] = rand(starts[-1], (h + 2 * kv) * d)
        inv = 1.0 / (500000.0 ** (torch.arange(0, d, 2, dtype=torch.float32, device="cuda") / d))
        ang = torch.arange(max(lens), dtype=torch.float32, device="cuda")[:, None] * inv
        s["cos"], s["sin"] = ang.cos(), ang.sin()
    else:
        s["q"] = rand(starts[-1], h, d)
        s["slopes"] = s["prefix"] = None
        if case["slopes"]:
            s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, dtype=torch.float32, device="cuda") / h)
        if case["prefix"]:
            s["prefix"] = (s["kv_lens"].double() * case["prefix"]).int()
    return s


# -- the plain form ------------------------------------------------------------------------------
def _token_rows(s, tokens):
    """The sequence and position of every token of the call."""
    t = torch.arange(tokens, device="cuda")
    starts = s["q_start"].long()
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    pos = s["kv_lens"].long()[seq] - (starts[seq + 1] - starts[seq]) + (t - starts[seq])
    return seq, t - starts[seq], pos


def _values(cache):
    """(q - z) * s of 4-bit rows, in 32 bits."""
    codes, scales, zeros = cache
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    c = c.unflatten(-1, (-1, 32))
    return ((c - zeros.float().unsqueeze(-1)) * scales.float().unsqueeze(-1)).flatten(-2)


def _quantised(x):
    """Codes, scale and zero point of each 32 fp16 values of the last dimension: minimum and maximum, the range, the
    scale and the zero point rounded to fp16 as the 4-bit cache holds them."""
    x = x.float().unflatten(-1, (-1, 32))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low).half().float() / 15.0).half().float()
    zero = torch.nan_to_num((-low / scale).half().float().round(), nan=0.0).clamp(0, 15)
    code = torch.nan_to_num(((x + zero * scale) / scale).round(), nan=0.0).clamp(0, 15)
    code = code.flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.squeeze(-1).half(), zero.squeeze(-1).to(torch.uint8)


def _plain_append(s):
    qkv, h, kv, d = s["qkv"], s["heads"], s["kv_heads"], s["head_dim"]
    seq, _, pos = _token_rows(s, qkv.shape[0])
    row = qkv.float().view(-1, h + 2 * kv, d)
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
    a, b = row[:, :h + kv, :d // 2], row[:, :h + kv, d // 2:]
    rot = torch.cat([a * c - b * sn, b * c + a * sn], -1).to(qkv.dtype)
    page = s["table"][seq, pos // s["page"]].long()
    at = pos % s["page"]
    for cache, x in ((s["k"], rot[:, h:]), (s["v"], row[:, h + kv:].to(qkv.dtype))):
        if s["kind"] == "4bit":
            for pool, new in zip(cache, _quantised(x)):
                pool[page, :, at] = new
        else:
            cache[page, :, at] = x
    q = rot[:, :h].contiguous()
    if s["kind"] == "4bit":
        return dict(q=q, k=_values(s["k"]).bfloat16(), v=_values(s["v"]).bfloat16())
    return dict(q=q, k=s["k"], v=s["v"])


def _gathered(s, cache):
    """A cache's rows by sequence [batch, kv_heads, keys, d], in 32 bits; 4-bit values rounded to fp16, as the operator
    defines them."""
    at = s["table"].long().clamp(min=0)
    x = _values(tuple(p[at] for p in cache)).half().float() if s["kind"] == "4bit" else cache[at].float()
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    q, h, kv, d, g = s["q"], s["heads"], s["kv_heads"], s["head_dim"], s["heads"] // s["kv_heads"]
    tokens, mq = q.shape[0], s["max_q"]
    k, v = _gathered(s, s["k"]), _gathered(s, s["v"])
    b, keys = k.shape[0], k.shape[2]
    starts, lens = s["q_start"].long(), s["kv_lens"].long()
    t = torch.arange(mq, device="cuda")
    qp = q[(starts[:-1, None] + t).clamp(max=tokens - 1)].float()
    qp = qp.view(b, mq, kv, g, d).permute(0, 2, 1, 3, 4).reshape(b, kv, mq * g, d)
    x = torch.matmul(qp, k.transpose(2, 3)) / math.sqrt(d)
    del k
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    i = (lens - (starts[1:] - starts[:-1]))[:, None] + t  # positions of the queries
    j = torch.arange(keys, device="cuda")
    far = i[:, :, None] - j
    see = far >= 0
    if s["prefix"] is not None:
        see = see | (j < s["prefix"].long()[:, None, None])
    see = see & (j < lens[:, None, None])
    if s["window"]:
        see = see & (far < s["window"])
    x = x.view(b, kv, mq, g, keys)
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, kv, 1, g, 1) * far.abs().float()[:, None, :, None]
    x = x.masked_fill(~see[:, None, :, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == float("-inf"), 0.0, top))
    total = x.sum(-1, keepdim=True)
    x = x / torch.where(total == 0.0, 1.0, total)
    o = torch.matmul(x.view(b, kv, mq * g, keys), v).view(b, kv, mq, g, d)
    seq, tok, _ = _token_rows(s, tokens)
    return o.permute(0, 2, 1, 3, 4).reshape(b, mq, h, d)[seq, tok].to(q.dtype)


# -- one pass ------------------------------------------------------------------------------------
def _own_append(s):
    from spectra_amd import kernels as K
    q = K.paged_rope_append(s["qkv"], s["kv_lens"], s["q_start"], s["table"], s["cos"], s["sin"], s["heads"], s["k"], s["v"])
    if s["kind"] == "4bit":
        return dict(q=q, k=K.kv4_dequantize(*s["k"]), v=K.kv4_dequantize(*s["v"]))
    return dict(q=q, k=s["k"], v=s["v"])


def _own_attend(s):
    from spectra_amd import kernels as K
    if "workspace" not in s:  # kept for all layers and steps, as a serving loop does
        s["workspace"] = K.paged_attend_workspace(s["head_dim"], s["q"].device)
    return K.paged_attend(s["q"], s["kv_lens"], s["q_start"], s["table"], s["k"], s["v"], cap=s["cap"], window=s["window"],
                          slopes=s["slopes"], prefix=s["prefix"], workspace=s["workspace"])


@torch.no_grad()
def run(state):
    if state["op"] == "append":
        return _own_append(state) if own else _plain_append(state)
    return _own_attend(state) if own else _plain_attend(state)


# -- what a pass cannot do without ---------------------------------------------------------------
def _row_bytes(case):
    """One head's key (or value) of one position."""
    d = case["head_dim"]
    return d / 2 + 3 * d / 32 if case["kind"] == "4bit" else 2 * d


def work(case):
    nq, lens = _lengths(case)
    h, kv, d, tokens = case["heads"], case["kv_heads"], case["head_dim"], sum(nq)
    if case["op"] == "append":
        b = tokens * ((2 * h + 2 * kv) * 2 * d + 2 * kv * _row_bytes(case) + 4 * d)
        if case["kind"] == "4bit":  # the pages' values read back
            rows = kv * case["page"] * (sum(-(-n // case["page"]) for n in lens) + 2)
            b += 2 * rows * (_row_bytes(case) + 2 * d)
        return {"bytes": b, "flops": tokens * (h + kv) * 3 * d}
    pairs = keys = 0
    for n, m in zip(nq, lens):
        pre = min(int(m * case["prefix"]), m)
        first = None
        for i in range(m - n, m):
            lo = max(0, i - case["window"] + 1) if case["window"] else 0
            hi = max(i + 1, pre)
            pairs += hi - lo
            first = lo if first is None else first
        keys += m - first
    return {"bytes": 2 * kv * keys * _row_bytes(case) + 2 * tokens * h * d * 2, "flops": 4 * h * d * pairs}


# -- the same in 64 bits -------------------------------------------------------------------------
def _wide(cache, kind, dt=torch.float64):
    """What the pages stand for, in 64 bits; 4-bit values rounded to ``dt`` first where it is smaller."""
    if kind != "4bit":
        return cache.double()
    codes, scales, zeros = cache
    lo, hi = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
    x = torch.cat([lo.unsqueeze(-1), hi.unsqueeze(-1)], -1).reshape(*codes.shape[:-1], -1)
    x = (x - zeros.double().repeat_interleave(32, -1)) * scales.double().repeat_interleave(32, -1)
    return x.to(dt).double()


def _exact_append(s, lens, nq):
    h, kv, d, page = s["heads"], s["kv_heads"], s["head_dim"], s["page"]
    table = s["table"].tolist()
    quantised = s["kind"] == "4bit"
    k, v = _wide(s["k"], s["kind"]), _wide(s["v"], s["kind"])
    qs, at = [], 0
    for i, (n, m) in enumerate(zip(nq, lens)):
        row = s["qkv"][at: at + n].double().view(n, h + 2 * kv, d)
        at += n
        c, sn = s["cos"][m - n: m].double()[:, None], s["sin"][m - n: m].double()[:, None]
        a, b = row[:, :h + kv].chunk(2, -1)
        rot = torch.cat([a * c - b * sn, b * c + a * sn], -1)
        qs.append(rot[:, :h])
        for pool, x in ((k, rot[:, h:]), (v, row[:, h + kv:])):
            if quantised:
                y = x.half().double().reshape(n, kv, d // 32, 32)
                low = y.min(-1, keepdim=True).values
                step = ((y.max(-1, keepdim=True).values - low).half().double() / 15).half().double()
                z = (-low / step).half().double().round().clamp(0, 15)
                x = ((((y + z * step) / step).round().clamp(0, 15) - z) * step).reshape(n, kv, d)
            first = m - n
            while first < m:  # the run of positions in one page
                end = min(m, (first // page + 1) * page)
                pool[table[i][first // page], :, first % page: first % page + end - first] = \
                    x[first - (m - n): end - (m - n)].transpose(0, 1)
                first = end
    return dict(q=torch.cat(qs), k=k, v=v)


def _exact_attend(s, lens, nq):
    h, kv, d, g = s["heads"], s["kv_heads"], s["head_dim"], s["heads"] // s["kv_heads"]
    table = s["table"].long()
    prefix = s["prefix"].tolist() if s["prefix"] is not None else [0] * len(nq)
    out, at = torch.zeros(sum(nq), h, d, dtype=torch.float64, device="cuda"), 0
    for i, (n, m) in enumerate(zip(nq, lens)):
        ids = table[i, : -(-m // s["page"])]
        pools = [_wide(tuple(p[ids] for p in c) if s["kind"] == "4bit" else c[ids], s["kind"], torch.float16)
                 for c in (s["k"], s["v"])]
        qpos, kpos = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
        hidden = (kpos > qpos) & (kpos >= prefix[i])
        if s["window"]:
            hidden |= kpos <= qpos - s["window"]
        for head in range(h):
            k, v = (p[:, head // g].reshape(-1, d)[:m] for p in pools)
            x = (s["q"][at: at + n, head].double() @ k.t()) * d ** -0.5
            if s["cap"]:
                x = (x / s["cap"]).tanh() * s["cap"]
            if s["slopes"] is not None:
                x = x - float(s["slopes"][head]) * (qpos - kpos).abs()
            x[hidden] = -math.inf
            out[at: at + n, head] = torch.softmax(x, -1) @ v
        at += n
    return out


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    nq, lens = _lengths(case)
    return (_exact_append if case["op"] == "append" else _exact_attend)(s, lens, nq)
