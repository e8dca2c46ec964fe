"""What a served batch's step adds to the paged KV cache, as measurable cases:

* ``axes``    ``kernels.paged_rope_axes_append``: queries and keys rotated by positions of several axes (time, height,
              width of images and video beside text), keys and values written to the sequences' pages.
* ``bounds``  ``kernels.paged_key_bounds``: upper and lower bounds, in 8 bits, of the keys of every page that a call's
              tokens lie in.
* ``select``  ``kernels.paged_select``: the pages of each token and KV head whose bounds allow the largest products.
* ``attend``  ``kernels.paged_attend_blocks``: attention over the selected pages.
* ``adjust``  ``kernels.adjust_logits``: penalties for repeated tokens, biases and grammar masks on a batch's logits.
* ``pick``    ``kernels.next_tokens``: the greedy choice from logits so adjusted.

A sequence of ``kv_lens[b]`` keys has its last ``q_start[b + 1] - q_start[b]`` tokens in the call; position p of it is
row p % page of page ``block_table[b, p // page]``, and a block is a page.  Sizes are the head layouts and the vocabulary
of the 3B-shaped decoder (24 query / 8 KV heads of 128, 128256 tokens) and generic ones; ``own`` picks the framework's
calls instead of the plain form.
"""
import math
import random

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "4bit": torch.float16}


def _paged(op, kind="fp16", batch=1, heads=24, kv_heads=8, head_dim=128, page=64, q=(1, 1), ctx=(0, 0), shape=0, count=32,
           cap=0.0, sections="16,24,24", interleaved=False, name=None):
    """``q``: tokens of a sequence in the call, ``ctx``: keys before them, both from .. to; the first sequence has the
    most of both, the others are spread by ``shape``.  ``count``: blocks a token and KV head attends to."""
    c = dict(op=op, kind=kind, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, q_lo=q[0],
             q_hi=q[1], ctx_lo=ctx[0], ctx_hi=ctx[1], shape=shape)
    if op == "axes":
        c.update(sections=sections, interleaved=interleaved)
    if op in ("select", "attend"):
        c["count"] = count
    if op == "attend":
        c["cap"] = cap
    return c if name is None else dict(c, name=name)


def _logits(op, kind="fp16", batch=1, vocab=128256, history=0, penalties=False, biases=0, masks=0, shape=0, name=None):
    """``history``: the longest row of tokens so far (0: none); ``biases``: biased tokens a row; ``masks``: grammar
    states whose masks the rows share (0: no masks)."""
    c = dict(op=op, kind=kind, batch=batch, vocab=vocab, history=history, penalties=penalties, biases=biases, masks=masks,
             shape=shape)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one token of each user of a served batch enters the cache, some of them after images
        _paged("axes", name="axes_tokens_b48", batch=48, ctx=(0, 4000), shape=1),
        # prompts with pictures in them enter a bf16 cache, axes interleaved over the pairs
        _paged("axes", name="axes_prompts_bf16", kind="bf16", batch=3, heads=32, page=32, q=(700, 2901), sections="24,20,20",
               interleaved=True, shape=2),
        # the pages that a served batch's new tokens lie in
        _paged("bounds", name="bounds_tokens_b64", batch=64, ctx=(0, 3000), shape=3),
        # all pages of prompts that a 4-bit cache has just taken
        _paged("bounds", name="bounds_prompts_4bit", kind="4bit", batch=3, heads=16, kv_heads=16, head_dim=64, page=32,
               q=(900, 8001), shape=4),
        # a served batch at all stages of long answers
        _paged("select", name="select_b64", batch=64, ctx=(0, 16000), shape=5),
        # one user with a very long document: latency, thousands of candidates a head
        _paged("select", name="select_one_long_bf16", kind="bf16", heads=32, page=32, ctx=(262000, 262000), count=64),
        # a served batch of long sequences: 4096 keys each instead of up to 32768
        _paged("attend", name="attend_b64", batch=64, ctx=(1000, 32767), count=64, shape=6),
        # one user with a very long document: 2048 keys of 131071, latency
        _paged("attend", name="attend_one_long_bf16", kind="bf16", heads=32, ctx=(131070, 131070), count=32),
        # five drafted tokens a sequence on a 4-bit cache, small heads, capped scores, each with blocks of its own
        _paged("attend", name="attend_drafts_4bit", kind="4bit", batch=12, heads=32, head_dim=64, q=(5, 5), ctx=(700, 9000),
               count=24, cap=30.0, shape=7),
        # the smallest: one user's next token under a grammar
        _logits("pick", name="pick_one_grammar", masks=1),
        # a served batch's logits on their way to a sampler: everything at once
        _logits("adjust", name="adjust_b64", batch=64, history=4096, penalties=True, biases=40, masks=5, shape=8),
        # many short chats on a small vocabulary, fp32 logits, penalties only
        _logits("pick", name="pick_b256_fp32", kind="fp32", batch=256, vocab=32003, history=900, penalties=True, shape=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choices(["axes", "bounds", "select", "attend", "adjust", "pick"], [3, 2, 4, 5, 2, 2])[0]
    shape = rng.randrange(1 << 20)
    if op in ("adjust", "pick"):
        return _logits(op, kind=rng.choice(["fp16", "bf16", "fp32"]), batch=_log(rng, 1, 64), vocab=_log(rng, 1000, 128256),
                       history=rng.choice([0, _log(rng, 1, 4096)]), penalties=rng.random() < 0.7,
                       biases=rng.choice([0, 0, _log(rng, 1, 300)]), masks=rng.choice([0, 1, 7]), shape=shape)
    heads, kv = rng.choice([(24, 8), (24, 8), (32, 8), (32, 4), (16, 16), (14, 2), (8, 1), (20, 1)])
    d, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 64, 128])
    c = dict(kind=rng.choice(["fp16", "bf16", "4bit"]), heads=heads, kv_heads=kv, head_dim=d, page=page, shape=shape)
    if op == "axes":
        a = rng.randint(1, d // 4)
        b = rng.randint(0, (d // 2 - a) // 2)
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, max(1, 4000 // batch))
        return _paged(op, batch=batch, q=(max(1, hi // 4), hi), ctx=(0, _log(rng, 1, max(1, 3000 // batch))),
                      sections="%d,%d,%d" % (d // 2 - a - b, a, b), interleaved=rng.random() < 0.5, **c)
    if op == "bounds":
        batch = _log(rng, 1, 64)
        hi = rng.choice([1, _log(rng, 1, max(1, 6000 // batch))])
        return _paged(op, batch=batch, q=(max(1, hi // 4), hi), ctx=(0, _log(rng, 1, max(1, 20000 // batch))), **c)
    stage = rng.choice(["tokens", "tokens", "drafts", "chunk"])
    if stage == "tokens":
        batch = _log(rng, 1, 64)
        return _paged(op, batch=batch, ctx=(0, _log(rng, 16, 260000 // batch)),
                      count=min(_log(rng, 4, 64), max(4, 260000 // (batch * page))), **c)
    if stage == "drafts":
        batch, q = _log(rng, 1, 16), rng.randint(2, 16)
        return _paged(op, batch=batch, q=(max(1, q // 2), q), ctx=(0, _log(rng, 16, 130000 // batch)),
                      count=min(_log(rng, 4, 64), max(4, 160000 // (batch * q * page))), **c)
    batch = rng.randint(1, 3)
    hi = _log(rng, 17, 384 // batch)
    return _paged(op, batch=batch, q=(max(1, hi // 3), hi), ctx=(0, _log(rng, 16, 60000 // batch)),
                  count=min(_log(rng, 4, 32), max(4, 160000 // (batch * hi * page))), **c)


def _lengths(case):
    """Tokens in the call and keys after it, per sequence."""
    r = random.Random(case["shape"])
    nq = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    nq[0], ctx[0] = case["q_hi"], case["ctx_hi"]
    return nq, [a + b for a, b in zip(nq, ctx)]


def _history_lengths(case):
    r = random.Random(case["shape"])
    lens = [r.randint(0, case["history"]) for _ in range(case["batch"])]
    lens[0] = case["history"]
    return lens, [r.randint(0, n) for n in lens]


# -- inputs --------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1 + int(seed))
    return (_prepare_logits if case["op"] in ("adjust", "pick") else _prepare_paged)(case, gen)


def _prepare_logits(case, gen):
    b, v = case["batch"], case["vocab"]

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s = dict(op=case["op"], logits=torch.randn(b, v, generator=gen, device="cuda").mul_(2.5).to(_DT[case["kind"]]),
             history=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None, bias_ids=None,
             bias=None, allowed=None, allowed_rows=None)
    if case["history"]:
        lens, prompts = _history_lengths(case)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["prompt_lens"] = torch.tensor(prompts, dtype=torch.int32, device="cuda")
        # some tokens are frequent, and what is likely now is often what was said before
        ids = (rand(b, case["history"]) ** 4 * v).long().clamp(max=v - 1)
        top = s["logits"].float().topk(min(v, 50), dim=1).indices
        again = top.gather(1, (rand(b, case["history"]) * top.shape[1]).long().clamp(max=top.shape[1] - 1))
        s["history"] = torch.where(rand(b, case["history"]) < 0.05, again, ids)
        if case["penalties"]:
            s["repetition"] = 1.0 + 0.3 * rand(b)
            s["presence"] = 0.5 * rand(b)
            s["frequency"] = 0.2 * rand(b)
    if case["biases"]:  # a row's biased tokens are distinct; rows with fewer are filled with -1
        n = min(case["biases"], v)
        step = v // n
        ids = torch.arange(n, device="cuda") * step + (rand(b, n) * step).long().clamp(max=step - 1)
        s["bias_ids"] = torch.where(rand(b, n) < 0.1, -1, ids)
        s["bias"] = torch.randn(b, n, generator=gen, device="cuda").mul_(4.0)
    if case["masks"]:  # grammar states allow few tokens or most; some rows have none
        m, words = case["masks"], -(-v // 32)
        share = rand(m, 1) ** 3
        share[0] = 0.02
        bits = rand(m, words * 32) < share
        power = 2 ** torch.arange(32, device="cuda")
        packed = (bits.view(m, words, 32) * power).sum(-1)
        s["allowed"] = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
        rows = (rand(b) * (m + 1)).int().clamp(max=m) - 1
        rows[0] = 0
        s["allowed_rows"] = rows.to(torch.int32)
    return s


def _codes_pool(gen, *shape):
    """Codes, scales and zero points as the 4-bit quantiser leaves them for values of deviation 1."""
    d = 2 * shape[-1]
    codes = torch.randint(0, 256, shape, generator=gen, device="cuda", dtype=torch.uint8)
    scales = torch.rand(*shape[:-1], d // 32, generator=gen, device="cuda").mul_(0.15).add_(0.2).half()
    zeros = torch.randint(5, 11, scales.shape, generator=gen, device="cuda", dtype=torch.uint8)
    return codes, scales, zeros


def _prepare_paged(case, gen):
    op, kind = case["op"], case["kind"]
    nq, lens = _lengths(case)
    b, h, kv, d, page = (case[k] for k in ("batch", "heads", "kv_heads", "head_dim", "page"))
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
    tokens = starts[-1]
    s = dict(op=op, kind=kind, heads=h, kv_heads=kv, head_dim=d, page=page, tokens=tokens, max_q=max(nq), table=table,
             kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
             q_start=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    if op in ("axes", "bounds", "attend"):
        s["k"] = _codes_pool(gen, pages, kv, page, d // 2) if kind == "4bit" else rand(pages, kv, page, d)
    if op in ("axes", "attend"):
        s["v"] = _codes_pool(gen, pages, kv, page, d // 2) if kind == "4bit" else rand(pages, kv, page, d)
    if op == "axes":
        s["qkv"] = rand(tokens, (h + 2 * kv) * d)
        # text moves all axes on together; a picture's rows and columns move two of them
        r = random.Random(case["shape"] + 1)
        pos = []
        for n, m in zip(nq, lens):
            first, wide = m - n, r.randint(4, 40)
            pos += [(first + i, first + i // wide, first + i % wide) if r.random() < 0.7 else (first + i,) * 3 for i in range(n)]
        s["positions"] = torch.tensor(pos, dtype=torch.int32, device="cuda").t().contiguous()
        sections = [int(x) for x in case["sections"].split(",")]
        pair = torch.arange(d // 2, device="cuda")
        if case["interleaved"]:
            which = pair % 3
            s["axis"] = torch.where(pair < 3 * torch.tensor(sections, device="cuda")[which], which, 0).to(torch.uint8)
        else:
            ends = torch.tensor(sections, device="cuda").cumsum(0)
            s["axis"] = torch.searchsorted(ends, pair, right=True).to(torch.uint8)
        inv = 1.0 / (500000.0 ** (torch.arange(0, d, 2, dtype=torch.float32, device="cuda") / d))
        ang = torch.arange(max(lens) + 40, dtype=torch.float32, device="cuda")[:, None] * inv
        s["cos"], s["sin"] = ang.cos(), ang.sin()
    if op in ("bounds", "select"):  # bounds of normal keys: about two and a half deviations each way
        codes = torch.randint(40, 128, (pages, kv, 2, d), generator=gen, device="cuda", dtype=torch.int8)
        codes[:, :, 1] *= -1
        s["bounds"] = codes, torch.rand(pages, kv, generator=gen, device="cuda").mul_(0.01).add_(0.02)
    if op in ("select", "attend"):
        s["q"], s["count"] = rand(tokens, h, d), case["count"]
    if op == "attend":
        s["cap"] = case["cap"]
        # as a selection leaves them: the first block, the last two, others at random; ascending, then -1
        seq, i = _positions(s, tokens)
        cur, j = i // page, torch.arange(max(need), device="cuda")
        x = torch.rand(tokens, kv, max(need), generator=gen, device="cuda")
        x[:, :, 0] = 2.0
        x = torch.where((j > cur[:, None] - 2)[:, None], 2.0, x)
        s["blocks"] = _best(torch.where((j > cur[:, None])[:, None], float("-inf"), x), case["count"])
    return s


# -- the plain form ------------------------------------------------------------------------------
def _positions(s, tokens):
    """The sequence and position of every token of the call."""
    t = torch.arange(tokens, device="cuda")
    starts = s["q_start"].long()
    seq = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return seq, s["kv_lens"].long()[seq] - starts[seq + 1] + t


def _best(x, count):
    """Where the `count` largest of the last dimension are, the lowest index on ties, -inf left out; ascending, then -1."""
    n = x.shape[-1]
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    at = torch.where(order.values > float("-inf"), order.indices, n)[..., :count].sort(-1).values
    at = torch.where(at == n, -1, at)
    return torch.nn.functional.pad(at, (0, max(0, count - n)), value=-1).to(torch.int32)


def _values(cache):
    """(q - z) * s of 4-bit rows, in 32 bits."""
    codes, scales, zeros = cache
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    c = c.unflatten(-1, (-1, 32))
    return ((c - zeros.float().unsqueeze(-1)) * scales.float().unsqueeze(-1)).flatten(-2)


def _rows(cache, at, kind):
    """Pages of a cache in 32 bits; 4-bit values rounded to fp16, as the operators define them."""
    return _values(tuple(p[at] for p in cache)).half().float() if kind == "4bit" else cache[at].float()


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


def _stored(cache, kind, page, at, x):
    """Writes rows x [tokens, kv, d] at row `at` of each token's page."""
    if kind == "4bit":
        codes, scales, zeros = _quantised(x)
        cache[0][page, :, at], cache[1][page, :, at], cache[2][page, :, at] = codes, scales, zeros
        return _values(cache).bfloat16()
    cache[page, :, at] = x
    return cache


def _plain_axes(s):
    qkv, h, kv, d = s["qkv"], s["heads"], s["kv_heads"], s["head_dim"]
    seq, i = _positions(s, qkv.shape[0])
    row = qkv.float().view(-1, h + 2 * kv, d)
    pair = torch.arange(d // 2, device="cuda")
    p = s["positions"].long().t()[:, s["axis"].long()]  # [tokens, d / 2]
    c, sn = s["cos"][p, pair][:, None], s["sin"][p, pair][:, None]
    a, b = row[:, :h + kv, :d // 2], row[:, :h + kv, d // 2:]
    rot = torch.cat([a * c - b * sn, b * c + a * sn], -1).to(qkv.dtype)
    page, at = s["table"][seq, i // s["page"]].long(), i % s["page"]
    return dict(q=rot[:, :h].contiguous(), k=_stored(s["k"], s["kind"], page, at, rot[:, h:]),
                v=_stored(s["v"], s["kind"], page, at, row[:, h + kv:].to(qkv.dtype)))


def _plain_bounds(s):
    page, kind = s["page"], s["kind"]
    lens, starts = s["kv_lens"].long(), s["q_start"].long()
    j = torch.arange(s["table"].shape[1], device="cuda")
    first = (lens - (starts[1:] - starts[:-1])) // page
    seq, block = torch.nonzero((j >= first[:, None]) & (j * page < lens[:, None]), as_tuple=True)
    at = s["table"][seq, block].long()
    k = _rows(s["k"], at, kind)
    hidden = (block * page)[:, None] + torch.arange(page, device="cuda") >= lens[seq][:, None]
    hidden = hidden[:, None, :, None]
    high, low = k.masked_fill(hidden, float("-inf")).amax(2), k.masked_fill(hidden, float("inf")).amin(2)
    most = torch.maximum(high.abs(), low.abs()).amax(-1)
    top = torch.full_like(most, 127.0)
    inv = (top / most)[..., None]
    codes, scales = s["bounds"]
    codes[at] = torch.stack([(high * inv).ceil(), (low * inv).floor()], 2).clamp(-127, 127).to(torch.int8)
    scales[at] = most / top
    return (codes.float() * scales[:, :, None, None]).to(_DT[kind])


def _plain_select(s):
    q, h, kv, d, g = s["q"], s["heads"], s["kv_heads"], s["head_dim"], s["heads"] // s["kv_heads"]
    tokens = q.shape[0]
    seq, i = _positions(s, tokens)
    cur = i // s["page"]
    starts = s["q_start"].long()
    t = torch.arange(s["max_q"], device="cuda")
    x = q.float().view(tokens, kv, g, d)
    most = x.abs().amax((2, 3), keepdim=True)
    code = (x * (torch.full_like(most, 127.0) / most)).round()
    code = code[(starts[:-1, None] + t).clamp(max=tokens - 1)].permute(0, 2, 1, 3, 4)  # [b, kv, q, g, d]
    b, n = code.shape[0], s["table"].shape[1]
    at = s["table"].long().clamp(min=0)
    codes, scales = s["bounds"][0][at].float(), s["bounds"][1][at].transpose(1, 2)  # whole numbers: exact in 32 bits
    high, low = codes[:, :, :, 0].permute(0, 2, 3, 1), codes[:, :, :, 1].permute(0, 2, 3, 1)
    code = code.reshape(b, kv, -1, d)
    x = torch.matmul(code.clamp(min=0.0), high.contiguous()) + torch.matmul(code.clamp(max=0.0), low.contiguous())
    x = x.view(b, kv, t.numel(), g, n).amax(3) * scales[:, :, None]
    at = torch.arange(tokens, device="cuda") - starts[seq]
    x = x.permute(0, 2, 1, 3)[seq, at]  # [tokens, kv, n]
    j = torch.arange(n, device="cuda")
    x = torch.where(((j < 1) | (j > cur[:, None] - 2))[:, None], float("inf"), x)
    return _best(torch.where((j > cur[:, None])[:, None], float("-inf"), x), s["count"])


def _plain_attend(s):
    q, h, kv, d, g = s["q"], s["heads"], s["kv_heads"], s["head_dim"], s["heads"] // s["kv_heads"]
    tokens, page, blocks = q.shape[0], s["page"], s["blocks"].long()
    seq, i = _positions(s, tokens)
    at = s["table"].long()[seq[:, None, None], blocks.clamp(min=0)].clamp(min=0)
    head = torch.arange(kv, device="cuda")[:, None]
    both = [(tuple(p[at, head] for p in c) if s["kind"] == "4bit" else c[at, head]) for c in (s["k"], s["v"])]
    k, v = [(_values(c).half().float() if s["kind"] == "4bit" else c.float()).view(tokens * kv, -1, d) for c in both]
    x = torch.matmul(q.float().view(tokens * kv, g, d), k.transpose(1, 2).contiguous()) / math.sqrt(d)
    if s["cap"]:
        x = s["cap"] * torch.tanh(x / s["cap"])
    j = blocks[..., None] * page + torch.arange(page, device="cuda")
    see = ((blocks >= 0)[..., None] & (j <= i[:, None, None, None])).view(tokens * kv, 1, -1)
    x = x.masked_fill(~see, float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    return (torch.matmul(x, v) / x.sum(-1, keepdim=True)).view(tokens, h, d).to(q.dtype)


def _plain_adjusted(s):
    """The adjusted logits in 32 bits."""
    x = s["logits"].float()
    b, v = x.shape
    if s["repetition"] is not None:
        at = torch.arange(s["history"].shape[1], device="cuda")
        here = at < s["lens"].long()[:, None]
        said = here & (at >= s["prompt_lens"].long()[:, None])
        seen = torch.zeros(b, v, device="cuda").scatter_add_(1, s["history"], here.float()) > 0
        count = torch.zeros(b, v, device="cuda").scatter_add_(1, s["history"], said.float())
        r = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None] * count
        x = x - s["presence"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        ids = s["bias_ids"]
        row = torch.zeros(b, v + 1, device="cuda").scatter_(1, torch.where(ids < 0, v, ids), s["bias"])
        x = x + row[:, :v]
    if s["allowed"] is not None:
        at = torch.arange(v, device="cuda")
        ok = ((s["allowed"].long()[:, at // 32] >> (at % 32)) & 1) > 0
        rows = s["allowed_rows"].long()
        x = x.masked_fill(~(ok[rows.clamp(min=0)] | (rows < 0)[:, None]), float("-inf"))
    return x


def _plain_pick(s):
    x = _plain_adjusted(s)
    top = x.amax(1, keepdim=True)
    at = torch.where(x == top, torch.arange(x.shape[1], device="cuda"), x.shape[1]).amin(1)
    return torch.where(top[:, 0] == float("-inf"), -1, at)


# -- one pass ------------------------------------------------------------------------------------
def _own(s):
    from spectra_amd import kernels as K
    op = s["op"]
    if op in ("adjust", "pick"):
        more = dict(history=s["history"], lens=s["lens"], prompt_lens=s["prompt_lens"], repetition=s["repetition"],
                    presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"], bias=s["bias"],
                    allowed=s["allowed"], allowed_rows=s["allowed_rows"])
        if op == "adjust":
            return K.adjust_logits(s["logits"], **more)
        if "workspace" not in s:  # kept from step to step, as a serving loop does
            s["workspace"] = K.next_tokens_workspace(s["logits"].device)
        return K.next_tokens(s["logits"], workspace=s["workspace"], **more)
    where = s["kv_lens"], s["q_start"], s["table"]
    if op == "axes":
        q = K.paged_rope_axes_append(s["qkv"], s["positions"], s["axis"], *where, s["cos"], s["sin"], s["heads"], s["k"], s["v"])
        if s["kind"] == "4bit":
            return dict(q=q, k=K.kv4_dequantize(*s["k"]), v=K.kv4_dequantize(*s["v"]))
        return dict(q=q, k=s["k"], v=s["v"])
    if op == "bounds":
        K.paged_key_bounds(s["tokens"], *where, s["k"], s["bounds"])
        return K.paged_bounds_values(s["bounds"], _DT[s["kind"]])
    if op == "select":
        if "workspace" not in s:
            s["workspace"] = K.paged_select_workspace(s["q"].device)
        return K.paged_select(s["q"], *where, s["bounds"], s["page"], s["count"], sink=1, local=2, workspace=s["workspace"])
    if "workspace" not in s:
        s["workspace"] = K.paged_attend_workspace(s["head_dim"], s["q"].device)
    return K.paged_attend_blocks(s["q"], s["blocks"], *where, s["k"], s["v"], cap=s["cap"], workspace=s["workspace"])


@torch.no_grad()
def run(state):
    if own:
        return _own(state)
    op = state["op"]
    if op == "adjust":
        return _plain_adjusted(state).to(state["logits"].dtype)
    return {"axes": _plain_axes, "bounds": _plain_bounds, "select": _plain_select, "attend": _plain_attend,
            "pick": _plain_pick}[op](state)


# -- what a pass cannot do without ---------------------------------------------------------------
def _row_bytes(case):
    """One head's key (or value) of one position."""
    d = case["head_dim"]
    return d / 2 + 3 * d / 32 if case["kind"] == "4bit" else 2 * d


def work(case):
    op, b = case["op"], case["batch"]
    if op in ("adjust", "pick"):
        each = 4 if case["kind"] == "fp32" else 2
        n = b * case["vocab"] * each * (2 if op == "adjust" else 1) + 12 * b * case["biases"]
        n += 8 * sum(_history_lengths(case)[0]) if case["history"] and case["penalties"] else 0
        return {"bytes": n + case["masks"] * case["vocab"] / 8 + 8 * b, "flops": 8 * b * case["vocab"]}
    nq, lens = _lengths(case)
    h, kv, d, page, tokens = case["heads"], case["kv_heads"], case["head_dim"], case["page"], sum(nq)
    pages = sum(-(-n // page) for n in lens) + 2
    if op == "axes":
        n = tokens * ((2 * h + 2 * kv) * 2 * d + 2 * kv * _row_bytes(case) + 4 * d + 12)
        if case["kind"] == "4bit":  # the pages' values read back
            n += 2 * kv * page * pages * (_row_bytes(case) + 2 * d)
        return {"bytes": n, "flops": tokens * (h + kv) * 3 * d}
    if op == "bounds":  # the rows of the pages that tokens lie in; the bounds' values read back
        rows = sum(m - (m - n) // page * page for n, m in zip(nq, lens))
        blocks = sum((m - 1) // page - (m - n) // page + 1 for n, m in zip(nq, lens))
        return {"bytes": kv * (rows * _row_bytes(case) + blocks * (2 * d + 4) + pages * (2 * d + 4 + 4 * d)), "flops": kv * rows * 2 * d}
    if op == "select":
        pairs = sum(i // page + 1 for n, m in zip(nq, lens) for i in range(m - n, m))
        blocks = sum((m - 1) // page + 1 for m in lens)
        return {"bytes": blocks * kv * (2 * d + 4) + tokens * (2 * h * d + 4 * kv * case["count"]), "flops": pairs * h * 4 * d}
    keys = read = 0.0
    for n, m in zip(nq, lens):
        seen, rest = 0, 1.0  # keys that the tokens see; the share of the sequence's blocks that no token does
        for i in range(m - n, m):
            all_, got = i // page + 1, min(case["count"], i // page + 1)
            seen += got * page - (page - 1 - i % page)
            rest *= 1.0 - got / all_
        keys += seen
        read += (1.0 - rest) * m
    return {"bytes": 2 * kv * read * _row_bytes(case) + 2 * tokens * h * d * 2 + 4 * tokens * kv * case["count"], "flops": 4 * h * d * keys}


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


def _exact_axes(s, nq, lens):
    h, kv, d, page = s["heads"], s["kv_heads"], s["head_dim"], s["page"]
    table = s["table"].tolist()
    k, v = _wide(s["k"], s["kind"]), _wide(s["v"], s["kind"])
    axis = s["axis"].tolist()
    where = s["positions"].long()
    c = torch.stack([s["cos"].double()[where[a], e] for e, a in enumerate(axis)], -1)[:, None]
    sn = torch.stack([s["sin"].double()[where[a], e] for e, a in enumerate(axis)], -1)[:, None]
    row = s["qkv"].double().view(-1, h + 2 * kv, d)
    a, b = row[:, :h + kv].chunk(2, -1)
    rot = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    at = 0
    for b_, (n, m) in enumerate(zip(nq, lens)):
        for pool, x in ((k, rot[at: at + n, h:]), (v, row[at: at + n, h + kv:])):
            if s["kind"] == "4bit":
                y = x.half().double().reshape(n, kv, d // 32, 32)
                low = y.min(-1, keepdim=True).values
                step = ((y.max(-1, keepdim=True).values - low).half().double() / 15).half().double()
                z = (-low / step).half().double().round().clamp(0, 15)
                x = ((((y + z * step) / step).round().clamp(0, 15) - z) * step).reshape(n, kv, d)
            first = m - n
            while first < m:  # the run of positions in one page
                end = min(m, (first // page + 1) * page)
                pool[table[b_][first // page], :, first % page: first % page + end - first] = \
                    x[first - (m - n): end - (m - n)].transpose(0, 1)
                first = end
        at += n
    return dict(q=rot[:, :h], k=k, v=v)


def _exact_bounds(s, nq, lens):
    page, (codes, scales) = s["page"], s["bounds"]
    out = codes.double() * scales.double()[:, :, None, None]
    for row, n, m in zip(s["table"].tolist(), nq, lens):
        for j in range((m - n) // page, (m - 1) // page + 1):
            cache = tuple(p[row[j]] for p in s["k"]) if s["kind"] == "4bit" else s["k"][row[j]]
            x = _wide(cache, s["kind"], torch.float16)[:, : m - j * page]
            step = x.abs().amax((1, 2))[:, None] / 127.0  # outwards to whole steps, the largest of all being 127
            out[row[j], :, 0] = (x.max(1).values / step).ceil().clamp(-127, 127) * step
            out[row[j], :, 1] = (x.min(1).values / step).floor().clamp(-127, 127) * step
    return out


def _exact_attend(s, nq, lens):
    h, kv, d, g, page = s["heads"], s["kv_heads"], s["head_dim"], s["heads"] // s["kv_heads"], s["page"]
    out, at = torch.zeros(sum(nq), h, d, dtype=torch.float64, device="cuda"), 0
    for b, (n, m) in enumerate(zip(nq, lens)):
        ids = s["table"][b, : -(-m // page)].long()
        k, v = [_wide(tuple(p[ids] for p in c) if s["kind"] == "4bit" else c[ids], s["kind"], torch.float16)
                for c in (s["k"], s["v"])]  # [blocks, kv, page, d]
        named = torch.zeros(n, kv, len(ids) + 1, dtype=torch.bool, device="cuda")
        blocks = s["blocks"][at: at + n].long()
        named.scatter_(2, torch.where(blocks < 0, len(ids), blocks), True)
        i = torch.arange(m - n, m, device="cuda")[:, None]
        for head in range(h):
            see = named[:, head // g, :-1].repeat_interleave(page, 1) & (torch.arange(len(ids) * page, device="cuda") <= i)
            x = s["q"][at: at + n, head].double() @ k[:, head // g].reshape(-1, d).t().contiguous() * d ** -0.5
            if s["cap"]:
                x = (x / s["cap"]).tanh() * s["cap"]
            x[~see] = -math.inf
            out[at: at + n, head] = torch.softmax(x, -1) @ v[:, head // g].reshape(-1, d)
        at += n
    return out


def _exact_logits(s, case):
    x = s["logits"].double()
    if s["repetition"] is not None:
        lens, prompts = _history_lengths(case)
        for b, (n, p) in enumerate(zip(lens, prompts)):
            row = s["history"][b, :n]
            ids = row.unique()
            r = s["repetition"][b].double()
            x[b, ids] = torch.where(x[b, ids] > 0, x[b, ids] / r, x[b, ids] * r)
            ids, times = row[p:].unique(return_counts=True)
            x[b, ids] -= s["frequency"][b].double() * times + s["presence"][b].double()
    for b in range(x.shape[0]):
        if s["bias_ids"] is not None:
            ids = s["bias_ids"][b]
            x[b, ids[ids >= 0]] += s["bias"][b][ids >= 0].double()
        if s["allowed"] is not None and int(s["allowed_rows"][b]) >= 0:
            words = s["allowed"][int(s["allowed_rows"][b])].long()
            bits = torch.stack([words >> e & 1 for e in range(32)], -1).flatten()[: x.shape[1]]
            x[b, bits == 0] = -math.inf
    if s["op"] == "adjust":
        return x
    return torch.where(x.amax(1) == -math.inf, -1, x.argmax(1))


@torch.no_grad()
def exact(case, seed):
    if case["op"] == "select":  # what 8-bit codes and 32-bit scores choose: nothing that 64 bits would say better
        return None
    s = prepare(case, seed)
    if case["op"] in ("adjust", "pick"):
        return _exact_logits(s, case)
    nq, lens = _lengths(case)
    return {"axes": _exact_axes, "bounds": _exact_bounds, "attend": _exact_attend}[case["op"]](s, nq, lens)
