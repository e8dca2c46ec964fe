"""The paged KV cache: appending with the rotation on the way, and attention over the pages, against plain
computations in 64 bits.

Tolerances of attention, elementwise, from the roundings that the operator has: u = eps / 2 of the activations' type
for the output and for every weight (relative to the sum A of weight times |value|; half the smallest subnormal for
weights below fp16's range); and the scores' error delta, which scales every weight by exp(delta) and thus moves
numerator and denominator by at most 2 delta A: fp32 products and sums of d terms (d 2^-24 of the sum of |q k|), a cap
(a few 2^-23 of it, from exp2 and the reciprocal) and the bias (2^-22 of it)."""
import ctypes
import math

import pytest
import torch

from spectra_amd import _lib as L

KINDS = ["fp16", "bf16", "4bit"]
_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "4bit": torch.float16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _values(cache, kind):
    """What 4-bit rows stand for, in 64 bits."""
    if kind != "4bit":
        return cache.double()
    codes, scales, zeros = cache
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    z, s = (t.double().repeat_interleave(32, -1) for t in (zeros, scales))
    return ((q - z) * s).half().double()


class Batch:
    """A batch on scattered pages: ``n`` tokens of the call and ``lens`` keys per sequence.  Rows of the pool that no
    sequence fills hold NaN; table entries that none needs, ids outside the pool."""

    def __init__(self, kind, n, lens, heads, kv, d, page, seed=0, pad=0, pages_apart=False):
        g = _gen(seed)
        self.kind, self.n, self.lens, self.heads, self.kv, self.d, self.page = kind, n, lens, heads, kv, d, page
        dt = _DT[kind]
        need = [-(-m // page) for m in lens]
        pages = sum(need) + 1
        order = torch.randperm(pages, generator=g, device="cuda").int()
        self.table = torch.full((len(n), max(need + [1]) + 1), 1 << 30, dtype=torch.int32, device="cuda")
        self.table[:, ::2] = -7
        self.valid = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        at = 0
        for b, (m, w) in enumerate(zip(lens, need)):
            self.table[b, :w] = order[at: at + w]
            at += w
            for p in range(w):
                self.valid[self.table[b, p].long(), : min(page, m - p * page)] = True
        step = 2 if pages_apart else 1  # pages apart: every second page of a larger pool

        def pool(last, dtype):
            return torch.zeros(pages * step, kv, page, last, dtype=dtype, device="cuda")[::step]

        def rand(*shape):
            return torch.randn(*shape, generator=g, device="cuda").to(dt)

        if kind == "4bit":
            from spectra_amd import kernels as K
            self.k, self.v = [], []
            for out in (self.k, self.v):
                for t in K.kv4_quantize(rand(pages * kv, page, d)):
                    x = pool(t.shape[-1], t.dtype)
                    x.copy_(t.view(pages, kv, page, -1))
                    out.append(x)
                out[1].masked_fill_(~self.valid[:, None, :, None], float("nan"))
            self.k, self.v = tuple(self.k), tuple(self.v)
        else:
            self.k, self.v = pool(d, dt), pool(d, dt)
            for x in (self.k, self.v):
                x.copy_(rand(pages, kv, page, d).masked_fill(~self.valid[:, None, :, None], float("nan")))
        starts = [0]
        for m in n:
            starts.append(starts[-1] + m)
        self.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.tokens = starts[-1] + pad
        self.q = rand(self.tokens, heads, d)
        self.rand = rand

    def rows(self, b):
        """Keys and values of sequence b [kv, len, d], 64 bits."""
        ids = self.table[b, : -(-self.lens[b] // self.page)].long()
        return [_values(tuple(t[ids] for t in c) if self.kind == "4bit" else c[ids], self.kind).transpose(0, 1)
                .reshape(self.kv, -1, self.d)[:, : self.lens[b]] for c in (self.k, self.v)]

    def reference(self, scale=None, cap=0.0, window=0, slopes=None, prefix=None):
        """Output and elementwise tolerance, by sequence and head."""
        scale = 1.0 / math.sqrt(self.d) if scale is None else scale
        u = torch.finfo(_DT[self.kind]).eps / 2
        sub = 2.0 ** -25 if self.kind != "bf16" else 0.0
        out = torch.zeros(self.tokens, self.heads, self.d, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(out)
        at = 0
        for b, (n, m) in enumerate(zip(self.n, self.lens)):
            if n == 0:
                continue
            k, v = self.rows(b)
            i = torch.arange(m - n, m, device="cuda")[:, None]
            j = torch.arange(m, device="cuda")[None]
            see = (j <= i) | (j < (int(prefix[b]) if prefix is not None else 0))
            if window:
                see &= i - j < window
            for h in range(self.heads):
                kh, vh = k[h * self.kv // self.heads], v[h * self.kv // self.heads]
                qh = self.q[at: at + n, h].double()
                x = qh @ kh.T * scale
                delta = self.d * 2.0 ** -24 * (qh.abs() @ kh.abs().T * scale).amax(-1, keepdim=True) if m else 0.0
                if cap:
                    x = cap * torch.tanh(x / cap)
                    delta = delta + cap * 2.0 ** -20
                if slopes is not None:
                    bias = float(slopes[h]) * (i - j).abs()
                    x = x - bias
                    delta = delta + 2.0 ** -22 * bias.amax() if m else delta
                x = x.masked_fill(~see, -math.inf)
                top = x.amax(-1, keepdim=True) if m else torch.zeros(n, 1, device="cuda", dtype=torch.float64)
                e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
                e = torch.where(see, e, 0.0)
                total = e.sum(-1, keepdim=True)
                vis = torch.where(see, 1.0, 0.0).double()
                clean = vh.masked_fill(~torch.isfinite(vh), 0.0)
                o = (e @ clean) / torch.where(total == 0, 1.0, total)
                lost = ~torch.isfinite(vh)  # a value that is not finite reaches the rows that see it, no others
                o = o.masked_fill((vis @ lost.double()) > 0, math.nan)
                a = (e @ clean.abs()) / torch.where(total == 0, 1.0, total)
                out[at: at + n, h] = o
                tol[at: at + n, h] = u * o.abs() + (u + 2 * delta + 2.0 ** -20) * a + \
                    sub * (1 + (vis @ clean.abs()) / torch.where(total == 0, 1.0, total))
            at += n
        return out, tol

    def attend(self, **kw):
        from spectra_amd import kernels as K
        return K.paged_attend(self.q, self.kv_lens, self.q_start, self.table, self.k, self.v, **kw)

    def check(self, **kw):
        """Runs on an output that already holds something, compares, and returns the output."""
        out = torch.full_like(self.q, 7.0)
        got = self.attend(out=out, **kw)
        assert got is out
        kw.pop("workspace", None)
        want, tol = self.reference(**kw)
        used = sum(self.n)
        assert torch.all(out[used:] == 7.0), "rows behind the last sequence were written"
        x, y = out[:used].double(), want[:used]
        assert torch.equal(torch.isnan(x), torch.isnan(y))
        off = ((x - y).abs() - tol[:used]).nan_to_num(-1.0).max()
        assert off <= 0, f"{float(off):.3g} outside the tolerance"
        return out


# -- attention: forms, sizes, masks --------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,d", [(24, 8, 128), (4, 4, 64), (14, 2, 64), (16, 1, 128), (5, 1, 128)])
@pytest.mark.parametrize("page", [16, 64])
def test_single_tokens(hip, kind, heads, kv, d, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 300, 517, 0]
    n = [1] * 15 + [0]
    Batch(kind, n, lens, heads, kv, d, page, seed=heads + page, pad=3).check()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,d", [(8, 4, 64), (24, 8, 128), (32, 1, 64)])
def test_drafted_tokens(hip, kind, heads, kv, d):
    n = [5, 1, 4, 2, 0, 7, 3]
    lens = [5, 40, 131, 700, 12, 263, 64]
    Batch(kind, n, lens, heads, kv, d, 32, seed=3, pad=1).check()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,d,page", [(6, 2, 128, 16), (4, 4, 64, 128), (7, 1, 64, 32)])
@pytest.mark.parametrize("n,lens", [([1, 90, 257, 0, 33], [70, 90, 300, 0, 512]), ([129], [129]), ([64, 200], [1000, 200])])
def test_prompts(hip, kind, heads, kv, d, page, n, lens):
    Batch(kind, n, lens, heads, kv, d, page, seed=len(n), pad=2).check()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [[1, 1, 1], [3, 2, 4], [150, 40, 77]])
@pytest.mark.parametrize("mods", [dict(cap=2.0), dict(slopes=True), dict(window=50), dict(prefix=True),
                                  dict(window=1), dict(cap=30.0, slopes=True, window=200, prefix=True), dict(scale=0.4)])
def test_scores_and_masks(hip, kind, n, mods):
    b = Batch(kind, n, [200, 333, 150], 6, 2, 64, 16, seed=5)
    mods = dict(mods)
    if "slopes" in mods:
        mods["slopes"] = torch.exp2(-torch.arange(1, 7, device="cuda").float())
    if "prefix" in mods:
        mods["prefix"] = torch.tensor([64, 0, 1000], dtype=torch.int32, device="cuda")
    b.check(**mods)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [[1, 1, 1], [3, 2, 4], [150, 40, 77]])
@pytest.mark.parametrize("cap,scale", [(200.0, 0.125), (300.0, 0.125), (1e5, 0.125), (1e6, 0.3), (1e8, 0.125), (3e29, 0.125),
                                       (300.0, 30.0), (2000.0, 400.0)])
def test_large_caps(hip, kind, n, cap, scale):
    """Caps far above the scores, and large ones that the scores reach.  A cap's error: 2^-20 of it up to 256 (its form is a
    constant plus the score); past that 2^-19 of the score, whatever the cap: 10 roundings of 2^-24 where tanh is a
    polynomial, and where it is 1 - 2 / (1 + 2^t), at least 0.24, 6 of 2^-24 in all (exp2 and the reciprocal are off by a
    unit)."""
    b = Batch(kind, n, [200, 333, 150], 6, 2, 64, 16, seed=41)
    got, u, at = b.attend(cap=cap, scale=scale), torch.finfo(_DT[kind]).eps / 2, 0
    sub = 2.0 ** -25 if kind != "bf16" else 0.0
    for s, (t, m) in enumerate(zip(b.n, b.lens)):
        k, v = b.rows(s)
        see = torch.arange(m, device="cuda")[None] <= torch.arange(m - t, m, device="cuda")[:, None]
        for h in range(6):
            qh, kh, vh = b.q[at: at + t, h].double(), k[h // 3], v[h // 3]
            x = cap * torch.tanh(qh @ kh.T * scale / cap)
            delta = 64 * 2.0 ** -24 * (qh.abs() @ kh.abs().T * scale).amax(-1, keepdim=True)
            delta = delta + (2.0 ** -20 * cap if cap <= 256 else 2.0 ** -19 * x.abs().amax(-1, keepdim=True))
            x = x.masked_fill(~see, -math.inf)
            p = torch.softmax(x, -1)
            total = torch.exp(x - x.amax(-1, keepdim=True)).sum(-1, keepdim=True)
            want, a = p @ vh, p @ vh.abs()
            tol = u * want.abs() + (u + 2 * delta + 2.0 ** -20) * a + sub * (1 + (see.double() @ vh.abs()) / total)
            assert torch.all((got[at: at + t, h].double() - want).abs() <= tol)
        at += t


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "4bit"])
@pytest.mark.parametrize("n", [1, 6, 40])
def test_long_caches_split(hip, kind, n):
    """Few tiles of long caches: every tile's keys in many pieces, joined in order."""
    b = Batch(kind, [n, n], [9001, 4000], 4, 2, 128, 64, seed=9)
    from spectra_amd import kernels as K
    ws = K.paged_attend_workspace(128)
    first = b.check(workspace=ws)
    for _ in range(3):
        assert torch.equal(b.attend(workspace=ws), first), "the same call gave other bits"


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("prefix", [False, True])
def test_distances_of_far_positions(hip, n, prefix):
    """Positions past 2^24, which fp32 does not hold: the distances, which the bias takes, are small.  The long
    sequence names the same few pages over and over, and a window leaves its last keys."""
    from spectra_amd import kernels as K
    g, page, d, window, m = _gen(n), 4096, 64, 48, (1 << 27) + 77
    k, v = (torch.randn(4, 1, page, d, generator=g, device="cuda").half() for _ in range(2))
    table = (torch.arange(m // page + 1, device="cuda") % 4).int()[None]
    q = torch.randn(n, 2, d, generator=g, device="cuda").half()
    slopes = torch.tensor([0.5, 0.125], device="cuda")
    got = K.paged_attend(q, torch.tensor([m], dtype=torch.int32, device="cuda"),
                         torch.tensor([0, n], dtype=torch.int32, device="cuda"), table, k, v, window=window, slopes=slopes,
                         prefix=torch.tensor([m], dtype=torch.int32, device="cuda") if prefix else None)
    i = torch.arange(m - n, m, device="cuda")[:, None]
    j = torch.arange(m - n - window, m, device="cuda")[None]
    see = (i - j < window) & ((j <= i) | prefix)
    kk, vv = (x[table[0, j[0] // page].long(), 0, j[0] % page].double() for x in (k, v))
    for h in range(2):
        bias = float(slopes[h]) * (i - j).abs()
        qh = q[:, h].double()
        delta = d * 2.0 ** -24 * (qh.abs() @ kk.abs().T / 8).amax(-1, keepdim=True) + 2.0 ** -22 * bias.amax()
        p = torch.softmax((qh @ kk.T / 8 - bias).masked_fill(~see, -math.inf), -1)
        want, a = p @ vv, p @ vv.abs()
        tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2 * delta + 2.0 ** -20) * a + 2.0 ** -25 * (1 + see.double() @ vv.abs())
        assert torch.all((got[:, h].double() - want).abs() <= tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [[1, 1], [3, 4], [70, 40]])
def test_pages_gigabytes_apart(hip, kind, n):
    """Offsets past 32 bits, in elements and in bytes: the same rows in pages that lie 3 GiB apart give the same bits."""
    from spectra_amd import kernels as K
    b = Batch(kind, n, [90, 75], 4, 2, 64, 64, seed=31)
    heads, kv, d = b.heads, b.kv, b.d

    def apart(x):
        step = 3 * (1 << 30) // x.element_size() if x.dtype != torch.half or kind != "4bit" else 1 << 30
        far = torch.empty(step * (x.shape[0] - 1) + x[0].numel(), dtype=x.dtype, device="cuda")
        far = far.as_strided(x.shape, (step,) + tuple(x.stride()[1:]))
        far.copy_(x)
        return far

    near = b.check()
    held = b.k, b.v
    b.k, b.v = (tuple(apart(t) for t in c) if kind == "4bit" else apart(c) for c in held)
    assert torch.equal(b.attend()[: sum(n)], near[: sum(n)])
    qkv = b.rand(b.tokens, (heads + 2 * kv) * d)
    for c in (held, (b.k, b.v)):
        K.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, None, None, heads, *c)
    for x, y in zip(held, (b.k, b.v)):
        for s, t in zip(x, y) if kind == "4bit" else [(x, y)]:
            assert torch.equal(torch.nan_to_num(s.float(), 99.0), torch.nan_to_num(t.float(), 99.0))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [[1, 1, 1], [4, 2, 4], [50, 64, 30]])
def test_sequences_that_share_pages(hip, kind, n):
    """A common beginning held once, and a whole sequence named twice."""
    b = Batch(kind, n, [150, 170, 150], 6, 2, 64, 16, seed=23)
    b.table[1, :6] = b.table[0, :6]
    b.table[2] = b.table[0]
    b.check()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "4bit"])
@pytest.mark.parametrize("kw", [dict(), dict(window=700, cap=20.0), dict(prefix=True)])
def test_cut_prompts(hip, kind, kw):
    """Chunks on long contexts, few enough that their keys are cut: 13 key steps (the least that are), 16, and many; a last
    tile that is not full, rows of a cut tile that see different keys."""
    lens = [780, 1024, 5003]
    b = Batch(kind, [30, 43, 77], lens, 6, 2, 128, 32, seed=29)
    if "prefix" in kw:
        kw = dict(kw, prefix=torch.tensor([0, 1024, 4000], dtype=torch.int32, device="cuda"))
    b.check(**kw)
    alone = Batch(kind, [40], [1000], 3, 1, 64, 64, seed=30)
    alone.check(**dict(kw, prefix=torch.tensor([990], dtype=torch.int32, device="cuda")))


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [65, 200])
def test_many_sequences(hip, batch):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 300, (batch,), generator=g).tolist()
    n = [min(m, 1) for m in lens]
    Batch("fp16", n, lens, 3, 1, 64, 16, seed=batch, pad=5).check()
    n = [min(m, int(x)) for m, x in zip(lens, torch.randint(0, 60, (batch,), generator=g))]
    Batch("bf16", n, lens, 3, 1, 64, 16, seed=batch).check()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "4bit"])
def test_large_batch(hip, kind):
    """So many tiles that a sum of padded ones would be 2^32: 65536 sequences, which share the pages of 64."""
    from spectra_amd import kernels as K
    times = 1024
    few = Batch(kind, [1] * 64, [1024 - 2 * b for b in range(64)], 8, 8, 64, 64, seed=37)
    want, tol = few.reference()
    got = torch.full((64 * times, 8, 64), 7.0, dtype=few.q.dtype, device="cuda")
    K.paged_attend(few.q.repeat(times, 1, 1), few.kv_lens.repeat(times), torch.arange(64 * times + 1, dtype=torch.int32, device="cuda"),
                   few.table.repeat(times, 1), few.k, few.v, out=got)
    for part in got.view(times, 64, 8, 64).split(64):
        assert torch.all((part.double() - want).abs() <= tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("far", [False, True])
def test_tables_past_32_bits(hip, kind, n, far):
    """Tables of so many key steps in all that shares are counted in steps of several: with short sequences, and with
    long ones of which a window leaves the last keys (their lengths are counted whole beside a prefix)."""
    from spectra_amd import kernels as K
    g, page, d, kv, heads, batch, window = _gen(n), 65536, 64, 4, 8, 72, 300
    pool = lambda: torch.randn(3, kv, page, d, generator=g, device="cuda").to(_DT[kind])  # noqa: E731
    k, v = pool(), pool()
    if kind == "4bit":
        k, v = (tuple(t.view(3, kv, page, -1) for t in K.kv4_quantize(x.view(3 * kv, page, d))) for x in (k, v))
    table = (torch.arange(batch * 8193, device="cuda") % 3).int().view(batch, -1)
    lens = [((1 << 29) - 77 * b if far else 20 + 11 * b) for b in range(batch)]
    q = torch.randn(batch * n, heads, d, generator=g, device="cuda").to(_DT[kind])
    got = K.paged_attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                         torch.arange(0, batch * n + 1, n, dtype=torch.int32, device="cuda"), table, k, v, window=window,
                         prefix=torch.zeros(batch, dtype=torch.int32, device="cuda"))
    u, sub = torch.finfo(_DT[kind]).eps / 2, 2.0 ** -25 if kind != "bf16" else 0.0
    for b, m in enumerate(lens):
        i = torch.arange(m - n, m, device="cuda")[:, None]
        j = torch.arange(max(0, m - n - window), m, device="cuda")[None]
        see = (i - j < window) & (j <= i)
        at = table[b, j[0] // page].long(), slice(None), j[0] % page
        kk, vv = (_values(tuple(t[at] for t in c) if kind == "4bit" else c[at], kind) for c in (k, v))
        for h in range(heads):
            qh, kh, vh = q[b * n: b * n + n, h].double(), kk[:, h * kv // heads], vv[:, h * kv // heads]
            delta = d * 2.0 ** -24 * (qh.abs() @ kh.abs().T / 8).amax(-1, keepdim=True)
            x = (qh @ kh.T / 8).masked_fill(~see, -math.inf)
            p = torch.softmax(x, -1)
            total = torch.exp(x - x.amax(-1, keepdim=True)).sum(-1, keepdim=True)
            want, a = p @ vh, p @ vh.abs()
            tol = u * want.abs() + (u + 2 * delta + 2.0 ** -20) * a + sub * (1 + (see.double() @ vh.abs()) / total)
            assert torch.all((got[b * n: b * n + n, h].double() - want).abs() <= tol), (b, h)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [[1, 1], [3, 4], [70, 40]])
@pytest.mark.parametrize("size", [7e37, 1e-24])
def test_values_at_the_ends_of_the_range(hip, n, size):
    """bf16 values whose unweighted sums pass fp32's range, and tiny ones."""
    b = Batch("bf16", n, [90, 3000], 6, 2, 128, 32, seed=47)
    b.v = (b.v.float().clamp(-4.0, 4.0) * size).bfloat16()
    assert torch.all(torch.isfinite(b.check()[: sum(n)]))
    b.q.zero_()  # (all weights alike)
    assert torch.all(torch.isfinite(b.check()[: sum(n)]))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("n", [[1] * 40, [3, 4] * 20, [70, 40]])
def test_means_of_the_largest_value(hip, kind, n):
    """Values that are all the type's largest: so is their mean, whatever the weights' roundings."""
    b = Batch(kind, n, [90 + 7 * s for s in range(len(n))], 6, 2, 128, 32, seed=63)
    b.q *= 3
    most = torch.finfo(b.q.dtype).max
    for sign in (1, -1):
        b.v[:] = sign * most
        assert torch.all(b.attend()[: sum(n)] == sign * most)
    b.v[:] = 0.75  # (and of another: half a unit in the last place, and the sums' own roundings, away at most)
    assert torch.all((b.attend()[: sum(n)].float() - 0.75).abs() <= torch.finfo(b.q.dtype).eps / 4)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("n", [1, 3, 30])
def test_weights_that_round_alike(hip, kind, n):
    """One key, and others whose weights are one number each time and round up or down together: the mean of the type's
    largest value is that value."""
    b = Batch(kind, [n], [32], 6, 2, 128, 32, seed=67)
    most = torch.finfo(b.q.dtype).max
    b.v[:], b.k[:], b.q[:] = most, 0, 0
    b.q[..., 0] = 1
    b.k[:, :, 0, 0] = 1
    for j in range(1, 400):
        assert torch.all(b.attend(scale=math.log(2) * (1 - j / 1000)) == most), j


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("ones,chunk", [(64, 300), (30, 150), (16, 700)])
def test_single_tokens_beside_a_chunk(hip, kind, ones, chunk):
    """One call, as a serving loop makes it: users' next tokens and a part of a new prompt, in tiles of the few rows' kernel
    (the first two) and of the many rows'."""
    r = torch.Generator().manual_seed(ones)
    lens = torch.randint(1, 900, (ones,), generator=r).tolist()
    n = [1] * (ones // 2) + [chunk] + [1] * (ones - ones // 2)
    lens[ones // 2: ones // 2] = [chunk + 250]
    b = Batch(kind, n, lens, 6, 2, 128, 32, seed=71, pad=1)
    first = b.check()
    assert torch.equal(b.attend(out=torch.full_like(b.q, 7.0)), first)
    b.check(cap=20.0, window=300)


@pytest.mark.gpu
def test_many_prompts_at_far_positions(hip):
    """Prompts whose key steps, counted whole beside a prefix, are more for each unit of work than a tile can have; a window
    leaves the last keys."""
    from spectra_amd import kernels as K
    g, page, d, kv, batch, n, window = _gen(73), 65536, 64, 8, 64, 5500, 300
    k, v = (torch.randn(3, kv, page, d, generator=g, device="cuda").half() for _ in range(2))
    table = (torch.arange(batch * 8193, device="cuda") % 3).int().view(batch, -1)
    lens = [(1 << 29) - 999 * b for b in range(batch)]
    q = torch.randn(batch * n, kv, d, generator=g, device="cuda", dtype=torch.float16)
    out = torch.full_like(q, 7.0)
    K.paged_attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                   torch.arange(0, batch * n + 1, n, dtype=torch.int32, device="cuda"), table, k, v, window=window,
                   prefix=torch.zeros(batch, dtype=torch.int32, device="cuda"), out=out)
    assert not torch.any((out == 7.0).all(-1)), "rows were left as they were"
    for b in (0, 31, 63):
        m = lens[b]
        for at in (0, 2741, n - 40):  # 40 rows
            i = torch.arange(m - n + at, m - n + at + 40, device="cuda")[:, None]
            j = torch.arange(int(i[0]) - window, int(i[-1]) + 1, device="cuda")[None]
            see = (i - j < window) & (j <= i)
            rows = table[b, j[0] // page].long(), slice(None), j[0] % page
            kk, vv = k[rows].double(), v[rows].double()
            for h in range(kv):
                qh = q[b * n + at: b * n + at + 40, h].double()
                delta = d * 2.0 ** -24 * (qh.abs() @ kk[:, h].abs().T / 8).amax(-1, keepdim=True)
                x = (qh @ kk[:, h].T / 8).masked_fill(~see, -math.inf)
                p = torch.softmax(x, -1)
                total = torch.exp(x - x.amax(-1, keepdim=True)).sum(-1, keepdim=True)
                want, a = p @ vv[:, h], p @ vv[:, h].abs()
                tol = 2.0 ** -11 * want.abs() + (2.0 ** -11 + 2 * delta + 2.0 ** -20) * a + \
                    2.0 ** -25 * (1 + (see.double() @ vv[:, h].abs()) / total)
                assert torch.all((out[b * n + at: b * n + at + 40, h].double() - want).abs() <= tol), (b, at, h)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_rows_without_keys(hip, kind):
    """More tokens than keys (positions below zero), and scores that are all -inf: zeros."""
    b = Batch(kind, [4, 2, 150], [2, 0, 100], 4, 2, 64, 16, seed=1)
    out = torch.full_like(b.q, 7.0)
    b.attend(out=out)
    assert torch.all(out[:2] == 0) and torch.all(out[4:6] == 0) and torch.all(out[6:56] == 0)
    assert torch.all(torch.isfinite(out)) and torch.all(out[2:4].abs().amax(-1) > 0)
    if kind == "fp16":
        b = Batch(kind, [1, 1], [20, 20], 4, 2, 64, 32, seed=1)
        b.k[:] = 60000.0
        b.q[0] = -60000.0  # every product is -inf in the scores' type times nothing: -2.3e11 each, finite and equal
        v = b.rows(0)[1].mean(1)
        got = b.attend()[0].double().view(2, 2, 64)
        assert torch.allclose(got, v[:, None].expand(2, 2, 64), atol=2e-3)
        b.k[:] = float("inf")
        b.q[0] = -1.0  # scores of -inf weigh nothing
        assert torch.all(b.attend()[0] == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("n,lens", [([1, 1], [40, 70]), ([4, 3], [40, 70]), ([40, 130], [40, 300])])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_stays_out(hip, kind, n, lens, what):
    """Values of the last token, and of keys before a window, that are not finite reach only the rows that see them."""
    b = Batch(kind, n, lens, 4, 2, 64, 16, seed=4)
    for s, m in enumerate(lens):
        page = b.table[s].long()
        b.v[page[(m - 1) // 16], :, (m - 1) % 16] = what
        b.v[page[0], :, 3] = what
        b.k[page[0], :, 4] = what
    for kw in (dict(window=30), dict(window=20, cap=5.0)):
        out = b.attend(**kw)
        keep = (b.k.clone(), b.v.clone())
        for s in range(len(n)):  # keys before every window of the call's tokens: cleaned, they change nothing
            if lens[s] - n[s] - 30 > 5:
                page = b.table[s].long()
                b.v[page[0], :, 3] = 0.0
                b.k[page[0], :, 4] = 0.0
        assert torch.equal(torch.isnan(out), torch.isnan(b.attend(**kw)))
        assert torch.equal(out.nan_to_num(5.0), b.attend(**kw).nan_to_num(5.0))
        b.k, b.v = keep
    out = b.attend(window=20)
    at = 0
    for s, (m, t) in enumerate(zip(lens, n)):
        pos = torch.arange(m - t, m, device="cuda")
        sees = (pos == m - 1) | (pos < 3 + 20) & (pos >= 3) | (pos < 4 + 20) & (pos >= 4)
        fine = torch.isfinite(out[at: at + t]).all(-1).all(-1)
        assert torch.all(fine[~sees]), "a row that sees only finite keys is not finite"
        assert not torch.any(fine[(pos == m - 1)])
        at += t
    # the rows that see only finite keys are those of the same batch without the others
    clean = Batch(kind, n, lens, 4, 2, 64, 16, seed=4)
    want, tol = clean.reference(window=20)
    at = 0
    for s, (m, t) in enumerate(zip(lens, n)):
        pos = torch.arange(m - t, m, device="cuda")
        far = (pos != m - 1) & (pos >= 4 + 20)
        x = (out[at: at + t].double() - want[at: at + t]).abs() <= tol[at: at + t]
        assert torch.all(x[far])
        at += t


def _least_us(f):
    f()
    least = math.inf
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        f()
        b.record()
        b.synchronize()
        least = min(least, 1e3 * a.elapsed_time(b))
    return least


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,lens", [([2500], [2500]), ([400, 300], [9000, 300]), ([5] * 9, [4000] * 9)])
@pytest.mark.parametrize("what", ["value", "values", "key", "page"])
def test_what_is_not_finite_costs_little(hip, kind, n, lens, what):
    """A value, all values, a key that are not finite, or a page that is missing, where every row sees it: no row is computed
    by itself for that, and the call takes about as long as with finite ones.  (One by one the prompt's rows took
    some hundred times as long.)"""
    b = Batch(kind, n, lens, 6, 2, 128, 16, seed=51)
    from spectra_amd import kernels as K
    ws = K.paged_attend_workspace(128)
    out = torch.empty_like(b.q)
    clean = _least_us(lambda: b.attend(workspace=ws, out=out))
    row, first = b.table[:, 0].long(), (slice(None), 3)
    if what == "page":
        b.table[:, 0] = -1
    else:
        x = (b.k if what == "key" else b.v)
        x = x[1] if kind == "4bit" else x
        x[(slice(None),) * 3 if what == "values" else (row, *first)] = float("nan")
    spoilt = _least_us(lambda: b.attend(workspace=ws, out=out))
    at = 0
    for t, m in zip(n, lens):
        pos = torch.arange(m - t, m, device="cuda")
        sees = pos >= (0 if what in ("values", "page") else 3)
        lost = torch.isnan(out[at: at + t]).all(-1).all(-1)
        assert torch.equal(lost, sees) and torch.all(torch.isfinite(out[at: at + t][~sees]))
        at += t
    assert spoilt < 4 * clean + 100, (clean, spoilt)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("n", [[1, 1], [3, 4], [40, 130]])
def test_infinite_values_where_every_score_is(hip, kind, n):
    """Rows that see only scores of -inf are zero, whatever the values are."""
    b = Batch(kind, n, [40, 300], 4, 2, 64, 16, seed=53)
    b.k[:] = float("inf")
    b.q[:] = -1.0
    for what in (float("inf"), float("nan")):
        b.v[:] = what
        assert torch.all(b.attend()[: sum(n)] == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kw", [dict(), dict(cap=5.0, slopes=True), dict(cap=1e4), dict(window=30, prefix=True)])
def test_rows_computed_by_themselves(hip, kind, d, kw):
    """One value of the last tokens that is not finite: the rows of its tile that do not see it are as without it."""
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = torch.exp2(-torch.arange(1, 7, device="cuda").float())
    if "prefix" in kw:
        kw["prefix"] = torch.tensor([10, 0, 60], dtype=torch.int32, device="cuda")
    b = Batch(kind, [4, 50, 140], [90, 77, 500], 6, 2, d, 16, seed=57)
    want, tol = b.reference(**kw)
    for s, (t, m) in enumerate(zip(b.n, b.lens)):
        x = b.v[1] if kind == "4bit" else b.v
        x[b.table[s, (m - 2) // 16].long(), :, (m - 2) % 16, 0] = float("inf")
    out, at = b.attend(**kw), 0
    for t, m in zip(b.n, b.lens):
        x, keep = out[at: at + t].double(), slice(0, t - 2)
        assert torch.all((x[keep] - want[at: at + t][keep]).abs() <= tol[at: at + t][keep])
        assert not torch.any(torch.isfinite(x[t - 2:]).all(-1))
        at += t


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 3, 100])
def test_pages_outside_the_pool(hip, kind, n):
    """A page id outside the pool, or a position past the table: NaN for the rows that see it, nobody else."""
    b = Batch(kind, [n, n], [200, 200], 4, 2, 64, 16, seed=6)
    fine = b.attend()
    for bad in (-1, 1 << 30, b.valid.shape[0]):
        keep = b.table[0, 11].clone()
        b.table[0, 11] = bad  # positions 176 .. 191
        out = b.attend()
        sees = torch.arange(200 - n, 200, device="cuda") >= 176
        assert torch.all(torch.isnan(out[:n][sees])) and torch.equal(out[:n][~sees], fine[:n][~sees])
        assert torch.equal(out[n:], fine[n:])
        assert torch.equal(b.attend(window=8)[n - 1], Batch(kind, [n, n], [200, 200], 4, 2, 64, 16, seed=6)
                           .attend(window=8)[n - 1])  # the last token's window is past it
        b.table[0, 11] = keep
    lens = b.kv_lens.clone()
    b.kv_lens[0] = 1 << 20  # far past the table
    out = b.attend()
    assert torch.all(torch.isnan(out[:n])) and torch.equal(out[n:], fine[n:])
    b.kv_lens.copy_(lens)
    assert torch.equal(b.attend(), fine)


# -- appending ------------------------------------------------------------------------------------
def _tables(rows, d):
    inv = 1.0 / (500000.0 ** (torch.arange(0, d, 2, dtype=torch.float32, device="cuda") / d))
    ang = torch.arange(rows, dtype=torch.float32, device="cuda")[:, None] * inv
    return ang.cos(), ang.sin()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,d,page", [(24, 8, 128, 16), (4, 4, 64, 64), (5, 1, 64, 32)])
@pytest.mark.parametrize("n,lens", [([1], [1]), ([1, 1, 0, 1], [17, 300, 5, 64]), ([70, 3, 0, 129], [70, 40, 9, 400])])
@pytest.mark.parametrize("turn", [True, False])
def test_append(hip, kind, heads, kv, d, page, n, lens, turn):
    from spectra_amd import kernels as K
    b = Batch(kind, n, lens, heads, kv, d, page, seed=2, pad=2, pages_apart=True)
    wide = b.rand(b.tokens, (heads + 2 * kv) * d + 16)
    qkv = wide[:, 8:-8]  # rows inside wider ones
    cos, sin = _tables(max(lens), d)
    before = [t.clone() for c in (b.k, b.v) for t in (c if kind == "4bit" else (c,))]
    q_out = torch.full((b.tokens, heads, d), 7.0, dtype=qkv.dtype, device="cuda")
    q = K.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, cos if turn else None, sin if turn else None, heads,
                            b.k, b.v, q_out=q_out)
    assert q is q_out and torch.all(q[sum(n):] == 7.0)
    after = [t for c in (b.k, b.v) for t in (c if kind == "4bit" else (c,))]
    # every row of the pool: the appended ones by the contiguous cache's kernels or in 64 bits, the rest as it was
    at = 0
    want = [t.clone() for t in before]
    u = torch.finfo(_DT[kind]).eps / 2
    for s, (t, m) in enumerate(zip(n, lens)):
        if t == 0:
            continue
        pos = torch.arange(m - t, m, device="cuda")
        x = qkv[at: at + t].double().view(t, heads + 2 * kv, d)
        c, sn = (y[pos].double()[:, None] for y in (cos, sin))
        lo, hi = x[:, :heads + kv].chunk(2, -1)
        rot = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1) if turn else x[:, :heads + kv]
        size = torch.cat([(lo * c).abs() + (hi * sn).abs(), (hi * c).abs() + (lo * sn).abs()], -1)
        # one rounding to 16 bits of a sum that fp32 holds to 3 roundings of its parts
        tol = u * rot.abs() + (1 + u) * 3 * 2.0 ** -24 * size + (2.0 ** -25 if kind != "bf16" else 0.0)
        assert torch.all((q[at: at + t].double() - rot[:, :heads]).abs() <= tol[:, :heads])
        ids, r = b.table[s][pos // page].long(), pos % page
        if kind == "bf16":
            got = after[0][ids, :, r].double()
            assert torch.all((got - rot[:, heads:]).abs() <= tol[:, heads:])
            want[0][ids, :, r] = after[0][ids, :, r]
            want[1][ids, :, r] = x[:, heads + kv:].to(torch.bfloat16)
        else:  # bit for bit what the contiguous cache gets
            ones, zeros = torch.ones(m, d // 2, device="cuda"), torch.zeros(m, d // 2, device="cuda")
            kc, vc = (torch.zeros(kv, m, d, dtype=torch.float16, device="cuda") for _ in range(2))
            qr = K.rope_append(qkv[at: at + t].contiguous(), pos, cos[:m].contiguous() if turn else ones,
                               sin[:m].contiguous() if turn else zeros, heads, kv, kc, vc)
            assert torch.equal(qr, q[at: at + t])
            new = [kc[:, m - t:], vc[:, m - t:]]
            if kind == "4bit":
                new = [y for c4 in new for y in K.kv4_quantize(c4.contiguous())]
            for w, y in zip(want, new):
                w[ids, :, r] = y.transpose(0, 1)
        at += t
    for w, a in zip(want, after):
        assert torch.equal(w.view(torch.uint8) if w.is_floating_point() else w, a.contiguous().view(torch.uint8)
                           if a.is_floating_point() else a)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_append_outside(hip, kind):
    """Tokens without a row to write: page ids outside the pool, positions past the block table, past the rope table
    (NaN queries) or below zero.  Nothing is written for them; the others go on."""
    from spectra_amd import kernels as K
    heads, kv, d = 4, 2, 64
    b = Batch(kind, [3, 4, 2, 2, 5], [20, 40, 64, 30, 3], heads, kv, d, 16, seed=8)
    qkv = b.rand(b.tokens, (heads + 2 * kv) * d)
    cos, sin = _tables(48, d)
    b.table[0, 1] = -5                     # positions 16 .. 19: sequence 0's tokens are 17 .. 19
    b.table[1, 2] = b.valid.shape[0]       # positions 32 .. 47: sequence 1's tokens are 36 .. 39
    parts = lambda: [t for c in (b.k, b.v) for t in (c if kind == "4bit" else (c,))]  # noqa: E731
    before = [t.clone() for t in parts()]
    b.kv_lens[2] = 64                      # positions 62, 63: past the rope table of 48
    q = K.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, cos, sin, heads, b.k, b.v)
    assert torch.all(torch.isfinite(q[:7])) and torch.all(torch.isnan(q[7:9])) and torch.all(torch.isnan(q[11:13]))
    assert torch.all(torch.isfinite(q[9:11])) and torch.all(torch.isfinite(q[13:]))
    changed = torch.zeros_like(b.valid)
    for x, y in zip(before, parts()):
        same = x.view(torch.uint8) == y.contiguous().view(torch.uint8)
        changed |= ~same.all(-1).all(1)
    want = torch.zeros_like(b.valid)
    want[b.table[3, 1].long(), 28 - 16: 30 - 16] = True
    want[b.table[4, 0].long(), 0:3] = True
    assert torch.equal(changed, want)
    b.kv_lens[3] = 1 << 20                 # past the block table, no rotation: no row either
    before = [t.clone() for t in parts()]
    K.paged_rope_append(qkv[9:11], b.kv_lens[3:4], torch.tensor([0, 2], dtype=torch.int32, device="cuda"), b.table[3:4],
                        None, None, heads, b.k, b.v)
    for x, y in zip(before, parts()):
        assert torch.equal(x.view(torch.uint8), y.contiguous().view(torch.uint8))


# -- together, as a serving loop uses them --------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_generation_together(hip, kind):
    """Prompts in two chunks, then captured single-token steps whose lengths advance on the device: every step against
    attention in 64 bits over all that was appended, and against the same step run eagerly."""
    from spectra_amd import kernels as K
    heads, kv, d, page, steps = 6, 2, 64, 16, 5
    n0 = [50, 3, 131]
    batch, most = len(n0), 160
    b = Batch(kind, n0, [most] * batch, heads, kv, d, page, seed=11)
    cos, sin = _tables(most, d)
    ws = K.paged_attend_workspace(d)
    hist = [[] for _ in n0]  # per sequence: (k rotated, v) rows as stored, 64 bits

    def note(qkv, n, lens):
        at = 0
        for s, (t, m) in enumerate(zip(n, lens)):
            ids, pos = b.table[s], torch.arange(m - t, m, device="cuda")
            rows = [_values(tuple(y[ids[pos // page].long(), :, pos % page] for y in c) if kind == "4bit"
                            else c[ids[pos // page].long(), :, pos % page], kind) for c in (b.k, b.v)]
            hist[s].append(rows)
            x = qkv[at: at + t].double().view(t, -1, d)[:, heads + kv:]
            # v as stored: itself, or within half a step of its group (a scale of range / 15, and fp16's roundings)
            step = (x.unflatten(-1, (-1, 32)).amax(-1) - x.unflatten(-1, (-1, 32)).amin(-1)) / 15
            bound = (0.51 * step.repeat_interleave(32, -1) + 2.0 ** -9) if kind == "4bit" else 0.0
            assert torch.all((rows[1] - x).abs() <= bound + (0.5 * step.repeat_interleave(32, -1) if kind == "4bit" else 0))
            at += t

    def want(q, n):
        outs, at = [], 0
        for s, t in enumerate(n):
            k, v = (torch.cat([r[i] for r in hist[s]]) for i in (0, 1))  # [len, kv, d]
            m = k.shape[0]
            see = torch.arange(m, device="cuda")[None] <= torch.arange(m - t, m, device="cuda")[:, None]
            g = heads // kv
            x = torch.einsum("thd,mhd->htm", q[at: at + t].double(), k.repeat_interleave(g, 1)) / math.sqrt(d)
            p = torch.softmax(x.masked_fill(~see, -math.inf), -1)
            outs.append(torch.einsum("htm,mhd->thd", p, v.repeat_interleave(g, 1)))
            at += t
        return torch.cat(outs)

    u = torch.finfo(_DT[kind]).eps / 2

    def step(qkv, lens, starts):
        q = K.paged_rope_append(qkv, lens, starts, b.table, cos, sin, heads, b.k, b.v)
        return q, K.paged_attend(q, lens, starts, b.table, b.k, b.v, workspace=ws)

    def close(got, q, n):
        y = want(q, n)
        # values of deviation 1: an output's own rounding, and the weights' against a sum of weight times |value| <= 6
        assert torch.all((got.double() - y).abs() <= u * y.abs() + (u + 2.0 ** -12) * 6)

    lens = [0] * batch
    for chunk in ([20, 1, 100], [30, 2, 31]):
        lens = [m + t for m, t in zip(lens, chunk)]
        starts = torch.tensor([0] + torch.tensor(chunk).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        qkv = b.rand(sum(chunk), (heads + 2 * kv) * d)
        q, o = step(qkv, torch.tensor(lens, dtype=torch.int32, device="cuda"), starts)
        note(qkv, chunk, lens)
        close(o, q, chunk)
    ones = torch.arange(batch + 1, dtype=torch.int32, device="cuda")
    dev_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qkv = b.rand(batch, (heads + 2 * kv) * d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(qkv, dev_lens + 1, ones)  # warm-up; the capture's first replay writes the same rows again
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dev_lens += 1
        q, o = step(qkv, dev_lens, ones)
    for i in range(steps):
        qkv.copy_(b.rand(batch, (heads + 2 * kv) * d))
        graph.replay()
        torch.cuda.synchronize()
        lens = [m + 1 for m in lens]
        assert dev_lens.tolist() == lens
        note(qkv, [1] * batch, lens)
        close(o, q, [1] * batch)
        eq, eo = step(qkv, dev_lens, ones)  # eager, between the replays
        assert torch.equal(eq, q) and torch.equal(eo, o)


@pytest.mark.gpu
def test_against_the_contiguous_kernels(hip):
    """One sequence: within the two kernels' roundings of attend_decode and attend_prefill on a contiguous cache."""
    from spectra_amd import kernels as K
    heads, kv, d, m = 24, 8, 128, 777
    b = Batch("fp16", [m], [m], heads, kv, d, 64, seed=12)
    k, v = (x.half().contiguous() for x in b.rows(0))
    old = K.attend_prefill(b.q, torch.arange(m, device="cuda"), m, k, v)
    _, tol = b.reference()
    assert torch.all((b.attend().double() - old.double()).abs() <= 2 * tol)
    one = Batch("fp16", [1], [m], heads, kv, d, 64, seed=12)
    kk, vv = (x.half().contiguous() for x in one.rows(0))
    qkv = torch.cat([one.q.reshape(-1), kk[:, -1].reshape(-1), vv[:, -1].reshape(-1)])
    old = K.attend_decode(qkv, torch.tensor([m - 1], device="cuda"), None, None, heads, kv, kk, vv)
    _, tol = one.reference()
    assert torch.all((one.attend()[0].double() - old.double()).abs() <= 2 * tol[0])


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,d,m", [(24, 8, 128, 700), (8, 2, 64, 90)])
def test_against_the_contiguous_4bit_cache(hip, heads, kv, d, m):
    """The same codes in the contiguous 4-bit cache stand for bf16 values there, and for fp16 ones on pages: the two differ
    by that rounding and their kernels', no more."""
    from spectra_amd import kernels as K
    w, page = 16, 64
    b = Batch("4bit", [1], [m], heads, kv, d, page, seed=61)
    g = _gen(62)
    # the newest rows, which the contiguous cache takes from qkv: exact in 4 bits (every group holds codes 0 and 15)
    code = torch.randint(0, 16, (2, kv, d // 32, 32), generator=g, device="cuda")
    code[..., 0], code[..., 1] = 0, 15
    new = ((code - 6) * 0.125).half().view(2, kv, d)
    at = (int(b.table[0, (m - 1) // page]), slice(None), (m - 1) % page)
    for c, x in zip((b.k, b.v), new):
        for t, y in zip(c, K.kv4_quantize(x.view(kv, 1, d).contiguous())):
            t[at] = y.view(kv, -1)
    ids = b.table[0, : -(-m // page)].long()
    codes = [tuple(t[ids].transpose(0, 1).reshape(kv, -1, t.shape[-1])[:, :m].contiguous() for t in c) for c in (b.k, b.v)]
    rows = b.rows(0)
    ring = [torch.zeros(kv, w, d, dtype=torch.float16, device="cuda") for _ in rows]  # the window: the same values
    last = torch.arange(m - w, m, device="cuda")
    for r, x in zip(ring, rows):
        r[:, last % w] = x[:, last].half()
    one, zero = torch.ones(m, d // 2, device="cuda"), torch.zeros(m, d // 2, device="cuda")
    qkv = torch.cat([b.q.reshape(-1), new.reshape(-1)])
    old = K.attend_decode_q4(qkv, torch.tensor([m - 1], device="cuda"), one, zero, heads, kv, *ring, *codes)
    want, tol = b.reference()
    u, g = 2.0 ** -8 + 2.0 ** -11, heads // kv
    k, v = (x.repeat_interleave(g, 0) for x in rows)
    size = (b.q[0].double().abs()[:, None] @ k.abs().transpose(1, 2)).squeeze(1) / math.sqrt(d)
    p = torch.softmax((b.q[0].double()[:, None] @ k.transpose(1, 2)).squeeze(1) / math.sqrt(d), -1)
    a = (p[:, None] @ v.abs()).squeeze(1)
    assert torch.all((old.double() - b.attend()[0].double()).abs() <= 2 * tol[0] + u * (1 + 2 * size.amax(-1, keepdim=True)) * a)


@pytest.mark.gpu
def test_strided_queries_and_streams(hip):
    """Queries inside wider rows, and calls on another stream than the current default, with a workspace each."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [1, 1, 1, 1], [100, 3000, 64, 7], 8, 2, 64, 32, seed=13)
    want = b.attend()
    wide = torch.randn(4, 12, 64, device="cuda").half()
    wide[:, 2:10] = b.q
    b.q = wide[:, 2:10]
    assert torch.equal(b.attend(), want)
    odd = torch.zeros(4 * 8 * 64 + 4, dtype=torch.float16, device="cuda")[4:].view(4, 8, 64)
    odd.copy_(wide[:, 2:10])
    b.q = odd  # 8-byte aligned: copied
    assert torch.equal(b.attend(), want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [K.paged_attend_workspace(64) for _ in streams]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s, ws in zip(streams, spaces):
            with torch.cuda.stream(s):
                outs.append(b.attend(workspace=ws))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.gpu
def test_empty_calls(hip):
    from spectra_amd import kernels as K
    b = Batch("fp16", [0, 0], [5, 9], 4, 2, 64, 16, seed=14)
    assert b.attend().shape == (0, 4, 64)
    q = K.paged_rope_append(torch.empty(0, 8 * 64, dtype=torch.float16, device="cuda"), b.kv_lens, b.q_start, b.table,
                            None, None, 4, b.k, b.v)
    assert q.shape == (0, 4, 64)
    b = Batch("fp16", [0, 0], [5, 9], 4, 2, 64, 16, seed=14, pad=3)  # tokens, none of a sequence
    out = torch.full_like(b.q, 7.0)
    assert torch.all(b.attend(out=out) == 7.0)
    b = Batch("4bit", [0, 0], [5, 9], 4, 2, 64, 16, seed=14, pad=200)  # the same for the prompts' tiles
    out = torch.full_like(b.q, 7.0)
    assert torch.all(b.attend(out=out) == 7.0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_captured_with_a_workspace_of_its_own(hip, n):
    """No workspace given: the call's own, also in a graph, whose replays follow the lengths."""
    b = Batch("fp16", [n, n], [3000, 700], 4, 2, 64, 16, seed=17)
    lens = b.kv_lens.clone()
    b.attend()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.attend()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.attend()
    for step in range(4):
        b.kv_lens.copy_(lens - 100 * step)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, b.attend())


@pytest.mark.gpu
def test_refusals(hip):
    from spectra_amd import kernels as K
    b = Batch("fp16", [2, 1], [40, 20], 4, 2, 64, 16, seed=15)
    good = dict(q=b.q, kv_lens=b.kv_lens, q_start=b.q_start, block_table=b.table, k_pages=b.k, v_pages=b.v)

    def bad(match, **kw):
        with pytest.raises(ValueError, match=match):
            K.paged_attend(**{**good, **kw})

    bad("fp16", q=b.q.float())
    bad("pages of head size", q=b.q.bfloat16())
    bad("q has head size", q=b.q[..., :32].contiguous())
    bad("multiple", q=b.q[:, :3])
    bad("kv_lens", kv_lens=b.kv_lens.long())
    bad("q_start", q_start=b.q_start.float())
    bad("block_table", block_table=b.table.t())
    bad("sequences need", q_start=b.q_start[:2])
    bad("pages of head size", v_pages=b.v[:-1])
    bad("contiguous", k_pages=b.k.transpose(1, 2).contiguous().transpose(1, 2))
    bad("k_pages and v_pages", k_pages=(b.k, b.k), v_pages=(b.v, b.v))
    bad("power of two", k_pages=b.k[:, :, :8].contiguous(), v_pages=b.v[:, :, :8].contiguous())
    bad("slopes", slopes=torch.ones(3, device="cuda"))
    bad("prefix", prefix=torch.ones(2, device="cuda"))
    bad("cap", cap=-1.0)
    bad("cap", cap=float("nan"))
    bad("scale", scale=0.0)
    bad("window", window=-1)
    bad("out", out=torch.empty(2, 4, 64, dtype=torch.float16, device="cuda"))
    with pytest.raises(L.SpectraError) as e:
        K.paged_attend(**good, workspace=torch.zeros(1024, dtype=torch.uint8, device="cuda"))
    assert e.value.status == L.ERR_WORKSPACE
    with pytest.raises(ValueError, match="head sizes"):
        K.paged_attend_workspace(96)
    with pytest.raises(L.SpectraError) as e:
        c = Batch("fp16", [1], [4], 2, 2, 32, 16, seed=15)
        K.paged_attend(c.q, c.kv_lens, c.q_start, c.table, c.k, c.v, workspace=K.paged_attend_workspace(64))
    assert e.value.status == L.ERR_UNSUPPORTED
    rows = torch.zeros(3, 8 * 64, dtype=torch.float16, device="cuda")
    args = [rows, b.kv_lens, b.q_start, b.table, None, None, 4, b.k, b.v]

    def bad_append(match, at, value):
        with pytest.raises(ValueError, match=match):
            K.paged_rope_append(*[value if i == at else x for i, x in enumerate(args)])

    bad_append("rows must hold", 0, rows[:, :-8])
    bad_append("fp16", 0, rows.float())
    bad_append("both", 4, torch.ones(40, 32, device="cuda"))
    bad_append("multiple", 6, 3)
    with pytest.raises(ValueError, match="cos"):
        K.paged_rope_append(*args[:4], torch.ones(40, 16, device="cuda"), torch.ones(40, 16, device="cuda"), *args[6:])


@pytest.mark.gpu
def test_rope_tables_without_rows(hip):
    """Not the same as no tables: no position has an angle."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [1], [4], 2, 2, 64, 16, seed=15)
    none = torch.empty(0, 32, device="cuda")
    with pytest.raises(ValueError, match="at least a row"):
        K.paged_rope_append(torch.zeros(1, 6 * 64, dtype=torch.float16, device="cuda"), b.kv_lens, b.q_start, b.table, none, none, 2,
                            b.k, b.v)


# -- the C entries' refusals, without a GPU -------------------------------------------------------
def _desc(**kw):
    p = L.PagedKv()
    p.kind, p.kv_heads, p.head_dim, p.page_size, p.num_pages = L.KV_F16, 2, 64, 16, 10
    p.k, p.v, p.page_stride = 0x10000, 0x20000, 2 * 16 * 64
    p.batch, p.table_width, p.table_stride = 3, 4, 4
    p.block_table, p.kv_lens, p.q_start = 0x30000, 0x31000, 0x32000
    for k, v in kw.items():
        setattr(p, k, v)
    return p


_BAD = [(dict(kind=3), "kind"), (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=3), "multiple"), (dict(head_dim=96), "64 or 128"),
        (dict(page_size=8), "power of two"), (dict(page_size=48), "power of two"), (dict(num_pages=0), "num_pages"),
        (dict(batch=0), "batch"), (dict(table_width=0), "table"), (dict(table_stride=3), "stride"), (dict(k=None), "NULL"),
        (dict(kv_lens=None), "NULL"), (dict(page_stride=100), "page stride"), (dict(k=0x10008), "16-byte"),
        (dict(page_stride=2 * 16 * 64 + 4), "16-byte"), (dict(kind=L.KV_4BIT), "scales"),
        (dict(table_width=1 << 28, table_stride=1 << 28), "positions")]


@pytest.mark.parametrize("bad,msg", _BAD)
def test_descriptor_refusals(bad, msg):
    lib = L.load()
    p = _desc(**bad)
    st = lib.spectra_paged_rope_append(ctypes.byref(p), 0x40000, 8 * 64, 5, None, None, 0, 4, 0x50000, None)
    assert st in (L.ERR_INVALID, L.ERR_UNSUPPORTED) and msg in lib.spectra_last_error().decode()
    st = lib.spectra_paged_attend(ctypes.byref(p), 0x40000, 4 * 64, 5, 4, 0.125, 0.0, 0, None, None, 0x60000, 1 << 40,
                                  0x50000, None)
    assert st in (L.ERR_INVALID, L.ERR_UNSUPPORTED) and msg in lib.spectra_last_error().decode()


@pytest.mark.parametrize("bad,heads,msg", [(dict(block_table=0x30002), 4, "aligned"), (dict(kv_lens=0x31001), 4, "aligned"),
                                           (dict(q_start=0x32002), 4, "aligned"), (dict(kv_heads=1), 1 << 25, "range")])
def test_descriptor_refusals_of_addresses_and_heads(bad, heads, msg):
    """Integers that lie across words, which scalar loads would read elsewhere, and heads past 32-bit offsets of a row."""
    lib = L.load()
    p = _desc(**bad)
    st = lib.spectra_paged_rope_append(ctypes.byref(p), 0x40000, (1 << 26) * 64, 5, None, None, 0, heads, 0x50000, None)
    assert st == L.ERR_INVALID and msg in lib.spectra_last_error().decode()
    st = lib.spectra_paged_attend(ctypes.byref(p), 0x40000, (1 << 26) * 64, 5, heads, 0.125, 0.0, 0, None, None, 0x60000, 1 << 40,
                                  0x50000, None)
    assert st == L.ERR_INVALID and msg in lib.spectra_last_error().decode()


@pytest.mark.parametrize("change,status,msg", [
    (dict(q=None), L.ERR_INVALID, "NULL"), (dict(q=0x40008), L.ERR_INVALID, "16-byte"), (dict(ldq=100), L.ERR_INVALID, "stride"),
    (dict(ldq=4 * 64 + 4), L.ERR_INVALID, "stride"), (dict(tokens=0), L.ERR_INVALID, "tokens"),
    (dict(tokens=1 << 31), L.ERR_INVALID, "tokens"), (dict(scale=float("nan")), L.ERR_INVALID, "scale"),
    (dict(cap=float("inf")), L.ERR_INVALID, "cap"), (dict(window=-3), L.ERR_INVALID, "window"),
    (dict(ws=None), L.ERR_WORKSPACE, "workspace"), (dict(size=1 << 20), L.ERR_WORKSPACE, "workspace"),
    (dict(ws=0x60008), L.ERR_INVALID, "workspace"), (dict(q=0x50000), L.ERR_INVALID, "overlap"),
    (dict(q=0x50000 - 16), L.ERR_INVALID, "overlap"), (dict(q=0x50000 + 5 * 4 * 64 * 2 - 16), L.ERR_INVALID, "overlap")])
def test_attend_refusals(change, status, msg):
    lib = L.load()
    a = dict(q=0x40000, ldq=4 * 64, tokens=5, scale=0.125, cap=0.0, window=0, ws=0x60000, size=1 << 40)
    a.update(change)
    p = _desc()
    st = lib.spectra_paged_attend(ctypes.byref(p), a["q"], a["ldq"], a["tokens"], 4, a["scale"], a["cap"], a["window"],
                                  None, None, a["ws"], a["size"], 0x50000, None)
    assert st == status and msg in lib.spectra_last_error().decode()


@pytest.mark.parametrize("change,msg", [
    (dict(qkv=None), "NULL"), (dict(ld=8 * 64 - 8), "stride"), (dict(ld=8 * 64 + 4), "16-byte"), (dict(cos=0x70000), "both"),
    (dict(cos=0x70000, sin=0x80000, rows=0), "rope_rows"), (dict(cos=0x70004, sin=0x80000, rows=9), "16-byte"),
    (dict(tokens=0), "tokens"), (dict(qkv=0x50000), "overlap")])
def test_append_refusals(change, msg):
    lib = L.load()
    a = dict(qkv=0x40000, ld=8 * 64, tokens=5, cos=None, sin=None, rows=0)
    a.update(change)
    p = _desc()
    st = lib.spectra_paged_rope_append(ctypes.byref(p), a["qkv"], a["ld"], a["tokens"], a["cos"], a["sin"], a["rows"], 4,
                                       0x50000, None)
    assert st == L.ERR_INVALID and msg in lib.spectra_last_error().decode()


_POOL = 10 * 2 * 16 * 64 * 2  # bytes of the descriptor's pools


def _desc4(**kw):
    """4-bit pages, all operands apart."""
    d = dict(kind=L.KV_4BIT, page_stride=2 * 16 * 32, k_scales=0x90000, v_scales=0x94000, k_zeros=0x98000, v_zeros=0x9c000,
             scale_stride=2 * 16 * 2, zero_stride=2 * 16 * 2)
    return _desc(**{**d, **kw})


@pytest.mark.parametrize("what", ["k", "v", "k end", "table", "lens", "starts", "workspace", "slopes", "prefix", "4-bit scales",
                                  "4-bit zeros", "workspace on k", "workspace on q", "workspace on lens"])
def test_attend_refuses_outputs_in_other_operands(what):
    lib, p, out, ws, sl, pre, q = L.load(), _desc(), 0x50000, 0x100000, None, None, 0x40000
    if what.startswith("4-bit"):
        p = _desc4()
        out = 0x94000 + 9 * 2 * 16 * 2 * 2 if "scales" in what else 0x9c000
    elif what in ("k", "v", "k end"):
        out = {"k": 0x10000, "v": 0x20000 + _POOL - 16, "k end": 0x10000 - 5 * 4 * 64 * 2 + 16}[what]
    elif what in ("table", "lens", "starts"):
        setattr(p, {"table": "block_table", "lens": "kv_lens", "starts": "q_start"}[what], out + 64)
    elif what == "workspace":
        out = ws + 4096
    elif what == "slopes":
        sl = out + 16
    elif what == "prefix":
        pre = out + 5 * 4 * 64 * 2 - 4
    else:
        ws = {"workspace on k": 0x10000 - 4096, "workspace on q": 0x40000, "workspace on lens": 0x31000 - 4096}[what]
    st = lib.spectra_paged_attend(ctypes.byref(p), q, 4 * 64, 5, 4, 0.125, 0.0, 0, sl, pre, ws, 1 << 40, out, None)
    assert st == L.ERR_INVALID and "must not overlap" in lib.spectra_last_error().decode()


@pytest.mark.parametrize("what", ["q on k", "q on v", "q on cos", "q on table", "k on v", "k on qkv", "v on lens", "k on sin",
                                  "k on scales", "scales on zeros", "zeros on keys' zeros", "strides"])
def test_append_refuses_operands_that_it_writes_twice(what):
    lib, p, q, qkv, cos, sin = L.load(), _desc4() if "scales" in what or "zeros" in what else _desc(), 0x50000, 0x40000, 0x70000, 0x80000
    if what == "q on k":
        q = 0x10000 + _POOL - 16
    elif what == "q on v":
        q = 0x20000 - 16
    elif what == "q on cos":
        q = cos + 9 * 32 * 4 - 16
    elif what == "q on table":
        p.block_table = q
    elif what == "k on v":
        p.v = p.k
    elif what == "k on qkv":
        qkv = 0x10000 + 32
    elif what == "v on lens":
        p.kv_lens = 0x20000 + 12
    elif what == "k on sin":
        sin = 0x10000 + _POOL - 16
    elif what == "k on scales":
        p.k_scales = 0x10000 + 16
    elif what == "scales on zeros":
        p.v_zeros = p.k_scales + 32
    elif what == "zeros on keys' zeros":
        p.v_zeros = p.k_zeros
    else:  # 4-bit scales between the codes' pages, but farther apart: the second lies in a page
        p = _desc4(page_stride=2 * 16 * 32 + 128, k_scales=0x10000 + 2 * 16 * 32, scale_stride=2 * 16 * 2 + 576)
    st = lib.spectra_paged_rope_append(ctypes.byref(p), qkv, 8 * 64, 5, cos, sin, 9, 4, q, None)
    assert st == L.ERR_INVALID and "must not overlap" in lib.spectra_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [[1, 1], [40, 70]])
def test_pools_among_each_other(hip, kind, n):
    """Keys and values (and scales and zero points) of a page beside each other in one allocation, the outputs between
    the last ones: apart, and the same results."""
    from spectra_amd import kernels as K
    b = Batch(kind, n, [90, 75], 4, 2, 64, 16, seed=43)
    parts = [t for c in zip(b.k, b.v) for t in c] if kind == "4bit" else [b.k, b.v]
    sizes = [t[0].numel() * t.element_size() for t in parts]
    pages, rest = parts[0].shape[0], b.q.numel() * 2
    step = sum(sizes) + 64
    room = torch.zeros(pages * step + 2 * rest, dtype=torch.uint8, device="cuda")
    views, at = [], 0
    for t, size in zip(parts, sizes):
        x = room[at:].view(t.dtype).as_strided(t.shape, (step // t.element_size(),) + t.stride()[1:])
        x.copy_(t)
        views.append(x)
        at += size
    ends = [room[pages * step + i * rest:][:rest].view(b.q.dtype).view(b.q.shape) for i in (0, 1)]
    qkv = b.rand(b.tokens, 8 * 64)
    near = K.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, None, None, 4, b.k, b.v)
    want = b.attend()
    c = (tuple(views[0::2]), tuple(views[1::2])) if kind == "4bit" else views
    q = K.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, None, None, 4, *c, q_out=ends[0])
    assert torch.equal(q, near)
    assert torch.equal(K.paged_attend(b.q, b.kv_lens, b.q_start, b.table, *c, out=ends[1]), want)


@pytest.mark.parametrize("scale,cap", [(3e38, 0.0), (1.0, 1e-38), (1.0, 3e38), (0.0, 0.0)])
def test_scales_out_of_range(scale, cap):
    lib, p = L.load(), _desc()
    st = lib.spectra_paged_attend(ctypes.byref(p), 0x40000, 4 * 64, 5, 4, scale, cap, 0, None, None, 0x60000, 1 << 40, 0x50000,
                                  None)
    assert st == L.ERR_INVALID and "scale" in lib.spectra_last_error().decode()


def test_descriptor_layout_matches_c(tmp_path):
    import os
    import subprocess
    fields = [f[0] for f in L.PagedKv._fields_]
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "spectra_hip.h"\nint main(void){\n'
    src += 'printf("%zu %d\\n", sizeof(spectra_paged_kv_t), SPECTRA_PAGED_COUNTER_BYTES);\n'
    for f in fields:
        src += f'printf("%zu\\n", offsetof(spectra_paged_kv_t, {f}));\n'
    c, exe = tmp_path / "layout.c", tmp_path / "layout"
    c.write_text(src + "return 0;}\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(c), "-o", str(exe)], check=True)
    v = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert v[:2] == [ctypes.sizeof(L.PagedKv), L.PAGED_COUNTER_BYTES]
    for f, off in zip(fields, v[2:]):
        assert getattr(L.PagedKv, f).offset == off, f


def test_wrapper_refuses_host_tensors():
    from spectra_amd import kernels as K
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    one = torch.ones(1, dtype=torch.int32)
    pages = torch.zeros(2, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        K.paged_attend(q, one, torch.tensor([0, 1], dtype=torch.int32), one[:, None], pages, pages)
    with pytest.raises(ValueError, match="GPU"):
        K.paged_rope_append(torch.zeros(1, 8 * 64, dtype=torch.float16), one, torch.tensor([0, 1], dtype=torch.int32),
                            one[:, None], None, None, 4, pages, pages)


@pytest.mark.gpu
def test_registered_operators(hip):
    """The registered operators give what the functions give, and a whole-graph compilation traces them."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [1, 3], [70, 33], 4, 2, 64, 16, seed=16)
    ops = L.load_torch_ops()
    ws = K.paged_attend_workspace(64)
    args = (b.q, b.kv_lens, b.q_start, b.table, [b.k], [b.v], 0.125, 2.0, 20, None, None, ws)
    want = b.attend(cap=2.0, window=20)
    assert torch.equal(ops.paged_attend(*args), want)
    out = torch.empty_like(want)
    ops.paged_attend_out(*args, out)
    assert torch.equal(out, want)
    qkv = b.rand(b.tokens, 8 * 64)
    cos, sin = _tables(80, 64)
    q = K.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, cos, sin, 4, b.k, b.v)
    rows = (b.k.clone(), b.v.clone())
    assert torch.equal(ops.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, cos, sin, 4, [b.k], [b.v]), q)
    into = torch.empty_like(q)
    ops.paged_rope_append_out(qkv, b.kv_lens, b.q_start, b.table, cos, sin, 4, [b.k], [b.v], into)
    assert torch.equal(into, q) and all(torch.equal(x.view(torch.int16), y.contiguous().view(torch.int16))
                                        for x, y in zip(rows, (b.k, b.v)))

    def step(qkv, k, v):
        q = ops.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, cos, sin, 4, [k], [v])
        return ops.paged_attend(q, b.kv_lens, b.q_start, b.table, [k], [v], 0.125, 0.0, 0, None, None, ws)

    eager = step(qkv, b.k, b.v)
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    assert torch.equal(compiled(qkv, b.k, b.v), eager)

    def functions(qkv, k, v):
        q = K.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, cos, sin, 4, k, v)
        return K.paged_attend(q, b.kv_lens, b.q_start, b.table, k, v, workspace=ws)

    assert torch.equal(torch.compile(functions, backend="aot_eager", fullgraph=True)(qkv, b.k, b.v), eager)


@pytest.mark.gpu
def test_operands_that_gradients_are_asked_of(hip):
    """There is no derivative: the results are the registered operators', which say so when one is asked for."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [1, 3], [70, 33], 4, 2, 64, 16, seed=16)
    ws, want = K.paged_attend_workspace(64), b.attend()
    qkv = b.rand(b.tokens, 8 * 64)
    batch = b.kv_lens, b.q_start, b.table
    rows = K.paged_rope_append(qkv, *batch, None, None, 4, b.k, b.v)
    want = b.attend()
    q = b.q.clone().requires_grad_()
    got = [K.paged_attend(q, *batch, b.k, b.v, workspace=ws), K.paged_attend(b.q, *batch, b.k, b.v.clone().requires_grad_()),
           K.paged_attend(b.q, *batch, b.k, b.v, slopes=torch.zeros(4, device="cuda", requires_grad=True))]
    for o in got:
        assert o.requires_grad and torch.equal(o, want)
        with pytest.warns(UserWarning, match="autograd kernel was not registered"):
            o.sum().backward()
    r = K.paged_rope_append(qkv.clone().requires_grad_(), *batch, None, None, 4, b.k, b.v)
    assert r.requires_grad and torch.equal(r, rows)
    with torch.no_grad():
        assert not K.paged_attend(q, *batch, b.k, b.v, workspace=ws).requires_grad
    # a negated view of one number, which only the dispatcher would resolve
    one = Batch("fp16", [1], [40], 1, 1, 64, 16, seed=17)
    slope = torch.complex(torch.zeros(1), torch.full((1,), -0.25)).cuda().conj().imag
    assert slope.is_neg() and torch.equal(one.attend(slopes=slope), one.attend(slopes=torch.full((1,), 0.25, device="cuda")))


def test_registered_operators_have_shapes():
    """The operators' Meta kernels (what a compiler traces with)."""
    ops = L.load_torch_ops()
    m = dict(device="meta")
    q = torch.empty(5, 4, 64, dtype=torch.float16, **m)
    i32 = lambda *s: torch.empty(*s, dtype=torch.int32, **m)  # noqa: E731
    pages = [torch.empty(3, 2, 16, 64, dtype=torch.float16, **m)]
    o = ops.paged_attend(q, i32(2), i32(3), i32(2, 4), pages, pages, 0.1, 0.0, 0, None, None, None)
    assert o.shape == q.shape and o.dtype == q.dtype
    q4 = [torch.empty(3, 2, 16, 32, dtype=torch.uint8, **m), torch.empty(3, 2, 16, 2, dtype=torch.float16, **m),
          torch.empty(3, 2, 16, 2, dtype=torch.uint8, **m)]
    for p in (pages, q4):
        r = ops.paged_rope_append(torch.empty(5, 8 * 64, dtype=torch.float16, **m), i32(2), i32(3), i32(2, 4), None, None, 4, p, p)
        assert r.shape == (5, 4, 64)


@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("what", ["none", "two", "values"])
def test_registered_operators_refuse_other_lists(out, what):
    """Lists of no pages, or of neither one tensor nor three, without memory: an error, also for a tracing compiler."""
    ops = L.load_torch_ops()
    m = dict(device="meta")
    i32 = lambda *s: torch.empty(*s, dtype=torch.int32, **m)  # noqa: E731
    p = torch.empty(3, 2, 16, 64, dtype=torch.float16, **m)
    k, v = {"none": ([], []), "two": ([p, p], [p, p]), "values": ([p], [])}[what]
    q, qkv = torch.empty(5, 4, 64, dtype=torch.float16, **m), torch.empty(5, 8 * 64, dtype=torch.float16, **m)
    append = (qkv, i32(2), i32(3), i32(2, 4), None, None, 4, k, v)
    attend = (q, i32(2), i32(3), i32(2, 4), k, v, 0.1, 0.0, 0, None, None, None)
    with pytest.raises(ValueError, match="k_pages"):
        ops.paged_rope_append_out(*append, q) if out else ops.paged_rope_append(*append)
    with pytest.raises(ValueError, match="k_pages"):
        ops.paged_attend_out(*attend, q) if out else ops.paged_attend(*attend)
