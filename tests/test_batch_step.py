"""What a served batch's step adds to the paged cache: appending with rotary positions of several axes, bounds of the
pages' keys, the selection of pages, attention over them, and the adjustment of logits with the choice of the next tokens.

Positions, bounds, selections and logits are defined by single fp32 operations, so they are compared bit by bit with the
same operations in numpy.  Attention is compared with 64 bits, by test_paged.py's tolerances: u = eps / 2 of the
activations' type for the output and for every weight (relative to the sum A of weight times |value|, half the smallest
subnormal for weights below fp16's range), and the scores' error delta, which moves numerator and denominator by at most 2
delta A: d 2^-24 of the sum of |q k|, 2^-20 of a cap, and 2^-20 for the exponentials and sums in fp32."""
import ctypes
import math

import numpy as np
import pytest
import torch

from spectra_amd import _lib as L
from test_paged import _DT, KINDS, Batch, _gen, _tables


# -- rotary axes ---------------------------------------------------------------------------------
def _rotated(x, c, s):
    """Rows x [T, heads, d] turned by c, s [T, d / 2] with fp32 operations; where c is NaN the pair stays."""
    half = x.shape[-1] // 2
    a, b = x[..., :half].float(), x[..., half:].float()
    c, s = c[:, None], s[:, None]
    still = torch.isnan(c)
    return torch.cat([torch.where(still, a, a * c - b * s), torch.where(still, b, b * c + a * s)], -1).to(x.dtype)


def _angles(positions, axis, cos, sin):
    n = positions.shape[0]
    pair = torch.arange(axis.numel(), device="cuda")
    p = positions.long().t()[:, axis.long().clamp(max=n - 1)]
    c, s = cos[p, pair], sin[p, pair]
    return c.masked_fill(axis >= n, math.nan), s.masked_fill(axis >= n, math.nan)


def _bits(x):
    return x.contiguous().view(torch.int16 if x.element_size() == 2 else torch.uint8)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,d,page", [(24, 8, 128, 16), (4, 4, 64, 64), (5, 1, 128, 32)])
@pytest.mark.parametrize("n,lens", [([1], [1]), ([1, 1, 0, 1], [17, 300, 5, 64]), ([70, 3, 0, 129], [70, 40, 9, 400])])
@pytest.mark.parametrize("axes", ["sections", "interleaved", "mixed"])
def test_axes_append(hip, kind, heads, kv, d, page, n, lens, axes):
    """Queries, and the rows that the pages get: the plain append's of rows rotated beforehand."""
    from spectra_amd import kernels as K
    b = Batch(kind, n, lens, heads, kv, d, page, seed=21, pad=2)
    half = d // 2
    if axes == "sections":
        axis, count = K.rope_axes([half - 2 * (half // 3), half // 3, half // 3], d), 3
    elif axes == "interleaved":
        axis, count = K.rope_axes([half - half // 2, half // 4, half // 4], d, interleaved=True), 3
    else:  # four axes without order, some pairs of none
        axis, count = torch.randint(0, 6, (half,), generator=_gen(1), device="cuda").to(torch.uint8), 4
    cos, sin = _tables(500, d)
    pos = torch.randint(0, 500, (count, b.tokens), generator=_gen(2), device="cuda", dtype=torch.int32)
    qkv = b.rand(b.tokens, (heads + 2 * kv) * d)
    rows = qkv.view(b.tokens, heads + 2 * kv, d)
    c, s = _angles(pos, axis, cos, sin)
    turned = rows.clone()
    turned[:, : heads + kv] = _rotated(rows[:, : heads + kv], c, s)
    caches = [tuple(t.clone() for t in x) if kind == "4bit" else x.clone() for x in (b.k, b.v)]
    want = K.paged_rope_append(turned.view(b.tokens, -1), b.kv_lens, b.q_start, b.table, None, None, heads, *caches)
    q_out = torch.full_like(want, 7.0)
    got = K.paged_rope_axes_append(qkv, pos, axis, b.kv_lens, b.q_start, b.table, cos, sin, heads, b.k, b.v, q_out)
    used = sum(n)
    assert got is q_out and torch.equal(_bits(got[:used]), _bits(want[:used]))
    assert torch.all(got[used:] == 7.0)
    for x, y in zip((b.k, b.v), caches):
        for p, r in zip(*((x, y) if kind == "4bit" else ([x], [y]))):
            assert torch.equal(_bits(p), _bits(r))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_axes_of_one_position_are_the_plain_append(hip, kind):
    from spectra_amd import kernels as K
    b = Batch(kind, [40, 1, 3], [90, 64, 3], 6, 2, 128, 32, seed=22)
    cos, sin = _tables(100, 128)
    qkv = b.rand(b.tokens, 10 * 128)
    caches = [tuple(t.clone() for t in x) if kind == "4bit" else x.clone() for x in (b.k, b.v)]
    want = K.paged_rope_append(qkv, b.kv_lens, b.q_start, b.table, cos, sin, 6, *caches)
    p = torch.cat([torch.arange(m - n, m) for n, m in zip(b.n, b.lens)]).int().cuda().expand(3, -1)
    wide = torch.zeros(b.tokens, 10 * 128 + 24, dtype=qkv.dtype, device="cuda")  # rows of a wider matrix, too
    wide[:, : 10 * 128] = qkv
    axis = K.rope_axes([24, 20, 20], 128, interleaved=True)
    odd = torch.zeros(65, dtype=torch.uint8, device="cuda")  # axes that start at an odd address
    odd[1:] = axis
    got = K.paged_rope_axes_append(wide[:, : 10 * 128], p, odd[1:], b.kv_lens, b.q_start, b.table, cos, sin, 6, b.k, b.v)
    assert torch.equal(_bits(got), _bits(want))
    for x, y in zip((b.k, b.v), caches):
        for u, r in zip(*((x, y) if kind == "4bit" else ([x], [y]))):
            assert torch.equal(_bits(u), _bits(r))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_axes_outside(hip, kind):
    """Positions outside the tables: NaN queries, nothing appended; pairs that do not turn keep infinite partners."""
    from spectra_amd import kernels as K
    b = Batch(kind, [4], [20], 2, 1, 64, 16, seed=23)
    cos, sin = _tables(30, 64)
    qkv = b.rand(4, 4 * 64)
    pos = torch.tensor([[3, 30, 4, 5], [3, 4, -1, 2147483647]], dtype=torch.int32, device="cuda")
    axis = K.rope_axes([10, 12], 64)  # ten pairs stay as they are
    if kind != "4bit":
        qkv[0, 31], qkv[0, 63] = math.inf, 2.0
    before = [_bits(x).clone() for x in ((*b.k, *b.v) if kind == "4bit" else (b.k, b.v))]
    q = K.paged_rope_axes_append(qkv, pos, axis, b.kv_lens, b.q_start, b.table, cos, sin, 2, b.k, b.v)
    c, s = _angles(pos[:, :1], axis, cos, sin)
    assert torch.equal(_bits(q[:1]), _bits(_rotated(qkv[:1].view(1, 4, 64)[:, :2], c, s)))
    assert torch.isnan(q[1:]).all()
    page, row = int(b.table[0, 1]), torch.tensor([1, 2, 3], device="cuda")  # positions 17 .. 19
    for x, y in zip(((*b.k, *b.v) if kind == "4bit" else (b.k, b.v)), before):
        now = _bits(x)
        assert torch.equal(now[page][:, row], y[page][:, row])
        other = torch.ones(x.shape[0], dtype=torch.bool, device="cuda")
        other[page] = False
        assert torch.equal(now[other], y[other]) and not torch.equal(now[page], y[page])


def test_rope_axes():
    from spectra_amd import kernels as K
    cpu = torch.device("cpu")
    assert K.rope_axes([2, 3], 16, device=cpu).tolist() == [0, 0, 1, 1, 1, 255, 255, 255]
    assert K.rope_axes([4, 2, 2], 16, True, cpu).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert K.rope_axes([8], 16, device=cpu).tolist() == [0] * 8
    for bad in ([], [1] * 5, [-1, 3], [5, 4]):
        with pytest.raises(ValueError, match="sections"):
            K.rope_axes(bad, 16, device=cpu)
    with pytest.raises(ValueError, match="must hold"):
        K.rope_axes([2, 2], 16, True, cpu)


# -- bounds --------------------------------------------------------------------------------------
def _bounds_of(k):
    """Codes and scale of keys [rows, d], by the fp32 operations of the definition."""
    k = k.float().cpu().numpy()
    hi, lo, f = k.max(0), k.min(0), np.float32
    zero = np.zeros((2, k.shape[1]), np.int8)
    if not np.isfinite(k).all():
        return zero, f(np.inf)
    a = np.abs(k).max()
    if a < f(2.0 ** -100):
        return zero, f(0)
    inv = f(127) / a
    codes = np.stack([np.ceil(hi * inv), np.floor(lo * inv)])
    return np.clip(codes, -127, 127).astype(np.int8), a / f(127)


def _check_bounds(b, bounds, before):
    codes, scales = (t.clone() for t in before)
    for s, (n, m) in enumerate(zip(b.n, b.lens)):
        if n == 0:
            continue
        k, _ = b.rows(s)
        for j in range(max(m - n, 0) // b.page, (m - 1) // b.page + 1):
            for h in range(b.kv):
                c, a = _bounds_of(k[h, j * b.page: (j + 1) * b.page])
                codes[b.table[s, j].long(), h] = torch.from_numpy(c).cuda()
                scales[b.table[s, j].long(), h] = float(a)
    assert torch.equal(bounds[0], codes) and torch.equal(bounds[1], scales)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,d,page", [(4, 2, 128, 64), (3, 3, 64, 16), (1, 1, 128, 256)])
@pytest.mark.parametrize("n,lens", [([1], [1]), ([1, 0, 1, 1], [64, 5, 65, 300]), ([200, 1, 17], [200, 128, 333])])
def test_bounds(hip, kind, heads, kv, d, page, n, lens):
    from spectra_amd import kernels as K
    b = Batch(kind, n, lens, heads, kv, d, page, seed=31)
    codes, scales = K.paged_bounds(b.k)
    codes.random_(-100, 100)
    scales.uniform_()
    before = codes.clone(), scales.clone()
    got = K.paged_key_bounds(b.tokens, b.kv_lens, b.q_start, b.table, b.k, (codes, scales))
    assert got[0] is codes and got[1] is scales
    _check_bounds(b, got, before)
    values = K.paged_bounds_values(got, torch.float32)
    assert torch.equal(values, got[0].float() * got[1][:, :, None, None])
    half = K.paged_bounds_values(got, _DT[kind])
    assert torch.equal(half, values.to(_DT[kind]))


@pytest.mark.gpu
def test_bounds_hold_every_key(hip):
    """Every key lies between the values, up to the last bit of the scale."""
    from spectra_amd import kernels as K
    b = Batch("bf16", [300, 77], [300, 77], 4, 4, 128, 32, seed=32)
    bounds = K.paged_key_bounds(b.tokens, b.kv_lens, b.q_start, b.table, b.k, K.paged_bounds(b.k))
    values = K.paged_bounds_values(bounds, torch.float32).double()
    for s in range(2):
        k, _ = b.rows(s)
        for j in range(-(-b.lens[s] // 32)):
            page = int(b.table[s, j])
            x = k[:, 32 * j: 32 * j + 32]
            slack = 127 * 2.0 ** -22 * bounds[1][page].double()[:, None]
            assert (x.amax(1) <= values[page, :, 0] + slack).all() and (x.amin(1) >= values[page, :, 1] - slack).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
def test_bounds_of_odd_keys(hip, kind):
    """Infinities, NaN, zeros, subnormals, and the largest values; rows behind the length do not count."""
    from spectra_amd import kernels as K
    b = Batch(kind, [70], [70], 2, 2, 64, 16, seed=33)
    p = [int(x) for x in b.table[0, :5]]
    b.k[p[0], 0, 3, 5] = math.inf
    b.k[p[0], 1, 15, 63] = math.nan
    b.k[p[1], 0] = 0.0
    b.k[p[1], 1] = -0.0
    b.k[p[2], 0] = torch.finfo(_DT[kind]).smallest_normal / 4 if kind == "fp16" else 1e-39
    b.k[p[2], 1] = torch.finfo(_DT[kind]).max
    b.k[p[3], 0, :, 0] = -torch.finfo(_DT[kind]).max
    b.k[p[3], 1] = -2.0 ** (-14 if kind == "fp16" else -99)
    before = K.paged_bounds(b.k)
    bounds = K.paged_key_bounds(70, b.kv_lens, b.q_start, b.table, b.k, K.paged_bounds(b.k))
    _check_bounds(b, bounds, before)
    assert math.isinf(float(bounds[1][p[0], 0])) and math.isinf(float(bounds[1][p[0], 1]))
    values = K.paged_bounds_values(bounds)
    assert (values[p[0], :, 0] == math.inf).all() and (values[p[0], :, 1] == -math.inf).all()


@pytest.mark.gpu
def test_bounds_outside(hip):
    """Pages outside the pool, positions past the table, tokens behind the last sequence and starts that are no batch's:
    nothing is written for them."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [40, 30], [40, 30], 2, 1, 64, 16, seed=34)
    b.table[0, 1] = 1 << 29
    b.table[1, 0] = -1
    codes, scales = K.paged_bounds(b.k)
    codes.fill_(3)
    before = codes.clone(), scales.clone()
    K.paged_key_bounds(b.tokens + 50, b.kv_lens, b.q_start, b.table, b.k, (codes, scales))
    for s, j in ((0, 0), (0, 2), (1, 1)):
        page = int(b.table[s, j])
        c, a = _bounds_of(b.k[page, 0, : min(16, b.lens[s] - 16 * j)])
        before[0][page, 0], before[1][page, 0] = torch.from_numpy(c).cuda(), float(a)
    assert torch.equal(codes, before[0]) and torch.equal(scales, before[1])
    narrow = b.table[:, :1].contiguous()  # lengths past the table
    K.paged_key_bounds(b.tokens, b.kv_lens, b.q_start, narrow, b.k, (codes, scales))
    assert torch.equal(codes, before[0])
    for starts in ([0, 0, 0], [50, 20, 10], [-5, 1000, 3], [70, 70, 70]):
        K.paged_key_bounds(b.tokens, b.kv_lens, torch.tensor(starts, dtype=torch.int32, device="cuda"), b.table, b.k, (codes, scales))
    K.paged_key_bounds(0, b.kv_lens, b.q_start, b.table, b.k, (codes, scales))
    torch.cuda.synchronize()


# -- selection -----------------------------------------------------------------------------------
def _selected(q, codes, scales, table, visible, count, sink, local):
    """One token's blocks of one KV head: q [g, d], codes [pages, 2, d], scales [pages]."""
    f = np.float32
    q = q.float().cpu().numpy()
    a = np.abs(q).max()
    c = np.zeros(q.shape, np.int64)
    if np.isfinite(q).all() and a >= f(2.0 ** -100):
        c = np.rint(q * (f(127) / a)).astype(np.int64)
    keys = []
    for j in range(visible):
        page = int(table[j])
        if j < sink or j >= visible - local:
            keys.append((2, 0.0))
        elif not 0 <= page < codes.shape[0] or scales[page] == np.inf:
            keys.append((1, 0.0))
        else:
            hi, lo = codes[page].astype(np.int64)
            with np.errstate(over="ignore"):
                keys.append((0, float(f(max((np.maximum(c, 0) * hi + np.minimum(c, 0) * lo).sum(1))) * scales[page])))
    got = sorted(sorted(range(visible), key=lambda j: (-keys[j][0], -keys[j][1], j))[:count])
    return got + [-1] * (count - len(got))


def _check_select(b, bounds, count, sink, local, got, pad=None):
    codes, scales = (t.cpu().numpy() for t in bounds)
    table, g = b.table.cpu().numpy(), b.heads // b.kv
    got = got.cpu()
    at = 0
    for s, (n, m) in enumerate(zip(b.n, b.lens)):
        for t in range(n):
            i = m - n + t
            for h in range(b.kv):
                want = _selected(b.q[at + t, h * g: (h + 1) * g], codes[:, h], scales[:, h], table[s],
                                 min(i // b.page + 1, table.shape[1]), count, sink, local)
                assert got[at + t, h].tolist() == want, (s, t, h)
        at += n
    if pad is not None:
        assert (got[at:] == pad).all()


def _random_bounds(b, seed, levels=None):
    """Bounds of random keys; ``levels``: only so many different ones, so that scores tie."""
    g = _gen(seed)
    pages = (b.k[0] if b.kind == "4bit" else b.k).shape[0]
    codes = torch.randint(-30, 128, (pages, b.kv, 2, b.d), generator=g, device="cuda", dtype=torch.int8)
    codes[:, :, 1] = -codes[:, :, 1]
    scales = torch.rand(pages, b.kv, generator=g, device="cuda") * 0.01 + 0.001
    if levels is not None:
        of = torch.randint(0, levels, (pages,), generator=g, device="cuda")
        codes, scales = codes[of].contiguous(), scales[of].contiguous()
    return codes, scales


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv,d", [(3, 1, 64), (24, 8, 128), (14, 2, 128), (8, 8, 64), (16, 1, 128), (40, 2, 64), (20, 1, 128)])
@pytest.mark.parametrize("count,sink,local", [(1, 0, 1), (5, 1, 2), (8, 3, 5), (9, 0, 1), (40, 1, 1)])
def test_select(hip, kind, heads, kv, d, count, sink, local):
    from spectra_amd import kernels as K
    b = Batch(kind, [1, 1, 0, 1], [513, 1, 20, 200], heads, kv, d, 16, seed=41, pad=2)
    bounds = _random_bounds(b, 5)
    out = torch.full((b.tokens, kv, count), 77, dtype=torch.int32, device="cuda")
    got = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, bounds, 16, count, sink=sink, local=local, out=out)
    assert got is out
    _check_select(b, bounds, count, sink, local, got, pad=77)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,d,page", [(24, 8, 128, 16), (6, 1, 64, 32), (16, 2, 128, 16), (12, 1, 128, 16), (20, 1, 64, 16)])
@pytest.mark.parametrize("n,lens", [([5, 3, 4], [400, 3, 257]), ([70, 1, 0, 33], [150, 600, 9, 33])])
def test_select_drafts_and_chunks(hip, heads, kv, d, page, n, lens):
    from spectra_amd import kernels as K
    b = Batch("fp16", n, lens, heads, kv, d, page, seed=42, pad=3)
    bounds = _random_bounds(b, 6)
    wide = torch.zeros(b.tokens, heads + 3, d, dtype=b.q.dtype, device="cuda")[:, 2: 2 + heads]  # strided queries
    wide.copy_(b.q)
    for q in (b.q, wide):
        out = torch.full((b.tokens, kv, 6), 77, dtype=torch.int32, device="cuda")
        K.paged_select(q, b.kv_lens, b.q_start, b.table, bounds, page, 6, out=out)
        _check_select(b, bounds, 6, 1, 2, out, pad=77)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 7])
@pytest.mark.parametrize("levels", [1, 2, 40])
def test_select_ties_take_the_lowest_block(hip, n, levels):
    from spectra_amd import kernels as K
    b = Batch("fp16", [n, n], [3000, 900], 4, 2, 64, 16, seed=43)
    bounds = _random_bounds(b, 7, levels)
    for count in (4, 63, 64, 130):
        got = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, bounds, 16, count, sink=1, local=1)
        _check_select(b, bounds, count, 1, 1, got)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("m,page", [(16 * 1025, 16), (16 * 8190 + 5, 16), (32 * 3000, 32)])
def test_select_long_tables(hip, n, m, page):
    """Many candidates, with and without a workspace, which serves calls of other shapes in between."""
    from spectra_amd import kernels as K
    b = Batch("bf16", [n], [m], 8, 2, 64, page, seed=44)
    small = Batch("bf16", [1, 1], [300, 100], 4, 2, 64, 16, seed=45)
    bounds, few = _random_bounds(b, 8), _random_bounds(small, 9)
    ws = K.paged_select_workspace()
    want = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, bounds, page, 40)
    _check_select(b, bounds, 40, 1, 2, want)
    for _ in range(3):
        assert torch.equal(K.paged_select(b.q, b.kv_lens, b.q_start, b.table, bounds, page, 40, workspace=ws), want)
        got = K.paged_select(small.q, small.kv_lens, small.q_start, small.table, few, 16, 5, workspace=ws)
        _check_select(small, few, 5, 1, 2, got)
    short = b.kv_lens.clone().fill_(page * 30)  # few blocks in a wide table: nothing to choose
    got = K.paged_select(b.q, short, b.q_start, b.table, bounds, page, 40, workspace=ws)
    assert got[-1, 0].tolist() == list(range(30)) + [-1] * 10


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 4])
def test_select_odd_blocks_and_queries(hip, n):
    """Infinite bounds and pages outside the pool come first; queries that are not finite, or vanish, score nothing."""
    from spectra_amd import kernels as K
    b = Batch("bf16", [n, n, n], [800, 800, 640], 4, 2, 128, 16, seed=46)
    codes, scales = _random_bounds(b, 10)
    scales[b.table[0, 7].long(), 0] = math.inf
    codes[b.table[0, 7].long()] = 0
    scales[b.table[0, 9].long()] = 0.0
    b.table[0, 20], b.table[0, 21] = -1, 1 << 30
    b.q[n, 1, 3] = math.inf  # the second sequence's first token, first KV head
    b.q[n, 2, 3] = math.nan
    b.q[2 * n] = 1e-38  # below 2^-100 of one scale
    got = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, (codes, scales), 16, 6)
    _check_select(b, (codes, scales), 6, 1, 2, got)
    assert got[n, 0].tolist() == [0, 1, 2, 3, 48, 49]


@pytest.mark.gpu
def test_select_outside(hip):
    """Positions past the table see its blocks; starts that are no batch's and lengths of zero end, and stay inside."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [2, 1], [400, 90], 4, 2, 64, 16, seed=47)
    bounds = _random_bounds(b, 11)
    got = K.paged_select(b.q, b.kv_lens + 5000, b.q_start, b.table, bounds, 16, 4)
    w = b.table.shape[1]
    assert (got[:, :, -1] == w - 1).all() and (got[:, :, -2] == w - 2).all() and (got[:, :, 0] == 0).all()
    got = K.paged_select(b.q, torch.zeros_like(b.kv_lens), b.q_start, b.table, bounds, 16, 4)
    assert (got[:2] == -1).all() and (got[2] == -1).all()
    for starts in ([50, 20, 10], [-5, 1000, 3], [3, 3, 3], [0, 0, 0], [2, 1, 3]):
        K.paged_select(b.q, b.kv_lens, torch.tensor(starts, dtype=torch.int32, device="cuda"), b.table, bounds, 16, 4)
    torch.cuda.synchronize()
    empty = K.paged_select(b.q[:0], b.kv_lens, b.q_start, b.table, bounds, 16, 4)
    assert empty.shape == (0, 2, 4)


# -- attention over blocks -----------------------------------------------------------------------
def _random_blocks(b, count, seed, holes=True):
    """Blocks of each token and KV head: some of those that it sees, in any order, holes among them."""
    g = torch.Generator().manual_seed(seed)
    out = torch.full((b.tokens, b.kv, count), -1, dtype=torch.int32)
    at = 0
    for n, m in zip(b.n, b.lens):
        for t in range(n):
            blocks = (m - n + t) // b.page + 1
            for h in range(b.kv):
                p = torch.randperm(blocks, generator=g)[: count - (count // 3 if holes else 0)]
                slots = torch.randperm(count, generator=g)[: len(p)] if holes else torch.arange(len(p))
                out[at + t, h, slots] = p.int()
        at += n
    return out.cuda()


def _blocks_reference(b, blocks, scale=None, cap=0.0):
    scale = 1.0 / math.sqrt(b.d) if scale is None else scale
    u = torch.finfo(_DT[b.kind]).eps / 2
    sub = 2.0 ** -25 if b.kind != "bf16" else 0.0
    out = torch.zeros(b.tokens, b.heads, b.d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    at = 0
    for s, (n, m) in enumerate(zip(b.n, b.lens)):
        k, v = b.rows(s)
        for t in range(n):
            for kv in range(b.kv):
                j = torch.cat([torch.arange(x * b.page, (x + 1) * b.page) for x in blocks[at + t, kv].tolist() if x >= 0] +
                              [torch.zeros(0, dtype=torch.long)]).cuda()
                j = j[j <= m - n + t]
                if j.numel() == 0:
                    continue
                heads = slice(kv * b.heads // b.kv, (kv + 1) * b.heads // b.kv)
                q, kk, vv = b.q[at + t, heads].double(), k[kv, j], v[kv, j]
                x = q @ kk.T * scale
                delta = b.d * 2.0 ** -24 * (q.abs() @ kk.abs().T * scale).amax(-1, keepdim=True)
                if cap:
                    x, delta = cap * torch.tanh(x / cap), delta + cap * 2.0 ** -20
                e = torch.exp(x - x.amax(-1, keepdim=True))
                total = e.sum(-1, keepdim=True)
                o, a = e @ vv / total, e @ vv.abs() / total
                out[at + t, heads] = o
                tol[at + t, heads] = u * o.abs() + (u + 2 * delta + 2.0 ** -20) * a + sub * (1 + vv.abs().sum(0) / total)
        at += n
    return out, tol


def _close(got, want, tol, rows=None):
    err = (got.double() - want).abs()
    if rows is not None:
        err, tol = err[:rows], tol[:rows]
    assert torch.isfinite(got[:rows]).all()
    assert (err <= tol).all(), float((err - tol).max())


def _attend(b, blocks, **kw):
    from spectra_amd import kernels as K
    return K.paged_attend_blocks(b.q, blocks, b.kv_lens, b.q_start, b.table, b.k, b.v, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,d,page", [(24, 8, 128, 16), (4, 4, 64, 64), (14, 2, 64, 32), (16, 1, 128, 128), (5, 1, 128, 16),
                                             (40, 2, 64, 16), (20, 1, 128, 64)])
@pytest.mark.parametrize("count", [1, 3, 10])
def test_blocks_single_tokens(hip, kind, heads, kv, d, page, count):
    b = Batch(kind, [1, 1, 0, 1, 1], [300, 1, 9, 17, 900], heads, kv, d, page, seed=51, pad=2)
    blocks = _random_blocks(b, count, 1)
    out = torch.full_like(b.q, 7.0)
    assert _attend(b, blocks, out=out) is out
    want, tol = _blocks_reference(b, blocks)
    _close(out, want, tol, 4)
    assert (out[4:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cap,scale", [(0.0, 0.3), (2.0, None), (400.0, None), (1e6, 0.2)])
def test_blocks_drafts_and_chunks(hip, kind, cap, scale):
    b = Batch(kind, [5, 40, 3], [400, 40, 3000], 6, 2, 128 if cap else 64, 16, seed=52)
    blocks = _random_blocks(b, 21, 2)
    want, tol = _blocks_reference(b, blocks, scale, cap)
    _close(_attend(b, blocks, cap=cap, scale=scale), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,tokens", [(8, 1, 1), (24, 8, 1), (16, 16, 3)])
def test_blocks_split_long_lists(hip, kind, heads, kv, tokens):
    """A long list is shared among workgroups and joined; a workspace serves calls of other shapes in between."""
    from spectra_amd import kernels as K
    b = Batch(kind, [tokens], [9000], heads, kv, 128, 32, seed=53)
    small = Batch(kind, [1, 1], [64, 30], 4, 2, 128, 16, seed=54)
    blocks, few = _random_blocks(b, 250, 3, holes=False), _random_blocks(small, 4, 4)
    ws = K.paged_attend_workspace(128)
    want, tol = _blocks_reference(b, blocks)
    other, slack = _blocks_reference(small, few)
    first = _attend(b, blocks, workspace=ws)
    _close(first, want, tol)
    for _ in range(3):
        _close(_attend(small, few, workspace=ws), other, slack)
        assert torch.equal(_attend(b, blocks, workspace=ws), first)  # whatever order the parts arrive in
        b.attend(workspace=ws)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_all_blocks_are_the_dense_attention(hip, kind):
    b = Batch(kind, [1, 4, 60], [700, 90, 200], 8, 2, 128, 32, seed=55)
    n = 700 // 32 + 1
    every = torch.arange(n, device="cuda", dtype=torch.int32).expand(b.tokens, 2, n)  # ones past a sequence's table, too
    want, tol = b.reference()
    _close(_attend(b, every), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "bf16"])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_blocks_hide_what_is_not_seen(hip, kind, what):
    """Rows behind the position, and pages that are not listed, hold anything."""
    b = Batch(kind, [1, 3], [37, 70], 4, 2, 64, 16, seed=56)
    blocks = _random_blocks(b, 4, 5)
    want, tol = _blocks_reference(b, blocks)
    blocks[1:, :, 0] = torch.where(blocks[1:, :, 0] < 0, 6, blocks[1:, :, 0])  # a block of later positions: nothing of it is seen
    b.k.masked_fill_(~b.valid[:, None, :, None], what)
    b.v.masked_fill_(~b.valid[:, None, :, None], what)
    b.k[b.table[1, 4].long(), :, 5:] = what  # keys 69 ..: seen by the last token alone
    b.v[b.table[1, 4].long(), :, 5:] = what
    got = _attend(b, blocks)
    sees = (blocks[3] == 4).any(-1).repeat_interleave(2)
    _close(got[:3], want[:3], tol[:3])
    assert torch.isnan(got[3, sees]).all() if math.isnan(what) else not torch.isfinite(got[3, sees]).all(-1).any()
    _close(got[3][~sees], want[3][~sees], tol[3][~sees])
    listed = blocks.clone()
    listed[0, :, :] = torch.tensor([0, -1, -1, -1], device="cuda", dtype=torch.int32)
    b.v[b.table[0, 1].long()] = what  # not listed any more
    assert torch.isfinite(_attend(b, listed)[0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_blocks_without_keys_and_outside(hip, kind):
    b = Batch(kind, [1, 1, 1, 1], [70, 70, 300, 40], 4, 2, 128, 16, seed=57)
    blocks = torch.tensor([[-1, -1, -7], [9, 1 << 30, -1], [3, 0, 18], [2, 0, 1]], dtype=torch.int32, device="cuda")
    blocks = blocks[:, None].expand(4, 2, 3)
    b.table[2, 3] = 1 << 30  # a page that is not there
    got = _attend(b, blocks)
    assert (got[0] == 0).all() and (got[1] == 0).all() and torch.isnan(got[2]).all()
    b.table[2, 3] = 0
    want, tol = _blocks_reference(b, torch.where(blocks > 18, -1, blocks))
    _close(got[3:], want[3:], tol[3:])
    b.kv_lens[3] = 16 * b.table.shape[1] + 1  # a position past the table
    assert torch.isnan(_attend(b, blocks)[3]).all()
    for starts in ([9, 9, 1, 0, 2], [0, 0, 0, 0, 0], [-4, 100, 3, 2, 1]):
        bad = torch.tensor(starts, dtype=torch.int32, device="cuda")
        from spectra_amd import kernels as K
        K.paged_attend_blocks(b.q, blocks, b.kv_lens, bad, b.table, b.k, b.v)
    torch.cuda.synchronize()
    assert _attend(Batch(kind, [0], [5], 4, 2, 64, 16), torch.zeros(0, 2, 1, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)


@pytest.mark.gpu
def test_blocks_named_twice_and_strided(hip):
    """A block named twice counts twice: with one other, two thirds of the weight at equal scores."""
    b = Batch("fp16", [1], [32], 2, 1, 64, 16, seed=58)
    b.k.zero_()
    b.v[b.table[0, 0].long()], b.v[b.table[0, 1].long()] = 3.0, 6.0
    blocks = torch.tensor([[[1, 0, 1]]], dtype=torch.int32, device="cuda")
    assert (_attend(b, blocks) - 5.0).abs().max() <= 5 * 2.0 ** -10
    wide = torch.zeros(1, 1, 6, dtype=torch.int32, device="cuda")
    wide[..., ::2] = blocks
    assert torch.equal(_attend(b, wide[..., ::2]), _attend(b, blocks))
    c = Batch("bf16", [3, 1], [100, 60], 4, 2, 128, 16, seed=59)
    lists = _random_blocks(c, 3, 6)
    want = _attend(c, lists)
    from spectra_amd import kernels as K
    for q in (torch.zeros(4, 9, 128, dtype=c.q.dtype, device="cuda")[:, 3: 7], torch.zeros(4, 128, 4, dtype=c.q.dtype, device="cuda").transpose(1, 2)):
        q.copy_(c.q)
        assert torch.equal(K.paged_attend_blocks(q, lists, c.kv_lens, c.q_start, c.table, c.k, c.v), want)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [7e37, 1e-24])
def test_blocks_of_values_at_the_ends_of_the_range(hip, size):
    b = Batch("bf16", [1, 3], [600, 600], 8, 2, 128, 16, seed=60)
    b.v.mul_(size)
    blocks = _random_blocks(b, 30, 7)
    want, tol = _blocks_reference(b, blocks)
    _close(_attend(b, blocks), want, tol)


# -- logits --------------------------------------------------------------------------------------
def _adjusted(x, history=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None, bias_ids=None,
              bias=None, allowed=None, allowed_rows=None):
    """The adjusted logits in numpy, each operation in fp32."""
    f = np.float32
    x = x.float().cpu().numpy().copy()
    host = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    history, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias, allowed, allowed_rows = map(
        host, (history, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias, allowed, allowed_rows))
    n, vocab = x.shape
    with np.errstate(all="ignore"):
        for b in range(n):
            if any(t is not None for t in (repetition, presence, frequency)):
                m = history.shape[1] if lens is None else min(max(int(lens[b]), 0), history.shape[1])
                p = 0 if prompt_lens is None else int(prompt_lens[b])
                row = history[b, :m]
                ok = (row >= 0) & (row < vocab)
                seen = np.unique(row[ok])
                count = np.bincount(row[ok & (np.arange(m) >= p)], minlength=vocab).astype(f)
                r = f(1) if repetition is None else repetition[b]
                x[b, seen] = np.where(x[b, seen] > 0, x[b, seen] / r, x[b, seen] * r)
                if frequency is not None:
                    x[b, seen] = np.where(count[seen] > 0, x[b, seen] - frequency[b] * count[seen], x[b, seen])
                if presence is not None:
                    x[b, seen] = np.where(count[seen] > 0, x[b, seen] - presence[b], x[b, seen])
            if bias is not None:
                last = {int(v): bias[b, e] for e, v in enumerate(bias_ids[b]) if 0 <= v < vocab}
                for v, w in last.items():
                    x[b, v] += w
            if allowed is not None:
                s = b if allowed_rows is None else int(allowed_rows[b])
                if 0 <= s < allowed.shape[0]:
                    bits = np.unpackbits(allowed[s].view(np.uint8), bitorder="little")[:vocab]
                    x[b, bits == 0] = -np.inf
    return torch.from_numpy(x)


def _picked(x):
    """The largest of each row, NaN before all, the lowest on ties; -1 where nothing is left."""
    at = torch.where(torch.isnan(x).any(1), torch.isnan(x).int().argmax(1), (x == x.amax(1, keepdim=True)).int().argmax(1))
    return torch.where((x == -math.inf).all(1), -1, at)


def _case(rows, vocab, dtype, seed, history=0, penalties="rpf", biases=0, masks=0, lens=True, row_masks=False):
    g = _gen(seed)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype)
    kw = {}
    if history:
        kw["history"] = (torch.rand(rows, history, generator=g, device="cuda") ** 3 * vocab).long() - int(vocab > 3)
        kw["history"][:, ::7] = vocab + 5
        if lens:
            kw["lens"] = torch.randint(-1, history + 3, (rows,), generator=g, device="cuda", dtype=torch.int32)
            kw["prompt_lens"] = torch.randint(0, history + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
        for name in penalties:
            key = dict(r="repetition", p="presence", f="frequency")[name]
            kw[key] = torch.rand(rows, generator=g, device="cuda") + (0.7 if name == "r" else 0.0)
    if biases:
        kw["bias_ids"] = torch.randint(-1, vocab + 1, (rows, biases), generator=g, device="cuda")
        kw["bias"] = torch.randn(rows, biases, generator=g, device="cuda") * 4
    if masks:
        words = -(-vocab // 32)
        kw["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (masks, words), generator=g, device="cuda").int()
        kw["allowed"][0] = 0  # nothing is left
        if not row_masks:
            kw["allowed_rows"] = torch.randint(-1, masks + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return x, kw


def _check_logits(x, kw, workspace=None):
    from spectra_amd import kernels as K
    want = _adjusted(x, **kw)
    got = K.adjust_logits(x, **kw)
    assert got.dtype == x.dtype and torch.equal(got.cpu().nan_to_num(nan=1e30), want.to(x.dtype).nan_to_num(nan=1e30))
    token = K.next_tokens(x, workspace=workspace, **kw)
    assert token.dtype == torch.int64 and torch.equal(token.cpu(), _picked(want))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (3, 2047), (2, 2048), (2, 2049), (5, 8193), (1, 32003), (2, 128256)])
@pytest.mark.parametrize("kw", [dict(), dict(history=50), dict(history=3000, penalties="r", lens=False), dict(history=1, penalties="pf"),
                                dict(biases=7), dict(masks=3), dict(history=300, biases=40, masks=2)])
def test_logits(hip, dtype, rows, vocab, kw):
    _check_logits(*_case(rows, vocab, dtype, 61, **kw))


@pytest.mark.gpu
def test_logits_of_a_large_batch(hip):
    """Larger slices, and a workspace that serves calls of other shapes in between."""
    from spectra_amd import kernels as K
    ws = K.next_tokens_workspace()
    for rows, vocab in ((700, 8200), (4096, 33), (64, 70001), (1, 128256)):
        x, kw = _case(rows, vocab, torch.float16, 62, history=120, biases=3, masks=5)
        _check_logits(x, kw, ws)
        _check_logits(x[:1], {k: v[:1] if k != "allowed" else v for k, v in kw.items()}, ws)
    assert (ws == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(60, 16384), (60, 16385), (40, 40003), (9, 128256)])
@pytest.mark.parametrize("kw", [dict(history=4000), dict(history=3001, biases=1100, masks=3), dict(biases=5000, masks=2)])
def test_logits_in_large_slices(hip, dtype, rows, vocab, kw):
    """So many tokens to adjust that a slice is 16384 logits, the last one of a row shorter."""
    _check_logits(*_case(rows, vocab, dtype, 71, **kw))


@pytest.mark.gpu
def test_logits_masks_by_row(hip):
    x, kw = _case(3, 1000, torch.float32, 63, masks=3, row_masks=True)
    _check_logits(x, kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_logits_that_are_odd(hip, dtype):
    """NaN, infinities, zeros of both signs, ties, the type's lowest value; an infinite bias."""
    from spectra_amd import kernels as K
    x = torch.zeros(8, 5000, dtype=dtype, device="cuda")
    x[1, 4000], x[1, 3000] = math.nan, math.inf
    x[2, 4000], x[2, 10] = math.inf, math.inf
    x[3] = -math.inf
    x[4] = -math.inf
    x[4, 4999] = torch.finfo(dtype).min
    x[5, 1], x[5, 0] = 0.0, -0.0
    x[6, ::2] = math.nan
    x[7] = torch.finfo(dtype).min
    kw = dict(history=torch.tensor([[10, 3000, 4000, 4999, 0, 2, 2, 2]], device="cuda").repeat(8, 1),
              repetition=torch.full((8,), 1.5, device="cuda"), frequency=torch.full((8,), 0.25, device="cuda"),
              presence=torch.full((8,), -0.5, device="cuda"))
    _check_logits(x, {})
    _check_logits(x, kw)
    bias = dict(bias_ids=torch.tensor([[5, 6, 5, -1]], device="cuda").repeat(8, 1),
                bias=torch.tensor([[9.0, math.inf, -math.inf, 3.0]], device="cuda").repeat(8, 1))
    _check_logits(x, bias)
    none = torch.zeros(1, 157, dtype=torch.int32, device="cuda")
    rows = torch.zeros(8, dtype=torch.int32, device="cuda")
    _check_logits(x, dict(allowed=none, allowed_rows=rows, **bias))
    assert (K.next_tokens(x, allowed=none, allowed_rows=rows) == -1).all()
    assert int(K.next_tokens(x)[3]) == -1 and int(K.next_tokens(x)[5]) == 0
    assert int(K.greedy_next(x[0].half(), torch.zeros(1, dtype=torch.int64, device="cuda"))) == int(K.next_tokens(x)[0])


@pytest.mark.gpu
def test_logits_infinite_penalties(hip):
    """They forbid the answer's tokens, not the prompt's; ids at the ends of their type count nothing."""
    x = torch.randn(2, 3000, generator=_gen(67), device="cuda")
    ends = [-2 ** 63, 2 ** 63 - 1, -1, 3000]
    history = torch.tensor([[5, 2500, 7, 2600, 5] + ends] * 2, device="cuda")
    kw = dict(history=history, prompt_lens=torch.tensor([2, 0], dtype=torch.int32, device="cuda"),
              bias_ids=torch.tensor([ends] * 2, device="cuda"), bias=torch.ones(2, 4, device="cuda"))
    for name in ("frequency", "presence"):
        got = _check_logits(x, {**kw, name: torch.full((2,), math.inf, device="cuda")})
        assert got[0, 2500] == x[0, 2500] and (got[0, [5, 7, 2600]] == -math.inf).all() and (got[1, [5, 7, 2500, 2600]] == -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_logits_in_place_strided_and_from_odd_addresses(hip, dtype):
    from spectra_amd import kernels as K
    x, kw = _case(4, 4099, dtype, 64, history=100, biases=5, masks=2)
    want = K.adjust_logits(x, **kw)
    token = K.next_tokens(x, **kw)
    room = torch.full((4, 4200), 7.0, dtype=dtype, device="cuda")
    view = room[:, 3: 3 + 4099]
    view.copy_(x)
    assert torch.equal(K.adjust_logits(view, **kw), want) and torch.equal(K.next_tokens(view, **kw), token)
    assert K.adjust_logits(view, **kw, out=view) is view and torch.equal(view, want)
    assert (room[:, :3] == 7.0).all() and (room[:, 3 + 4099:] == 7.0).all()
    other = torch.full((4, 5000), 7.0, dtype=dtype, device="cuda")
    K.adjust_logits(x, **kw, out=other[:, 1: 4100])
    assert torch.equal(other[:, 1: 4100], want) and (other[:, 4100:] == 7.0).all() and (other[:, 0] == 7.0).all()
    t = x.t().contiguous().t()  # columns beside each other: copied first
    assert torch.equal(K.adjust_logits(t, **kw), want) and torch.equal(K.next_tokens(t, **kw), token)
    strided = {**kw, "history": kw["history"].t().contiguous().t(), "allowed": kw["allowed"].repeat(1, 2)[:, : kw["allowed"].shape[1]],
               "bias_ids": kw["bias_ids"].repeat(1, 3)[:, :5], "bias": kw["bias"].t().contiguous().t()}
    assert torch.equal(K.adjust_logits(x, **strided), want)
    one = {k: (v[:1].expand(4, -1) if k == "history" else v) for k, v in kw.items()}  # one history for all rows
    same = {k: (v.contiguous() if k == "history" else v) for k, v in one.items()}
    assert torch.equal(K.adjust_logits(x, **one), K.adjust_logits(x, **same))
    out = torch.full((4,), 9, dtype=torch.int64, device="cuda")
    assert K.next_tokens(x, **kw, out=out) is out and torch.equal(out, token)
    assert K.adjust_logits(x[:0]).shape == (0, 4099) and K.next_tokens(x[:0]).shape == (0,)


# -- together ------------------------------------------------------------------------------------
def _step(b, s):
    """One step of a batch: append, bounds, selection, attention, logits by the tied embedding, the next tokens."""
    from spectra_amd import kernels as K
    where = b.kv_lens, b.q_start, b.table
    q = K.paged_rope_axes_append(s["qkv"], s["pos"], s["axis"], *where, s["cos"], s["sin"], b.heads, b.k, b.v)
    K.paged_key_bounds(b.tokens, *where, b.k, s["bounds"])
    blocks = K.paged_select(q, *where, s["bounds"], b.page, s["count"], workspace=s["select"])
    o = K.paged_attend_blocks(q, blocks, *where, b.k, b.v, workspace=s["attend"])
    logits = K.w4a16_linear(s["head"], o.view(b.tokens, -1))
    return blocks, o, K.next_tokens(logits, history=s["history"], lens=s["lens"], repetition=s["repetition"], allowed=s["allowed"],
                                    allowed_rows=s["rows"], workspace=s["next"])


def _session(kind, seed, n=(1, 1, 1), lens=(400, 33, 700)):
    from spectra_amd import compressor as C
    from spectra_amd import kernels as K
    b = Batch(kind, list(n), list(lens), 4, 2, 64, 16, seed=seed)
    if kind != "4bit":  # (rows that no sequence has filled hold NaN, and a step's lengths go back over them)
        for x in (b.k, b.v):
            x.nan_to_num_(0.0)
    vocab = 500
    q = C.quantize_nf4(b.rand(vocab, 256) * 0.1, 64, 0, None, True)
    ops = K.QWeightOperands(q.packed, q.absmax, None, 256, codebook="nf4", group_size=64, marlin_layout=True)
    cos, sin = _tables(800, 64)
    full = torch.tensor([0, b.tokens], dtype=torch.int32, device="cuda")
    bounds = K.paged_bounds(b.k)
    for i, m in enumerate(b.lens):  # the bounds of what is there
        K.paged_key_bounds(m, b.kv_lens[i: i + 1], full.clone().fill_(m) * torch.tensor([0, 1], device="cuda", dtype=torch.int32),
                           b.table[i: i + 1], b.k, bounds)
    s = dict(qkv=b.rand(b.tokens, 8 * 64), pos=torch.randint(0, 800, (3, b.tokens), device="cuda", dtype=torch.int32, generator=_gen(seed)),
             axis=K.rope_axes([12, 10, 10], 64, interleaved=True), cos=cos, sin=sin, bounds=bounds, count=6, head=ops,
             history=torch.randint(0, vocab, (b.tokens, 40), device="cuda", generator=_gen(seed + 1)),
             lens=torch.full((b.tokens,), 30, dtype=torch.int32, device="cuda"),
             repetition=torch.full((b.tokens,), 1.3, device="cuda"),
             allowed=torch.randint(-2 ** 31, 2 ** 31, (2, 16), device="cuda", generator=_gen(seed + 2)).int(),
             rows=torch.tensor(([0, -1, 1] * b.tokens)[: b.tokens], dtype=torch.int32, device="cuda"),
             select=K.paged_select_workspace(), attend=K.paged_attend_workspace(64), next=K.next_tokens_workspace())
    return b, s


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_a_step_together(hip, kind):
    """Each part against its reference on what the part before it left."""
    from spectra_amd import kernels as K
    b, s = _session(kind, 71)
    blocks, o, tokens = _step(b, s)
    where = b.kv_lens, b.q_start, b.table
    c, sn = _angles(s["pos"], s["axis"], s["cos"], s["sin"])
    b.q = _rotated(s["qkv"].view(3, 8, 64)[:, :4], c, sn)
    assert torch.equal(_bits(K.paged_rope_axes_append(s["qkv"], s["pos"], s["axis"], *where, s["cos"], s["sin"], 4, b.k, b.v)), _bits(b.q))
    for i, m in enumerate(b.lens):
        k, _ = b.rows(i)
        for j in range(-(-m // 16)):
            for h in range(2):
                codes, a = _bounds_of(k[h, 16 * j: 16 * j + 16])
                page = int(b.table[i, j])
                assert np.array_equal(s["bounds"][0][page, h].cpu().numpy(), codes) and float(s["bounds"][1][page, h]) == float(a)
    _check_select(b, s["bounds"], 6, 1, 2, blocks)
    want, tol = _blocks_reference(b, blocks)
    _close(o, want, tol)
    logits = K.w4a16_linear(s["head"], o.view(3, -1))
    kw = dict(history=s["history"], lens=s["lens"], repetition=s["repetition"], allowed=s["allowed"], allowed_rows=s["rows"])
    assert torch.equal(tokens.cpu(), _picked(_adjusted(logits, **kw)))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_a_step_captured(hip, kind):
    """Replays follow lengths, positions, histories and masks, and give what eager steps give, two graphs in turn."""
    sessions = [_session(kind, 72), _session(kind, 73, (2, 1), (300, 90))]
    graphs = []
    for b, s in sessions:
        _step(b, s)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(b, s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(b, s)
        graphs.append((g, out))
    for turn in range(4):
        for (b, s), (g, out) in zip(sessions, graphs):
            b.kv_lens.sub_(17 * (turn % 2))
            s["pos"].add_(turn).clamp_(max=799)
            s["lens"].sub_(5)
            s["allowed"].bitwise_not_()
            s["qkv"].mul_(-1.0)
            g.replay()
            torch.cuda.synchronize()
            got = [x.clone() for x in out]
            for x, y in zip(got, _step(b, s)):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_steps_on_two_streams(hip):
    b, s = _session("fp16", 74)
    other = {**s}
    from spectra_amd import kernels as K
    other.update(select=K.paged_select_workspace(), attend=K.paged_attend_workspace(64), next=K.next_tokens_workspace())
    _step(b, s)
    want = [x.clone() for x in _step(b, s)]  # (the rows that the step writes are those that are there)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for st, mine in zip(streams, (s, other)):
            with torch.cuda.stream(st):
                q = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, mine["bounds"], 16, 6, workspace=mine["select"])
                o = K.paged_attend_blocks(b.q, q, b.kv_lens, b.q_start, b.table, b.k, b.v, workspace=mine["attend"])
                t = K.next_tokens(o.view(3, -1).float(), workspace=mine["next"])
                outs.append((q, o, t))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for one in outs for x, y in zip(one, outs[0])) and len(want) == 3


# -- refusals ------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_refusals(hip):
    from spectra_amd import kernels as K
    b = Batch("fp16", [2, 1], [40, 20], 4, 2, 64, 16, seed=81)
    where = b.kv_lens, b.q_start, b.table
    i32 = lambda *x: torch.zeros(*x, dtype=torch.int32, device="cuda")  # noqa: E731
    cos, sin = _tables(50, 64)
    rows, pos, axis = b.rand(3, 8 * 64), i32(3, 3), K.rope_axes([32], 64)

    def bad(match, f, *args, **kw):
        with pytest.raises(ValueError, match=match):
            f(*args, **kw)

    append = K.paged_rope_axes_append
    bad("positions", append, rows, pos.long(), axis, *where, cos, sin, 4, b.k, b.v)
    bad("positions", append, rows, i32(5, 3), axis, *where, cos, sin, 4, b.k, b.v)
    bad("positions", append, rows, i32(3, 4), axis, *where, cos, sin, 4, b.k, b.v)
    bad("positions", append, rows, i32(3), axis, *where, cos, sin, 4, b.k, b.v)
    bad("axis", append, rows, pos, axis[:31], *where, cos, sin, 4, b.k, b.v)
    bad("axis", append, rows, pos, axis.int(), *where, cos, sin, 4, b.k, b.v)
    bad("at least a row", append, rows, pos, axis, *where, cos[:0], sin[:0], 4, b.k, b.v)
    bad("cos and sin", append, rows, pos, axis, *where, cos, sin[:-1], 4, b.k, b.v)
    bad("q_out", append, rows, pos, axis, *where, cos, sin, 4, b.k, b.v, torch.empty(3, 4, 32, device="cuda"))
    codes, scales = K.paged_bounds(b.k)
    bad("codes", K.paged_key_bounds, 3, *where, b.k, (codes.int(), scales))
    bad("codes", K.paged_key_bounds, 3, *where, b.k, (codes[:-1], scales[:-1]))
    bad("scales", K.paged_key_bounds, 3, *where, b.k, (codes, scales.half()))
    bad("tokens", K.paged_key_bounds, -1, *where, b.k, (codes, scales))
    bad("k_pages", K.paged_key_bounds, 3, *where, (b.k, b.k), (codes, scales))
    bad("fp16", K.paged_key_bounds, 3, *where, b.k.float(), (codes, scales))
    bad("out_dtype", K.paged_bounds_values, (codes, scales), torch.int8)
    bad("codes", K.paged_bounds_values, (codes[:, :, :1], scales))
    sel = K.paged_select
    bad("count", sel, b.q, *where, (codes, scales), 16, 2)
    bad("count", sel, b.q, *where, (codes, scales), 16, 4, sink=2, local=3)
    bad("count", sel, b.q, *where, (codes, scales), 16, 4, local=0)
    bad("count", sel, b.q, *where, (codes, scales), 16, 40000)
    bad("power of two", sel, b.q, *where, (codes, scales), 24, 4)
    bad("sizes", sel, b.q, *where, (codes, scales), 1 << 17, 4)
    bad("q must", sel, b.q.float(), *where, (codes, scales), 16, 4)
    bad("codes", sel, b.q[..., :32].contiguous(), *where, (codes, scales), 16, 4)
    bad("multiple", sel, b.q[:, :3], *where, (codes, scales), 16, 4)
    bad("out", sel, b.q, *where, (codes, scales), 16, 4, out=i32(3, 2, 5))
    bad("kv_lens", sel, b.q, b.kv_lens.long(), *where[1:], (codes, scales), 16, 4)
    with pytest.raises(L.SpectraError) as e:
        sel(b.q, *where, (codes, scales), 16, 4, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    assert e.value.status == L.ERR_WORKSPACE
    with pytest.raises(L.SpectraError) as e:
        sel(b.q, *where[:2], i32(2, 32769), (codes, scales), 16, 4)
    assert e.value.status == L.ERR_UNSUPPORTED
    att, blocks = K.paged_attend_blocks, i32(3, 2, 4)
    bad("blocks", att, b.q, blocks.long(), *where, b.k, b.v)
    bad("blocks", att, b.q, blocks[:2], *where, b.k, b.v)
    bad("blocks", att, b.q, blocks[:, :1], *where, b.k, b.v)
    bad("blocks", att, b.q, blocks[..., :0], *where, b.k, b.v)
    bad("scale", att, b.q, blocks, *where, b.k, b.v, scale=-1.0)
    bad("cap", att, b.q, blocks, *where, b.k, b.v, cap=math.nan)
    bad("out", att, b.q, blocks, *where, b.k, b.v, out=b.q.float())
    bad("overlap", att, b.q, blocks, *where, b.k, b.v, out=b.q)
    with pytest.raises(L.SpectraError) as e:
        att(b.q, blocks, *where, b.k, b.v, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    assert e.value.status == L.ERR_WORKSPACE
    x = torch.zeros(2, 100, device="cuda")
    h, one = torch.zeros(2, 5, dtype=torch.int64, device="cuda"), torch.ones(2, device="cuda")
    for f in (K.adjust_logits, K.next_tokens):
        bad("logits", f, x.double())
        bad("logits", f, x[0])
        bad("need a history", f, x, repetition=one)
        bad("of a history", f, x, lens=i32(2))
        bad("history", f, x, history=h.int(), repetition=one)
        bad("history", f, x, history=h[:1], repetition=one)
        bad("repetition", f, x, history=h, repetition=one.double())
        bad("presence", f, x, history=h, presence=one[:1])
        bad("lens", f, x, history=h, presence=one, lens=i32(3))
        bad("prompt_lens", f, x, history=h, presence=one, prompt_lens=i32(2).long())
        bad("bias", f, x, bias=one[:, None])
        bad("bias", f, x, bias=one[:, None], bias_ids=h[:, :2])
        bad("allowed", f, x, allowed=i32(2, 3))
        bad("allowed", f, x, allowed=i32(1, 4))
        bad("allowed_rows", f, x, allowed_rows=i32(2))
        bad("allowed_rows", f, x, allowed=i32(1, 4), allowed_rows=i32(1))
        bad("vocab", f, x[:, :0])
    bad("out", K.adjust_logits, x, out=x.half())
    bad("out", K.adjust_logits, x, out=torch.zeros(100, 2, device="cuda").t())
    bad("overlap", K.adjust_logits, x.view(-1)[:100].view(1, 100), out=x.view(-1)[50:150].view(1, 100))
    bad("out", K.next_tokens, x, out=i32(2))
    bad("at most", K.next_tokens, torch.zeros(4097, 2, device="cuda"))
    with pytest.raises(L.SpectraError) as e:
        K.next_tokens(x, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    assert e.value.status == L.ERR_WORKSPACE
    for f in (lambda t: K.adjust_logits(t), lambda t: K.next_tokens(t)):
        with pytest.raises(ValueError, match="on the GPU"):
            f(torch.zeros(1, 4))


def _desc(**kw):
    d = dict(kind=L.KV_F16, kv_heads=2, head_dim=64, page_size=16, num_pages=4, k=0x10000, v=0x20000, page_stride=2 * 16 * 64,
             batch=2, table_width=3, block_table=0x30000, table_stride=3, kv_lens=0x31000, q_start=0x32000)
    d.update(kw)
    return L.PagedKv(**d)


def _refused(status, msg, want, text):
    assert status == want and text in msg.decode(), (status, msg)


@pytest.mark.parametrize("change,status,text", [
    (dict(), L.ERR_INVALID, "axes"), (dict(axes=5), L.ERR_INVALID, "axes"), (dict(axes=2, ldpos=1), L.ERR_INVALID, "stride"),
    (dict(axes=1, positions=0x50002), L.ERR_INVALID, "aligned"),
    (dict(axes=1, positions=0), L.ERR_INVALID, "NULL"), (dict(axes=1, axis=0), L.ERR_INVALID, "NULL"),
    (dict(axes=1, cos=0, sin=0), L.ERR_INVALID, "NULL"), (dict(axes=1, positions=0x90000), L.ERR_INVALID, "overlap"),
    (dict(axes=1, axis=0x90000), L.ERR_INVALID, "overlap")])
def test_axes_refusals(change, status, text):
    lib = L.load()
    a = dict(positions=0x50000, ldpos=3, axes=0, axis=0x60000, cos=0x70000, sin=0x80000)
    a.update(change)
    st = lib.spectra_paged_rope_axes_append(ctypes.byref(_desc()), 0xA0000, 8 * 64, 3, a["positions"], a["ldpos"], a["axes"],
                                            a["axis"], a["cos"], a["sin"], 50, 4, 0x90000, None)
    _refused(st, lib.spectra_last_error(), status, text)


@pytest.mark.parametrize("kv,bounds,text", [
    (dict(), dict(codes=0), "NULL"), (dict(), dict(scales=0), "NULL"), (dict(), dict(code_stride=200), "stride"),
    (dict(), dict(scale_stride=1), "stride"), (dict(), dict(codes=0x40008), "aligned"), (dict(), dict(code_stride=264), "aligned"),
    (dict(), dict(codes=0x10000), "overlap"), (dict(), dict(scales=0x31000), "overlap"), (dict(page_size=24), dict(), "power of two")])
def test_bounds_refusals(kv, bounds, text):
    lib = L.load()
    b = dict(codes=0x40000, code_stride=256, scales=0x50000, scale_stride=2)
    b.update(bounds)
    st = lib.spectra_paged_key_bounds(ctypes.byref(_desc(**kv)), 3, ctypes.byref(L.PagedBounds(**b)), None)
    _refused(st, lib.spectra_last_error(), L.ERR_INVALID, text)
    if not kv and "overlap" not in text:
        st = lib.spectra_paged_bounds_values(ctypes.byref(L.PagedBounds(**b)), 4, 2, 64, 0x90000, L.F16, None)
        _refused(st, lib.spectra_last_error(), L.ERR_INVALID, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(count=2), L.ERR_INVALID, "count"), (dict(local=0), L.ERR_INVALID, "count"), (dict(sink=-1), L.ERR_INVALID, "count"),
    (dict(sink=2147483647, local=2147483647, count=5), L.ERR_INVALID, "count"), (dict(dtype=L.F32), L.ERR_INVALID, "fp16"),
    (dict(q=0), L.ERR_INVALID, "NULL"), (dict(blocks=0), L.ERR_INVALID, "NULL"), (dict(q=0x90008), L.ERR_INVALID, "aligned"),
    (dict(ldq=250), L.ERR_INVALID, "stride"), (dict(blocks=0x90000), L.ERR_INVALID, "overlap"),
    (dict(blocks=0x40000), L.ERR_INVALID, "overlap"), (dict(ws=0x90000), L.ERR_INVALID, "overlap"), (dict(bytes=100, ws=0x1000000), L.ERR_WORKSPACE, "workspace"),
    (dict(ws=0x1000004), L.ERR_INVALID, "aligned"), (dict(kv=dict(table_width=32769, table_stride=32769)), L.ERR_UNSUPPORTED, "32768"),
    (dict(heads=1024, ldq=65536), L.ERR_UNSUPPORTED, "heads"), (dict(kv=dict(head_dim=96)), L.ERR_UNSUPPORTED, "head_dim")])
def test_select_refusals(change, status, text):
    lib = L.load()
    a = dict(q=0x90000, ldq=256, dtype=L.F16, heads=4, count=4, sink=1, local=2, ws=0, bytes=1 << 30, blocks=0xA0000, kv={})
    a.update(change)
    b = L.PagedBounds(0x40000, 256, 0x50000, 2)
    st = lib.spectra_paged_select(ctypes.byref(_desc(k=0, v=0, page_stride=0, **a["kv"])), ctypes.byref(b), a["q"], a["ldq"], a["dtype"], 3,
                                  a["heads"], a["count"], a["sink"], a["local"], a["ws"], a["bytes"], a["blocks"], None)
    _refused(st, lib.spectra_last_error(), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(q=0), L.ERR_INVALID, "NULL"), (dict(blocks=0), L.ERR_INVALID, "NULL"), (dict(count=0), L.ERR_INVALID, "count"),
    (dict(count=1 << 27), L.ERR_INVALID, "count"), (dict(scale=0.0), L.ERR_INVALID, "scale"), (dict(scale=math.nan), L.ERR_INVALID, "scale"),
    (dict(cap=-1.0), L.ERR_INVALID, "cap"), (dict(cap=math.inf), L.ERR_INVALID, "cap"), (dict(ws=0), L.ERR_WORKSPACE, "workspace"),
    (dict(bytes=1000), L.ERR_WORKSPACE, "workspace"), (dict(out=0x90000), L.ERR_INVALID, "overlap"), (dict(out=0xA0000), L.ERR_INVALID, "overlap"),
    (dict(out=0x20000), L.ERR_INVALID, "overlap"), (dict(out=0xB0008), L.ERR_INVALID, "aligned"), (dict(blocks=0xA0002), L.ERR_INVALID, "aligned"),
    (dict(ldq=8), L.ERR_INVALID, "stride")])
def test_blocks_refusals(change, status, text):
    lib = L.load()
    a = dict(q=0x90000, ldq=256, blocks=0xA0000, count=4, scale=0.1, cap=0.0, ws=0x1000000, bytes=1 << 30, out=0xB0000)
    a.update(change)
    st = lib.spectra_paged_attend_blocks(ctypes.byref(_desc()), a["q"], a["ldq"], 3, 4, a["blocks"], a["count"], a["scale"], a["cap"],
                                         a["ws"], a["bytes"], a["out"], None)
    _refused(st, lib.spectra_last_error(), status, text)


def test_refusals_of_more_tokens_than_are_counted():
    """Sizes are checked before they are multiplied: sums of bytes past 64 bits would pass for none."""
    lib = L.load()
    kv, b = _desc(k=0, v=0, page_stride=0, kv_heads=8), L.PagedBounds(0x40000, 8 * 128, 0x50000, 8)
    st = lib.spectra_paged_select(ctypes.byref(kv), ctypes.byref(b), 0x90000, 8 * 64, L.F16, 1 << 29, 8, 32768, 1, 2, 0, 0, 1 << 60, None)
    _refused(st, lib.spectra_last_error(), L.ERR_INVALID, "tokens")
    kv = _desc(kv_heads=8, page_stride=8 * 16 * 64)
    st = lib.spectra_paged_attend_blocks(ctypes.byref(kv), 0x90000, 8 * 64, 1 << 29, 8, 1 << 60, 1 << 25, 0.1, 0.0, 0x1000000, 1 << 30, 1 << 61, None)
    _refused(st, lib.spectra_last_error(), L.ERR_INVALID, "tokens")


@pytest.mark.parametrize("change,text", [
    (dict(logits=0), "NULL"), (dict(dtype=7), "dtype"), (dict(rows=0), "range"), (dict(vocab=0), "range"), (dict(ld=90), "stride"),
    (dict(repetition=0x20000), "history"), (dict(repetition=0x20000, history=0x30000, history_width=9, history_ld=5), "stride"),
    (dict(biases=3), "NULL"), (dict(biases=3, bias=0x40000, bias_ids=0x50000, bias_ld=2, bias_ids_ld=3), "stride"),
    (dict(allowed=0x60000, states=0), "stride"), (dict(allowed=0x60000, states=2, allowed_ld=3), "stride"),
    (dict(allowed=0x60000, states=1, allowed_ld=4), "mask"), (dict(logits=0x10001), "aligned"), (dict(state=0x70002), "aligned"),
    (dict(history=0x90010, history_width=2, history_ld=2, presence=0x20000), "overlap"), (dict(prompt_lens=0x90000), "overlap")])
def test_logits_refusals(change, text):
    lib = L.load()
    a = dict(logits=0x10000, ld=100, dtype=L.F16, rows=2, vocab=100)
    a.update(change)
    l = L.Logits(**a)
    _refused(lib.spectra_next_tokens(ctypes.byref(l), 0x90010, 0x1000000, 1 << 30, None) if "overlap" in text and "history" in change else
             lib.spectra_adjust_logits(ctypes.byref(l), 0x90000, 100, None), lib.spectra_last_error(), L.ERR_INVALID, text)


def test_logits_refuse_outputs():
    lib = L.load()
    l = L.Logits(logits=0x10000, ld=100, dtype=L.F16, rows=2, vocab=100)
    for out, ldo, text in ((0, 100, "out"), (0x90001, 100, "out"), (0x90000, 99, "stride"), (0x10002, 100, "overlap"), (0x10000, 120, "overlap")):
        _refused(lib.spectra_adjust_logits(ctypes.byref(l), out, ldo, None), lib.spectra_last_error(), L.ERR_INVALID, text)
    for out, ws, size, want in ((0, 0x1000000, 1 << 30, L.ERR_INVALID), (0x90004, 0x1000000, 1 << 30, L.ERR_INVALID), (0x90000, 0, 1 << 30, L.ERR_WORKSPACE),
                                (0x90000, 0x1000000, 16, L.ERR_WORKSPACE), (0x90000, 0x90000, 1 << 30, L.ERR_INVALID), (0x10000, 0x1000000, 1 << 30, L.ERR_INVALID)):
        assert lib.spectra_next_tokens(ctypes.byref(l), out, ws, size, None) == want
    many = L.Logits(logits=0x10000, ld=100, dtype=L.F16, rows=4097, vocab=100)
    assert lib.spectra_next_tokens(ctypes.byref(many), 0x90000, 0x1000000, 1 << 30, None) == L.ERR_INVALID


def test_registered_operators_have_shapes():
    """The operators' Meta kernels (what a compiler traces with)."""
    ops = L.load_torch_ops()
    m = dict(device="meta")
    q = torch.empty(5, 4, 64, dtype=torch.float16, **m)
    i32 = lambda *s: torch.empty(*s, dtype=torch.int32, **m)  # noqa: E731
    pages = [torch.empty(3, 2, 16, 64, dtype=torch.float16, **m)]
    codes, scales = torch.empty(3, 2, 2, 64, dtype=torch.int8, **m), torch.empty(3, 2, **m)
    where = i32(2), i32(3), i32(2, 4)
    tab = torch.empty(9, 32, **m)
    r = ops.paged_rope_axes_append(torch.empty(5, 8 * 64, dtype=torch.float16, **m), i32(3, 5), torch.empty(32, dtype=torch.uint8, **m), *where,
                                   tab, tab, 4, pages, pages)
    assert r.shape == q.shape
    ops.paged_key_bounds(5, *where, pages, codes, scales)
    assert ops.paged_bounds_values(codes, scales, L.BF16).dtype == torch.bfloat16
    s = ops.paged_select(q, *where, codes, scales, 16, 6, 1, 2, None)
    assert s.shape == (5, 2, 6) and s.dtype == torch.int32
    assert ops.paged_attend_blocks(q, s, *where, pages, pages, 0.1, 0.0, None).shape == q.shape
    x = torch.empty(4, 100, **m)
    assert ops.adjust_logits(x, *[None] * 10).shape == x.shape
    t = ops.next_tokens(x, *[None] * 11)
    assert t.shape == (4,) and t.dtype == torch.int64
    for bad in ([], [pages[0], pages[0]]):
        with pytest.raises(ValueError, match="k_pages"):
            ops.paged_key_bounds(5, *where, bad, codes, scales)
        with pytest.raises(ValueError, match="k_pages"):
            ops.paged_attend_blocks(q, s, *where, bad, bad, 0.1, 0.0, None)


@pytest.mark.gpu
def test_registered_operators(hip):
    """The registered operators give what the functions give, a whole-graph compilation traces them, and operands that
    gradients are asked of go to them."""
    from spectra_amd import kernels as K
    b, s = _session("fp16", 91)
    eager = [x.clone() for x in _step(b, s)]
    eager = [x.clone() for x in _step(b, s)]

    def functions(qkv, k, v, codes, scales):
        where = b.kv_lens, b.q_start, b.table
        q = K.paged_rope_axes_append(qkv, s["pos"], s["axis"], *where, s["cos"], s["sin"], 4, k, v)
        K.paged_key_bounds(b.tokens, *where, k, (codes, scales))
        blocks = K.paged_select(q, *where, (codes, scales), 16, 6)
        o = K.paged_attend_blocks(q, blocks, *where, k, v)
        x = K.adjust_logits(o.view(b.tokens, -1), bias_ids=s["history"], bias=s["history"].float())
        return blocks, o, x, K.next_tokens(x), K.paged_bounds_values((codes, scales))

    args = s["qkv"], b.k, b.v, *s["bounds"]
    plain = functions(*args)
    assert torch.equal(plain[0], eager[0]) and torch.equal(plain[1], eager[1])
    for x, y in zip(torch.compile(functions, backend="aot_eager", fullgraph=True)(*args), plain):
        assert torch.equal(x, y)
    ops = L.load_torch_ops()
    where = b.kv_lens, b.q_start, b.table
    q = torch.empty_like(b.q)
    ops.paged_rope_axes_append_out(s["qkv"], s["pos"], s["axis"], *where, s["cos"], s["sin"], 4, [b.k], [b.v], q)
    ops.paged_key_bounds(b.tokens, *where, [b.k], *s["bounds"])
    blocks = torch.empty_like(eager[0])
    ops.paged_select_out(q, *where, *s["bounds"], 16, 6, 1, 2, s["select"], blocks)
    assert torch.equal(blocks, eager[0])
    o = torch.empty_like(q)
    ops.paged_attend_blocks_out(q, blocks, *where, [b.k], [b.v], 0.125, 0.0, s["attend"], o)
    assert torch.equal(o, eager[1])
    logits = torch.randn(3, 500, device="cuda")
    kw = (s["history"], s["lens"], None, s["repetition"], None, None, None, None, s["allowed"], s["rows"])
    want = K.adjust_logits(logits, history=s["history"], lens=s["lens"], repetition=s["repetition"], allowed=s["allowed"], allowed_rows=s["rows"])
    out = torch.empty_like(logits)
    ops.adjust_logits_out(logits, *kw, out)
    tokens = torch.empty(3, dtype=torch.int64, device="cuda")
    ops.next_tokens_out(logits, *kw, s["next"], tokens)
    assert torch.equal(out, want) and torch.equal(tokens, K.next_tokens(want))
    assert torch.equal(ops.adjust_logits(logits, *kw), want)
    leaf = logits.clone().requires_grad_()
    got = K.adjust_logits(leaf, history=s["history"], lens=s["lens"], repetition=s["repetition"], allowed=s["allowed"], allowed_rows=s["rows"])
    assert got.requires_grad and torch.equal(got, want)
    over = logits.clone()
    ops.adjust_logits_(over, *kw)
    assert torch.equal(over, want)
    grad = K.paged_attend_blocks(b.q.clone().requires_grad_(), blocks, *where, b.k, b.v)
    assert grad.requires_grad and torch.equal(grad, K.paged_attend_blocks(b.q, blocks, *where, b.k, b.v))


# -- the paths of larger and rarer shapes ----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 9])
@pytest.mark.parametrize("levels", [1, 3, 300])
def test_select_ties_of_many(hip, n, levels):
    """More candidates than one wave holds, so many alike that no bound leaves few; more wanted than there are lanes."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [n], [16 * 1300 + 9], 4, 2, 64, 16, seed=48)
    bounds = _random_bounds(b, 12, levels)
    for count in (5, 70, 400, 700):
        got = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, bounds, 16, count, workspace=K.paged_select_workspace())
        _check_select(b, bounds, count, 1, 2, got)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 9])
def test_select_infinite_bounds_of_many(hip, n):
    """More pages come before all scores than are wanted."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [n], [16 * 900], 4, 2, 64, 16, seed=49)
    codes, scales = _random_bounds(b, 13)
    scales[::2] = math.inf
    got = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, (codes, scales), 16, 30)
    _check_select(b, (codes, scales), 30, 1, 2, got)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 9])
def test_select_scores_past_the_range(hip, n):
    """More scores past fp32's range than are wanted, the others below zero: they tie, whatever range their keys are
    counted in."""
    from spectra_amd import kernels as K
    b = Batch("bf16", [n], [16 * 1300], 2, 2, 64, 16, seed=50)
    codes, scales = _random_bounds(b, 16)
    b.q.zero_()
    b.q[..., 0] = 1.0
    codes[:, :, :, 0] = -100  # (of queries with one positive dim the scores are its codes', times 127)
    codes[::2, :, :, 0] = 127
    scales[::2] = 3e38
    for count in (5, 400, 600):
        got = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, (codes, scales), 16, count)
        _check_select(b, (codes, scales), count, 1, 2, got)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_many_sequences(hip, kind):
    """More sequences than a wave has lanes, some without tokens, pages apart in a larger pool."""
    from spectra_amd import kernels as K
    g = torch.Generator().manual_seed(6)
    lens = torch.randint(1, 400, (150,), generator=g).tolist()
    n = [min(m, x) for m, x in zip(lens, torch.randint(0, 3, (150,), generator=g).tolist())]
    b = Batch(kind, n, lens, 4, 2, 64, 16, seed=61, pages_apart=True)
    before = K.paged_bounds(b.k)
    bounds = K.paged_key_bounds(b.tokens, b.kv_lens, b.q_start, b.table, b.k, K.paged_bounds(b.k))
    _check_bounds(b, bounds, before)
    bounds = _random_bounds(b, 14)
    blocks = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, bounds, 16, 5)
    _check_select(b, bounds, 5, 1, 2, blocks)
    want, tol = _blocks_reference(b, blocks)
    _close(_attend(b, blocks), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_a_long_chunk(hip, kind):
    """Many tokens of one sequence beside single ones; their tiles are shared out unevenly."""
    from spectra_amd import kernels as K
    b = Batch(kind, [1, 300, 1], [2000, 700, 5], 6, 1, 128, 32, seed=62)
    bounds = _random_bounds(b, 15)
    blocks = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, bounds, 32, 7, sink=2, local=1)
    _check_select(b, bounds, 7, 2, 1, blocks)
    want, tol = _blocks_reference(b, blocks)
    _close(_attend(b, blocks), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_pages_gigabytes_apart(hip, kind):
    """Pages further apart than 32 bits of bytes: the same as side by side."""
    from spectra_amd import kernels as K
    b = Batch(kind, [1, 3], [90, 40], 4, 2, 64, 16, seed=63)
    pages = (b.k[0] if kind == "4bit" else b.k).shape[0]

    def far(t):
        step = (3 << 29) // t.element_size()
        room = torch.zeros((pages - 1) * step + t[0].numel(), dtype=t.dtype, device="cuda")
        x = room.as_strided(t.shape, (step, *t.stride()[1:]))
        x.copy_(t)
        return x

    near = K.paged_key_bounds(4, b.kv_lens, b.q_start, b.table, b.k, K.paged_bounds(b.k))
    blocks = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, near, 16, 4)
    want = _attend(b, blocks)
    k, v = [tuple(far(t) for t in c) if kind == "4bit" else far(c) for c in (b.k, b.v)]
    bounds = far(near[0]).zero_(), far(near[1]).zero_()
    K.paged_key_bounds(4, b.kv_lens, b.q_start, b.table, k, bounds)
    assert torch.equal(bounds[0], near[0]) and torch.equal(bounds[1], near[1])
    assert torch.equal(K.paged_bounds_values(bounds), K.paged_bounds_values(near))
    assert torch.equal(K.paged_select(b.q, b.kv_lens, b.q_start, b.table, bounds, 16, 4), blocks)
    assert torch.equal(K.paged_attend_blocks(b.q, blocks, b.kv_lens, b.q_start, b.table, k, v), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(2, 3001), (300, 700)])
def test_logits_of_long_histories(hip, rows, vocab):
    """Histories and lists of biases whose counts and places need more than 16 bits."""
    x, kw = _case(rows, vocab, torch.float16, 65, history=40000 if rows == 2 else 33000)
    kw["history"][:, : 32800] = 3  # one token, more often than 15 bits hold
    kw["lens"].fill_(32900)
    kw["prompt_lens"].fill_(5)
    _check_logits(x, kw)
    if rows == 2:
        x, kw = _case(rows, vocab, torch.float32, 66, history=10, biases=70000)
        _check_logits(x, kw)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 300, 6000, 32767, 32768])
def test_select_the_largest_tables(hip, count):
    """32768 pages a sequence, as many as a selection takes; all of them, all but one, and few."""
    from spectra_amd import kernels as K
    n, pages = 32768, 500
    g = _gen(68)
    q = torch.randn(2, 4, 128, generator=g, device="cuda").half()
    codes = torch.randint(-30, 128, (pages, 1, 2, 128), generator=g, device="cuda", dtype=torch.int8)
    codes[:, :, 1] = -codes[:, :, 1]
    scales = torch.rand(pages, 1, generator=g, device="cuda") + 0.1
    table = torch.randint(0, pages, (1, n), generator=g, device="cuda", dtype=torch.int32)  # the pages again and again
    lens, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([16 * n], [0, 2]))
    got = K.paged_select(q, lens, starts, table, (codes, scales), 16, count, sink=0, local=1)
    c, s, t = codes.cpu().numpy(), scales.cpu().numpy(), table.cpu().numpy()
    for i in range(2):
        assert got[i, 0].tolist() == _selected(q[i], c[:, 0], s[:, 0], t[0], n, count, 0, 1)
    assert torch.equal(got, K.paged_select(q, lens, starts, table, (codes, scales), 16, count, sink=0, local=1,
                                           workspace=K.paged_select_workspace()))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [256, 2048])
def test_large_pages(hip, kind, page):
    """Pages of more rows than a wave or a step takes at once."""
    from spectra_amd import kernels as K
    b = Batch(kind, [1, 3], [5 * page - 7, page + 130], 4, 2, 128, page, seed=69)
    before = K.paged_bounds(b.k)
    _check_bounds(b, K.paged_key_bounds(b.tokens, b.kv_lens, b.q_start, b.table, b.k, K.paged_bounds(b.k)), before)
    bounds = _random_bounds(b, 17)
    blocks = K.paged_select(b.q, b.kv_lens, b.q_start, b.table, bounds, page, 3)
    _check_select(b, bounds, 3, 1, 2, blocks)
    want, tol = _blocks_reference(b, blocks)
    _close(_attend(b, blocks), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,page", [(6, 16), (16, 64), (2, 32), (18, 16)])
@pytest.mark.parametrize("cap", [0.0, 20.0, 1e6])
def test_blocks_of_4_bits_and_64_dims_in_numbers(hip, heads, page, cap):
    """As many steps that workgroups have several each: two tiles' scores share the registers of one, up to 8 heads a KV
    head.  Rows that no sequence has hold NaN; a page that is not there makes the rows that see it NaN, and no others."""
    b = Batch("4bit", [5, 40, 3], [3900, 900, 3001], heads, 2, 64, page, seed=70)
    blocks = _random_blocks(b, 2560 // page, 8)
    blocks[7:11] = -1
    blocks[8, :, 5] = 0  # a row with 17 keys of two tiles, one with 16, rows without
    blocks[8, :, 9], blocks[9, :, 0] = 874 // page, 0
    want, tol = _blocks_reference(b, blocks, cap=cap)
    got = _attend(b, blocks, cap=cap)
    _close(got, want, tol)
    assert (got[7] == 0).all() and (got[10] == 0).all()
    last = (blocks[45:] * page).clamp(min=0) + 15  # the third sequence loses a page
    gone = int(blocks[46, 0][blocks[46, 0] > 3].min())
    b.table[2, gone] = -5
    sees = ((blocks[45:] == gone) & (last <= 3000)).any(-1).repeat_interleave(heads // 2, 1)
    bad = _attend(b, blocks, cap=cap)
    assert torch.isnan(bad[45:][sees]).all() and torch.equal(bad[45:][~sees], got[45:][~sees]) and torch.equal(bad[:45], got[:45])


@pytest.mark.gpu
def test_larger_calls_captured(hip):
    """Many drafts on 4-bit pages of 64 dims, a long table split among workgroups, a batch's logits in large slices: each
    replay of a captured graph, with eager calls of other shapes on the same workspaces between them, is the eager call's."""
    from spectra_amd import kernels as K
    b = Batch("4bit", [5, 40, 3], [3900, 900, 3001], 6, 2, 64, 16, seed=72)
    blocks = _random_blocks(b, 160, 9)
    long = Batch("bf16", [1], [16 * 8100 + 3], 8, 2, 64, 16, seed=73)
    bounds = _random_bounds(long, 18)
    x, kw = _case(40, 40003, torch.float16, 74, history=3001, biases=40, masks=3)
    small, few = _case(3, 500, torch.float16, 75, history=20)
    at, sel, nx = K.paged_attend_workspace(64), K.paged_select_workspace(), K.next_tokens_workspace()

    def calls():
        return (_attend(b, blocks, workspace=at, cap=9.0), K.paged_select(long.q, long.kv_lens, long.q_start, long.table, bounds, 16, 60, workspace=sel),
                K.next_tokens(x, workspace=nx, **kw), K.adjust_logits(x, **kw))

    want = calls()
    _check_select(long, bounds, 60, 1, 2, want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        calls()
        with torch.cuda.graph(graph, stream=side):
            got = calls()
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(4):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g.nan_to_num(), w.nan_to_num()) for g, w in zip(got, want))
        _check_logits(small, few, nx)
        K.paged_attend_blocks(b.q[:5], blocks[:5, :, :3].contiguous(), b.kv_lens[:1], b.q_start[:2], b.table[:1], b.k, b.v, workspace=at)
        K.paged_select(long.q, torch.full_like(long.kv_lens, 16 * 1100), long.q_start, long.table, bounds, 16, 5, workspace=sel)


def _one_token(b, s, t, row, blocks, cap):
    """The output [heads, d] of token t of sequence s (row `row` of the call) and its tolerance, whose keys may score infinities."""
    u, sub = torch.finfo(_DT[b.kind]).eps / 2, 2.0 ** -25 if b.kind != "bf16" else 0.0
    k, v = b.rows(s)
    out, tol = [], []
    for h in range(b.heads):
        kv = h * b.kv // b.heads
        j = torch.cat([torch.arange(x * b.page, (x + 1) * b.page) for x in blocks[row, kv].tolist() if x >= 0]).cuda()
        j = j[j <= b.lens[s] - b.n[s] + t]
        kk, vv = k[kv, j], v[kv, j]
        q = b.q[row, h].double()
        x = (kk * q).sum(-1) / math.sqrt(b.d)
        size = (kk * q).abs().sum(-1) / math.sqrt(b.d)
        delta = b.d * 2.0 ** -24 * size[torch.isfinite(size)].max()
        if cap:
            x, delta = cap * torch.tanh(x / cap), delta + cap * 2.0 ** -20
        e = torch.exp(x - x.max())
        p = e / e.sum()
        o, a = (p[:, None] * vv).sum(0), (p[:, None] * vv.abs()).sum(0)
        out.append(o)
        tol.append(u * o.abs() + (u + 2 * delta + 2.0 ** -20) * a + sub * (1 + vv.abs().sum(0) / e.sum()))
    return torch.stack(out), torch.stack(tol)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,d", [(2, 2, 64), (12, 2, 64), (18, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("what", ["values", "keys above", "keys below"])
def test_blocks_of_4_bits_with_infinite_scales(hip, heads, kv, d, cap, what):
    """A row that sees an infinite scale has what the formula gives, in a batch whose workgroups have many tiles and alone:
    infinite values are infinite in their dims, a score of -inf weighs nothing, one of +inf is NaN (with a cap: the cap)."""
    from spectra_amd import kernels as K
    b = Batch("4bit", [5, 40, 3], [3900, 900, 3001], heads, kv, d, 16, seed=76)
    blocks = _random_blocks(b, 160, 10, holes=False)
    before = _attend(b, blocks, cap=cap)
    page, row = 50, 7  # key 807 of the third sequence, which its second token lists in every KV head
    blocks[46, :, 3] = torch.where((blocks[46] == page).any(-1), blocks[46, :, 3], page)
    blocks[45], blocks[47] = torch.where(blocks[45] == page, -1, blocks[45]), torch.where(blocks[47] == page, -1, blocks[47])
    at = b.table[2, page].long()
    codes, scales, zeros = b.v if what == "values" else b.k
    codes[at, :, row, :16] = 0x5A
    zeros[at, :, row, 0] = 7 if what == "values" else 2
    scales[at, :, row, 0] = math.inf
    if what != "values":
        b.q[46, :, :32] = b.q[46, :, :32].abs().clamp(min=0.01) * (1 if what == "keys above" else -1)
    got = _attend(b, blocks, cap=cap)
    want, tol = _one_token(b, 2, 1, 46, blocks, cap)
    alone = K.paged_attend_blocks(b.q[46:47], blocks[46:47], torch.tensor([3000], dtype=torch.int32, device="cuda"), b.q_start.new_tensor([0, 1]),
                                  b.table[2:], b.k, b.v, cap=cap)
    finite = torch.isfinite(want)
    assert finite.all(-1).all() == (what == "keys below" or (what == "keys above" and cap > 0))
    for x in (got[46], alone[0]):
        assert torch.equal(torch.isnan(x), torch.isnan(want))
        assert torch.equal(torch.isposinf(x), torch.isposinf(want)) and torch.equal(torch.isneginf(x), torch.isneginf(want))
        err = (x.double() - want).abs()
        assert (err <= tol)[finite].all(), float((err - tol)[finite].max())
    assert torch.equal(got[:45], before[:45])


@pytest.mark.gpu
def test_scores_bound_products_of_rounded_queries(hip):
    """A block's score is at least the product of each rounded query with each of its keys; a dim below half a step of the
    queries' scale counts nothing, however large the keys are in it."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [1], [400], 6, 2, 64, 16, seed=77)
    codes, scales = K.paged_key_bounds(400, b.kv_lens, b.q_start.new_tensor([0, 400]), b.table, b.k, K.paged_bounds(b.k))
    k, _ = b.rows(0)
    for h in range(2):
        q = b.q[0, 3 * h: 3 * h + 3].float()
        c = torch.round(q * (127 / q.abs().max())).double()
        for j in range(25):
            page = b.table[0, j].long()
            hi, lo = codes[page, h].double()
            score = float(scales[page, h]) * float((c.clamp(min=0) @ hi + c.clamp(max=0) @ lo).max())
            assert float((c @ k[h, 16 * j: 16 * j + 16].T).max()) <= score + 127 * 2.0 ** -22 * float(scales[page, h]) * float(c.abs().sum(-1).max())
    one = Batch("fp16", [1], [80], 1, 1, 64, 16, seed=78)
    one.q.zero_()
    one.q[0, 0, 0], one.q[0, 0, 1] = 127.0, 0.4
    one.k.zero_()
    one.k[one.table[0, 1].long(), 0, 5, 1] = 100.0  # a product of 40, a score of 0
    one.k[one.table[0, 2].long(), 0, 5, 0] = 0.01   # of 1.27, and a score as large
    bounds = K.paged_key_bounds(80, one.kv_lens, one.q_start.new_tensor([0, 80]), one.table, one.k, K.paged_bounds(one.k))
    got = K.paged_select(one.q, one.kv_lens, one.q_start, one.table, bounds, 16, 3, sink=1, local=1)
    assert got[0, 0].tolist() == [0, 2, 4]


@pytest.mark.gpu
def test_calls_that_meet_in_workspaces_on_two_streams(hip):
    """A selection split among workgroups, lists whose tiles are cut, choices over small and over large slices, on two streams
    at once, each with workspaces of its own: what each gives alone."""
    from spectra_amd import kernels as K
    sides = []
    for i in range(2):
        long = Batch("bf16", [1, 1], [16 * 1100 + 3, 16 * 1300], 4, 2, 64, 16, seed=91 + i)
        near = Batch("fp16", [1, 3], [1500, 1400], 8, 2, 64, 16, seed=93 + i)
        sides.append(dict(long=long, bounds=_random_bounds(long, 95 + i), near=near, lists=_random_blocks(near, 80, 11 + i, holes=False),
                          small=_case(3, 7001, torch.float16, 97 + i, history=50, masks=2),
                          large=_case(40, 40003, torch.float32, 99 + i, history=3001, biases=20),
                          select=K.paged_select_workspace(), attend=K.paged_attend_workspace(64), next=K.next_tokens_workspace(),
                          busy=torch.randn(4096, 4096, device="cuda", dtype=torch.float16)))

    def calls(s):
        long, near = s["long"], s["near"]
        return (K.paged_select(long.q, long.kv_lens, long.q_start, long.table, s["bounds"], 16, 70, workspace=s["select"]),
                _attend(near, s["lists"], workspace=s["attend"]),
                *[K.next_tokens(x, workspace=s["next"], **kw) for x, kw in (s["small"], s["large"])])

    wants = [calls(s) for s in sides]
    torch.cuda.synchronize()
    for s, want in zip(sides, wants):
        _check_select(s["long"], s["bounds"], 70, 1, 2, want[0])
        _close(want[1], *_blocks_reference(s["near"], s["lists"]))
        for (x, kw), t in zip((s["small"], s["large"]), want[2:]):
            assert torch.equal(t.cpu(), _picked(_adjusted(x, **kw)))
        assert s["select"][16384:].any() and s["attend"][16384:].any()  # (partial results have met there)
    assert not any(torch.equal(x, y) for x, y in zip(*wants))
    streams, outs = [torch.cuda.Stream() for _ in range(2)], ([], [])
    for st, s in zip(streams, sides):  # (work that the calls of both queue up behind)
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _ in range(4):
                s["busy"] @ s["busy"]
    for _ in range(25):
        for st, s, out in zip(streams, sides, outs):
            with torch.cuda.stream(st):
                out.append(calls(s))
    torch.cuda.synchronize()
    for want, out in zip(wants, outs):
        assert all(torch.equal(x, y) for one in out for x, y in zip(one, want))
    for s in sides:
        assert not s["select"][:16384].any() and not s["attend"][:16384].any() and not s["next"].any()


@pytest.mark.gpu
def test_clamped_starts_reach_only_what_they_name(hip):
    """Starts that are no batch's are clamped to the call's tokens (a start below the one before it: no tokens).  Bounds are
    worked out for the pages that they then name, and for no others; a selection leaves rows behind the last start alone."""
    from spectra_amd import kernels as K
    b = Batch("fp16", [40, 30], [40, 30], 2, 1, 64, 16, seed=79)
    for starts, touched in (([0, 0, 0], ()), ([50, 20, 10], ()), ([70, 70, 70], ()), ([-5, 1000, 3], (0,)), ([0, 1, 1], (0,))):
        # sequence 0 with all of the call's tokens, or one; its pages from the first of its tokens on
        bad = b.q_start.new_tensor(starts)
        codes, scales = K.paged_bounds(b.k)
        codes.fill_(3)
        scales.fill_(5.0)
        want = codes.clone(), scales.clone()
        K.paged_key_bounds(b.tokens, b.kv_lens, bad, b.table, b.k, (codes, scales))
        for s in touched:
            first = 0 if starts[1] > 1 else 39
            for j in range(first // 16, 3):
                page = int(b.table[s, j])
                c, a = _bounds_of(b.k[page, 0, : min(16, 40 - 16 * j)])
                want[0][page, 0], want[1][page, 0] = torch.from_numpy(c).cuda(), float(a)
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1]), starts
    b = Batch("fp16", [2, 1], [400, 90], 4, 2, 64, 16, seed=80)
    bounds = _random_bounds(b, 19)
    for starts in ([0, 0, 0], [2, 1, 1], [0, 1, 1], [-5, 1, 2], [0, 2, 2]):
        out = torch.full((3, 2, 4), 77, dtype=torch.int32, device="cuda")
        K.paged_select(b.q, b.kv_lens, b.q_start.new_tensor(starts), b.table, bounds, 16, 4, out=out)
        last = max(starts[-1], 0)
        assert (out[last:] == 77).all() and not (out[:last] == 77).any(), starts


@pytest.mark.gpu
@pytest.mark.parametrize("g", [3, 6])
@pytest.mark.parametrize("width", [9000, 10000, 32768])
def test_select_chunks_on_wide_tables(hip, g, width):
    """Tokens beside each other on tables so wide that their keys do not fit: groups of fewer tokens than a tile holds, or one,
    with their pages split among workgroups or not."""
    from spectra_amd import kernels as K
    n, pages, d = 9, 700, 64
    gen = _gen(82)
    q = torch.randn(n, g, d, generator=gen, device="cuda").half()
    codes = torch.randint(-30, 128, (pages, 1, 2, d), generator=gen, device="cuda", dtype=torch.int8)
    codes[:, :, 1] = -codes[:, :, 1]
    scales = torch.rand(pages, 1, generator=gen, device="cuda") + 0.1
    table = torch.randint(0, pages, (1, width), generator=gen, device="cuda", dtype=torch.int32)  # the pages again and again
    last = 16 * (width - 1) + 4  # (the tokens' own page changes after the fifth)
    lens, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([last], [0, n]))
    c, s, t = codes.cpu().numpy(), scales.cpu().numpy(), table.cpu().numpy()
    for count in (40, 300):
        got = K.paged_select(q, lens, starts, table, (codes, scales), 16, count)
        assert torch.equal(got, K.paged_select(q, lens, starts, table, (codes, scales), 16, count, workspace=K.paged_select_workspace()))
        for i in range(n) if width < 32768 else (0, 4, 5, 8):
            want = _selected(q[i], c[:, 0], s[:, 0], t[0], (last - n + i) // 16 + 1, count, 1, 2)
            assert got[i, 0].tolist() == want, (count, i)


@pytest.mark.parametrize("heads,d,width", [(97, 128, 32768), (209, 64, 32768), (257, 128, 16), (257, 64, 1)])
def test_select_refuses_more_heads_than_fit(heads, d, width):
    """Query heads a KV head: 256, and 96 of 128 dims or 208 of 64 beside a table of 32768 pages."""
    lib = L.load()
    kv = _desc(k=0, v=0, page_stride=0, kv_heads=1, head_dim=d, table_width=width, table_stride=width)
    b = L.PagedBounds(0x40000, 2 * d, 0x50000, 1)
    st = lib.spectra_paged_select(ctypes.byref(kv), ctypes.byref(b), 0x100000, heads * d, L.F16, 3, heads, 4, 1, 2, 0, 0, 0x200000, None)
    _refused(st, lib.spectra_last_error(), L.ERR_UNSUPPORTED, "heads")


@pytest.mark.gpu
@pytest.mark.parametrize("heads,d,width", [(96, 128, 32768), (208, 64, 32768), (256, 128, 100), (256, 64, 100)])
def test_select_with_the_most_heads(hip, heads, d, width):
    from spectra_amd import kernels as K
    gen = _gen(83)
    q = torch.randn(1, heads, d, generator=gen, device="cuda").half()
    codes = torch.randint(-30, 128, (300, 1, 2, d), generator=gen, device="cuda", dtype=torch.int8)
    codes[:, :, 1] = -codes[:, :, 1]
    scales = torch.rand(300, 1, generator=gen, device="cuda") + 0.1
    table = torch.randint(0, 300, (1, width), generator=gen, device="cuda", dtype=torch.int32)
    lens, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([16 * width], [0, 1]))
    want = _selected(q[0], codes[:, 0].cpu().numpy(), scales[:, 0].cpu().numpy(), table[0].cpu().numpy(), width, 20, 1, 2)
    for ws in (None, K.paged_select_workspace()):
        assert K.paged_select(q, lens, starts, table, (codes, scales), 16, 20, workspace=ws)[0, 0].tolist() == want


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(40, 40003), (3, 40003)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_logits_in_place_of_large_and_small_slices(hip, dtype, rows, vocab):
    """Logits that are their own output, adjusted tokens spread over all slices."""
    from spectra_amd import kernels as K
    x, kw = _case(rows, vocab, dtype, 84, history=3001, biases=1100, masks=3)
    want = K.adjust_logits(x, **kw)
    for _ in range(3):
        mine = x.clone()
        assert K.adjust_logits(mine, **kw, out=mine) is mine and torch.equal(_bits(mine), _bits(want))
