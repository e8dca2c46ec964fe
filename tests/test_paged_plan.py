"""How the paged attention's work is shared out, on the CPU: the kernels' own plans, compiled for the host, cover every key
step of every tile once and give partial sums records of their own (tests/paged_plan.cpp), up to the batches and lines
whose sums leave 32 bits."""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F16, Q4 = 0, 2


@pytest.fixture(scope="session")
def program(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("plan") / "paged_plan")
    r = subprocess.run([shutil.which("hipcc") or "/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only",
                        "--offload-arch=gfx950", "-O2", "-std=c++17", "-w", f"-I{ROOT}/spectra_amd/csrc", f"-I{ROOT}/include",
                        os.path.join(ROOT, "tests", "paged_plan.cpp"), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return exe


@pytest.fixture(scope="session")
def plan(program):
    def run(n, lens, heads=8, kv_heads=8, d=64, page=64, kind=F16, width=0, pad=0, window=0, prefix=None):
        """``width``: pages a sequence that the table holds (0: what the longest needs)."""
        head = f"{kind} {heads} {kv_heads} {d} {page} {width} {len(n)} {pad} {window}\n"
        rows = "\n".join(f"{a} {b} {-1 if prefix is None else prefix[i]}" for i, (a, b) in enumerate(zip(n, lens)))
        r = subprocess.run([program], input=head + rows + "\n", capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stdout + r.stderr
        return r.stdout

    return run


def test_regions_that_meet(program):
    """Which operands share memory, runs with gaps between them included (what lies between pages is not the pool's)."""
    r = subprocess.run([program, "7"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout


# sums of padded steps of exactly 2^32, of a little more, and past it without a wrap to something small
@pytest.mark.parametrize("batch,kv_heads,lo,hi,kind", [
    (16384, 32, 897, 1024, F16), (65536, 8, 1024, 1024, F16), (8192, 32, 4096, 4096, Q4), (262144, 8, 128, 128, F16),
    (65536, 8, 900, 1100, Q4), (20000, 31, 1, 1500, F16), (1 << 20, 1, 1, 200, Q4)])
def test_large_batches(plan, batch, kv_heads, lo, hi, kind):
    r = random.Random(batch + kv_heads)
    out = plan([1] * batch, [r.randint(lo, hi) for _ in range(batch)], heads=kv_heads, kv_heads=kv_heads, kind=kind)
    assert f"ok few: {batch * kv_heads} tiles" in out


@pytest.mark.parametrize("lens", [[(1 << 29) + 5] * 64, [(1 << 29) - 1, 3, 1 << 20] * 30, [1 << 28] + [100] * 70])
@pytest.mark.parametrize("kv_heads", [4, 8])
def test_lines_past_32_bits(plan, lens, kv_heads):
    """Tables so wide that the line is counted in steps of several steps; the lengths may be shorter."""
    kw = dict(heads=2 * kv_heads, kv_heads=kv_heads, page=65536, width=(1 << 13) + 1)
    assert "(wide)" in plan([1] * len(lens), lens, **kw)
    assert "(wide)" in plan([1, 3] * (len(lens) // 2) + [2] * (len(lens) % 2), [m // 4096 + 3 for m in lens], kind=Q4, **kw)
    plan([1] * len(lens), lens, window=48, **kw)
    plan([1] * len(lens), lens, window=48, prefix=[0] * len(lens), **kw)


@pytest.mark.parametrize("batch,chunk,kv_heads", [(33, 1800, 64), (129, 2600, 32), (3000, 30, 32), (64, 900, 8)])
@pytest.mark.parametrize("prefix", [False, True])
def test_many_tiles_of_long_caches(plan, batch, chunk, kv_heads, prefix):
    """So much work that a share of it has more steps than any tile: none is cut, and none is lost."""
    r = random.Random(batch)
    lens = [r.randint(1 << 28, (1 << 30) - 70000) for _ in range(batch)]
    out = plan([chunk - b % 7 for b in range(batch)], lens, heads=6 * kv_heads, kv_heads=kv_heads, page=4096,
               window=300 if prefix else 0, prefix=[0] * batch if prefix else None)
    assert "ok many" in out


@pytest.mark.parametrize("seed", range(40))
def test_ragged_batches(plan, seed):
    r = random.Random(seed)
    batch = r.choice([1, 2, 7, 63, 64, 65, 130, 300])
    kv_heads, g = r.choice([1, 2, 8, 16]), r.choice([1, 3, 4, 7, 16, 33])
    hi = r.choice([1, 1, 2, 5, 16, 100, 700] if batch < 100 else [1, 1, 4])
    n = [r.randint(0 if r.random() < 0.2 else 1, hi) for _ in range(batch)]
    n[0] = max(n[0], 1)
    ctx = r.choice([0, 3, 200, 5000, 100000])
    lens = [max(0, m + r.randint(-2 if r.random() < 0.1 else 0, ctx)) for m in n]
    page = r.choice([16, 64, 128])
    kw = dict(heads=g * kv_heads, kv_heads=kv_heads, d=r.choice([64, 128]), page=page, kind=r.choice([0, 1, 2]),
              pad=r.choice([0, 0, 5]), window=r.choice([0, 0, 1, 100, 3000]))
    if r.random() < 0.3:
        kw["prefix"] = [r.choice([0, 10, 10 ** 6]) for _ in n]
    kw["width"] = r.choice([0, 0, max(lens) // page + 9, max(1, max(lens) // page // 2)])
    if max(lens) == 0:
        kw["width"] = 1
    assert "ok" in plan(n, lens, **kw)
