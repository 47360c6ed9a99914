"""The paged key/value operators (mocha_kv.h through mocha_kv.py) on a B200 against their
formulas in 64 bits (kv_reference.py derives the bounds)."""
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEV = "cuda:0"


@pytest.fixture(scope="module")
def kv(native):
    import mocha_kv
    return mocha_kv


def pool(lens, kv_heads, dim, page, dtype, by_token=False, seed=0, spare=2, fill=float("nan")):
    """(k, v, table): pages in random order; every row of a page that no sequence holds is `fill`."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    count = sum(need) + spare
    ids = torch.randperm(count, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(max(need), 1)
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    kvs = []
    for _ in range(2):
        shape = (count, page, kv_heads, dim) if by_token else (count, kv_heads, page, dim)
        t = torch.full(shape, fill, device=DEV, dtype=dtype)
        kvs.append(t.transpose(1, 2) if by_token else t)
    at = 0
    for s, n in enumerate(lens):
        for i in range(need[s]):
            table[s, i] = ids[at]
            rows = min(page, n - i * page)
            for t in kvs:
                t[ids[at], :, :rows] = torch.randn(kv_heads, rows, dim, device=DEV, generator=g).to(dtype)
            at += 1
    return kvs[0], kvs[1], table.to(DEV)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def queries(rows, heads, dim, dtype, seed=1, scale=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(rows, heads, dim, device=DEV, generator=g) * scale).to(dtype)


def close(got, want, tol, name=""):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((err / tol.clamp_min(1e-300))[bad].max()), bad.nonzero()[0].tolist())


def check(kv, lens, qlens, heads, kv_heads, dim, page, dtype, window=0, prefix=None, cap=0.0, slopes=False, by_token=False,
          scale=None, seed=0, run=None):
    """decode (qlens None) or prefill of random data, out and lse, against the formula."""
    k, v, table = pool(lens, kv_heads, dim, page, dtype, by_token, seed)
    cache = kv.KvPages(k, v)
    prefill = qlens is not None
    counts = qlens if prefill else [1] * len(lens)
    rows = sum(counts)
    q = queries(rows, heads, dim, dtype, seed + 1)
    sl = (2.0 ** (-4.0 * (torch.arange(heads, device=DEV) + 1) / heads)).float() if slopes else None
    pre = None if prefix is None else ints(prefix)
    lse = torch.full((rows, heads), 5.0, device=DEV)
    out = torch.full((rows, heads, dim), 7.0, device=DEV, dtype=dtype)
    more = dict(window=window, prefix=pre, cap=cap, slopes=sl, scale=scale, lse=lse, out=out)
    start = np.concatenate([[0], np.cumsum(counts)]).astype(int).tolist()
    if prefill:
        cache.prefill(q, ints(start), table, ints(lens), **more)
    else:
        cache.decode(q, table, ints(lens), **more)
    torch.cuda.synchronize()
    for s, n in enumerate(lens):
        a, b = start[s], start[s + 1]
        p = [n - (b - a) + i for i in range(b - a)]
        want, wl, tol, tol_l = ref.attend(q[a:b], ref.gather(k, table, s, n), ref.gather(v, table, s, n), p,
                                          dim ** -0.5 if scale is None else scale, window,
                                          0 if prefix is None else min(prefix[s], n), cap, sl, dtype)
        close(out[a:b], want, tol, f"sequence {s}")
        none = torch.isinf(wl)
        assert torch.equal(torch.isinf(lse[a:b]), none)
        close(lse[a:b][~none], wl[~none], tol_l[~none], f"lse {s}")
    return k, v, table, q, out


# ---- append ----------------------------------------------------------------------------

@pytest.mark.parametrize("tin", [F32, F16, BF16])
@pytest.mark.parametrize("tout", [F32, F16, BF16])
@pytest.mark.parametrize("dim,dims,interleaved,by_token,page", [
    (64, 64, False, False, 16), (128, 128, True, True, 24), (96, 32, False, True, 8), (32, 16, True, False, 64),
    (128, 0, False, False, 8),
])
def test_append(kv, tin, tout, dim, dims, interleaved, by_token, page):
    heads, kvh = 6, 2
    lens = [1, 37, 130]
    k, v, table = pool(lens, kvh, dim, page, tout, by_token, seed=3)
    k0, v0 = k.clone(), v.clone()
    # every position of sequence 2 in reverse, one of each other, two skipped rows
    where = [(2, p) for p in range(129, -1, -1)] + [(-1, 5), (0, 0), (1, 36), (7, 0), (0, -1)]
    rows = len(where)
    fused = queries(rows, heads + 2 * kvh, dim, tin, seed=4)
    q, kn, vn = fused.split([heads, kvh, kvh], 1)
    angle = torch.arange(200, device=DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(max(dims, 16) // 2, device=DEV) / 16.0)
    cos, sin = angle.cos().float(), angle.sin().float()
    q_out = torch.full((rows, heads, dim), 9.0, device=DEV, dtype=tout)
    kv.KvPages(k, v).append(q, kn, vn, ints([s for s, _ in where]), ints([p for _, p in where]), table,
                            cos=cos if dims else None, sin=sin if dims else None, interleaved=interleaved, q_out=q_out)
    torch.cuda.synchronize()
    pos = torch.tensor([max(p, 0) for _, p in where])
    turn = [ref.rotate(x, cos[pos][:, :dims // 2], sin[pos][:, :dims // 2], interleaved) for x in (q, kn)]
    u = ref.unit(tout)
    tiny = torch.finfo(tout).tiny
    for i, (s, p) in enumerate(where):
        if not 0 <= s < 3 or p < 0:
            assert (q_out[i] == 9.0).all()
            continue
        page_id, row = int(table[s, p // page]), p % page
        close(q_out[i], turn[0][0][i], u * turn[0][0][i].abs() + (1 + u) * turn[0][1][i] + tiny)
        close(k[page_id, :, row], turn[1][0][i], u * turn[1][0][i].abs() + (1 + u) * turn[1][1][i] + tiny)
        assert torch.equal(v[page_id, :, row], vn[i].to(tout))
        for new, old in ((k, k0), (v, v0)):
            new[page_id, :, row] = old[page_id, :, row]
    for new, old in ((k, k0), (v, v0)):  # nothing else was written
        assert torch.equal(torch.nan_to_num(new.float(), 123.0), torch.nan_to_num(old.float(), 123.0))


def test_append_in_place_without_queries_and_status(kv):
    k, v, table = pool([40], 2, 64, 16, F32)
    cache = kv.KvPages(k, v)
    angle = torch.arange(64, device=DEV)[:, None] * torch.linspace(1, 0.1, 32, device=DEV)
    cos, sin = angle.cos(), angle.sin()
    q = queries(3, 4, 64, F32)
    want = ref.rotate(q, cos[[3, 4, 5]], sin[[3, 4, 5]], False)
    new = queries(3, 2, 64, F32, 5)
    cache.append(q, new, new, ints([0] * 3), ints([3, 4, 5]), table, cos=cos, sin=sin, q_out=q)
    close(q, want[0], want[0].abs() * 2.0 ** -24 + 1.001 * want[1] + 1e-38)
    before = k.clone()
    status = ints([0])
    cache.append(None, new[:0], new[:0], ints([]), ints([]), table, status=status)
    cache.append(None, new[:1], new[:1], ints([0]), ints([6]), table, status=status)
    assert int(status) == 0
    got = k.clone()
    # position 48 lies past the table, 63 past nothing but the table too; page -7 past the pool
    cache.append(None, new[:2], new[:2], ints([0, 0]), ints([48, 64]), table, status=status)
    assert int(status) == 1
    status.zero_()
    table[0, 2] = 1000
    cache.append(None, new[:1], new[:1], ints([0]), ints([33]), table, status=status)
    assert int(status) == 1
    status.zero_()
    cache.append(None, new[:1], new[:1], ints([0]), ints([5]), table, cos=cos[:5], sin=sin[:5], status=status)
    assert int(status) == 1  # the angles end at position 4
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(k))
    page = int(table[0, 0])
    assert torch.equal(k[page, :, 6], new[0]) and torch.equal(k[page, :, :6], before[page, :, :6])


# ---- decode ----------------------------------------------------------------------------

LENS = [0, 1, 2, 7, 8, 9, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,by_token", [
    (14, 2, 64, 16, False), (4, 1, 128, 24, True), (3, 3, 32, 8, False), (32, 2, 96, 64, True), (9, 1, 64, 8, True),
    (40, 1, 128, 16, False),
])
def test_decode(kv, dtype, heads, kv_heads, dim, page, by_token):
    check(kv, LENS, None, heads, kv_heads, dim, page, dtype, by_token=by_token)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window,prefix,cap,slopes", [
    (1, None, 0.0, False), (64, None, 0.0, False), (65, [3] * 16, 0.0, False), (17, list(range(0, 160, 10)), 5.0, True),
    (0, [400] * 16, 1.0, False), (0, None, 0.0, True), (1000, [-4] * 16, 0.0, False),
])
def test_decode_scores(kv, dtype, window, prefix, cap, slopes):
    check(kv, LENS, None, 6, 2, 64, 8, dtype, window=window, prefix=prefix, cap=cap, slopes=slopes, scale=0.31)


@pytest.mark.parametrize("dtype,lens", [(F32, [5000]), (BF16, [40001, 1]), (F16, [1, 9999, 0, 3]), (BF16, [130] * 700)])
def test_decode_split(kv, dtype, lens):
    """Long sequences are cut over the CTAs and joined; many short ones share them."""
    if len(lens) > 100:
        k, v, table = pool(lens, 1, 64, 8, dtype)
        q = queries(len(lens), 2, 64, dtype)
        out = kv.KvPages(k, v).decode(q, table, ints(lens))
        for s in range(0, len(lens), 97):
            want, _, tol, _ = ref.attend(q[s:s + 1], ref.gather(k, table, s, 130), ref.gather(v, table, s, 130), [129], 0.125, dtype=dtype)
            close(out[s:s + 1], want, tol)
        return
    check(kv, lens, None, 8, 2, 128, 64, dtype)


# ---- prefill ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,by_token", [
    (7, 1, 64, 16, False), (4, 2, 128, 24, True), (2, 2, 32, 8, False), (16, 1, 96, 64, True), (64, 1, 64, 128, False),
    (1, 1, 128, 256, False),
])
def test_prefill(kv, dtype, heads, kv_heads, dim, page, by_token):
    check(kv, [1, 5, 64, 130, 9, 257, 0, 128], [1, 3, 64, 17, 0, 40, 0, 128], heads, kv_heads, dim, page, dtype,
          by_token=by_token)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window,prefix,cap,slopes", [
    (1, None, 0.0, False), (64, None, 0.0, False), (33, [3, 0, 130, 64], 0.0, False), (17, [200, 20, 20, 1], 5.0, True),
    (0, [400] * 4, 1.0, False), (0, None, 0.0, True), (1000, [-4] * 4, 0.0, False),
])
def test_prefill_scores(kv, dtype, window, prefix, cap, slopes):
    check(kv, [201, 131, 300, 65], [150, 131, 7, 65], 6, 2, 64, 8, dtype, window=window, prefix=prefix, cap=cap,
          slopes=slopes, scale=0.31)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale,cap", [(-0.3, 0.0), (0.0, 0.0), (-2.0, 3.0), (0.7, 0.25), (1e-3, 40.0), (4e4, 100.0), (-1e9, 1e-9)])
def test_scales_and_caps(kv, dtype, scale, cap):
    """Scales of any sign, and caps that scores stay far below or pass by far."""
    check(kv, [150, 9], None, 4, 2, 64, 8, dtype, scale=scale, cap=cap)
    check(kv, [150, 9], [40, 9], 4, 2, 64, 8, dtype, scale=scale, cap=cap, slopes=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_zero_scores_under_a_steep_cap(kv, dtype):
    """Scores of zero stay zero whatever scale and cap are: every key has the same weight."""
    k, v, table = pool([150], 2, 64, 8, dtype, False, 5)
    cache = kv.KvPages(k.zero_(), v)
    q = queries(150, 4, 64, dtype, 6)
    mean = ref.gather(v, table, 0, 150).mean(1).repeat_interleave(2, 0)
    for scale, cap in [(2.0**40, 2.0**-40), (1.0, 2.0**-40), (2.0**40, 2.0**40)]:
        for got in (cache.prefill(q, ints([0, 150]), table, ints([150]), scale=scale, cap=cap)[-1],
                    cache.decode(q[-1:].contiguous(), table, ints([150]), scale=scale, cap=cap)[0]):
            # 150 terms and two roundings of values below 5: fp32 150 2^-24 5, bf16 2^-8 of weights and result
            assert (got.double() - mean).abs().max() <= (5e-5 if dtype == F32 else 2 * 2.0**-8 * 5)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_small_scores_below_a_wide_cap(kv, dtype):
    """A cap far above most scores leaves them as they are, also beside one that reaches it."""
    lens = [150]
    k, v, table = pool(lens, 2, 64, 8, dtype, False, 5)
    cache = kv.KvPages(k, v)
    q = queries(150, 4, 64, dtype, 6)
    q[140] *= 5e3
    for scale, cap in [(0.125, 1e6), (0.125, 2.0**40), (0.125, 1e3)]:
        want, wl, tol, tol_l = ref.attend(q, ref.gather(k, table, 0, 150), ref.gather(v, table, 0, 150), range(150), scale,
                                          cap=cap, dtype=dtype)
        got = cache.prefill(q, ints([0, 150]), table, ints([150]), scale=scale, cap=cap)
        ok = torch.arange(150, device=DEV) != 140
        close(got[ok], want[ok], tol[ok], f"cap {cap}")
        close(cache.decode(q[-1:].contiguous(), table, ints([150]), scale=scale, cap=cap), want[-1:], tol[-1:], f"decode, cap {cap}")


def test_prefill_more_rows_than_keys(kv):
    """Rows at negative positions see at most the prefix; without one they are zeros."""
    for prefix in (None, [2, 0, 9]):
        check(kv, [3, 0, 20], [10, 4, 25], 4, 2, 64, 8, BF16, prefix=prefix)
        check(kv, [3, 0, 20], [10, 4, 25], 4, 2, 64, 8, F32, prefix=prefix)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [190, 205, 2 ** 31 - 1])
def test_windows_wider_than_the_sequence(kv, dtype, window):
    """Rows at negative positions do not wrap a wide window round."""
    check(kv, [3, 0, 200], [10, 4, 205], 4, 2, 64, 8, dtype, window=window)
    check(kv, [3, 0, 200], None, 4, 2, 64, 8, dtype, window=window)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_calls_without_rows(kv, dtype):
    k, v, table = pool([20], 2, 64, 8, dtype)
    cache = kv.KvPages(k, v)
    none, q = queries(0, 4, 64, dtype), queries(3, 4, 64, dtype)
    out = torch.full_like(q, 7.0)
    k0 = k.clone()
    assert cache.decode(none, table[:0], ints([])).shape == (0, 4, 64)
    assert cache.prefill(none, ints([0]), table[:0], ints([])).shape == (0, 4, 64)
    assert cache.prefill(none, ints([0, 0]), table, ints([20])).shape == (0, 4, 64)
    cache.prefill(q, ints([0]), table[:0], ints([]), out=out)
    cache.prefill(q, ints([2, 2]), table, ints([20]), out=out)
    assert (out == 7).all()
    assert cache.append(none, none[:, :2], none[:, :2], ints([]), ints([]), table).shape == (0, 4, 64)
    assert torch.equal(k.nan_to_num(0.0), k0.nan_to_num(0.0))


_FIRST = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, mocha_kv
d = dict(device="cuda", dtype=torch.bfloat16)
ints = lambda *x: torch.tensor(x, device="cuda", dtype=torch.int32)
k, v = torch.randn(6, 2, 16, 64, **d), torch.randn(6, 2, 16, 64, **d)
q, new = torch.randn(2, 8, 64, **d), torch.randn(2, 2, 64, **d)
cache, table, lens = mocha_kv.KvPages(k, v), ints(5, 0, 3, 1, 4, 2).view(2, 3), ints(40, 17)
start, seq, pos = ints(0, 1, 2), ints(0, 1), ints(39, 16)
def step():
    r = cache.append(q, new, new, seq, pos, table)
    return cache.decode(r, table, lens), cache.prefill(r, start, table, lens)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
torch.cuda.synchronize()
want = step()
assert all(torch.equal(a, b) and a.isfinite().all() for a, b in zip(got, want))
"""


def test_first_calls_of_a_process_captured(kv):
    import os
    import subprocess
    import sys
    subprocess.run([sys.executable, "-c", _FIRST, os.path.dirname(kv.__file__)], check=True, timeout=240)


@pytest.mark.parametrize("dtype,lens,qlens", [(F32, [3000], [3]), (BF16, [20000, 200], [5, 2]), (F16, [9000], [130])])
def test_prefill_split(kv, dtype, lens, qlens):
    check(kv, lens, qlens, 8, 2, 128, 64, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_prefill_many_sequences(kv, dtype):
    """More sequences than a CTA keeps tile counts of; sequences without rows among them."""
    lens = [(s * 7) % 40 for s in range(600)]
    qlens = [min(n, s % 3) for s, n in enumerate(lens)]
    k, v, table = pool(lens, 1, 64, 8, dtype)
    start = np.concatenate([[0], np.cumsum(qlens)]).astype(int).tolist()
    q = queries(start[-1], 2, 64, dtype)
    out = kv.KvPages(k, v).prefill(q, ints(start), table, ints(lens))
    for s in range(0, 600, 41):
        a, b, n = start[s], start[s + 1], lens[s]
        want, _, tol, _ = ref.attend(q[a:b], ref.gather(k, table, s, n), ref.gather(v, table, s, n),
                                     range(n - (b - a), n), 0.125, dtype=dtype)
        close(out[a:b], want, tol)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_prefill_unseen_values_stay_out(kv, dtype, value):
    """Infinite and NaN keys and values at positions that a row does not see never reach it,
    although other rows of its tile see them; rows that see them carry them on."""
    n, at = 150, [100, 149]
    k, v, table = pool([n], 2, 64, 8, dtype)
    for p in at:
        page, row = int(table[0, p // 8]), p % 8
        k[page, 0, row] = value
        v[page, :, row] = value
    q = queries(n, 4, 64, dtype)
    out = kv.KvPages(k, v).prefill(q, ints([0, n]), table, ints([n]), window=20)
    kk, vv = ref.gather(k, table, 0, n), ref.gather(v, table, 0, n)
    clean = [p for p in range(n) if not any(a <= p < a + 20 for a in at)]
    want, _, tol, _ = ref.attend(q[clean], torch.nan_to_num(kk, 0, 0, 0), torch.nan_to_num(vv, 0, 0, 0), clean, 0.125,
                                 20, dtype=dtype)
    close(out[clean], want, tol)
    assert not torch.isfinite(out[100:120]).all(-1).any() and not torch.isfinite(out[149]).all(-1).any()


def test_prefill_unseen_values_in_a_split_unit(kv):
    n = 5000
    k, v, table = pool([n], 1, 128, 16, BF16)
    page = int(table[0, (n - 1) // 16])
    v[page, :, (n - 1) % 16] = float("nan")
    q = queries(4, 2, 128, BF16)
    out = kv.KvPages(k, v).prefill(q, ints([0, 4]), table, ints([n]))
    kk, vv = ref.gather(k, table, 0, n), torch.nan_to_num(ref.gather(v, table, 0, n))
    want, _, tol, _ = ref.attend(q[:3], kk, vv, [n - 4, n - 3, n - 2], 128 ** -0.5, dtype=BF16)
    close(out[:3], want, tol)
    assert out[3].isnan().all()


# ---- both ------------------------------------------------------------------------------

@pytest.mark.parametrize("prefill", [False, True])
def test_infinite_scores(kv, prefill):
    """All visible scores -infinity: zeros; NaN queries: NaN; +infinity: NaN, as inf - inf is."""
    k, v, table = pool([40], 1, 64, 8, BF16)
    k.fill_(1.0)
    q = torch.ones(1, 3, 64, device=DEV, dtype=BF16)
    q[:, 0] = -math.inf
    q[:, 1] = math.nan
    q[:, 2] = math.inf
    lse = torch.zeros(1, 3, device=DEV)
    cache = kv.KvPages(k, v)
    out = cache.prefill(q, ints([0, 1]), table, ints([40]), lse=lse) if prefill else cache.decode(q, table, ints([40]), lse=lse)
    assert (out[0, 0] == 0).all() and lse[0, 0] == -math.inf
    assert out[0, 1].isnan().all() and out[0, 2].isnan().all() and lse[0, 1].isnan() and lse[0, 2].isnan()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("prefill", [False, True])
def test_bad_pages_read_as_zeros(kv, prefill, dtype):
    n = 200
    k, v, table = pool([n], 2, 64, 16, dtype)
    status = ints([0])
    q = queries(3 if prefill else 1, 4, 64, dtype)
    cache = kv.KvPages(k, v)

    def go(**more):
        if prefill:
            return cache.prefill(q, ints([0, 3]), table, ints([n]), status=status, **more)
        return cache.decode(q, table, ints([n]), status=status, **more)

    go()
    assert int(status) == 0
    table[0, 1], table[0, 5], table[0, 7] = -1, 1 << 30, len(k)
    # pages that no query sees may hold anything
    out = go(window=40)
    assert int(status) == 0
    first = n - q.shape[0]
    kk, vv = ref.gather(k, table, 0, n), ref.gather(v, table, 0, n)
    want, _, tol, _ = ref.attend(q, kk, vv, range(first, n), 0.125, 40, dtype=dtype)
    close(out, want, tol)
    out = go()
    assert int(status) == 1
    want, _, tol, _ = ref.attend(q, kk, vv, range(first, n), 0.125, dtype=dtype)
    close(out, want, tol)


@pytest.mark.parametrize("prefill", [False, True])
def test_lengths_past_the_table(kv, prefill):
    """A length that the table cannot hold counts as what it holds."""
    k, v, table = pool([64], 1, 64, 16, BF16)
    q = queries(1, 2, 64, BF16)
    cache = kv.KvPages(k, v)
    for n in (64, 65, 2 ** 31 - 1):
        out = cache.prefill(q, ints([0, 1]), table, ints([n])) if prefill else cache.decode(q, table, ints([n]))
        want, _, tol, _ = ref.attend(q, ref.gather(k, table, 0, 64), ref.gather(v, table, 0, 64), [63], 0.125, dtype=BF16)
        close(out, want, tol)


def test_prefill_rows_behind_the_last_sequence(kv):
    """Rows outside the ranges stay as they were; ranges are cut to the rows there are."""
    for dtype in (F32, BF16):
        k, v, table = pool([30, 30], 1, 64, 8, dtype)
        q = queries(20, 2, 64, dtype)
        out = torch.full((20, 2, 64), 3.0, device=DEV, dtype=dtype)
        cache = kv.KvPages(k, v)
        cache.prefill(q, ints([4, 9, 15]), table, ints([30, 30]), out=out)
        assert (out[:4] == 3).all() and (out[15:] == 3).all() and (out[4:15] != 3).any()
        want = out.clone()
        again = torch.full_like(out, 3.0)
        cache.prefill(q[:15], ints([4, 9, 15]), table, ints([30, 30]), out=again[:15])
        assert torch.equal(again, want)


def test_strided_queries_and_outputs(kv):
    """q out of a fused projection, out into one; the same values as contiguous ones."""
    for dtype in (F32, BF16):
        k, v, table = pool([70, 33], 2, 64, 8, dtype)
        cache = kv.KvPages(k, v)
        fused = queries(12, 4 + 2 + 2, 64, dtype)
        wide = torch.zeros(12, 9, 96, device=DEV, dtype=dtype)
        out = wide[:, 1:9:2, :64]
        q = fused[:, :4]
        cache.prefill(q, ints([0, 7, 12]), table, ints([70, 33]), out=out)
        assert torch.equal(out, cache.prefill(q.contiguous(), ints([0, 7, 12]), table, ints([70, 33])))
        assert (wide[:, 0::2] == 0).all() and (wide[:, :, 64:] == 0).all()
        wide.zero_()
        cache.decode(q[3:11:5], table, ints([70, 33]), out=out[:2])
        assert torch.equal(out[:2], cache.decode(q[3:11:5].contiguous(), table, ints([70, 33])))
        assert (wide[:, 0::2] == 0).all() and (wide[2:] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_offsets_past_32_bits(kv, dtype):
    """Pages further apart than 2^32 elements of the pool in all."""
    far = (1 << 31) + 64
    store = torch.empty(2 * far + 2 * 8 * 64 * 2, device=DEV, dtype=dtype)
    k = store.as_strided((3, 1, 8, 64), (far, 8 * 64, 64, 1))
    v = store.as_strided((3, 1, 8, 64), (far, 8 * 64, 64, 1), 8 * 64)
    g = torch.Generator(device=DEV).manual_seed(0)
    for t in (k, v):
        t.copy_(torch.randn(3, 1, 8, 64, device=DEV, generator=g))
    table = ints([2, 0, 1]).view(1, 3)
    cache = kv.KvPages(k, v)
    new = queries(1, 1, 64, dtype, 9)
    cache.append(None, new, new, ints([0]), ints([5]), table)
    assert torch.equal(k[2, 0, 5], new[0, 0]) and torch.equal(v[2, 0, 5], new[0, 0])
    q = queries(2, 2, 64, dtype)
    kk, vv = ref.gather(k, table, 0, 24), ref.gather(v, table, 0, 24)
    want, _, tol, _ = ref.attend(q, kk, vv, [22, 23], 0.125, dtype=dtype)
    close(cache.prefill(q, ints([0, 2]), table, ints([24])), want, tol)
    close(cache.decode(q[1:], table, ints([24])), want[1:], tol[1:])


def serving(kv, dtype, k, v, table, new, cos, sin, pos, seq, kv_len, start):
    cache = kv.KvPages(k, v)
    q, kn, vn = new.split([4, 2, 2], 1)
    q = cache.append(q, kn, vn, seq, pos, table, cos=cos, sin=sin)
    return cache.prefill(q, start, table, kv_len) if start is not None else cache.decode(q, table, kv_len)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_prompt_pieces_then_tokens(kv, dtype):
    """Two sequences' prompts in two pieces each, then single tokens, against the formula
    over the keys as they were rounded into the pages."""
    page, dim = 16, 64
    k, v, table = pool([80, 80], 2, dim, page, dtype)
    k.fill_(math.nan), v.fill_(math.nan)
    angle = torch.arange(80, device=DEV)[:, None] * torch.logspace(0, -3, 32, device=DEV)
    cos, sin = angle.cos(), angle.sin()
    have = [0, 0]
    for step, counts in enumerate([(33, 5), (20, 0), (1, 1), (1, 1), (1, 1)]):
        rows = sum(counts)
        new = queries(rows, 8, dim, dtype, 100 + step)
        pos = [have[s] + i for s in range(2) for i in range(counts[s])]
        seq = [s for s in range(2) for _ in range(counts[s])]
        have = [have[s] + counts[s] for s in range(2)]
        start = None if counts == (1, 1) else ints([0, counts[0], rows])
        out = serving(kv, dtype, k, v, table, new, cos, sin, ints(pos), ints(seq), ints(have), start)
        q = ref.rotate(new[:, :4], cos[pos], sin[pos], False)
        qs = kv.KvPages(k, v).append(new[:, :4], new[:, 4:6], new[:, 6:], ints(seq), ints(pos), table, cos=cos, sin=sin)
        close(qs, q[0], ref.unit(dtype) * q[0].abs() + 1.01 * q[1] + torch.finfo(dtype).tiny)
        for s in range(2):
            rws = [i for i in range(rows) if seq[i] == s]
            want, _, tol, _ = ref.attend(qs[rws], ref.gather(k, table, s, have[s]), ref.gather(v, table, s, have[s]),
                                         [pos[i] for i in rws], 0.125, dtype=dtype)
            close(out[rws], want, tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("prefill", [False, True])
def test_captured_and_replayed(kv, dtype, prefill):
    """A captured step follows lengths, positions and tables that change between replays."""
    lens = [300, 17]
    k, v, table = pool([320, 320], 2, 64, 16, dtype, fill=0.0)
    angle = torch.arange(320, device=DEV)[:, None] * torch.logspace(0, -3, 32, device=DEV)
    cos, sin = angle.cos(), angle.sin()
    new = queries(2, 8, 64, dtype)
    pos, kv_len, seq = ints([n - 1 for n in lens]), ints(lens), ints([0, 1])
    start = ints([0, 1, 2]) if prefill else None
    args = (kv, dtype, k, v, table, new, cos, sin, pos, seq, kv_len, start)
    serving(*args)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = serving(*args)
    for step in range(3):
        new.copy_(queries(2, 8, 64, dtype, 50 + step))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, serving(*args))
        pos += 1
        kv_len += 1
    seq[1] = -1  # a padded batch: the second row is skipped, its sequence has no keys
    kv_len[1] = 0
    g.replay()
    torch.cuda.synchronize()
    if not prefill:
        assert (out[1] == 0).all()


def test_two_streams_and_threads_at_once(kv):
    """Calls on two streams from two threads: the results of calls one after the other."""
    k, v, table = pool([3000, 50, 700], 2, 128, 32, BF16)
    cache = kv.KvPages(k, v)
    q = queries(3, 8, 128, BF16)
    qp = queries(60, 8, 128, BF16, 7)
    lens, start = ints([3000, 50, 700]), ints([0, 20, 30, 60])
    want = cache.decode(q, table, lens), cache.prefill(qp, start, table, lens)
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got[i].append(cache.prefill(qp, start, table, lens) if i else cache.decode(q, table, lens))
        s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_same_bits_every_time(kv, dtype):
    k, v, table = pool([5000, 900, 3], 2, 64, 16, dtype)
    cache = kv.KvPages(k, v)
    q, qp = queries(3, 8, 64, dtype), queries(300, 8, 64, dtype)
    lens, start = ints([5000, 900, 3]), ints([0, 200, 297, 300])
    want = cache.decode(q, table, lens), cache.prefill(qp, start, table, lens)
    for _ in range(10):
        assert torch.equal(cache.decode(q, table, lens), want[0])
        assert torch.equal(cache.prefill(qp, start, table, lens), want[1])


def test_refusals(kv):
    k, v, table = pool([40, 40], 2, 64, 16, BF16)
    cache = kv.KvPages(k, v)
    lens, q = ints([40, 40]), queries(2, 4, 64, BF16)
    start = ints([0, 1, 2])
    bad = [
        lambda: cache.decode(q.float(), table, lens),
        lambda: cache.decode(q[:1], table, lens),
        lambda: cache.decode(q[:, :, :32], table, lens),
        lambda: cache.decode(q, table.long(), lens),
        lambda: cache.decode(q, table, lens.long()),
        lambda: cache.decode(q, table, lens[:1]),
        lambda: cache.decode(q, table, lens, prefix=ints([1])),
        lambda: cache.decode(q, table, lens, slopes=torch.ones(3, device=DEV)),
        lambda: cache.decode(q.cpu(), table, lens),
        lambda: cache.decode(q, table, lens, lse=torch.zeros(2, 3, device=DEV)),
        lambda: cache.prefill(q, start[:2], table, lens),
        lambda: cache.append(q, q[:, :1], q[:, :2], lens, lens, table),
        lambda: cache.append(q, q[:, :2], q[:, :2], lens, lens, table, cos=torch.zeros(9, 32, device=DEV)),
        lambda: cache.decode(q.clone().requires_grad_(), table, lens),
        lambda: kv.KvPages(k, v[:, :1]),
        lambda: kv.KvPages(k, v.float()),
        lambda: kv.KvPages(k.clone().requires_grad_(), v),
        lambda: kv.KvPages(k.cpu(), v.cpu()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
    errors = [
        lambda: cache.decode(queries(2, 3, 64, BF16), table, lens),       # heads not a multiple
        lambda: cache.decode(queries(2, 130, 64, BF16), table, lens),     # more than 64 per kv head
        lambda: cache.decode(q, table, lens, window=-1),
        lambda: cache.decode(q, table, lens, cap=-1.0),
        lambda: cache.decode(q, table, lens, scale=math.nan),
        lambda: cache.decode(torch.zeros(2, 4, 65, device=DEV, dtype=BF16)[:, :, :64], table, lens),  # stride of 130 bytes
        lambda: cache.decode(torch.zeros(2 * 4 * 64 + 1, device=DEV, dtype=BF16)[1:].view(2, 4, 64), table, lens),
        lambda: cache.append(q, q[:, :2], q[:, :2], lens, lens, table, cos=torch.zeros(9, 36, device=DEV),
                             sin=torch.zeros(9, 36, device=DEV)),         # 72 rotated dims of 64
    ]
    for call in errors:
        with pytest.raises(RuntimeError):
            call()
    assert cache.decode(q, table, lens).isfinite().all()
    with torch.no_grad():
        assert cache.decode(q.clone().requires_grad_(), table, lens).isfinite().all()
    one = torch.zeros(16, device=DEV).as_strided((1, 16), (3, 1))  # a table of one row has no stride between rows
    cache.append(q, q[:, :2], q[:, :2], ints([0, 1]), ints([0, 0]), table, cos=one, sin=one)


def test_c_calls_refuse_a_small_workspace(kv, native, capfd):
    k, v, table = pool([40], 2, 64, 16, BF16)
    cache = kv.KvPages(k, v)
    lib = kv._load()
    q = queries(1, 4, 64, BF16)
    out = torch.zeros_like(q)
    lens = ints([40])
    rows = kv._Rows(q.data_ptr(), 0, 64), kv._Rows(out.data_ptr(), 0, 64)
    seqs, scores = cache._seqs(table, lens, None), cache._scores(4, 1, None, 0, None, 0.0, None)
    need = ctypes.c_ulonglong()
    assert lib.mocha_kv_workspace(cache._pages, 4, 0, ctypes.byref(need)) == 0
    space = torch.empty(need.value + 16, dtype=torch.uint8, device=DEV)
    at = ctypes.addressof

    def go(ptr, size):
        return lib.mocha_kv_decode(cache._pages, at(seqs), at(scores), at(rows[0]), at(rows[1]), None, ptr, size, None)

    assert go(space.data_ptr(), need.value - 1) == 1
    assert go(space.data_ptr() + 8, need.value) == 1
    assert go(None, need.value) == 1
    assert "workspace" in capfd.readouterr().err
    torch.cuda.synchronize()
    assert (out == 0).all()
    assert go(space.data_ptr(), need.value) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, cache.decode(q, table, lens))
