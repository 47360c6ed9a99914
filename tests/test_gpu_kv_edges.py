"""The paged key/value operators at the edges of what they take: waits that run out, tensors
that gradients are asked of."""
import ctypes
import math

import pytest
import torch

import kv_reference as ref
from test_gpu_kv import BF16, DEV, F16, F32, close, ints, kv, pool, queries  # noqa: F401 (kv is a fixture)

pytestmark = pytest.mark.gpu


# ---- waits that run out ----------------------------------------------------------------

@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64)])
def test_waits_that_run_out(kv, dtype, dim):
    """CTAs that never get some values give up: status 2, and every row is what it always is or
    NaN, also rows that others had parts of.  The next call is as if nothing had been."""
    lens, counts = [9000, 700, 40], [300, 200, 40]
    rows, heads, kvh = sum(counts), 8, 2
    k, v, table = pool(lens, kvh, dim, 16, dtype)
    cache = kv.KvPages(k, v)
    q, start = queries(rows, heads, dim, dtype), ints([0, 300, 500, 540])
    lse = torch.empty(rows, heads, device=DEV)
    want = cache.prefill(q, start, table, ints(lens), lse=lse)
    want_l = lse.clone()
    torch.cuda.synchronize()
    assert want.isfinite().all() and want_l.isfinite().all()
    lib, at = kv._load(), ctypes.addressof
    for drop in (0, 1, 2, 8, 70):
        out, status = torch.full_like(q, 7.0), ints([0])
        lse.fill_(5.0)
        held = ints(lens)
        args = [cache._seqs(table, held, status), cache._scores(heads, 3, None, 0, None, 0.0, None),
                cache._rows(q, "q", dtype, rows), cache._rows(out, "out", dtype, rows)]
        size, space = cache._space(lib, heads, 1)
        assert lib.mocha_kv_prefill_check(cache._pages, at(args[0]), at(args[1]), rows, start.data_ptr(), at(args[2]),
                                          at(args[3]), lse.data_ptr(), space.data_ptr(), size,
                                          torch.cuda.current_stream().cuda_stream, 64 if drop else 1 << 18, drop) == 0
        torch.cuda.synchronize()
        lost = out.isnan().any(-1)
        assert torch.equal(lost, out.isnan().all(-1)) and torch.equal(lost, lse.isnan())
        assert torch.equal(out[~lost], want[~lost]) and torch.equal(lse[~lost], want_l[~lost])
        assert int(status) == (2 if lost.any() else 0)
        # drop 1 stops every CTA; 70 the first ones and those from 70 on, of the 134 that have shares of 6
        assert lost.any() == (drop > 0) and lost.all() >= (drop == 1) and not (drop == 70 and lost.all())
    assert torch.equal(cache.prefill(q, start, table, ints(lens)), want)


# ---- gradients -------------------------------------------------------------------------

def test_gradients_and_tangents_are_refused(kv):
    """Every floating tensor of every call, by reverse and by forward mode; none of them would
    get anything."""
    k, v, table = pool([40, 40], 2, 64, 16, BF16)
    cache = kv.KvPages(k, v)
    lens, start, seq, pos = ints([40, 40]), ints([0, 1, 2]), ints([0, 1]), ints([3, 4])
    q, new = queries(2, 4, 64, BF16), queries(2, 2, 64, BF16)
    cos, sin = torch.ones(9, 32, device=DEV), torch.zeros(9, 32, device=DEV)
    slopes = torch.ones(4, device=DEV)

    def calls(x):
        """name -> the call with that tensor put through x"""
        lse = torch.zeros(2, 4, device=DEV)
        out = torch.zeros_like(q)
        return {
            "append q": lambda: cache.append(x(q), new, new, seq, pos, table, cos=cos, sin=sin),
            "append k": lambda: cache.append(q, x(new), new, seq, pos, table, cos=cos, sin=sin),
            "append v": lambda: cache.append(q, new, x(new), seq, pos, table, cos=cos, sin=sin),
            "append cos": lambda: cache.append(q, new, new, seq, pos, table, cos=x(cos), sin=sin),
            "append sin": lambda: cache.append(q, new, new, seq, pos, table, cos=cos, sin=x(sin)),
            "append q_out": lambda: cache.append(q, new, new, seq, pos, table, cos=cos, sin=sin, q_out=x(out)),
            "decode q": lambda: cache.decode(x(q), table, lens),
            "decode slopes": lambda: cache.decode(q, table, lens, slopes=x(slopes)),
            "decode out": lambda: cache.decode(q, table, lens, out=x(out)),
            "decode lse": lambda: cache.decode(q, table, lens, lse=x(lse)),
            "prefill q": lambda: cache.prefill(x(q), start, table, lens),
            "prefill slopes": lambda: cache.prefill(q, start, table, lens, slopes=x(slopes)),
            "prefill lse": lambda: cache.prefill(q, start, table, lens, lse=x(lse)),
            "pages k": lambda: kv.KvPages(x(k), v).decode(q, table, lens),
            "pages v": lambda: kv.KvPages(k, x(v)).decode(q, table, lens),
        }

    for call in calls(lambda t: t).values():
        call()
    for call in calls(lambda t: t.clone().requires_grad_()).values():
        with pytest.raises(ValueError):
            call()
        with torch.no_grad():
            call()
    with torch.autograd.forward_ad.dual_level():
        for call in calls(lambda t: torch.autograd.forward_ad.make_dual(t.clone(), torch.ones_like(t))).values():
            with pytest.raises(ValueError):
                call()
        cache.decode(q, table, lens, slopes=slopes)
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda t: cache.decode(t, table, lens), (q,), (q,))
    with torch.no_grad():
        late = kv.KvPages(k.clone().requires_grad_(), v)
        late.decode(q, table, lens)
    with pytest.raises(ValueError):
        late.decode(q, table, lens)


# ---- options ---------------------------------------------------------------------------

def test_windows_past_32_bits(kv):
    """A window that no 32-bit number holds is wider than any sequence, or negative."""
    k, v, table = pool([40, 9], 2, 64, 16, BF16)
    cache = kv.KvPages(k, v)
    lens, q, start = ints([40, 9]), queries(2, 4, 64, BF16), ints([0, 1, 2])
    for window in (2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1, 2 ** 64 + 1):
        assert torch.equal(cache.decode(q, table, lens, window=window), cache.decode(q, table, lens))
        assert torch.equal(cache.prefill(q, start, table, lens, window=window), cache.prefill(q, start, table, lens))
    for window in (-1, -2 ** 32 + 5, -2 ** 63):
        with pytest.raises(RuntimeError):
            cache.decode(q, table, lens, window=window)
        with pytest.raises(RuntimeError):
            cache.prefill(q, start, table, lens, window=window)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [36, 5])
def test_caps_do_not_see_other_calls(kv, dtype, rows):
    """The same bits whatever ran before: a group of 7 heads leaves the last two of a tile's 128
    rows without queries, a short piece more, and what a call before left there is no score."""
    k, v, table = pool([600], 2, 64, 16, dtype)
    cache = kv.KvPages(k, v)
    lens, start = ints([600]), ints([0, rows])
    q = queries(rows, 14, 64, dtype, scale=0.5)
    full = queries(600, 16, 64, dtype, 3)
    got = []
    for size in (0.0, 1e3, 1.0):
        for _ in range(3):
            cache.prefill(full * size, ints([0, 600]), table, lens)
        got.append(cache.prefill(q, start, table, lens, cap=30.0))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("prefill", [False, True])
def test_caps_do_not_see_other_keys(kv, dtype, prefill):
    """The same bits whatever lies behind the sequence's end in its last page, in pages that its
    window has left, in other caches, and at positions that a row does not see."""
    n, rows = 420, 30 if prefill else 1
    k, v, table = pool([n], 2, 64, 16, dtype, fill=0.0)
    cache = kv.KvPages(k, v)
    other = kv.KvPages(torch.zeros_like(k), torch.zeros_like(v))
    far = torch.arange(len(k), device=DEV, dtype=torch.int32).view(1, -1)
    q = queries(rows, 4, 64, dtype, scale=0.5)
    seen_by_last = k[int(table[0, 26]), :, 1:4].clone()
    got = []
    for size in (0.0, 1e3, -30.0):
        k[int(table[0, 26]), :, 4:] = size  # 420 = 26 * 16 + 4
        k[int(table[0, 2])] = size  # positions 32 .. 47, before the window
        k[int(table[0, 26]), :, 1:4] = size if prefill else seen_by_last  # the last three, which the rows before do not see
        other.k.fill_(size)
        big = queries(300, 4, 64, dtype, 7)
        other.prefill(big, ints([0, 300]), far, ints([16 * len(k)]))
        other.decode(big[:1], far, ints([16 * len(k)]))
        if prefill:
            got.append(cache.prefill(q, ints([0, rows]), table, ints([n]), cap=30.0, window=300)[:rows - 3])
        else:
            got.append(cache.decode(q, table, ints([n]), cap=30.0, window=300))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("scale,cap,size", [(2.0 ** -30, 50.0, 12000.0), (2.0 ** -39, 1.0, 2.0 ** 17),
                                            (2.0 ** 10, 2.0 ** -10, 2.0 ** -42), (0.125, 50.0, 9e-5)])
def test_caps_over_scores_of_any_size(kv, prefill, scale, cap, size):
    """Products far from 1 under a small or large scale: scores of a tenth of the cap and up to
    half of it, where tanh is neither its argument nor 1."""
    k, v, table = pool([300], 2, 64, 16, BF16)
    k *= 2.0 ** 16
    cache = kv.KvPages(k, v)
    q = queries(40, 4, 64, BF16, scale=size)
    z = (ref.gather(k, table, 0, 300)[0] @ q[:, 0].double().T * scale / cap).abs()
    assert 0.05 < z.median() < 0.2 and z.max() < 0.6, (float(z.median()), float(z.max()))
    want, _, tol, _ = ref.attend(q, ref.gather(k, table, 0, 300), ref.gather(v, table, 0, 300), range(260, 300), scale,
                                 cap=cap, dtype=BF16)
    if prefill:
        close(cache.prefill(q, ints([0, 40]), table, ints([300]), scale=scale, cap=cap), want, tol)
    else:
        close(cache.decode(q[-1:].contiguous(), table, ints([300]), scale=scale, cap=cap), want[-1:], tol[-1:])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("top", [0.0, 1.0])
def test_many_weights_far_below_the_largest(kv, prefill, dtype, top):
    """One key 25.5 powers of two above 131071 others, whose weights together are W = 0.28 % of its
    own, in so many sequences (over the same pages) that whole ones fall to one CTA: with a value
    of `top` against theirs of -1 the output is (top - W) / (1 + W).  It may be off by
      u |o|, its own rounding;
      n 2^-32: an fp16 weight is off by at most 2^-25, the largest being 2^7 (bf16: 2^-8 W);
      n 2^-24 times the largest sum on the way, top + W, for a product that is added to an fp32
      sum loses what lies below that sum's last place (beside a top of 1, more than all of W);
      60 2^-24 W, the exponents' last places (scores of 25.5), and 2^-22 W for the rest.
    lse is a sum of n fp32 weights, at most 2048 of them one after the other."""
    n, page = 131072, 64
    seqs, rows = (160, 256) if prefill else (640, 1)
    k = torch.zeros(n // page, 1, page, 64, device=DEV, dtype=dtype)
    v = torch.full_like(k, -1.0)
    k[..., 0] = -1.0
    k[0, 0, 0, 0] = 0.0
    v[0, 0, 0] = top
    table = torch.arange(n // page, device=DEV, dtype=torch.int32).repeat(seqs, 1)
    q = torch.zeros(seqs * rows, 1, 64, device=DEV, dtype=dtype)
    q[:, 0, 0] = 1.0
    lens = ints([n] * seqs)
    cache = kv.KvPages(k, v)
    lse = torch.empty(seqs * rows, 1, device=DEV)
    scale = 25.5 * math.log(2.0)
    if prefill:
        out = cache.prefill(q, ints(range(0, seqs * rows + 1, rows)), table, lens, scale=scale, lse=lse)
    else:
        out = cache.decode(q, table, lens, scale=scale, lse=lse)
    w = torch.arange(n - rows, n, device=DEV, dtype=torch.float64).repeat(seqs) * 2.0 ** -25.5
    want = ((top - w) / (1 + w))[:, None, None]
    most = float(w.max())
    weights = n * 2.0 ** -32 if dtype == F16 else 2.0 ** -8 * most
    tol = ref.unit(dtype) * want.abs() + weights + n * 2.0 ** -24 * (top + most) + (60 * 2.0 ** -24 + 2.0 ** -22) * most
    close(out, want, tol)
    assert float((lse[:, 0].double() - torch.log1p(w)).abs().max()) <= 2048 * 2.0 ** -24 + 60 * 2.0 ** -24 * most + 2.0 ** -22


# ---- infinite and NaN values -----------------------------------------------------------

def plain(q, k, v, positions, window=0, prefix=0):
    """The formula by torch in 64 bits, so that infinities and NaN go where they go."""
    rows, heads, dim = q.shape
    group = heads // k.shape[0]
    k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
    z = torch.einsum("rhd,hjd->hrj", q.double(), k) * dim ** -0.5
    p, j = torch.tensor(list(positions), device=DEV)[:, None], torch.arange(k.shape[1], device=DEV)
    seen = (j <= p) & ((p - j < window) if window else True) | (j < prefix)
    out = torch.empty(rows, heads, dim, dtype=torch.float64, device=DEV)
    for r in range(rows):
        at = seen[r].nonzero().flatten()
        if len(at) == 0 or not (z[:, r, at] > -math.inf).any():
            out[r] = 0.0
            continue
        out[r] = torch.einsum("hj,hjd->hd", torch.softmax(z[:, r, at], -1), v[:, at])
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("where", ["seen by all", "seen by some", "one dim", "both", "values everywhere", "keys too"])
@pytest.mark.parametrize("window,prefix", [(0, 0), (70, 3)])
def test_values_that_are_not_finite(kv, dtype, where, window, prefix):
    """Infinities and NaN in keys and values that rows see, do not see, or both, beside finite ones:
    what a row sees shows in its dims as the formula has it, what it does not see nowhere."""
    n, rows = 300, 170
    k, v, table = pool([n], 2, 64, 16, dtype, fill=0.0)

    def put(t, pos, value, dims=slice(None)):
        t[int(table[0, pos // 16]), :, pos % 16, dims] = value

    if where == "seen by all":
        put(v, 1, math.nan)
    if where in ("seen by some", "both"):
        put(v, 200, math.inf), put(v, 231, math.nan, slice(3, 9))
    if where in ("one dim", "both"):
        put(v, 2, math.inf, slice(17, 18)), put(v, 140, -math.inf, slice(17, 20))
    if where in ("values everywhere", "keys too"):
        v.fill_(math.nan)
    if where == "keys too":
        put(k, 150, math.nan), put(k, 151, math.inf)
    q, lse, lse0 = queries(rows, 6, 64, dtype), torch.zeros(rows, 6, device=DEV), torch.zeros(rows, 6, device=DEV)
    more = dict(window=window, prefix=ints([prefix]) if prefix else None)
    cache = kv.KvPages(k, v)
    out = cache.prefill(q, ints([0, rows]), table, ints([n]), lse=lse, **more)
    kv.KvPages(k, torch.zeros_like(v)).prefill(q, ints([0, rows]), table, ints([n]), lse=lse0, **more)
    kk, vv = ref.gather(k, table, 0, n), ref.gather(v, table, 0, n)
    want = plain(q, kk, vv, range(n - rows, n), window, prefix)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.isinf(), want.isinf()) and torch.equal(out[out.isinf()].double(), want[want.isinf()])
    _, _, tol, _ = ref.attend(q, torch.nan_to_num(kk, 0, 0, 0), torch.nan_to_num(vv, 0, 0, 0), range(n - rows, n), 0.125, window,
                              prefix, dtype=dtype)
    ok = want.isfinite()
    close(out[ok], want[ok], tol[ok])
    assert torch.equal(lse.nan_to_num(7.0), lse0.nan_to_num(7.0))  # the values are no part of it
    one = cache.decode(q[-1:].contiguous(), table, ints([n]), **more)[0]
    assert torch.equal(one.isnan(), want[-1].isnan())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_of_minus_infinity_over_nan_values(kv, dtype):
    """Rows whose visible scores are all -infinity are zeros, whatever the values hold."""
    for n, rows in ((40, 1), (40, 30), (3000, 2)):
        k, v, table = pool([n], 1, 64, 8, dtype)
        k.fill_(1.0), v.fill_(math.nan)
        q = torch.full((rows, 2, 64), -math.inf, device=DEV, dtype=dtype)
        cache = kv.KvPages(k, v)
        assert (cache.prefill(q, ints([0, rows]), table, ints([n])) == 0).all()
        assert (cache.decode(q[:1].contiguous(), table, ints([n])) == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_nan_does_not_cost_a_prompt_its_speed(kv, dtype):
    """A NaN that every row sees makes every row NaN: each is looked at once more, but not done
    once more (some 100 times the call's time)."""
    n = 4096 if dtype == BF16 else 1024
    k, v, table = pool([n], 2, 64, 64, dtype)
    q = queries(n, 8, 64, dtype)
    start, lens = ints([0, n]), ints([n])
    cache = kv.KvPages(k, v)
    out = torch.empty_like(q)

    def time():
        best = math.inf
        for _ in range(3):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            cache.prefill(q, start, table, lens, out=out)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    usual = time()
    assert out.isfinite().all()
    v[int(table[0, 0]), :, 0] = math.nan
    slow = time()
    print("ms", usual, slow)
    assert out.isnan().all() and slow < 30 * usual


# ---- roundings -------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,heads,kvh,dim,more", [
    ([1, 2, 40, 300, 3000], 6, 2, 64, {}), ([777], 32, 4, 128, {}), ([130, 2000], 24, 2, 96, {}),
    ([130, 900], 40, 1, 128, {"window": 400, "prefix": 5}), ([1500, 9], 4, 4, 32, {"cap": 20.0}),
])
def test_decode_rounds_its_outputs_alone(kv, dtype, lens, heads, kvh, dim, more):
    """Single-token attention in 16 bits: u |o| for the output, 2^-16 A for weights in two parts (the
    second at most 2u of the weight and rounded by u of itself: 2^-15 in bf16), n 2^-32 of the largest
    value for fp16's last bit, and what the same formula in fp32 may be off by; no u A for weights
    of 16 bits."""
    k, v, table = pool(lens, kvh, dim, 16, dtype)
    q = queries(len(lens), heads, dim, dtype)
    window, prefix, cap = (more.get(x, 0) for x in ("window", "prefix", "cap"))
    out = kv.KvPages(k, v).decode(q, table, ints(lens), window=window, cap=cap, prefix=ints([prefix] * len(lens)))
    for s, n in enumerate(lens):
        kk, vv = ref.gather(k, table, s, n), ref.gather(v, table, s, n)
        args = ([n - 1], dim ** -0.5, window, min(prefix, n), cap)
        want, _, tol, _ = ref.attend(q[s:s + 1], kk, vv, *args)
        size = ref.attend(q[s:s + 1], kk, vv.abs(), *args)[0]
        u = ref.unit(dtype)
        close(out[s:s + 1], want, u * want.abs() + max(2.0 ** -16, 2 * u * u) * size + n * 2.0 ** -32 * vv.abs().max() + tol)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("prefill", [False, True])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("scale,cap", [(4e4, 100.0), (-1e9, 1e-9), (3.0, 4.0), (-0.7, 0.25), (0.125, 50.0), (2.0 ** 40, 2.0 ** -40)])
def test_caps_that_scores_reach(kv, prefill, dtype, slopes, scale, cap):
    """Scores around a cap and far past it, under a bound that stays far below the outputs."""
    n, rows = 200, 60
    k, v, table = pool([n], 2, 64, 16, dtype)
    q = queries(rows, 4, 64, dtype)
    sl = torch.tensor([0.5, 0.125, 0.03, 0.004], device=DEV) if slopes else None
    want, tol = ref.capped(q, ref.gather(k, table, 0, n), ref.gather(v, table, 0, n), range(n - rows, n), scale, cap, sl, dtype)
    assert float(tol.median()) < 0.1 * float(want.abs().median())
    cache = kv.KvPages(k, v)
    if prefill:
        close(cache.prefill(q, ints([0, rows]), table, ints([n]), scale=scale, cap=cap, slopes=sl), want, tol)
    else:
        close(cache.decode(q[-1:].contiguous(), table, ints([n]), scale=scale, cap=cap, slopes=sl), want[-1:], tol[-1:])


# ---- strides ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_broadcast_queries_and_pages(kv, dtype):
    """One query row for all rows, and one page under several ids (strides of 0): as if copied."""
    k, v, table = pool([70, 33], 2, 64, 16, dtype)
    cache = kv.KvPages(k, v)
    lens, start = ints([70, 33]), ints([0, 7, 12])
    q = queries(1, 4, 64, dtype)
    for n, call in ((12, lambda x: cache.prefill(x, start, table, lens)), (2, lambda x: cache.decode(x, table, lens))):
        assert torch.equal(call(q.expand(n, 4, 64)), call(q.expand(n, 4, 64).contiguous()))
    q = queries(12, 4, 64, dtype)
    k1, v1 = (queries(2, 16, 64, dtype, seed=s).view(1, 2, 16, 64).expand(5, 2, 16, 64) for s in (3, 4))
    wide, copied = kv.KvPages(k1, v1), kv.KvPages(k1.contiguous(), v1.contiguous())
    ids = ints([4, 0, 2, 1, 3, 1, 0, 2, 2, 4]).view(2, 5)
    for call in (lambda c: c.prefill(q, start, ids, lens), lambda c: c.decode(q[:2], ids, lens)):
        assert torch.equal(call(wide), call(copied))
