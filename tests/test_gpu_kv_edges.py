"""The paged key/value operators at the edges of what they take: waits that run out."""
import ctypes

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
