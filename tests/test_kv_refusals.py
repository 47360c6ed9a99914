"""Argument checks of mocha_kv.h: bad calls return 1 with their message before any CUDA call
is made, so they are refused the same on a machine without a GPU."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def kv(native):
    import mocha_kv
    return mocha_kv


def pages(kv, **more):
    p = dict(device=0, type=2, pages=10, page_size=16, kv_heads=2, head_dim=64, page_stride=2048, head_stride=1024,
             token_stride=64, k=1 << 20, v=1 << 21)
    p.update(more)
    return kv._Pages(**p)


def refs(*structs):
    return [s if s is None or isinstance(s, int) else C.addressof(s) for s in structs]


def decode(kv, p=None, s=None, z=None, q=None, out=None, n=2):
    p = p or pages(kv)
    s = s or kv._Seqs(n, 4, 4, 4096, 8192, None)
    z = z or kv._Scores(4, 0, 0.125, 0.0, None, None)
    q = q or kv._Rows(1 << 16, 256, 64)
    out = out or kv._Rows(1 << 17, 256, 64)
    a = [p, s, z, q, out]
    return kv._load().mocha_kv_decode(*refs(*a), None, 1 << 18, 1 << 40, None)


@pytest.mark.parametrize("more,message", [
    ({"type": 3}, "type"), ({"pages": 0}, "pages"), ({"kv_heads": 0}, "kv_heads"), ({"page_size": 12}, "page_size"),
    ({"page_size": 0}, "page_size"), ({"page_size": 1 << 17}, "page_size"), ({"head_dim": 48}, "head_dim"),
    ({"head_dim": 160}, "head_dim"), ({"token_stride": 60}, "token_stride"), ({"token_stride": 68}, "16 bytes"),
    ({"page_stride": -8}, "negative"), ({"page_stride": 1 << 40}, "large"), ({"k": 0}, "aligned"),
    ({"v": (1 << 21) + 8}, "aligned"),
])
def test_pages(kv, capfd, more, message):
    assert decode(kv, pages(kv, **more)) == 1
    err = capfd.readouterr().err
    assert err.startswith("mocha_kv_decode: ") and message in err
    got = C.c_ulonglong()
    assert kv._load().mocha_kv_workspace(*refs(pages(kv, **more)), 4, 0, C.byref(got)) == 1


@pytest.mark.parametrize("what,message", [
    (dict(s=(-1, 4, 4, 4096, 8192, None)), "seqs"), (dict(s=(2, 0, 4, 4096, 8192, None)), "table_width"),
    (dict(s=(2, 4, 3, 4096, 8192, None)), "table_stride"), (dict(s=(2, 4, 4, None, 8192, None)), "null table"),
    (dict(s=(2, 4, 4, 4096, None, None)), "kv_len"), (dict(z=(3, 0, 0.1, 0.0, None, None)), "multiple of kv_heads"),
    (dict(z=(130, 0, 0.1, 0.0, None, None)), "64 times"), (dict(z=(4, -1, 0.1, 0.0, None, None)), "window"),
    (dict(z=(4, 0, float("inf"), 0.0, None, None)), "finite"), (dict(z=(4, 0, 0.1, -1.0, None, None)), "cap"),
    (dict(z=(4, 0, 2.0**41, 0.0, None, None)), "scale"), (dict(z=(4, 0, float("nan"), 0.0, None, None)), "scale"),
    (dict(z=(4, 0, 0.1, 2.0**-41, None, None)), "cap"), (dict(z=(4, 0, 0.1, 2.0**41, None, None)), "cap"),
    (dict(z=(4, 0, 0.1, float("nan"), None, None)), "cap"),
    (dict(q=(None, 256, 64)), "null q"), (dict(q=((1 << 16) + 2, 256, 64)), "q must be"),
    (dict(q=(1 << 16, 257, 64)), "q must be"), (dict(out=(1 << 17, 256, 32)), "out must be"),
    (dict(out=(1 << 17, -256, 64)), "out must be"),
])
def test_decode(kv, capfd, what, message):
    kinds = {"s": kv._Seqs, "z": kv._Scores, "q": kv._Rows, "out": kv._Rows}
    assert decode(kv, **{n: kinds[n](*a) for n, a in what.items()}) == 1
    assert message in capfd.readouterr().err


def test_null_structs(kv, capfd):
    lib = kv._load()
    assert lib.mocha_kv_decode(None, None, None, None, None, None, None, 0, None) == 1
    assert lib.mocha_kv_prefill(None, None, None, 0, None, None, None, None, None, 0, None) == 1
    assert lib.mocha_kv_append(None, None, 0, None, None, 0, 0, None, None, None, None, None, None) == 1
    assert lib.mocha_kv_workspace(None, 4, 0, None) == 1
    p = pages(kv)
    assert lib.mocha_kv_decode(*refs(p), None, None, None, None, None, None, 0, None) == 1
    assert lib.mocha_kv_workspace(*refs(p), 4, 0, None) == 1
    assert capfd.readouterr().err.count("null") >= 5


def append(kv, p=None, rows=3, seq=4096, pos=4096, in_type=0, heads=4, q=1, k=1, v=1, q_out=1, rope=1):
    row = kv._Rows(1 << 16, 512, 64)
    out = kv._Rows(1 << 24, 512, 64)
    keep = [p or pages(kv), kv._Seqs(2, 4, 4, 4096, None, None)]
    pick = [row if x == 1 else x for x in (q, k, v)] + [out if q_out == 1 else q_out,
                                                       kv._Rope(4096, 8192, 32, 100, 64, 0) if rope == 1 else rope]
    a = refs(*keep)
    b = refs(*pick)
    return kv._load().mocha_kv_append(*a, rows, seq, pos, in_type, heads, *b, None)


@pytest.mark.parametrize("what,message", [
    (dict(in_type=5), "in_type"), (dict(rows=-1), "rows"), (dict(seq=None), "seq"), (dict(pos=None), "pos"),
    (dict(q=None), "together"), (dict(q_out=None), "together"), (dict(heads=0), "heads"), (dict(k=None), "null k"),
    (dict(v=None), "null v"), (dict(rope=None), "rope"), (dict(rows=2 ** 31 - 1, heads=1 << 24), "too many"),
])
def test_append(kv, capfd, what, message):
    assert append(kv, **what) == 1
    assert message in capfd.readouterr().err


@pytest.mark.parametrize("rope,message", [
    ((4096, 8192, 32, 100, 24, 0), "dims"), ((4096, 8192, 32, 100, 80, 0), "dims"), ((4096, 8192, 32, 100, -16, 0), "dims"),
    ((None, 8192, 32, 100, 64, 0), "cos"), ((4096, 8196, 32, 100, 64, 0), "cos"), ((4096, 8192, 31, 100, 64, 0), "cos"),
    ((4096, 8192, 34, 100, 64, 0), "cos"), ((4096, 8192, 32, 0, 64, 0), "cos"),
])
def test_append_angles(kv, capfd, rope, message):
    assert append(kv, rope=kv._Rope(*rope)) == 1
    assert message in capfd.readouterr().err


def test_append_in_place_needs_one_type(kv, capfd):
    assert append(kv, q_out=kv._Rows(1 << 16, 512, 64)) == 1
    assert "only with the same type" in capfd.readouterr().err


def test_prefill_rows(kv, capfd):
    keep = [pages(kv), kv._Seqs(2, 4, 4, 4096, 8192, None), kv._Scores(4, 0, 0.125, 0.0, None, None)]
    row = kv._Rows(1 << 16, 256, 64)
    lib = kv._load()
    a, r = refs(*keep), C.addressof(row)
    assert lib.mocha_kv_prefill(*a, -1, 4096, r, r, None, 1 << 18, 1 << 40, None) == 1
    assert "rows" in capfd.readouterr().err
    assert lib.mocha_kv_prefill(*a, 3, None, r, r, None, 1 << 18, 1 << 40, None) == 1
    assert "q_start" in capfd.readouterr().err


@pytest.mark.parametrize("polls,drop", [(-1, 0), (1, -1)])
def test_prefill_check(kv, capfd, polls, drop):
    assert kv._load().mocha_kv_prefill_check(None, None, None, 0, None, None, None, None, None, 0, None, polls, drop) == 1
    assert "wait_polls" in capfd.readouterr().err


def test_workspace(kv):
    lib = kv._load()
    got = C.c_ulonglong()
    for t in (0, 1, 2):
        for d in (32, 64, 96, 128):
            for prefill in (0, 1):
                p = pages(kv, type=t, head_dim=d, token_stride=128, head_stride=2048, page_stride=4096)
                assert lib.mocha_kv_workspace(*refs(p), 28, prefill, C.byref(got)) == 0
                assert 0 < got.value < 64 << 20 and got.value % 8 == 0


@pytest.mark.parametrize("kv_type,page_size,pages", [(3, 16, 10), (-1, 16, 10), (2, 12, 10), (2, 0, 10), (2, 2048, 10), (2, 16, 0),
                                                    (2, 16, 2 ** 31 - 1)])
def test_open_paged(native, capfd, kv_type, page_size, pages):
    out = C.c_void_p()
    assert native.load().mocha_q8b_open_paged(0, None, 0, 64, 2, kv_type, page_size, pages, C.byref(out)) == 1
    assert "mocha_q8b_open_paged" in capfd.readouterr().err


def test_open_paged_type_by_name(native):
    with pytest.raises(ValueError, match="kv_type"):
        native.Q8BatchHandle(0, b"", kv_type="int8")
