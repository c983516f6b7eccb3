"""Attention of sequences that begin alike against the definition in 64 bits (tests/paged_util.py: the tolerance counts the roundings of one pass over all keys; the pieces' sums are
added up in 32 bits beside them).  In the tables of all but a group's first sequence the pages in common are not there."""
import numpy as np
import pytest

from tests import paged_more_util as M
from tests import paged_util as P

pytestmark = pytest.mark.gpu

CASES = [
    # sequences (new, cached), groups, tokens in common, heads, kv heads, hd, page
    ([(1, 2), (1, 2)], [0, 2], [1], 1, 1, 64, 16),
    ([(1, 640), (1, 620), (1, 601), (1, 605)], [0, 4], [600], 32, 32, 128, 64),
    ([(1, 900), (1, 700), (1, 690), (1, 1000), (1, 40)], [0, 3, 4], [650, 999], 8, 2, 128, 16),
    ([(1, 500)] * 20, [0, 20], [480], 8, 2, 64, 32),             # 80 rows of a group: a tile of 128
    ([(1, 300 + i) for i in range(70)], [0, 33, 33, 68], [288, 0, 17], 4, 4, 128, 16),
    ([(1, 50)] * 3 + [(1, 1500)] * 3, [3, 6], [1490], 6, 2, 256, 64),       # sequences before the first group
    ([(40, 340), (17, 317), (1, 301), (100, 400)], [0, 4], [300], 4, 2, 128, 32),
    ([(130, 530), (1, 900), (64, 464), (0, 400), (64, 64)], [0, 4], [400], 6, 2, 64, 64),
    ([(60, 260), (90, 290), (33, 33)], [0, 2, 3], [200, 0], 2, 1, 256, 16),
    ([(2, 2000), (3, 2100), (5, 1990)], [0, 3], [1983], 4, 4, 64, 128),
    ([(1, 40)] * 140, list(range(0, 141, 2)), [33] * 70, 2, 1, 64, 16),     # more groups than lanes
    ([(1, 3000)], [0, 1], [2999], 10, 2, 128, 256),              # a group of one
    ([(300, 700), (200, 600)], [0, 2], [400], 5, 5, 128, 1024),
    ([(0, 90), (1, 100), (0, 95)], [0, 3], [90], 4, 2, 128, 16),
    # more pieces of a row than there are lanes to a head
    ([(1, 6500), (1, 6450)], [0, 2], [6300], 16, 2, 64, 128),
    ([(1, 11000), (3, 10900)], [0, 2], [10500], 4, 2, 128, 64),
    ([(1, 19000), (1, 18900)], [0, 2], [18800], 2, 1, 256, 256),
    ([(2, 9000), (1, 8000), (1, 700)], [0, 2], [300], 8, 1, 64, 16),
]


def _batch(rng, case, q8=False):
    seqs, start, length, heads, kv_heads, hd, page = CASES[case]
    p = M.PagedQ8(rng, seqs, heads, kv_heads, hd, page, token_major=case % 2 == 1)
    M.share(p, start, length)
    p.store()
    p.quantize() if q8 else None
    M.PagedQ8.upload(p) if q8 else P.Paged.upload(p)
    M.shared_batch(p, start, length, gone=[-1, p.n_page, 1 << 30][case % 3])
    return p, (rng.standard_normal((p.rows, heads, hd)) * 1.5).astype(np.float16)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_shared(hip, case, f32, q8):
    print("shared case %d" % case, flush=True)
    p, q = _batch(np.random.default_rng(300 + case), case, q8)
    got = M.run_shared(p, q, f32, q8)
    assert P.flag() == 0
    print("worst error / bound %.2f" % P.check_attention(p, q, got, f32), flush=True)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("new", [1, 70])
def test_what_is_not_finite(hip, new, f32):
    """Infinities and NaN in V, in common and not: they reach the rows that see them and no others."""
    rng = np.random.default_rng(new)
    p = P.Paged(rng, [(new, 200 + new), (new, 215 + new), (new, 230)], 4, 2, 128, 16)
    p.v_rows[0][7, 0, 3], p.v_rows[0][190, 1, 100] = np.inf, np.nan
    M.share(p, [0, 2], [200])
    p.v_rows[0][200, 0, 5], p.v_rows[1][214 + new, 0, 9], p.v_rows[1][200, 1, 0] = -np.inf, np.inf, np.nan
    p.store()
    p.upload()
    M.shared_batch(p, [0, 2], [200])
    q = (rng.standard_normal((p.rows, 4, 128)) * 1.5).astype(np.float16)
    got = M.run_shared(p, q, f32)
    assert P.flag() == 0
    P.check_attention(p, q, got, f32)


@pytest.mark.parametrize("new", [1, 70])
def test_missing_pages(hip, new):
    """Of the keys in common, which hides them from the whole group, and of a sequence's own."""
    rng = np.random.default_rng(new)
    p = P.Paged(rng, [(new, 200 + new), (new, 215 + new), (new, 230)], 4, 2, 64, 16)
    M.share(p, [0, 2], [192])
    p.store()
    p.upload()
    p.table[0, 3] = -1
    p.table[1, 12] = p.n_page
    M.shared_batch(p, [0, 2], [192])
    q = rng.standard_normal((p.rows, 4, 64)).astype(np.float16)
    got = M.run_shared(p, q, True)
    assert P.flag() != 0 and P.flag() == 0
    P.check_attention(p, q, got, True, hidden={(0, 3), (1, 3), (1, 12)})


@pytest.mark.parametrize("new", [1, 40])
def test_groups_that_do_not_fit_take_no_part(hip, new):
    """Each kind of wrong entry: the flag, the rows concerned are left alone, the others are right."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(5)
    p = P.Paged(rng, [(new, 90 + new), (new, 100 + new), (new, 70 + new), (new, 80 + new), (new, 60 + new)], 4, 2, 64, 16)
    start, length = [0, 2, 4], [90, 64]
    M.share(p, start, length)
    p.store()
    p.upload()
    M.shared_batch(p, start, length)
    q = rng.standard_normal((p.rows, 4, 64)).astype(np.float16)
    whole = M.run_shared(p, q, True)
    assert P.flag() == 0
    P.check_attention(p, q, whole, True)

    def check(left, other=(), **kw):
        """sequences `left` are left alone; those in `other` see other tokens than before"""
        fields = {n: getattr(p.prefix, n) for n in ("max_rows", "max_prefix")}
        p.d_groups.upload(np.asarray(kw.pop("start", start), np.int32))
        p.d_length.upload(np.asarray(kw.pop("length", length), np.int32))
        for n, v in kw.items():
            setattr(p.prefix, n, v)
        got = M.run_shared(p, q, True)
        assert P.flag() != 0 and P.flag() == 0
        for s in range(5):
            a, b = int(p.row_start[s]), int(p.row_start[s + 1])
            if s in left:
                assert (got[a:b] == 77).all(), s
            elif s in other:
                assert (got[a:b] != 77).all() and np.isfinite(got[a:b]).all(), s
            else:
                assert (np.abs(got[a:b] - whole[a:b]) <= 1e-5).all(), s
        assert (got[int(p.row_start[-1]):] == 77).all()
        for n, v in fields.items():
            setattr(p.prefix, n, v)

    check({0, 1}, max_prefix=80)
    check({0, 1, 2, 3}, max_rows=2 * new - 1)
    check({0, 1}, length=[91, 64])                               # more than max_prefix
    check({0}, other={1}, length=[91, 64], max_prefix=91)        # the first new token of sequence 0 would be in common
    check({0, 1}, length=[-1, 64])
    check({2, 3}, length=[90, 1 << 20])
    check({2, 3, 4}, start=[0, 2, 6])                            # sequences outside the batch
    p.batch.max_new = new                                        # a sequence that does not fit by itself: the others of its group take part
    p.d_kv.upload(np.array([90 + new, 1 << 20, 70 + new, 80 + new, 60 + new], np.int32))
    check({1})
    p.d_kv.upload(p.kv.astype(np.int32))
    assert isinstance(p.prefix, H.PagedPrefix)


def test_strided_rows_and_a_stream_of_its_own(hip):
    """q as a part of wider rows, the output as a part of wider rows, neither touched elsewhere; the same bits on another stream."""
    import ctypes as C

    from spy_amd import _lib as H
    B = C.byref
    rng = np.random.default_rng(9)
    p = P.Paged(rng, [(1, 50), (40, 90), (1, 60)], 4, 2, 64, 16)
    M.share(p, [0, 3], [48])
    p.store()
    p.upload()
    M.shared_batch(p, [0, 3], [48])
    wide = rng.standard_normal((p.rows, 8, 64)).astype(np.float16)
    dq = H.DeviceBuffer.from_numpy(wide.view(np.uint16))
    L = H.load()
    st = C.c_void_p()
    H.check(L.spy_hip_stream_create(B(st)))
    results = []
    for stream in (None, st):
        out = H.DeviceBuffer.from_numpy(np.full((p.rows, 6, 64), 77, np.float32))
        tq = H.tensor(dq, H.F16, [64, 4, p.rows], [2, 128, 1024], offset=256)
        to = H.tensor(out, H.F32, [64, 4, p.rows], [4, 256, 1536], offset=256)
        need = L.spy_hip_paged_attention_shared_scratch_size(B(tq), B(p.t_k), B(p.batch), B(p.prefix))
        scratch = H.DeviceBuffer(need)
        H.check(L.spy_hip_paged_attention_shared(stream, B(tq), B(p.t_k), None, B(p.t_v), None, B(to), B(p.batch), B(p.prefix), 0.125, scratch.ptr, need))
        H.sync(stream)
        got = out.download(np.float32).reshape(p.rows, 6, 64)
        assert (got[:, 0] == 77).all() and (got[:, 5] == 77).all()
        P.check_attention(p, wide[:, 2:6], got[:, 1:5], True)
        results.append(got)
    assert np.array_equal(results[0], results[1])
    H.check(L.spy_hip_stream_destroy(st))
