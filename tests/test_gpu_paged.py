"""Appending to a cache in pages and attention over it, against their definitions in 64 bits (tests/paged_util.py, whose tolerances count the kernels' roundings)."""
import ctypes as C

import numpy as np
import pytest

from tests import paged_util as P

pytestmark = pytest.mark.gpu
B = C.byref


def _rope(mode, dims, base=10000.0, scale=1.0, factor=1.0):
    from spy_amd import _lib as H
    return H.RopeParam(mode=mode, num_dim=dims, freq_base=base, freq_scale=scale, attention_factor=factor)


def _check_append(p, q, k, v, qo, before, mode, dims, base, scale, factor):
    want_k, want_v = before[0].astype(np.float64), before[1].astype(np.float64)
    tol_k = np.zeros_like(want_k)
    rows = set()
    for row, s, pos in p.rows_of():
        rows.add(row)
        if q is not None:
            y, size = P.rotated(q[row].astype(np.float64), pos, mode, dims, base, scale, factor)
            assert (np.abs(qo[row] - y) <= P.EPS16 * np.abs(y) + 8 * P.EPS32 * size + 2.0 ** -25).all(), (row, s, pos)
        if pos < 0:
            continue
        y, size = P.rotated(k[row].astype(np.float64), pos, mode, dims, base, scale, factor)
        p.k_at(want_k, s, pos)[:] = y
        p.k_at(tol_k, s, pos)[:] = P.EPS16 * np.abs(y) + 8 * P.EPS32 * size + 2.0 ** -25
        p.v_at(want_v, s, pos)[:] = v[row].astype(np.float16)
    got_k, got_v = p.pools()
    same = np.isnan(want_k) & np.isnan(got_k)
    assert (same | (np.abs(got_k - want_k) <= tol_k)).all()
    assert np.array_equal(got_v.astype(np.float64), want_v, equal_nan=True)
    if q is not None:
        assert (qo[[r for r in range(p.rows) if r not in rows]] == 77).all()


APPENDS = [
    # sequences (new, cached), heads, kv heads, hd, page, mode, rotated elements
    ([(1, 1)], 1, 1, 64, 16, 0, 64),
    ([(1, 1001)], 32, 32, 128, 64, 0, 128),
    ([(1, 16), (0, 40), (1, 17), (1, 64), (1, 5000)], 8, 2, 128, 16, 2, 128),
    ([(3, 3), (2, 33), (7, 100)], 6, 3, 64, 32, 0, 32),
    ([(8, 8), (1, 9), (0, 0), (30, 77)], 4, 4, 256, 16, 2, 256),
    ([(65, 130), (64, 64), (63, 200), (129, 129)], 6, 2, 128, 64, 2, 64),
    ([(200, 1111)], 5, 1, 128, 128, 0, 16),
    ([(1, 7)] * 70 + [(2, 9)], 2, 1, 64, 16, 2, 64),             # more sequences than lanes
    ([(9, 40), (0, 3)] * 40, 1, 1, 64, 1024, -1, 64),
    ([(8, 8), (1, 9), (0, 0), (130, 177)], 4, 4, 256, 16, 2, 256),
    ([(1, 700)] * 120 + [(8, 13)], 3, 1, 64, 32, 0, 48),
    ([(7, 70)] * 19, 4, 2, 128, 16, 2, 128),
]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(hip, case, dtype):
    seqs, heads, kv_heads, hd, page, mode, dims = APPENDS[case]
    print("append case %d %s" % (case, dtype.__name__), flush=True)
    rng = np.random.default_rng(case)
    p = P.Paged(rng, seqs, heads, kv_heads, hd, page, token_major=case % 2 == 1)
    p.store(upto=np.maximum(p.kv - p.n_new, 0))
    p.upload()
    q, k, v = (rng.standard_normal((p.rows, n, hd)).astype(dtype) for n in (heads, kv_heads, kv_heads))
    if case % 3 == 2:
        q = None
    base, scale, factor = (500000.0, 0.25, 1.1) if case % 2 else (10000.0, 1.0, 1.0)
    rc, qo = P.run_append(p, q, k, v, None if mode < 0 and case % 2 else _rope(mode, dims, base, scale, factor), dtype)
    assert rc == 0 and P.flag() == 0
    _check_append(p, q, k, v, qo, (p.k_pool, p.v_pool), mode, dims, base, scale, factor)


def test_append_at_far_positions(hip):
    """Angles of positions up to 2^24: a 32-bit product would be off by whole radians there."""
    rng = np.random.default_rng(5)
    for pos in (99999, 1048575, (1 << 24) - 1):
        p = P.Paged(rng, [(1, 40)], 2, 1, 128, 1024, table_spare=1)
        p.kv[:] = pos + 1                                        # the sequence's pages before the last one are not there
        p.table = np.full((1, pos // 1024 + 2), -1, np.int32)
        p.table[0, pos // 1024] = 1
        p.upload()
        q, k, v = (rng.standard_normal((p.rows, n, 128)).astype(np.float32) for n in (2, 1, 1))
        rc, qo = P.run_append(p, q, k, v, _rope(0, 128), np.float32)
        assert rc == 0 and P.flag() == 0
        _check_append(p, q, k, v, qo, (p.k_pool, p.v_pool), 0, 128, 10000.0, 1.0, 1.0)


@pytest.mark.parametrize("new", [1, 40, 45])
def test_append_without_a_place_raises_the_flag_and_stores_nothing(hip, new):
    """Pages that are not there, positions before the first: the other sequences' tokens are stored."""
    rng = np.random.default_rng(3)
    p = P.Paged(rng, [(new, 60), (new, 50), (new, 45)], 2, 1, 64, 16)
    p.upload()
    p.table[1, 49 // 16] = p.n_page                              # the last page of the second sequence
    p.d_table.upload(p.table)
    q, k, v = (rng.standard_normal((p.rows, n, 64)).astype(np.float16) for n in (2, 1, 1))
    rc, qo = P.run_append(p, q, k, v, _rope(2, 64), np.float16)
    assert rc == 0 and P.flag() != 0 and P.flag() == 0
    got_k, got_v = p.pools()
    for row, s, pos in p.rows_of():
        if s == 1 and pos // 16 == 49 // 16:
            continue
        assert np.isfinite(p.k_at(got_k, s, pos)).all() and np.array_equal(p.v_at(got_v, s, pos), v[row])
    n_stored = sum(1 for row, s, pos in p.rows_of() if not (s == 1 and pos // 16 == 49 // 16))
    assert np.isfinite(got_k).sum() == n_stored * 64 and np.isfinite(got_v).sum() == n_stored * 64


ATTENDS = [
    # sequences, heads, kv heads, hd, page, causal, window
    ([(1, 1)], 1, 1, 64, 16, 1, 0),
    ([(1, 1), (1, 31), (1, 32), (1, 33), (1, 64), (1, 127), (1, 128), (1, 129)], 4, 4, 128, 16, 1, 0),
    ([(1, 4096)], 32, 32, 128, 64, 1, 0),
    ([(1, 700), (0, 900), (1, 3000), (1, 15)], 8, 2, 128, 32, 1, 0),
    ([(1, 2500), (1, 37)], 40, 2, 64, 128, 1, 0),               # twenty query heads to a K/V head: more than one tile of rows
    ([(1, 1500), (1, 90)], 6, 2, 256, 64, 1, 0),
    ([(2, 2), (3, 50), (5, 333), (1, 600)], 6, 2, 128, 16, 1, 0),
    ([(17, 17), (16, 48), (40, 300)], 4, 4, 64, 64, 1, 0),
    ([(130, 130), (1, 400), (70, 512), (64, 64)], 6, 2, 128, 64, 1, 0),
    ([(100, 250), (33, 33)], 2, 1, 256, 32, 1, 0),
    ([(129, 1000)], 3, 1, 64, 16, 1, 0),
    ([(1, 1000), (1, 5), (1, 64)], 4, 2, 128, 16, 1, 64),
    ([(150, 700), (20, 20), (1, 300)], 4, 2, 128, 64, 1, 100),
    ([(70, 300), (1, 9)], 4, 4, 64, 32, 1, 1),                  # a window of one: every token sees itself
    ([(40, 100), (5, 5)], 2, 2, 128, 16, 0, 0),                 # all cached tokens, the later ones too
    ([(40, 100), (200, 500)], 4, 1, 64, 32, 0, 37),
    ([(1, 20)] * 70, 2, 2, 64, 16, 1, 0),
    ([(300, 300)], 5, 5, 128, 1024, 1, 0),
    ([(17, 1500)] * 60 + [(18, 2100), (40, 1040), (17, 1024), (19, 1025)], 4, 4, 64, 16, 1, 0),      # so many that no sequence's keys are shared out: long runs of tiles
    ([(17, 2200)] * 32, 8, 8, 128, 128, 1, 2050),
    ([(17, 1090)] * 64, 4, 4, 256, 32, 0, 0),
]


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention(hip, case, f32):
    """What no sequence holds is NaN in K and V."""
    seqs, heads, kv_heads, hd, page, causal, window = ATTENDS[case]
    print("attention case %d" % case, flush=True)
    rng = np.random.default_rng(100 + case)
    p = P.Paged(rng, seqs, heads, kv_heads, hd, page, token_major=case % 2 == 1)
    p.store()
    p.upload()
    q = (rng.standard_normal((p.rows, heads, hd)) * 1.5).astype(np.float16)
    got = P.run_attention(p, q, f32, causal, window)
    assert P.flag() == 0
    print("worst error / bound %.2f" % P.check_attention(p, q, got, f32, causal, window), flush=True)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("new", [1, 3, 150])
def test_attention_keeps_what_it_does_not_see_out(hip, new, f32):
    """Infinities and NaN in K and V of tokens that some rows see and others do not, behind the window and ahead of the causal limit: they reach the rows that see them
    and no others.  Few of them, so that most outputs stay finite."""
    rng = np.random.default_rng(new)
    p = P.Paged(rng, [(new, 400), (new, new + 1)], 4, 2, 128, 16)
    for s, at in ((0, 399), (0, 400 - new), (0, 330), (0, 5), (1, new)):
        d = int(rng.integers(0, 128))
        p.v_rows[s][at, 0, d] = [np.inf, -np.inf, np.nan][int(rng.integers(0, 3))]
        p.v_rows[s][at, 1, (d + 3) % 128] = np.inf
    p.store()
    p.upload()
    q = (rng.standard_normal((p.rows, 4, 128)) * 1.5).astype(np.float16)
    for window in (0, 60):
        got = P.run_attention(p, q, f32, 1, window)
        assert P.flag() == 0
        P.check_attention(p, q, got, f32, 1, window)


def test_attention_with_keys_of_nan(hip):
    """A NaN in K makes the rows that see it NaN, and no other row."""
    rng = np.random.default_rng(8)
    p = P.Paged(rng, [(60, 200)], 2, 2, 64, 32)
    p.k_rows[0][170, 1, 9] = np.nan
    p.store()
    p.upload()
    q = rng.standard_normal((p.rows, 2, 64)).astype(np.float16)
    got = P.run_attention(p, q, True)[:60]
    assert np.isfinite(got[:, 0]).all() and np.isfinite(got[:30, 1]).all() and np.isnan(got[30:, 1]).all()


@pytest.mark.parametrize("new,kv", [(1, 300), (64, 300)])
def test_attention_of_missing_pages(hip, new, kv):
    """Pages outside the pool hold nothing and raise the flag; a row all of whose pages are missing gets zeros."""
    rng = np.random.default_rng(4)
    p = P.Paged(rng, [(new, kv), (new, new), (new, kv)], 4, 2, 64, 32)
    p.store()
    hidden = {(0, 0), (0, 4)} | {(1, i) for i in range(-(-new // 32))}
    for s, i in hidden:
        p.table[s, i] = [-1, p.n_page, 1 << 30][i % 3]
    p.upload()
    q = rng.standard_normal((p.rows, 4, 64)).astype(np.float16)
    got = P.run_attention(p, q, True)
    assert P.flag() != 0
    P.check_attention(p, q, got, True, hidden=hidden)
    assert (got[p.row_start[1]:p.row_start[2]] == 0).all()
    # a window whose tokens all lie behind the missing pages: nobody asks for them
    p.table[1, :] = 0
    p.d_table.upload(p.table)
    P.run_attention(p, q, True, 1, 50)
    assert P.flag() == 0


def test_sequences_that_do_not_fit_the_launch_take_no_part(hip):
    """More cached tokens than max_kv, more new ones than max_new, rows past the tensor: the flag, and their rows are left alone."""
    rng = np.random.default_rng(6)
    p = P.Paged(rng, [(2, 90), (2, 40), (2, 60)], 2, 2, 64, 16)
    p.store()
    p.upload()
    q = rng.standard_normal((p.rows, 2, 64)).astype(np.float16)
    p.batch.max_kv = 60
    got = P.run_attention(p, q, True)
    assert P.flag() != 0 and (got[:2] == 77).all() and (got[2:6] != 77).all()
    p.batch.max_kv, p.batch.max_new = 90, 1
    got = P.run_attention(p, q, True)
    assert P.flag() != 0 and (got == 77).all()
    p.batch.max_new = 2
    p.d_start.upload(np.array([0, 2, 4, p.rows + 1], np.int32))
    got = P.run_attention(p, q, True)
    assert P.flag() != 0 and (got[:4] != 77).all() and (got[4:] == 77).all()


@pytest.mark.parametrize("heads,new,kv", [(2, 1, 200), (2, 70, 200)])
def test_pages_beyond_32_bit_offsets(hip, heads, new, kv):
    """A pool of 9 GB whose used pages lie at both ends."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(7)
    small = P.Paged(rng, [(new, kv)], heads, 2, 128, 64)
    small.store()
    bytes_page = 2 * 64 * 128 * 2
    n_page = (9 << 30) // bytes_page
    pool_k, pool_v = H.DeviceBuffer(n_page * bytes_page), H.DeviceBuffer(n_page * bytes_page)
    small.upload()
    where = {int(pg): (n_page - 1 - i if i % 2 == 0 else i) for i, pg in enumerate(small.table[0][small.table[0] >= 0])}
    for pg, to in where.items():
        pool_k.upload(small.k_pool[pg].view(np.uint16), to * bytes_page)
        pool_v.upload(small.v_pool[pg].view(np.uint16), to * bytes_page)
    table = np.array([[where.get(int(x), -1) for x in small.table[0]]], np.int32)
    small.d_table.upload(table)
    small.t_k, small.t_v = H.tensor(pool_k, H.F16, [128, 64, 2, n_page]), H.tensor(pool_v, H.F16, [64, 128, 2, n_page])
    q = rng.standard_normal((small.rows, heads, 128)).astype(np.float16)
    got = P.run_attention(small, q, True)
    assert P.flag() == 0
    P.check_attention(small, q, got, True)
    k, v = (rng.standard_normal((small.rows, 2, 128)).astype(np.float16) for _ in range(2))
    rc, _ = P.run_append(small, None, k, v, None, np.float16)
    assert rc == 0 and P.flag() == 0
    for row, s, pos in small.rows_of():
        to = int(table[0, pos // 64]) * bytes_page
        page = pool_k.download(np.float16, 2 * 64 * 128, to).reshape(2, 64, 128)
        assert np.array_equal(page[:, pos % 64], k[row])
        page = pool_v.download(np.float16, 2 * 64 * 128, to).reshape(2, 128, 64)
        assert np.array_equal(page[:, :, pos % 64], v[row])


def test_attention_of_strided_rows(hip):
    """q as a part of fused rows of q, k and v, the output as a part of wider rows, neither of which is touched elsewhere."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(9)
    p = P.Paged(rng, [(1, 50), (40, 90)], 4, 2, 64, 16)
    p.store()
    p.upload()
    wide = rng.standard_normal((p.rows, 8, 64)).astype(np.float16)
    dq = H.DeviceBuffer.from_numpy(wide.view(np.uint16))
    out = H.DeviceBuffer.from_numpy(np.full((p.rows, 6, 64), 77, np.float32))
    L = H.load()
    tq = H.tensor(dq, H.F16, [64, 4, p.rows], [2, 128, 1024], offset=256)
    to = H.tensor(out, H.F32, [64, 4, p.rows], [4, 256, 1536], offset=256)
    need = L.spy_hip_paged_attention_scratch_size(B(tq), B(p.t_k), B(p.batch))
    scratch = H.DeviceBuffer(max(need, 1))
    H.check(L.spy_hip_paged_attention(None, B(tq), B(p.t_k), B(p.t_v), B(to), B(p.batch), 0.125, 1, 0, scratch.ptr, need))
    got = out.download(np.float32).reshape(p.rows, 6, 64)
    assert (got[:, 0] == 77).all() and (got[:, 5] == 77).all()
    P.check_attention(p, wide[:, 2:6], got[:, 1:5], True)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("new", [1, 2, 64])
def test_many_keys_of_little_weight(hip, new, f32):
    """One key weighs e^10.4 times as much as each of the others, whose probabilities are subnormal fp16 numbers, and all of which together have a tenth of its weight."""
    rng = np.random.default_rng(new)
    p = P.Paged(rng, [(new, 4000)], 2, 2, 64, 64)
    p.k_rows[0][:] = 0
    p.k_rows[0][5, :, 0] = 10.4
    p.v_rows[0][:] = 1
    p.v_rows[0][5] = 0
    p.store()
    p.upload()
    q = np.zeros((p.rows, 2, 64), np.float16)
    q[:, :, 0] = 1
    got = P.run_attention(p, q, f32, scale=1.0)
    P.check_attention(p, q, got, f32, scale=1.0)


def test_missing_pages_far_into_a_long_run_of_tiles(hip):
    rng = np.random.default_rng(19)
    p = P.Paged(rng, [(17, 2200)] * 64, 4, 4, 64, 16)
    p.store()
    hidden = {(s, int(i)) for s in (0, 3, 63) for i in rng.integers(0, 136, 5)} | {(1, 64), (1, 127), (2, 63), (2, 128)}
    for s, i in hidden:
        p.table[s, i] = [-1, p.n_page][i % 2]
    p.upload()
    q = rng.standard_normal((p.rows, 4, 64)).astype(np.float16)
    got = P.run_attention(p, q, True)
    assert P.flag() != 0
    P.check_attention(p, q, got, True, hidden=hidden)


@pytest.mark.parametrize("causal", [1, 0])
def test_fewer_cached_tokens_than_new_ones(hip, causal):
    """Tokens at negative positions, an empty cache: rows that see nothing get zeros."""
    rng = np.random.default_rng(17)
    p = P.Paged(rng, [(70, 0), (1, 0), (70, 3), (20, 5), (3, 1), (2, 40)], 2, 1, 128, 16)
    p.store()
    p.upload()
    q = rng.standard_normal((p.rows, 2, 128)).astype(np.float16)
    got = P.run_attention(p, q, True, causal)
    assert P.flag() == 0
    P.check_attention(p, q, got, True, causal)
    assert (got[:71] == 0).all()


@pytest.mark.parametrize("new", [1, 40])
def test_sequences_that_share_pages(hip, new):
    """The first pages of one sequence in the table of another, as for prompts that begin alike."""
    rng = np.random.default_rng(13)
    p = P.Paged(rng, [(new, 200), (new, 150)], 4, 2, 128, 32)
    p.table[1, :3] = p.table[0, :3]
    p.k_rows[1][:96], p.v_rows[1][:96] = p.k_rows[0][:96], p.v_rows[0][:96]
    p.store()
    p.upload()
    q = rng.standard_normal((p.rows, 4, 128)).astype(np.float16)
    got = P.run_attention(p, q, True)
    assert P.flag() == 0
    P.check_attention(p, q, got, True)
