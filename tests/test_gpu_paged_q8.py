"""A cache in pages of 8 bits: what is stored against Q8_0's arithmetic and the definition in 64 bits; attention over it against attention over fp16 pages that hold the same
values, bit for bit, and against its definition."""
import ctypes as C

import numpy as np
import pytest

from tests import paged_more_util as M
from tests import paged_util as P
from tests.test_gpu_paged import APPENDS, ATTENDS, _rope

pytestmark = pytest.mark.gpu
B = C.byref


def _stored(p, before, rows, new):
    """that the pools on the device are `before` but for the new tokens' places; those of token (sequence, position): (K numbers, K scales, V numbers, V scales)"""
    after = [x.copy() for x in p.q8_pools()]
    got = {}
    for row, s, pos in rows:
        page, at = p.table[s, pos // p.page], pos % p.page
        k = (page, at) if p.token_major else (page, slice(None), at)
        places = (k, (page, slice(None), at), (page, slice(None), slice(None), at), (page, slice(None), slice(None), at))
        got[row] = [after[i][w].copy() for i, w in enumerate(places)]
        for i, w in enumerate(places):
            after[i][w] = before[i][w]
    assert all(np.array_equal(x.view(np.uint8), y.view(np.uint8)) for x, y in zip(after, before)), "places of no new token"
    return got


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(hip, case, dtype):
    seqs, heads, kv_heads, hd, page, mode, dims = APPENDS[case]
    print("append case %d %s" % (case, dtype.__name__), flush=True)
    rng = np.random.default_rng(case)
    p = M.PagedQ8(rng, seqs, heads, kv_heads, hd, page, token_major=case % 2 == 1)
    p.quantize()
    p.upload()
    before = [x.copy() for x in p.q8_pools()]
    q, k, v = ((rng.standard_normal((p.rows, n, hd)) * np.exp(rng.uniform(-6, 3, (p.rows, n, 1)))).astype(dtype) for n in (heads, kv_heads, kv_heads))
    if case % 3 == 2:
        q = None
    base, scale, factor = (500000.0, 0.25, 1.1) if case % 2 else (10000.0, 1.0, 1.0)
    rope = None if mode < 0 and case % 2 else _rope(mode, dims, base, scale, factor)
    rc, qo = M.run_append_q8(p, q, k, v, rope, dtype)
    assert rc == 0 and P.flag() == 0
    rows = [r for r in p.rows_of() if r[2] >= 0]
    got = _stored(p, before, rows, p.n_new)
    for row, s, pos in rows:
        kq, kd, vq, vd = got[row]
        wq, wd = M.q8_blocks(v[row])                             # V as Q8_0 has it, bit for bit
        assert np.array_equal(vq, wq) and np.array_equal(vd, wd), (row, s, pos)
        if mode < 0:
            wq, wd = M.q8_blocks(k[row])
            assert np.array_equal(kq, wq) and np.array_equal(kd, wd), (row, s, pos)
            continue
        # K is turned first, in 32 bits: off by 8 steps of the pair's size; then a step of the block at most half, its scale's rounding and that of the value read back
        y, size = P.rotated(k[row].astype(np.float64), pos, mode, dims, base, scale, factor)
        off = 8 * P.EPS32 * size
        top = (np.abs(y) + off).reshape(kv_heads, -1, 32).max(axis=2)
        d = top / 127
        tol = np.repeat(d * (0.5 + 2.0 ** -15) + 127 * (P.EPS16 * d + 2.0 ** -25), 32, axis=1) + off + P.EPS16 * (np.abs(y) + np.repeat(d, 32, axis=1)) + 2.0 ** -25
        value = M.q8_values(kq, kd).astype(np.float64)
        assert (np.abs(value - y) <= tol).all(), (row, s, pos, np.abs(value - y).max())
        assert (np.abs(kq.reshape(kv_heads, -1, 32).astype(int)).max(axis=2) == 127).all()
    # q_out is that of appending to fp16 pages
    if q is not None:
        rc, want = P.run_append(p, q, k, v, rope, dtype)
        assert rc == 0 and np.array_equal(qo.view(np.uint16), want.view(np.uint16))
        assert (qo[int(p.row_start[-1]):] == 77).all()


@pytest.mark.parametrize("new", [1, 40, 130])
def test_append_of_blocks_that_are_not_numbers(hip, new):
    """Infinities, NaN, magnitudes past what fp16 scales hold, blocks of zeros and of the smallest numbers: their blocks, and no others."""
    rng = np.random.default_rng(new)
    p = M.PagedQ8(rng, [(new, new + 30), (new, new)], 2, 2, 128, 16)
    p.quantize()
    p.upload()
    k, v = (rng.standard_normal((p.rows, 2, 128)).astype(np.float32) for _ in range(2))
    for x in (k, v):
        for value in (np.inf, -np.inf, np.nan, 8.4e6, 8.3e6, 3e38, 0.0, 1e-30, 1e-40):
            row, head, block = (int(rng.integers(0, n)) for n in (2 * new, 2, 4))
            if abs(value) < 1:
                x[row, head, 32 * block:32 * block + 32] = value
            else:
                x[row, head, 32 * block + int(rng.integers(0, 32))] = value
    rc, _ = M.run_append_q8(p, None, k, v, None, np.float32)
    assert rc == 0 and P.flag() == 0
    kq, kd, vq, vd = p.q8_pools()
    for row, s, pos in p.rows_of():
        page, at = p.table[s, pos // p.page], pos % p.page
        for got_q, got_d, x in ((kq[page, :, at], kd[page, :, at], k[row]), (vq[page, :, :, at], vd[page, :, :, at], v[row])):
            wq, wd = M.q8_blocks(x)
            assert np.array_equal(got_d, wd, equal_nan=True)
            fine = np.repeat(np.isfinite(wd), 32, axis=1)
            assert np.array_equal(got_q[fine], wq[fine])


@pytest.mark.parametrize("new", [1, 40, 130])
def test_append_without_a_place_raises_the_flag_and_stores_nothing(hip, new):
    rng = np.random.default_rng(3)
    p = M.PagedQ8(rng, [(new, 160), (new, 150), (new, 145)], 2, 1, 64, 16)
    p.quantize()
    p.upload()
    before = [x.copy() for x in p.q8_pools()]
    lost = p.table[1, 149 // 16]
    p.table[1, 149 // 16] = p.n_page
    p.d_table.upload(p.table)
    q, k, v = (rng.standard_normal((p.rows, n, 64)).astype(np.float16) for n in (2, 1, 1))
    rc, _ = M.run_append_q8(p, q, k, v, _rope(2, 64), np.float16)
    assert rc == 0 and P.flag() != 0 and P.flag() == 0
    rows = [r for r in p.rows_of() if not (r[1] == 1 and r[2] // 16 == 149 // 16)]
    got = _stored(p, before, rows, p.n_new)
    for row, s, pos in rows:
        wq, wd = M.q8_blocks(v[row])
        assert np.array_equal(got[row][2], wq) and np.array_equal(got[row][3], wd)
    assert lost != p.n_page


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention(hip, case, f32):
    """What no sequence holds has scales of NaN."""
    seqs, heads, kv_heads, hd, page, causal, window = ATTENDS[case]
    print("attention case %d" % case, flush=True)
    rng = np.random.default_rng(100 + case)
    p = M.PagedQ8(rng, seqs, heads, kv_heads, hd, page, token_major=case % 2 == 1)
    p.store()
    p.quantize()
    p.upload()
    q = (rng.standard_normal((p.rows, heads, hd)) * 1.5).astype(np.float16)
    got = M.run_attention_q8(p, q, f32, causal, window)
    assert P.flag() == 0
    want = P.run_attention(p, q, f32, causal, window)
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
    if case in (1, 5, 8, 9, 11, 13):
        print("worst error / bound %.2f" % P.check_attention(p, q, got, f32, causal, window), flush=True)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("new", [1, 3, 150])
def test_attention_keeps_what_it_does_not_see_out(hip, new, f32):
    """Blocks of NaN in V, of tokens that some rows see and others do not; scales so large that values are infinite."""
    rng = np.random.default_rng(new)
    p = M.PagedQ8(rng, [(new, 400), (new, new + 1)], 4, 2, 128, 16)
    for s, at in ((0, 399), (0, 400 - new), (0, 330), (0, 5), (1, new)):
        p.v_rows[s][at, 0, int(rng.integers(0, 128))] = np.nan
    p.store()
    p.quantize()
    for s, at in ((0, 399 - new // 2), (0, 12)):                 # one block: -inf, +inf and zeros
        page, o = p.table[s, at // 16], at % 16
        p.v_d[page, 1, 2, o] = 60000
        p.v_pool[page, 1, 64:96, o] = M.q8_values(p.v_q[page, 1, 64:96, o], p.v_d[page, 1, 2:3, o])
        p.v_rows[s][at, 1] = p.v_pool[page, 1, :, o]
    assert np.isinf(p.v_pool).any() and np.isnan(p.v_rows[0]).sum() == 4 * 32
    p.upload()
    q = (rng.standard_normal((p.rows, 4, 128)) * 1.5).astype(np.float16)
    for window in (0, 60):
        got = M.run_attention_q8(p, q, f32, 1, window)
        assert P.flag() == 0
        P.check_attention(p, q, got, f32, 1, window)


def test_attention_with_keys_of_nan(hip):
    rng = np.random.default_rng(8)
    p = M.PagedQ8(rng, [(60, 200)], 2, 2, 64, 32)
    p.k_rows[0][170, 1, 9] = np.nan
    p.store()
    p.quantize()
    p.upload()
    q = rng.standard_normal((p.rows, 2, 64)).astype(np.float16)
    got = M.run_attention_q8(p, q, True)[:60]
    assert np.isfinite(got[:, 0]).all() and np.isfinite(got[:30, 1]).all() and np.isnan(got[30:, 1]).all()


@pytest.mark.parametrize("new,kv", [(1, 300), (64, 300)])
def test_attention_of_missing_pages(hip, new, kv):
    rng = np.random.default_rng(4)
    p = M.PagedQ8(rng, [(new, kv), (new, new), (new, kv)], 4, 2, 64, 32)
    p.store()
    p.quantize()
    hidden = {(0, 0), (0, 4)} | {(1, i) for i in range(-(-new // 32))}
    for s, i in hidden:
        p.table[s, i] = [-1, p.n_page, 1 << 30][i % 3]
    p.upload()
    q = rng.standard_normal((p.rows, 4, 64)).astype(np.float16)
    got = M.run_attention_q8(p, q, True)
    assert P.flag() != 0
    P.check_attention(p, q, got, True, hidden=hidden)
    assert (got[p.row_start[1]:p.row_start[2]] == 0).all()


@pytest.mark.parametrize("causal", [1, 0])
def test_fewer_cached_tokens_than_new_ones(hip, causal):
    rng = np.random.default_rng(17)
    p = M.PagedQ8(rng, [(70, 0), (1, 0), (70, 3), (20, 5), (3, 1), (2, 40)], 2, 1, 128, 16)
    p.store()
    p.quantize()
    p.upload()
    q = rng.standard_normal((p.rows, 2, 128)).astype(np.float16)
    got = M.run_attention_q8(p, q, True, causal)
    assert P.flag() == 0
    P.check_attention(p, q, got, True, causal)
    assert (got[:71] == 0).all()


@pytest.mark.parametrize("new,kv", [(1, 200), (70, 200)])
def test_pages_beyond_32_bit_offsets(hip, new, kv):
    """Pools of 5 GB (and scales of 0.3 GB) whose used pages lie at both ends."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(7)
    small = M.PagedQ8(rng, [(new, kv)], 2, 2, 128, 64)
    small.store()
    small.quantize()
    small.upload()
    size, scales = 2 * 64 * 128, 2 * 64 * 4 * 2
    n_page = (5 << 30) // size
    pools = [H.DeviceBuffer(n_page * n) for n in (size, scales, size, scales)]
    where = {int(pg): (n_page - 1 - i if i % 2 == 0 else i) for i, pg in enumerate(small.table[0][small.table[0] >= 0])}
    for pg, to in where.items():
        for buf, x, n in zip(pools, (small.k_q, small.k_d, small.v_q, small.v_d), (size, scales, size, scales)):
            buf.upload(x[pg].view(np.uint8), to * n)
    small.d_table.upload(np.array([[where.get(int(x), -1) for x in small.table[0]]], np.int32))
    small.t_kq, small.t_vq = H.tensor(pools[0], H.I8, [128, 64, 2, n_page]), H.tensor(pools[2], H.I8, [64, 128, 2, n_page])
    small.t_kd, small.t_vd = H.tensor(pools[1], H.F16, [4, 64, 2, n_page]), H.tensor(pools[3], H.F16, [64, 4, 2, n_page])
    q = rng.standard_normal((small.rows, 2, 128)).astype(np.float16)
    got = M.run_attention_q8(small, q, True)
    assert P.flag() == 0
    P.check_attention(small, q, got, True)
    k, v = (rng.standard_normal((small.rows, 2, 128)).astype(np.float16) for _ in range(2))
    rc, _ = M.run_append_q8(small, None, k, v, None, np.float16)
    assert rc == 0 and P.flag() == 0
    for row, s, pos in small.rows_of():
        to, at = where[int(small.table[0, pos // 64])], pos % 64
        for i, x in ((0, k[row]), (2, v[row])):
            wq, wd = M.q8_blocks(x)
            page, d = pools[i].download(np.int8, size, to * size), pools[i + 1].download(np.float16, scales // 2, to * scales)
            page, d = (page.reshape(2, 64, 128)[:, at], d.reshape(2, 64, 4)[:, at]) if i == 0 else (page.reshape(2, 128, 64)[:, :, at], d.reshape(2, 4, 64)[:, :, at])
            assert np.array_equal(page, wq) and np.array_equal(d, wd)
