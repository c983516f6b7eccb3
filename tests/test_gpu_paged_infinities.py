"""Infinities and NaN in V: an output is what the kinds that its row sees in its dimension add up to (+inf, -inf, or NaN for both or a NaN), whatever the weight, the place
in a tile, the window or the causal limit; rows that see none have finite outputs."""
import numpy as np
import pytest

from tests import paged_util as P

pytestmark = pytest.mark.gpu


def _kinds(v, seen):
    """[rows][hd]: 0 finite, else the value that an output has to be"""
    plus, minus, nan = (seen @ m.astype(np.int64) > 0 for m in (np.isposinf(v), np.isneginf(v), np.isnan(v)))
    out = np.where(plus, np.inf, np.where(minus, -np.inf, 0.0))
    return np.where(nan | (plus & minus), np.nan, out)


def _check(p, q, got, f32, causal, window, scale):
    n_kinds = set()
    g = p.heads // p.kv_heads
    for s in range(len(p.seqs)):
        new, kv, r0 = int(p.n_new[s]), int(p.kv[s]), int(p.row_start[s])
        pos, j = np.arange(kv - new, kv), np.arange(kv)
        seen = (j[None] <= pos[:, None]) | (not causal)
        if window:
            seen = seen & (j[None] > pos[:, None] - window)
        for h in range(p.heads):
            k, v = p.k_rows[s][:, h // g], p.v_rows[s][:, h // g]
            kinds = _kinds(v, seen.astype(np.int64))
            have = got[r0:r0 + new, h].astype(np.float64)
            finite = kinds == 0
            assert np.array_equal(np.isfinite(have), finite) and np.array_equal(have[~finite], kinds[~finite], equal_nan=True), (s, h, have[~finite][:4], kinds[~finite][:4])
            n_kinds |= {str(x) for x in np.unique(kinds[~finite])}
            want, tol = P.attention(q[r0:r0 + new, h], k, np.where(np.isfinite(v), v, 0), pos, scale, causal, window, f32)
            assert (np.abs(have - want)[finite] <= tol[finite]).all(), (s, h)
    return n_kinds


CASES = [
    # sequences, heads, kv heads, hd, page, causal, window
    ([(1, 700), (3, 300), (1, 40)], 4, 2, 128, 16, 1, 0),
    ([(1, 3000)], 2, 2, 64, 64, 1, 0),
    ([(1, 900), (2, 500)], 4, 2, 256, 32, 1, 100),
    ([(150, 700), (20, 333), (1, 300)], 4, 2, 128, 64, 1, 0),
    ([(300, 300)], 4, 4, 64, 16, 1, 0),
    ([(150, 400), (40, 200)], 2, 2, 256, 64, 1, 0),
    ([(70, 900), (33, 400)], 2, 2, 128, 32, 1, 130),
    ([(40, 900)], 4, 1, 64, 32, 0, 0),
    ([(17, 1100)] * 70, 4, 4, 128, 64, 1, 0),                    # no sequence's keys shared out
    ([(1, 200)] * 900, 2, 2, 64, 64, 1, 0),
]


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_kinds_of_infinities(hip, case, f32):
    seqs, heads, kv_heads, hd, page, causal, window = CASES[case]
    print("infinities: case %d f32 %d" % (case, f32), flush=True)
    rng = np.random.default_rng(case)
    p = P.Paged(rng, seqs, heads, kv_heads, hd, page)
    for s, (new, kv) in enumerate(seqs):
        for at in {0, kv - 1, kv - new, kv // 2, *rng.integers(0, kv, 6).tolist()}:
            for h in range(kv_heads):
                for value in (np.inf, -np.inf, np.nan):
                    if rng.random() < 0.6:
                        p.v_rows[s][at, h, int(rng.integers(0, hd))] = value
        for h in range(kv_heads):                                # one dimension with many of one sign, one with both
            p.v_rows[s][rng.integers(0, kv, 20), h, 1] = np.inf
            p.v_rows[s][rng.integers(0, kv, 2), h, 2] = [np.inf, -np.inf]
    p.store()
    p.upload()
    q = (rng.standard_normal((p.rows, heads, hd)) * 1.5).astype(np.float16)
    scale = 1.0 / np.sqrt(hd)
    got = P.run_attention(p, q, f32, causal, window)
    assert P.flag() == 0
    kinds = _check(p, q, got, f32, causal, window, scale)
    assert kinds == {"inf", "-inf", "nan"}
    assert (got[int(p.row_start[-1]):].astype(np.float64) == 77).all()
    again = P.run_attention(p, q, f32, causal, window)
    assert np.array_equal(got, again, equal_nan=True)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("gap", [12.0, 60.0, 400.0])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("n_seq", [1, 400])
def test_an_infinity_of_hardly_any_weight(hip, n_seq, new, gap, f32):
    """Keys whose weight is e^-gap of the row's largest, down to less than a float holds, in tiles that all rows see whole, before and behind the heavy one."""
    print("light infinities: n_seq %d new %d gap %g" % (n_seq, new, gap), flush=True)
    rng = np.random.default_rng(new)
    kv = 1000
    p = P.Paged(rng, [(new, kv)] * n_seq, 2, 2, 128, 64)
    for s in range(n_seq):
        p.k_rows[s][:] = 0
        p.k_rows[s][500, :, 0] = gap
        p.v_rows[s][3, :, 0], p.v_rows[s][700, :, 1], p.v_rows[s][130, :, 2], p.v_rows[s][131, :, 3], p.v_rows[s][800, :, 3] = np.inf, -np.inf, np.nan, -np.inf, np.inf
    p.store()
    p.upload()
    q = np.zeros((p.rows, 2, 128), np.float16)
    q[:, :, 0] = 1
    got = P.run_attention(p, q, f32, scale=1.0)[:int(p.row_start[-1])].astype(np.float64)
    assert P.flag() == 0
    want = np.array([np.inf, -np.inf, np.nan, np.nan])
    assert np.array_equal(got[:, :, :4], np.broadcast_to(want, got[:, :, :4].shape), equal_nan=True), got[0, 0, :4]
    assert np.isfinite(got[:, :, 4:]).all()


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("what", [np.nan, np.inf])
@pytest.mark.parametrize("new", [1, 60])
def test_a_key_of_nan_or_infinity_voids_the_rows_that_see_it(hip, new, what, f32):
    """A score of NaN, or of +inf, which a softmax turns into NaN: the row is NaN in all dimensions, infinities in V or not; the others are as they were."""
    rng = np.random.default_rng(8)
    p = P.Paged(rng, [(new, 200), (new, 150)], 2, 2, 64, 32)
    at = 170 if new > 1 else 100
    p.k_rows[0][at, 1, 9] = what
    p.v_rows[0][20, :, 5] = np.inf
    p.store()
    p.upload()
    q = rng.standard_normal((p.rows, 2, 64)).astype(np.float16)
    q[:, :, 9] = 1
    got = P.run_attention(p, q, f32).astype(np.float64)
    first = max(at - (200 - new), 0)
    assert np.isnan(got[first:new, 1]).all() and np.isposinf(got[:first, 1, 5]).all() and np.isposinf(got[:new, 0, 5]).all()
    rest = np.arange(64) != 5
    assert np.isfinite(got[:first, 1][:, rest]).all() and np.isfinite(got[:new, 0][:, rest]).all() and np.isfinite(got[new:2 * new]).all()
