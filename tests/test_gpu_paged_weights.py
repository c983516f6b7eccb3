"""Weights far below a row's largest one in the product of attention over pages, against the definition in 64 bits.

Every score is one product (a query has a single element, a key one that counts), so that a weight w = e^x, x = scale * q * k <= 0, is known but for the roundings of
scale * log2(e) (two), of the score, of its distance to a reference up to 15 above it and of the exponential: relative, (4 |x| + 14) * 2^-24 counts them.  A sum of
n weights of one sign is off by at most one rounding per addition on the longest way through it: in F32 outputs two per 32 keys for the sequences of few rows, 32 and one per 64
for the others (n / 16 + 64 is more than both), 16 per 64 where fp16 weights are added (n / 4 + 64).  128 more count the merging of waves and workgroups.  A weight enters
the product as fp16 (2^-11 of it) or as two (2^-22), or off by 2^-35 of the row's largest where that is more."""
import numpy as np
import pytest

from tests import paged_util as P

pytestmark = pytest.mark.gpu

MANY = {1: 768, 20: 128}             # sequences, two K/V heads each, from which on a row's keys are not shared out (256 compute units)


def _batch(new, n_seq, hd, k, v, page=64):
    """n_seq sequences over the same pages, which hold k and v [keys][hd] for two heads"""
    from spy_amd import _lib as H
    n = len(k)
    p = P.Paged(np.random.default_rng(n), [(new, n)], 2, 2, hd, page)
    p.k_rows[0][:], p.v_rows[0][:] = k[:, None], v[:, None]
    p.store()
    p.upload()
    up = H.DeviceBuffer.from_numpy
    p.seqs, p.n_new, p.kv = [(new, n)] * n_seq, np.full(n_seq, new), np.full(n_seq, n)
    p.table = np.repeat(p.table, n_seq, axis=0)
    p.row_start = (np.arange(n_seq + 1) * new).astype(np.int32)
    p.rows = int(p.row_start[-1]) + 3
    p.d_start, p.d_kv, p.d_table = up(p.row_start), up(p.kv.astype(np.int32)), up(p.table)
    p.batch = H.PagedBatch(n_seq, new, n, p.d_start.ptr, p.d_kv.ptr, p.d_table.ptr, p.table.shape[1])
    return p


def _check(p, q0, x, v, f32, scale=1.0):
    """outputs of all rows (not causal: all see all keys) where a query is q0 in its first element and x the scores"""
    q = np.zeros((p.rows, 2, p.hd), np.float16)
    q[:, :, 0] = q0
    got = P.run_attention(p, q, f32, causal=0, scale=scale)[:int(p.row_start[-1])].astype(np.float64)
    assert P.flag() == 0
    n, v = len(x), v.astype(np.float64)
    x = x - x.max()
    w = np.exp(x)
    total = w.sum()
    far = np.where((v != 0) & (w[:, None] > 0), -x[:, None], 0).max(axis=0)      # of the keys that an output is made of
    out = w @ v / total
    arith = 2 * (4 * far + 14) + (n / 16 if f32 else n / 4) + 64 + 128
    spread = (w * -x).sum() / total                                       # the total's own weights, each with its distance
    tol = np.abs(out) * ((arith + 4 * spread) * P.EPS32 + (2.0 ** -22 if f32 else 3 * P.EPS16)) + 2.0 ** -35 * np.abs(v).sum(axis=0) / total + (1e-30 if f32 else 2.0 ** -25)
    if not f32:
        tol = tol + np.abs(out) * n * 2.0 ** -35 / total                  # (fp16 weights in the total as well)
    off = np.abs(got - out) / tol
    print("worst error / bound %.3f" % off.max(), flush=True)
    assert np.isfinite(got).all() and off.max() <= 1, np.argwhere(~(off <= 1))[:4].tolist()


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("gap", [10.4, 14.0, 17.0])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_light_keys_beside_a_heavy_one(hip, hd, new, gap, f32):
    """A heavy key in the first tile of every wave, thousands of keys that weigh e^-gap as much behind it, which the outputs consist of."""
    print("light keys: hd %d new %d gap %g f32 %d" % (hd, new, gap, f32), flush=True)
    n = 4000
    k, v = np.zeros((n, hd), np.float16), np.ones((n, hd), np.float16)
    heavy = [5, 37, 69, 101]
    k[heavy, 0], v[heavy] = gap, 0
    _check(_batch(new, MANY[new], hd, k, v), 1.0, k[:, 0].astype(np.float64), v, f32)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("order", ["any", "ascending", "descending"])
@pytest.mark.parametrize("shared_out", [True, False])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_every_output_from_a_key_of_its_own(hip, hd, new, shared_out, order, f32):
    """V is 0 but for one key in each dimension, weights between 1 and e^-14: an output is a single weight, divided by the sum of all."""
    print("own keys: hd %d new %d shared_out %d %s f32 %d" % (hd, new, shared_out, order, f32), flush=True)
    rng = np.random.default_rng(hd + new)
    n = 4000 if shared_out else 3001
    k, v = np.zeros((n, hd), np.float16), np.zeros((n, hd), np.float16)
    x = -14 * rng.random(n)
    x = x if order == "any" else np.sort(x) if order == "ascending" else -np.sort(-x)
    k[:, 0] = x
    v[rng.permutation(n)[:hd], np.arange(hd)] = 2.0 ** 14
    _check(_batch(new, 1 if shared_out else MANY[new], hd, k, v), 1.0, k[:, 0].astype(np.float64), v, f32)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("scale", [1.0, -1.0, 3e-3, 1e24])
def test_scores_past_the_whole_numbers_of_a_float(hip, scale, new, f32):
    """Scores up to 10^9 and, by the scale, 10^33, where a float's neighbours are further apart than a reference lies below the largest: V is 1, and so are the outputs."""
    print("far scores: scale %g new %d f32 %d" % (scale, new, f32), flush=True)
    rng = np.random.default_rng(new)
    n, hd = 1500, 128
    k = np.zeros((n, hd), np.float16)
    k[:, 0] = 2.0 ** rng.uniform(0, 15, n) * rng.choice([-1, 1], n)
    for n_seq in (1, MANY[new]):
        p = _batch(new, n_seq, hd, k, np.ones((n, hd), np.float16))
        for q0 in (30000.0, 1.0, 77.0):
            q = np.zeros((p.rows, 2, hd), np.float16)
            q[:, :, 0] = q0
            got = P.run_attention(p, q, f32, causal=0, scale=scale)[:int(p.row_start[-1])].astype(np.float64)
            # a sum of weights divided by the same sum: (n / 4 + 192) additions on either side, a weight as it enters the one and the other
            assert np.abs(got - 1).max() <= 2 * (n / 4 + 192) * P.EPS32 + (2.0 ** -22 if f32 else 2 * P.EPS16), (n_seq, q0, np.abs(got - 1).max())


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n_seq", [1, MANY[1]])
def test_f16_outputs_of_few_rows_are_rounded_f32_outputs(hip, hd, n_seq):
    """Sequences of few rows take probabilities as two terms for either type: the F16 output is the F32 output rounded, to the bit."""
    print("f16 as f32: hd %d n_seq %d" % (hd, n_seq), flush=True)
    rng = np.random.default_rng(hd)
    k, v = (rng.standard_normal((1700, hd)).astype(np.float16) for _ in range(2))
    p = _batch(1, n_seq, hd, k, v)
    q = rng.standard_normal((p.rows, 2, hd)).astype(np.float16)
    a, b = P.run_attention(p, q, True, causal=0), P.run_attention(p, q, False, causal=0)
    assert np.array_equal(a[:n_seq].astype(np.float16), b[:n_seq])
