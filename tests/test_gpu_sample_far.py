"""Tokens drawn where the distance of two logits is past the largest float and the temperature as large, so that both still weigh something; and what weights are off by."""
import numpy as np
import pytest

from tests.test_gpu_sample import check, draw, logits_of

pytestmark = pytest.mark.gpu

TEMPERATURES = np.array([1e10, 1.5e18, 3e30, 1e37, 3e37, 1e38, 2e38, 3.4e38, np.inf], np.float32)


def _wide(rng, n):
    l = (rng.uniform(-3.4e38, 3.4e38, (len(TEMPERATURES), n))).astype(np.float32)
    l[:, :3] = [3.4e38, -3.4e38, 0.0]
    l[:, rng.integers(3, n, n // 8)] = -np.inf
    l[:, rng.integers(3, n, 2)] = np.nan
    return l


@pytest.mark.parametrize("n", [5, 900, 33000, 70001])
def test_distances_past_the_largest_float(hip, n):
    rng = np.random.default_rng(n)
    l = _wide(rng, n) if n > 5 else np.repeat(np.array([[3e38, -3e38, 1e38, -np.inf, 0.0]], np.float32), len(TEMPERATURES), axis=0)
    for u in (0.001, 0.5, 0.999):
        u = (u + rng.uniform(-1e-3, 1e-3, len(TEMPERATURES))).astype(np.float32)
        for a in (dict(), dict(top_p=0.9), dict(min_p=0.004), dict(top_k=max(n - 2, 1)), dict(top_k=n // 2 + 1, top_p=0.8), dict(top_k=min(n // 3 + 1, 400))):
            check(hip, l, uniform=u, temperature=TEMPERATURES, **a)


def test_the_weight_of_two_logits_at_the_ends_of_a_float(hip):
    """3e38 and -3e38 at temperature 1e38: e^-6, not what the largest float as their distance would make it."""
    l = np.repeat(np.array([[3e38, -3e38]], np.float32), 2, axis=0)
    got, prob = draw(hip, l, uniform=np.array([0.5, 0.9995], np.float32), temperature=np.float32(1e38))
    w = np.exp((l[0].astype(np.float64) - np.float64(l[0, 0])) / np.float64(np.float32(1e38)))
    assert got.tolist() == [0, 1]
    assert (np.abs(prob - w / w.sum()) <= w / w.sum() * 2.0 ** -20).all(), (prob, w / w.sum())


def test_small_logits_keep_their_rank_beside_a_large_temperature(hip):
    """Logits far below what a unit of the distances is: still ranked by their values, not by index."""
    rng = np.random.default_rng(3)
    l = (rng.permutation(2000).astype(np.float32) * np.float32(1e-42))[None].repeat(2, axis=0)
    order = np.argsort(-l[0], kind="stable")
    for k in (1, 7, 700, 1999):
        got, prob = draw(hip, l, uniform=np.array([0.0, 0.99999994], np.float32), temperature=np.float32(1e30), top_k=k)
        kept = np.sort(order[:k])
        assert got.tolist() == [kept[0], kept[-1]] and np.abs(prob - 1 / k).max() <= 2.0 ** -22 / k


@pytest.mark.parametrize("temperature", [0.3, 0.7, 1.0, 1.3, 40.0])
def test_what_a_weight_is_off_by(hip, temperature):
    """Tokens of every weight down to 2^-40 drawn one by one.  With y = log2(1 / w): max - l is off by 2^-24 of itself, y once more, which is y ln 2 * 2^-23 of the weight,
    the exponential by an ulp (2^-23), the weight's step is 2^-44; the sum by what its weights are, and the probability is rounded (2^-24)."""
    rng = np.random.default_rng(7)
    t = np.float64(np.float32(temperature))
    n = 400
    l = np.sort(rng.uniform(-40, 0, n) * np.log(2) * t + 5 * t).astype(np.float32)      # light tokens first, where uniform has fine steps
    y = (np.float64(l[-1]) - l.astype(np.float64)) * np.log2(np.e) / t
    w = 2.0 ** -y
    run = np.cumsum(w)
    u = ((run - w / 2) / run[-1]).astype(np.float32)
    off = w * (0.7 * y + 1) * 2.0 ** -23 + 2.0 ** -44
    clear = np.minimum(w / 2, run[-1] - run + w / 2) > 4 * (np.cumsum(off) + u * off.sum() + run * 2.0 ** -23)      # (some weigh less than all before them are off by)
    assert clear.sum() > n * 3 // 4 and y[clear].max() > 35
    got, prob = draw(hip, np.repeat(l[None], n, axis=0), uniform=u, temperature=np.float32(temperature))
    assert np.array_equal(got[clear], np.arange(n)[clear])
    tol = (off / w + off.sum() / run[-1] + 2.0 ** -24) * w / run[-1]
    have = np.abs(prob - w / run[-1])[clear] / tol[clear]
    print("worst error / bound %.2f, in 2^-23 of the weight %.1f" % (have.max(), (np.abs(prob * run[-1] / w - 1) * 2 ** 23)[clear][y[clear] < 20].max()), flush=True)
    assert have.max() <= 1
