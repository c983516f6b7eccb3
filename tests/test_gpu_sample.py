"""Tokens drawn from rows of logits against the definition in 64 bits.  A token may differ from it only where the random number or a setting lies closer to a border
between tokens than the kernel's roundings: a weight is off by at most 2^-22 of itself (one rounding of max - l, relative, times a distance of at most 30, the
exponential's last bits) or 2^-44 of the largest."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
B = C.byref


def plan(l, t=1.0, k=0, p=1.0, m=0.0, u=0.0, slack=0.0):
    """(token, probability) of one row in 64 bits; slack: top-p's and the draw's borders moved by that share of the sums"""
    x = l.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    top = x.max()
    if top == -np.inf:
        return -1, 0.0
    if not t > 0:
        return int(np.argmax(x)), 1.0
    order = np.lexsort((np.arange(x.size), -x))
    with np.errstate(all="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - top) / np.float64(t))))[order]
    if 0 < k < w.size:
        w[k:] = 0
    n = w.size
    if p < 1:
        n = int(np.searchsorted(np.cumsum(w), np.float64(p) * w.sum() * (1 + slack))) + 1
    if m > 0:
        n = min(n, int((w >= min(np.float64(m), 1.0)).sum()))
    n = max(1, min(n, int((w > 0).sum())))
    kept = np.sort(order[:n])
    w = np.where(x[kept] == top, 1.0, np.exp((x[kept] - top) / np.float64(t)))
    at = int(np.searchsorted(np.cumsum(w), np.float64(u) * w.sum() * (1 + slack), side="right"))
    at = min(at, n - 1)
    return int(kept[at]), w[at] / w.sum()


def draw(hip, logits, **settings):
    from spy_amd import _lib as H
    L = H.load()
    rows, n = logits.shape
    dl = H.DeviceBuffer.from_numpy(logits)
    dev = {}
    for name, v in settings.items():
        dev[name] = H.DeviceBuffer.from_numpy(np.broadcast_to(np.asarray(v, np.int32 if name == "top_k" else np.float32), rows).copy())
    param = H.SampleParam(*(dev[n].ptr if n in dev else None for n in ("temperature", "top_k", "top_p", "min_p", "uniform")))
    tokens, probs = H.DeviceBuffer.from_numpy(np.full(rows + 1, -7, np.int32)), H.DeviceBuffer.from_numpy(np.full(rows + 1, -7, np.float32))
    tl = H.tensor(dl, H.F32, [n, rows])
    need = L.spy_hip_sample_scratch_size(B(tl))
    scratch = H.DeviceBuffer(need + 256)
    scratch.fill(0xFF)
    H.check(L.spy_hip_sample(None, B(tl), B(param), tokens.ptr, probs.ptr, scratch.ptr, need), "spy_hip_sample")
    H.sync()
    t, p = tokens.download(np.int32), probs.download(np.float32)
    assert t[-1] == -7 and p[-1] == -7 and (scratch.download(np.uint8, offset=need) == 0xFF).all()
    return t[:-1], p[:-1]


def check(hip, logits, **settings):
    rows = logits.shape[0]
    got, prob = draw(hip, logits, **settings)
    at = lambda name, r, other: np.broadcast_to(np.asarray(settings.get(name, other)), rows)[r]   # noqa: E731
    for r in range(rows):
        a = dict(t=np.float32(at("temperature", r, 1.0)), k=int(at("top_k", r, 0)), p=np.float32(at("top_p", r, 1.0)), m=np.float32(at("min_p", r, 0.0)), u=np.float32(at("uniform", r, 0.0)))
        allowed = [plan(logits[r], slack=s, **a) for s in (0.0, 2.0 ** -21, -2.0 ** -21)]
        hits = [w for tok, w in allowed if tok == got[r]]
        assert hits, (r, got[r], allowed, a)
        assert abs(prob[r] - hits[0]) <= 2.0 ** -21 * hits[0] + 2.0 ** -30, (r, prob[r], hits, a)


def logits_of(rng, rows, n):
    l = rng.standard_normal((rows, n)) * 2.5
    for r in range(rows):
        l[r, rng.integers(0, n, 12)] += 4 + 5 * rng.random(12)
    return l.astype(np.float32)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 1000, 1024, 1025, 4097, 32000, 50257, 100003, 131072, 262144])
def test_settings_of_every_kind(hip, n):
    rng = np.random.default_rng(n)
    rows = 14
    l = logits_of(rng, rows, n)
    u = rng.random(rows).astype(np.float32)
    t = (0.5 + rng.random(rows)).astype(np.float32)
    check(hip, l, uniform=u)
    check(hip, l, uniform=u, temperature=t)
    check(hip, l, uniform=u, temperature=t, top_k=np.array([1, 2, 3, 40, 0, -5, n, n + 1, max(n - 1, 1), 500, 7, 64, 5000, 100]))
    check(hip, l, uniform=u, temperature=t, top_p=np.array([0, 0.1, 0.5, 0.9, 0.95, 0.999, 0.9999, 1, 2, -1, 0.3, 0.7, 0.99999, 1e-6]))
    check(hip, l, uniform=u, temperature=t, min_p=np.array([0, 0.05, 0.1, 0.5, 1, 2, -1, 1e-6, 0.2, 0.9, 1e-12, 0.01, 0.001, 0.3]))
    check(hip, l, uniform=u, temperature=t, top_k=40, top_p=0.95, min_p=0.05)
    check(hip, l, uniform=u, temperature=np.tile([0.0, 1.0], 7), top_k=np.arange(14) * 3, top_p=0.8)
    check(hip, l, uniform=u, temperature=100.0, top_p=0.5)      # nearly flat: half of the tokens
    check(hip, l, uniform=u, temperature=0.02, top_k=9, min_p=0.2)


@pytest.mark.parametrize("n", [100, 5000, 32000, 100003])
def test_equal_logits_rank_by_index(hip, n):
    """All alike; a few values only; all alike but one: the cut falls among equal logits, by thousands."""
    rng = np.random.default_rng(n)
    u = rng.random(6).astype(np.float32)
    flat = np.full((6, n), 3.25, np.float32)
    check(hip, flat, uniform=u, top_k=[1, 7, n // 2, n - 1, 0, 99])
    check(hip, flat, uniform=u, top_p=[0.1, 0.25, 0.5, 0.75, 0.3, 0.999])
    few = rng.integers(0, 4, (6, n)).astype(np.float32)
    check(hip, few, uniform=u, top_k=[1, 7, n // 2, n - 1, n // 3, 99], top_p=[1, 0.5, 0.9, 0.95, 0.2, 0.6])
    one = flat.copy()
    one[np.arange(6), rng.integers(0, n, 6)] = 9.0
    check(hip, one, uniform=u, top_k=[1, 2, n // 2, 5, n - 1, 50], min_p=[0, 0, 1e-4, 1e-2, 0.5, 0])
    zero = np.where(rng.random((6, n)) < 0.5, np.float32(0.0), np.float32(-0.0))
    check(hip, zero, uniform=u, top_k=[1, 2, 3, n // 2, n - 1, 9])


@pytest.mark.parametrize("n", [70, 32000, 100003])
def test_masked_tokens_infinities_and_nan(hip, n):
    rng = np.random.default_rng(n)
    l = logits_of(rng, 10, n)
    hidden = rng.random((10, n)) < 0.99
    hidden[:, 5] = False
    l[hidden] = -np.inf
    l[1, 6] = np.nan
    l[2, :] = -np.inf
    l[3, :] = np.nan
    l[4, :] = np.finfo(np.float32).min                          # masked with the type's lowest value: all alike
    l[5, hidden[5]] = np.finfo(np.float32).min
    l[6, [3, 9, 60]] = np.inf
    l[7, [3, 9]] = np.inf
    l[7, 4] = np.nan
    l[8, :] = -np.inf
    l[8, n - 1] = -3e38
    u = rng.random(10).astype(np.float32)
    u[9] = 0.99999994
    for kw in ({}, {"top_k": 3}, {"top_p": 0.7}, {"min_p": 0.1}, {"top_k": 50, "top_p": 0.9, "min_p": 0.01}, {"temperature": 0.0}, {"temperature": 1e-38}, {"temperature": np.inf}):
        check(hip, l, uniform=u, **kw)
    got, prob = draw(hip, l, uniform=u)
    assert got[2] == -1 and got[3] == -1 and prob[2] == 0 and prob[3] == 0 and got[8] == n - 1 and got[6] in (3, 9, 60) and got[7] in (3, 9)


@pytest.mark.parametrize("n", [1000, 40000])
def test_temperatures_next_to_zero_and_far_masks(hip, n):
    """Masks of -inf and of the type's lowest value beside temperatures by which their distance is past the largest float: only what is as large as the maximum weighs."""
    rng = np.random.default_rng(n)
    temps = np.array([1e-3, 1e-6, 9e-8, 7e-8, 3e-8, 1e-8, 1e-12, 1e-20, 1e-30, 1e-37, 1e-40], np.float32)
    logits = np.repeat(logits_of(rng, 1, n), len(temps), axis=0)
    logits[:, rng.permutation(n)[:n // 3]] = -np.inf
    logits[:, rng.permutation(n)[:n // 3]] = np.finfo(np.float32).min
    logits[:, rng.permutation(n)[:3]] = logits[0].max()
    for a in (dict(top_p=0.9), dict(top_k=n // 2 + 600, top_p=0.9), dict(top_k=50), dict(min_p=0.1, top_p=0.5), dict()):
        check(hip, logits, temperature=temps, uniform=rng.random(len(temps)).astype(np.float32), **a)


def test_logits_further_apart_than_a_float(hip):
    """A largest and a least logit whose difference is infinite, every temperature, the flat one too."""
    rng = np.random.default_rng(2)
    logits = rng.standard_normal((4, 1500)).astype(np.float32)
    logits[:, :700] = -3e38
    logits[:, rng.permutation(1500)[:3]] = 3e38
    temps = np.array([1.0, 1e30, np.inf, 1e-9], np.float32)
    for a in (dict(top_k=40), dict(top_k=1400), dict(top_p=0.7), dict()):
        check(hip, logits, temperature=temps, uniform=np.array([0.1, 0.9, 0.999, 0.4], np.float32), **a)


def test_random_numbers_at_and_past_their_ends(hip):
    rng = np.random.default_rng(2)
    l = np.repeat(logits_of(rng, 1, 777), 8, axis=0)
    u = np.array([0.0, -0.0, -3.0, np.nan, 1.0, 7.0, np.inf, 1e-40], np.float32)
    got, _ = draw(hip, l, uniform=u, top_k=20)
    kept = np.sort(np.argsort(-l[0], kind="stable")[:20])
    assert got.tolist() == [kept[0]] * 4 + [kept[-1]] * 3 + [kept[0]]


def test_weights_of_one_row_are_drawn_as_often_as_they_weigh(hip):
    """65536 equally spaced numbers: every token as often as its probability says, to within one."""
    rng = np.random.default_rng(4)
    l = np.repeat((rng.standard_normal(40) * 1.5).astype(np.float32)[None], 65536, axis=0)
    u = (np.arange(65536) / 65536).astype(np.float32)
    got, prob = draw(hip, l, uniform=u, temperature=0.7)
    w = np.exp(l[0].astype(np.float64) / np.float64(np.float32(0.7)))
    w /= w.sum()
    assert np.abs(np.bincount(got, minlength=40) - 65536 * w).max() <= 1.01 and (np.diff(got) >= 0).all()
    assert np.abs(prob - w[got]).max() <= 2.0 ** -21


def test_results_do_not_change_from_call_to_call(hip):
    """Counts and sums come from atomics, in any order: whole numbers, so the same every time."""
    rng = np.random.default_rng(9)
    l = logits_of(rng, 64, 20000)
    u = rng.random(64).astype(np.float32)
    a = draw(hip, l, uniform=u, temperature=1.3, top_k=3000, top_p=0.97)
    for _ in range(4):
        b = draw(hip, l, uniform=u, temperature=1.3, top_k=3000, top_p=0.97)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_rows_with_a_stride(hip):
    from spy_amd import _lib as H
    rng = np.random.default_rng(1)
    wide = logits_of(rng, 5, 1003)
    dl, du, out = H.DeviceBuffer.from_numpy(wide), H.DeviceBuffer.from_numpy(rng.random(5).astype(np.float32)), H.DeviceBuffer(20)
    tl = H.tensor(dl, H.F32, [1000, 5], [4, 4012], offset=4)
    param = H.SampleParam(uniform=du.ptr)
    L = H.load()
    need = L.spy_hip_sample_scratch_size(B(tl))
    scratch = H.DeviceBuffer(max(need, 1))
    H.check(L.spy_hip_sample(None, B(tl), B(param), out.ptr, None, scratch.ptr, need))
    got, u = out.download(np.int32), du.download(np.float32)
    for r in range(5):
        assert got[r] in [plan(wide[r, 1:1001], u=u[r], slack=s)[0] for s in (0, 2.0 ** -21, -2.0 ** -21)]
