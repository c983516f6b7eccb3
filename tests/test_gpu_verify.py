"""Drafted tokens against the definition in 64 bits: which are taken, what is drawn behind them, and that what comes out is distributed as the target's tokens are.
A result may differ from the definition's only where a comparison is closer than the weights' roundings: those of tests/test_gpu_sample.py, 2^-22 of a probability, and twice that for a difference
of two sums up to which every probability counts with its own; 2^-20 of the sums is allowed."""
import ctypes as C

import numpy as np
import pytest

from tests.test_gpu_paged import P
from tests.test_gpu_sample import logits_of

pytestmark = pytest.mark.gpu
B = C.byref
SLACK = 2.0 ** -20
NAMES = ("temperature", "top_k", "top_p", "min_p")


def distribution(l, t=1.0, k=0, p=1.0, m=0.0, slack=0.0):
    """probabilities of one row in 64 bits; slack: top-p's border moved by that share of the sum"""
    x = l.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    top, out = x.max(), np.zeros(x.size)
    if top == -np.inf:
        return out
    if not t > 0:
        out[np.argmax(x)] = 1.0
        return out
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
    out[order[:n]] = w[:n]
    return out / out.sum()


def run(H, logits, drafted, start, accept, uniform, settings=None, draft=None, draft_settings=None, in_place=False, stream=None):
    """tokens, accepted, probs; what lies behind them is looked at"""
    L = H.load()
    rows, n = logits.shape
    keep = []

    def up(x, t):
        keep.append(H.DeviceBuffer.from_numpy(np.ascontiguousarray(np.asarray(x, t))))
        return keep[-1].ptr

    def param(s, u=None):
        a = {n: up(np.broadcast_to(v, rows), np.int32 if n == "top_k" else np.float32) for n, v in (s or {}).items()}
        return H.SampleParam(*(a.get(n) for n in NAMES), None if u is None else up(u, np.float32))

    up(logits, np.float32)
    tl = H.tensor(keep[-1], H.F32, [n, rows])
    td = None
    if draft is not None:
        up(draft, np.float32)
        td = H.tensor(keep[-1], H.F32, [n, rows])
    pt, pd = param(settings, uniform), param(draft_settings) if draft_settings else None
    d_drafted = H.DeviceBuffer.from_numpy(np.append(np.asarray(drafted, np.int32), np.int32(-7)))
    tokens = d_drafted if in_place else H.DeviceBuffer.from_numpy(np.full(rows + 1, -7, np.int32))
    accepted, probs = H.DeviceBuffer.from_numpy(np.full(len(start), -7, np.int32)), H.DeviceBuffer.from_numpy(np.full(rows + 1, -7, np.float32))
    need = L.spy_hip_sample_verify_scratch_size(B(tl), len(start) - 1)
    scratch = H.DeviceBuffer(need + 256)
    scratch.fill(0xFF)
    H.check(L.spy_hip_sample_verify(stream, B(tl), B(pt), None if td is None else B(td), None if pd is None else B(pd), d_drafted.ptr, up(start, np.int32), len(start) - 1,
                                    up(accept, np.float32), tokens.ptr, accepted.ptr, probs.ptr, scratch.ptr, need))
    H.sync()
    assert (scratch.download(np.uint8, offset=need) == 0xFF).all()
    t, a, p = tokens.download(np.int32), accepted.download(np.int32), probs.download(np.float32)
    assert t[-1] == -7 and a[-1] == -7 and p[-1] == -7
    return t[:-1], a[:-1], p[:-1]


def number(u):
    return min(float(u), float(np.float32(0.99999994))) if u > 0 else 0.0


def fits(p, q, u_accept, u, drafted, token, prob, taken, at_end):
    """whether one row's outcome is the definition's for the distributions p and q, but for SLACK"""
    if not at_end:
        dp, dq = (p[drafted], q[drafted]) if 0 <= drafted < p.size else (0.0, 0.0)
        left, right = number(u_accept) * dq, dp
        if taken:
            return left < right + SLACK * (left + right) and token == drafted and abs(prob - dp) <= SLACK * dp + 1e-37
        if left < right - SLACK * (left + right):
            return False
    rest = p if at_end else np.maximum(p - q, 0)
    if p.sum() == 0:
        return token == -1 and prob == 0
    if not 0 <= token < p.size or not p[token] > 0 or abs(prob - p[token]) > SLACK * p[token] + 1e-37:
        return False
    if not at_end and rest.sum() <= 4 * SLACK:
        return True                                              # p and q are all but the same: any token of p's
    upto = np.cumsum(rest)
    want, off = number(u) * upto[-1], (SLACK if at_end else 2 * SLACK)
    return upto[token] >= want - off and (upto[token - 1] if token else 0.0) <= want + off


def check(got, logits, drafted, start, accept, uniform, settings=None, draft=None, draft_settings=None):
    tokens, accepted, probs = got

    def dists(l, s, r):
        a = {n: np.broadcast_to(np.asarray(v), len(logits))[r] for n, v in (s or {}).items()}
        kw = dict(t=np.float32(a.get("temperature", 1.0)), k=int(a.get("top_k", 0)), p=np.float32(a.get("top_p", 1.0)), m=np.float32(a.get("min_p", 0.0)))
        base = [distribution(l[r], **kw)]
        return base + [distribution(l[r], slack=x, **kw) for x in (SLACK, -SLACK)] if kw["p"] < 1 else base

    for s in range(len(start) - 1):
        a, b = int(start[s]), int(start[s + 1])
        if a == b:
            assert accepted[s] == -7
            continue
        stop = a + int(accepted[s])
        assert a <= stop < b, (s, accepted[s])
        for r in range(a, stop + 1):
            ps = dists(logits, settings, r)
            d = int(drafted[r])
            if r == b - 1:
                qs = [np.zeros(logits.shape[1])]
            elif draft is not None:
                qs = dists(draft, draft_settings, r)
            else:
                qs = [np.zeros(logits.shape[1])]
                if 0 <= d < logits.shape[1]:
                    qs[0][d] = 1.0
            assert any(fits(p, q, accept[r], uniform[r], d, int(tokens[r]), float(probs[r]), r < stop, r == b - 1) for p in ps for q in qs), \
                (s, r - a, stop - a, b - a, tokens[r], probs[r], d, accept[r], uniform[r])
        assert (tokens[stop + 1:b] == -1).all() and (probs[stop + 1:b] == 0).all()
    for r in [r for r in range(len(logits)) if not any(start[s] <= r < start[s + 1] for s in range(len(start) - 1))]:
        assert tokens[r] == -7 and probs[r] == -7


def case_of(rng, lens, n, near=0.7, spare=2):
    """requests with so many drafted tokens each (-1: no row at all): logits, the draft's, drafted tokens drawn from the draft's, random numbers"""
    start = np.concatenate([[0], np.cumsum([x + 1 for x in lens])])
    rows = int(start[-1]) + spare
    logits = logits_of(rng, rows, n)
    draft = (logits + near * rng.standard_normal(logits.shape)).astype(np.float32)
    accept, uniform = rng.random(rows).astype(np.float32), rng.random(rows).astype(np.float32)
    return logits, draft, start, accept, uniform


def drawn_from(rng, draft, settings=None):
    out = []
    for r in range(len(draft)):
        a = {n: np.broadcast_to(np.asarray(v), len(draft))[r] for n, v in (settings or {}).items()}
        q = distribution(draft[r], t=np.float32(a.get("temperature", 1.0)), k=int(a.get("top_k", 0)), p=np.float32(a.get("top_p", 1.0)), m=np.float32(a.get("min_p", 0.0)))
        out.append(int(np.searchsorted(np.cumsum(q), rng.random() * q.sum(), side="right")) if q.sum() else 0)
    return np.minimum(np.array(out, np.int32), draft.shape[1] - 1)


LENS = [[4], [0], [1, 0, -1, 3, 8, 2], [5] * 20, [70, 2]]
SETTINGS = [
    (None, None),
    (dict(temperature=0.8, top_k=40, top_p=0.9, min_p=0.02), dict(temperature=0.7, top_k=20)),
    (dict(temperature=1.2, top_p=0.95), dict(temperature=1.0, top_p=0.8)),
    (dict(temperature=0.9, top_k=500), dict(temperature=0.9, top_k=2000, top_p=0.97)),
    (dict(temperature=0.0), dict(temperature=0.0)),
    (dict(temperature=0.0), dict(temperature=1.0, min_p=0.1)),
    (dict(temperature=1.0, min_p=0.05), dict(temperature=0.0)),
]


@pytest.mark.parametrize("n", [7, 1000, 32000, 70001])
@pytest.mark.parametrize("case", range(len(SETTINGS)))
def test_drafts_of_a_model(hip, case, n):
    from spy_amd import _lib as H
    for lens in LENS if n <= 1000 else LENS[:3]:
        rng = np.random.default_rng(1000 * case + n + len(lens))
        logits, draft, start, accept, uniform = case_of(rng, lens, n)
        s, d = SETTINGS[case]
        drafted = drawn_from(rng, draft, d)
        got = run(H, logits, drafted, start, accept, uniform, s, draft, d, in_place=len(lens) == 1)
        if len(lens) == 1:                                       # in place: rows of no request keep what was drafted
            rest = int(start[-1])
            assert np.array_equal(got[0][rest:], drafted[rest:])
            got[0][rest:] = -7
        assert P.flag() == 0
        check(got, logits, drafted, start, accept, uniform, s, draft, d)


@pytest.mark.parametrize("n", [5, 1000, 100003])
def test_drafts_that_were_looked_up(hip, n):
    """No distribution: taken with the target's probability; else a token that is not the drafted one."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(n)
    for s in (None, dict(temperature=0.6, top_p=0.9), dict(top_k=3), dict(temperature=0.0)):
        logits, _, start, accept, uniform = case_of(rng, [3, 1, 0, 2], n)
        drafted = np.where(rng.random(len(logits)) < 0.6, logits.argmax(axis=1), rng.integers(0, n, len(logits))).astype(np.int32)
        drafted[1] = [-1, n, -(1 << 31)][n % 3]                  # outside the vocabulary: not taken
        got = run(H, logits, drafted, start, accept, uniform, s)
        assert P.flag() == 0
        check(got, logits, drafted, start, accept, uniform, s)
        assert got[1][0] <= 1


def test_settings_by_row(hip):
    from spy_amd import _lib as H
    rng = np.random.default_rng(2)
    logits, draft, start, accept, uniform = case_of(rng, [6] * 12, 5000)
    rows = len(logits)

    def some():
        return dict(temperature=np.where(rng.random(rows) < 0.2, 0, rng.uniform(0.3, 1.5, rows)).astype(np.float32), top_k=rng.choice([0, 1, 5, 60, 400, 3000], rows).astype(np.int32),
                    top_p=rng.choice([0.0, 0.3, 0.9, 1.0], rows).astype(np.float32), min_p=rng.choice([0.0, 0.01, 0.5, 2.0], rows).astype(np.float32))

    s, d = some(), some()
    drafted = drawn_from(rng, draft, d)
    check(run(H, logits, drafted, start, accept, uniform, s, draft, d), logits, drafted, start, accept, uniform, s, draft, d)


def test_same_distributions(hip):
    """The draft is the target: every token is taken, and none is refused for a rounding."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(3)
    logits, _, start, accept, uniform = case_of(rng, [7] * 30, 3001)
    accept[:] = np.float32(0.99999994)
    s = dict(temperature=0.9, top_p=0.95)
    drafted = drawn_from(rng, logits, s)
    tokens, accepted, probs = run(H, logits, drafted, start, accept, uniform, s, logits.copy(), s)
    assert (accepted == 7).all()
    check((tokens, accepted, probs), logits, drafted, start, accept, uniform, s, logits, s)


def test_infinities_nan_and_rows_without_a_token(hip):
    from spy_amd import _lib as H
    rng = np.random.default_rng(4)
    logits, draft, start, accept, uniform = case_of(rng, [2] * 16 + [0] * 4, 901)
    rows = len(logits)
    for x in (logits, draft):
        for r in range(rows):
            kind = int(rng.integers(0, 6))
            if kind == 0:
                x[r] = -np.inf
            elif kind == 1:
                x[r, rng.integers(0, 901, 3)] = np.inf
            elif kind == 2:
                x[r, rng.random(901) < 0.9] = -np.inf
            elif kind == 3:
                x[r, rng.random(901) < 0.5] = np.nan
    accept[::7], uniform[::5], accept[3], uniform[4], accept[5], uniform[6] = np.nan, np.nan, 1.5, 1.0, -1, -2
    drafted = drawn_from(rng, draft)
    got = run(H, logits, drafted, start, accept, uniform, None, draft)
    assert P.flag() == 0
    check(got, logits, drafted, start, accept, uniform, None, draft)
    assert (got[0] == -1).any()


@pytest.mark.parametrize("drafter", [True, False])
def test_what_comes_out_is_distributed_as_the_target(hip, drafter):
    """20000 requests with one drafted token over the same 12 logits: how often each token comes first, against p.  A count's deviation is sqrt(n p (1 - p)): five of them are allowed (of
    12 counts one beyond in two million), and the seed is fixed."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(6)
    n, vocab = 20000, 12
    l, d = rng.standard_normal(vocab).astype(np.float32) * 1.5, rng.standard_normal(vocab).astype(np.float32) * 1.5
    logits, draft = np.broadcast_to(l, (2 * n, vocab)), np.broadcast_to(d, (2 * n, vocab))
    start = np.arange(0, 2 * n + 1, 2)
    accept, uniform = rng.random(2 * n).astype(np.float32), rng.random(2 * n).astype(np.float32)
    p, q = distribution(l, p=np.float32(0.9)), distribution(d)
    drafted = rng.choice(vocab, 2 * n, p=q if drafter else np.full(vocab, 1 / vocab)).astype(np.int32)
    tokens, accepted, _ = run(H, logits, drafted, start, accept, uniform, dict(top_p=0.9), draft if drafter else None)
    count = np.bincount(tokens[::2], minlength=vocab)
    assert (np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p)) + 1e-9).all(), (count / n, p)
    share = np.minimum(p, q).sum() if drafter else p.mean()      # of the drafts that are taken
    assert abs(accepted.mean() - share) <= 5 * np.sqrt(share * (1 - share) / n)
    second = tokens[1::2][accepted == 1]                         # behind a taken draft: the target's again
    count = np.bincount(second, minlength=vocab)
    assert (np.abs(count - len(second) * p) <= 5 * np.sqrt(len(second) * p * (1 - p)) + 1e-9).all()


def test_requests_that_do_not_fit_are_left_alone(hip):
    from spy_amd import _lib as H
    rng = np.random.default_rng(7)
    logits, draft, start, accept, uniform = case_of(rng, [2, 1, 3], 300)
    drafted = drawn_from(rng, draft)
    want = run(H, logits, drafted, start, accept, uniform, None, draft)
    bad = start.copy()
    bad[-1] = len(logits) + 1
    got = run(H, logits, drafted, bad, accept, uniform, None, draft)
    assert P.flag() != 0 and P.flag() == 0
    assert got[1][-1] == -7 and (got[0][start[2]:] == -7).all()
    assert all(np.array_equal(g[:k], w[:k]) for g, w, k in zip(got, want, (start[2], 2, start[2])))
    bad = start.copy()
    bad[0] = -1
    got = run(H, logits, drafted, bad, accept, uniform, None, draft)
    assert P.flag() != 0 and got[1][0] == -7 and np.array_equal(got[0][start[1]:], want[0][start[1]:])


@pytest.mark.parametrize("start, alone", [([0, 3, 1, 6], [1, 2]), ([0, 2, 9, 1, 4], [1, 2, 3]), ([5, 7, 0, 4], [1, 2]), ([2, 4, 4, 3, 8], [2, 3])])
@pytest.mark.parametrize("drafter", [True, False])
def test_requests_that_begin_before_one_in_front_of_them(hip, start, alone, drafter):
    """Left alone, whatever their rows; the others are as if by themselves."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(8)
    logits, draft = (rng.standard_normal((8, 1500)).astype(np.float32) for _ in range(2))
    accept, uniform = rng.random(8).astype(np.float32), rng.random(8).astype(np.float32)
    drafted = drawn_from(rng, draft)
    tokens, accepted, probs = run(H, logits, drafted, np.asarray(start, np.int32), accept, uniform, dict(top_p=0.9), draft if drafter else None)
    assert P.flag() != 0
    sound = np.zeros(8, bool)
    for s in range(len(start) - 1):
        if s in alone:
            assert accepted[s] == -7
            continue
        a, b = start[s], start[s + 1]
        sound[a:b] = True
        if a < b:
            one = np.array([0, b - a])
            check((tokens[a:b], accepted[s:s + 1], probs[a:b]), logits[a:b], drafted[a:b], one, accept[a:b], uniform[a:b], dict(top_p=0.9), draft[a:b] if drafter else None)
    assert (tokens[~sound] == -7).all() and (probs[~sound] == -7).all()


def test_strided_rows_and_replays(hip):
    """Rows that are parts of wider ones, 4 bytes aligned; a recorded call replayed with other drafts, rows and numbers between eager calls."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(8)
    L = H.load()
    n, rows = 1001, 12
    wide = H.DeviceBuffer.from_numpy(np.zeros((rows, 2 * n + 3), np.float32))
    tl = H.tensor(wide, H.F32, [n, rows], [4, 4 * (2 * n + 3)], offset=4)
    td = H.tensor(wide, H.F32, [n, rows], [4, 4 * (2 * n + 3)], offset=4 * (n + 2))
    full = lambda t, k=rows: H.DeviceBuffer.from_numpy(np.zeros(k, t))                            # noqa: E731
    drafted, start, accept, uniform, tokens, accepted, probs = full(np.int32), full(np.int32, 4), full(np.float32), full(np.float32), full(np.int32), full(np.int32, 3), full(np.float32)
    top_p = H.DeviceBuffer.from_numpy(np.full(rows, 0.9, np.float32))
    param, dparam = H.SampleParam(None, None, top_p.ptr, None, uniform.ptr), H.SampleParam(None, None, top_p.ptr, None, None)
    need = L.spy_hip_sample_verify_scratch_size(B(tl), 3)
    scratch = H.DeviceBuffer(need)
    call = lambda st: H.check(L.spy_hip_sample_verify(st, B(tl), B(param), B(td), B(dparam), drafted.ptr, start.ptr, 3, accept.ptr, tokens.ptr, accepted.ptr, probs.ptr, scratch.ptr, need))   # noqa: E731
    st, graph = C.c_void_p(), C.c_void_p()
    H.check(L.spy_hip_stream_create(B(st)))
    s = dict(top_p=0.9)
    for turn in range(6):
        lens = [[3, 3, 3], [0, 5, 1], [4, -1, 2], [1, 1, 7], [10, -1, 0], [2, 2, 2]][turn]
        logits, draft, at, a, u = case_of(rng, lens, n, spare=rows - sum(x + 1 for x in lens))
        d = drawn_from(rng, draft, s)
        host = np.full((rows, 2 * n + 3), np.nan, np.float32)
        host[:, 1:n + 1], host[:, n + 2:2 * n + 2] = logits, draft
        for buf, x, t in ((wide, host, np.float32), (drafted, d, np.int32), (start, at, np.int32), (accept, a, np.float32), (uniform, u, np.float32), (tokens, np.full(rows, -7), np.int32),
                          (accepted, np.full(3, -7), np.int32), (probs, np.full(rows, -7), np.float32)):
            buf.upload(np.asarray(x, t))
        H.sync()
        if turn == 0:
            call(st)
        elif turn == 1:
            H.check(L.spy_hip_capture_begin(st))
            call(st)
            H.check(L.spy_hip_capture_end(st, B(graph)))
        if turn:
            H.check(L.spy_hip_graph_launch(graph, st))
        H.sync(st)
        got = tokens.download(np.int32), accepted.download(np.int32), probs.download(np.float32)
        check(got, logits, d, at, a, u, s, draft, s)
        call(None)
        H.sync()
        assert all(np.array_equal(x, y) for x, y in zip(got, (tokens.download(np.int32), accepted.download(np.int32), probs.download(np.float32))))
    H.check(L.spy_hip_graph_destroy(graph))
    H.check(L.spy_hip_stream_destroy(st))
