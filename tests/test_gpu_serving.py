"""Requests served together: rows of an embedding table as q, k and v, appended to a paged cache, attention over it, its rows as logits, tokens drawn from them, which are
the next step's rows.  Each step against the definitions in 64 bits (tests/paged_util.py, tests/test_gpu_sample.py), as eager calls and as one recorded graph."""
import ctypes as C

import numpy as np
import pytest

from tests import paged_util as P
from tests.test_gpu_sample import plan

pytestmark = pytest.mark.gpu
B = C.byref
HEADS, KV, HD, PAGE = 4, 2, 64, 16
VOCAB = HEADS * HD


class Step:
    """The buffers of one kind of step (so many rows at most) and its four calls."""

    def __init__(self, H, p, table, rope, rows, max_new, max_kv, rng):
        self.H, self.p, self.rows, self.rope = H, p, rows, rope
        width = (HEADS + 2 * KV) * HD
        full = lambda shape, t, v: H.DeviceBuffer.from_numpy(np.full(shape, v, t))                # noqa: E731
        self.ids, self.x = full(rows, np.int32, 0), full((rows, width), np.float32, 0)
        self.q16, self.out = full((rows, HEADS, HD), np.float16, 77), full((rows, VOCAB), np.float32, 77)
        self.tokens, self.uniform = full(rows, np.int32, -7), full(rows, np.float32, 0)
        self.temperature, self.top_k = full(rows, np.float32, 0.25), full(rows, np.int32, 40)
        self.start, self.kv = full(len(p.seqs) + 1, np.int32, 0), full(len(p.seqs), np.int32, 0)
        self.batch = H.PagedBatch(len(p.seqs), max_new, max_kv, self.start.ptr, self.kv.ptr, p.d_table.ptr, p.table.shape[1])
        self.table = table
        self.t_ids, self.t_x = H.tensor(self.ids, H.I32, [rows]), H.tensor(self.x, H.F32, [width, rows])
        part = lambda heads, first: H.tensor(self.x, H.F32, [HD, heads, rows], [4, HD * 4, width * 4], offset=first * HD * 4)   # noqa: E731
        self.t_q, self.t_k, self.t_v = part(HEADS, 0), part(KV, HEADS), part(KV, HEADS + KV)
        self.t_q16, self.t_out = H.tensor(self.q16, H.F16, [HD, HEADS, rows]), H.tensor(self.out, H.F32, [HD, HEADS, rows])
        self.t_logits = H.tensor(self.out, H.F32, [VOCAB, rows])
        self.param = H.SampleParam(self.temperature.ptr, self.top_k.ptr, None, None, self.uniform.ptr)
        L = H.load()
        self.need = L.spy_hip_paged_attention_scratch_size(B(self.t_q16), B(p.t_k), B(self.batch))
        self.scratch = H.DeviceBuffer(self.need + 256)
        self.scratch.fill(0xFF)
        assert L.spy_hip_sample_scratch_size(B(self.t_logits)) == 0

    def run(self, st, tokens=None):
        L, H, p = self.H.load(), self.H, self.p
        H.check(L.spy_hip_op_get_row(st, B(self.table), B(self.t_ids), B(self.t_x)))
        H.check(L.spy_hip_paged_append(st, B(self.t_q), B(self.t_k), B(self.t_v), B(self.batch), B(self.rope), B(self.t_q16), B(p.t_k), B(p.t_v)))
        H.check(L.spy_hip_paged_attention(st, B(self.t_q16), B(p.t_k), B(p.t_v), B(self.t_out), B(self.batch), 0.125, 1, 0, self.scratch.ptr, self.need))
        H.check(L.spy_hip_sample(st, B(self.t_logits), B(self.param), (tokens or self.tokens).ptr, None, None, 0))

    def set(self, ids, start, kv, uniform):
        self.ids.upload(np.asarray(ids, np.int32))
        self.start.upload(np.asarray(start, np.int32))
        self.kv.upload(np.asarray(kv, np.int32))
        self.uniform.upload(np.asarray(uniform, np.float32))


def check_step(p, emb, step, ids, start, kv, uniform, history):
    """the step's queries, attention and tokens; history: the tokens of each sequence, the new ones last"""
    q16 = step.q16.download(np.float16).reshape(step.rows, HEADS, HD)
    out = step.out.download(np.float32).reshape(step.rows, VOCAB)
    tokens = step.tokens.download(np.int32)
    pool_k, pool_v = p.pools()
    for s in range(len(p.seqs)):
        new, n = int(start[s + 1] - start[s]), int(kv[s])
        if not new:
            continue
        x = emb[np.asarray(history[s][:n])].astype(np.float64).reshape(n, HEADS + 2 * KV, HD)
        k, v = (np.array([at(pool, s, j) for j in range(n)]) for at, pool in ((p.k_at, pool_k), (p.v_at, pool_v)))
        for j in range(n):
            y, size = P.rotated(x[j, HEADS:HEADS + KV], j, 2, HD, 10000.0, 1.0)
            assert (np.abs(k[j] - y) <= P.EPS16 * np.abs(y) + 8 * P.EPS32 * size + 2.0 ** -25).all(), (s, j)
            assert np.array_equal(v[j], x[j, HEADS + KV:].astype(np.float16)), (s, j)
        for i in range(new):
            row, pos = int(start[s]) + i, n - new + i
            y, size = P.rotated(x[pos, :HEADS], pos, 2, HD, 10000.0, 1.0)
            assert (np.abs(q16[row] - y) <= P.EPS16 * np.abs(y) + 8 * P.EPS32 * size + 2.0 ** -25).all(), (s, i)
            for h in range(HEADS):
                want, tol = P.attention(q16[row:row + 1, h], k[:, h // 2], v[:, h // 2], np.array([pos]), 0.125, 1, 0, True)
                assert (np.abs(out[row, h * HD:h * HD + HD] - want[0]) <= tol[0]).all(), (s, i, h)
            assert tokens[row] in [plan(out[row], t=np.float32(0.25), k=40, u=np.float32(uniform[row]), slack=d)[0] for d in (0.0, 2.0 ** -21, -2.0 ** -21)], (s, i)
    rest = int(start[-1])
    assert (q16[rest:] == step.left_q[rest:]).all() and (out[rest:] == step.left_out[rest:]).all(), "rows behind the last sequence"
    step.left_q, step.left_out = q16, out
    return tokens


@pytest.mark.parametrize("captured", [False, True])
def test_requests_served_together(hip, captured):
    from spy_amd import _lib as H
    rng = np.random.default_rng(11)
    L = H.load()
    prompt, steps = [1, 37, 130, 16, 5], 6
    p = P.Paged(rng, [(0, n + steps) for n in prompt], HEADS, KV, HD, PAGE, spare=0)
    p.upload()
    emb = rng.standard_normal((VOCAB, (HEADS + 2 * KV) * HD)).astype(np.float32)
    d_emb = H.DeviceBuffer.from_numpy(emb)
    table = H.tensor(d_emb, H.F32, [emb.shape[1], VOCAB])
    rope = H.RopeParam(mode=2, num_dim=HD, freq_base=10000.0, freq_scale=1.0, attention_factor=1.0)
    history = [list(map(int, rng.integers(0, VOCAB, n))) for n in prompt]
    # the prompts, all at once
    first = Step(H, p, table, rope, sum(prompt) + 2, max(prompt), max(prompt), rng)
    start, kv = np.concatenate([[0], np.cumsum(prompt)]), np.array(prompt)
    ids, uniform = np.zeros(first.rows, np.int32), rng.random(first.rows).astype(np.float32)
    ids[:sum(prompt)] = np.concatenate(history)
    first.left_q, first.left_out = np.full((first.rows, HEADS, HD), 77, np.float16), np.full((first.rows, VOCAB), 77, np.float32)
    first.set(ids, start, kv, uniform)
    first.run(None)
    H.sync()
    tokens = check_step(p, emb, first, ids, start, kv, uniform, history)
    tokens = [int(tokens[start[s + 1] - 1]) for s in range(len(prompt))]
    # one token per request and step; request 2 ends after the third
    one = Step(H, p, table, rope, len(prompt), 1, max(prompt) + steps, rng)
    one.left_q, one.left_out = np.full((one.rows, HEADS, HD), 77, np.float16), np.full((one.rows, VOCAB), 77, np.float32)
    other = H.DeviceBuffer.from_numpy(np.full(one.rows, -7, np.int32))
    st, graph = C.c_void_p(), C.c_void_p()
    H.check(L.spy_hip_stream_create(B(st)))
    live = list(range(len(prompt)))
    for n in range(steps):
        if n == 3:
            tokens = [t for t, s in zip(tokens, live) if s != 2]
            live.remove(2)
        for t, s in zip(tokens, live):
            history[s].append(t)
        kv = np.array([len(h) for h in history])
        start = np.concatenate([[0], np.cumsum([s in live for s in range(len(prompt))])])
        ids, uniform = np.zeros(one.rows, np.int32), rng.random(one.rows).astype(np.float32)
        ids[:len(live)] = tokens
        one.set(ids, start, kv, uniform)
        H.sync()                                                           # uploads are on the null stream, which the other one does not wait for
        if captured:
            if not graph.value:
                H.check(L.spy_hip_capture_begin(st))
                one.run(st)
                H.check(L.spy_hip_capture_end(st, B(graph)))
            H.check(L.spy_hip_graph_launch(graph, st))
        else:
            one.run(st)
        H.sync(st)
        tokens = check_step(p, emb, one, ids, start, kv, uniform, history)
        before = one.left_out.copy()
        one.run(None, other)                                               # the same step as eager calls between the replays: the same bits
        H.sync()
        assert np.array_equal(other.download(np.int32), tokens) and np.array_equal(one.out.download(np.uint32).reshape(before.shape), before.view(np.uint32))
        tokens = [int(t) for t in tokens[:len(live)]]
        print("step %d tokens %s" % (n, tokens), flush=True)
    assert (one.scratch.download(np.uint8, offset=one.need) == 0xFF).all() and P.flag() == 0
    if graph.value:
        H.check(L.spy_hip_graph_destroy(graph))
    H.check(L.spy_hip_stream_destroy(st))


def test_calls_on_two_streams_at_once(hip):
    """Attention (single tokens, keys shared out; a chunk), appending and sampling on two streams, each with its own scratch: the results of one call alone."""
    from spy_amd import _lib as H
    L = H.load()
    sides = []
    for seed, seqs in ((21, [(1, 3000), (1, 77), (1, 1500)]), (22, [(70, 900), (1, 2000)])):
        rng = np.random.default_rng(seed)
        p = P.Paged(rng, seqs, 8, 2, 128, 32)
        p.store()
        p.upload()
        dq = H.DeviceBuffer.from_numpy(rng.standard_normal((p.rows, 8, 128)).astype(np.float16).view(np.uint16))
        out = H.DeviceBuffer.from_numpy(np.full((p.rows, 8, 128), 77, np.float32))
        logits = H.DeviceBuffer.from_numpy(rng.standard_normal((p.rows, 5001)).astype(np.float32))
        uniform, tokens = H.DeviceBuffer.from_numpy(rng.random(p.rows).astype(np.float32)), H.DeviceBuffer.from_numpy(np.full(p.rows, -7, np.int32))
        tq, to, tl = H.tensor(dq, H.F16, [128, 8, p.rows]), H.tensor(out, H.F32, [128, 8, p.rows]), H.tensor(logits, H.F32, [5001, p.rows])
        need = L.spy_hip_paged_attention_scratch_size(B(tq), B(p.t_k), B(p.batch))
        st = C.c_void_p()
        H.check(L.spy_hip_stream_create(B(st)))
        new = H.DeviceBuffer.from_numpy(rng.standard_normal((p.rows, 4, 128)).astype(np.float16).view(np.uint16))
        tk, tv = (H.tensor(new, H.F16, [128, 2, p.rows], [2, 256, 1024], offset=o) for o in (0, 512))
        sides.append(dict(p=p, keep=(dq, logits, uniform, new), out=out, tokens=tokens, tq=tq, to=to, tl=tl, tk=tk, tv=tv, need=need, scratch=H.DeviceBuffer(max(need, 1)), st=st,
                          param=H.SampleParam(None, None, None, None, uniform.ptr)))
    assert all(s["need"] for s in sides)

    def run(s, st):
        p = s["p"]
        H.check(L.spy_hip_paged_append(st, None, B(s["tk"]), B(s["tv"]), B(p.batch), None, None, B(p.t_k), B(p.t_v)))
        H.check(L.spy_hip_paged_attention(st, B(s["tq"]), B(p.t_k), B(p.t_v), B(s["to"]), B(p.batch), 0.1, 1, 0, s["scratch"].ptr, s["need"]))
        H.check(L.spy_hip_sample(st, B(s["tl"]), B(s["param"]), s["tokens"].ptr, None, None, 0))

    want = []
    for s in sides:
        run(s, None)
        H.sync()
        want.append((s["out"].download(np.uint32), s["tokens"].download(np.int32)))
    for again in range(5):
        for s in sides:
            s["out"].fill(0x33)
            s["tokens"].fill(0x33)
        H.sync()
        for _ in range(4):
            for s in sides:
                run(s, s["st"])
        for s in sides:
            H.sync(s["st"])
        for s, (o, t) in zip(sides, want):
            rows = int(s["p"].row_start[-1]) * 8 * 128
            assert np.array_equal(s["out"].download(np.uint32)[:rows], o[:rows]) and np.array_equal(s["tokens"].download(np.int32), t), again
    for s in sides:
        H.check(L.spy_hip_stream_destroy(s["st"]))


@pytest.mark.parametrize("seqs", [[(1, 3000), (1, 77), (1, 1500)], [(70, 2900), (1, 2000), (3, 3)], [(200, 2200)]])
def test_a_recorded_call_follows_the_lengths(hip, seqs):
    """Keys shared out and joined, recorded once, replayed with other lengths and pages in the device arrays, other calls on the same stream in between: the bits of an eager call."""
    from spy_amd import _lib as H
    L = H.load()
    rng = np.random.default_rng(31)
    p = P.Paged(rng, seqs, 4, 2, 128, 16)
    p.store()
    p.upload()
    q = (rng.standard_normal((p.rows, 4, 128)) * 1.5).astype(np.float16)
    dq = H.DeviceBuffer.from_numpy(q.view(np.uint16))
    outs = [H.DeviceBuffer.from_numpy(np.full(q.shape, 77, np.float32)) for _ in range(2)]
    tq, to = H.tensor(dq, H.F16, [128, 4, p.rows]), [H.tensor(o, H.F32, [128, 4, p.rows]) for o in outs]
    need = L.spy_hip_paged_attention_scratch_size(B(tq), B(p.t_k), B(p.batch))
    assert need > 0
    scratch = [H.DeviceBuffer(need) for _ in range(2)]
    st, graph = C.c_void_p(), C.c_void_p()
    H.check(L.spy_hip_stream_create(B(st)))
    call = lambda i, s: H.check(L.spy_hip_paged_attention(s, B(tq), B(p.t_k), B(p.t_v), B(to[i]), B(p.batch), 0.09, 1, 0, scratch[i].ptr, need))     # noqa: E731
    H.check(L.spy_hip_capture_begin(st))
    call(0, st)
    H.check(L.spy_hip_capture_end(st, B(graph)))
    full, starts = p.kv.copy(), p.row_start.copy()
    for n in range(4):
        p.kv = np.maximum(full - np.array([0, 500, 37, 1400])[n], p.n_new)            # shorter caches: the same tokens, fewer of them
        if n == 2:                                                                    # the first sequence has ended
            p.row_start = np.concatenate([[0], starts[1:] - starts[1]]).astype(np.int32)
        else:
            p.row_start = starts
        p.n_new = np.diff(p.row_start)
        p.d_kv.upload(p.kv.astype(np.int32))
        p.d_start.upload(p.row_start)
        for i in range(2):
            outs[i].upload(np.full(q.shape, 77, np.float32))
            scratch[i].fill(0xFF)
        H.sync()
        H.check(L.spy_hip_graph_launch(graph, st))
        H.sync(st)
        got = outs[0].download(np.float32).reshape(q.shape)
        call(1, st)
        H.sync(st)
        assert np.array_equal(got.view(np.uint32), outs[1].download(np.uint32).reshape(q.shape)), n
        k_rows, v_rows = p.k_rows, p.v_rows
        p.k_rows, p.v_rows = [k[:x] for k, x in zip(k_rows, p.kv)], [v[:x] for v, x in zip(v_rows, p.kv)]
        P.check_attention(p, q, got, True, scale=0.09)
        p.k_rows, p.v_rows = k_rows, v_rows
        p.n_new = np.diff(starts)
    assert P.flag() == 0
    H.check(L.spy_hip_graph_destroy(graph))
    H.check(L.spy_hip_stream_destroy(st))
