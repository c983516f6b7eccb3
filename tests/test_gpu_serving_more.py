"""Requests behind one prompt, served together from a cache of 8 bits with drafted tokens: rows of an embedding table as q, k and v, stored and attended to, the output's rows as logits, the drafts
drawn from logits of their own and verified.  Each step against the definitions in 64 bits, as eager calls and as one recorded graph; calls on two streams at once; a recorded call whose groups change."""
import ctypes as C

import numpy as np
import pytest

from tests import paged_more_util as M
from tests import paged_util as P
from tests.test_gpu_verify import check as check_verify

pytestmark = pytest.mark.gpu
B = C.byref
HEADS, KV, HD, PAGE = 4, 2, 64, 16
VOCAB = HEADS * HD
SETTINGS, DRAFT_SETTINGS = dict(temperature=0.25, top_k=200), dict(temperature=0.3, top_p=0.9)


class Step:
    """The buffers of one kind of step (so many rows at most) and its calls."""

    def __init__(self, H, p, table, rope, rows, max_new, max_kv, prefix):
        self.H, self.p, self.rows, self.rope, self.table, self.prefix = H, p, rows, rope, table, prefix
        width = (HEADS + 2 * KV) * HD
        full = lambda shape, t, v: H.DeviceBuffer.from_numpy(np.full(shape, v, t))                # noqa: E731
        self.ids, self.x = full(rows, np.int32, 0), full((rows, width), np.float32, 0)
        self.q16, self.out, self.draft = full((rows, HEADS, HD), np.float16, 77), full((rows, VOCAB), np.float32, 77), full((rows, VOCAB), np.float32, 0)
        self.start, self.kv, n = full(len(p.seqs) + 1, np.int32, 0), full(len(p.seqs), np.int32, 0), len(p.seqs)
        self.drafted, self.tokens, self.accepted, self.probs = full(rows, np.int32, 0), full(rows, np.int32, -7), full(n, np.int32, -7), full(rows, np.float32, -7)
        self.uniform, self.accept, self.u_draft = (full(rows, np.float32, 0) for _ in range(3))
        self.settings = [full(rows, np.float32, 0.25), full(rows, np.int32, 200), full(rows, np.float32, 0.3), full(rows, np.float32, 0.9)]
        self.batch = H.PagedBatch(n, max_new, max_kv, self.start.ptr, self.kv.ptr, p.d_table.ptr, p.table.shape[1])
        part = lambda heads, first: H.tensor(self.x, H.F32, [HD, heads, rows], [4, HD * 4, width * 4], offset=first * HD * 4)   # noqa: E731
        self.t_q, self.t_k, self.t_v = part(HEADS, 0), part(KV, HEADS), part(KV, HEADS + KV)
        self.t_ids, self.t_x = H.tensor(self.ids, H.I32, [rows]), H.tensor(self.x, H.F32, [width, rows])
        self.t_q16, self.t_out = H.tensor(self.q16, H.F16, [HD, HEADS, rows]), H.tensor(self.out, H.F32, [HD, HEADS, rows])
        self.t_logits, self.t_draft = H.tensor(self.out, H.F32, [VOCAB, rows]), H.tensor(self.draft, H.F32, [VOCAB, rows])
        self.param = H.SampleParam(self.settings[0].ptr, self.settings[1].ptr, None, None, self.uniform.ptr)
        self.draft_param = H.SampleParam(self.settings[2].ptr, None, self.settings[3].ptr, None, self.u_draft.ptr)
        L = H.load()
        need = L.spy_hip_paged_attention_shared_scratch_size(B(self.t_q16), B(p.t_kq), B(self.batch), B(prefix)), L.spy_hip_sample_verify_scratch_size(B(self.t_logits), n)
        self.need = need
        self.scratch = [H.DeviceBuffer(x + 256) for x in need]
        for s in self.scratch:
            s.fill(0xFF)

    def draw_drafts(self):
        """what a small model would propose"""
        L, H = self.H.load(), self.H
        H.check(L.spy_hip_sample(None, B(self.t_draft), B(self.draft_param), self.drafted.ptr, None, None, 0))
        H.sync()
        return self.drafted.download(np.int32)

    def run(self, st, tokens=None):
        L, H, p = self.H.load(), self.H, self.p
        H.check(L.spy_hip_op_get_row(st, B(self.table), B(self.t_ids), B(self.t_x)))
        H.check(L.spy_hip_paged_append_q8(st, B(self.t_q), B(self.t_k), B(self.t_v), B(self.batch), B(self.rope), B(self.t_q16), B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd)))
        H.check(L.spy_hip_paged_attention_shared(st, B(self.t_q16), B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd), B(self.t_out), B(self.batch), B(self.prefix), 0.125, self.scratch[0].ptr, self.need[0]))
        H.check(L.spy_hip_sample_verify(st, B(self.t_logits), B(self.param), B(self.t_draft), B(self.draft_param), self.drafted.ptr, self.start.ptr, len(p.seqs), self.accept.ptr,
                                        (tokens or self.tokens).ptr, self.accepted.ptr, self.probs.ptr, self.scratch[1].ptr, self.need[1]))

    def set(self, rng, start, kv):
        self.start.upload(np.asarray(start, np.int32))
        self.kv.upload(np.asarray(kv, np.int32))
        self.u, self.a = rng.random(self.rows).astype(np.float32), rng.random(self.rows).astype(np.float32)
        self.uniform.upload(self.u)
        self.accept.upload(self.a)
        self.u_draft.upload(rng.random(self.rows).astype(np.float32))
        for buf, t, n in ((self.tokens, np.int32, self.rows), (self.accepted, np.int32, len(kv)), (self.probs, np.float32, self.rows)):
            buf.upload(np.full(n, -7, t))


def check_step(p, emb, step, start, kv, drafted, draft, history, common):
    """what is cached, the attention and the verified tokens; history: the tokens of each sequence, its new rows' last"""
    out = step.out.download(np.float32).reshape(step.rows, VOCAB)
    q16 = step.q16.download(np.float16).reshape(step.rows, HEADS, HD)
    kq, kd, vq, vd = p.q8_pools()
    for s in range(len(p.seqs)):
        new, n = int(start[s + 1] - start[s]), int(kv[s])
        if not new:
            continue
        x = emb[np.asarray(history[s][:n])].reshape(n, HEADS + 2 * KV, HD)
        k, v = np.zeros((n, KV, HD), np.float16), np.zeros((n, KV, HD), np.float16)
        for j in range(n):
            page, at = p.table[0 if j < common else s, j // PAGE], j % PAGE
            k[j], v[j] = M.q8_values(kq[page, :, at], kd[page, :, at]), M.q8_values(vq[page, :, :, at], vd[page, :, :, at])
            y, size = P.rotated(x[j, HEADS:HEADS + KV].astype(np.float64), j, 2, HD, 10000.0, 1.0)
            off = 8 * P.EPS32 * size                             # as in tests/test_gpu_paged_q8.py
            d = np.repeat((np.abs(y) + off).reshape(KV, -1, 32).max(axis=2) / 127, 32, axis=1)
            assert (np.abs(k[j] - y) <= d * (0.5 + 2.0 ** -15) + 127 * (P.EPS16 * d + 2.0 ** -25) + off + P.EPS16 * (np.abs(y) + d) + 2.0 ** -25).all(), (s, j)
            assert np.array_equal(v[j], M.q8_values(*M.q8_blocks(x[j, HEADS + KV:]))), (s, j)
        for i in range(new):
            row, pos = int(start[s]) + i, n - new + i
            y, size = P.rotated(x[pos, :HEADS].astype(np.float64), pos, 2, HD, 10000.0, 1.0)
            assert (np.abs(q16[row] - y) <= P.EPS16 * np.abs(y) + 8 * P.EPS32 * size + 2.0 ** -25).all(), (s, i)
            for h in range(HEADS):
                want, tol = P.attention(q16[row:row + 1, h], k[:, h // 2], v[:, h // 2], np.array([pos]), 0.125, 1, 0, True)
                assert (np.abs(out[row, h * HD:h * HD + HD] - want[0]) <= tol[0]).all(), (s, i, h)
    got = step.tokens.download(np.int32), step.accepted.download(np.int32), step.probs.download(np.float32)
    check_verify(got, out, drafted, np.asarray(start), step.a, step.u, SETTINGS, draft, DRAFT_SETTINGS)
    return got


@pytest.mark.parametrize("captured", [False, True])
def test_requests_behind_one_prompt_with_drafts(hip, captured):
    from spy_amd import _lib as H
    rng = np.random.default_rng(12)
    L = H.load()
    common, own, steps, most = 100, [3, 37, 1, 18, 9], 6, 4      # tokens in common, each request's own, steps, drafts at most
    n = len(own)
    longest = common + max(own) + steps * (most + 1)
    p = M.PagedQ8(rng, [(0, longest)] * n, HEADS, KV, HD, PAGE, spare=0)
    p.quantize()
    p.upload()
    emb = rng.standard_normal((VOCAB, (HEADS + 2 * KV) * HD)).astype(np.float32)
    d_emb = H.DeviceBuffer.from_numpy(emb)
    table = H.tensor(d_emb, H.F32, [emb.shape[1], VOCAB])
    rope = H.RopeParam(mode=2, num_dim=HD, freq_base=10000.0, freq_scale=1.0, attention_factor=1.0)
    prompt = list(map(int, rng.integers(0, VOCAB, common)))
    history = [prompt + list(map(int, rng.integers(0, VOCAB, x))) for x in own]
    # the prompt once, by the first request, then each request's own tokens behind it: without drafts, the last row of each is what counts
    d_groups, d_length = H.DeviceBuffer.from_numpy(np.array([0, n], np.int32)), H.DeviceBuffer.from_numpy(np.array([0], np.int32))
    prefix = H.PagedPrefix(1, sum(own) + common, longest, d_groups.ptr, d_length.ptr)
    first = Step(H, p, table, rope, common, common, common, prefix)
    first.set(rng, [0] + [common] * n, [common] + [0] * (n - 1))
    first.ids.upload(np.asarray(prompt, np.int32))
    H.sync()
    H.check(L.spy_hip_op_get_row(None, B(table), B(first.t_ids), B(first.t_x)))
    H.check(L.spy_hip_paged_append_q8(None, B(first.t_q), B(first.t_k), B(first.t_v), B(first.batch), B(rope), B(first.t_q16), B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd)))
    d_length.upload(np.array([common], np.int32))
    # whole pages in common are the first request's alone
    lost = p.table.copy()
    lost[1:, :common // PAGE] = -1
    p.d_table.upload(lost)
    step = Step(H, p, table, rope, max(sum(own), n * (most + 1)) + 2, max(max(own), most + 1), longest, prefix)
    other = H.DeviceBuffer.from_numpy(np.full(step.rows, -7, np.int32))
    st, graph = C.c_void_p(), C.c_void_p()
    H.check(L.spy_hip_stream_create(B(st)))
    news = own
    n_accepted = n_drafted = 0
    last = [0] * n
    for turn in range(steps + 1):
        start = np.concatenate([[0], np.cumsum(news)])
        kv = [len(h) for h in history]
        draft = (rng.standard_normal((step.rows, VOCAB)) * 0.02).astype(np.float32)
        if turn:                                                 # a small model: what the large one had at the request's last token, and something added
            for i in range(n):
                draft[start[i]:start[i + 1]] += step.out.download(np.float32).reshape(step.rows, VOCAB)[last[i]]
        step.draft.upload(draft)
        step.set(rng, start, kv)
        H.sync()
        drafted = step.draw_drafts()
        ids = np.zeros(step.rows, np.int32)
        seen = []
        for s in range(n):
            h = list(history[s])
            if turn:                                             # [last token, drafts ...]: the drafts are cached as well
                h += [int(drafted[start[s] + i]) for i in range(news[s] - 1)]
                kv[s] = len(h)
            else:                                                # a prompt's own tokens: they are what is verified, and all are taken or not
                drafted[start[s]:start[s + 1] - 1] = h[len(h) - news[s] + 1:]
            ids[start[s]:start[s + 1]] = h[len(h) - news[s]:]
            seen.append(h)
        step.drafted.upload(drafted)
        step.kv.upload(np.asarray(kv, np.int32))
        step.ids.upload(ids)
        H.sync()                                                 # uploads are on the null stream, which the other one does not wait for
        if captured and turn:
            if not graph.value:
                H.check(L.spy_hip_capture_begin(st))
                step.run(st)
                H.check(L.spy_hip_capture_end(st, B(graph)))
            H.check(L.spy_hip_graph_launch(graph, st))
        else:
            step.run(st)
        H.sync(st)
        tokens, accepted, _ = check_step(p, emb, step, start, kv, drafted, draft, seen, common)
        before = step.out.download(np.uint32)
        step.run(None, other)                                    # the same step as eager calls between the replays: the same bits
        H.sync()
        assert np.array_equal(other.download(np.int32)[:start[-1]], tokens[:start[-1]]) and np.array_equal(step.out.download(np.uint32), before)
        for s in range(n):
            if turn:
                took = int(accepted[s])
                last[s] = start[s] + took
                n_accepted += took
                n_drafted += news[s] - 1
                history[s] = history[s] + [int(t) for t in tokens[start[s]:start[s] + took + 1]]
            else:
                last[s] = start[s + 1] - 1
                history[s].append(int(rng.integers(0, VOCAB)))
        news = [1 + int(x) for x in rng.integers(0, most + 1, n)]
        print("step %d: %d of %d drafts taken so far" % (turn, n_accepted, n_drafted), flush=True)
    for s, need in zip(step.scratch, step.need):
        assert (s.download(np.uint8, offset=need) == 0xFF).all()
    assert P.flag() == 0
    if graph.value:
        H.check(L.spy_hip_graph_destroy(graph))
    H.check(L.spy_hip_stream_destroy(st))


def _side(H, seed, seqs, start, length, q8):
    rng = np.random.default_rng(seed)
    p = M.PagedQ8(rng, seqs, 8, 2, 128, 32)
    M.share(p, start, length)
    p.store()
    p.quantize()
    p.upload()
    M.shared_batch(p, start, length)
    L, n = H.load(), len(seqs)
    s = dict(p=p, st=C.c_void_p(), q8=q8)
    s["q"] = H.DeviceBuffer.from_numpy(rng.standard_normal((p.rows, 8, 128)).astype(np.float16).view(np.uint16))
    s["out"] = [H.DeviceBuffer.from_numpy(np.full((p.rows, 8, 128), 77, np.float32)) for _ in range(2)]
    s["tq"], s["to"] = H.tensor(s["q"], H.F16, [128, 8, p.rows]), [H.tensor(o, H.F32, [128, 8, p.rows]) for o in s["out"]]
    s["new"] = H.DeviceBuffer.from_numpy(rng.standard_normal((p.rows, 4, 128)).astype(np.float16).view(np.uint16))
    s["tk"], s["tv"] = (H.tensor(s["new"], H.F16, [128, 2, p.rows], [2, 256, 1024], offset=o) for o in (0, 512))
    s["logits"], s["draft"] = (H.DeviceBuffer.from_numpy(rng.standard_normal((p.rows, 5001)).astype(np.float32)) for _ in range(2))
    s["tl"], s["td"] = (H.tensor(s[x], H.F32, [5001, p.rows]) for x in ("logits", "draft"))
    s["u"] = H.DeviceBuffer.from_numpy(rng.random(p.rows).astype(np.float32))
    s["drafted"] = H.DeviceBuffer.from_numpy(rng.integers(0, 5001, p.rows).astype(np.int32))
    s["tokens"], s["accepted"], s["probs"] = H.DeviceBuffer(4 * p.rows), H.DeviceBuffer(4 * n), H.DeviceBuffer(4 * p.rows)
    s["param"] = H.SampleParam(None, None, None, None, s["u"].ptr)
    pages = (B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd)) if q8 else (B(p.t_k), None, B(p.t_v), None)
    need = (L.spy_hip_paged_attention_q8_scratch_size(B(s["tq"]), B(p.t_kq), B(p.batch)), L.spy_hip_paged_attention_shared_scratch_size(B(s["tq"]), pages[0], B(p.batch), B(p.prefix)),
            L.spy_hip_sample_verify_scratch_size(B(s["tl"]), n))
    scratch = [H.DeviceBuffer(max(x, 1)) for x in need]
    H.check(L.spy_hip_stream_create(B(s["st"])))

    def run(st):
        H.check(L.spy_hip_paged_append_q8(st, None, B(s["tk"]), B(s["tv"]), B(p.batch), None, None, B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd)))
        H.check(L.spy_hip_paged_attention_q8(st, B(s["tq"]), B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd), B(s["to"][0]), B(p.batch), 0.1, 1, 0, scratch[0].ptr, need[0]))
        H.check(L.spy_hip_paged_attention_shared(st, B(s["tq"]), *pages, B(s["to"][1]), B(p.batch), B(p.prefix), 0.1, scratch[1].ptr, need[1]))
        H.check(L.spy_hip_sample_verify(st, B(s["tl"]), B(s["param"]), B(s["td"]), None, s["drafted"].ptr, p.d_start.ptr, n, s["u"].ptr, s["tokens"].ptr, s["accepted"].ptr, s["probs"].ptr,
                                        scratch[2].ptr, need[2]))

    def results():
        rows = int(p.row_start[-1])
        return [o.download(np.uint32)[:rows * 1024] for o in s["out"]] + [s["tokens"].download(np.int32)[:rows], s["accepted"].download(np.int32), s["probs"].download(np.uint32)[:rows]]

    return dict(s, run=run, results=results, need=need, keep=scratch)


def test_calls_on_two_streams_at_once(hip):
    """Each call with scratch of its own: the results of one call alone.  Pages whose own rows hold the common tokens, so that both kinds of attention see the same."""
    from spy_amd import _lib as H
    L = H.load()
    sides = [_side(H, 41, [(1, 3000), (1, 2907), (2, 2950), (1, 60)], [0, 3], [2880], True), _side(H, 42, [(70, 900), (3, 850), (1, 2000)], [0, 2], [800], False)]
    for s in sides:                                              # (spy_hip_paged_attention_q8 reads every sequence's own table)
        s["p"].d_table.upload(s["p"].table)
    assert all(x for s in sides for x in s["need"])
    want = []
    for s in sides:
        s["run"](None)
        H.sync()
        want.append(s["results"]())
        rows = int(s["p"].row_start[-1])
        if s["q8"]:
            a, b = (x.view(np.float32).reshape(rows, 8, 128) for x in want[-1][:2])
            assert (np.abs(a - b) <= 1e-5).all()                 # fp32 sums in another order of values below 1
    for again in range(5):
        for s in sides:
            for o in s["out"] + [s["tokens"], s["accepted"], s["probs"]]:
                o.fill(0x33)
        H.sync()
        for _ in range(4):
            for s in sides:
                s["run"](s["st"])
        for s in sides:
            H.sync(s["st"])
        for s, w in zip(sides, want):
            assert all(np.array_equal(x, y) for x, y in zip(s["results"](), w)), again
    assert P.flag() == 0
    for s in sides:
        H.check(L.spy_hip_stream_destroy(s["st"]))


@pytest.mark.parametrize("q8", [False, True])
def test_a_recorded_call_follows_groups_and_lengths(hip, q8):
    """Recorded once, replayed with other groups, lengths in common and rows in the device arrays, eager calls between: the bits of an eager call, and the definition."""
    from spy_amd import _lib as H
    L = H.load()
    rng = np.random.default_rng(51)
    seqs, common = [(1, 700), (40, 560), (1, 900), (3, 520), (17, 600)], 500
    p = M.PagedQ8(rng, seqs, 4, 2, 128, 16)
    M.share(p, [0, 5], [common])
    p.store()
    if q8:
        p.quantize()
        p.upload()
    else:
        P.Paged.upload(p)
    M.shared_batch(p, [0, 3, 5], [common, common])
    p.d_table.upload(p.table)
    p.prefix.max_rows, p.prefix.max_prefix = p.rows, common
    q = (rng.standard_normal((p.rows, 4, 128)) * 1.5).astype(np.float16)
    dq = H.DeviceBuffer.from_numpy(q.view(np.uint16))
    outs = [H.DeviceBuffer.from_numpy(np.full(q.shape, 77, np.float32)) for _ in range(2)]
    tq, to = H.tensor(dq, H.F16, [128, 4, p.rows]), [H.tensor(o, H.F32, [128, 4, p.rows]) for o in outs]
    pages = (B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd)) if q8 else (B(p.t_k), None, B(p.t_v), None)
    need = L.spy_hip_paged_attention_shared_scratch_size(B(tq), pages[0], B(p.batch), B(p.prefix))
    scratch = [H.DeviceBuffer(need) for _ in range(2)]
    st, graph = C.c_void_p(), C.c_void_p()
    H.check(L.spy_hip_stream_create(B(st)))
    call = lambda i, s: H.check(L.spy_hip_paged_attention_shared(s, B(tq), *pages, B(to[i]), B(p.batch), B(p.prefix), 0.09, scratch[i].ptr, need))      # noqa: E731
    H.check(L.spy_hip_capture_begin(st))
    call(0, st)
    H.check(L.spy_hip_capture_end(st, B(graph)))
    starts = p.row_start.copy()
    for turn, (start, length) in enumerate([([0, 3, 5], [500, 500]), ([0, 5, 5], [499, 0]), ([1, 3, 5], [64, 1]), ([0, 0, 2], [0, 500]), ([0, 2, 5], [0, 0]), ([0, 3, 5], [500, 33])]):
        p.row_start = starts if turn != 3 else np.concatenate([[0], starts[1:] - starts[1]]).astype(np.int32)       # the first sequence has ended
        p.n_new = np.diff(p.row_start)
        p.d_start.upload(p.row_start)
        p.d_groups.upload(np.asarray(start, np.int32))
        p.d_length.upload(np.asarray(length, np.int32))
        for i in range(2):
            outs[i].upload(np.full(q.shape, 77, np.float32))
            scratch[i].fill(0xFF)
        H.sync()
        H.check(L.spy_hip_graph_launch(graph, st))
        H.sync(st)
        got = outs[0].download(np.float32).reshape(q.shape)
        call(1, st)
        H.sync(st)
        assert np.array_equal(got.view(np.uint32), outs[1].download(np.uint32).reshape(q.shape)), turn
        P.check_attention(p, q, got, True, scale=0.09)
    assert P.flag() == 0
    H.check(L.spy_hip_graph_destroy(graph))
    H.check(L.spy_hip_stream_destroy(st))
