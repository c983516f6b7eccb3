"""Batches over a cache in pages for the tests: inputs on the host, their copies on the device, and the operators' definitions in 64 bits."""
import ctypes as C

import numpy as np

from spy_amd import _lib as H

EPS16, EPS32 = 2.0 ** -11, 2.0 ** -24                # half a step of fp16 and fp32, relative to the value


class Paged:
    """seqs: (new tokens, cached tokens) of each sequence.  Pages lie in the pool in a random order, with pages of nobody between them; what no sequence holds is
    `fill`.  token_major: pages as [position][head][hd] rows instead of one block per head.  spare: rows of q, k, v and out behind the last sequence."""

    def __init__(self, rng, seqs, heads, kv_heads, hd, page, fill=np.nan, token_major=False, spare=3, table_spare=2):
        self.rng, self.seqs, self.heads, self.kv_heads, self.hd, self.page = rng, seqs, heads, kv_heads, hd, page
        self.n_new = np.array([s[0] for s in seqs])
        self.kv = np.array([s[1] for s in seqs])
        self.row_start = np.concatenate([[0], np.cumsum(self.n_new)]).astype(np.int32)
        self.rows = int(self.row_start[-1]) + spare
        need = [-(-int(k) // page) for k in self.kv]
        self.n_page = sum(need) + 3
        order = rng.permutation(self.n_page)
        self.table = np.full((len(seqs), max(need + [1]) + table_spare), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        # logical contents, one row per cached token: [sequence][position][head][hd]
        self.k_rows = [rng.standard_normal((int(n), kv_heads, hd)).astype(np.float16) for n in self.kv]
        self.v_rows = [rng.standard_normal((int(n), kv_heads, hd)).astype(np.float16) for n in self.kv]
        self.token_major = token_major
        if token_major:
            self.k_shape, self.v_shape = (self.n_page, page, kv_heads, hd), (self.n_page, kv_heads, hd, page)
        else:
            self.k_shape, self.v_shape = (self.n_page, kv_heads, page, hd), (self.n_page, kv_heads, hd, page)
        self.k_pool = np.full(self.k_shape, fill, np.float16)
        self.v_pool = np.full(self.v_shape, fill, np.float16)

    def k_at(self, pool, seq, pos):
        """view of the K rows of a cached token, [head][hd]"""
        p, o = self.table[seq, pos // self.page], pos % self.page
        return pool[p, o] if self.token_major else pool[p, :, o]

    def v_at(self, pool, seq, pos):
        return pool[self.table[seq, pos // self.page], :, :, pos % self.page]

    def store(self, upto=None):
        """the sequences' rows into the pools; upto: positions below that many (of each sequence)"""
        for s in range(len(self.seqs)):
            n = int(self.kv[s]) if upto is None else int(upto[s])
            for pos in range(n):
                self.k_at(self.k_pool, s, pos)[:] = self.k_rows[s][pos]
                self.v_at(self.v_pool, s, pos)[:] = self.v_rows[s][pos]

    def upload(self):
        up = H.DeviceBuffer.from_numpy
        self.d_k, self.d_v = up(self.k_pool.view(np.uint16)), up(self.v_pool.view(np.uint16))
        self.d_start, self.d_kv, self.d_table = up(self.row_start), up(self.kv.astype(np.int32)), up(self.table)
        self.batch = H.PagedBatch(len(self.seqs), max(1, int(self.n_new.max())), max(1, int(self.kv.max())), self.d_start.ptr, self.d_kv.ptr, self.d_table.ptr, self.table.shape[1])
        hd, ps, G, es = self.hd, self.page, self.kv_heads, 2
        if self.token_major:
            self.t_k = H.tensor(self.d_k, H.F16, [hd, ps, G, self.n_page], [es, G * hd * es, hd * es, ps * G * hd * es])
        else:
            self.t_k = H.tensor(self.d_k, H.F16, [hd, ps, G, self.n_page])
        self.t_v = H.tensor(self.d_v, H.F16, [ps, hd, G, self.n_page])

    def pools(self):
        return self.d_k.download(np.float16).reshape(self.k_shape), self.d_v.download(np.float16).reshape(self.v_shape)

    def rows_of(self):
        """(row, sequence, position) of every new token"""
        for s, (new, kv) in enumerate(zip(self.n_new, self.kv)):
            for i in range(int(new)):
                yield int(self.row_start[s]) + i, s, int(kv) - int(new) + i


def rotated(x, pos, mode, dims, base, freq_scale, factor=1.0):
    """x: [head][hd] of one token in 64 bits, and what |x| a result can be off by (the sum of the magnitudes of the pair)"""
    y, size = x.copy(), np.abs(x)
    if mode < 0:
        return y, size
    i = np.arange(dims // 2)
    angle = np.float64(pos) * freq_scale * np.power(np.float64(base), -2.0 * i / dims)
    c, s = np.cos(angle) * factor, np.sin(angle) * factor
    a, b = (slice(0, dims, 2), slice(1, dims, 2)) if mode == 0 else (slice(0, dims // 2), slice(dims // 2, dims))
    y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, a] * s + x[:, b] * c
    size[:, a] = size[:, b] = (np.abs(x[:, a]) + np.abs(x[:, b])) * abs(factor)
    return y, size


def attention(q, k, v, pos, scale, causal, window, f32):
    """q [rows][hd], k and v [keys][hd] of one K/V head, pos [rows]: the outputs in 64 bits and how far off the kernel's may be, from the roundings it makes:
    hd fp32 additions to a score of at most A = scale * max sum |q k|, one fma and an exponential (together (hd A + 8) eps of a probability), n additions to a sum;
    a probability as fp16 (half a step of it, or of the least subnormal) or as two, whose second has half a step of a half step; the output's own rounding."""
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    j = np.arange(len(k))
    seen = np.ones((len(q), len(k)), bool)
    if causal:
        seen &= j[None] <= pos[:, None]
    if window:
        seen &= j[None] > pos[:, None] - window
    with np.errstate(all="ignore"):
        x = np.where(seen, scale * (q @ np.where(np.isnan(k), 0, k).T), -np.inf)
        size = np.where(seen, abs(scale) * (np.abs(q) @ np.abs(np.where(np.isnan(k), 0, k)).T), 0).max(axis=1, initial=0)
        top = x.max(axis=1, initial=-np.inf, keepdims=True)
        e = np.where(seen, np.exp(x - np.where(np.isfinite(top), top, 0)), 0)
        total = np.maximum(e.sum(axis=1, keepdims=True), 1e-300)
        vz = np.where(np.isfinite(v), v, 0)
        out = (e / total) @ vz
        mass = (e / total) @ np.abs(vz)
        for d in np.argwhere(~np.isfinite(v)):                   # an infinity or NaN reaches the rows that see it, and no others
            out[:, d[1]] = np.where(seen[:, d[0]], out[:, d[1]] + e[:, d[0]] * v[d[0], d[1]], out[:, d[1]])
        few = np.abs(vz).max(initial=0) * seen.sum(axis=1)[:, None] * 2.0 ** -25 / total
    arith = ((q.shape[1] * size + len(k) + 8) * EPS32)[:, None]
    tol = mass * (2 * arith + (EPS16 ** 2 if f32 else EPS16)) + few * (2.0 ** -11 if f32 else 1.0) + (EPS32 if f32 else EPS16) * np.abs(out) + (1e-30 if f32 else 2.0 ** -25)
    return np.where(seen.any(axis=1)[:, None], out, 0.0), tol


def run_append(p, q, k, v, rope, dtype, stream=None):
    """q, k, v: [rows][heads][hd] arrays (q may be None); returns the return code and q_out's array"""
    t = {np.float32: H.F32, np.float16: H.F16}[dtype]
    L, B = H.load(), C.byref
    bufs = [None if x is None else H.DeviceBuffer.from_numpy(x.view(np.uint32 if dtype is np.float32 else np.uint16)) for x in (q, k, v)]
    tq, tk, tv = (None if x is None else H.tensor(b, t, [x.shape[2], x.shape[1], x.shape[0]]) for x, b in zip((q, k, v), bufs))
    qo = None if q is None else H.DeviceBuffer.from_numpy(np.full(q.shape, 77, np.float16).view(np.uint16))
    tqo = None if q is None else H.tensor(qo, H.F16, [q.shape[2], q.shape[1], q.shape[0]])
    ref = lambda x: None if x is None else B(x)                                                   # noqa: E731
    rc = L.spy_hip_paged_append(stream, ref(tq), B(tk), B(tv), B(p.batch), ref(rope), ref(tqo), B(p.t_k), B(p.t_v))
    H.sync()
    return rc, None if q is None else qo.download(np.float16).reshape(q.shape)


def run_attention(p, q, f32, causal=1, window=0, scale=None):
    L, B = H.load(), C.byref
    scale = 1.0 / np.sqrt(p.hd) if scale is None else scale
    dq = H.DeviceBuffer.from_numpy(q.view(np.uint16))
    out = H.DeviceBuffer.from_numpy(np.full(q.shape, 77, np.float32 if f32 else np.float16).view(np.uint32 if f32 else np.uint16))
    tq, to = H.tensor(dq, H.F16, [p.hd, p.heads, p.rows]), H.tensor(out, H.F32 if f32 else H.F16, [p.hd, p.heads, p.rows])
    need = L.spy_hip_paged_attention_scratch_size(B(tq), B(p.t_k), B(p.batch))
    scratch = H.DeviceBuffer(need + 256)
    scratch.fill(0xFF)                                           # NaN wherever something is read before it is written
    H.check(L.spy_hip_paged_attention(None, B(tq), B(p.t_k), B(p.t_v), B(to), B(p.batch), scale, causal, window, scratch.ptr, need), "spy_hip_paged_attention")
    H.sync()
    assert (scratch.download(np.uint8, offset=need) == 0xFF).all()
    return out.download(np.float32 if f32 else np.float16).reshape(q.shape)


def flag():
    f = C.c_int32()
    H.check(H.load().spy_hip_take_error(C.byref(f)), "spy_hip_take_error")
    return f.value


def check_attention(p, q, got, f32, causal=1, window=0, scale=None, hidden=()):
    """every row against the definition; hidden: (sequence, page index) whose positions hold nothing"""
    scale = 1.0 / np.sqrt(p.hd) if scale is None else scale
    g = p.heads // p.kv_heads
    worst = 0.0
    for s in range(len(p.seqs)):
        new, kv, r0 = int(p.n_new[s]), int(p.kv[s]), int(p.row_start[s])
        if not new:
            continue
        pos = np.arange(kv - new, kv)
        keep = np.array([j for j in range(kv) if (s, j // p.page) not in hidden], int)
        for h in range(p.heads):
            k, v = p.k_rows[s][:, h // g], p.v_rows[s][:, h // g]
            if len(keep) < kv:                                   # hidden positions: give them a place no row sees
                want, tol = _with_hidden(q[r0:r0 + new, h], k, v, pos, scale, causal, window, f32, keep)
            else:
                want, tol = attention(q[r0:r0 + new, h], k, v, pos, scale, causal, window, f32)
            have = got[r0:r0 + new, h].astype(np.float64)
            fine = np.isfinite(want)
            assert np.array_equal(fine, np.isfinite(have)), (s, h, "infinities or NaN in other places")
            off = np.abs(have[fine] - want[fine]) / tol[fine]
            worst = max(worst, off.max(initial=0))
            assert off.max(initial=0) <= 1, (s, h, off.max(), np.argwhere(np.abs(have - want) > tol)[:4].tolist())
    assert (got[int(p.row_start[-1]):].astype(np.float64) == 77).all(), "rows behind the last sequence"
    return worst


def _with_hidden(q, k, v, pos, scale, causal, window, f32, keep):
    """attention over the positions in `keep` only, masks by their true positions"""
    seen_pos = pos
    kk, vv = k[keep], v[keep]
    outs, tols = [], []
    for i in range(len(q)):
        ok = np.ones(len(keep), bool)
        if causal:
            ok &= keep <= seen_pos[i]
        if window:
            ok &= keep > seen_pos[i] - window
        o, t = attention(q[i:i + 1], kk[ok], vv[ok], np.array([1 << 30]), scale, 0, 0, f32) if ok.any() else (np.zeros((1, q.shape[1])), np.full((1, q.shape[1]), 1e-30))
        outs.append(o[0])
        tols.append(t[0])
    return np.array(outs), np.array(tols)
