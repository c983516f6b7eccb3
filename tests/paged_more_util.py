"""Caches in pages of 8 bits, and batches whose sequences begin alike, for the tests (beside tests/paged_util.py)."""
import ctypes as C

import numpy as np

from spy_amd import _lib as H
from tests import paged_util as P

B = C.byref


def q8_blocks(x):
    """float32 values, blocks of 32 along the last axis: whole numbers and scales as Q8_0 has them, every step rounded to 32 bits (a float's division and product)"""
    x = np.asarray(x, np.float32)
    b = x.reshape(x.shape[:-1] + (-1, 32))
    top = np.abs(b).max(axis=-1, keepdims=True)                  # NaN if any is
    with np.errstate(all="ignore"):
        inv = np.where(top > np.float32(1e-36), np.float32(127) / top, np.float32(0)).astype(np.float32)
        q = np.nan_to_num(np.rint(b * inv), nan=0).astype(np.int8).reshape(x.shape)
        d = (top / np.float32(127)).astype(np.float16)[..., 0]
    d[~np.isfinite(d)] = np.nan
    return q, d


def q8_values(q, d):
    """what the blocks stand for, as fp16"""
    with np.errstate(all="ignore"):
        return (q.astype(np.float32) * np.repeat(d, 32, axis=-1).astype(np.float32)).astype(np.float16)


class PagedQ8(P.Paged):
    """A batch whose pools are held in 8 bits as well: `k_pool` and `v_pool` have what they stand for.  K scales are [page][head][position][block] whatever the pages' order."""

    def quantize(self):
        """the pools as they are, to 8 bits; what is NaN gets whole numbers that are not 0 and scales of NaN"""
        turn = np.swapaxes
        for name in ("k", "v"):
            pool = getattr(self, name + "_pool").astype(np.float32)
            pool = pool if name == "k" else turn(pool, 2, 3)
            q, d = q8_blocks(pool)
            q[np.repeat(np.isnan(d), 32, axis=-1)] = 85
            value = q8_values(q, d)
            setattr(self, name + "_pool", np.ascontiguousarray(value if name == "k" else turn(value, 2, 3)))
            if name == "v":
                q, d = turn(q, 2, 3), turn(d, 2, 3)
            elif self.token_major:
                d = turn(d, 1, 2)
            setattr(self, name + "_q", np.ascontiguousarray(q))
            setattr(self, name + "_d", np.ascontiguousarray(d))
        for s in range(len(self.seqs)):
            for pos in range(int(self.kv[s])):
                if self.table[s, pos // self.page] >= 0:
                    self.k_rows[s][pos], self.v_rows[s][pos] = self.k_at(self.k_pool, s, pos), self.v_at(self.v_pool, s, pos)

    def upload(self):
        super().upload()
        up = H.DeviceBuffer.from_numpy
        self.d_kq, self.d_vq, self.d_kd, self.d_vd = up(self.k_q), up(self.v_q), up(self.k_d.view(np.uint16)), up(self.v_d.view(np.uint16))
        hd, ps, G, n = self.hd, self.page, self.kv_heads, self.n_page
        self.t_kq = H.tensor(self.d_kq, H.I8, [hd, ps, G, n], [1, G * hd, hd, ps * G * hd] if self.token_major else None)
        self.t_vq = H.tensor(self.d_vq, H.I8, [ps, hd, G, n])
        self.t_kd, self.t_vd = H.tensor(self.d_kd, H.F16, [hd // 32, ps, G, n]), H.tensor(self.d_vd, H.F16, [ps, hd // 32, G, n])

    def q8_pools(self):
        """(whole numbers, scales) of K and of V^T, as they are on the device"""
        get = lambda buf, like, t: buf.download(t).view(like.dtype).reshape(like.shape)           # noqa: E731
        return get(self.d_kq, self.k_q, np.int8), get(self.d_kd, self.k_d, np.uint16), get(self.d_vq, self.v_q, np.int8), get(self.d_vd, self.v_d, np.uint16)


def _run(p, q, f32, need, call, stream=None):
    """call(tensors of q and out, scratch, its size); the output, with checks of what lies behind the scratch"""
    L = H.load()
    dq = H.DeviceBuffer.from_numpy(q.view(np.uint16))
    out = H.DeviceBuffer.from_numpy(np.full(q.shape, 77, np.float32 if f32 else np.float16).view(np.uint32 if f32 else np.uint16))
    tq, to = H.tensor(dq, H.F16, [p.hd, p.heads, p.rows]), H.tensor(out, H.F32 if f32 else H.F16, [p.hd, p.heads, p.rows])
    size = need(L, tq)
    scratch = H.DeviceBuffer(size + 256)
    scratch.fill(0xFF)                                           # NaN wherever something is read before it is written
    H.check(call(L, tq, to, scratch.ptr, size))
    H.sync()
    assert (scratch.download(np.uint8, offset=size) == 0xFF).all()
    return out.download(np.float32 if f32 else np.float16).reshape(q.shape)


def run_attention_q8(p, q, f32, causal=1, window=0, scale=None, stream=None):
    scale = 1.0 / np.sqrt(p.hd) if scale is None else scale
    return _run(p, q, f32, lambda L, tq: L.spy_hip_paged_attention_q8_scratch_size(B(tq), B(p.t_kq), B(p.batch)),
                lambda L, tq, to, scratch, size: L.spy_hip_paged_attention_q8(stream, B(tq), B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd), B(to), B(p.batch), scale, causal, window, scratch, size))


def share(p, start, length):
    """the first length[g] tokens of the sequences start[g] .. start[g + 1] - 1 made alike (before store())"""
    for g, n in enumerate(length):
        for s in range(start[g] + 1, start[g + 1]):
            p.k_rows[s][:n], p.v_rows[s][:n] = p.k_rows[start[g]][:n], p.v_rows[start[g]][:n]


def shared_batch(p, start, length, gone=-1):
    """the groups on the device (after upload()); pages that lie in what a group has in common are taken out of the other sequences' tables"""
    table = p.table.copy()
    for g, n in enumerate(length):
        for s in range(start[g] + 1, start[g + 1]):
            table[s, :n // p.page] = gone
    p.d_table.upload(table)
    p.d_groups, p.d_length = H.DeviceBuffer.from_numpy(np.asarray(start, np.int32)), H.DeviceBuffer.from_numpy(np.asarray(length, np.int32))
    rows = [int(p.row_start[start[g + 1]] - p.row_start[start[g]]) for g in range(len(length))]
    p.prefix = H.PagedPrefix(len(length), max(1, max(rows)), max(1, max(length)), p.d_groups.ptr, p.d_length.ptr)


def run_shared(p, q, f32, q8=False, scale=None, stream=None):
    scale = 1.0 / np.sqrt(p.hd) if scale is None else scale
    k, ks, v, vs = (B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd)) if q8 else (B(p.t_k), None, B(p.t_v), None)
    return _run(p, q, f32, lambda L, tq: L.spy_hip_paged_attention_shared_scratch_size(B(tq), k, B(p.batch), B(p.prefix)),
                lambda L, tq, to, scratch, size: L.spy_hip_paged_attention_shared(stream, B(tq), k, ks, v, vs, B(to), B(p.batch), B(p.prefix), scale, scratch, size))


def run_append_q8(p, q, k, v, rope, dtype, stream=None):
    """q, k, v: [rows][heads][hd] arrays (q may be None); returns the return code and q_out's array"""
    t = {np.float32: H.F32, np.float16: H.F16}[dtype]
    L = H.load()
    bufs = [None if x is None else H.DeviceBuffer.from_numpy(x.view(np.uint32 if dtype is np.float32 else np.uint16)) for x in (q, k, v)]
    tq, tk, tv = (None if x is None else H.tensor(b, t, [x.shape[2], x.shape[1], x.shape[0]]) for x, b in zip((q, k, v), bufs))
    qo = None if q is None else H.DeviceBuffer.from_numpy(np.full(q.shape, 77, np.float16).view(np.uint16))
    tqo = None if q is None else H.tensor(qo, H.F16, [q.shape[2], q.shape[1], q.shape[0]])
    ref = lambda x: None if x is None else B(x)                                                   # noqa: E731
    rc = L.spy_hip_paged_append_q8(stream, ref(tq), B(tk), B(tv), B(p.batch), ref(rope), ref(tqo), B(p.t_kq), B(p.t_kd), B(p.t_vq), B(p.t_vd))
    H.sync()
    return rc, None if q is None else qo.download(np.float16).reshape(q.shape)
