"""What the batch entry points refuse, before any device call: no GPU needed, and the pointers here are never used."""
import ctypes as C

import pytest

from spy_amd import _lib as H

B = C.byref


def batch(**kw):
    b = H.PagedBatch(2, 4, 100, 4096, 4096, 4096, 8)
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def rows(n_head, n_row=8, hd=128, t=H.F16, at=4096, nb=None):
    return H.tensor(at, t, [hd, n_head, n_row], nb)


def pages(kind, hd=128, ps=16, G=2, n=10, t=H.F16, at=4096, nb=None):
    return H.tensor(at, t, [hd, ps, G, n] if kind == "k" else [ps, hd, G, n], nb)


def rope(**kw):
    return H.RopeParam(**{"mode": 0, "num_dim": 128, "freq_base": 1e4, "freq_scale": 1.0, "attention_factor": 1.0, **kw})


def append(**kw):
    a = {"q": rows(4), "k": rows(2), "v": rows(2), "b": batch(), "rope": rope(), "qo": rows(4), "kp": pages("k"), "vp": pages("v"), **kw}
    ref = lambda x: None if x is None else B(x)                                                   # noqa: E731
    return H.load().spy_hip_paged_append(None, *(ref(a[n]) for n in ("q", "k", "v", "b", "rope", "qo", "kp", "vp")))


def attend(scale=0.1, window=0, scratch=4096, room=None, **kw):
    a = {"q": rows(4), "kp": pages("k"), "vp": pages("v"), "out": rows(4, at=8192), "b": batch(), **kw}
    ref = lambda x: None if x is None else B(x)                                                   # noqa: E731
    L = H.load()
    if room is None:
        room = L.spy_hip_paged_attention_scratch_size(ref(a["q"]), ref(a["kp"]), ref(a["b"]))
    return L.spy_hip_paged_attention(None, *(ref(a[n]) for n in ("q", "kp", "vp", "out", "b")), scale, 1, window, scratch, room)


INVALID_BATCH = [dict(b=None), dict(b=batch(n_seq=0)), dict(b=batch(n_seq=-1)), dict(b=batch(max_new=0)), dict(b=batch(max_kv=0)), dict(b=batch(row_start=None)), dict(b=batch(kv_len=None)),
                 dict(b=batch(pages=None)), dict(b=batch(pages=4097)), dict(b=batch(page_stride=0)), dict(b=batch(max_kv=(1 << 30) + 1)), dict(b=batch(max_new=(1 << 24) + 1)),
                 dict(kp=None), dict(vp=None), dict(kp=pages("k", at=0)), dict(kp=pages("k", at=4104)), dict(vp=pages("v", at=4104)), dict(vp=pages("v", G=1)), dict(vp=pages("v", n=11)),
                 dict(vp=pages("v", ps=32)), dict(kp=pages("k", nb=[2, 264, 4224, 8448])), dict(vp=pages("v", nb=[2, 40, 4096, 8192])), dict(kp=pages("k", n=0)), dict(kp=pages("k", G=0))]


@pytest.mark.parametrize("kw", INVALID_BATCH + [
    dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(q=rows(3)), dict(q=rows(5)), dict(k=rows(3)), dict(v=rows(2, n_row=9)), dict(q=rows(4, hd=64)), dict(q=rows(4, at=4104)),
    dict(qo=rows(4, nb=[2, 264, 1056])), dict(k=rows(2, n_row=0), v=rows(2, n_row=0)), dict(rope=rope(num_dim=0)), dict(rope=rope(num_dim=24)), dict(rope=rope(num_dim=144)),
    dict(rope=rope(freq_base=0.0)), dict(rope=rope(freq_base=-1.0)), dict(rope=rope(freq_scale=float("nan"))), dict(rope=rope(freq_base=float("inf"))), dict(q=rows(4, nb=[4, 256, 1024]))])
def test_append_refuses(kw):
    assert append(**kw) == H.EINVAL


@pytest.mark.parametrize("kw", [dict(kp=pages("k", hd=96), vp=pages("v", hd=96)), dict(kp=pages("k", ps=8), vp=pages("v", ps=8)), dict(kp=pages("k", ps=48), vp=pages("v", ps=48)),
                                dict(kp=pages("k", ps=2048), vp=pages("v", ps=2048)), dict(k=rows(2, t=H.F32)), dict(v=rows(2, t=H.F32)), dict(qo=rows(4, t=H.F32)), dict(q=rows(4, t=H.F32)),
                                dict(k=rows(2, t=H.I32)), dict(rope=rope(mode=4)), dict(rope=rope(mode=1)), dict(rope=rope(extend_factor=1.0)), dict(rope=rope(xpos_base=512.0))])
def test_append_does_not_support(kw):
    assert append(**kw) == H.EUNSUPPORTED


@pytest.mark.parametrize("kw", INVALID_BATCH + [dict(q=None), dict(out=None), dict(q=rows(3), out=rows(3)), dict(out=rows(4, n_row=9)), dict(out=rows(2)), dict(q=rows(4, hd=64)), dict(q=rows(4, at=0)),
                                                dict(out=rows(4, at=4100)), dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=0.0), dict(scale=1e-38), dict(scale=-1e25),
                                                dict(out=rows(4))])
def test_attention_refuses(kw):
    assert attend(**kw) == H.EINVAL


def test_attention_types_and_scratch():
    assert attend(q=rows(4, t=H.F32)) == H.EUNSUPPORTED
    assert attend(out=rows(4, t=H.I32)) == H.EUNSUPPORTED
    long = batch(max_kv=100000, page_stride=10000)
    need = H.load().spy_hip_paged_attention_scratch_size(B(rows(4)), B(pages("k")), B(long))
    assert need > 0
    assert attend(b=long, room=need - 1) == H.ENOSPACE
    assert attend(b=long, scratch=None, room=need) == H.EINVAL
    assert attend(b=long, scratch=4096 + 16, room=need) == H.EINVAL
    assert H.load().spy_hip_paged_attention_scratch_size(None, B(pages("k")), B(long)) == 0


def sample(t=H.F32, n=1000, n_row=3, at=4096, nb=None, uniform=4096, tokens=4096, param=True, ne2=1):
    l = H.tensor(at, t, [n, n_row, ne2], nb)
    p = H.SampleParam(uniform=uniform)
    L = H.load()
    return L.spy_hip_sample(None, B(l), B(p) if param else None, tokens, None, 4096, L.spy_hip_sample_scratch_size(B(l)))


@pytest.mark.parametrize("kw", [dict(n=0), dict(n_row=0), dict(n=(1 << 18) + 1), dict(at=0), dict(at=4097), dict(uniform=None), dict(uniform=4098), dict(tokens=None), dict(tokens=4099), dict(param=False),
                                dict(nb=[4, 4002]), dict(nb=[8, 8000]), dict(ne2=2)])
def test_sample_refuses(kw):
    assert sample(**kw) == H.EINVAL


def test_sample_does_not_support_other_types():
    assert sample(t=H.F16) == H.EUNSUPPORTED
