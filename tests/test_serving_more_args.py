"""What the entry points over pages of 8 bits, and those for sequences that begin alike, refuse before any device call: no GPU needed, and the pointers here are never used."""
import ctypes as C

import pytest

from spy_amd import _lib as H
from tests.test_serving_args import batch, pages, rope, rows

B = C.byref


def _ref(x):
    return None if x is None else B(x)


def q8(kind, hd=128, ps=16, G=2, n=10, t=H.I8, at=4096, nb=None):
    return H.tensor(at, t, [hd, ps, G, n] if kind == "k" else [ps, hd, G, n], nb)


def scales(kind, hd=128, ps=16, G=2, n=10, t=H.F16, at=4096, nb=None):
    return H.tensor(at, t, [hd // 32, ps, G, n] if kind == "k" else [ps, hd // 32, G, n], nb)


CACHE = {"kp": q8("k"), "ks": scales("k"), "vp": q8("v"), "vs": scales("v")}


def append(**kw):
    a = {"q": rows(4), "k": rows(2), "v": rows(2), "b": batch(), "rope": rope(), "qo": rows(4), **CACHE, **kw}
    return H.load().spy_hip_paged_append_q8(None, *(_ref(a[n]) for n in ("q", "k", "v", "b", "rope", "qo", "kp", "ks", "vp", "vs")))


def attend(scale=0.1, window=0, scratch=4096, room=None, **kw):
    a = {"q": rows(4), "out": rows(4, at=8192), "b": batch(), **CACHE, **kw}
    L = H.load()
    if room is None:
        room = L.spy_hip_paged_attention_q8_scratch_size(_ref(a["q"]), _ref(a["kp"]), _ref(a["b"]))
    return L.spy_hip_paged_attention_q8(None, *(_ref(a[n]) for n in ("q", "kp", "ks", "vp", "vs", "out", "b")), scale, 1, window, scratch, room)


def prefix(**kw):
    p = H.PagedPrefix(1, 8, 64, 4096, 4096)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def shared(scale=0.1, scratch=4096, room=None, **kw):
    a = {"q": rows(4), "kp": pages("k"), "ks": None, "vp": pages("v"), "vs": None, "out": rows(4, at=8192), "b": batch(), "p": prefix(), **kw}
    L = H.load()
    if room is None:
        room = L.spy_hip_paged_attention_shared_scratch_size(_ref(a["q"]), _ref(a["kp"]), _ref(a["b"]), _ref(a["p"]))
    return L.spy_hip_paged_attention_shared(None, *(_ref(a[n]) for n in ("q", "kp", "ks", "vp", "vs", "out", "b", "p")), scale, scratch, room)


INVALID_BATCH = [dict(b=None), dict(b=batch(n_seq=0)), dict(b=batch(max_new=0)), dict(b=batch(max_kv=0)), dict(b=batch(row_start=None)), dict(b=batch(kv_len=4098)), dict(b=batch(pages=None)),
                 dict(b=batch(page_stride=0))]
INVALID_CACHE = [dict(kp=None), dict(ks=None), dict(vp=None), dict(vs=None), dict(kp=q8("k", at=0)), dict(kp=q8("k", at=4104)), dict(ks=scales("k", at=4100)), dict(vs=scales("v", at=0)),
                 dict(vp=q8("v", G=1), vs=scales("v", G=1)), dict(vp=q8("v", n=11), vs=scales("v", n=11)), dict(vp=q8("v", ps=32), vs=scales("v", ps=32)), dict(ks=scales("k", n=9)), dict(ks=scales("k", hd=64)),
                 dict(vs=scales("v", ps=32)), dict(vs=scales("v", hd=256)), dict(kp=q8("k", nb=[1, 136, 2176, 4352])), dict(kp=q8("k", nb=[2, 256, 4096, 8192])), dict(vp=q8("v", nb=[1, 24, 4096, 8192])),
                 dict(ks=scales("k", nb=[2, 16, 256, 512])), dict(vs=scales("v", nb=[2, 36, 144, 288])), dict(kp=q8("k", n=0), ks=scales("k", n=0)), dict(vs=scales("v", nb=[4, 64, 256, 512]))]
UNSUPPORTED_CACHE = [dict(kp=q8("k", t=H.F16)), dict(ks=scales("k", t=H.F32)), dict(vs=scales("v", t=H.F32)), dict(kp=q8("k", hd=96), ks=scales("k", hd=96)), dict(kp=q8("k", ps=48), ks=scales("k", ps=48)),
                     dict(kp=pages("k"))]


@pytest.mark.parametrize("kw", INVALID_BATCH + INVALID_CACHE + [
    dict(q=None), dict(qo=None), dict(k=None), dict(v=None), dict(q=rows(3)), dict(k=rows(3)), dict(v=rows(2, n_row=9)), dict(q=rows(4, hd=64)), dict(q=rows(4, at=4104)),
    dict(k=rows(2, n_row=0), v=rows(2, n_row=0)), dict(rope=rope(num_dim=0)), dict(rope=rope(num_dim=24)), dict(rope=rope(num_dim=144)), dict(rope=rope(freq_base=0.0)),
    dict(qo=rows(4, at=4096 + 256), q=rows(4))])
def test_append_refuses(kw):
    assert append(**kw) == H.EINVAL


@pytest.mark.parametrize("kw", UNSUPPORTED_CACHE + [dict(k=rows(2, t=H.F32)), dict(qo=rows(4, t=H.F32)), dict(k=rows(2, t=H.I8)), dict(rope=rope(mode=4)), dict(rope=rope(extend_factor=1.0))])
def test_append_does_not_support(kw):
    assert append(**kw) == H.EUNSUPPORTED


@pytest.mark.parametrize("kw", INVALID_BATCH + INVALID_CACHE + [dict(q=None), dict(out=None), dict(q=rows(3), out=rows(3, at=8192)), dict(out=rows(4, n_row=9, at=8192)), dict(q=rows(4, hd=64)),
                                                                dict(out=rows(4, at=8196)), dict(window=-1), dict(scale=float("nan")), dict(scale=0.0), dict(out=rows(4))])
def test_attention_refuses(kw):
    assert attend(**kw) == H.EINVAL


@pytest.mark.parametrize("kw", UNSUPPORTED_CACHE + [dict(q=rows(4, t=H.F32)), dict(out=rows(4, t=H.I8, at=8192))])
def test_attention_does_not_support(kw):
    assert attend(**kw) == H.EUNSUPPORTED


@pytest.mark.parametrize("kw", INVALID_BATCH + [
    dict(p=None), dict(p=prefix(n_group=0)), dict(p=prefix(n_group=(1 << 20) + 1)), dict(p=prefix(max_rows=0)), dict(p=prefix(max_prefix=0)), dict(p=prefix(max_prefix=(1 << 30) + 1)),
    dict(p=prefix(seq_start=None)), dict(p=prefix(length=None)), dict(p=prefix(length=4098)), dict(kp=None), dict(vp=None), dict(q=None), dict(out=None), dict(out=rows(4)), dict(scale=float("nan")),
    dict(ks=scales("k")), dict(ks=scales("k"), vs=scales("v")), dict(kp=q8("k"), vp=q8("v")), dict(kp=q8("k"), vp=q8("v"), ks=scales("k")), dict(kp=q8("k"), vp=q8("v"), ks=scales("k"), vs=scales("v", n=9)),
    dict(vp=q8("v")), dict(vp=pages("v", n=11)), dict(q=rows(3), out=rows(3, at=8192))])
def test_shared_refuses(kw):
    assert shared(**kw) == H.EINVAL


@pytest.mark.parametrize("kw", [dict(q=rows(4, t=H.F32)), dict(out=rows(4, t=H.I32, at=8192)), dict(kp=pages("k", hd=96), vp=pages("v", hd=96))])
def test_shared_does_not_support(kw):
    assert shared(**kw) == H.EUNSUPPORTED


def test_scratch():
    L = H.load()
    long = batch(max_kv=100000, page_stride=10000)
    need = L.spy_hip_paged_attention_q8_scratch_size(B(rows(4)), B(q8("k")), B(long))
    assert need == L.spy_hip_paged_attention_scratch_size(B(rows(4)), B(pages("k")), B(long)) > 0
    assert attend(b=long, room=need - 1) == H.ENOSPACE
    assert attend(b=long, scratch=None, room=need) == H.EINVAL
    assert attend(b=long, scratch=4096 + 16, room=need) == H.EINVAL
    assert L.spy_hip_paged_attention_q8_scratch_size(B(rows(4)), B(pages("k")), B(long)) == 0
    need = L.spy_hip_paged_attention_shared_scratch_size(B(rows(4)), B(pages("k")), B(batch()), B(prefix()))
    assert need == L.spy_hip_paged_attention_shared_scratch_size(B(rows(4)), B(q8("k")), B(batch()), B(prefix())) > 0
    assert shared(room=need - 1) == H.ENOSPACE
    assert shared(scratch=None) == H.EINVAL
    assert shared(scratch=4096 + 16) == H.EINVAL
    assert L.spy_hip_paged_attention_shared_scratch_size(B(rows(4)), B(pages("k")), B(batch()), None) == 0


@pytest.mark.parametrize("n_row,seqs,groups,new", [(1 << 27, 1 << 20, 1, 1), (1 << 20, 1 << 20, 1, 1), (64, 4, 1 << 20, 16), (1 << 24, 16, 1, 1 << 20)])
def test_shared_batches_that_no_launch_can_hold(n_row, seqs, groups, new):
    kw = dict(q=rows(32, n_row=n_row, at=1 << 44), out=rows(32, n_row=n_row, at=1 << 45), kp=pages("k", G=16), vp=pages("v", G=16), b=batch(n_seq=seqs, max_new=new),
              p=prefix(n_group=groups, max_rows=n_row))
    assert shared(**kw, room=1 << 60) == H.EINVAL


@pytest.mark.parametrize("n_row,new", [((1 << 24) + 5, 1), (1 << 27, 9)])
def test_append_of_more_rows_than_threads(n_row, new):
    a = {n: rows(16, n_row=n_row, at=(i + 1) << 44) for i, n in enumerate(("q", "k", "v", "qo"))}
    assert append(**a, kp=q8("k", G=16), ks=scales("k", G=16), vp=q8("v", G=16), vs=scales("v", G=16), b=batch(n_seq=1, max_new=new)) == H.EINVAL


def verify(t=H.F32, n=1000, n_row=5, at=4096, nb=None, uniform=4096, param=True, draft=True, drafted=4096, row_start=4096, n_seq=2, accept=4096, tokens=4096, accepted=4096, probs=None, scratch=4096,
           room=1 << 30, draft_param=True, **kw):
    l = H.tensor(at, t, [n, n_row], nb)
    d = H.tensor(kw.get("draft_at", 8192), kw.get("draft_t", H.F32), [kw.get("draft_n", n), kw.get("draft_row", n_row)])
    p = H.SampleParam(uniform=uniform, top_p=kw.get("top_p"))
    q = H.SampleParam(top_p=kw.get("draft_top_p"))
    return H.load().spy_hip_sample_verify(None, B(l), B(p) if param else None, B(d) if draft else None, B(q) if draft_param else None, drafted, row_start, n_seq, accept, tokens, accepted, probs, scratch,
                                          room)


@pytest.mark.parametrize("kw", [dict(n=0), dict(n_row=0), dict(n=(1 << 18) + 1), dict(at=0), dict(at=4097), dict(nb=[8, 8000]), dict(nb=[4, 4002]), dict(uniform=None), dict(uniform=4098), dict(param=False),
                                dict(drafted=None), dict(drafted=4097), dict(row_start=None), dict(row_start=4098), dict(n_seq=0), dict(n_seq=-1), dict(n_seq=(1 << 20) + 1), dict(accept=None),
                                dict(accept=4099), dict(tokens=None), dict(tokens=4097), dict(accepted=None), dict(accepted=4098), dict(probs=4097), dict(scratch=None), dict(scratch=4112),
                                dict(draft_at=0), dict(draft_at=8194), dict(draft_n=999), dict(draft_row=6), dict(draft_top_p=4098), dict(top_p=4097), dict(n_row=1 << 21), dict(n_row=1 << 22, draft=False)])
def test_verify_refuses(kw):
    assert verify(**kw) == H.EINVAL


def test_verify_types_and_scratch():
    assert verify(t=H.F16) == H.EUNSUPPORTED
    assert verify(draft_t=H.F16) == H.EUNSUPPORTED
    L = H.load()
    need = L.spy_hip_sample_verify_scratch_size(B(H.tensor(4096, H.F32, [1000, 5])), 2)
    assert need > 0
    assert verify(room=need - 1) == H.ENOSPACE
    assert L.spy_hip_sample_verify_scratch_size(None, 2) == 0
