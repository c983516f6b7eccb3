"""Batches that no launch can hold are refused, before any device call; no GPU needed."""
import ctypes as C

import pytest

from spy_amd import _lib as H
from tests.test_serving_args import append, attend, batch, pages, rows, sample

B = C.byref


@pytest.mark.parametrize("n_row", [1 << 22, 1 << 30])
def test_sampling_of_more_rows_than_threads(n_row):
    assert sample(n=4, n_row=n_row) == H.EINVAL


@pytest.mark.parametrize("new,seqs", [(1, 1), (9, 1), (9, 1 << 20)])
def test_append_of_more_rows_than_threads(new, seqs):
    """rows one by one; in tiles; tiles for many sequences"""
    n_row = (1 << 24) + 5 if seqs == 1 else 1 << 20
    h = 2 if new == 1 else 16
    a = {n: rows(h, n_row=n_row * (8 if new == 9 and seqs == 1 else 1), at=(i + 1) << 44) for i, n in enumerate(("q", "k", "v", "qo"))}
    assert append(**a, kp=pages("k", G=h), vp=pages("v", G=h), b=batch(n_seq=seqs, max_new=new)) == H.EINVAL


@pytest.mark.parametrize("seqs,new,hd", [(1 << 20, 1, 128), (1 << 20, 1, 256), (1 << 19, 40, 128), (1 << 20, 40, 256)])
def test_attention_of_more_sequences_than_threads(seqs, new, hd):
    kw = dict(q=rows(32, n_row=1 << 20, hd=hd, at=1 << 44), out=rows(32, n_row=1 << 20, hd=hd, at=1 << 45), kp=pages("k", G=16, hd=hd), vp=pages("v", G=16, hd=hd), b=batch(n_seq=seqs, max_new=new))
    assert attend(**kw, room=1 << 50) == H.EINVAL
    assert H.load().spy_hip_paged_attention_scratch_size(B(kw["q"]), B(kw["kp"]), B(kw["b"])) == 0
