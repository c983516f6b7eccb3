"""Outputs that lie over inputs are refused, rows side by side in one buffer are not: no GPU needed."""
import os
import subprocess

import numpy as np
import pytest

from spy_amd import _lib as H
from tests.test_serving_args import append, attend, rows

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HD = 128


def _held(at, es, n_head, n_row, h, r):
    """what a tensor of rows holds, in units of 16 bytes"""
    return set(((at + np.arange(n_row)[:, None, None] * r + np.arange(n_head)[None, :, None] * h + np.arange(0, HD * es, 16)) // 16).ravel().tolist())


def _random(rng, n_head, n_row):
    es = int(rng.choice([2, 4]))
    w = HD * es
    kind = rng.random()
    if kind < 0.35:
        h, r = w, w * n_head
    elif kind < 0.8:                                             # a part of wider rows, heads next to each other or with something between them
        h = w * int(rng.integers(1, 3))
        r = max(int(rng.choice([4096, 8192])), h * n_head)
    else:                                                        # one block per head
        h, r = w * n_row, w
    return (1 << 20) + int(rng.integers(0, 600)) * 64, es, n_head, n_row, h, r


def test_what_is_told_to_meet_meets_and_fused_and_dense_rows_are_told(tmp_path):
    """Pairs at random against the sets of what they hold: never told to meet where they do not, always where both have no gaps or both are parts of rows of one width."""
    out = str(tmp_path / "rows_meet")
    subprocess.check_call(["g++", "-O1", "-std=c++20", "-o", out, os.path.join(ROOT, "tests", "host", "rows_meet.cpp")])
    rng = np.random.default_rng(0)
    pairs = []
    for _ in range(4000):
        n_row = int(rng.integers(1, 6))
        pairs.append((_random(rng, int(rng.choice([1, 2, 4, 8])), n_row), _random(rng, int(rng.choice([1, 2, 4, 8])), n_row)))
    told = subprocess.run([out], input="".join("%d %d %d %d %d %d\n" % t for p in pairs for t in p), capture_output=True, text=True, check=True).stdout.split()
    assert len(told) == len(pairs)
    span = lambda t: (t[2] - 1) * t[4] + HD * t[1]                                                # noqa: E731  (of a row)
    dense = lambda t: span(t) + (t[3] - 1) * t[5] == HD * t[1] * t[2] * t[3]                      # noqa: E731
    n = {"meet": 0, "apart": 0, "fused": 0}
    for (a, b), says in zip(pairs, told):
        meet, fused = bool(_held(*a) & _held(*b)), a[5] == b[5] and span(a) <= a[5] and span(b) <= b[5]
        assert meet or says == "0", (a, b)
        assert says == "1" or not (meet and (fused or (dense(a) and dense(b)))), (a, b)
        n["meet" if meet else "apart"] += 1
        n["fused"] += fused and not dense(a) and not dense(b)
    assert min(n.values()) > 300, n


@pytest.mark.parametrize("at", [4096, 4096 + 16, 4096 + 768, 4096 - 256, 4096 + 8 * 4 * 256 - 16])
def test_attention_refuses_out_over_q(at):
    assert attend(out=rows(4, at=at)) == H.EINVAL


@pytest.mark.parametrize("which", ["q", "k", "v"])
@pytest.mark.parametrize("off", [0, 256, -256])
def test_append_refuses_q_out_over_an_input(which, off):
    at = {"q": 1 << 16, "k": 1 << 17, "v": 1 << 18}
    assert append(**{n: rows(4 if n == "q" else 2, at=at[n]) for n in at}, qo=rows(4, at=at[which] + off)) == H.EINVAL


@pytest.mark.parametrize("off", [2048 - 256, 2048 + 256, 512, 1024 - 5 * 3200])
def test_append_refuses_q_out_over_a_part_of_the_same_wide_rows(off):
    """q | k | v | q_out in one row; q_out one head early, one late (over the next row's q), over q, and over k of rows before"""
    nb = [2, 256, 3200]
    a = dict(q=rows(4, at=1 << 20, nb=nb), k=rows(2, at=(1 << 20) + 1024, nb=nb), v=rows(2, at=(1 << 20) + 1536, nb=nb))
    assert append(**a, qo=rows(4, at=(1 << 20) + off, nb=nb)) == H.EINVAL
