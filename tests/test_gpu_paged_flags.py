"""Batches whose arrays do not fit the launch raise the flag in both entry points, whichever way the rows are gone through, also where no row belongs to the entry."""
import numpy as np
import pytest

from tests import paged_util as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wrong", ["none", "descending", "ended and too long", "ended and negative", "past the rows", "past the pages"])
@pytest.mark.parametrize("new", [2, 90])
def test_append_and_attention_raise_the_flag(hip, new, wrong):
    """new 2: a row per workgroup, 90: V in tiles.  Sequences 40 and 69 take no part, behind the first 64 that are looked at together one of them."""
    print("flags: new %d %s" % (new, wrong), flush=True)
    rng = np.random.default_rng(new)
    seqs = [(1, 20)] * 70
    seqs[3] = (new, 100)
    seqs[40] = seqs[69] = (0, 20)
    p = P.Paged(rng, seqs, 2, 1, 64, 16)
    p.store()
    p.upload()
    start, kv = p.row_start.copy(), p.kv.astype(np.int32)
    if wrong == "descending":
        start[70] = start[69] - 1
    elif wrong == "ended and too long":
        kv[69] = int(p.kv.max()) + 1
    elif wrong == "ended and negative":
        kv[40] = -1
    elif wrong == "past the rows":
        start[70] = p.rows + 1
    elif wrong == "past the pages":
        p.batch.max_kv = 4096
        kv[69] = p.table.shape[1] * 16 + 1
    p.d_start.upload(start)
    p.d_kv.upload(kv)
    q, k, v = (rng.standard_normal((p.rows, n, 64)).astype(np.float16) for n in (2, 1, 1))
    P.flag()
    rc, _ = P.run_append(p, q, k, v, None, np.float16)
    assert rc == 0 and (P.flag() != 0) == (wrong != "none") and P.flag() == 0
    got_k, got_v = p.pools()
    for row, s, pos in p.rows_of():
        assert np.array_equal(p.k_at(got_k, s, pos), k[row]) and np.array_equal(p.v_at(got_v, s, pos), v[row])
    P.run_attention(p, q, True)
    assert (P.flag() != 0) == (wrong != "none")


@pytest.mark.parametrize("by_head", [False, True])
def test_append_of_parts_of_one_wide_row(hip, by_head):
    """q, k, v and q_out side by side in one buffer, as blocks of heads or head by head, which is no overlap: all of q_out is written, and nothing else."""
    from spy_amd import _lib as H
    rng = np.random.default_rng(1)
    p = P.Paged(rng, [(1, 20), (12, 30)], 2, 2, 64, 16)
    p.upload()
    wide = rng.standard_normal((p.rows, 9, 64)).astype(np.float16)
    at = {"q": 0, "k": 1, "v": 2, "qo": 3} if by_head else {"q": 0, "k": 2, "v": 4, "qo": 6}
    head = 4 if by_head else 1
    buf = H.DeviceBuffer.from_numpy(wide.view(np.uint16))
    t = {n: H.tensor(buf, H.F16, [64, 2, p.rows], [2, 128 * head, 9 * 128], offset=128 * o) for n, o in at.items()}
    B = P.C.byref
    H.check(H.load().spy_hip_paged_append(None, B(t["q"]), B(t["k"]), B(t["v"]), B(p.batch), None, B(t["qo"]), B(p.t_k), B(p.t_v)), "spy_hip_paged_append")
    got, n = buf.download(np.float16).reshape(wide.shape), int(p.row_start[-1])
    want = wide.copy()
    for h in range(2):
        want[:n, at["qo"] + head * h] = wide[:n, at["q"] + head * h]
    assert np.array_equal(got, want) and P.flag() == 0
