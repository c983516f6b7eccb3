"""How many bits of a probability reach an F16 output of sequences that begin alike: as many as with spy_hip_paged_attention, whose sequences of up to 16 rows have two fp16 terms, whatever the rows
of the whole group are.

Scores are 0 or -1 (times the scale), exact, for every third key and the others, and the scale is such that e^-1 of the largest is 2^-1 (1 + 2^-11.1): as one fp16 term it would be off by that 2^-11.1.
Both kinds weigh about half, with V of 1 and -1, so that this moves an output by 2 * 1/2 * 1/2 * 2^-11.1 = 2.2e-4.  What the kernels are off by, relative to the sum of p |v| = 1: the exponent, at most 16
in magnitude, by 2^-24 of itself for its rounding and 2^-23 of the score, times ln 2, and the exponential by 2^-23: 14 * 2^-24 in all; two terms by 2^-22; n additions above and below the line by
n 2^-24 each.  The output's own half step is 2^-11 of it, and it is near 0."""
import numpy as np
import pytest

from tests import paged_more_util as M
from tests import paged_util as P

pytestmark = pytest.mark.gpu

CASES = [
    # sequences (new, cached), groups, tokens in common, heads, kv heads, hd, page
    ([(1, 420 + i) for i in range(20)], [0, 20], [400], 8, 2, 64, 32),                 # single tokens: 80 rows of a group
    ([(1, 300 + i) for i in range(12)], [0, 12], [290], 16, 2, 128, 16),
    ([(2, 400)] * 9, [0, 9], [390], 4, 1, 256, 64),
    ([(1, 440)] + [(1, 390)] * 40, [0, 41], [380], 4, 4, 128, 64),                     # 41 rows, heads by themselves
    ([(1, 320), (150, 460), (1, 310), (4, 330)], [0, 4], [300], 8, 2, 128, 32),        # single tokens beside a chunk: before it, and behind it in the same tile and in one of their own
    ([(31, 331), (1, 301), (97, 397), (1, 309)], [0, 4], [300], 4, 4, 64, 16),         # (the last token in a tile that begins with it)
    ([(60, 260), (3, 203)] * 3, [0, 2, 6], [200, 190], 4, 2, 256, 16),
    ([(1, 270)] * 70 + [(20, 290)], [0, 71], [256], 2, 1, 128, 128),                   # more sequences than lanes
]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_two_terms_for_sequences_of_few_rows(hip, case, q8):
    seqs, start, length, heads, kv_heads, hd, page = CASES[case]
    print("case %d" % case, flush=True)
    rng = np.random.default_rng(700 + case)
    p = M.PagedQ8(rng, seqs, heads, kv_heads, hd, page)
    sign = rng.choice([-1.0, 1.0], (kv_heads, hd))
    for s in range(len(seqs)):
        near = np.arange(int(p.kv[s])) % 3 == 0
        p.k_rows[s][:] = 0
        p.k_rows[s][~near, :, 5] = -1
        p.v_rows[s][:] = np.where(near[:, None, None], sign, -sign)
    M.share(p, start, length)
    p.store()
    p.quantize() if q8 else None
    M.PagedQ8.upload(p) if q8 else P.Paged.upload(p)
    M.shared_batch(p, start, length)
    q = np.zeros((p.rows, heads, hd), np.float16)
    q[:, :, 5] = 1
    q[:, :, 6] = rng.standard_normal((p.rows, heads))            # (meets zeros)
    scale = float(np.float32((1 - np.log2(1 + 2.0 ** -11.1)) * np.log(2)))
    got = M.run_shared(p, q, False, q8, scale=scale).astype(np.float64)
    assert P.flag() == 0
    checked = 0
    for s, (new, kv) in enumerate(seqs):
        if new * heads // kv_heads > 16:
            continue
        assert kv < 450 and set(np.unique(np.abs(p.v_rows[s].astype(np.float64)))) == {1.0} and set(np.unique(p.k_rows[s][:, :, 5].astype(np.float64))) == {-1.0, 0.0}
        for i in range(new):
            pos = np.arange(kv - new + i + 1)
            w = np.where(pos % 3 == 0, 1.0, np.exp(-scale))
            want = (w * np.where(pos % 3 == 0, 1, -1)).sum() / w.sum() * sign
            tol = 2 * (len(pos) + 14) * P.EPS32 + 2.0 ** -22
            tol = tol + P.EPS16 * (np.abs(want) + tol) + 2.0 ** -25
            assert tol.max() < 1.2e-4
            off = np.abs(got[int(p.row_start[s]) + i].reshape(kv_heads, -1, hd) - want[:, None])
            assert (off <= tol[:, None]).all(), (s, i, off.max(), tol.max())
            checked += off.size
    assert checked > 500
