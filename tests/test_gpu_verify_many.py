"""Verification of drafts with so many rows that numbers of threads pass 31 bits: the bits of calls of an eighth of the rows, and the definition where requests are short."""
import numpy as np
import pytest

from tests.test_gpu_paged import P
from tests.test_gpu_verify import check, drawn_from, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,drafter", [((1 << 20) + 1000, True), ((1 << 21) + 1000, False)])
def test_rows_past_31_bits_of_threads(hip, rows, drafter):
    from spy_amd import _lib as H
    rng = np.random.default_rng(31)
    vocab = 12
    start = np.concatenate([np.arange(0, 4000, 4), np.arange(4000, rows, 1000), [rows]])
    logits = rng.standard_normal((rows, vocab), dtype=np.float32) * 2
    draft = logits + rng.standard_normal((rows, vocab), dtype=np.float32) * np.float32(0.5) if drafter else None
    accept, uniform = rng.random(rows, dtype=np.float32), rng.random(rows, dtype=np.float32)
    drafted = rng.integers(0, vocab, rows).astype(np.int32)
    drafted[:4000] = drawn_from(rng, draft[:4000]) if drafter else logits[:4000].argmax(axis=1)
    settings = dict(top_p=0.95)
    tokens, accepted, probs = run(H, logits, drafted, start, accept, uniform, settings, draft)
    assert P.flag() == 0
    print("%d rows in one call" % rows, flush=True)
    short = slice(0, 4000)
    check((tokens[short], accepted[:1000], probs[short]), logits[short], drafted[short], start[:1001], accept[short], uniform[short], settings, draft[short] if drafter else None)
    ends = np.linspace(0, len(start) - 1, 9).astype(int)
    for a, b in zip(ends, ends[1:]):
        r = slice(int(start[a]), int(start[b]))
        part = run(H, logits[r], drafted[r], start[a:b + 1] - start[a], accept[r], uniform[r], settings, draft[r] if drafter else None)
        for got, want in zip((tokens[r], accepted[a:b], probs[r]), part):
            assert np.array_equal(got.view(np.uint32), want.view(np.uint32)), (a, b)
