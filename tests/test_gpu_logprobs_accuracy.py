"""Token log probabilities of enough rows that a thread's share has a thousand values, some shares with a clear candidate, next to whose one the bulk's terms
are below half a step: the sums' rounding stays below that of the results.

Bound. ln p = (x - m) - ln Z: two F32 differences (2^-24 each of at most |ln p| where ln Z <= |ln p|) and ln Z itself (logf: 2^-23; Z's sum of n / 16 batches a thread, of random sign
over 256 threads, less): 2^-24 (1 + 1 + 2) / sqrt(3) as a root mean square, 1.4e-7. The entropy is a difference of two such terms, the smaller of which is
at most the entropy's size here."""
import numpy as np
import pytest

from parity import rel_l2
from test_gpu_logprobs import backend, run  # noqa: F401

pytestmark = pytest.mark.gpu


def test_long_shares(backend):
    rows, count, k = 444, 248000, 3
    rng = np.random.default_rng(1)
    x = rng.standard_normal((rows, count), dtype=np.float32) * np.float32(2.5)
    at = rng.integers(0, count, (rows, 8))
    x[np.arange(rows)[:, None], at] += rng.random((rows, 8), dtype=np.float32) * 16
    tokens = rng.integers(0, count, rows)
    lp, ent, top, tlp = run(backend, x, tokens, k)
    want = np.empty((3, rows))
    wtop = np.empty((rows, k))
    for i in range(rows):
        z = x[i].astype(np.float64)
        z -= z.max()
        e = np.exp(z)
        ln = np.log(e.sum())
        want[:2, i] = z[tokens[i]] - ln, ln - (e @ z) / e.sum()
        wtop[i] = z[top[i]] - ln
    assert rel_l2(lp, want[0]) <= 1.4e-7
    assert rel_l2(ent, want[1]) <= 1.4e-7
    assert rel_l2(tlp, wtop) <= 1.4e-7
