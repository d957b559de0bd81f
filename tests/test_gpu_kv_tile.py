"""The kernel for many rows to BF16, from the fewest query rows a key/value head that it takes (128) on. That it is the one that runs shows in its 16-bit
operands: some of its results are not those of the F32 form rounded."""
import threading

import numpy as np
import pytest

import kv_oracle
from nuclis_b200 import Backend, KvCache, encoding as enc
from parity import rel_l2
from test_gpu_kv_cache import Held, PAIRS, attend, backend, case  # noqa: F401

pytestmark = pytest.mark.gpu


def rounded(x):
    """F32 to BF16 and back, to nearest even."""
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7fff + (b >> 16 & 1)) >> 16 << 16).astype(np.uint32).view(np.float32).reshape(x.shape)


# width, group, rows, length (after the rows): one tile that is half full, just full, a row over
FEWEST = [(128, 1, 128, 128), (128, 5, 26, 26), (128, 1, 256, 256), (128, 1, 257, 300), (64, 1, 128, 500), (64, 8, 16, 129), (256, 4, 32, 32), (256, 1, 128, 1000), (256, 1, 129, 129)]


@pytest.mark.parametrize("width,group,rows,length", FEWEST)
@pytest.mark.parametrize("kenc,venc", PAIRS)
def test_the_fewest_rows(backend, kenc, venc, width, group, rows, length):
    b = backend
    heads = 2
    shape = KvCache(2, (length + 15) // 16 * 16, heads, width, kenc, venc)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [5, length], length + width + rows)
        q = rng.standard_normal((rows, heads * group, width)) * 1.5
        spans = [(1, length - rows, rows)]
        want = kv_oracle.attention(q.astype(np.float32), k[1], v[1], length - rows, group)
        got = attend(b, held, cache, shape, spans, rows, q, heads * group, dtype=enc.BF16)
        assert rel_l2(got, want) <= 2.0 ** -8
        assert np.any(got != rounded(attend(b, held, cache, shape, spans, rows, q, heads * group)))
        np.testing.assert_array_equal(got, attend(b, held, cache, shape, spans, rows, q, heads * group, pad=3, dtype=enc.BF16))


@pytest.mark.parametrize("width", [64, 128, 256])
def test_two_handles_with_many_rows_at_once(backend, width):
    """A handle a thread, each with its own stream and scratch, both with parts to join: the results are those of one alone."""
    shape = KvCache(1, 4096, 2, width, enc.Q8_0, enc.Q4_0)

    def work(b, seed, turns, results):
        with Held(b) as held:
            cache, k, v, rng = case(b, held, shape, [3000], seed)
            q = rng.standard_normal((80, 4, width)).astype(np.float32)
            for _ in range(turns):
                results.append(attend(b, held, cache, shape, [(0, 2920, 80)], 80, q, 4, dtype=enc.BF16))
            want = kv_oracle.attention(q, k[0], v[0], 2920, 2)
            assert rel_l2(results[0], want) <= 2.0 ** -8
            results.append("fine")

    other = Backend(0)
    try:
        results = [[], []]
        threads = [threading.Thread(target=work, args=(b, 40 + i, 20, results[i])) for i, b in enumerate((backend, other))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for r in results:
            assert len(r) == 21 and r[20] == "fine"
            for x in r[1:20]:
                np.testing.assert_array_equal(x, r[0])
    finally:
        other.deinit()
