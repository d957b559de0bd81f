"""The cache's Q8_0 blocks against the format's own rule, d = amax / 127 divided exactly and code = round(x / d): the library multiplies by the
F32 reciprocals instead.

What that may change, before any rounding to fewer bits: fl(1 / 127) is off by at most 2^-24 of itself and the product rounds once more, so d is within
2^-23 (1 + 2^-24) of the quotient. In f16 that is the same number or, where a border lies between, the next one: a step, at most 2^-10. 1 / d and the
product with x round once each (2^-24): x / d <= 127 is within 127 x 2^-22 of the exact one, so a code is off the exact quotient by no more than half and that."""
import numpy as np
import pytest

from nuclis_b200 import KvCache, encoding as enc
from test_gpu_kv_cache import Held, backend, read, write  # noqa: F401

pytestmark = pytest.mark.gpu


def test_blocks_beside_the_exact_division(backend):
    b = backend
    rows, heads, width = 2048, 4, 128
    shape = KvCache(1, rows, heads, width, enc.Q8_0, enc.Q8_0)
    rng = np.random.default_rng(127)
    k, v = (rng.standard_normal((rows, heads, width)).astype(np.float32) * np.float32(s) for s in (1.0, 0.05))
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, rows)], rows, k, v)
        for got, x in zip(read(b, held, cache, shape, [(0, 0, rows)], rows), (k, v)):
            got, x = (a.astype(np.float64).reshape(-1, 32) for a in (got, x))
            d = np.abs(x).max(1) / 127
            scale = np.abs(got).max(1) / 127  # the largest of a block has code 127
            assert np.all(scale == scale.astype(np.float16))
            exact = d.astype(np.float16).astype(np.float64)
            assert np.all(np.abs(scale - exact) <= 2.0 ** -10 * exact)
            assert np.mean(scale != exact) <= 2.0 ** -23 / 2.0 ** -11 * 8  # the share of quotients that lie so near a border, eight times over
            codes = got / scale[:, None]
            assert np.all(codes == np.round(codes))
            assert np.all(np.abs(codes - x / d[:, None]) <= 0.5 + 127 * 2.0 ** -22)
