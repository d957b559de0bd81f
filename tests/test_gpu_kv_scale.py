"""The ends of attention's scale: what the call takes gives the formula's result, the rest is refused."""
import numpy as np
import pytest

import kv_oracle
from nuclis_b200 import KvCache, NuclisError, encoding as enc, kv_spans
from parity import rel_l2
from test_gpu_kv_cache import Held, attend, backend, case  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width,rows,dtype", [(128, 2, 0), (96, 2, 0), (128, 140, enc.BF16), (256, 140, enc.BF16)])
def test_a_scale_near_the_end_of_f32(backend, width, rows, dtype):
    """Queries that take it back: scores of some units."""
    b = backend
    shape = KvCache(1, 208, 1, width, enc.Q8_0, enc.Q8_0)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [200], 3)
        scale = np.float32(2.0 ** 127)  # 1.7e38
        q = (rng.standard_normal((rows, 1, width)) * 0.1 * 2.0 ** -122).astype(np.float32)
        want = kv_oracle.attention(q.astype(np.float64) * float(scale), k[0], v[0], 200 - rows, 1, scale=1.0)
        got = attend(b, held, cache, shape, [(0, 200 - rows, rows)], rows, q, 1, dtype=dtype, scale=float(scale))
        # scores of some tens: their F32 rounding, 2^-24 of the score for each block, is that of the probability
        assert rel_l2(got, want) <= (1e-4 if dtype == 0 else 2.0 ** -8 + 1e-2)


def test_scales_that_are_refused(backend):
    b = backend
    shape = KvCache(1, 32, 1, 64)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [20], 4)
        q = rng.standard_normal((1, 1, 64)).astype(np.float32)
        sp, queries, out = held.up(kv_spans([(0, 19, 1)])), held.up(q), held.new(256)
        for scale in (0.0, 1e-60, 2.5e38, 3e38, float("inf"), -1.0):
            b.begin()
            with pytest.raises(NuclisError) as e:
                b.attention(cache, shape, sp, 1, 1, queries, 64, 1, out, 64, scale=scale)
            assert e.value.name == "InvalidShape", scale
            b.discard()
        b.begin()
        b.attention(cache, shape, sp, 1, 1, queries, 64, 1, out, 64, scale=1e-30)  # next to none: the values' mean
        b.commit()
        assert rel_l2(out.floats(), v[0, :20, 0].mean(0)) <= 1e-5
