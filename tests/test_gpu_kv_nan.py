"""A block of values that was stored from a NaN reaches every row that sees its position, however little weight the row has there."""
import numpy as np
import pytest

import kv_oracle
from nuclis_b200 import KvCache, encoding as enc
from parity import rel_l2
from test_gpu_kv_cache import Held, attend, backend, write  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("venc", [enc.Q8_0, enc.Q4_0])
@pytest.mark.parametrize("width", [64, 128, 256, 96])
@pytest.mark.parametrize("at,window", [(30, 0), (200, 0), (300, 150), (399, 0)])
def test_a_nan_of_next_to_no_weight(backend, width, venc, at, window):
    b = backend
    length, rows = 400, 140
    shape = KvCache(1, length, 1, width, enc.Q8_0, venc)
    rng = np.random.default_rng(at)
    u = rng.standard_normal(width)
    u /= np.linalg.norm(u)
    q, k, v = (rng.standard_normal((n, 1, width)) for n in (rows, length, length))
    # the key at `at` lies 40 nats below the others, those of its step among them
    q -= (q @ u)[..., None] * u
    q += np.sqrt(40 * np.sqrt(width)) * u
    k[at] -= np.sqrt(40 * np.sqrt(width)) * u
    q, k, v = (x.astype(np.float32) for x in (q, k, v))
    v[at, 0, 33] = np.nan
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, length)], length, k, v)
        clean = kv_oracle.stored(v, venc)
        clean[at, 0, 32:64] = 0
        want = kv_oracle.attention(q, kv_oracle.stored(k, enc.Q8_0), clean, length - rows, 1, window=window)
        pos = length - rows + np.arange(rows)
        sees = (pos >= at) & ((pos < at + window) if window else True)
        for dtype, bound in ((0, 1e-5), (enc.BF16, 2.0 ** -8)):
            got = attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, 1, window=window, dtype=dtype)
            bad = np.zeros(got.shape, bool)
            bad[sees, :, 32:64] = True
            assert np.all(np.isnan(got[bad])) and np.all(np.isfinite(got[~bad]))
            assert rel_l2(got[~bad], want[~bad]) <= bound


@pytest.mark.parametrize("venc", [enc.Q8_0, enc.Q4_0])
@pytest.mark.parametrize("width", [64, 128, 256, 96])
@pytest.mark.parametrize("at,window", [(30, 0), (270, 0), (390, 0), (399, 0), (254, 150)])
def test_a_nan_of_a_weight_that_f32_ends_above(backend, width, venc, at, window):
    """The key at `at` lies 120 nats below the others: its weight is zero in F32, in steps that all rows see as in those that some do."""
    b = backend
    length, rows = 400, 140
    shape = KvCache(1, length, 1, width, enc.Q8_0, venc)
    rng = np.random.default_rng(at)
    u = rng.standard_normal(width)
    u /= np.linalg.norm(u)
    q, k, v = (rng.standard_normal((n, 1, width)) for n in (rows, length, length))
    gain = np.sqrt(120 * np.sqrt(width))
    q += (gain - q @ u)[..., None] * u
    k -= (k @ u)[..., None] * u
    k[at] -= gain * u
    q, k, v = (x.astype(np.float32) for x in (q, k, v))
    v[at, 0, 33] = np.nan
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, length)], length, k, v)
        clean = kv_oracle.stored(v, venc)
        clean[at, 0, 32:64] = 0
        want = kv_oracle.attention(q, kv_oracle.stored(k, enc.Q8_0), clean, length - rows, 1, window=window)
        pos = length - rows + np.arange(rows)
        sees = (pos >= at) & ((pos < at + window) if window else True)
        assert at < length - rows or 0 < sees.sum() < rows
        for dtype, bound in ((0, 1e-5), (enc.BF16, 2.0 ** -8)):
            got = attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, 1, window=window, dtype=dtype)
            bad = np.zeros(got.shape, bool)
            bad[sees, :, 32:64] = True
            assert np.all(np.isnan(got[bad])) and np.all(np.isfinite(got[~bad]))
            assert rel_l2(got[~bad], want[~bad]) <= bound
