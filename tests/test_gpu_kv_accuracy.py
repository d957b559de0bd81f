"""Attention over the quantized cache on data that is not unit normal: positions whose values dwarf the others', one key that holds
nearly all the weight, queries and keys with a mean, channels that set their block's scale, long sums of one sign.

Bounds. To BF16 a result is rounded by at most half a step, 2^-8 of the value; the 16-bit operands of a call of many rows are rounded
to 11 bits each (2^-12 of random sign on average: together below 1e-3 of the result), so relative L2 stays within 2^-8, whose root mean square over a binade is
1.7e-3. To F32 the library's bound for F32 accumulation holds, relative L2 1e-5."""
import numpy as np
import pytest

import kv_oracle
from nuclis_b200 import KvCache, encoding as enc
from parity import rel_l2
from test_gpu_kv_cache import Held, PAIRS, attend, backend, write  # noqa: F401

pytestmark = pytest.mark.gpu


def one_key_and_one_value(width, length, rows, dominant, large, ratio, seed):
    """q, k, v of one head: the key at `dominant` holds some 95 % of every row's weight, that at `large` next to none, whose values are
    `ratio` times the others'."""
    rng = np.random.default_rng(seed)
    u = rng.standard_normal(width)
    u /= np.linalg.norm(u)
    gain = np.sqrt((np.log(length) + 3.5) * np.sqrt(width))  # q . k / sqrt(width) of the two along u
    k, v, q = (rng.standard_normal((n, 1, width)) for n in (length, length, rows))
    k -= (k @ u)[..., None] * u
    q -= (q @ u)[..., None] * u
    q += gain * u
    k[dominant] += gain * u
    k[large] -= gain * u
    v *= 2.0 ** -6
    v[large] *= ratio
    return (x.astype(np.float32) for x in (q, k, v))


@pytest.mark.parametrize("ratio", [2 ** 7, 2 ** 10, 2 ** 12, 2 ** 20])
@pytest.mark.parametrize("venc", [enc.Q8_0, enc.Q4_0])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_large_values_ahead_of_those_that_count(backend, width, venc, ratio):
    """The probabilities of later steps keep their bits, whatever the values of an earlier one were."""
    b = backend
    length, rows = 4096, 140
    shape = KvCache(1, length, 1, width, enc.Q8_0, venc)
    q, k, v = one_key_and_one_value(width, length, rows, 3000, 100, ratio, 5)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, length)], length, k, v)
        want = kv_oracle.attention(q, kv_oracle.stored(k, enc.Q8_0), kv_oracle.stored(v, venc), length - rows, 1)
        spans = [(0, length - rows, rows)]
        assert rel_l2(attend(b, held, cache, shape, spans, rows, q, 1, dtype=enc.BF16), want) <= 2.0 ** -8
        assert rel_l2(attend(b, held, cache, shape, spans, rows, q, 1), want) <= 1e-5


@pytest.mark.parametrize("venc", [enc.Q8_0, enc.Q4_0])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_large_values_ahead_in_one_block_to_f32(backend, width, venc):
    """More units than blocks, so that one block (and of it the warp that has both positions) walks past the large values to those that count."""
    b = backend
    length, rows = 4096, 592
    shape = KvCache(1, length, 1, width, enc.Q8_0, venc)
    q, k, v = one_key_and_one_value(width, length, rows * 8, 2661, 101, 2 ** 20, 7)  # granules 166 and 6, 160 apart
    q = q.reshape(rows, 8, width)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, length)], length, k, v)
        got = attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, 8)
        k, v = kv_oracle.stored(k, enc.Q8_0), kv_oracle.stored(v, venc)
        for i in (0, 300, 591):
            assert rel_l2(got[i:i + 1], kv_oracle.attention(q[i:i + 1], k, v, length - rows + i, 8)) <= 1e-5, i


@pytest.mark.parametrize("ratio", [2 ** 7, 2 ** 12, 2 ** 16, 2 ** 20])
@pytest.mark.parametrize("kenc,venc", PAIRS)
@pytest.mark.parametrize("width", [64, 128, 256])
def test_large_values_beside_those_that_count(backend, width, kenc, venc, ratio):
    """The same with both positions in one step of either kernel: the values keep their bits beside larger ones. To F32 a position's product of
    probability and scale has its halves' end, 2^-36 of the largest value beside it, of random sign over the positions."""
    b = backend
    length, rows = 700, 140
    shape = KvCache(1, 704, 1, width, kenc, venc)
    q, k, v = one_key_and_one_value(width, length, rows, 129, 130, ratio, 6)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, length)], length, k, v)
        want = kv_oracle.attention(q, kv_oracle.stored(k, kenc), kv_oracle.stored(v, venc), length - rows, 1)
        spans = [(0, length - rows, rows)]
        assert rel_l2(attend(b, held, cache, shape, spans, rows, q, 1, dtype=enc.BF16), want) <= 2.0 ** -8
        got = attend(b, held, cache, shape, spans, rows, q, 1)
        lost = np.sqrt(length) * 2.0 ** -36 * np.abs(v).max() * np.sqrt(want.size)
        assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want) + lost


@pytest.mark.parametrize("venc", [enc.Q8_0, enc.Q4_0])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_steps_of_zeros_and_of_alternating_sizes(backend, width, venc):
    """Values that are zero for a while (a cache written in part), then tiny, then large, step by step: their exponent moves both ways.
    Row by row within half a step of BF16, and f16's end: a probability times 2^7 and the power of two of its step's values over the largest so far is
    rounded by at most 2^-25 where it is next to zero, so a position adds at most 2^-32 max|v|, of random sign, and the norm of a row's result
    is off by sqrt(length) x 2^-32 max|v| sqrt(width). It shows in the rows that look at a position of zeros: all they hold is the share of the others,
    whose probabilities are near e^-20."""
    b = backend
    length, rows = 2000, 140
    shape = KvCache(1, length, 1, width, enc.Q8_0, venc)
    rng = np.random.default_rng(9)
    k, v = (rng.standard_normal((length, 1, width)).astype(np.float32) for _ in range(2))
    v[:300] = 0
    step = np.arange(length) // 128
    v[300:] *= np.where(step % 3 == 0, 2.0 ** -8, np.where(step % 3 == 1, 1.0, 2.0 ** 6))[300:, None, None].astype(np.float32)
    v[900:1300] = 0
    q = rng.standard_normal((rows, 1, width)).astype(np.float32)
    q[::2] = 4 * k[rng.integers(300, 1800, rows // 2)]  # every other row looks at one position
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, length)], length, k, v)
        want = kv_oracle.attention(q, kv_oracle.stored(k, enc.Q8_0), kv_oracle.stored(v, venc), length - rows, 1)
        got = attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, 1, dtype=enc.BF16)
        assert np.all(np.isfinite(got))
        lost = np.sqrt(length) * 2.0 ** -32 * np.abs(v).max() * np.sqrt(width)
        assert np.all(np.linalg.norm(got - want, axis=-1) <= 2.0 ** -8 * np.linalg.norm(want, axis=-1) + lost)


@pytest.mark.parametrize("width", [64, 128, 256])
def test_queries_with_a_mean_and_keys_with_large_channels(backend, width):
    """What projections write: a channel in each block of the keys sets its scale, the other codes lie near zero, and a block's queries
    do not cancel. The scores are far smaller than what an offset of the codes would contribute."""
    b = backend
    length, rows, group = 4000, 3, 2
    shape = KvCache(1, length, 1, width, enc.Q8_0, enc.Q8_0)
    rng = np.random.default_rng(width)
    k, v = (rng.standard_normal((length, 1, width)) for _ in range(2))
    k *= 0.3
    k[..., 5::32] += 60
    q = rng.standard_normal((rows, group, width)) + 2
    q[..., 5::32] *= 0.02
    q, k, v = (x.astype(np.float32) for x in (q, k, v))
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, length)], length, k, v)
        want = kv_oracle.attention(q, kv_oracle.stored(k, enc.Q8_0), kv_oracle.stored(v, enc.Q8_0), length - rows, group)
        assert rel_l2(attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, group), want) <= 1e-5


@pytest.mark.parametrize("length", [24100, 100000])
@pytest.mark.parametrize("width,heads,group", [(256, 1, 8), (128, 2, 4), (64, 1, 8)])
def test_long_sums_of_whole_units(backend, width, heads, group, length):
    """More units than blocks over a long cache, to F32: a block sums all positions of a unit, and values of one sign make the sums grow."""
    b = backend
    rows = 592
    shape = KvCache(1, (length + 15) // 16 * 16, heads, width, enc.Q8_0, enc.Q4_0)
    rng = np.random.default_rng(length)
    k, v = (rng.standard_normal((length, heads, width), dtype=np.float32) for _ in range(2))
    v += 3
    q = rng.standard_normal((rows, heads * group, width), dtype=np.float32) * np.float32(0.3)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, length)], length, k, v)
        got = attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, heads * group)
        k, v = kv_oracle.stored(k, enc.Q8_0), kv_oracle.stored(v, enc.Q4_0)
        for i in (0, 301, 591):
            assert rel_l2(got[i:i + 1], kv_oracle.attention(q[i:i + 1], k, v, length - rows + i, group)) <= 1e-5, i


@pytest.mark.parametrize("width,length", [(32, 2000000), (96, 400001), (512, 60001)])
def test_long_sums_of_other_widths(backend, width, length):
    """A warp sums all positions of a row, whose values have one sign."""
    b = backend
    shape = KvCache(1, (length + 15) // 16 * 16, 1, width, enc.Q8_0, enc.Q4_0)
    rng = np.random.default_rng(width)
    k, v = (rng.standard_normal((length, 1, width), dtype=np.float32) for _ in range(2))
    v += 3
    q = rng.standard_normal((2, 2, width), dtype=np.float32) * np.float32(0.3)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        for at in range(0, length, 1 << 20):  # (what a call takes)
            n = min(1 << 20, length - at)
            write(b, held, cache, shape, [(0, at, n)], n, k[at:at + n], v[at:at + n])
        got = attend(b, held, cache, shape, [(0, length - 2, 2)], 2, q, 2)
        want = kv_oracle.attention(q, kv_oracle.stored(k, enc.Q8_0), kv_oracle.stored(v, enc.Q4_0), length - 2, 2)
        assert rel_l2(got, want) <= 1e-5


@pytest.mark.parametrize("venc", [enc.Q8_0, enc.Q4_0])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_long_sums_of_many_rows(backend, width, venc):
    """More units of the many-row kernel than blocks over 24 times the same 65,536 positions, values of one sign: a row counts a position as often as it sees it."""
    b = backend
    piece, times, rows = 65536, 24, 20000 if width == 256 else 40000
    length = piece * times
    shape = KvCache(1, length, 1, width, enc.Q8_0, venc)
    rng = np.random.default_rng(width)
    k, v = (rng.standard_normal((piece, 1, width), dtype=np.float32) for _ in range(2))
    v += 3
    q = rng.standard_normal((rows, 1, width), dtype=np.float32) * np.float32(0.3)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        for at in range(times):
            write(b, held, cache, shape, [(0, at * piece, piece)], piece, k, v)
        got = attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, 1, dtype=enc.BF16)
    k, v = kv_oracle.stored(k, enc.Q8_0)[:, 0], kv_oracle.stored(v, venc)[:, 0]
    for i in (0, rows // 2 + 1, rows - 1):
        weight = np.exp(k @ q[i, 0].astype(np.float64) / np.sqrt(width)) * ((length - rows + i - np.arange(piece)) // piece + 1)
        assert rel_l2(got[i, 0], weight @ v / weight.sum()) <= 2.0 ** -8, i


@pytest.mark.parametrize("rows,group,window", [(140, 1, 0), (20000, 2, 270000), (20000, 2, 0)])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_many_rows_over_a_long_cache(backend, width, rows, group, window):
    """Unit normal values, whose sums do not grow, so that a wrong share of any of them shows: units cut into parts, and whole ones under a window."""
    b = backend
    length = 400000
    shape = KvCache(1, length, 1, width, enc.Q8_0, enc.Q8_0)
    rng = np.random.default_rng(width)
    k, v = (rng.standard_normal((length, 1, width), dtype=np.float32) for _ in range(2))
    v[:200000] *= 2  # exponents and, with the keys' growth, maxima that move on the way
    k *= np.linspace(0.2, 1.5, length, dtype=np.float32)[:, None, None]
    q = rng.standard_normal((rows, group, width), dtype=np.float32)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, length)], length, k, v)
        got = attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, group, dtype=enc.BF16, window=window)
    k, v = kv_oracle.stored(k, enc.Q8_0), kv_oracle.stored(v, enc.Q8_0)
    for i in (0, rows // 2 + 1, rows - 1):
        want = kv_oracle.attention(q[i:i + 1], k, v, length - rows + i, group, window=window)
        assert rel_l2(got[i:i + 1], want) <= 2.0 ** -8, i
