"""The quantized key/value cache: rows written and read back (exactly what the rule of a block gives), and the causal
grouped-query attention over it against 64 bits.

Bounds. A read is d * code, both exact in F32: equal to the last bit; BF16 is that, rounded once. Attention to F32 is held to the
library's bound for F32 accumulation, relative L2 1e-5: the query and the probabilities keep 22 bits (2^-23 each), a
score of width/32 blocks has that many F32 roundings on terms of its own size (8 x 2^-24 of sum |q k| scale, about 10 for unit
normal rows of 256: 5e-6 of a probability at worst, and of random sign), and a sum over n positions on the tensor cores truncates
once per 16 positions and warp (n / 128 x 2^-23: below 1e-6 for the lengths here). To BF16 the rounding comes on top: half a step, 2^-8 of
the value."""
import threading

import numpy as np
import pytest

import kv_oracle
from nuclis_b200 import Backend, KvCache, NuclisError, encoding as enc, kv_spans
from parity import rel_l2

pytestmark = pytest.mark.gpu

PAIRS = [(enc.Q8_0, enc.Q8_0), (enc.Q4_0, enc.Q4_0), (enc.Q8_0, enc.Q4_0), (enc.Q4_0, enc.Q8_0)]


@pytest.fixture(scope="module")
def backend():
    b = Backend(0)
    yield b
    b.deinit()


class Held:
    """Buffers of one test, released at its end."""

    def __init__(self, b):
        self.b, self.all = b, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for x in self.all:
            self.b.release(x)

    def new(self, size):
        self.all.append(self.b.create(size))
        return self.all[-1]

    def up(self, data):
        data = np.ascontiguousarray(data)
        buf = self.new(data.nbytes)
        buf.write(data)
        return buf


def bf16(buf, shape):
    return (buf.read(np.uint16).astype(np.uint32) << 16).view(np.float32).reshape(shape)


def write(b, held, cache, shape, spans, rows, keys, values):
    """keys, values: [sequences * rows][heads][width]."""
    n = shape.heads * shape.width
    fused = np.concatenate([keys.reshape(-1, n), values.reshape(-1, n)], 1).astype(np.float32)
    buf = held.up(fused)
    sp = held.up(kv_spans(spans))
    b.begin()
    b.kv_write(cache, shape, sp, len(spans), rows, buf, 2 * n, buf.slice(n * 4, buf.len - n * 4), 2 * n)
    b.commit()


def read(b, held, cache, shape, spans, rows, dtype=0):
    n = shape.heads * shape.width
    size = 4 if dtype == 0 else 2
    out = held.new(len(spans) * rows * 2 * n * size)  # keys and values of a row side by side
    sp = held.up(kv_spans(spans))
    b.begin()
    b.kv_read(cache, shape, sp, len(spans), rows, out, 2 * n, out.slice(n * size, out.len - n * size), 2 * n, out_dtype=dtype)
    b.commit()
    x = out.floats().reshape(-1, 2, shape.heads, shape.width) if dtype == 0 else bf16(out, (-1, 2, shape.heads, shape.width))
    return x[:, 0], x[:, 1]


def attend(b, held, cache, shape, spans, rows, q, heads, dtype=0, pad=0, **kw):
    n = heads * shape.width
    qb = held.up(np.concatenate([q.reshape(-1, n).astype(np.float32), np.full((q.shape[0], pad), np.nan, np.float32)], 1) if pad else q.astype(np.float32))
    size = 4 if dtype == 0 else 2
    out = held.up(np.full(len(spans) * rows * n * size, 0xc1, np.uint8))
    sp = held.up(kv_spans(spans))
    b.begin()
    b.attention(cache, shape, sp, len(spans), rows, qb, n + pad, heads, out, n, out_dtype=dtype, **kw)
    b.commit()
    return out.floats().reshape(-1, heads, shape.width) if dtype == 0 else bf16(out, (-1, heads, shape.width))


UNTOUCHED = np.full(4, 0xc1, np.uint8).view(np.float32)[0]


@pytest.mark.parametrize("width,heads", [(32, 1), (64, 3), (96, 2), (128, 8), (160, 1), (256, 4), (512, 2)])
@pytest.mark.parametrize("kenc,venc", PAIRS)
def test_rows_come_back_as_the_rule_gives_them(backend, kenc, venc, width, heads):
    b = backend
    shape = KvCache(3, 48, heads, width, kenc, venc)
    rng = np.random.default_rng(width + heads)
    rows = 21
    k, v = (rng.standard_normal((2 * rows, heads, width)).astype(np.float32) * np.float32(s) for s in (3.0, 0.02))
    with Held(b) as held:
        cache = held.new(shape.bytes)
        spans = [(2, 5, rows), (0, 27, rows - 4)]
        write(b, held, cache, shape, spans, rows, k, v)
        gk, gv = read(b, held, cache, shape, [(2, 5, rows), (0, 27, rows)], rows)
        live = np.r_[0:rows, rows:2 * rows - 4]
        for got, x, e in ((gk, k, kenc), (gv, v, venc)):
            np.testing.assert_array_equal(got[live].astype(np.float64), kv_oracle.stored(x[live], e))
            assert np.all(got[2 * rows - 4:] == 0)  # padding rows were not written
        others = read(b, held, cache, shape, [(1, 0, 48), (2, 0, 5), (2, 26, 22), (0, 0, 27)], 48)
        for x in others:
            x = x.reshape(4, 48, heads, width)
            assert np.all(x[0] == 0) and np.all(x[1, :5] == 0) and np.all(x[2, :22] == 0) and np.all(x[3, :27] == 0)
        hk, hv = read(b, held, cache, shape, spans, rows, dtype=enc.BF16)
        for got, x, e in ((hk, k, kenc), (hv, v, venc)):
            want = kv_oracle.stored(x[:rows], e)
            assert np.all(np.abs(got[:rows] - want) <= 2.0 ** -8 * np.abs(want))


@pytest.mark.parametrize("encoding", [enc.Q8_0, enc.Q4_0])
def test_blocks_at_the_ends_of_the_scale(backend, encoding):
    """Zeros, equal magnitudes of both signs, scales that vanish in f16 or pass its range, NaN and infinity."""
    b = backend
    shape = KvCache(1, 16, 1, 256, encoding, encoding)
    x = np.zeros((16, 1, 256), np.float32)
    rng = np.random.default_rng(3)
    x[1] = rng.standard_normal(256) * 1e-7       # scales near f16's smallest
    x[2] = rng.standard_normal(256) * 1e-9       # scales that round to zero
    x[3] = rng.standard_normal(256) * 1e6
    x[4] = rng.standard_normal(256) * 1e9        # scales beyond f16
    x[5] = np.tile([1.0, -1.0], 128)             # the first of equals decides Q4_0's sign
    x[6] = np.tile([-2.5, 2.5], 128)
    x[7] = np.arange(256) - 128                  # halves of a code
    x[8, 0, 40] = np.nan
    x[8, 0, 70] = 1.0
    x[9, 0, 130] = np.inf
    x[10, 0, 200] = -np.inf
    x[11] = np.finfo(np.float32).max
    x[12] = np.finfo(np.float32).tiny / 4
    x[13] = rng.standard_normal(256)
    x[13, 0, 255] = 60.0
    x[14] = -x[13]
    x[15] = np.repeat(rng.standard_normal(8), 32)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, 16)], 16, x, x[::-1])
        for got, want in zip(read(b, held, cache, shape, [(0, 0, 16)], 16), (x, x[::-1])):
            np.testing.assert_array_equal(got.astype(np.float64), kv_oracle.stored(want, encoding))


def test_the_later_of_two_spans_keeps_a_position(backend):
    b = backend
    shape = KvCache(2, 64, 2, 64, enc.Q8_0, enc.Q4_0)
    rng = np.random.default_rng(8)
    k, v = (rng.standard_normal((3 * 40, 2, 64)).astype(np.float32) for _ in range(2))
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, 40), (0, 10, 40), (0, 10, 3)], 40, k, v)
        got = read(b, held, cache, shape, [(0, 0, 50)], 50)
        at = np.r_[0:10, 80:83, 43:80]
        for g, x, e in zip(got, (k, v), (enc.Q8_0, enc.Q4_0)):
            np.testing.assert_array_equal(g.astype(np.float64), kv_oracle.stored(x[at], e))


def test_unaligned_rows_and_strides(backend):
    b = backend
    shape = KvCache(1, 32, 3, 64, enc.Q4_0, enc.Q8_0)
    rng = np.random.default_rng(9)
    n, rows, stride = 192, 7, 2 * 192 + 5
    x = rng.standard_normal(rows * stride + 1).astype(np.float32)
    with Held(b) as held:
        cache, sp = held.new(shape.bytes), held.up(kv_spans([(0, 3, rows)]))
        rowsb, out = held.up(x), held.new(x.nbytes)
        b.begin()
        b.kv_write(cache, shape, sp, 1, rows, rowsb.slice(4, rowsb.len - 4), stride, rowsb.slice(4 + 4 * (n + 2), rowsb.len - 4 - 4 * (n + 2)), stride)
        b.kv_read(cache, shape, sp, 1, rows, out.slice(4, out.len - 4), stride, out.slice(4 + 4 * (n + 2), out.len - 4 - 4 * (n + 2)), stride)
        b.commit()
        got, want = out.floats()[1:].reshape(rows, stride), x[1:].reshape(rows, stride)
        np.testing.assert_array_equal(got[:, :n].astype(np.float64), kv_oracle.stored(want[:, :n], enc.Q4_0))
        np.testing.assert_array_equal(got[:, n + 2:2 * n + 2].astype(np.float64), kv_oracle.stored(want[:, n + 2:2 * n + 2], enc.Q8_0))
        assert np.all(got[:, n:n + 2] == 0) and np.all(got[:, 2 * n + 2:] == 0)


def case(b, held, shape, lengths, seed, gain=1.0):
    """A cache with `lengths[s]` written positions in slot s; what it holds, in 64 bits, per slot."""
    rng = np.random.default_rng(seed)
    cache = held.new(shape.bytes)
    most = max(lengths)
    k, v = (rng.standard_normal((len(lengths), most, shape.heads, shape.width)).astype(np.float32) for _ in range(2))
    v *= np.float32(gain)
    write(b, held, cache, shape, [(s, 0, n) for s, n in enumerate(lengths)], most, k.reshape(-1, shape.heads, shape.width), v.reshape(-1, shape.heads, shape.width))
    return cache, kv_oracle.stored(k, shape.key_encoding), kv_oracle.stored(v, shape.value_encoding), rng


# width, group, rows, length (after the rows), window
SHAPES = [(128, 5, 1, 1, 0), (128, 5, 1, 2, 0), (128, 1, 1, 16, 0), (128, 8, 1, 17, 0), (128, 5, 1, 700, 0), (128, 5, 1, 4099, 0), (128, 3, 6, 333, 0),
          (128, 5, 8, 129, 100), (64, 3, 1, 1000, 0), (64, 16, 3, 257, 31), (64, 1, 40, 40, 0), (256, 5, 1, 515, 0), (256, 4, 5, 900, 0), (256, 10, 2, 77, 1),
          (96, 2, 3, 70, 0), (32, 4, 1, 65, 20), (512, 2, 2, 50, 0), (128, 5, 70, 300, 64), (256, 2, 100, 100, 0)]


@pytest.mark.parametrize("width,group,rows,length,window", SHAPES)
@pytest.mark.parametrize("kenc,venc", PAIRS)
def test_attention_against_64_bits(backend, kenc, venc, width, group, rows, length, window):
    b = backend
    heads = 2
    shape = KvCache(2, (length + 15) // 16 * 16 + 16, heads, width, kenc, venc)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [3, length], length + width)
        q = rng.standard_normal((rows, heads * group, width)) * 1.5
        spans = [(1, length - rows, rows)]
        want = kv_oracle.attention(q.astype(np.float32), k[1], v[1], length - rows, group, window=window)
        got = attend(b, held, cache, shape, spans, rows, q, heads * group, window=window)
        assert rel_l2(got, want) <= 1e-5
        again = attend(b, held, cache, shape, spans, rows, q, heads * group, window=window, pad=3)
        np.testing.assert_array_equal(got, again)  # the same from run to run, whatever the rows' alignment
        half = attend(b, held, cache, shape, spans, rows, q, heads * group, window=window, dtype=enc.BF16)
        assert rel_l2(half, want) <= 2.0 ** -8
        b.generic_only = True
        try:
            plain = attend(b, held, cache, shape, spans, rows, q, heads * group, window=window)
        finally:
            b.generic_only = False
        assert rel_l2(plain, want) <= 1e-5


# many rows to BF16: the tensor-core kernel's tiles of 256 rows (128 at width 256) and steps of 128 keys (64)
PROMPTS = [(128, 1, 64, 64, 0), (128, 5, 13, 13, 0), (128, 5, 60, 300, 0), (128, 8, 33, 1000, 0), (128, 1, 300, 300, 0), (128, 2, 200, 777, 130), (64, 1, 70, 500, 0),
           (64, 4, 100, 129, 0), (64, 16, 20, 2000, 5), (256, 4, 16, 16, 0), (256, 5, 50, 700, 0), (256, 1, 200, 260, 64), (256, 3, 129, 400, 0)]


@pytest.mark.parametrize("width,group,rows,length,window", PROMPTS)
@pytest.mark.parametrize("kenc,venc", PAIRS)
def test_many_rows_to_bf16(backend, kenc, venc, width, group, rows, length, window):
    """16-bit operands: q, k, v and p are rounded to 11 bits once each (2^-11 of a term at most, 4 x 2^-12 / sqrt(3) of random sign: 6e-4 of the
    result and less), the result to BF16's 8 (2^-8 at most): relative L2 within one half step, 2^-8."""
    b = backend
    heads = 2
    shape = KvCache(2, (length + 15) // 16 * 16, heads, width, kenc, venc)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [5, length], length + width + rows)
        q = rng.standard_normal((rows, heads * group, width)) * 1.5
        spans = [(1, length - rows, rows)]
        want = kv_oracle.attention(q.astype(np.float32), k[1], v[1], length - rows, group, window=window)
        got = attend(b, held, cache, shape, spans, rows, q, heads * group, window=window, dtype=enc.BF16)
        assert rel_l2(got, want) <= 2.0 ** -8
        np.testing.assert_array_equal(got, attend(b, held, cache, shape, spans, rows, q, heads * group, window=window, pad=3, dtype=enc.BF16))


@pytest.mark.parametrize("width", [64, 128, 256])
def test_many_rows_of_a_batch_to_bf16(backend, width):
    b = backend
    group, rows = 3, 90
    lengths = [90, 91, 300, 1, 650, 40]
    shape = KvCache(len(lengths), 656, 2, width, enc.Q8_0, enc.Q4_0)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, lengths, 78)
        q = rng.standard_normal((len(lengths) * rows, 2 * group, width)).astype(np.float32)
        spans = [(0, 0, 90), (1, 1, 90), (2, 230, 70), (3, 0, 1), (4, 0, 0), (4, 600, 50)]
        for window in (0, 33):
            got = attend(b, held, cache, shape, spans, rows, q, 2 * group, window=window, dtype=enc.BF16).reshape(len(spans), rows, 2 * group, width)
            for s, (slot, first, count) in enumerate(spans):
                if count:
                    want = kv_oracle.attention(q[s * rows: s * rows + count], k[slot], v[slot], first, group, window=window)
                    assert rel_l2(got[s, :count], want) <= 2.0 ** -8, s
                assert np.all(got[s, count:].view(np.uint32) == 0xc1c10000), s  # padding rows are left as they were


@pytest.mark.parametrize("kenc,venc", PAIRS[:2])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_many_rows_beside_values_they_do_not_see(backend, width, kenc, venc):
    """NaN and huge values ahead of a window and behind the last position, a NaN that some rows of the call see, queries of all sizes."""
    b = backend
    group, rows, length, window = 2, 100, 400, 200
    shape = KvCache(1, 480, 1, width, kenc, venc)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [length], 15)
        bad = np.full((60, 1, width), np.nan, np.float32)
        huge = np.full((60, 1, width), 3e38, np.float32)
        write(b, held, cache, shape, [(0, length, 40)], 60, bad, bad)
        write(b, held, cache, shape, [(0, length + 40, 10)], 60, huge, huge)
        write(b, held, cache, shape, [(0, 0, 55)], 60, bad, huge)
        q = (rng.standard_normal((rows, group, width)) * np.array([1e-30, 2.0])[:, None]).astype(np.float32)
        q[7, 0] = 0
        spans = [(0, length - rows, rows)]
        want = kv_oracle.attention(q, k[0], v[0], length - rows, group, window=window)
        got = attend(b, held, cache, shape, spans, rows, q, group, window=window, dtype=enc.BF16)
        assert rel_l2(got[:, 0], want[:, 0]) <= 2.0 ** -8 and rel_l2(got[:, 1], want[:, 1]) <= 2.0 ** -8
        # position 350 (row 50): NaN keys for every row that sees it
        write(b, held, cache, shape, [(0, 350, 1)], 1, bad[:1], v[0, 350:351].astype(np.float32))
        got = attend(b, held, cache, shape, spans, rows, q, group, window=window, dtype=enc.BF16)
        assert rel_l2(got[:50], want[:50]) <= 2.0 ** -8 and np.all(np.isnan(got[50:]))
        # a NaN block of its values: those dimensions of the rows that see it
        one = v[0, 350:351].astype(np.float32)
        one[0, 0, 40] = np.nan
        write(b, held, cache, shape, [(0, 350, 1)], 1, k[0, 350:351].astype(np.float32), one)
        got = attend(b, held, cache, shape, spans, rows, q, group, window=window, dtype=enc.BF16)
        assert rel_l2(got[:50], want[:50]) <= 2.0 ** -8
        assert np.all(np.isnan(got[50:, :, 32:64])) and np.all(np.isfinite(np.delete(got[50:], np.s_[32:64], 2)))
        # a NaN query stays in its row
        q[3, 1, 5] = np.nan
        got = attend(b, held, cache, shape, spans, rows, q, group, window=window, dtype=enc.BF16)
        assert np.all(np.isnan(got[3, 1])) and np.all(np.isfinite(got[3, 0])) and rel_l2(got[10:50], want[10:50]) <= 2.0 ** -8


@pytest.mark.parametrize("gain", [1e-6, 1e4])
@pytest.mark.parametrize("venc", [enc.Q8_0, enc.Q4_0])
def test_many_rows_and_values_of_all_sizes(backend, gain, venc):
    """Scales that rise and fall by orders of magnitude along the sequence, beyond what f16 holds of the values themselves."""
    b = backend
    shape = KvCache(1, 912, 1, 128, enc.Q4_0, venc)
    rng = np.random.default_rng(12)
    k, v = (rng.standard_normal((900, 1, 128)).astype(np.float32) for _ in range(2))
    v *= np.exp(rng.uniform(-3, 3, (900, 1, 1))).astype(np.float32) * np.float32(gain)
    k *= np.float32(gain)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, 900)], 900, k, v)
        q = (rng.standard_normal((150, 2, 128)) / gain).astype(np.float32)
        sk, sv = kv_oracle.stored(k, enc.Q4_0), kv_oracle.stored(v, venc)
        want = kv_oracle.attention(q, sk, sv, 750, 2)
        assert rel_l2(attend(b, held, cache, shape, [(0, 750, 150)], 150, q, 2, dtype=enc.BF16), want) <= 2.0 ** -8


@pytest.mark.parametrize("width", [64, 128, 256, 96])
def test_a_batch_of_unlike_sequences(backend, width):
    """Lengths from one position to many, an absent sequence, padding rows, two sequences on one slot."""
    b = backend
    group, rows = 5, 3
    lengths = [1, 2, 15, 16, 17, 500, 33, 1300]
    shape = KvCache(len(lengths), 1312, 2, width, enc.Q8_0, enc.Q4_0)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, lengths, 77)
        q = rng.standard_normal((len(lengths) * rows, 2 * group, width)).astype(np.float32)
        spans = [(0, 0, 1), (1, 0, 2), (2, 12, 3), (7, 1297, 3), (4, 0, 0), (5, 498, 2), (5, 200, 3), (7, 5, 1)]
        for window in (0, 10):
            got = attend(b, held, cache, shape, spans, rows, q, 2 * group, window=window).reshape(len(spans), rows, 2 * group, width)
            for s, (slot, first, count) in enumerate(spans):
                if count:
                    want = kv_oracle.attention(q[s * rows: s * rows + count], k[slot], v[slot], first, group, window=window)
                    assert rel_l2(got[s, :count], want) <= 1e-5, s
                assert np.all(got[s, count:].view(np.uint32) == UNTOUCHED.view(np.uint32)), s  # padding rows are left as they were


@pytest.mark.parametrize("pad,at", [(1, 0), (24, 1), (8, 8)])
@pytest.mark.parametrize("dtype,length,rows", [(0, 500, 3), (0, 9000, 1), (enc.BF16, 500, 3), (enc.BF16, 300, 90), (enc.BF16, 9000, 70)])
@pytest.mark.parametrize("width", [64, 128, 256, 96])
def test_output_rows_apart(backend, width, dtype, length, rows, pad, at):
    """A stride beyond the row, and rows that start anywhere: the same values, and nothing between or around them is written."""
    b = backend
    heads, size = 4, 4 if dtype == 0 else 2
    n = heads * width
    shape = KvCache(1, 9008, 2, width, enc.Q8_0, enc.Q8_0)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [length], 60)
        q = rng.standard_normal((rows, heads, width)).astype(np.float32)
        spans = [(0, length - rows, rows)]
        plain = attend(b, held, cache, shape, spans, rows, q, heads, dtype=dtype)
        word = np.uint32 if dtype == 0 else np.uint16
        out = held.up(np.full((rows + 1) * (n + pad) + at, 0xc1c1, word))
        qb, sp = held.up(q), held.up(kv_spans(spans))
        b.begin()
        b.attention(cache, shape, sp, 1, rows, qb, n, heads, out.slice(at * size, out.len - at * size), n + pad, out_dtype=dtype)
        b.commit()
        got = out.read(word)
        assert np.all(got[:at] == 0xc1c1) and np.all(got[at + rows * (n + pad):] == 0xc1c1)
        got = got[at: at + rows * (n + pad)].reshape(rows, n + pad)
        assert np.all(got[:, n:] == 0xc1c1)
        bits = plain.view(np.uint32) if dtype == 0 else (plain.view(np.uint32) >> 16).astype(np.uint16)
        np.testing.assert_array_equal(got[:, :n], bits.reshape(rows, n))


@pytest.mark.parametrize("count,rows,dtype", [(300, 2, 0), (45, 64, enc.BF16), (150, 9, 0)])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_many_sequences(backend, width, count, rows, dtype):
    """More sequences than a warp has lanes, a third of them absent, their lengths from one position to hundreds, on slots in no order."""
    b = backend
    group = 2
    rng = np.random.default_rng(count + width)
    lengths = rng.integers(1, 40000 // count, count)
    shape = KvCache(count, (40000 // count + 15) // 16 * 16, 2, width, enc.Q4_0, enc.Q8_0)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [int(n) for n in lengths], 50)
        q = rng.standard_normal((count * rows, 2 * group, width)).astype(np.float32)
        spans = []
        for slot in rng.permutation(count):
            n = int(min(rng.integers(1, rows + 1), lengths[slot]))
            spans.append((int(slot), int(lengths[slot]) - n, 0 if slot % 3 == 0 else n))
        got = attend(b, held, cache, shape, spans, rows, q, 2 * group, dtype=dtype).reshape(count, rows, 2 * group, width)
        untouched = UNTOUCHED.view(np.uint32) if dtype == 0 else 0xc1c10000
        for s, (slot, first, n) in enumerate(spans):
            if n:
                want = kv_oracle.attention(q[s * rows: s * rows + n], k[slot], v[slot], first, group)
                assert rel_l2(got[s, :n], want) <= (1e-5 if dtype == 0 else 2.0 ** -8), s
            assert np.all(got[s, n:].view(np.uint32) == untouched), s


@pytest.mark.parametrize("kenc,venc", PAIRS[:2])
@pytest.mark.parametrize("width", [64, 128, 256, 160])
def test_what_a_row_does_not_see_may_hold_anything(backend, width, kenc, venc):
    """NaN and huge values behind the last position, ahead of the window, and between the rows of a call."""
    b = backend
    group, rows, length, window = 3, 4, 150, 40
    shape = KvCache(1, 208, 1, width, kenc, venc)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [length], 5)
        bad = np.full((60, 1, width), np.nan, np.float32)
        huge = np.full((60, 1, width), 3e38, np.float32)
        write(b, held, cache, shape, [(0, length, 40)], 60, bad, bad)
        write(b, held, cache, shape, [(0, length + 40, 10)], 60, huge, huge)
        write(b, held, cache, shape, [(0, 0, 55)], 60, bad, huge)
        q = rng.standard_normal((rows, group, width)).astype(np.float32)
        got = attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, group, window=window)
        want = kv_oracle.attention(q, k[0], v[0], length - rows, group, window=window)
        assert rel_l2(got, want) <= 1e-5
        # a NaN that only the last row sees stays with it
        write(b, held, cache, shape, [(0, length - 1, 1)], 1, bad[:1], bad[:1])
        got = attend(b, held, cache, shape, [(0, length - rows, rows)], rows, q, group, window=window)
        assert rel_l2(got[:-1], want[:-1]) <= 1e-5 and np.all(np.isnan(got[-1]))


@pytest.mark.parametrize("gain", [1e-6, 1e-3, 1e4])
@pytest.mark.parametrize("encoding", [enc.Q8_0, enc.Q4_0])
def test_values_and_queries_of_all_sizes(backend, gain, encoding):
    b = backend
    shape = KvCache(1, 304, 2, 128, encoding, encoding)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [300], 6, gain)
        q = (rng.standard_normal((2, 4, 128)) * np.array([1e-30, 1e-3, 1.0, 30.0])[:, None]).astype(np.float32)
        want = kv_oracle.attention(q, k[0], v[0], 298, 2)
        got = attend(b, held, cache, shape, [(0, 298, 2)], 2, q, 4)
        # scores of some hundred (the last head): their F32 rounding, 2^-24 of the score for each of the 4 blocks, is that of the probability.
        # The split of x = p d bias into f16 halves has an absolute end as well: lo = x - hi is rounded to a multiple of 2^-24 at its smallest,
        # half a step of which is 2^-25. The largest scale seen has bias dmax >= 2^11, so that is at most 2^-36 dmax of p d and, the largest
        # code of a block times its scale being its largest value, 2^-36 max|v| a position of the result (the sum of the p, by which it is
        # divided, is at least 1). It shows where the row's likeliest positions hold zeros: values of 1e-6, whose Q8_0 scales vanish in f16
        # for some blocks and not for others.
        lost = 300 * 2.0 ** -36 * np.abs(v).max() * np.sqrt(want[:, 0].size)
        for h in range(4):
            assert np.linalg.norm(got[:, h] - want[:, h]) <= (1e-5 if h < 3 else 1e-4) * np.linalg.norm(want[:, h]) + lost, h
        q[0, 1] = 0.0
        got = attend(b, held, cache, shape, [(0, 298, 2)], 2, q, 4, scale=0.25)
        want = kv_oracle.attention(q, k[0], v[0], 298, 2, scale=0.25)
        assert rel_l2(got[0, 1], want[0, 1]) <= 1e-5  # every position the same
        q[1, 2, 7] = np.nan
        got = attend(b, held, cache, shape, [(0, 298, 2)], 2, q, 4)
        assert np.all(np.isnan(got[1, 2])) and np.all(np.isfinite(np.delete(got.reshape(8, 128), 6, 0)))


def test_the_values_of_one_sequence_may_grow(backend):
    """Scales that rise and fall by orders of magnitude along the sequence."""
    b = backend
    shape = KvCache(1, 1024, 1, 128, enc.Q4_0, enc.Q8_0)
    rng = np.random.default_rng(12)
    k, v = (rng.standard_normal((1000, 1, 128)).astype(np.float32) for _ in range(2))
    v *= np.exp(rng.uniform(-8, 8, (1000, 1, 1))).astype(np.float32)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        write(b, held, cache, shape, [(0, 0, 1000)], 1000, k, v)
        q = rng.standard_normal((1, 4, 128)).astype(np.float32)
        want = kv_oracle.attention(q, kv_oracle.stored(k, enc.Q4_0), kv_oracle.stored(v, enc.Q8_0), 999, 4)
        assert rel_l2(attend(b, held, cache, shape, [(0, 999, 1)], 1, q, 4), want) <= 1e-5


@pytest.mark.parametrize("width", [64, 128, 256])
def test_a_unit_of_many_blocks(backend, width):
    """One head over a long cache: its steps go to most of the device's blocks, and one joins more than 32 parts."""
    b = backend
    length, rows = 20001, 130
    shape = KvCache(1, 20016, 1, width, enc.Q4_0, enc.Q8_0)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [length], 31)
        q = rng.standard_normal((rows, 1, width)).astype(np.float32)
        spans = [(0, length - rows, rows)]
        want = kv_oracle.attention(q, k[0], v[0], length - rows, 1)
        assert rel_l2(attend(b, held, cache, shape, spans, rows, q, 1), want) <= 1e-5
        assert rel_l2(attend(b, held, cache, shape, spans, rows, q, 1, dtype=enc.BF16), want) <= 2.0 ** -8
        one = attend(b, held, cache, shape, [(0, length - 1, 1)], 1, q[-1:], 1)
        assert rel_l2(one, want[-1:]) <= 1e-5


@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("width", [64, 128, 256])
def test_more_units_than_blocks(backend, width, window):
    """A prompt whose units outnumber the device's blocks for either kernel, so that blocks take several whole ones."""
    b = backend
    heads, group, rows = 8, 4, 1300
    shape = KvCache(1, 1312, heads, width, enc.Q8_0, enc.Q4_0)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [rows], 32)
        q = rng.standard_normal((rows, heads * group, width)).astype(np.float32)
        want = kv_oracle.attention(q, k[0], v[0], 0, group, window=window)
        spans = [(0, 0, rows)]
        assert rel_l2(attend(b, held, cache, shape, spans, rows, q, heads * group, window=window), want) <= 1e-5
        assert rel_l2(attend(b, held, cache, shape, spans, rows, q, heads * group, window=window, dtype=enc.BF16), want) <= 2.0 ** -8


def test_graphs_that_join_in_one_scratch(backend):
    """Two recordings whose calls all leave partial results in the handle's scratch, launched in turn: each result is the first one's, bit for bit."""
    b = backend
    shape = KvCache(2, 4096, 2, 128, enc.Q8_0, enc.Q8_0)
    with Held(b) as held:
        cache, k, v, rng = case(b, held, shape, [4000, 2500], 33)
        graphs = []
        for rows, dtype, n in ((1, 0, 4000), (70, enc.BF16, 2500)):
            q = held.up(rng.standard_normal(rows * 4 * 128).astype(np.float32))
            out = held.new(rows * 4 * 128 * (4 if dtype == 0 else 2))
            sp = held.up(kv_spans([(0, n - rows, rows), (1, 2500 - rows, rows)][: 2 if rows == 70 else 1]))
            count = 2 if rows == 70 else 1
            if count == 2:
                q, out = held.up(np.tile(q.floats(), 2)), held.new(2 * out.len)
            logits, tokens, logp = held.up(rng.standard_normal((3, 200001)).astype(np.float32)), held.up(np.array([5, 200000, 77], np.uint32)), held.new(12)
            entropies = held.new(12)
            b.begin()
            b.attention(cache, shape, sp, count, rows, q, 512, 4, out, 512, out_dtype=dtype)
            b.token_logprobs(logits, 3, 200001, 200001, tokens, logp, entropies)
            graphs.append((b.commit_retain(), out, logp))
        first = []
        for g, out, logp in graphs:
            b.graph_launch(g)
            first.append((out.read(np.uint16).copy(), logp.read(np.uint32).copy()))
        for _ in range(5):
            for g, out, logp in graphs:
                b.graph_launch(g, 3)
            for (g, out, logp), (a, l) in zip(graphs, first):
                np.testing.assert_array_equal(out.read(np.uint16), a)
                np.testing.assert_array_equal(logp.read(np.uint32), l)
        for g in graphs:
            b.graph_release(g[0])


def test_two_handles_at_once(backend):
    """A handle a thread, each with its own stream and scratch: the results are those of one alone."""
    shape = KvCache(1, 4096, 2, 128, enc.Q8_0, enc.Q8_0)

    def work(b, seed, turns, results):
        with Held(b) as held:
            cache, k, v, rng = case(b, held, shape, [3000], seed)
            q = rng.standard_normal((40, 4, 128)).astype(np.float32)
            for _ in range(turns):
                results.append(attend(b, held, cache, shape, [(0, 2960, 40)], 40, q, 4, dtype=enc.BF16))
                results.append(attend(b, held, cache, shape, [(0, 2999, 1)], 1, q[-1:], 4))
            want = kv_oracle.attention(q, k[0], v[0], 2960, 2)
            assert rel_l2(results[0], want) <= 2.0 ** -8 and rel_l2(results[1], want[-1:]) <= 1e-5

    other = Backend(0)
    try:
        results = [[], []]
        threads = [threading.Thread(target=work, args=(b, 40 + i, 20, results[i])) for i, b in enumerate((backend, other))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for r in results:
            assert len(r) == 40
            for i in range(2, 40):
                np.testing.assert_array_equal(r[i], r[i % 2])
    finally:
        other.deinit()


@pytest.mark.parametrize("width", [64, 128, 256, 96])
def test_a_recorded_step_follows_its_spans(backend, width):
    """One recording of write + attention, replayed token by token with the spans buffer moved on; a second graph in between."""
    b = backend
    group, steps = 4, 40
    shape = KvCache(2, 64, 2, width, enc.Q8_0, enc.Q8_0)
    n, m = 2 * width, 2 * group * width
    rng = np.random.default_rng(21)
    x = rng.standard_normal((2, steps, m + 2 * n)).astype(np.float32)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        graphs = []
        for s in range(2):  # one graph a sequence: they share the handle's scratch
            row, sp, out = held.up(x[s, 0]), held.up(kv_spans([(s, 0, 1)])), held.new(m * 4)
            b.begin()
            b.kv_write(cache, shape, sp, 1, 1, row.slice(m * 4, n * 4), n, row.slice((m + n) * 4, n * 4), n)
            b.attention(cache, shape, sp, 1, 1, row, m, 2 * group, out, m)
            graphs.append((b.commit_retain(), row, sp, out))
        for step in range(1, steps):
            for s, (graph, row, sp, out) in enumerate(graphs):
                row.write(x[s, step])
                sp.write(kv_spans([(s, step, 1)]))
                b.graph_launch(graph)
                k, v = (kv_oracle.stored(x[s, : step + 1, m + i * n: m + (i + 1) * n].reshape(-1, 2, width), enc.Q8_0) for i in range(2))
                want = kv_oracle.attention(x[s, step, :m].reshape(1, 2 * group, width), k, v, step, group)
                assert rel_l2(out.floats().reshape(want.shape), want) <= 1e-5, (s, step)
        for g in graphs:
            b.graph_release(g[0])


def test_a_bad_span_is_reported_and_left_out(backend):
    b = backend
    shape = KvCache(2, 32, 1, 64, enc.Q8_0, enc.Q8_0)
    rng = np.random.default_rng(2)
    k = rng.standard_normal((4 * 5, 1, 64)).astype(np.float32)
    bad = [(2, 0, 1), (0, 30, 3), (0, 0, 6), (0xffffffff, 0xffffffff, 5)]
    with Held(b) as held:
        cache = held.new(shape.bytes)
        for span in bad:
            with pytest.raises(NuclisError) as e:
                write(b, held, cache, shape, [span, (1, 0, 5)], 5, k[:10], k[:10])
            assert e.value.name == "ExecutionFailed"
            got = read(b, held, cache, shape, [(0, 0, 32), (1, 0, 5)], 32)  # the next call is as ever
            assert np.all(got[0][:32] == 0)
            np.testing.assert_array_equal(got[0][32:37].astype(np.float64), kv_oracle.stored(k[5:10], enc.Q8_0))
            with pytest.raises(NuclisError) as e:
                attend(b, held, cache, shape, [span, (1, 0, 5)], 5, k[:10], 1)
            assert e.value.name == "ExecutionFailed"
            with pytest.raises(NuclisError) as e:
                read(b, held, cache, shape, [(1, 0, 5), span], 5)
            assert e.value.name == "ExecutionFailed"
        # a span that is absent may name anything
        assert np.all(np.isfinite(attend(b, held, cache, shape, [(9, 9, 0), (1, 0, 5)], 5, k[:10], 1)[5:]))


def test_a_cache_beyond_32_bits(backend):
    """Byte offsets past 2^32: the last positions of the last slot, under a window."""
    b = backend
    shape = KvCache(2, 1 << 20, 8, 128, enc.Q8_0, enc.Q8_0)
    assert shape.bytes > 1 << 32
    rng = np.random.default_rng(4)
    with Held(b) as held:
        cache = held.new(shape.bytes)
        first = (1 << 20) - 300
        k, v = (rng.standard_normal((300, 8, 128)).astype(np.float32) for _ in range(2))
        write(b, held, cache, shape, [(1, first, 300)], 300, k, v)
        got = read(b, held, cache, shape, [(1, first, 300), (0, first, 300)], 300)
        np.testing.assert_array_equal(got[0][:300].astype(np.float64), kv_oracle.stored(k, enc.Q8_0))
        np.testing.assert_array_equal(got[1][:300].astype(np.float64), kv_oracle.stored(v, enc.Q8_0))
        assert np.all(got[0][300:] == 0)
        q = rng.standard_normal((1, 40, 128)).astype(np.float32)
        out = attend(b, held, cache, shape, [(1, (1 << 20) - 1, 1)], 1, q, 40, window=290)
        want = kv_oracle.attention(q, kv_oracle.stored(k, enc.Q8_0)[10:], kv_oracle.stored(v, enc.Q8_0)[10:], 289, 5)
        assert rel_l2(out, want) <= 1e-5


def test_rows_whose_bytes_pass_64_bits_are_refused(backend):
    """97 x 172,961 rows are 2^24 + 1: at a stride of 2^40 the last one's offset is 2^64 elements."""
    b = backend
    with Held(b) as held:
        shape = KvCache(1, 32, 1, 64)
        cache, sp, rows = held.new(shape.bytes), held.up(kv_spans([(0, 0, 1)] * 97)), held.new(4096)
        for call in (lambda: b.kv_write(cache, shape, sp, 97, 172961, rows, 1 << 40, rows, 1 << 40),
                     lambda: b.kv_read(cache, shape, sp, 97, 172961, rows.slice(0, 1024), 1 << 40, rows.slice(2048, 1024), 1 << 40),
                     lambda: b.attention(cache, shape, sp, 97, 172961, rows.slice(0, 1024), 1 << 40, 1, rows.slice(2048, 1024), 1 << 40)):
            b.begin()
            with pytest.raises(NuclisError) as e:
                call()
            assert e.value.name == "InvalidShape"
            b.discard()


def test_refusals(backend):
    b = backend
    with Held(b) as held:
        shape = KvCache(2, 32, 2, 64)
        cache, sp, rows, out = held.new(shape.bytes), held.up(kv_spans([(0, 0, 1)] * 4)), held.new(4 * 256 * 4), held.new(4 * 512 * 4)

        def refused(name, call, *args, **kw):
            b.begin()
            with pytest.raises(NuclisError) as e:
                call(*args, **kw)
            assert e.value.name == name
            b.discard()

        def kvw(cache=cache, shape=shape, sp=sp, s=1, t=1, k=rows, ks=128, v=rows, vs=128):
            b.kv_write(cache, shape, sp, s, t, k, ks, v, vs)

        def kvr(k=out, ks=256, v=out.slice(512, out.len - 512), vs=256, dtype=0, s=1, t=1):
            b.kv_read(cache, shape, sp, s, t, k, ks, v, vs, out_dtype=dtype)

        def att(q=rows, qs=256, heads=4, o=out, os=256, s=1, t=1, **kw):
            b.attention(cache, shape, sp, s, t, q, qs, heads, o, os, **kw)

        for call in (kvw, kvr, att):
            refused("InvalidShape", call, s=0)
            refused("InvalidShape", call, t=0)
            refused("InvalidShape", call, s=5)      # the spans buffer holds four
            refused("InvalidShape", call, t=9)      # rows past the buffers
            refused("InvalidShape", call, s=-1)
        other = KvCache(2, 32, 2, 64, enc.Q6_K, enc.Q8_0)
        refused("UnsupportedTensorEncoding", kvw, shape=other)
        for bad in (KvCache(2, 33, 2, 64), KvCache(2, 32, 2, 48), KvCache(2, 32, 2, 544), KvCache(0, 32, 2, 64), KvCache(2, 0, 2, 64), KvCache(2, 32, 0, 64), KvCache(3, 32, 2, 64)):
            refused("InvalidShape", kvw, shape=bad)
        refused("InvalidShape", kvw, ks=127)
        refused("InvalidShape", kvw, cache=cache.slice(8, cache.len - 8))
        refused("InvalidShape", kvw, sp=sp.slice(4, 16))
        refused("InvalidShape", kvw, k=cache)
        refused("InvalidShape", kvr, dtype=1)
        refused("InvalidShape", kvr, v=out.slice(256, out.len - 256))   # values on top of the keys
        refused("InvalidShape", kvr, v=out.slice(512, out.len - 512), ks=250, t=2)
        refused("InvalidShape", kvr, k=cache)
        refused("InvalidShape", att, heads=3)
        refused("InvalidShape", att, heads=0)
        refused("InvalidShape", att, scale=-1.0)
        refused("InvalidShape", att, scale=float("nan"))
        refused("InvalidShape", att, scale=float("inf"))
        refused("InvalidShape", att, out_dtype=1)
        refused("InvalidShape", att, qs=255)
        refused("InvalidShape", att, o=rows)
        refused("InvalidShape", att, o=cache)
        with pytest.raises(NuclisError) as e:
            kvw()
        assert e.value.name == "NotRecording"
