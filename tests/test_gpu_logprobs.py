"""Log probabilities of given tokens, entropies and alternatives against 64 bits.

Bounds. x - m is exact or rounded once; ex2 of it is off by 2^-22 and its argument's rounding (2^-24 of up to 150, weighted by a term that
small); Z's sum runs over a thread's share in F32 (n / 65536 x 2^-24 and less, of random sign). So ln Z is off by some 1e-6 at most, and
a log probability by that plus 2^-23 of its own size: 4e-6 + 4e-7 |log p| covers both. The entropy is ln Z minus a mean of the same kind.
Indexes are exact, the lowest first among equals."""
import numpy as np
import pytest

from nuclis_b200 import Backend, NuclisError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    b = Backend(0)
    yield b
    b.deinit()


def run(b, logits, tokens, k, stride=None, offset=0):
    """logits [rows][count]; laid out at `stride` floats a row, `offset` floats into the buffer."""
    rows, count = logits.shape
    stride = stride or count
    flat = np.full(offset + rows * stride, 1e30, np.float32)
    np.lib.stride_tricks.as_strided(flat[offset:], (rows, count), (stride * 4, 4))[:] = logits
    bufs = []

    def up(x):
        bufs.append(b.create(x.nbytes))
        bufs[-1].write(x)
        return bufs[-1]

    x, t = up(flat), up(np.asarray(tokens, np.uint32))
    lp, ent = up(np.zeros(rows, np.float32)), up(np.zeros(rows, np.float32))
    top, tlp = (up(np.zeros(rows * k, np.uint32)), up(np.zeros(rows * k, np.float32))) if k else (None, None)
    b.begin()
    b.token_logprobs(x.slice(offset * 4, x.len - offset * 4), rows, count, stride, t, lp, ent, k, top, tlp)
    b.commit()
    out = lp.floats(), ent.floats(), top.read(np.uint32).reshape(rows, k) if k else None, tlp.floats().reshape(rows, k) if k else None
    for buf in bufs:
        b.release(buf)
    return out


def check(logits, tokens, k, got):
    lp, ent, top, tlp = got
    x = logits.astype(np.float64)
    m = x.max(1, keepdims=True)
    z = np.exp(x - m).sum(1, keepdims=True)
    logp = x - m - np.log(z)
    want = logp[np.arange(len(x)), tokens]
    finite = np.isfinite(want)
    np.testing.assert_array_equal(lp[~finite], want[~finite])
    assert np.all(np.abs(lp[finite] - want[finite]) <= 4e-6 + 4e-7 * np.abs(want[finite]))
    p = np.exp(logp)
    h = -np.where(p > 0, p * np.where(p > 0, logp, 0), 0).sum(1)
    assert np.all(np.abs(ent - h) <= 4e-6 + 4e-7 * h)
    if k:
        order = np.argsort(-logits, axis=1, kind="stable")[:, :k]
        np.testing.assert_array_equal(top, order)
        want = np.take_along_axis(logp, order, 1)
        finite = np.isfinite(want)
        np.testing.assert_array_equal(tlp[~finite], want[~finite])
        assert np.all(np.abs(tlp[finite] - want[finite]) <= 4e-6 + 4e-7 * np.abs(want[finite]))


@pytest.mark.parametrize("rows,count,k", [(1, 1, 1), (1, 2, 0), (1, 5, 5), (3, 31, 31), (2, 32, 32), (1, 4095, 20), (1, 4097, 1), (7, 5000, 3), (1, 32001, 20), (1, 248320, 20),
                                          (1, 248320, 0), (2, 248321, 32), (40, 10007, 5), (300, 4099, 7), (700, 1500, 2), (65, 131072, 1)])
@pytest.mark.parametrize("stride,offset", [(0, 0), (3, 1)])
def test_against_64_bits(backend, rows, count, k, stride, offset):
    rng = np.random.default_rng(rows * 7 + count)
    x = (rng.standard_normal((rows, count)) * rng.uniform(0.01, 6, (rows, 1))).astype(np.float32)
    x[rng.integers(0, rows, 3), rng.integers(0, count, 3)] += 20
    tokens = rng.integers(0, count, rows)
    got = run(backend, x, tokens, k, count + stride, offset)
    check(x, tokens, k, got)
    for a, b in zip(got, run(backend, x, tokens, k, count + stride, offset)):
        assert a is b or np.array_equal(a, b)  # the same from run to run


@pytest.mark.parametrize("rows,count", [(1, 248320), (1, 9000), (600, 9000), (2, 50)])
def test_ties_go_to_the_lowest_index(backend, rows, count):
    k = 20
    rng = np.random.default_rng(count)
    for x in (np.zeros((rows, count)), rng.integers(0, 3, (rows, count)), np.where(rng.random((rows, count)) < 0.5, 0.0, -0.0), np.sort(rng.standard_normal((rows, count)), 1),
              -np.sort(rng.standard_normal((rows, count)), 1), np.floor(np.linspace(0, 50, count))[None].repeat(rows, 0)):
        x = x.astype(np.float32)
        tokens = rng.integers(0, count, rows)
        check(x, tokens, k, run(backend, x, tokens, k))


@pytest.mark.parametrize("rows,count", [(2, 248320), (600, 9001), (3, 40)])
def test_masks(backend, rows, count):
    """Minus infinity and the type's lowest value, few tokens left, one left."""
    k = 20
    rng = np.random.default_rng(count)
    x = rng.standard_normal((rows, count)).astype(np.float32) * 3
    for mask in (-np.inf, np.finfo(np.float32).min):
        for left in (count // 2, 25, 3, 1):
            y = np.full_like(x, mask)
            keep = rng.permutation(count)[:left]
            y[:, keep] = x[:, keep]
            tokens = np.where(rng.random(rows) < 0.5, keep[0], rng.integers(0, count, rows))
            check(y, tokens, k, run(backend, y, tokens, k))


def test_large_and_close_values(backend):
    rng = np.random.default_rng(1)
    x = np.stack([rng.standard_normal(20000) * 1e-3 + 5000, rng.standard_normal(20000) * 1e4, np.r_[100.0, np.zeros(19999)], np.full(20000, 3e38)]).astype(np.float32)
    tokens = np.array([7, int(x[1].argmax()), 0, 19999])
    check(x, tokens, 10, run(backend, x, tokens, 10))


@pytest.mark.parametrize("rows,count", [(4, 248320), (600, 5000)])
def test_rows_without_an_answer(backend, rows, count):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((rows, count)).astype(np.float32)
    x[0] = -np.inf
    x[1, count // 3] = np.nan
    x[2, count - 1] = np.inf
    tokens = np.full(rows, 3)
    tokens[3] = count
    lp, ent, top, tlp = run(backend, x, tokens, 4)
    assert lp[0] == -np.inf and ent[0] == 0 and np.all(tlp[0] == -np.inf)
    np.testing.assert_array_equal(top[0], np.arange(4))
    for r in (1, 2):
        assert np.isnan(lp[r]) and np.isnan(ent[r]) and np.all(np.isnan(tlp[r])) and np.all(top[r] == 0xffffffff)
    assert np.isnan(lp[3]) and np.isfinite(ent[3])  # a token outside the vocabulary
    tokens[3] = 3
    rest = np.arange(3, rows)
    check(x[rest], tokens[rest], 4, tuple(a[rest] for a in run(backend, x, tokens, 4)))


def test_alternatives_agree_with_argmax_in_one_recording(backend):
    """The head's last steps together: the greedy token into the tokens buffer, then its log probability."""
    b = backend
    count = 32007
    rng = np.random.default_rng(9)
    x = rng.standard_normal(count).astype(np.float32)
    bufs = [b.create(n) for n in (count * 4, 4, 4, 4, 4, 4)]
    logits, token, lp, ent, top, tlp = bufs
    logits.write(x)
    b.begin()
    b.argmax(logits, count, token)
    b.token_logprobs(logits, 1, count, count, token, lp, ent, 1, top, tlp)
    graph = b.commit_retain()
    for step in range(3):
        logits.write(x + np.float32(step) * rng.standard_normal(count).astype(np.float32))
        b.graph_launch(graph)
        y = logits.floats()
        assert token.read(np.uint32)[0] == top.read(np.uint32)[0] == y.argmax()
        assert lp.floats()[0] == tlp.floats()[0]
    b.graph_release(graph)
    for buf in bufs:
        b.release(buf)


def test_refusals(backend):
    b = backend
    x, small, other = b.create(4000), b.create(40), b.create(400)

    def refused(*args):
        b.begin()
        with pytest.raises(NuclisError) as e:
            b.token_logprobs(*args)
        assert e.value.name == "InvalidShape"
        b.discard()

    a, c, d, f = (other.slice(i * 100, 100) for i in range(4))
    for args in ((x, 0, 10, 10, a, c, d), (x, 1, 0, 10, a, c, d), (x, 2, 10, 9, a, c, d), (x, 11, 100, 100, a, c, d), (x, 30, 10, 10, a, c, d), (x, 1, 10, 10, a, c, c),
                 (x, 1, 10, 10, a, c, x), (x, 1, 10, 10, a, a, d), (x, 1, 10, 10, a, c, d, 11, f, small), (x, 1, 100, 100, a, c, d, 33, f, small),
                 (x, 1, 100, 100, a, c, d, 5, None, small), (x, 1, 100, 100, a, c, d, 5, f, f), (x, 1, 100, 100, a, c, d, 11, f, small), (x.slice(2, 400), 1, 10, 10, a, c, d)):
        refused(*args)
    with pytest.raises(NuclisError) as e:
        b.token_logprobs(x, 1, 10, 10, a, c, d)
    assert e.value.name == "NotRecording"
    for buf in (x, small, other):
        b.release(buf)
