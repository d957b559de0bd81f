"""The decode stack with attention between QKV and O: the operators as a model plan records them (projections, cache write,
attention, projections), replayed step by step, against the CPU oracle of the projections and the 64-bit attention."""
import numpy as np
import pytest

import kv_oracle
import oracle
from nuclis_b200 import Backend, encoding as enc
from nuclis_b200.shard import LayerShapes, rank_shapes
from nuclis_b200.stack import Stack, make_stack
from parity import rel_l2

pytestmark = pytest.mark.gpu

SHAPES = LayerShapes(hidden=1024, ffn=2048, kv=256)  # 8 query heads on 2 key/value heads of 128


@pytest.fixture(scope="module")
def backend():
    b = Backend(0)
    yield b
    b.deinit()


def host_weights(w):
    return {name: getattr(w, name).read() for name in ("qkv", "o", "gate", "up", "down")}


def layer(x, host, cache, kenc, venc, window=0, width=128):
    """One layer's outputs for the rows x, appended to `cache` (lists of keys and of values), in the oracle's arithmetic and 64 bits."""
    s = SHAPES
    qkv = oracle.matmul(enc.Q4_K, s.qkv_rows, s.hidden, host["qkv"], x)
    q, k, v = np.split(qkv, [s.hidden, s.hidden + s.kv], axis=1)
    first = len(cache[0])
    cache[0].extend(kv_oracle.stored(k.reshape(len(x), -1, width), kenc))
    cache[1].extend(kv_oracle.stored(v.reshape(len(x), -1, width), venc))
    a = kv_oracle.attention(q.reshape(len(x), -1, width), np.array(cache[0]), np.array(cache[1]), first, s.hidden // s.kv, window=window)
    a = a.reshape(len(x), -1).astype(np.float32)
    o = oracle.matmul(enc.Q4_K, s.hidden, s.hidden, host["o"], a)
    g, u = (oracle.matmul(enc.Q4_K, s.ffn, s.hidden, host[n], o) for n in ("gate", "up"))
    return oracle.matmul(enc.Q6_K, s.hidden, s.ffn, host["down"], (oracle.silu(g) * u).astype(np.float32)), a


@pytest.mark.parametrize("kenc,venc,window", [(enc.Q8_0, enc.Q8_0, 0), (enc.Q4_0, enc.Q4_0, 6)])
def test_a_recorded_step_replayed_along_the_sequence(backend, kenc, venc, window):
    """One token a step. The bound of a chain: five F32 products and the attention at 1e-5 each, the SwiGLU product doubling one: 1e-4."""
    b = backend
    st = make_stack(b, 1, 2, shapes=SHAPES, seed=31, prepare=False)
    st.enable_attention(64, key_encoding=kenc, value_encoding=venc, window=window)
    host = [host_weights(w) for w in st.layers]
    rng = np.random.default_rng(3)
    caches = [([], []), ([], [])]
    b.begin()
    assert st.record() == 2 * 6
    graph = b.commit_retain()
    for step in range(20):
        x = rng.standard_normal((1, SHAPES.hidden)).astype(np.float32)
        st.h.write(x)
        st.seek(step)
        b.graph_launch(graph)
        for i in range(2):  # every layer reads the same input row; the last one's output is in d
            want, a = layer(x, host[i], caches[i], kenc, venc, window)
        assert rel_l2(st.att.floats(), a[0]) <= 1e-4, step
        assert rel_l2(st.d.floats(), want[0]) <= 1e-4, step
    b.graph_release(graph)


def test_a_prompt_and_then_single_tokens(backend):
    """40 rows through the prefill products (BF16 operands: relative L2 2e-2 a product, as the prefill tests hold them), then steps of one
    token on the same caches with the folded norms, and a verified draft of three."""
    b = backend
    st = make_stack(b, 40, 1, shapes=SHAPES, seed=32, prepare=False)
    st.enable_attention(64)
    host = host_weights(st.layers[0])
    rng = np.random.default_rng(4)
    x = rng.standard_normal((40, SHAPES.hidden)).astype(np.float32)
    st.h.write(x)
    b.begin()
    st.record()
    b.commit()
    cache = ([], [])
    want, a = layer(x, host, cache, enc.Q8_0, enc.Q8_0)
    got = (st.att.read(np.uint16).astype(np.uint32) << 16).view(np.float32)[: a.size].reshape(a.shape)
    assert rel_l2(got, a) <= 2e-2 and rel_l2(st.d.floats()[: want.size].reshape(want.shape), want) <= 4e-2

    for rows in (1, 3):
        nx = Stack(b, SHAPES, rank_shapes(SHAPES, 1, 0), rows)
        nx.layers = st.layers
        nx.enable_attention(64)
        b.release(nx.caches[0])
        nx.caches = st.caches
        # the oracle goes on from the cache as the prompt left it
        n = SHAPES.kv
        out, spans = b.create(64 * 2 * n * 4), b.create(16)
        from nuclis_b200 import kv_spans
        first = 40 if rows == 1 else 41
        spans.write(kv_spans([(0, 0, first)]))
        b.begin()
        b.kv_read(st.caches[0], st.kv_shape, spans, 1, first, out, 2 * n, out.slice(n * 4, out.len - n * 4), 2 * n)
        b.commit()
        held = out.floats()[: first * 2 * n].reshape(first, 2, -1, 128).astype(np.float64)
        cache = (list(held[:, 0]), list(held[:, 1]))
        x = rng.standard_normal((rows, SHAPES.hidden)).astype(np.float32)
        nx.h.write(x)
        nx.seek(first)
        b.begin()
        nx.record()
        b.commit()
        want, a = layer(x, host, cache, enc.Q8_0, enc.Q8_0)
        assert rel_l2(nx.att.floats()[: a.size].reshape(a.shape), a) <= 1e-4
        assert rel_l2(nx.d.floats()[: want.size].reshape(want.shape), want) <= 1e-4


def test_attention_between_the_folded_norms(backend):
    b = backend
    st = make_stack(b, 1, 1, shapes=SHAPES, seed=33, prepare=False)
    st.enable_norms(7)
    st.enable_attention(32, width=64)
    host = host_weights(st.layers[0])
    b.begin()
    assert st.record() == 6
    graph = b.commit_retain()
    cache = ([], [])
    residual = st.residual0.copy()
    for step in range(3):
        if step:
            st.seek(step)
            b.graph_launch(graph)
        def norm(r, w):
            r = r.astype(np.float64)
            return (r / np.sqrt(np.mean(r * r) + 1e-6) * w).astype(np.float32)[None]
        s = SHAPES
        qkv = oracle.matmul(enc.Q4_K, s.qkv_rows, s.hidden, host["qkv"], norm(residual, st.norm_attn_host))
        q, k, v = np.split(qkv, [s.hidden, s.hidden + s.kv], axis=1)
        cache[0].extend(kv_oracle.stored(k.reshape(1, -1, 64), enc.Q8_0))
        cache[1].extend(kv_oracle.stored(v.reshape(1, -1, 64), enc.Q8_0))
        a = kv_oracle.attention(q.reshape(1, -1, 64), np.array(cache[0]), np.array(cache[1]), step, s.hidden // s.kv).reshape(1, -1).astype(np.float32)
        residual = residual + oracle.matmul(enc.Q4_K, s.hidden, s.hidden, host["o"], a)[0]
        f = norm(residual, st.norm_ffn_host)
        g, u = (oracle.matmul(enc.Q4_K, s.ffn, s.hidden, host[n], f) for n in ("gate", "up"))
        residual = residual + oracle.matmul(enc.Q6_K, s.hidden, s.ffn, host["down"], (oracle.silu(g) * u).astype(np.float32))[0]
        assert rel_l2(st.residual.floats(), residual) <= 1e-4, step
    b.graph_release(graph)


def test_heads_that_do_not_divide_are_refused(backend):
    st = Stack(backend, SHAPES, rank_shapes(SHAPES, 1, 0), 1)
    with pytest.raises(ValueError):
        st.enable_attention(16, width=384)
