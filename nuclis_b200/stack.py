"""The synthetic dense decode layer stack: 64 layers of QKV -> O -> SwiGLU gate/up -> down.

The matmul chain of a decoder layer: per layer

    qkv = Wqkv . h                      Q4_K  [hidden + 2 kv][hidden]
    o   = Wo . qkv[:hidden]             Q4_K  [hidden][hidden]         (+ allreduce)
    a   = silu(Wgate . o) * (Wup . o)   Q4_K  [ffn][hidden] each
    d   = Wdown . a                     Q6_K  [hidden][ffn]            (+ allreduce)

written against the backend's operator interface exactly as a model plan of
the reference would write it (``matvec``, ``matvecSegments`` with the SiLU pair
mode, ``matmul`` for a verify batch; inference/src/models/qwen35_metal.zig:589-640).
Every layer reads the same input hidden state: 64 un-normalised layers of
random weights overflow F32 within a dozen products, and the norms that keep a
real model bounded are not part of this path. Stream order keeps the layers
serial all the same, and every weight byte of every layer is read each step.

Norms and residuals come in with ``enable_norms``, attention over a quantized
key/value cache between QKV and O with ``enable_attention``; without the latter O
reads the Q slice as it is, which is what the matmul benchmark times.

With ``ranks`` > 1 the layer is row-split (see ``shard``): each rank holds its
rows of QKV/gate/up and its K slice of O/down, and the partial O and down
outputs are summed over the ranks.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np

from . import encoding as enc
from .backend import Backend, Buffer, KvCache, Matrix, Segment, SegmentMode, kv_spans
from .errors import NuclisError
from .shard import LayerShapes, RankShapes, rank_shapes


@dataclass
class LayerWeights:
    qkv: Buffer
    o: Buffer
    gate: Buffer
    up: Buffer
    down: Buffer


@dataclass
class Stack:
    backend: Backend
    shapes: LayerShapes
    local: RankShapes
    tokens: int
    layers: list[LayerWeights] = field(default_factory=list)

    def __post_init__(self):
        b, s, l, m = self.backend, self.shapes, self.local, self.tokens
        pad = Backend.matmul_padded(m) if m > 1 else 1
        self.m_qkv = Matrix(s.qkv_encoding, l.qkv_rows, s.hidden, enc.matrix_bytes(s.qkv_encoding, l.qkv_rows, s.hidden))
        self.m_o = Matrix(s.o_encoding, s.hidden, l.q_rows, enc.matrix_bytes(s.o_encoding, s.hidden, l.q_rows))
        self.m_gate = Matrix(s.gate_up_encoding, l.ffn_rows, s.hidden, enc.matrix_bytes(s.gate_up_encoding, l.ffn_rows, s.hidden))
        self.m_down = Matrix(s.down_encoding, s.hidden, l.ffn_rows, enc.matrix_bytes(s.down_encoding, s.hidden, l.ffn_rows))
        self.h = b.create(pad * s.hidden * 4)
        self.qkv = b.create(pad * l.qkv_rows * 4)
        self.o = b.create(pad * s.hidden * 4)
        self.g = b.create(pad * l.ffn_rows * 4)
        self.u = b.create(pad * l.ffn_rows * 4)
        self.d = b.create(pad * s.hidden * 4)

    # ---- weights ----
    def weight_bytes_per_layer(self) -> int:
        return self.m_qkv.bytes + self.m_o.bytes + 2 * self.m_gate.bytes + self.m_down.bytes

    def add_layer_buffers(self) -> LayerWeights:
        b = self.backend
        w = LayerWeights(b.create(self.m_qkv.bytes), b.create(self.m_o.bytes), b.create(self.m_gate.bytes),
                         b.create(self.m_gate.bytes), b.create(self.m_down.bytes))
        self.layers.append(w)
        return w

    def fill_layer_torch(self, w: LayerWeights, seed: int) -> None:
        """Random blocks drawn on the device (see ``synth``): local shard shapes, seeded per layer and rank."""
        from . import synth
        s, l = self.shapes, self.local
        for i, (buf, e, rows, cols) in enumerate([(w.qkv, s.qkv_encoding, l.qkv_rows, s.hidden), (w.o, s.o_encoding, s.hidden, l.q_rows),
                                                  (w.gate, s.gate_up_encoding, l.ffn_rows, s.hidden), (w.up, s.gate_up_encoding, l.ffn_rows, s.hidden),
                                                  (w.down, s.down_encoding, s.hidden, l.ffn_rows)]):
            synth.fill_matrix_torch(device_tensor(buf), e, rows, cols, seed * 8 + i)

    def prepare_layer(self, w: LayerWeights) -> None:
        """Load-time re-layout of the matrices whose GGUF rows the specialized kernels cannot address
        (the Q6_K down projection): same bytes, same values. The GGUF copy is released."""
        b = self.backend
        raw = Matrix(self.m_down.encoding, self.m_down.rows, self.m_down.columns, self.m_down.bytes)
        prepared, m = b.prepare(w.down, raw)
        b.release(w.down)
        w.down = prepared
        self.m_down = m

    # ---- attention ----
    def enable_attention(self, capacity: int, width: int = 128, key_encoding: int = enc.Q8_0, value_encoding: int = enc.Q8_0, window: int = 0) -> None:
        """Adds what a decoder layer has between its QKV and its O projection: the step's keys and values into the layer's quantized
        cache, and causal grouped-query attention over it (heads of ``width``; this rank's where the layer is split). The step's
        position is read on the device: ``seek`` moves a recorded step on."""
        b, l, m = self.backend, self.local, self.tokens
        if l.q_rows % width or l.kv_rows % width or l.q_rows % l.kv_rows:
            raise ValueError("the rows of Q and of K are whole heads, and a key/value head serves as many query heads as another")
        self.kv_shape = KvCache(1, (capacity + 15) // 16 * 16, l.kv_rows // width, width, key_encoding, value_encoding)
        self.kv_window = window
        self.caches = [b.create(self.kv_shape.bytes) for _ in self.layers]
        self.spans = b.create(16)
        # a prompt's rows go into O's prefill product as BF16, which rounds them anyway
        self.att_dtype = enc.BF16 if m > Backend.matvec_rows_max else enc.F32
        self.att = b.create((Backend.matmul_padded(m) if m > 1 else 1) * l.q_rows * (2 if self.att_dtype == enc.BF16 else 4))
        self.seek(0)

    def seek(self, position: int) -> None:
        """The next step's rows stand at ``position`` and behind it (between recordings: the spans are uploaded)."""
        self.spans.write(kv_spans([(0, position, self.tokens)]))

    def record_attention(self, layer: int) -> tuple[Buffer, int, int]:
        """O's input for the layer: buffer, row stride and dtype."""
        b, l, m = self.backend, self.local, self.tokens
        if getattr(self, "caches", None) is None:
            return self.qkv.slice(0, self.qkv.len), l.qkv_rows, enc.F32
        cache, shape = self.caches[layer], self.kv_shape
        keys = self.qkv.slice(l.q_rows * 4, self.qkv.len - l.q_rows * 4)
        values = self.qkv.slice((l.q_rows + l.kv_rows) * 4, self.qkv.len - (l.q_rows + l.kv_rows) * 4)
        b.kv_write(cache, shape, self.spans, 1, m, keys, l.qkv_rows, values, l.qkv_rows)
        b.attention(cache, shape, self.spans, 1, m, self.qkv, l.qkv_rows, l.q_rows // shape.width, self.att, l.q_rows, window=self.kv_window,
                    out_dtype=self.att_dtype)
        return self.att, l.q_rows, self.att_dtype

    # ---- the recording of one step ----
    def enable_norms(self, seed: int = 0) -> None:
        """Adds what a pre-norm decoder layer has around its projections (inference/src/models/qwen35_metal.zig:635-640):
        a residual row and the two RMS-norm weight rows (shared by the layers here: their values do not matter to the
        timing). ``record`` then uses the folded operators: four launches a layer, as without the norms."""
        import numpy as np
        b, s = self.backend, self.shapes
        rng = np.random.default_rng(seed + 17)
        self.residual = b.create(s.hidden * 4)
        self.residual0 = (rng.standard_normal(s.hidden) * 0.5).astype(np.float32)
        self.norm_attn, self.norm_ffn = b.create(s.hidden * 4), b.create(s.hidden * 4)
        self.norm_attn_host = (1.0 + 0.1 * rng.standard_normal(s.hidden)).astype(np.float32)
        self.norm_ffn_host = (1.0 + 0.1 * rng.standard_normal(s.hidden)).astype(np.float32)
        self.norm_attn.write(self.norm_attn_host)
        self.norm_ffn.write(self.norm_ffn_host)
        self.residual.write(self.residual0)

    def record_with_norms(self, reduce: bool = False) -> int:
        """One token: x += O(Q(norm(x))); x += down(silu(gate(norm(x))) * up(norm(x))) per layer, the norms folded into the
        staging passes of QKV and of the gate/up pair, the adds into the writes of O and down; with the layer split over
        ranks (``reduce``) the adds are folded into the gathers of the two sums instead."""
        b, hidden = self.backend, self.shapes.hidden
        attention = 2 if getattr(self, "caches", None) is not None else 0
        for i, w in enumerate(self.layers):
            b.matvec_segments_normed([Segment(w.qkv, self.m_qkv, self.qkv)], self.residual, self.norm_attn)
            a_in, _, _ = self.record_attention(i)
            if reduce:
                b.matvec(w.o, self.m_o, a_in, self.o)
                b.allreduce_sum_add_f32(self.o, self.residual, hidden)
            else:
                b.matvec_add(w.o, self.m_o, a_in, self.residual, self.residual)
            b.matvec_segments_normed([Segment(w.gate, self.m_gate, self.g), Segment(w.up, self.m_gate, self.g)], self.residual, self.norm_ffn,
                                     mode=SegmentMode.silu_mul_pair)
            if reduce:
                b.matvec(w.down, self.m_down, self.g, self.d)
                b.allreduce_sum_add_f32(self.d, self.residual, hidden)
            else:
                b.matvec_add(w.down, self.m_down, self.g, self.residual, self.residual)
        return ((6 if reduce else 4) + attention) * len(self.layers)

    def record(self, allreduce: bool | None = None) -> int:
        """Records every layer's chain into the open recording; returns how many operators it recorded."""
        b, s, l, m = self.backend, self.shapes, self.local, self.tokens
        reduce = l.ranks > 1 if allreduce is None else allreduce
        ops = 0
        attention = 2 if getattr(self, "caches", None) is not None else 0
        if getattr(self, "residual", None) is not None and m == 1:
            return self.record_with_norms(reduce)
        for i, w in enumerate(self.layers):
            ops += attention
            if m == 1:
                b.matvec(w.qkv, self.m_qkv, self.h, self.qkv)
                a_in, a_stride, a_dtype = self.record_attention(i)  # without attention the Q slice: the first q_rows floats of each token row
                b.matvec(w.o, self.m_o, a_in, self.o)
                ops += 2
                if reduce:
                    b.allreduce_sum_f32(self.o, s.hidden)
                    ops += 1
                try:
                    b.matvec_segments([Segment(w.gate, self.m_gate, self.g), Segment(w.up, self.m_gate, self.g)], self.o, SegmentMode.silu_mul_pair)
                    ops += 1
                except NuclisError as e:
                    if e.name != "MergeDeclined":
                        raise
                    # the caller's fallback of the reference: two projections and the activation (qwen35_metal.zig:597-600)
                    b.matvec(w.gate, self.m_gate, self.o, self.g)
                    b.matvec(w.up, self.m_gate, self.o, self.u)
                    b.silu_mul(self.g, self.u, l.ffn_rows)
                    ops += 3
                b.matvec(w.down, self.m_down, self.g, self.d)
                ops += 1
                if reduce:
                    b.allreduce_sum_f32(self.d, s.hidden)
                    ops += 1
            else:
                b.matmul(w.qkv, self.m_qkv, self.h, s.hidden, self.qkv, l.qkv_rows, m)
                a_in, a_stride, a_dtype = self.record_attention(i)
                b.matmul(w.o, self.m_o, a_in, a_stride, self.o, s.hidden, m, in_dtype=a_dtype)
                ops += 2
                if reduce:
                    b.allreduce_sum_f32(self.o, m * s.hidden)
                    ops += 1
                b.matmul(w.gate, self.m_gate, self.o, s.hidden, self.g, l.ffn_rows, m)
                b.matmul(w.up, self.m_gate, self.o, s.hidden, self.u, l.ffn_rows, m)
                b.silu_mul(self.g, self.u, m * l.ffn_rows)
                b.matmul(w.down, self.m_down, self.g, l.ffn_rows, self.d, s.hidden, m)
                ops += 4
                if reduce:
                    b.allreduce_sum_f32(self.d, m * s.hidden)
                    ops += 1
        return ops

    def algorithmic_bytes_per_step(self) -> int:
        """Weight bytes read plus activation bytes read and written by the matmuls, all layers."""
        s, l, m = self.shapes, self.local, self.tokens
        acts = m * 4 * (s.hidden + l.qkv_rows + l.q_rows + s.hidden + 2 * (s.hidden + l.ffn_rows) + l.ffn_rows + s.hidden)
        return len(self.layers) * (self.weight_bytes_per_layer() + acts)


def device_tensor(buf: Buffer):
    """A torch uint8 view of a backend buffer (no copy), for filling it on the device."""
    import torch

    class _Raw:
        pass

    raw = _Raw()
    raw.__cuda_array_interface__ = {"shape": (buf.len,), "typestr": "|u1", "data": (buf.device_ptr, False), "version": 2}
    return torch.as_tensor(raw, device=f"cuda:{buf.backend.device}")


def make_stack(backend: Backend, tokens: int, layers: int, ranks: int = 1, rank: int = 0, seed: int = 0,
               shapes: LayerShapes | None = None, prepare: bool = True) -> Stack:
    shapes = shapes or LayerShapes()
    st = Stack(backend, shapes, rank_shapes(shapes, ranks, rank), tokens)
    for i in range(layers):
        w = st.add_layer_buffers()
        st.fill_layer_torch(w, seed * 100003 + i * 64 + rank)
        if prepare:
            import torch
            torch.cuda.synchronize()
            st.prepare_layer(w)
    return st
