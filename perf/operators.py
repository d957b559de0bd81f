"""What is measured of the operators around a quantized key/value cache and of the token log probabilities.

Four operators of ``nuclis_b200.Backend``:

    kv_write         rows of keys and values, quantized as they are written into a cache (Q8_0 or Q4_0 blocks of 32)
    kv_read          rows of the cache decoded again, to F32 or BF16
    attention        causal grouped-query attention over the cache, from one token to a whole prompt
    token_logprobs   log probabilities of given tokens with the entropy of each row and its top alternatives

``run`` computes them in elementary torch operations, or, where ``own`` is set, with the calls that a program makes of
the library: the operators recorded once (``begin`` .. ``commit_retain``) and replayed with ``graph_launch``.
"""
import math

import torch

own = False

Q4_0, Q8_0 = 2, 8
F32, BF16 = 0, 30
DEVICE = "cuda"


# ---- the cases ---------------------------------------------------------------------------------------------------------
# Heads and widths: 40 query heads on 8 key/value heads of 128 are the layer of the 27B-shape stack (hidden 5120, 1024 rows of
# K and of V); 20 on 4 of 256 are the same layer with wide heads, 24 on 8 of 64 a small model. 248320 is the vocabulary of the
# output head. The sessions of a batch have lengths spread evenly up to `context` (`sessions`), in an order that comes from the seed.

def listed():
    return [
        # one decode step's row of keys and values into the cache, and back: the smallest call, all latency
        kv("write 1 row q4_0", "write", heads=8, width=128, kenc=Q4_0, venc=Q4_0, tokens=1, context=517, dtype=F32),
        # a prompt's keys and values into the cache and back for a dense consumer: wide keys, narrow values
        kv("write 4096 rows q8_0/q4_0", "write", heads=8, width=128, kenc=Q8_0, venc=Q4_0, tokens=4096, context=4096, dtype=F32),
        # a short saved prefix read back, wide heads, at odd positions
        kv("read 777 rows q8_0", "read", heads=4, width=256, kenc=Q8_0, venc=Q8_0, tokens=777, context=1001, dtype=F32),
        # a long session's cache decoded to BF16, the largest copy
        kv("read 65536 rows q4_0 bf16", "read", heads=8, width=128, kenc=Q4_0, venc=Q4_0, tokens=65536, context=65536, dtype=BF16),
        # a decode step early in a chat: latency counts
        attn("decode 1 at 700 q4_0", heads=8, group=5, width=128, kenc=Q4_0, venc=Q4_0, context=700),
        # a decode step at the end of a long document: the cache is the work
        attn("decode 1 at 131072 q4_0", heads=8, group=5, width=128, kenc=Q4_0, venc=Q4_0, context=131072),
        # a draft of six tokens verified at once, wide heads, eight-bit cache
        attn("verify 6 at 20000 q8_0", heads=4, group=5, width=256, kenc=Q8_0, venc=Q8_0, tokens=6, context=20000),
        # a batch of sessions of all lengths, one token each, under a sliding window
        attn("batch 24 to 9000 window", heads=8, group=3, width=64, kenc=Q8_0, venc=Q4_0, sequences=24, context=9000, window=4096),
        # a prompt from its first token, rounded to BF16 for the projection behind it
        attn("prompt 2048 q4_0 bf16", heads=8, group=5, width=128, kenc=Q4_0, venc=Q4_0, tokens=2048, context=2048, dtype=BF16),
        # the next chunk of a long prompt, wide heads, odd sizes
        attn("chunk 387 at 24100 bf16", heads=4, group=5, width=256, kenc=Q8_0, venc=Q4_0, tokens=387, context=24100, dtype=BF16),
        # one sampled token's log probability with the alternatives that an answer lists
        logp("logprobs 1 x 248320", rows=1, count=248320, k=20),
        # a scored prompt: every row of the head's logits
        logp("logprobs 509 x 248320", rows=509, count=248320, k=5),
    ]


def kv(name, op, heads, width, kenc, venc, tokens, context, dtype, sequences=1):
    return dict(name=name, op=op, sequences=sequences, heads=heads, width=width, kenc=kenc, venc=venc, tokens=tokens, context=context, dtype=dtype)


def attn(name, heads, group, width, kenc, venc, context, sequences=1, tokens=1, window=0, dtype=F32):
    return dict(name=name, op="attention", sequences=sequences, heads=heads, group=group, width=width, kenc=kenc, venc=venc, tokens=tokens, context=context, window=window,
                dtype=dtype)


def logp(name, rows, count, k):
    return dict(name=name, op="logprobs", rows=rows, count=count, k=k)


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["write", "read", "attention", "attention", "attention", "logprobs"])
    if op == "logprobs":
        rows = log(1, 500)
        c = logp("", rows, log(1000, 248320), rng.randint(0, 20))
    else:
        heads, width = rng.choice([(8, 128), (4, 256), (8, 64), (2, 128), (1, 256), (5, 128)])
        kenc, venc = rng.choice([(Q4_0, Q4_0), (Q8_0, Q8_0), (Q8_0, Q4_0), (Q4_0, Q8_0)])
        if op == "attention":
            form = rng.choice(["decode", "verify", "batch", "prompt"])
            sequences = log(2, 40) if form == "batch" else 1
            tokens = 1 if form == "decode" else log(2, 8) if form == "verify" else rng.randint(1, 3) if form == "batch" else log(9, 1500)
            context = log(1, 100000) if form in ("decode", "verify") else log(1, 8000) if form == "batch" else log(9, 12000)
            c = attn("", heads, rng.choice([1, 3, 4, 5, 8, 10]), width, kenc, venc, max(context, tokens), sequences, tokens, rng.choice([0, 0, 0, log(16, 8000)]),
                     BF16 if form == "prompt" and rng.random() < 0.7 else rng.choice([F32, F32, BF16]))
        else:
            sequences = rng.choice([1, 1, log(2, 16)])
            tokens = log(1, 24000 // sequences)
            c = kv("", op, heads, width, kenc, venc, tokens, tokens + rng.randint(0, 500), rng.choice([F32, BF16]), sequences)
    while work(c)["flops"] > 1.8e11:  # no more than the largest listed chunk
        c["tokens"] = max(1, c["tokens"] * 2 // 3)
    del c["name"]
    return c


def sessions(case):
    """(length, rows) of each sequence of an attention call. In a batch the first has ended and the second has a row fewer than the others."""
    s, t, n = case["sequences"], case["tokens"], case["context"]
    if s == 1:
        return [(n, t)]
    return [(max(t, -(-n * (i + 1) // s)), 0 if i == 0 else max(1, t - 1) if i == 1 else t) for i in range(s)]


# ---- inputs -------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    if case["op"] == "logprobs":
        state = logits_of(case, g)
    else:
        state = cache_of(case, g, seed)
    state["case"] = case
    if own:
        state["plan"] = Plan(state)  # what a program keeps between calls: the handle, its buffers, the recorded operators
    state.pop("raw", None)
    torch.cuda.synchronize()  # the library runs on a stream of its own
    return state


def logits_of(case, g):
    """Logits as a head writes them: a bulk, some rows with a few clear candidates, and on odd rows a mask over part of the vocabulary."""
    rows, count = case["rows"], case["count"]
    x = torch.randn(rows, count, generator=g, device=DEVICE) * 2.5
    at = torch.randint(0, count, (rows, 8), generator=g, device=DEVICE)
    x.scatter_add_(1, at, torch.rand(rows, 8, generator=g, device=DEVICE) * 16)
    x[1::2, count // 2: count // 2 + count // 9] = -math.inf
    x[2::4, : count // 7] = torch.finfo(torch.float32).min
    top = x.argmax(1)
    other = torch.randint(0, count, (rows,), generator=g, device=DEVICE)
    masked = x.gather(1, other[:, None])[:, 0] < -1e30
    tokens = torch.where((torch.rand(rows, generator=g, device=DEVICE) < 0.6) | masked, top, other)
    return {"logits": x, "tokens": tokens.to(torch.int32)}


def cache_of(case, g, seed):
    """Keys and values as projections write them (channels of unlike size, a few of them large), one span of rows for each sequence, and
    for the readers the quantized cache."""
    s, t, h, w, n = case["sequences"], case["tokens"], case["heads"], case["width"], case["context"]
    gain = torch.exp(torch.randn(2, 1, h, w, generator=g, device=DEVICE) * 0.4)
    rng = torch.Generator()
    rng.manual_seed(seed)
    slots = torch.randperm(s, generator=rng)
    if case["op"] == "attention":
        length, count = torch.tensor(sessions(case))[torch.randperm(s, generator=rng)].T
    else:
        length, count = torch.full((s,), n), torch.full((s,), t)
    spans = torch.stack([slots, length - count, count, torch.zeros(s, dtype=torch.long)], 1).to(torch.int32).to(DEVICE)
    state = {"spans": spans}
    if case["op"] == "write":
        # the fused rows of a projection: queries are not here, keys and values side by side, some floats between the rows
        state["rows"] = torch.randn(s * t, 2 * h * w + 4, generator=g, device=DEVICE)
        state["rows"][:, : 2 * h * w] *= gain.reshape(-1)
        return state
    raw = torch.randn(2, s, h, n, w, generator=g, device=DEVICE) * gain.reshape(2, 1, h, 1, w)  # [keys | values][slot][head][position][width]
    state["kcodes"], state["kscales"] = quantize(raw[0], case["kenc"])
    state["vcodes"], state["vscales"] = quantize(raw[1], case["venc"])
    if case["op"] == "attention":
        state["queries"] = torch.randn(s * t, h * case["group"] * w, generator=g, device=DEVICE) * 1.2
    if own:
        state["raw"] = raw
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return state["plan"].run()
    case = state["case"]
    if case["op"] == "logprobs":
        return plain_logprobs(state["logits"], state["tokens"], case["k"])
    if case["op"] == "write":
        h, w = case["heads"], case["width"]
        keys, values = (state["rows"][:, i * h * w: (i + 1) * h * w].reshape(-1, h, w) for i in (0, 1))
        out = [dequantize(*quantize(x, e)).to(dtype_of(case)).reshape(-1, h * w) for x, e in ((keys, case["kenc"]), (values, case["venc"]))]
        return {"keys": out[0], "values": out[1]}
    if case["op"] == "read":
        return {"keys": plain_read(state["kcodes"], state["kscales"], state["spans"], case), "values": plain_read(state["vcodes"], state["vscales"], state["spans"], case)}
    return plain_attention(state, case)


def dtype_of(case):
    return torch.bfloat16 if case["dtype"] == BF16 else torch.float32


def quantize(x, encoding):
    """Blocks of 32 along the last axis. Q8_0: d = amax / 127, code = round(x / d), halves away from zero. Q4_0: d = -m / 8 where m is the first
    value of the largest magnitude, code = min(15, trunc(x / d + 8.5)) standing for code - 8. The divisions are products with 1 / d; d is kept in 16 bits."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    if encoding == Q8_0:
        d = b.abs().amax(-1, keepdim=True) / 127
    else:
        d = b.gather(-1, b.abs().argmax(-1, keepdim=True)) / -8
    d = d.clamp(-65504.0, 65504.0)
    inverse = torch.where(d.half() == 0, 0.0, 1 / d)
    q = b * inverse
    if encoding == Q8_0:
        whole = torch.trunc(q)
        codes = (whole + torch.trunc((q - whole) * 2)).clamp(-127, 127)
    else:
        codes = torch.trunc(q + 8.5).clamp(0, 15) - 8
    return codes.to(torch.int8).reshape(x.shape), d.half().squeeze(-1)


def dequantize(codes, scales):
    return (codes.reshape(*scales.shape, 32).float() * scales.float()[..., None]).reshape(codes.shape)


def plain_read(codes, scales, spans, case):
    at = spans[:, 1, None].long() + torch.arange(case["tokens"], device=DEVICE)  # [sequence][row] -> position
    slot = spans[:, 0, None].long().expand_as(at)
    x = dequantize(codes[slot, :, at], scales[slot, :, at])  # [sequence][row][head][width]
    return x.reshape(-1, case["heads"] * case["width"]).to(dtype_of(case))


def plain_attention(state, case):
    s, t, h, g, w = case["sequences"], case["tokens"], case["heads"], case["group"], case["width"]
    spans = state["spans"].long()
    k = dequantize(state["kcodes"], state["kscales"])[spans[:, 0]]  # [sequence][head][position][width]
    v = dequantize(state["vcodes"], state["vscales"])[spans[:, 0]]
    q = state["queries"].reshape(s, t, h, g, w).permute(0, 2, 3, 1, 4).reshape(s, h, g * t, w)
    scores = (q @ k.transpose(2, 3)).reshape(s, h, g, t, -1) * w ** -0.5
    row = torch.arange(t, device=DEVICE)
    here = spans[:, 1, None] + row  # position of each row
    at = torch.arange(k.shape[2], device=DEVICE)
    seen = at <= here[..., None]
    if case["window"]:
        seen = seen & (at > here[..., None] - case["window"])
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (p.reshape(s, h, g * t, -1) @ v).reshape(s, h, g, t, w) / p.sum(-1, keepdim=True)
    live = (row < spans[:, 2, None])[:, None, None, :, None]  # rows behind a sequence's last stay as they were: zero
    return torch.where(live, out, 0.0).permute(0, 3, 1, 2, 4).reshape(s * t, h * g * w).to(dtype_of(case))


def plain_logprobs(logits, tokens, k):
    m = logits.amax(1, keepdim=True)
    e = torch.exp(logits - m)
    total = e.sum(1, keepdim=True)
    norm = m + torch.log(total)
    weighted = torch.where(e > 0, e * (logits - m), 0.0).sum(1, keepdim=True)
    out = {"logprobs": (logits.gather(1, tokens[:, None].long()) - m - torch.log(total))[:, 0], "entropy": (torch.log(total) - weighted / total)[:, 0]}
    if k:
        value, index = torch.sort(logits, dim=1, descending=True, stable=True)
        out["top"], out["top_logprobs"] = index[:, :k].to(torch.int32), value[:, :k] - norm
    return out


# ---- the library's calls ------------------------------------------------------------------------------------------------------

BACKEND = []


def backend():
    """One handle for the program, as a server keeps it."""
    if not BACKEND:
        from nuclis_b200 import Backend
        BACKEND.append(Backend(0))
    return BACKEND[0]


class Memory:
    """A buffer of the handle, and what torch reads it through: it lives as long as a tensor over it does."""

    def __init__(self, size):
        self.buffer = backend().create(size)
        self.__cuda_array_interface__ = {"shape": (size,), "typestr": "|u1", "data": (self.buffer.device_ptr, False), "version": 2}

    def __del__(self):
        backend().release(self.buffer)


class Plan:
    """A state's buffers on the handle and its recorded operators; torch sees the buffers without a copy."""

    def __init__(self, state):
        self.memory = {}  # of each buffer
        self.graph = None
        b = backend()
        case = state["case"]
        torch.cuda.synchronize()
        if case["op"] == "logprobs":
            rows, count, k = case["rows"], case["count"], case["k"]
            logits, tokens = self.given(state, "logits"), self.given(state, "tokens")
            logprobs, entropy = self.new((rows,)), self.new((rows,))
            self.out = {"logprobs": self.view(logprobs, (rows,)), "entropy": self.view(entropy, (rows,))}
            top = top_logprobs = None
            if k:
                top, top_logprobs = self.new((rows, k)), self.new((rows, k))
                self.out |= {"top": self.view(top, (rows, k), torch.int32), "top_logprobs": self.view(top_logprobs, (rows, k))}
            self.record(lambda: b.token_logprobs(logits, rows, count, count, tokens, logprobs, entropy, k, top, top_logprobs))
            return
        from nuclis_b200 import KvCache
        s, t, h, w = case["sequences"], case["tokens"], case["heads"], case["width"]
        shape = KvCache(slots=s, capacity=(case["context"] + 15) // 16 * 16, heads=h, width=w, key_encoding=case["kenc"], value_encoding=case["venc"])
        cache = self.buffer(shape.bytes)
        spans = self.given(state, "spans")
        size = 2 if case["dtype"] == BF16 else 4
        if case["op"] != "write":
            self.fill(cache, shape, state["raw"])
        if case["op"] == "attention":
            width = h * case["group"] * w
            queries, out = self.given(state, "queries"), self.buffer(s * t * width * size)
            self.out = self.view(out, (s * t, width), dtype_of(case))
            self.record(lambda: b.attention(cache, shape, spans, s, t, queries, width, h * case["group"], out, width, window=case["window"], out_dtype=case["dtype"]))
            return
        keys, values = self.buffer(s * t * h * w * size), self.buffer(s * t * h * w * size)
        self.out = {"keys": self.view(keys, (s * t, h * w), dtype_of(case)), "values": self.view(values, (s * t, h * w), dtype_of(case))}
        if case["op"] == "write":
            rows = self.given(state, "rows")
            stride, part = 2 * h * w + 4, h * w * 4

            def both():
                b.kv_write(cache, shape, spans, s, t, rows, stride, rows.slice(part, rows.len - part), stride)
                b.kv_read(cache, shape, spans, s, t, keys, h * w, values, h * w, out_dtype=case["dtype"])
            self.record(both)
        else:
            self.record(lambda: b.kv_read(cache, shape, spans, s, t, keys, h * w, values, h * w, out_dtype=case["dtype"]))

    def buffer(self, size):
        memory = Memory(size)
        self.memory[memory.buffer.id] = memory
        return memory.buffer

    def new(self, shape):
        return self.buffer(4 * math.prod(shape))

    def view(self, buffer, shape, dtype=torch.float32):
        return torch.as_tensor(self.memory[buffer.id], device=DEVICE).view(dtype).view(shape)

    def given(self, state, name):
        """The input's values in a buffer of the handle; the state keeps the tensor that shows them."""
        x = state[name]
        buffer = self.buffer(x.numel() * x.element_size())
        state[name] = self.view(buffer, x.shape, x.dtype).copy_(x)
        return buffer

    def fill(self, cache, shape, raw):
        """The keys and values of every slot and position, written as a program's prompts wrote them."""
        b = backend()
        _, s, h, n, w = raw.shape
        rows = self.buffer(2 * s * n * h * w * 4)
        self.view(rows, (2, s, n, h, w)).copy_(raw.transpose(2, 3))
        spans = self.buffer(s * 16)
        slot = torch.arange(s, device=DEVICE, dtype=torch.int32)
        self.view(spans, (s, 4), torch.int32).copy_(torch.stack([slot, slot * 0, slot * 0 + n, slot * 0], 1))
        torch.cuda.synchronize()
        half = s * n * h * w * 4
        b.begin()
        b.kv_write(cache, shape, spans, s, n, rows.slice(0, half), h * w, rows.slice(half, half), h * w)
        b.commit()
        del self.memory[rows.id], self.memory[spans.id]

    def record(self, operators):
        torch.cuda.synchronize()
        backend().begin()
        operators()
        self.graph = backend().commit_retain()

    def run(self):
        backend().graph_launch(self.graph)
        return self.out

    def __del__(self):
        if self.graph is not None:
            backend().graph_release(self.graph)


# ---- the work and the exact results ---------------------------------------------------------------------------------------------

def block_bytes(encoding, values):
    return values // 32 * (34 if encoding == Q8_0 else 18)


def work(case):
    if case["op"] == "logprobs":
        return {"bytes": 4 * case["rows"] * (case["count"] + 3 + 2 * case["k"]), "flops": 5 * case["rows"] * case["count"]}
    s, t, h, w, n = case["sequences"], case["tokens"], case["heads"], case["width"], case["context"]
    size = 2 if case["dtype"] == BF16 else 4
    if case["op"] != "attention":
        values = s * t * h * w
        quantized = block_bytes(case["kenc"], values) + block_bytes(case["venc"], values)
        read = quantized + 2 * values * size
        return {"bytes": read + (8 * values + quantized if case["op"] == "write" else 0) + 16 * s, "flops": 4 * values}
    pairs = keys = 0  # (row, key) pairs, and the keys that some row of a sequence sees
    for length, count in sessions(case):
        window = case["window"] or length
        keys += length - max(0, length - count - window + 1) if count else 0
        pairs += sum(min(window, length - count + i + 1) for i in range(count))
    cache = (block_bytes(case["kenc"], h * w) + block_bytes(case["venc"], h * w)) * keys
    return {"bytes": cache + s * t * h * case["group"] * w * (4 + size) + 16 * s, "flops": 4 * w * h * case["group"] * pairs}


def exact(case, seed):
    """The definitions in 64 bits. The codes of a quantized row are a matter of its 32-bit rule, so they are found with that rule; what they stand for is not rounded."""
    state = prepare(case, seed)
    if case["op"] == "logprobs":
        return exact_logprobs(state, case)
    if case["op"] == "write":
        h, w = case["heads"], case["width"]
        return {"keys": exact_blocks(state["rows"][:, : h * w], case["kenc"]), "values": exact_blocks(state["rows"][:, h * w: 2 * h * w], case["venc"])}
    both = [(state[c].double().unflatten(-1, (-1, 32)) * state[d].double().unsqueeze(-1)).flatten(-2) for c, d in (("kcodes", "kscales"), ("vcodes", "vscales"))]
    spans = state["spans"].tolist()
    t, h, w = case["tokens"], case["heads"], case["width"]
    if case["op"] == "read":
        parts = [torch.cat([x[slot, :, first: first + t].transpose(0, 1).reshape(t, h * w) for slot, first, _, _ in spans]) for x in both]
        return {"keys": parts[0], "values": parts[1]}
    g = case["group"]
    out = torch.zeros(case["sequences"], t, h, g, w, dtype=torch.float64, device=DEVICE)
    queries = state["queries"].double().reshape(case["sequences"], t, h, g, w)
    for i, (slot, first, count, _) in enumerate(spans):
        for begin in range(0, count, 256):  # rows in pieces, so that the scores stay small
            rows = range(begin, min(begin + 256, count))
            low = max(0, first + rows[0] - case["window"] + 1) if case["window"] else 0
            high = first + rows[-1] + 1
            where = torch.arange(low, high, device=DEVICE)[None]
            pos = torch.arange(first + rows[0], high, device=DEVICE)[:, None]
            hidden = where > pos
            if case["window"]:
                hidden |= where <= pos - case["window"]
            for j in range(h):
                z = torch.einsum("tgw,nw->gtn", queries[i, rows[0]: rows[-1] + 1, j], both[0][slot, j, low:high]) / math.sqrt(w)
                p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
                out[i, rows[0]: rows[-1] + 1, j] = torch.einsum("gtn,nw->tgw", p, both[1][slot, j, low:high])
    return out.reshape(case["sequences"] * t, h * g * w)


def exact_blocks(rows, encoding):
    x = rows.reshape(rows.shape[0], -1, 32)
    if encoding == Q8_0:
        d = (x.abs().max(-1, keepdim=True).values / 127).clamp(max=65504.0)
        q = x * torch.where(d.half() > 0, 1 / d, 0.0)
        codes = (torch.sign(q) * torch.floor(q.abs().double() + 0.5)).clamp(-127, 127)
    else:
        low, high = x.min(-1, keepdim=True), x.max(-1, keepdim=True)
        first_low = low.indices < high.indices
        m = torch.where((-low.values > high.values) | ((-low.values == high.values) & first_low), low.values, high.values)
        d = (m / -8).clamp(-65504.0, 65504.0)
        q = x * torch.where(d.half() != 0, 1 / d, 0.0)
        codes = torch.floor(q + 8.5).clamp(0, 15).double() - 8
    return (codes.double() * d.half().double()).reshape(rows.shape)


def exact_logprobs(state, case):
    pieces = []
    for x, token in zip(state["logits"].split(64), state["tokens"].split(64)):
        z = torch.log_softmax(x.double(), 1)
        piece = [z.gather(1, token[:, None].long())[:, 0], -torch.special.xlogy(z.exp(), z.exp()).sum(1)]
        if case["k"]:
            index = torch.sort(x, dim=1, descending=True, stable=True).indices[:, : case["k"]]
            piece += [index.to(torch.int32), z.gather(1, index)]
        pieces.append(piece)
    return dict(zip(("logprobs", "entropy", "top", "top_logprobs"), (torch.cat(p) for p in zip(*pieces))))
