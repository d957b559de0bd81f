"""Plain forms of the cache and attention operators: the quantization rule in the F32 arithmetic it is defined in, everything
else in 64 bits."""
import numpy as np

from nuclis_b200 import encoding as enc


def quantize(x, encoding):
    """Rows of whole 32-value blocks -> (codes, f16 scales) by GGUF's rule, with this library's answers where that has none."""
    x = np.asarray(x, dtype=np.float32)
    b = x.reshape(*x.shape[:-1], -1, 32)
    f = np.float32
    with np.errstate(all="ignore"):
        if encoding == enc.Q8_0:
            d = (np.max(np.abs(b), axis=-1) * (f(1) / f(127))).astype(np.float32)
        else:
            at = np.argmax(np.abs(b), axis=-1)
            d = (np.take_along_axis(b, at[..., None], -1)[..., 0] / f(-8)).astype(np.float32)
        d = np.clip(d, f(-65504), f(65504))
        bad = ~np.isfinite(b).all(-1)
        half = d.astype(np.float16)
        inverse = np.where(bad | (half == 0), f(0), f(1) / d).astype(np.float32)
        q = (np.where(bad[..., None], f(0), b) * inverse[..., None]).astype(np.float32)
        if encoding == enc.Q8_0:
            whole = np.trunc(q)
            codes = np.clip(whole + np.where(np.abs(q - whole) >= 0.5, np.sign(q), 0), -127, 127)
        else:
            codes = np.clip(np.trunc((q + f(8.5)).astype(np.float32)), 0, 15) - 8
    half = np.where(bad, np.float16(np.nan), half)
    return codes.reshape(x.shape).astype(np.int8), half


def dequantize(codes, scales):
    return (codes.reshape(*scales.shape, 32).astype(np.float64) * scales.astype(np.float64)[..., None]).reshape(codes.shape)


def stored(x, encoding):
    """What a cache gives back for the values x, in 64 bits."""
    return dequantize(*quantize(x, encoding))


def attention(q, k, v, first, group, scale=None, window=0):
    """q [rows][heads][width], k and v [positions][kv heads][width]; row i stands at position first + i. 64 bits."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    rows, heads, width = q.shape
    scale = 1 / np.sqrt(width) if scale is None else scale
    out = np.zeros_like(q)
    for i in range(rows):
        p = first + i
        low = max(0, p - window + 1) if window else 0
        for h in range(heads):
            s = k[low:p + 1, h // group] @ q[i, h] * scale
            e = np.exp(s - s.max())
            out[i, h] = e @ v[low:p + 1, h // group] / e.sum()
    return out
