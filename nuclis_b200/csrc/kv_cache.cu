// Writing rows of keys and values into the quantized cache, and reading them back. Both are one pass over the rows:
// bound by memory for a prompt, by the launch for a single row.
//
// The rule of a block of 32 (GGUF's, in F32 arithmetic): Q8_0 d = amax * (1 / 127), code = round(x * (1 / d)) with halves away
// from zero; Q4_0 d = m / -8 with m the first value of the largest magnitude, code = min(15, trunc(x * (1 / d) + 8.5)).
// The stored scale is d rounded to f16. A block whose scale rounds to zero stores zeros; one whose scale passes the f16
// range stores the largest scale and saturated codes; one that holds a NaN or an infinity stores a NaN scale, so that it
// reads back as NaN and cannot pass for data.
#include <cuda_bf16.h>

#include "kernels.hpp"
#include "kv_layout.cuh"
#include "launch.cuh"

namespace nu {

namespace {

constexpr int KV_THREADS = 128;

// Eight lanes hold a block, four values each. Returns this lane's four codes without sign (one a byte), and the scale.
template <bool Q8>
__device__ __forceinline__ uint32_t quantize4(const float x[4], float &scale) {
    float top = 0.0f;  // the value of the largest magnitude, the first of equals
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bad |= !isfinite(x[i]);
        if (fabsf(x[i]) > fabsf(top)) top = x[i];
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, top, o);
        const bool lower = (threadIdx.x & o) != 0;  // the other lane holds earlier values
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
        if (lower ? fabsf(other) >= fabsf(top) : fabsf(other) > fabsf(top)) top = other;
    }
    float d = Q8 ? __fmul_rn(fabsf(top), 1.0f / 127.0f) : top * -0.125f;
    d = fminf(fmaxf(d, -65504.0f), 65504.0f);
    scale = bad ? NAN : d;
    const float inverse = bad || __half2float(__float2half_rn(d)) == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = bad ? 0.0f : __fmul_rn(x[i], inverse);
        const int c = Q8 ? min(max((int)roundf(q), -127), 127) + 128 : min(max((int)__fadd_rn(q, 8.5f), 0), 15);
        codes |= (uint32_t)c << (8 * i);
    }
    return codes;
}

struct WriteParams {
    KvView c;
    const KvSpan *spans;
    uint32_t sequences, tokens, pieces;  // a piece: 128 consecutive values of a row, one warp's
    const float *rows[2];                // keys, values
    size_t stride[2];
};

__device__ __forceinline__ uint32_t nibbles(uint32_t bytes) { return (bytes & 15u) | (bytes >> 4 & 0xf0u) | (bytes >> 8 & 0xf00u) | (bytes >> 12 & 0xf000u); }

template <bool VALUES, bool Q8>
__device__ __forceinline__ void write_piece(const WriteParams &p, const float *row, uint32_t piece, uint32_t slot, uint32_t pos) {
    const uint32_t lane = threadIdx.x & 31, e = piece * 128 + lane * 4, width = p.c.l.width;
    const bool live = e < p.c.heads * width;  // blocks are whole: the eight lanes of one are live together
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
        if ((uintptr_t)(row + e) % 16 == 0) {
            const float4 v = *(const float4 *)(row + e);
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = row[e + i];
        }
    }
    float scale;
    const uint32_t codes = quantize4<Q8>(x, scale);
    const uint32_t head = e / width, dim = e % width, b = dim / 32, at = pos % KV_GRANULE;
    uint8_t *g = live ? kv_head(p.c, slot, head) + (size_t)(pos / KV_GRANULE) * p.c.l.bytes : nullptr;
    const uint32_t near = __shfl_xor_sync(0xffffffffu, codes, VALUES ? 2 : 1);  // keys: the other half of eight dimensions; values: the other nibbles
    if (!live) return;
    if (dim % 32 == 0) *(__half *)(g + (VALUES ? p.c.l.v_scales : p.c.l.k_scales) + (at * p.c.l.blocks + b) * 2) = __float2half_rn(scale);
    if (VALUES) {
        if (Q8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) g[kv_value_byte(p.c.l, at, dim + i)] = (uint8_t)(codes >> (8 * i));
        } else if (!(dim & 8)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) g[kv_value_byte(p.c.l, at, dim + i)] = (uint8_t)((codes >> (8 * i) & 15u) | (near >> (8 * i) & 15u) << 4);
        }
    } else {
        const uint32_t t = dim % 32 / 8, second = dim / 4 % 2;
        if (Q8) {  // bytes 0,4,1,5 by the lane of dimensions 0..3, bytes 2,6,3,7 by the other
            const uint32_t low = second ? near : codes, high = second ? codes : near;
            *(uint32_t *)(g + kv_key_word(p.c.l, at, b, t, second)) = __byte_perm(low, high, second ? 0x7362 : 0x5140);
        } else if (!second) {
            *(uint32_t *)(g + kv_key_word(p.c.l, at, b, t, 0)) = nibbles(codes) | nibbles(near) << 16;
        }
    }
}

// One warp a piece of a row. Where two spans of a call cover the same position, the row of the later span is written.
__global__ void __launch_bounds__(KV_THREADS) kv_write_kernel(const WriteParams p) {
    wait_for_previous_operator();
    const uint32_t lane = threadIdx.x & 31;
    const size_t item = (size_t)blockIdx.x * (KV_THREADS / 32) + threadIdx.x / 32;
    const uint32_t which = (uint32_t)(item % 2), piece = (uint32_t)(item / 2 % p.pieces);
    const size_t r = item / 2 / p.pieces;
    if (r >= (size_t)p.sequences * p.tokens) return;
    const uint32_t sequence = (uint32_t)(r / p.tokens), i = (uint32_t)(r % p.tokens);
    const KvSpan span = kv_span(p.c, p.spans, sequence, p.tokens);
    if (i >= span.count) return;
    const uint32_t pos = span.first + i;
    for (uint32_t later = sequence + 1; later < p.sequences; later += 32) {
        bool covered = false;
        if (later + lane < p.sequences) {
            const KvSpan s = kv_span(p.c, p.spans, later + lane, p.tokens);
            covered = s.slot == span.slot && pos >= s.first && pos - s.first < s.count;
        }
        if (__any_sync(0xffffffffu, covered)) return;
    }
    const float *row = p.rows[which] + r * p.stride[which];
    if (which) {
        if (p.c.l.v8) write_piece<true, true>(p, row, piece, span.slot, pos);
        else write_piece<true, false>(p, row, piece, span.slot, pos);
    } else {
        if (p.c.l.k8) write_piece<false, true>(p, row, piece, span.slot, pos);
        else write_piece<false, false>(p, row, piece, span.slot, pos);
    }
}

struct ReadParams {
    KvView c;
    const KvSpan *spans;
    uint32_t sequences, tokens, pieces;
    void *rows[2];
    size_t stride[2];
    bool bf16;
};

// One warp a piece of a row, a lane four values of it.
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const ReadParams p) {
    wait_for_previous_operator();
    const uint32_t lane = threadIdx.x & 31;
    const size_t item = (size_t)blockIdx.x * (KV_THREADS / 32) + threadIdx.x / 32;
    const uint32_t which = (uint32_t)(item % 2), piece = (uint32_t)(item / 2 % p.pieces);
    const size_t r = item / 2 / p.pieces;
    if (r >= (size_t)p.sequences * p.tokens) return;
    const uint32_t sequence = (uint32_t)(r / p.tokens), i = (uint32_t)(r % p.tokens);
    const KvSpan span = kv_span(p.c, p.spans, sequence, p.tokens);
    const uint32_t e = piece * 128 + lane * 4, width = p.c.l.width;
    if (i >= span.count || e >= p.c.heads * width) return;
    const uint32_t pos = span.first + i, at = pos % KV_GRANULE, head = e / width, dim = e % width, b = dim / 32;
    const uint8_t *g = kv_head(p.c, span.slot, head) + (size_t)(pos / KV_GRANULE) * p.c.l.bytes;
    const float d = __half2float(*(const __half *)(g + (which ? p.c.l.v_scales : p.c.l.k_scales) + (at * p.c.l.blocks + b) * 2));
    float x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        int code;
        if (which) {
            const uint32_t byte = g[kv_value_byte(p.c.l, at, dim + k)];
            code = p.c.l.v8 ? (int)byte - 128 : (int)(byte >> (dim & 8 ? 4 : 0) & 15u) - 8;
        } else if (p.c.l.k8) {
            const uint32_t w = *(const uint32_t *)(g + kv_key_word(p.c.l, at, b, dim % 32 / 8, k / 2));
            code = (int)(w >> (8 * (k % 2 * 2 + dim / 4 % 2)) & 255u) - 128;
        } else {
            const uint32_t w = *(const uint32_t *)(g + kv_key_word(p.c.l, at, b, dim % 32 / 8, 0));
            code = (int)(w >> (4 * (dim % 8 + k)) & 15u) - 8;
        }
        x[k] = __fmul_rn(d, (float)code);
    }
    const size_t out = r * p.stride[which] + e;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (p.bf16) ((__nv_bfloat16 *)p.rows[which])[out + k] = __float2bfloat16_rn(x[k]);
        else ((float *)p.rows[which])[out + k] = x[k];
    }
}

KvView view(const KvCacheJob &c) { return {c.base, kv_layout(c.width, c.k8, c.v8), c.slots, c.heads, c.capacity / KV_GRANULE, c.status}; }

}  // namespace

int launch_kv_write(cudaStream_t s, const KvCacheJob &c, const void *spans, uint32_t sequences, uint32_t tokens, const float *keys, size_t key_stride,
                    const float *values, size_t value_stride) {
    WriteParams p{view(c), (const KvSpan *)spans, sequences, tokens, (c.heads * c.width + 127) / 128, {keys, values}, {key_stride, value_stride}};
    const size_t items = (size_t)sequences * tokens * p.pieces * 2;
    launch_after_previous(kv_write_kernel, dim3((unsigned)((items + KV_THREADS / 32 - 1) / (KV_THREADS / 32))), dim3(KV_THREADS), s, p);
    return 1;
}

int launch_kv_read(cudaStream_t s, const KvCacheJob &c, const void *spans, uint32_t sequences, uint32_t tokens, void *keys, size_t key_stride, void *values,
                   size_t value_stride, bool bf16) {
    ReadParams p{view(c), (const KvSpan *)spans, sequences, tokens, (c.heads * c.width + 127) / 128, {keys, values}, {key_stride, value_stride}, bf16};
    const size_t items = (size_t)sequences * tokens * p.pieces * 2;
    launch_after_previous(kv_read_kernel, dim3((unsigned)((items + KV_THREADS / 32 - 1) / (KV_THREADS / 32))), dim3(KV_THREADS), s, p);
    return 1;
}

}  // namespace nu
