// Writing rows of keys and values into the quantized cache, and reading them back. Both are one pass over the rows:
// bound by memory for a prompt, by the launch for a single row.
//
// The rule of a block of 32 (in F32; GGUF's but for Q8_0's division by 127, here a product with the reciprocal: no slow division in a warp's chain
// of dependent steps, and d within 2^-23 of the quotient): Q8_0 d = amax * (1 / 127), code = round(x * (1 / d)) with halves away
// from zero; Q4_0 d = m / -8 with m the first value of the largest magnitude, code = min(15, trunc(x * (1 / d) + 8.5)).
// The stored scale is d rounded to f16. A block whose scale rounds to zero stores zeros; one whose scale passes the f16
// range stores the largest scale and saturated codes; one that holds a NaN or an infinity stores a NaN scale, so that it
// reads back as NaN and cannot pass for data.
//
// Measured (8 heads of width 128, against a copy's 6.46 TB/s): 65,536 rows of Q4_0 read to BF16 66 us, 5.2 TB/s; 4,096 rows written as
// Q8_0 / Q4_0 and read back to F32 23 us, 3.4 TB/s, of which the write waits for its own instructions more than for memory; one row
// written and read back 6.3 us, which is two launches and two chains of dependent loads.
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
    // magnitudes as integers: their order is the floats', and NaN and infinity come out on top
    uint32_t a[4], own = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = __float_as_uint(x[i]) & 0x7fffffffu;
        own = max(own, a[i]);
    }
    uint32_t top = own;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const bool bad = top >= 0x7f800000u;
    float d;
    if (Q8) {
        d = __fmul_rn(__uint_as_float(top), 1.0f / 127.0f);
    } else {  // with the sign of the first value of that magnitude
        const float first = a[0] == top ? x[0] : a[1] == top ? x[1] : a[2] == top ? x[2] : x[3];
        const uint32_t group = threadIdx.x & 24u, have = __ballot_sync(0xffffffffu, own == top) >> group & 0xffu;
        d = __shfl_sync(0xffffffffu, first, group + __ffs(have) - 1) * -0.125f;
    }
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

__device__ __forceinline__ uint32_t nibbles(uint32_t bytes) { return (bytes & 15u) | (bytes >> 4 & 0xf0u) | (bytes >> 8 & 0xf00u) | (bytes >> 12 & 0xf000u); }

// Both kernels give one warp the share of a granule (16 positions) that a piece of up to 128 dimensions of one head's keys
// or values has, of one sequence: the rows' side is then read or written in whole 512-byte runs, and so is the cache's,
// whose order puts four positions into one word of the values. A granule that the span covers in part is written byte by
// byte where a word has other positions in it.
struct Item {
    KvSpan span;
    uint32_t sequence, granule, head, dim0, dims;  // dimensions [dim0, dim0 + dims) of the head
    uint32_t which;                                // 0: keys, 1: values
    uint32_t live;                                 // bit i: position i of the granule is in the span
};

struct RowsParams {
    KvView c;
    const KvSpan *spans;
    uint32_t sequences, tokens, pieces;  // pieces of a head's width
    uint32_t granules;                   // that a span of `tokens` rows can touch
    void *rows[2];                       // keys, values
    size_t stride[2];
};

// (The host's limit on a call's rows keeps the count of items below 2^32.)
__device__ __forceinline__ bool item_of(const RowsParams &p, uint32_t index, Item &it) {
    it.which = index & 1;
    index >>= 1;
    it.dim0 = index % p.pieces * 128;
    index /= p.pieces;
    it.head = index % p.c.heads;
    index /= p.c.heads;
    it.granule = index % p.granules;
    it.sequence = index / p.granules;
    if (it.sequence >= p.sequences) return false;
    it.dims = min(128u, p.c.l.width - it.dim0);
    it.span = kv_span(p.c, p.spans, it.sequence, p.tokens);
    if (it.span.count == 0) return false;
    it.granule += it.span.first / KV_GRANULE;
    const uint32_t p0 = it.granule * KV_GRANULE, end = it.span.first + it.span.count;
    if (p0 >= end) return false;
    const uint32_t low = it.span.first > p0 ? it.span.first - p0 : 0, high = min(KV_GRANULE, end - p0);
    it.live = (0xffffu >> (16 - high)) & (0xffffu << low);
    return true;
}

// A 4 x 4 transposition of bytes: word i of the result has byte i of each of the four words, in their order.
__device__ __forceinline__ void transpose_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&out)[4]) {
    const uint32_t ab = __byte_perm(a, b, 0x5140), cd = __byte_perm(c, d, 0x5140), ab2 = __byte_perm(a, b, 0x7362), cd2 = __byte_perm(c, d, 0x7362);
    out[0] = __byte_perm(ab, cd, 0x5410);
    out[1] = __byte_perm(ab, cd, 0x7632);
    out[2] = __byte_perm(ab2, cd2, 0x5410);
    out[3] = __byte_perm(ab2, cd2, 0x7632);
}

constexpr int KV_WARPS = KV_THREADS / 32;

// FULL: the piece has 128 dimensions and the codes lie in vectors of 16 bytes (widths of whole 128s), so that every place is a
// matter of shifts (65,536 rows of width 128 read: 94 us without, 66 with it; 4,096 written and read 38 and 24).
// The second half of writing values: the rows' codes in `words` ([position][lane], four a word) become the cache's words.
template <bool Q8, bool FULL>
__device__ __forceinline__ void transpose_item(const KvLayout &l, const Item &it, uint8_t *g, uint32_t (&words)[512]) {
    const uint32_t lane = threadIdx.x & 31, mine = lane * 4, dims = FULL ? 128 : it.dims;
    const bool live = FULL || mine < dims;
    // this lane's words: four dimensions (four codes a byte of theirs, or with the partner's as nibbles), four groups of positions
    uint32_t codes[KV_GRANULE];
#pragma unroll
    for (uint32_t at = 0; at < KV_GRANULE; ++at) codes[at] = words[at * 32 + lane];
    __syncwarp();
    const uint32_t per = Q8 ? dims / 8 : dims / 16;  // words of a lane slot
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
        uint32_t c[4];
        transpose_bytes(codes[2 * tt], codes[2 * tt + 1], codes[8 + 2 * tt], codes[9 + 2 * tt], c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w = c[i];
            if (!Q8) {
                w = __byte_perm(w, 0, 0x3120) & 0x0f0f0f0fu;  // 2t, 8 + 2t, 2t + 1, 9 + 2t
                w |= __shfl_xor_sync(0xffffffffu, w, 2) << 4;
            }
            const uint32_t word = mine / (Q8 ? 8 : 16), slot = ((mine + i) % 8) * 4 + tt;
            // vectors of four words a slot, as the cache keeps them
            if (live && (Q8 || !(mine & 8))) words[word / 4 * 128 + slot * 4 + word % 4] = w;
        }
    }
    __syncwarp();
    const uint32_t word0 = Q8 ? it.dim0 / 8 : it.dim0 / 16;
    if (it.live == 0xffffu && (FULL || (l.v_vec == 16 && per % 4 == 0))) {
#pragma unroll
        for (uint32_t v = 0; v < (Q8 ? 4 : 2); ++v)
            if (FULL || v < per / 4) *(uint4 *)(g + l.v_codes + (word0 / 4 + v) * 512 + lane * 16) = *(const uint4 *)&words[v * 128 + lane * 4];
    } else {
        const uint32_t tt = lane % 4;
#pragma unroll 1
        for (uint32_t w = 0; w < per; ++w) {
            const uint32_t x = words[w / 4 * 128 + lane * 4 + w % 4];
            uint8_t *dst = g + l.v_codes + kv_word(FULL ? 16 : l.v_vec, lane, word0 + w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t at = Q8 ? 2 * tt + (i & 1) + (i >> 1) * 8 : 2 * tt + (i >> 1) + (i & 1) * 8;
                if (it.live >> at & 1u) dst[i] = (uint8_t)(x >> (8 * i));
            }
        }
    }
}

template <bool VALUES, bool Q8, bool FULL>
__device__ __forceinline__ void write_item(const RowsParams &p, const Item &it, uint32_t (&words)[512], __half (&scales)[64]) {
    const KvLayout &l = p.c.l;
    const uint32_t lane = threadIdx.x & 31, mine = lane * 4, dims = FULL ? 128 : it.dims;
    const bool live = FULL || mine < dims;  // blocks are whole: the eight lanes of one are live together
    const uint32_t dim = it.dim0 + mine, b = dim / 32;
    // row of position 0 of the granule, before the rows' start where the span begins inside it; only live positions are read
    const float *row0 = (const float *)p.rows[VALUES] + ((ptrdiff_t)it.sequence * p.tokens + (ptrdiff_t)it.granule * KV_GRANULE - it.span.first) * (ptrdiff_t)p.stride[VALUES] +
                        (size_t)it.head * l.width + dim;
    uint8_t *g = kv_head(p.c, it.span.slot, it.head) + (size_t)it.granule * l.bytes;
    const bool aligned = ((uintptr_t)row0 | p.stride[VALUES] * 4) % 16 == 0;
    const uint32_t t = dim % 32 / 8, second = dim / 4 % 2;
    // Four positions at a time, their loads together; not unrolled further: a warp runs this once, and fetching the code was
    // what it waited for when it was 16 positions long.
#pragma unroll 1
    for (uint32_t at0 = 0; at0 < KV_GRANULE; at0 += 4) {
        if (!(it.live >> at0 & 15u)) continue;
        float x[4][4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.0f;
            if ((it.live >> (at0 + i) & 1u) && live) {
                const float *row = row0 + (ptrdiff_t)(at0 + i) * (ptrdiff_t)p.stride[VALUES];
                if (aligned) {
                    const float4 v = __ldcs((const float4 *)row);
                    x[i][0] = v.x; x[i][1] = v.y; x[i][2] = v.z; x[i][3] = v.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[i][k] = row[k];
                }
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t at = at0 + i;
            if (!(it.live >> at & 1u)) continue;  // the same for the whole warp
            float scale;
            const uint32_t codes = quantize4<Q8>(x[i], scale);
            if (lane % 8 == 0 && live) scales[at * 4 + lane / 8] = __float2half_rn(scale);
            if (VALUES) {
                words[at * 32 + lane] = codes;
            } else {
                const uint32_t near = __shfl_xor_sync(0xffffffffu, codes, 1);  // the other half of eight dimensions
                uint32_t *dst = (uint32_t *)(g + kv_key_word(l, FULL ? 16 : l.k_vec, at, b, t, Q8 ? second : 0));
                if (live && Q8) {  // bytes 0,4,1,5 by the lane of dimensions 0..3, bytes 2,6,3,7 by the other
                    const uint32_t low = second ? near : codes, high = second ? codes : near;
                    *dst = __byte_perm(low, high, second ? 0x7362 : 0x5140);
                } else if (live && !second) {
                    *dst = nibbles(codes) | nibbles(near) << 16;
                }
            }
        }
    }
    __syncwarp();
    uint8_t *gs = g + (VALUES ? l.v_scales : l.k_scales);
    if (it.live == 0xffffu && FULL) {  // two blocks a word, two words a position
        *(uint32_t *)(gs + lane / 2 * l.blocks * 2 + it.dim0 / 16 + lane % 2 * 4) = ((const uint32_t *)scales)[lane];
    } else {
        const uint32_t blocks = dims / 32;
        for (uint32_t i = lane; i < KV_GRANULE * blocks; i += 32)
            if (it.live >> (i / blocks) & 1u) ((__half *)gs)[i / blocks * l.blocks + it.dim0 / 32 + i % blocks] = scales[i / blocks * 4 + i % blocks];
    }
    if (VALUES) transpose_item<Q8, FULL>(l, it, g, words);
}

__global__ void __launch_bounds__(KV_THREADS) kv_write_kernel(const RowsParams p) {
    __shared__ __align__(16) uint32_t words[KV_WARPS][512];
    __shared__ __align__(16) __half scales[KV_WARPS][64];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    wait_for_previous_operator();
    Item it;
    if (!item_of(p, blockIdx.x * KV_WARPS + warp, it)) return;
    // where two spans of a call cover the same position, the row of the later span is written
    for (uint32_t later = it.sequence + 1; later < p.sequences; later += 32) {
        uint32_t covered = 0;
        if (later + lane < p.sequences) {
            const KvSpan s = kv_span(p.c, p.spans, later + lane, p.tokens);
            if (s.count && s.slot == it.span.slot)
                for (uint32_t i = 0; i < KV_GRANULE; ++i) covered |= (uint32_t)(it.granule * KV_GRANULE + i >= s.first && it.granule * KV_GRANULE + i - s.first < s.count) << i;
        }
        it.live &= ~__reduce_or_sync(0xffffffffu, covered);
    }
    const bool full = p.c.l.width % 128 == 0;
    if (it.which) {
        if (p.c.l.v8) full ? write_item<true, true, true>(p, it, words[warp], scales[warp]) : write_item<true, true, false>(p, it, words[warp], scales[warp]);
        else full ? write_item<true, false, true>(p, it, words[warp], scales[warp]) : write_item<true, false, false>(p, it, words[warp], scales[warp]);
    } else {
        if (p.c.l.k8) full ? write_item<false, true, true>(p, it, words[warp], scales[warp]) : write_item<false, true, false>(p, it, words[warp], scales[warp]);
        else full ? write_item<false, false, true>(p, it, words[warp], scales[warp]) : write_item<false, false, false>(p, it, words[warp], scales[warp]);
    }
}

// A code without sign, placed in the low bits of 2^23, less 2^23 and its offset: exact, and the two operations run at four times a
// conversion's rate.
template <bool Q8>
__device__ __forceinline__ float code_value(uint32_t code) { return __uint_as_float(code | 0x4b000000u) - (Q8 ? 8388736.0f : 8388616.0f); }

template <typename T>
__device__ __forceinline__ T out_value(float x);
template <>
__device__ __forceinline__ float out_value<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 out_value<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Decoded rows of a piece, padded so that the values' scattered stores meet no bank twice.
template <typename T>
struct Staged {
    static constexpr int ROW = 128 + 16 / sizeof(T);
    T x[KV_GRANULE][ROW];
};

template <bool VALUES, bool Q8, bool FULL, typename T>
__device__ __forceinline__ void read_item(const RowsParams &p, const Item &it, Staged<T> &st) {
    const KvLayout &l = p.c.l;
    const uint32_t lane = threadIdx.x & 31, slot = lane / 4, t = lane % 4, b0 = it.dim0 / 32, dims = FULL ? 128 : it.dims;
    const uint8_t *g = kv_head(p.c, it.span.slot, it.head) + (size_t)it.granule * l.bytes;
    const __half *scales = (const __half *)(g + (VALUES ? l.v_scales : l.k_scales)) + b0;
    if (VALUES) {
        constexpr int PER = Q8 ? 4 : 2;  // words of a block
        const uint8_t *codes = g + l.v_codes;
#pragma unroll
        for (uint32_t b = 0; b < 4; ++b) {
            if (!FULL && b >= dims / 32) break;
            float d[4];  // of positions 2t, 2t + 1, 8 + 2t, 9 + 2t
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = __half2float(scales[(2 * t + (i & 1) + (i >> 1) * 8) * l.blocks + b]);
#pragma unroll
            for (int w = 0; w < PER; ++w) {
                const uint32_t word = *(const uint32_t *)(codes + kv_word(FULL ? 16 : l.v_vec, lane, (b0 + b) * PER + w));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t at = 2 * t + (i & 1) + (i >> 1) * 8;
                    if (Q8) {
                        st.x[at][b * 32 + w * 8 + slot] = out_value<T>(__fmul_rn(d[i], code_value<true>(__byte_perm(word, 0u, 0x4440 + i))));
                    } else {
                        const uint32_t byte = word >> (8 * ((i & 1) * 2 + (i >> 1)));
                        st.x[at][b * 32 + w * 16 + slot] = out_value<T>(__fmul_rn(d[i], code_value<false>(byte & 15u)));
                        st.x[at][b * 32 + w * 16 + 8 + slot] = out_value<T>(__fmul_rn(d[i], code_value<false>(byte >> 4 & 15u)));
                    }
                }
            }
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) {
            const uint32_t at = j * 8 + slot;
#pragma unroll
            for (uint32_t b = 0; b < 4; ++b) {
                if (!FULL && b >= dims / 32) break;
                const float d = __half2float(scales[at * l.blocks + b]);
                const uint32_t w0 = *(const uint32_t *)(g + kv_key_word(l, FULL ? 16 : l.k_vec, at, b0 + b, t, 0));
                const uint32_t w1 = Q8 ? *(const uint32_t *)(g + kv_key_word(l, FULL ? 16 : l.k_vec, at, b0 + b, t, 1)) : 0u;
                alignas(16) T x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t code = Q8 ? __byte_perm(i % 4 < 2 ? w0 : w1, 0u, 0x4440 + i % 2 * 2 + i / 4) : w0 >> (4 * i) & 15u;
                    x[i] = out_value<T>(__fmul_rn(d, code_value<Q8>(code)));
                }
#pragma unroll
                for (int v = 0; v < (int)sizeof(x) / 16; ++v) *(uint4 *)((uint8_t *)&st.x[at][b * 32 + t * 8] + v * 16) = ((const uint4 *)x)[v];
            }
        }
    }
    __syncwarp();
    // the rows, as whole runs
    T *row0 = (T *)p.rows[VALUES] + ((ptrdiff_t)it.sequence * p.tokens + (ptrdiff_t)it.granule * KV_GRANULE - it.span.first) * (ptrdiff_t)p.stride[VALUES] +
              (size_t)it.head * l.width + it.dim0;
    constexpr uint32_t V = 16 / sizeof(T);
    const uint32_t lanes = dims / V;  // vectors of a row
    if (((uintptr_t)row0 | p.stride[VALUES] * sizeof(T)) % 16 == 0) {
        if (FULL) {
            constexpr uint32_t LANES = 128 / V, TURN = 32 / LANES;  // rows a turn
            T *dst = row0 + (ptrdiff_t)(lane / LANES) * (ptrdiff_t)p.stride[VALUES] + lane % LANES * V;
#pragma unroll
            for (uint32_t at = 0; at < KV_GRANULE; at += TURN) {
                const uint32_t r = at + lane / LANES;
                if (it.live >> r & 1u) __stcs((uint4 *)dst, *(const uint4 *)&st.x[r][lane % LANES * V]);
                dst += (ptrdiff_t)TURN * (ptrdiff_t)p.stride[VALUES];
            }
        } else {
            for (uint32_t i = lane; i < KV_GRANULE * lanes; i += 32) {
                const uint32_t at = i / lanes, v = i % lanes;
                if (it.live >> at & 1u) *(uint4 *)(row0 + (ptrdiff_t)at * (ptrdiff_t)p.stride[VALUES] + v * V) = *(const uint4 *)&st.x[at][v * V];
            }
        }
    } else {
        for (uint32_t i = lane; i < KV_GRANULE * dims; i += 32) {
            const uint32_t at = i / dims, d = i % dims;
            if (it.live >> at & 1u) row0[(ptrdiff_t)at * (ptrdiff_t)p.stride[VALUES] + d] = st.x[at][d];
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(KV_THREADS) kv_read_kernel(const RowsParams p) {
    __shared__ __align__(16) Staged<T> staged[KV_WARPS];
    const uint32_t warp = threadIdx.x / 32;
    wait_for_previous_operator();
    Item it;
    if (!item_of(p, blockIdx.x * KV_WARPS + warp, it)) return;
    const bool full = p.c.l.width % 128 == 0;
    if (it.which) {
        if (p.c.l.v8) full ? read_item<true, true, true, T>(p, it, staged[warp]) : read_item<true, true, false, T>(p, it, staged[warp]);
        else full ? read_item<true, false, true, T>(p, it, staged[warp]) : read_item<true, false, false, T>(p, it, staged[warp]);
    } else {
        if (p.c.l.k8) full ? read_item<false, true, true, T>(p, it, staged[warp]) : read_item<false, true, false, T>(p, it, staged[warp]);
        else full ? read_item<false, false, true, T>(p, it, staged[warp]) : read_item<false, false, false, T>(p, it, staged[warp]);
    }
}

KvView view(const KvCacheJob &c) { return {c.base, kv_layout(c.width, c.k8, c.v8), c.slots, c.heads, c.capacity / KV_GRANULE, c.status}; }

RowsParams rows_params(const KvCacheJob &c, const void *spans, uint32_t sequences, uint32_t tokens, void *keys, size_t key_stride, void *values, size_t value_stride) {
    const uint32_t granules = (tokens + 2 * KV_GRANULE - 2) / KV_GRANULE;
    return {view(c), (const KvSpan *)spans, sequences, tokens, (c.width + 127) / 128, granules, {keys, values}, {key_stride, value_stride}};
}
unsigned blocks_of(const RowsParams &p) { return (unsigned)(((size_t)p.sequences * p.granules * p.c.heads * p.pieces * 2 + KV_WARPS - 1) / KV_WARPS); }

}  // namespace

int launch_kv_write(cudaStream_t s, const KvCacheJob &c, const void *spans, uint32_t sequences, uint32_t tokens, const float *keys, size_t key_stride,
                    const float *values, size_t value_stride) {
    const RowsParams p = rows_params(c, spans, sequences, tokens, (void *)keys, key_stride, (void *)values, value_stride);
    launch_after_previous(kv_write_kernel, dim3(blocks_of(p)), dim3(KV_THREADS), s, p);
    return 1;
}

int launch_kv_read(cudaStream_t s, const KvCacheJob &c, const void *spans, uint32_t sequences, uint32_t tokens, void *keys, size_t key_stride, void *values,
                   size_t value_stride, bool bf16) {
    const RowsParams p = rows_params(c, spans, sequences, tokens, keys, key_stride, values, value_stride);
    if (bf16) launch_after_previous(kv_read_kernel<__nv_bfloat16>, dim3(blocks_of(p)), dim3(KV_THREADS), s, p);
    else launch_after_previous(kv_read_kernel<float>, dim3(blocks_of(p)), dim3(KV_THREADS), s, p);
    return 1;
}

}  // namespace nu
