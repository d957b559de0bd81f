// Where a quantized key/value cache keeps its bytes.
//
// A cache holds `slots` sequences of `capacity` positions; every (slot, head) is one run of granules of 16 positions,
// and a granule is one contiguous run of bytes
//
//     [key codes][key scales][value codes][value scales]        (16 x 2 x width x 18 / 32 bytes when both are Q4_0)
//
// so that attention reads a head's history as one linear stream, whatever the two encodings are. Blocks are GGUF's
// (32 values of one position and head, one f16 scale); only the order of the codes is this library's own: it is that
// of the mma.sync.m16n8k16 B operand, so that a lane's share of a tile is its own 16-byte vectors, unpacked with two
// logical operations a pair and no exchange between lanes. With lane = 4 g + t:
//
//   keys     two tiles of eight positions; lane (g, t) holds position g, and of every block b the eight dimensions
//            32 b + 8 t + i. Q4_0: one word a block, nibble i. Q8_0: two words, bytes i = 0,4,1,5 and 2,6,3,7.
//   values   one tile of 16 positions; lane (g, t) holds positions 2t, 2t+1, 8+2t, 9+2t of dimensions 8 n + g.
//            Q4_0: word j has dimension 16 j + g in its low and 16 j + 8 + g in its high nibbles, bytes in the order
//            2t, 8+2t, 2t+1, 9+2t. Q8_0: word n, bytes 2t, 2t+1, 8+2t, 9+2t.
//   scales   [position][block] f16
//
// A code is stored without a sign: Q4_0 as GGUF does (code + 8), Q8_0 as code + 128. A zero-filled buffer is a cache of
// zeros (its scales are zero).
#pragma once
#include <cuda_fp16.h>
#include <stddef.h>
#include <stdint.h>

#include "kernels.hpp"

namespace nu {

constexpr uint32_t KV_GRANULE = 16;  // positions

struct KvLayout {
    uint32_t width, blocks;  // values and 32-value blocks of a head's row
    bool k8, v8;             // Q8_0 instead of Q4_0
    uint32_t k_vec, v_vec;   // bytes of the vectors a lane's codes are kept in
    uint32_t k_scales, v_codes, v_scales, bytes;
};

__host__ __device__ constexpr uint32_t kv_vector(uint32_t lane_bytes) { return lane_bytes % 16 == 0 ? 16 : lane_bytes % 8 == 0 ? 8 : 4; }
__host__ __device__ constexpr uint32_t kv_code_bytes(uint32_t width, bool q8) { return KV_GRANULE * width / (q8 ? 1 : 2); }

__host__ __device__ constexpr KvLayout kv_layout(uint32_t width, bool k8, bool v8) {
    KvLayout l{};
    l.width = width;
    l.blocks = width / 32;
    l.k8 = k8;
    l.v8 = v8;
    l.k_vec = kv_vector(kv_code_bytes(width, k8) / 64);  // two tiles of 32 lanes
    l.v_vec = kv_vector(kv_code_bytes(width, v8) / 32);
    const uint32_t scales = KV_GRANULE * l.blocks * 2;
    l.k_scales = kv_code_bytes(width, k8);
    l.v_codes = l.k_scales + scales;
    l.v_scales = l.v_codes + kv_code_bytes(width, v8);
    l.bytes = l.v_scales + scales;
    return l;
}

// One sequence's rows in a call, as the spans buffer holds them (nu_kv_span).
struct KvSpan {
    uint32_t slot, first, count, reserved;
};

struct KvView {
    uint8_t *base;
    KvLayout l;
    uint32_t slots, heads, granules;  // granules of a (slot, head)
    uint32_t *status;  // the status words
};

__device__ __forceinline__ uint8_t *kv_head(const KvView &c, uint32_t slot, uint32_t head) {
    return c.base + ((size_t)slot * c.heads + head) * c.granules * c.l.bytes;
}

// A span that names a slot or a position outside the cache, or more rows than the call has, counts as empty and raises
// its status word, which the next commit or graph launch reports.
__device__ __forceinline__ KvSpan kv_span(const KvView &c, const KvSpan *spans, uint32_t sequence, uint32_t tokens) {
    const uint4 w = *(const uint4 *)(spans + sequence);
    KvSpan s{w.x, w.y, w.z, 0};
    if (s.count && (s.slot >= c.slots || s.count > tokens || (uint64_t)s.first + s.count > (uint64_t)c.granules * KV_GRANULE)) {
        *(volatile uint32_t *)(c.status + STATUS_SPAN) = 1u;
        s.count = 0;
    }
    return s;
}

// Byte of the word `word` (of a lane's words in a tile) in the tile's codes.
__host__ __device__ constexpr uint32_t kv_word(uint32_t vec, uint32_t lane, uint32_t word) {
    return word * 4 / vec * 32 * vec + lane * vec + word * 4 % vec;
}
// Key codes: offset in the granule of the word(s) that hold dimensions 32 b + 8 t .. + 7 of position `at`.
// (`vec`: the layout's, which a caller that knows it to be 16 passes as that constant.)
__host__ __device__ inline uint32_t kv_key_word(const KvLayout &l, uint32_t vec, uint32_t at, uint32_t b, uint32_t t, uint32_t second) {
    return at / 8 * (l.k_scales / 2) + kv_word(vec, at % 8 * 4 + t, l.k8 ? 2 * b + second : b);
}
__host__ __device__ inline uint32_t kv_key_word(const KvLayout &l, uint32_t at, uint32_t b, uint32_t t, uint32_t second) { return kv_key_word(l, l.k_vec, at, b, t, second); }
// Value codes: offset of the byte that holds dimension `dim` of position `at`; Q4_0: the high nibble if dim & 8.
__host__ __device__ inline uint32_t kv_value_byte(const KvLayout &l, uint32_t at, uint32_t dim) {
    const uint32_t half = at / 8, t = at % 8 / 2, e = at % 2, lane = dim % 8 * 4 + t;
    return l.v_codes + kv_word(l.v_vec, lane, l.v8 ? dim / 8 : dim / 16) + (l.v8 ? half * 2 + e : e * 2 + half);
}

}  // namespace nu
