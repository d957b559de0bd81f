// What the attention kernels over the quantized cache share: their parameters, the split of the work over the blocks, and the
// unpacking of codes to f16.
#pragma once
#include <cuda_bf16.h>

#include "kernels.hpp"
#include "kv_layout.cuh"

namespace nu {
namespace attn {

constexpr uint32_t SPIN_LIMIT = 1u << 22;

struct AttentionParams {
    KvView c;
    const KvSpan *spans;
    uint32_t sequences, tokens;
    const float *q;
    size_t q_stride;
    uint32_t group;  // query heads of a key/value head
    uint32_t tiles;  // row tiles of a (sequence, head): ceil(tokens * group / rows of a tile)
    void *out;
    size_t out_stride;
    bool bf16;
    float scale;     // times log2(e)
    uint32_t window; // 0: none
    float *partials;      // [block][2][rows * (width + 2)], and behind them the sums of long units ([block][FOLDED] of the kernel)
    uint32_t *counters;   // one a block, zero between launches
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void store_out(const AttentionParams &p, size_t index, float v) {
    if (p.bf16) ((__nv_bfloat16 *)p.out)[index] = __float2bfloat16_rn(v);
    else ((float *)p.out)[index] = v;
}

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ uint32_t h2(__half2 x) { return *(const uint32_t *)&x; }
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *(const __half2 *)&x; }
// (w & mask) | high in one operation: `high` is a register the compiler cannot see into, as two constants do not fit one.
__device__ __forceinline__ uint32_t mask_or(uint32_t w, uint32_t mask, uint32_t high) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(high));
    return r;
}
// Four-bit codes in bits 0..3 / 4..7 of the bytes 0 and 2 of w, as whole numbers code - 8 in f16: the code is placed in the
// low bits of 1024 (or, shifted by four, of 1024 = 64 * 16), which one exact operation takes off again.
__device__ __forceinline__ uint32_t low_codes(uint32_t w, uint32_t k1024) { return h2(__hsub2(as_h2(mask_or(w, 0x000f000fu, k1024)), as_h2(0x64086408u))); }
__device__ __forceinline__ uint32_t high_codes(uint32_t w, uint32_t k1024) { return h2(__hfma2(as_h2(mask_or(w, 0x00f000f0u, k1024)), as_h2(0x2c002c00u), as_h2(0xd480d480u))); }
// Eight-bit codes in bytes 0, 1 (or 2, 3) of w, as code - 128.
__device__ __forceinline__ uint32_t byte_codes(uint32_t w, uint32_t selector) { return h2(__hsub2(as_h2(__byte_perm(w, 0x64646464u, selector)), as_h2(0x64806480u))); }

// The steps of STEP positions that the ROWS query rows of tile `tile` of a sequence see: [first, first + count).
template <uint32_t ROWS, uint32_t STEP>
__device__ __forceinline__ void unit_range(const AttentionParams &p, const KvSpan &s, uint32_t tile, uint32_t &first, uint32_t &count) {
    const uint32_t rows = s.count * p.group, r0 = tile * ROWS;  // below 2^31: the host's limit on a call's rows
    first = count = 0;
    if (r0 >= rows) return;
    const uint32_t r1 = min(rows, r0 + ROWS) - 1;
    const uint32_t low = s.first + r0 / p.group, high = s.first + r1 / p.group;
    first = (p.window && low >= p.window ? low - p.window + 1 : 0) / STEP;
    count = high / STEP + 1 - first;
}

// A unit costs its block SEGMENT steps before and after its own (queries, join, result): an equal share counts them as steps, ahead of
// the unit's.
//
// Where a block starts: which entry ((sequence, row tile), all of whose heads have the same steps) and how far into it.
struct Plan {
    bool even;                      // every block has one part of one unit
    bool whole;                     // every block has whole units, longest first; else an equal share of all steps (and segments)
    unsigned long long share, total;
    uint32_t entry, in;             // in: blocks (even) or steps into the entry; whole: the units
    bool idle;
};

// One warp's finding, the same in every warp: no barrier. Lanes take entries in turn.
template <uint32_t ROWS, uint32_t STEP, uint32_t SEGMENT, uint32_t LEAST, uint32_t JOIN>
__device__ __forceinline__ Plan plan(const AttentionParams &p) {
    const uint32_t lane = threadIdx.x & 31, entries = p.sequences * p.tiles, blocks = gridDim.x, heads = p.c.heads;
    uint32_t first, one = 0;  // the steps of this lane's first entry
    auto steps = [&](uint32_t e) {
        uint32_t count = 0;
        if (e < entries) unit_range<ROWS, STEP>(p, kv_span(p.c, p.spans, e / p.tiles, p.tokens), e % p.tiles, first, count);
        return count;
    };
    auto cached = [&](uint32_t e) { return e < 32 ? one : steps(e); };
    one = steps(lane);
    unsigned long long total = 0, units = 0;
    for (uint32_t e = lane; e < entries; e += 32) {
        const uint32_t c = cached(e);
        total += c;
        units += c != 0;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        units += __shfl_xor_sync(0xffffffffu, units, o);
    }
    total *= heads;
    units *= heads;
    Plan r{};
    r.total = total + units * SEGMENT;
    r.share = (r.total + blocks - 1) / blocks;
    if (total == 0) { r.idle = true; return r; }
    // Even parts: 1 + count * spare / total blocks for a unit of `count` steps, at most `blocks` together and of LEAST steps or more (what a
    // block's warps do at once: shorter parts would only be more to join). Taken if the longest part
    // is not much longer than an equal share, which costs most blocks a second segment. Where the block that joins takes JOIN
    // steps' time for a part, count / n + JOIN n is least at n = sqrt(count / JOIN); up to sqrt(2) more are as good (128 rows of 4 heads at
    // position 8,000, width 256: 37 parts a unit 126 us, 16 parts 86 us).
    const unsigned long long spare = units <= blocks ? blocks - units : 0;
    auto parts = [&](uint32_t count) {
        const uint32_t n = min(1 + (uint32_t)((unsigned long long)count * spare / total), (count + LEAST - 1) / LEAST);
        return JOIN ? min(n, 1 + (uint32_t)sqrtf(2.0f * (float)count / (float)max(JOIN, 1u))) : n;
    };
    if (units <= blocks) {
        uint32_t even = 0, equal = 0;  // the longest time of a unit, in steps
        for (uint32_t e = lane; e < entries; e += 32) {
            const uint32_t c = cached(e), n = parts(c);
            if (c == 0) continue;
            even = max(even, (c + n - 1) / n + JOIN * n);
            equal = max(equal, JOIN * (uint32_t)((c + r.share - 1) / r.share));
        }
        r.even = __reduce_max_sync(0xffffffffu, even) <= r.share + SEGMENT + __reduce_max_sync(0xffffffffu, equal);
    }
    // Whole units: a prompt has its units in order of length, so the blocks take them from the longest down, forwards and backwards in turn.
    // Nothing is joined then (a prompt of 2,048 rows to BF16: 172 us in equal shares, 109 so and with faster joins); taken where no block gets much more than an equal
    // share (with many rounds none does).
    if (p.sequences == 1 && units > blocks) {
        const uint32_t n = (uint32_t)units, rounds = (n + blocks - 1) / blocks;
        uint32_t longest = 0;
        if (rounds <= 8) {  // 32 blocks stand for all: their neighbours' units are as long to a step, but for the last round's end (all: 4 us more)
            const uint32_t rest = n - (rounds - 1) * blocks - 1, b = lane == 0 ? ((rounds - 1) & 1u ? blocks - 1 - rest : rest) : lane * blocks / 32;
            for (uint32_t j = 0; j < rounds; ++j) {
                const uint32_t u = j * blocks + (j & 1u ? blocks - 1 - b : b);
                if (u < n) longest += steps((n - 1 - u) / heads) + SEGMENT;
            }
        }
        r.whole = __reduce_max_sync(0xffffffffu, longest) <= r.share + SEGMENT;
        if (r.whole) {
            r.in = n;
            r.share = rounds;
            return r;
        }
    }
    const unsigned long long at = r.even ? blockIdx.x : blockIdx.x * r.share;
    unsigned long long before = 0;
    r.idle = true;
    for (uint32_t e0 = 0; e0 < entries; e0 += 32) {
        const uint32_t c = cached(e0 + lane);
        const unsigned long long mine = c == 0 ? 0 : (unsigned long long)(r.even ? parts(c) : c + SEGMENT) * heads;
        unsigned long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= (uint32_t)o) upto += x;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, at < before + upto);
        if (hit) {
            const int l = __ffs(hit) - 1;
            r.entry = e0 + l;
            r.in = (uint32_t)(at - before - __shfl_sync(0xffffffffu, upto - mine, l));
            r.idle = false;
            break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (r.even && !r.idle) {  // the unit's share: parts of one length
        const uint32_t c = steps(r.entry), n = parts(c);
        r.share = (c + n - 1) / n;
        r.total = n;
    }
    return r;
}

// The part of a unit that a block takes next: steps [skip, skip + n) of the `count` from `first`, and the blocks c0 .. c1 that share the unit.
struct Segment {
    KvSpan span;
    uint32_t sequence, tile, head, first, count, skip, n, c0, c1;
};

// Walks a block's plan; the same in every thread that walks it.
template <uint32_t ROWS, uint32_t STEP, uint32_t SEGMENT>
struct Walk {
    unsigned long long at, end, entry_begin;
    uint32_t entry;
    __device__ __forceinline__ explicit Walk(const Plan &pl) {
        at = pl.even || pl.whole ? 0 : blockIdx.x * pl.share;
        end = pl.idle ? 0 : pl.even ? 1 : pl.whole ? pl.share : min(pl.total, at + pl.share);  // even parts: one turn; whole units: one a round
        entry_begin = at - pl.in;
        entry = pl.entry;
    }
    __device__ __forceinline__ bool next(const AttentionParams &p, const Plan &pl, Segment &s) {
        while (at < end) {
            if (pl.whole) {
                const uint32_t j = (uint32_t)at++, u = j * gridDim.x + (j & 1u ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                if (u >= pl.in) continue;
                s.sequence = 0;
                s.tile = (pl.in - 1 - u) / p.c.heads;
                s.head = (pl.in - 1 - u) % p.c.heads;
                s.span = kv_span(p.c, p.spans, 0, p.tokens);
                unit_range<ROWS, STEP>(p, s.span, s.tile, s.first, s.count);
                s.skip = 0;
                s.n = s.count;
                s.c0 = s.c1 = blockIdx.x;
                return true;
            }
            s.sequence = entry / p.tiles;
            s.tile = entry % p.tiles;
            s.span = kv_span(p.c, p.spans, s.sequence, p.tokens);
            unit_range<ROWS, STEP>(p, s.span, s.tile, s.first, s.count);
            if (pl.even) {
                const uint32_t parts = (uint32_t)pl.total, share = (uint32_t)pl.share, k = pl.in % parts;
                s.head = pl.in / parts;
                s.skip = k * share;
                at = end;
                if (s.skip >= s.count) return false;  // fewer parts than blocks
                s.n = min(share, s.count - s.skip);
                s.c0 = blockIdx.x - k;
                s.c1 = s.c0 + (s.count - 1) / share;
                return true;
            }
            const uint32_t cost = s.count ? s.count + SEGMENT : 0;
            const unsigned long long all = (unsigned long long)cost * p.c.heads;
            if (at - entry_begin >= all) {  // all its heads are done (or it has no rows)
                entry_begin += all;
                ++entry;
                continue;
            }
            s.head = (uint32_t)((at - entry_begin) / cost);
            const unsigned long long unit_begin = entry_begin + (unsigned long long)s.head * cost;
            const uint32_t from = (uint32_t)(at - unit_begin), to = (uint32_t)min((unsigned long long)cost, end - unit_begin);
            at += to - from;
            if (to <= SEGMENT) continue;  // the share ends ahead of the unit's first step
            s.skip = max(from, SEGMENT) - SEGMENT;
            s.n = to - SEGMENT - s.skip;
            s.c0 = (uint32_t)((unit_begin + SEGMENT) / pl.share);
            s.c1 = (uint32_t)((unit_begin + cost - 1) / pl.share);
            return true;
        }
        return false;
    }
};

}  // namespace attn

// The kernel for many rows to BF16 (kv_attention_tile.cu); whether it serves the job.
bool attention_tile_configure();
bool attention_tile_supported(const AttentionJob &job);
int launch_attention_tile(cudaStream_t s, const AttentionJob &job, attn::AttentionParams p);

}  // namespace nu
