// Causal grouped-query attention over the quantized cache, in F32 accuracy.
//
//     out = sum_j softmax_j(scale q . k_j) v_j,   j in [max(0, p - window + 1), p]   for the row at position p
//
// split_kernel (widths 64, 128, 256) reads every cache byte of a head once for up to eight query rows and runs both products
// on mma.sync.m16n8k16 without losing F32 accuracy:
//
//   * Codes are whole numbers of at most eight bits, so they are exact in f16; a block's scale is applied to the product, not
//     to the codes. What is not exact in f16, the query and the probabilities, is split: x = hi + lo with both in
//     f16 (22 bits). The 16 rows of the A operand are the hi parts of eight query rows and their lo parts, so the split
//     costs no second instruction, and the two sums of a row come out in the same thread.
//   * q . k = sum_b d_b (q_b . c_b): one accumulator pair of instructions per block of 32, then F32 FMAs with d_b. Codes
//     get their sign on the way (two operations a pair), so that the sums are no larger than the scores. (Eight-bit key codes can stay as they lie, with the
//     share of their offset of 128, sum_b d_b * sum(q_b), taken off afterwards: an operation a pair less and no faster, six rows at 20,000 positions
//     49 us either way. Where a block's queries do not cancel and one channel sets the scale, the offset's share is many times the score:
//     the result was off by up to 9e-5.)
//   * p v = sum_j (p_j d_jb) c_j: the scale goes into the probability, once per block, before it is split. The products
//     p d are kept near 2^11 by a power of two per warp (`bias`), moved when a scale above 2^12 comes by or all that a warp takes at once (16 positions, 32
//     at width 64) lie below 2^6: f16's range is no limit, and what is lost of a position is below 2^-31 of the largest value beside it.
//   * A tensor core's sum is cut off, not rounded, at each step (about 2^-24 of it, always towards zero: a unit of 100,000 positions in one block was
//     up to 9e-5 off), so a warp adds its accumulators up elsewhere, rounded, every 64 products: 592 rows at 100,000 positions, width 256, 4,604 us
//     without and 4,667 with it (5,079 every 32, with the place of the sums kept in registers).
//   * The running maximum of a row is only raised when a score passes it by 3 (in log2): the accumulators are rarely rescaled.
//
// Work split: the granules of all (sequence, row tile, head) units are laid end to end and every block takes the same
// number of them, whatever the lengths are; they are counted on the device from the spans, so a recorded launch fits every
// later length. A unit that spans blocks is joined by the block that arrives last, in block order: nothing depends on timing.
// Within a block the warps take turns at stages of one or two granules, each through its own ring of bulk copies.
//
// Bound by fixed latencies more than by memory: a granule takes about 500 instructions, and a thread's accumulators leave room for four warps
// a scheduler, which keep its issue slots 55 % busy. Measured (Q4_0, 40 query heads on 8 of width 128, one row): position 131,072 68 us,
// 2.2 TB/s; position 700 14.5 us, launch, plan, one stage and join. Six rows (30 a head: four tiles of eight, each unpacks the cache
// again) over 20,000 positions of Q8_0 at width 256 49 us. 24 sequences at width 64 under a window 33 us, 2.0 TB/s.
//
// generic_kernel: one warp per query row and head, any width up to 512; also what generic_only selects. Its sums are compensated every 64
// positions: 2,000,000 positions in a plain F32 sum were 2e-5 off.
#include <type_traits>

#include "kv_attention.cuh"
#include "launch.cuh"

namespace nu {

using namespace attn;

namespace {

// ---- any width ---------------------------------------------------------------------------------------------------------

constexpr int GENERIC_WARPS = 4;
constexpr uint32_t GENERIC_WIDTH = 512;

__device__ __forceinline__ float key_value(const KvLayout &l, const uint8_t *g, uint32_t at, uint32_t dim) {
    const float d = __half2float(*(const __half *)(g + l.k_scales + (at * l.blocks + dim / 32) * 2));
    const uint32_t i = dim % 8, t = dim % 32 / 8;
    if (l.k8) {
        const uint32_t w = *(const uint32_t *)(g + kv_key_word(l, at, dim / 32, t, i % 4 / 2));
        return d * (float)((int)(w >> (8 * (i % 2 * 2 + i / 4)) & 255u) - 128);
    }
    return d * (float)((int)(*(const uint32_t *)(g + kv_key_word(l, at, dim / 32, t, 0)) >> (4 * i) & 15u) - 8);
}
__device__ __forceinline__ float value_value(const KvLayout &l, const uint8_t *g, uint32_t at, uint32_t dim) {
    const float d = __half2float(*(const __half *)(g + l.v_scales + (at * l.blocks + dim / 32) * 2));
    const uint32_t byte = g[kv_value_byte(l, at, dim)];
    return d * (float)(l.v8 ? (int)byte - 128 : (int)(byte >> (dim & 8 ? 4 : 0) & 15u) - 8);
}

__global__ void __launch_bounds__(GENERIC_WARPS * 32) generic_kernel(const AttentionParams p) {
    __shared__ float queries[GENERIC_WARPS][GENERIC_WIDTH];
    __shared__ float2 totals[GENERIC_WARPS][GENERIC_WIDTH];  // a lane's own: the registers are the loop's
    wait_for_previous_operator();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32, width = p.c.l.width, heads = p.c.heads * p.group;
    const size_t item = (size_t)blockIdx.x * GENERIC_WARPS + warp, r = item / heads;
    const uint32_t head = (uint32_t)(item % heads);
    if (r >= (size_t)p.sequences * p.tokens) return;
    const KvSpan span = kv_span(p.c, p.spans, (uint32_t)(r / p.tokens), p.tokens);
    const uint32_t i = (uint32_t)(r % p.tokens);
    if (i >= span.count) return;
    const uint32_t pos = span.first + i, low = p.window && pos >= p.window ? pos - p.window + 1 : 0;
    const float *q = p.q + r * p.q_stride + (size_t)head * width;
    for (uint32_t d = lane; d < width; d += 32) queries[warp][d] = q[d] * p.scale;
    __syncwarp();
    const uint8_t *base = kv_head(p.c, span.slot, head / p.group);
    // acc: the sums of up to 64 positions; totals: of those before, and what their last rounding added, which is taken off the next term
    float m = -INFINITY, acc[GENERIC_WIDTH / 32];
    float2 sum = make_float2(0.0f, 0.0f), *total = totals[warp] + lane;
#pragma unroll
    for (int k = 0; k < (int)GENERIC_WIDTH / 32; ++k) acc[k] = 0.0f;
    for (uint32_t d = 0; d < width; d += 32) total[d] = make_float2(0.0f, 0.0f);
    auto add = [](float2 to, float x) {
        const float y = x - to.y, next = to.x + y;
        return make_float2(next, (next - to.x) - y);
    };
    for (uint64_t j0 = low; j0 <= pos; j0 += 32) {
        const uint64_t j = j0 + lane;
        float s = -INFINITY;
        if (j <= pos) {
            const uint8_t *g = base + (size_t)(j / KV_GRANULE) * p.c.l.bytes;
            s = 0.0f;
            for (uint32_t d = 0; d < width; ++d) s = fmaf(queries[warp][d], key_value(p.c.l, g, (uint32_t)(j % KV_GRANULE), d), s);
        }
        float top = s;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float next = fmaxf(m, top), f = next == -INFINITY ? 1.0f : exp2f(m - next);
        const float w = j <= pos ? exp2f(s - (next == -INFINITY ? 0.0f : next)) : 0.0f;
        m = next;
        if (f != 1.0f) {  // the same in every lane
            sum = make_float2(sum.x * f, sum.y * f);
#pragma unroll
            for (int k = 0; k < (int)GENERIC_WIDTH / 32; ++k) acc[k] *= f;
            for (uint32_t d = 0; d < width; d += 32) total[d] = make_float2(total[d].x * f, total[d].y * f);
        }
        sum = add(sum, w);
        const uint32_t n = (uint32_t)min((uint64_t)32, pos - j0 + 1);
        for (uint32_t l = 0; l < n; ++l) {
            const float wl = __shfl_sync(0xffffffffu, w, l);
            const uint8_t *g = base + (size_t)((j0 + l) / KV_GRANULE) * p.c.l.bytes;
#pragma unroll
            for (int k = 0; k < (int)GENERIC_WIDTH / 32; ++k)
                if (k * 32 < (int)width) acc[k] = fmaf(wl, value_value(p.c.l, g, (uint32_t)((j0 + l) % KV_GRANULE), k * 32 + lane), acc[k]);
        }
        if ((j0 - low) % 64 == 32)
#pragma unroll
            for (int k = 0; k < (int)GENERIC_WIDTH / 32; ++k)
                if (k * 32 < (int)width) { total[k * 32] = add(total[k * 32], acc[k]); acc[k] = 0.0f; }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum.x += __shfl_xor_sync(0xffffffffu, sum.x, o);
#pragma unroll
    for (int k = 0; k < (int)GENERIC_WIDTH / 32; ++k)
        if (k * 32 < (int)width) store_out(p, r * p.out_stride + (size_t)head * width + k * 32 + lane, (total[k * 32].x + (acc[k] - total[k * 32].y)) / sum.x);
}

// ---- widths 64, 128, 256 -------------------------------------------------------------------------------------------------

constexpr int ROWS = 8;  // query rows of a unit

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma(float c[4], const uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// The same onto an accumulator of zeros.
__device__ __forceinline__ void mma_zero(float c[4], const uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t pack_hi_lo(float x, float y, uint32_t &lo) {
    const __half2 hi = __floats2half2_rn(x, y);
    const float2 f = __half22float2(hi);
    lo = h2(__floats2half2_rn(x - f.x, y - f.y));
    return h2(hi);
}

// N words of a lane's codes in a tile, kept in vectors.
template <int N, int VEC>
__device__ __forceinline__ void load_words(const uint8_t *tile, uint32_t lane, uint32_t (&w)[N]) {
#pragma unroll
    for (int v = 0; v < N * 4 / VEC; ++v) {
        const uint8_t *src = tile + v * 32 * VEC + lane * VEC;
        if (VEC == 16) {
            const uint4 x = *(const uint4 *)src;
            w[v * 4] = x.x; w[v * 4 + 1] = x.y; w[v * 4 + 2] = x.z; w[v * 4 + 3] = x.w;
        } else {
            const uint2 x = *(const uint2 *)src;
            w[v * 2] = x.x; w[v * 2 + 1] = x.y;
        }
    }
}
// The scales of positions at, at + 1 (NB each): N = NB words.
template <int NB>
__device__ __forceinline__ void load_scales(const uint8_t *scales, uint32_t at, uint32_t (&w)[NB]) {
    const uint8_t *src = scales + at * NB * 2;
#pragma unroll
    for (int i = 0; i < NB; i += 4) {
        if (NB == 2) {
            const uint2 x = *(const uint2 *)src;
            w[0] = x.x; w[1] = x.y;
        } else {
            const uint4 x = *(const uint4 *)(src + i * 4);
            w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
        }
    }
}
template <int NB>
__device__ __forceinline__ float scale_of(const uint32_t (&w)[NB], int e, int b) {
    const int i = e * NB + b;
    return __half2float(__ushort_as_half((unsigned short)(i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu)));
}

template <int W, bool K8, bool V8>
struct Split {
    // Two blocks share a multiprocessor, so that one's prologue and join run under the other's main loop; a thread holds W/2
    // accumulators, which leaves room for eight warps a block at 128 registers, or four at 255.
    static constexpr int WARPS = W == 256 ? 4 : 8, THREADS = WARPS * 32, RESIDENT = 2;
    static constexpr int NB = W / 32, KT = W / 16, NT = W / 8;
    static constexpr KvLayout L = kv_layout(W, K8, V8);
    static constexpr int SG = W == 64 ? 2 : 1;  // granules of a stage
    static constexpr int STAGE = SG * (int)L.bytes;
    static constexpr int RING = (W == 256 ? 98 : 100) * 1024 / WARPS;
    static constexpr int STAGES = RING / STAGE < 8 ? RING / STAGE : 8;
    static constexpr int JOIN = WARPS * ROWS * W * 4;  // the warps' accumulators; takes the ring's place
    static constexpr int BUFFER = WARPS * STAGES * STAGE > JOIN ? WARPS * STAGES * STAGE : JOIN;
    static constexpr int FRAGMENTS = KT * 512;
    static constexpr int SMEM = BUFFER + FRAGMENTS + WARPS * STAGES * 8 + (WARPS * 2 + 1) * ROWS * 4 + 64;
    static constexpr int PARTIAL = ROWS * (W + 2);
    static constexpr int FOLD = 64 / SG;               // stages that a warp's accumulators sum at most: 64 products each
    static constexpr int FOLDED = WARPS * (NT + 1) * 64;  // floats of a block's sums behind all blocks' partial results: a thread's own, and their m and bias
    // A second segment costs a block about 6 us of prologue and join; the bytes that its warps read in that time.
    static constexpr uint32_t SEGMENT = 96 * 1024 / L.bytes;
    static_assert(SCRATCH_SMS * RESIDENT * (2 * PARTIAL + FOLDED) <= SCRATCH_FLOATS && SCRATCH_SMS * RESIDENT <= SCRATCH_COUNTERS, "the handle's scratch");
    static_assert(STAGES >= 2, "a ring needs two stages");
    static_assert(SMEM <= 113 * 1024, "two blocks share a multiprocessor");
};

template <int W, bool K8, bool V8>
__global__ void __launch_bounds__(Split<W, K8, V8>::THREADS, 2) split_kernel(const __grid_constant__ AttentionParams p) {
    using S = Split<W, K8, V8>;
    constexpr int NB = S::NB, NT = S::NT, WARPS = S::WARPS, STAGES = S::STAGES, SG = S::SG;
    constexpr KvLayout L = S::L;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t *ring = smem;
    float *join = (float *)smem;
    uint4 *fragments = (uint4 *)(smem + S::BUFFER);                     // [KT][32]
    uint64_t *bars = (uint64_t *)(smem + S::BUFFER + S::FRAGMENTS);     // [WARPS][STAGES]
    float *join_m = (float *)(bars + WARPS * STAGES);                   // [WARPS][ROWS]
    float *join_l = join_m + WARPS * ROWS;                              // [WARPS][ROWS]
    float *row_scale = join_l + WARPS * ROWS;                           // [ROWS]
    uint32_t *word = (uint32_t *)(row_scale + ROWS);                    // broadcast words

    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = lane / 4, t = lane % 4;
    if (lane == 0)
        for (int i = 0; i < STAGES; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bars + warp * STAGES + i)), "r"(1));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    wait_for_previous_operator();

    const Plan pl = plan<ROWS, KV_GRANULE, S::SEGMENT, WARPS * SG, 0>(p);
    Walk<ROWS, KV_GRANULE, S::SEGMENT> walk(pl);
    Segment sg;

    uint32_t turn = 0, phase = 0;  // the warp's place in its ring, over all segments
    bool alive = true;
    while (walk.next(p, pl, sg)) {
        // ---- the segment: granules [g0, g0 + n) of one unit, which the blocks c0 .. c1 share ----
        const KvSpan &span = sg.span;
        const uint32_t sequence = sg.sequence, tile = sg.tile, head = sg.head, count = sg.count, skip = sg.skip, n = sg.n, c0 = sg.c0, c1 = sg.c1;
        const uint32_t g0 = sg.first + skip;
        const uint8_t *base = kv_head(p.c, span.slot, head) + (size_t)g0 * L.bytes;
        const uint32_t stages = (n + SG - 1) / SG, mystages = stages > warp ? (stages - warp + WARPS - 1) / WARPS : 0;
        // the ring: `turn` is the place of the warp's next stage, `phase` its barrier's parity; a place is filled again as soon as it is read
        const uint8_t *source = base + (size_t)warp * S::STAGE;
        uint32_t left = mystages, place = turn;
        auto request = [&]() {
            const uint32_t bytes = SG == 1 || left > 1 ? S::STAGE : min((uint32_t)SG, n - (warp + (mystages - 1) * WARPS) * SG) * L.bytes;
            bulk_load(smem_u32(ring + (warp * STAGES + place) * S::STAGE), source, bytes, smem_u32(bars + warp * STAGES + place));
            source += (size_t)WARPS * S::STAGE;
            --left;
            place = place + 1 == STAGES ? 0 : place + 1;
        };
        if (lane == 0)
            for (uint32_t i = 0; i < min(mystages, (uint32_t)STAGES); ++i) request();

        // ---- the rows, split into f16 halves after a power of two that brings each row's largest value to [2^13, 2^14) ----
        const size_t rows0 = (size_t)sequence * p.tokens;  // the sequence's first row in the call
        const uint32_t live_rows = span.count * p.group;
        for (uint32_t r = warp; r < ROWS; r += WARPS) {
            const uint32_t row = tile * ROWS + r;
            float x[8] = {};
            if (row < live_rows && lane < (uint32_t)W / 8) {
                const float *q = p.q + (rows0 + row / p.group) * p.q_stride + (size_t)(head * p.group + row % p.group) * W + lane * 8;
                if ((uintptr_t)q % 16 == 0) {
                    const float4 a = *(const float4 *)q, b = *(const float4 *)(q + 4);
                    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = q[i];
                }
            }
            uint32_t top = 0;  // as bits: NaN and infinity come out largest
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
            top = __reduce_max_sync(0xffffffffu, top);
            // 2^e: from the exponent's bits; rows of zeros and of subnormal values count as 2^-126
            const int e = (int)max(top >> 23, 1u) - 127;
            const float down = top >= 0x7f800000u ? NAN : scalbnf(1.0f, -e);
            if (lane == 0) row_scale[r] = scalbnf(p.scale, e - 13);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * down * 8192.0f;
            if (lane < (uint32_t)W / 8) {
                const uint32_t b = lane / 4, tt = lane % 4;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) hi[i] = pack_hi_lo(x[i], x[i + 4], lo[i]);
                // the pair of dimensions i, i + 4 of the eight is the k pair of step i / 2, half i % 2
                fragments[(2 * b) * 32 + r * 4 + tt] = make_uint4(hi[0], lo[0], hi[1], lo[1]);
                fragments[(2 * b + 1) * 32 + r * 4 + tt] = make_uint4(hi[2], lo[2], hi[3], lo[3]);
            }
        }
        __syncthreads();

        // positions that this thread's row sees, and those that every row of the tile sees
        const uint32_t row = tile * ROWS + g;
        const uint32_t pos = row < live_rows ? span.first + row / p.group : 0;
        const uint32_t row_high = pos, row_low = row < live_rows ? (p.window && pos >= p.window ? pos - p.window + 1 : 0) : 1;  // a dead row sees nothing
        const uint32_t last_row = min(live_rows, tile * ROWS + ROWS) - 1;
        const uint32_t tile_high = span.first + last_row / p.group, first_pos = span.first + tile * ROWS / p.group;
        const uint32_t tile_low = p.window && first_pos >= p.window ? first_pos - p.window + 1 : 0;   // some row sees [tile_low, tile_high]
        const uint32_t all_low = p.window && tile_high >= p.window ? tile_high - p.window + 1 : 0;    // every live row sees [all_low, first_pos]
        const float my_scale = row_scale[g];
        uint32_t k1024 = 0x64006400u;
        asm volatile("" : "+r"(k1024));

        float m = -INFINITY, l = 0.0f, bias = 0x1p40f, o[NT][4];  // the smallest scale is 2^-24
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

        // the sums of earlier stages, of a maximum and a bias of then
        auto sums_so_far = [&]() {
            uint32_t thread = threadIdx.x;
            asm volatile("" : "+r"(thread));  // (found anew each time: the loop has no registers to keep it in)
            return (float2 *)(p.partials + (size_t)gridDim.x * 2 * S::PARTIAL + (size_t)blockIdx.x * S::FOLDED) + thread / 32 * (NT + 1) * 32 + thread % 32;
        };
        auto weight_of = [&](float2 then) {
            return then.x == -INFINITY ? 0.0f : exp2_approx(then.x - m) * (bias / then.y);
        };
        for (uint32_t i = 0, upto = S::FOLD;; upto += S::FOLD) {
        for (const uint32_t end = min(upto, mystages); i < end && alive; ++i) {
            const uint32_t slot = turn;
            alive = mbar_wait(smem_u32(bars + warp * STAGES + slot), phase);
            if (!__all_sync(0xffffffffu, alive)) {  // a copy never came: report, let the others in flight land, give up the block's results
                *(volatile uint32_t *)(p.c.status + STATUS_WAIT) = 1u;
                for (uint32_t k = i + 1; k < min(i + STAGES, mystages); ++k) {
                    if (++turn == STAGES) { turn = 0; phase ^= 1u; }
                    mbar_wait(smem_u32(bars + warp * STAGES + turn), phase);
                }
                alive = false;
                break;
            }
            if (++turn == STAGES) { turn = 0; phase ^= 1u; }
            const uint8_t *stage = ring + (warp * STAGES + slot) * S::STAGE;
            const uint32_t st = warp + i * WARPS, key0 = (g0 + st * SG) * KV_GRANULE;
            const uint32_t here = SG == 1 ? KV_GRANULE : min((uint32_t)SG, n - st * SG) * KV_GRANULE;  // positions that were copied
            const bool at_edge = key0 < all_low || key0 + SG * KV_GRANULE - 1 > first_pos || here < SG * KV_GRANULE;
            auto take = [&](auto edge_tag) {
            constexpr bool edge = decltype(edge_tag)::value;

            float s[SG * 2][2];
            {
                uint32_t codes[SG * 2][K8 ? 2 * NB : NB], scales[SG * 2][NB];
#pragma unroll
                for (int j = 0; j < SG * 2; ++j) {
                    const uint8_t *gran = stage + j / 2 * L.bytes;
                    load_words<K8 ? 2 * NB : NB, L.k_vec>(gran + j % 2 * (L.k_scales / 2), lane, codes[j]);
                    load_scales<NB>(gran + L.k_scales, j % 2 * 8 + 2 * t, scales[j]);
                    s[j][0] = s[j][1] = 0.0f;
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint4 q0 = fragments[(2 * b) * 32 + lane], q1 = fragments[(2 * b + 1) * 32 + lane];
#pragma unroll
                    for (int j = 0; j < SG * 2; ++j) {
                        float c[4];
                        if (K8) {
                            mma_zero(c, q0, byte_codes(codes[j][2 * b], 0x4140), byte_codes(codes[j][2 * b], 0x4342));
                            mma(c, q1, byte_codes(codes[j][2 * b + 1], 0x4140), byte_codes(codes[j][2 * b + 1], 0x4342));
                        } else {
                            const uint32_t w = codes[j][b], w8 = w >> 8;
                            mma_zero(c, q0, low_codes(w, k1024), high_codes(w, k1024));
                            mma(c, q1, low_codes(w8, k1024), high_codes(w8, k1024));
                        }
                        s[j][0] = fmaf(scale_of<NB>(scales[j], 0, b), c[0] + c[2], s[j][0]);
                        s[j][1] = fmaf(scale_of<NB>(scales[j], 1, b), c[1] + c[3], s[j][1]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < SG * 2; ++j) {
                s[j][0] *= my_scale;
                s[j][1] *= my_scale;
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t in = j * 8 + 2 * t + e, key = key0 + in;
                        if (in >= here || key < row_low || key > row_high) s[j][e] = -INFINITY;
                    }
                }
            }

            // ---- the values' scales, and whether the maximum or the bias has to move ----
            uint32_t vs[SG * 2][NB];
            __half2 big = as_h2(0u);
#pragma unroll
            for (int j = 0; j < SG * 2; ++j) {
                load_scales<NB>(stage + j / 2 * L.bytes + L.v_scales, j % 2 * 8 + 2 * t, vs[j]);
                if (edge) {  // what no row of the tile sees may hold anything
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const uint32_t in = j * 8 + 2 * t + e, key = key0 + in;
                        if (in >= here || key < tile_low || key > tile_high) {
#pragma unroll
                            for (int k = 0; k < NB / 2; ++k) vs[j][e * NB / 2 + k] = 0u;
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < NB; ++k) big = __hmax2(big, __habs2(as_h2(vs[j][k])));  // a NaN loses
            }
            const float2 big2 = __half22float2(big);
            const float dmax = fmaxf(big2.x, big2.y);
            float top = s[0][0];
#pragma unroll
            for (int j = 0; j < SG * 2; ++j) top = fmaxf(top, fmaxf(s[j][0], s[j][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (__any_sync(0xffffffffu, top > m + 3.0f || dmax * bias > 4096.0f) || __all_sync(0xffffffffu, dmax * bias < 64.0f)) {
                float d = fmaxf(dmax, __shfl_xor_sync(0xffffffffu, dmax, 1));
                d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, 2));
                const float next = fmaxf(m, top);
                const float bias_next = d * bias > 4096.0f || (d * bias < 64.0f && d > 0.0f) ? scalbnf(1.0f, 127 + 11 - (int)(__float_as_uint(fminf(d, 65504.0f)) >> 23)) : bias;
                const float fl = m == -INFINITY ? 0.0f : exp2_approx(m - next), f = fl * (bias_next / bias);
                bias = bias_next;
                m = next;
                l *= fl;
#pragma unroll
                for (int k = 0; k < NT; ++k) { o[k][0] *= f; o[k][1] *= f; o[k][2] *= f; o[k][3] *= f; }
            }
            const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int j = 0; j < SG * 2; ++j) {
                s[j][0] = exp2_approx(s[j][0] - ref);
                s[j][1] = exp2_approx(s[j][1] - ref);
                l += s[j][0] + s[j][1];
            }

            // ---- p v ----
#pragma unroll
            for (int k = 0; k < SG; ++k) {
                uint32_t codes[V8 ? NT : NT / 2];
                load_words<V8 ? NT : NT / 2, L.v_vec>(stage + k * L.bytes + L.v_codes, lane, codes);
                const float p0 = s[2 * k][0] * bias, p1 = s[2 * k][1] * bias, p2 = s[2 * k + 1][0] * bias, p3 = s[2 * k + 1][1] * bias;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float x0 = p0 * scale_of<NB>(vs[2 * k], 0, b), x1 = p1 * scale_of<NB>(vs[2 * k], 1, b);
                    float x2 = p2 * scale_of<NB>(vs[2 * k + 1], 0, b), x3 = p3 * scale_of<NB>(vs[2 * k + 1], 1, b);
                    if (edge) {  // a position that this row does not see, another does, and whose scale is a NaN (one that it sees reaches it at any weight)
                        const uint32_t key = key0 + k * KV_GRANULE + 2 * t;
                        auto unseen = [&](uint32_t at) { return at < row_low || at > row_high; };
                        if (unseen(key)) x0 = 0.0f;
                        if (unseen(key + 1)) x1 = 0.0f;
                        if (unseen(key + 8)) x2 = 0.0f;
                        if (unseen(key + 9)) x3 = 0.0f;
                    }
                    uint4 a;
                    a.x = pack_hi_lo(x0, x1, a.y);
                    a.z = pack_hi_lo(x2, x3, a.w);
                    if (V8) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) mma(o[4 * b + q], a, byte_codes(codes[4 * b + q], 0x4140), byte_codes(codes[4 * b + q], 0x4342));
                    } else {
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const uint32_t w = codes[2 * b + q], w8 = w >> 8;
                            mma(o[4 * b + 2 * q], a, low_codes(w, k1024), low_codes(w8, k1024));
                            mma(o[4 * b + 2 * q + 1], a, high_codes(w, k1024), high_codes(w8, k1024));
                        }
                    }
                }
            }
            };
            if (at_edge) take(std::true_type{});
            else take(std::false_type{});
            __syncwarp();
            if (lane == 0 && left) request();
        }
            if (i == mystages || !alive) break;
            // (only its own thread reads what it writes)
            float2 *folded = sums_so_far();
            const float f = upto == S::FOLD ? 0.0f : weight_of(folded[NT * 32]);
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                float2 x = upto == S::FOLD ? make_float2(0.0f, 0.0f) : folded[k * 32];
                x.x = fmaf(x.x, f, o[k][0] + o[k][2]);
                x.y = fmaf(x.y, f, o[k][1] + o[k][3]);
                folded[k * 32] = x;
                o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.0f;
            }
            folded[NT * 32] = make_float2(m, bias);
        }
        if (mystages > (uint32_t)S::FOLD) {
            const float2 *folded = sums_so_far();
            const float f = weight_of(folded[NT * 32]);
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                const float2 x = folded[k * 32];
                o[k][0] = fmaf(x.x, f, o[k][0]);
                o[k][1] = fmaf(x.y, f, o[k][1]);
            }
        }

        // ---- join the warps ----
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (!__syncthreads_and(alive)) return;  // every warp is done with the ring, which the accumulators now take
        if (t == 0) { join_m[warp * ROWS + g] = m; join_l[warp * ROWS + g] = l; }
        const float back = 1.0f / bias;
#pragma unroll
        for (int k = 0; k < NT; ++k)
            *(float2 *)(join + (warp * ROWS + g) * W + k * 8 + 2 * t) = make_float2((o[k][0] + o[k][2]) * back, (o[k][1] + o[k][3]) * back);
        __syncthreads();
        const uint32_t used = min(stages, (uint32_t)WARPS);
        const bool whole = n == count;
        float *partial = p.partials + ((size_t)blockIdx.x * 2 + (skip == 0 && !whole)) * S::PARTIAL;  // a unit that starts here goes into the second place
        // a row's parts are weighted by 2^(their maximum - the row's): found once, by one thread a row
        if (tid < ROWS) {
            float top = -INFINITY, sum = 0.0f;
            for (uint32_t w = 0; w < used; ++w) top = fmaxf(top, join_m[w * ROWS + tid]);
            const float ref = top == -INFINITY ? 0.0f : top;
            for (uint32_t w = 0; w < used; ++w) {
                const float f = exp2f(join_m[w * ROWS + tid] - ref);
                sum += join_l[w * ROWS + tid] * f;
                join_m[w * ROWS + tid] = f;
            }
            if (whole) {
                row_scale[tid] = 1.0f / sum;
            } else {
                partial[ROWS * W + tid] = top;
                partial[ROWS * W + ROWS + tid] = sum;
            }
        }
        __syncthreads();
        auto put = [&](uint32_t e, float4 x) {  // four values of a row of the result
            const uint32_t r = e / W;
            const uint32_t out_row = tile * ROWS + r;
            if (out_row >= live_rows) return;
            const float f = row_scale[r];
            const size_t i = (rows0 + out_row / p.group) * p.out_stride + (size_t)(head * p.group + out_row % p.group) * W + e % W;
            store_out(p, i, x.x * f);
            store_out(p, i + 1, x.y * f);
            store_out(p, i + 2, x.z * f);
            store_out(p, i + 3, x.w * f);
        };
        for (uint32_t e = tid * 4; e < ROWS * W; e += S::THREADS * 4) {
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (uint32_t w = 0; w < used; ++w) {
                const float f = join_m[w * ROWS + e / W];
                const float4 x = *(const float4 *)(join + w * ROWS * W + e);
                acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
            }
            if (whole) put(e, acc);
            else *(float4 *)(partial + e) = acc;
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (tid == 0) *word = atomicAdd(p.counters + c0, 1u) == (c1 - c0);
            __syncthreads();
            if (*word) {  // this block arrived last: the parts of all blocks, in their order
                __threadfence();
                const uint32_t parts = (c1 - c0) + 1;
                const float *first_part = p.partials + ((size_t)c0 * 2 + 1) * S::PARTIAL, *other = p.partials + ((size_t)c0 + 1) * 2 * S::PARTIAL;
                auto part = [&](uint32_t c) { return c ? other + (size_t)(c - 1) * 2 * S::PARTIAL : first_part; };
                float *weight = join;  // [parts][ROWS]
                for (uint32_t r = warp; r < ROWS; r += WARPS) {  // a warp a row, a lane a part
                    float top = -INFINITY, sum = 0.0f;
                    for (uint32_t c = lane; c < parts; c += 32) {
                        const float x = __ldcg(part(c) + ROWS * W + r);
                        weight[c * ROWS + r] = x;
                        top = fmaxf(top, x);
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    const float ref = top == -INFINITY ? 0.0f : top;
                    for (uint32_t c = lane; c < parts; c += 32) {
                        const float f = exp2f(weight[c * ROWS + r] - ref);
                        sum += __ldcg(part(c) + ROWS * W + ROWS + r) * f;
                        weight[c * ROWS + r] = f;
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (lane == 0) row_scale[r] = 1.0f / sum;
                }
                __syncthreads();
                for (uint32_t e = tid * 4; e < ROWS * W; e += S::THREADS * 4) {
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                    for (uint32_t c = 0; c < parts; ++c) {
                        const float f = weight[c * ROWS + e / W];
                        const float4 x = __ldcg((const float4 *)(part(c) + e));
                        acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
                    }
                    put(e, acc);
                }
                if (tid == 0) p.counters[c0] = 0;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the ring's bytes go back to the copies
        __syncthreads();
    }
}

template <int W, bool K8, bool V8>
bool configure() {
    return cudaFuncSetAttribute(split_kernel<W, K8, V8>, cudaFuncAttributeMaxDynamicSharedMemorySize, Split<W, K8, V8>::SMEM) == cudaSuccess;
}
template <int W, bool K8, bool V8>
int launch(cudaStream_t s, const AttentionParams &p, int sm_count) {
    using S = Split<W, K8, V8>;
    launch_after_previous_smem(split_kernel<W, K8, V8>, dim3(sm_count * S::RESIDENT), dim3(S::THREADS), S::SMEM, s, p);
    return 1;
}
#define NU_EVERY(F, W, ...) (k8 ? (v8 ? F<W, true, true>(__VA_ARGS__) : F<W, true, false>(__VA_ARGS__)) : (v8 ? F<W, false, true>(__VA_ARGS__) : F<W, false, false>(__VA_ARGS__)))

}  // namespace

bool attention_configure() {
    bool ok = true;
    for (int i = 0; i < 4; ++i) {
        const bool k8 = i & 1, v8 = i & 2;
        ok = ok && NU_EVERY(configure, 64) && NU_EVERY(configure, 128) && NU_EVERY(configure, 256);
    }
    return ok && attention_tile_configure();
}

int launch_attention(cudaStream_t s, const AttentionJob &j) {
    const bool k8 = j.cache.k8, v8 = j.cache.v8;
    const uint32_t width = j.cache.width;
    AttentionParams p{};
    p.c = {j.cache.base, kv_layout(width, k8, v8), j.cache.slots, j.cache.heads, j.cache.capacity / KV_GRANULE, j.cache.status};
    p.spans = (const KvSpan *)j.spans;
    p.sequences = j.sequences; p.tokens = j.tokens;
    p.q = j.queries; p.q_stride = j.q_stride;
    p.group = j.heads / j.cache.heads;
    p.tiles = (uint32_t)(((uint64_t)j.tokens * p.group + ROWS - 1) / ROWS);
    p.out = j.out; p.out_stride = j.out_stride; p.bf16 = j.bf16;
    p.scale = j.scale * 1.4426950408889634f;
    p.window = j.window;
    p.partials = j.partials; p.counters = j.counters;
    if (!j.generic && attention_tile_supported(j)) return launch_attention_tile(s, j, p);
    if (!j.generic && width == 64) return NU_EVERY(launch, 64, s, p, j.sm_count);
    if (!j.generic && width == 128) return NU_EVERY(launch, 128, s, p, j.sm_count);
    if (!j.generic && width == 256) return NU_EVERY(launch, 256, s, p, j.sm_count);
    const size_t items = (size_t)j.sequences * j.tokens * j.heads;
    launch_after_previous(generic_kernel, dim3((unsigned)((items + GENERIC_WARPS - 1) / GENERIC_WARPS)), dim3(GENERIC_WARPS * 32), s, p);
    return 1;
}

}  // namespace nu
