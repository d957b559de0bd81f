// Attention over the quantized cache for many query rows, to BF16: the products on the 5th-generation tensor cores.
//
// One block a multiprocessor walks its share of all (sequence, row tile, head) units, as the kernel for few rows does
// (kv_attention.cu), in steps of 128 keys (64 at width 256). A unit's row tile is 256 query rows, two M = 128 tiles that share every key
// step (one tile at width 256, whose accumulator alone takes half the tensor memory).
//   * warps 8..15 decode: a step's keys and values become f16 in shared memory, in the 128-byte-swizzled K-major layout of
//     the tensor core: keys as rows of dimensions, values transposed as rows of positions. The dimensions of a key's eight
//     stand in the order 0,4,1,5,2,6,3,7 that unpacking gives, and the queries are laid out alike. Two more warps bring the
//     scales of the next step near f16's upper end meanwhile (done by the decoding warps themselves, with a barrier before and after,
//     387 rows at position 24,100 took 338 us instead of 267).
//   * warp 16 issues S = Q K^T and O += P V, in an order that keeps one tile's softmax under the other's products.
//   * warps 0..7 are the softmax: a thread has a row; it reads S from tensor memory, writes P = 2^(S scale - m) as f16 over it, and
//     the tensor core takes P from there. The maximum m is only moved when a score passes it by 8 (log2), so O is rarely rescaled.
//
// Range: a step's keys and values are brought into f16's range by a power of two each (their largest scale's), a row's query
// by one of its own; the score's factor takes the first and last back, O carries the values'. Where that moves by more than P has room for, O is
// multiplied by the power of two between them, up or down, so P's bits do not depend on what the values of other steps are. Products are exact and sums F32. Against 64 bits the result is off by
// its own BF16 rounding and little else (1.7e-3 relative). The tensor cores cut a sum off at each product (about 2^-24 of it, always towards zero: 1,500,000 positions in one
// block were 1.1e-2 off), so over a long cache (`launch`) the softmax warps add O up elsewhere, rounded, every 32,768 positions, and it starts again at zero.
//
// A value's scale that is NaN would reach rows that do not see its position (0 * NaN), so it is decoded as zeros and marked, and
// the rows that do see it write NaN in its block's dimensions.
//
// Bound by the work on both sides of the tensor core, not by memory: at width 256 a step of 64 keys costs the decoding warps more than its
// products take; at width 128 a softmax warp spends 3,300 cycles on 128 keys, of which the exponentials are a third and reading S from
// tensor memory twice most of the rest (its 128 columns do not fit in registers beside eight decoding warps). Measured: 387 rows
// of 20 heads on 4 (width 256) at position 24,100 271 us, 700 TFLOP/s; a prompt of 2,048 rows, 40 heads on 8 of width 128, 111 us, 388 TFLOP/s over
// the causal half.
//
// Every wait is bounded: a thread whose wait runs out raises the block's flag, all waits then fall through, and the block
// ends as ever with the status word raised.
#include <algorithm>

#include "kv_attention.cuh"
#include "launch.cuh"

namespace nu {

using namespace attn;

namespace {

template <int W, bool K8, bool V8>
struct Tile {
    static constexpr int QT = W == 256 ? 1 : 2;    // M = 128 tiles
    static constexpr int ROWS = QT * 128;
    static constexpr int KT = W == 256 ? 64 : 128; // keys of a step
    static constexpr int NB = W / 32;
    static constexpr KvLayout L = kv_layout(W, K8, V8);
    static constexpr int SOFT = 8, PROD = 8, THREADS = (SOFT + PROD + 4) * 32;  // + the warpgroup of the warp that issues
    // Registers a thread, of the 96 x 640 that the block starts with
    static constexpr int SOFT_REGS = 136, PROD_REGS = 80, MMA_REGS = 48;
    static_assert(SOFT * SOFT_REGS + PROD * PROD_REGS + 4 * MMA_REGS <= (SOFT + PROD + 4) * 96, "more registers than the block has");
    // shared memory
    static constexpr int Q_TILE = 128 * W * 2, Q = 0, K_BYTES = KT * W * 2, K = Q + QT * Q_TILE, V = K + 2 * K_BYTES, TABLE = V + 2 * K_BYTES;
    static constexpr int NANS = TABLE + 4 * NB * KT * 2, EXCHANGE = NANS + 4 * 128, SMALL = EXCHANGE + 3 * 256 * 4, BARS = SMALL + 128, BYTES = BARS + 32 * 8 + 1024;
    // tensor memory columns
    static constexpr int S_COLS = KT, O_COL = 2 * KT;
    static constexpr int PARTIAL = ROWS * (W + 2);
    static constexpr int FOLD = 32768 / KT;                        // steps that O sums at most
    static constexpr int FOLDED = 256 * (W / (QT == 2 ? 1 : 2) + 2);  // floats of a block's sums behind all blocks' partial results: a thread's columns of its row, m and exponent
    static_assert(SCRATCH_SMS * (2 * PARTIAL + FOLDED) <= SCRATCH_FLOATS && SCRATCH_SMS <= SCRATCH_COUNTERS, "the handle's scratch");
    // P is kept 2^P_UP above the probabilities (at most 2^8 before a maximum moves), so that it ends below 2^15. O carries the exponent of a
    // step's values; a step whose values' lies up to SPREAD below takes P down by that (a probability of one keeps 11 bits down to 2^-14, so a SPREAD of
    // 12 leaves those of 2^-9 all of theirs), any other moves O's exponent to its own, up or down. O is at most 2^31 positions of 2^15 times a value
    // below 2^16, and the exponents are 40 apart at most, so F32 holds it.
    static constexpr int P_UP = 7, SPREAD = 12, NO_VALUES = -1000;  // NO_VALUES: a step of zeros
    // The largest scale of a step goes to [2^TOP, 2^(TOP+1)), so that times the largest code it just ends in f16 (65,504). A value keeps f16's 11 bits down to 2^-29 of the
    // largest value of its step, and all to 2^-40 of it.
    static constexpr int K_TOP = K8 ? 8 : 12, V_TOP = V8 ? 8 : 12;
    static constexpr uint32_t SEGMENT = 6;         // steps that a block decodes in the time that a second segment costs it
};

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// Bounded; falls through at once when a thread of the block has given up.
__device__ __forceinline__ void wait_or_give_up(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag) {
    for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return;
        if (i % 64 == 63 && *abort_flag) return;
    }
    *abort_flag = 1;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar) : "memory");
}
template <int N>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// Two F32 operations at once.
__device__ __forceinline__ uint64_t two(float a, float b) { return (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float low_of(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float high_of(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
// Shared-memory descriptor of a K-major f16 tile in the 128-byte swizzle: rows of 128 bytes, groups of eight rows 1024 bytes
// apart (version 1, swizzle mode 2). The high word is the same for all; the low one has the address.
constexpr uint32_t DESC_HIGH = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t descriptor(uint32_t addr) { return (addr & 0x3ffffu) >> 4 | 1u << 16; }
// kind::f16, D f32, A and B f16, K-major.
constexpr uint32_t instruction(int m, int n) { return 1u << 4 | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24; }
// Four steps of 16 along K, one swizzle atom: 32 bytes, two units of a descriptor, further each. The whole warp comes here, so that
// the operands stay in uniform registers, and one lane issues: with a lane alone in a branch every operand had to be moved there,
// some 130 cycles a product that itself takes 32 to 64.
__device__ __forceinline__ void mma_ss4(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p, q;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.eq.u32 q, %4, %4;\n\t"
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t"
        "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %5};\n\tmov.b64 b, {y, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(DESC_HIGH)
        : "memory");
}
// The same with A in tensor memory: 16 f16 along K are eight columns.
__device__ __forceinline__ void mma_ts4(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred e, p, q;\n\t.reg .b64 b;\n\t.reg .b32 x, y;\n\t"
        "elect.sync _|e, 0xffffffff;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.eq.u32 q, %4, %4;\n\t"
        "mov.b64 b, {%2, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t"
        "add.u32 x, %1, 8;\n\tadd.u32 y, %2, 2;\n\tmov.b64 b, {y, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, q;\n\t"
        "add.u32 x, %1, 16;\n\tadd.u32 y, %2, 4;\n\tmov.b64 b, {y, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, q;\n\t"
        "add.u32 x, %1, 24;\n\tadd.u32 y, %2, 6;\n\tmov.b64 b, {y, %5};\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, q;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(DESC_HIGH)
        : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
          "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]),
          "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
                   "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
        "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
        "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
                 "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int ID, int N>
__device__ __forceinline__ void named_barrier() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory"); }
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// The 16-byte chunk that eight dimensions 32 b + 8 t .. of a row are kept in: an order in which the lanes (g, t) of a tile of keys, eight at
// a time, meet no bank twice.
__host__ __device__ constexpr uint32_t chunk_of(uint32_t b, uint32_t t) { return b / 2 * 8 + 2 * t + b % 2; }
// Byte of the 16-byte chunk `chunk` (of all a row's) of row `row` in a swizzled tile of `rows` rows.
__device__ __forceinline__ uint32_t swizzled(uint32_t rows, uint32_t row, uint32_t chunk) {
    return chunk / 8 * rows * 128 + row / 8 * 1024 + row % 8 * 128 + ((chunk % 8) ^ (row % 8)) * 16;
}
// Two codes with their sign, exact in f16, times their scales: a value is rounded once.
__device__ __forceinline__ uint32_t value2(uint32_t codes, uint32_t d) { return h2(__hmul2(as_h2(codes), as_h2(d))); }

// LONG: O is added up elsewhere every FOLD steps.
template <int W, bool K8, bool V8, bool LONG>
__global__ void __launch_bounds__(Tile<W, K8, V8>::THREADS, 1) tile_kernel(const __grid_constant__ AttentionParams p) {
    using T = Tile<W, K8, V8>;
    constexpr int QT = T::QT, ROWS = T::ROWS, KT = T::KT, NB = T::NB;
    constexpr KvLayout L = T::L;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);  // (an offset, so that the pointer stays one to shared memory)
    __half *value_scales = (__half *)(smem + T::TABLE);             // [2][NB][KT] of a step
    __half *key_scales = value_scales + 2 * NB * KT;                // [2][KT][NB]
    uint8_t *nans = smem + T::NANS;                                 // [4][128]: blocks of a key's values with a NaN scale
    float *exchange = (float *)(smem + T::EXCHANGE);                // [2][256] row maxima and sums between the two halves of a row (width 256), [256] row scales
    float *row_scale = exchange + 512;
    int *exponents = (int *)(smem + T::SMALL);                      // [4][2] of a step's keys and values
    uint32_t *largest = (uint32_t *)(smem + T::SMALL) + 8;          // [2][rating warp][keys, values] a step's largest scales, as bits
    uint32_t *any_nan = largest + 8;                                // [4]
    uint32_t *tmem_slot = any_nan + 4, *last = tmem_slot + 1;
    volatile uint32_t *abort_flag = last + 1;
    uint32_t *rated_nan = last + 2;                                 // [2][rating warp]
    const uint32_t bars = smem_u32(smem + T::BARS);
    auto bar = [&](int i) { return bars + i * 8; };
    constexpr int K_FULL = 0, K_EMPTY = 2, V_FULL = 4, V_EMPTY = 6, S_FULL = 8, P_FULL = 10, PV_DONE = 12, Q_FULL = 14, SCALES_FULL = 16, SCALES_EMPTY = 18;
    const uint32_t tid = threadIdx.x, warp = tid / 32, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar(K_FULL + i), T::PROD);
            mbar_init(bar(V_FULL + i), T::PROD);
            mbar_init(bar(K_EMPTY + i), 1);
            mbar_init(bar(V_EMPTY + i), 1);
            mbar_init(bar(S_FULL + i), 1);
            mbar_init(bar(P_FULL + i), T::SOFT / QT);
            mbar_init(bar(PV_DONE + i), 1);
            mbar_init(bar(SCALES_FULL + i), 2);
            mbar_init(bar(SCALES_EMPTY + i), T::PROD);
        }
        mbar_init(bar(Q_FULL), T::SOFT);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == T::SOFT + T::PROD) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    wait_for_previous_operator();

    const Plan pl = plan<ROWS, KT, T::SEGMENT, 2, 1>(p);
    Walk<ROWS, KT, T::SEGMENT> walk(pl);
    Segment sg;

    if (warp < T::SOFT) {
        more_registers<T::SOFT_REGS>();
        // ---- softmax: thread = row `row` of M tile `q` (width 256: columns `half` of the only tile) ----
        const uint32_t group = warp / 4, q = QT == 2 ? group : 0, row = warp % 4 * 32 + lane;
        const uint32_t lanes = (warp % 4 * 32) << 16;
        constexpr int COLS = QT == 2 ? KT : KT / 2;  // of S, a thread's
        constexpr int OCOLS = QT == 2 ? W : W / 2;   // of O
        const uint32_t ocol = tmem + lanes + T::O_COL + (QT == 2 ? q * W : group * OCOLS);
        uint32_t step = 0;  // over all segments
        while (walk.next(p, pl, sg)) {
            // the queries: a row's largest value is brought to [2^14, 2^15) by a power of two (or 2^126 times its own)
            const uint32_t live_rows = sg.span.count * p.group, tile_row0 = sg.tile * ROWS;
            const size_t rows0 = (size_t)sg.sequence * p.tokens;
            {
                constexpr uint32_t LPR = W / 8, RPI = 32 / LPR;  // lanes a row, rows a turn
                constexpr uint32_t MINE = ROWS / T::SOFT;        // rows of this warp: those of its threads
                const uint32_t base = QT == 2 ? warp * 32 : warp % 4 * 32 + group * 16, chunk = lane % LPR;
                constexpr uint32_t TURNS = MINE / RPI, BATCH = TURNS < 8 ? TURNS : 8;
                const bool aligned = ((uintptr_t)p.q | p.q_stride * 4) % 16 == 0;
                auto source = [&](uint32_t r) -> const float * {
                    const uint32_t all = tile_row0 + r;
                    return all < live_rows ? p.q + (rows0 + all / p.group) * p.q_stride + (size_t)(sg.head * p.group + all % p.group) * W + chunk * 8 : nullptr;
                };
#pragma unroll 1
                for (uint32_t i0 = 0; i0 < TURNS; i0 += BATCH) {
                    float x[BATCH][8];
#pragma unroll
                    for (uint32_t i = 0; i < BATCH; ++i) {
                        const float *src = source(base + (i0 + i) * RPI + lane / LPR);
#pragma unroll
                        for (int k = 0; k < 8; ++k) x[i][k] = 0.0f;
                        if (src && aligned) {
                            const float4 a = *(const float4 *)src, b = *(const float4 *)(src + 4);
                            x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w; x[i][4] = b.x; x[i][5] = b.y; x[i][6] = b.z; x[i][7] = b.w;
                        }
                    }
                    if (!aligned) {
#pragma unroll
                        for (uint32_t i = 0; i < BATCH; ++i) {
                            const float *src = source(base + (i0 + i) * RPI + lane / LPR);
                            if (src) {
#pragma unroll
                                for (int k = 0; k < 8; ++k) x[i][k] = src[k];
                            }
                        }
                    }
#pragma unroll
                    for (uint32_t i = 0; i < BATCH; ++i) {
                        const uint32_t r = base + (i0 + i) * RPI + lane / LPR;
                        uint32_t top = 0;
#pragma unroll
                        for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[i][k]) & 0x7fffffffu);
#pragma unroll
                        for (uint32_t o = 1; o < LPR; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                        const int e = top == 0 ? 0 : min(max((int)(top >> 23) - 127 - 14, -126), 126);
                        const bool bad = top >= 0x7f800000u;
                        const float down = power_of_two(-e);
                        if (chunk == 0) row_scale[r] = bad ? NAN : p.scale * power_of_two(e);
                        uint4 out;
                        out.x = h2(__floats2half2_rn(x[i][0] * down, x[i][4] * down));
                        out.y = h2(__floats2half2_rn(x[i][1] * down, x[i][5] * down));
                        out.z = h2(__floats2half2_rn(x[i][2] * down, x[i][6] * down));
                        out.w = h2(__floats2half2_rn(x[i][3] * down, x[i][7] * down));
                        if (bad) out = make_uint4(0u, 0u, 0u, 0u);
                        *(uint4 *)(smem + T::Q + r / 128 * T::Q_TILE + swizzled(128, r % 128, chunk_of(chunk / 4, chunk % 4))) = out;
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(Q_FULL));
            if (QT == 1) named_barrier<1, 256>();  // the two halves of a row share its scale
            const uint32_t all = tile_row0 + q * 128 + row;
            const bool live = all < live_rows;
            const uint32_t pos = live ? sg.span.first + all / p.group : 0;
            const uint32_t low = live ? (p.window && pos >= p.window ? pos - p.window + 1 : 0) : 1;  // sees [low, pos]; a dead row nothing
            const uint32_t first_pos = sg.span.first + tile_row0 / p.group, last_pos = sg.span.first + (min(live_rows, tile_row0 + ROWS) - 1) / p.group;
            const uint32_t all_low = p.window && last_pos >= p.window ? last_pos - p.window + 1 : 0;  // every live row sees [all_low, first_pos]
            const float rs = row_scale[q * 128 + row];
            float m = -INFINITY, l = 0.0f;
            int big = 0;            // exponent that O carries
            uint32_t nan_blocks = 0;

            // the sums of O of earlier steps ([column][thread]), of a maximum and an exponent of then
            auto sums_so_far = [&]() {
                uint32_t thread = threadIdx.x;
                asm volatile("" : "+r"(thread));  // (found anew each time: the loop has no registers to keep it in)
                return p.partials + (size_t)gridDim.x * 2 * T::PARTIAL + (size_t)blockIdx.x * T::FOLDED + thread;
            };
            auto weight_of_sums = [&]() {
                const float then = sums_so_far()[OCOLS * 256];
                return then == -INFINITY ? 0.0f : exp2_approx(then - m) * power_of_two(__float_as_int(sums_so_far()[OCOLS * 256 + 256]) - big);
            };

            for (uint32_t i = 0, upto = T::FOLD;; upto += T::FOLD) {
            for (const uint32_t end = LONG ? min(upto, sg.n) : sg.n; i < end; ++i, ++step) {
                const uint32_t buffer = QT == 2 ? q : step & 1u, ring = step & 3u;
                const uint32_t key0 = (sg.first + sg.skip + i) * KT + (QT == 1 ? group * COLS : 0);
                const bool edge = key0 < all_low || key0 + COLS - 1 > first_pos;
                wait_or_give_up(bar(S_FULL + buffer), (QT == 2 ? step : step >> 1) & 1u, abort_flag);
                fence_after();
                const int ek = exponents[ring * 2], ev = exponents[ring * 2 + 1];
                float factor = rs * power_of_two(ek);
                factor = factor < 1.2e-38f ? 1.2e-38f : factor;  // a masked score is minus infinity times this
                const uint32_t scol = tmem + lanes + buffer * T::S_COLS;
                // S in chunks of 32 columns, the next on its way while one is worked on; twice, first for the maximum (at width 256 a
                // thread's one chunk stays)
                constexpr int CHUNKS = COLS / 32;
                const uint32_t sfirst = scol + (QT == 1 ? group * COLS : 0);
                uint32_t v[QT][32];
                // columns [from, to] of this thread's are seen
                const int to = pos < key0 ? -1 : (int)min(pos - key0, (uint32_t)COLS), from = low > key0 ? (int)min(low - key0, (uint32_t)COLS) : 0;
                auto hide = [&](uint32_t (&x)[32], int c0) {
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (c > to - c0 || c < from - c0) x[c] = 0xff800000u;
                };
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                tmem_load32(sfirst, v[0]);
#pragma unroll
                for (int k = 0; k < CHUNKS; ++k) {
                    uint32_t (&x)[32] = v[k % QT];
                    tmem_load_wait();
                    if (QT == 2 && k + 1 < CHUNKS) tmem_load32(sfirst + (k + 1) * 32, v[(k + 1) % QT]);
                    if (edge) hide(x, k * 32);
#pragma unroll
                    for (int c = 0; c < 32; c += 8)
#pragma unroll
                        for (int j = 0; j < 4; ++j) tops[j] = fmaxf(tops[j], fmaxf(__uint_as_float(x[c + j]), __uint_as_float(x[c + 4 + j])));
                }
                float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                top *= factor;
                if (QT == 1) {  // both halves have S in registers now: P may take its place
                    exchange[(step & 1u) * 256 + tid] = top;
                    named_barrier<1, 256>();
                    top = fmaxf(top, exchange[(step & 1u) * 256 + (tid ^ 128u)]);
                }
                bool waited = i == 0;
                const int own = ev == T::NO_VALUES ? big : ev;  // a step of zeros goes with any exponent
                if (i == 0) {
                    m = top;
                    big = own;
                } else if (__any_sync(0xffffffffu, top > m + 8.0f) || own > big || own < big - T::SPREAD) {
                    const float next = fmaxf(m, top), fl = m == -INFINITY ? 0.0f : exp2_approx(m - next);
                    const int next_big = own;
                    const float f = fl * power_of_two(big - next_big);
                    m = next;
                    l *= fl;
                    big = next_big;
                    wait_or_give_up(bar(PV_DONE + q), (step - 1) & 1u, abort_flag);
                    waited = true;
                    fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < OCOLS; c0 += 32) {
                        uint32_t o[32];
                        tmem_load32(ocol + c0, o);
                        tmem_load_wait();
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
                        tmem_store32(ocol + c0, o);
                    }
                    tmem_store_wait();
                }
                const int shift = (ev == T::NO_VALUES ? 0 : ev - big) + T::P_UP;
                const float offset = (float)shift - (m == -INFINITY ? 0.0f : m);
                const uint64_t factor2 = two(factor, factor), offset2 = two(offset, offset);
                uint64_t sums[4] = {0, 0, 0, 0};
                // In pieces of 16 columns: one arrives, the next one's powers are taken, the one before is summed, packed and stored between
                // them (the unit of the powers takes 8 cycles an instruction). P lies over S: half as wide, over columns that have been read.
                constexpr int PIECES = COLS / 16;
                uint32_t y[3][16], pk[8];
                auto raise = [&](uint32_t (&x)[16], int pair) {
                    asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+r"(x[2 * pair]));
                    asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+r"(x[2 * pair + 1]));
                };
                auto gather = [&](const uint32_t (&x)[16], int pair) {
                    sums[pair % 4] = add2(sums[pair % 4], (uint64_t)x[2 * pair] | (uint64_t)x[2 * pair + 1] << 32);
                    pk[pair] = h2(__floats2half2_rn(__uint_as_float(x[2 * pair]), __uint_as_float(x[2 * pair + 1])));
                };
                const uint32_t pfirst = scol + (QT == 1 ? group * COLS : 0) / 2;
                if (QT == 2) {
                    tmem_load16(sfirst, y[0]);
                    tmem_load_wait();
                } else {
#pragma unroll
                    for (int c = 0; c < 16; ++c) { y[0][c] = v[0][c]; y[1][c] = v[0][16 + c]; }
                }
#pragma unroll
                for (int k = 0; k < PIECES; ++k) {
                    uint32_t (&x)[16] = y[k % 3];
                    if (QT == 2 && k + 1 < PIECES) tmem_load16(sfirst + (k + 1) * 16, y[(k + 1) % 3]);
                    if (QT == 2 && edge) {
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            if (c > to - k * 16 || c < from - k * 16) x[c] = 0xff800000u;
                    }
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        const uint64_t z = fma2((uint64_t)x[c] | (uint64_t)x[c + 1] << 32, factor2, offset2);
                        x[c] = (uint32_t)z;
                        x[c + 1] = (uint32_t)(z >> 32);
                    }
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        raise(x, c);
                        if (k > 0) gather(y[(k + 2) % 3], c);
                    }
                    if (k > 0) tmem_store8(pfirst + (k - 1) * 8, pk);
                    if (QT == 2 && k + 1 < PIECES) tmem_load_wait();
                }
#pragma unroll
                for (int c = 0; c < 8; ++c) gather(y[(PIECES - 1) % 3], c);
                tmem_store8(pfirst + (PIECES - 1) * 8, pk);
                sums[0] = add2(add2(sums[0], sums[1]), add2(sums[2], sums[3]));
                const float sum = low_of(sums[0]) + high_of(sums[0]);
                if (any_nan[ring]) {  // the blocks that are NaN at a position this row sees, whatever weight it has there
                    const uint8_t *mine = nans + ring * 128 + (QT == 1 ? group * COLS : 0);
#pragma unroll 1
                    for (int c = from; c <= min(to, COLS - 1); ++c) nan_blocks |= mine[c];
                }
                l += sum * power_of_two(-shift);
                tmem_store_wait();
                if (!waited) wait_or_give_up(bar(PV_DONE + q), (step - 1) & 1u, abort_flag);
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(P_FULL + q));
            }
                if (!LONG || i == sg.n) break;
                // (only its own thread reads what it writes)
                wait_or_give_up(bar(PV_DONE + q), (step - 1) & 1u, abort_flag);
                fence_after();
                const float g = upto == T::FOLD ? 0.0f : weight_of_sums();
#pragma unroll 1
                for (int c0 = 0; c0 < OCOLS; c0 += 32) {
                    uint32_t o[32];
                    float *to = sums_so_far() + c0 * 256;
                    tmem_load32(ocol + c0, o);
                    tmem_load_wait();
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(fmaf(upto == T::FOLD ? 0.0f : to[c * 256], g, __uint_as_float(o[c])));
#pragma unroll
                    for (int c = 0; c < 32; ++c) { to[c * 256] = __uint_as_float(o[c]); o[c] = 0u; }
                    tmem_store32(ocol + c0, o);
                }
                sums_so_far()[OCOLS * 256] = m;
                sums_so_far()[OCOLS * 256 + 256] = __int_as_float(big);
                tmem_store_wait();  // (the next step's arrival is for these too)
            }

            // ---- the result, or this block's part of it ----
            wait_or_give_up(bar(PV_DONE + q), (step - 1) & 1u, abort_flag);
            fence_after();
            if (QT == 1) {  // every thread has read the last maxima: the product that was waited for has all their rows
                exchange[tid] = l;
                exchange[256 + tid] = __uint_as_float(nan_blocks);
                named_barrier<1, 256>();
                l += exchange[tid ^ 128u];
                nan_blocks |= __float_as_uint(exchange[256 + (tid ^ 128u)]);
                named_barrier<1, 256>();
            }
            const bool whole = sg.n == sg.count;
            const float up = power_of_two(big - T::P_UP) * (whole ? 1.0f / l : 1.0f);
            float *partial = p.partials + ((size_t)blockIdx.x * 2 + (sg.skip == 0)) * T::PARTIAL;  // a unit that starts here goes into the second place
            const uint32_t dim0 = QT == 2 ? 0 : group * OCOLS;
            const bool folded = LONG && sg.n > (uint32_t)T::FOLD;
            const float g = folded ? weight_of_sums() : 0.0f;
#pragma unroll 1
            for (int c0 = 0; c0 < OCOLS; c0 += 32) {
                uint32_t o[32];
                tmem_load32(ocol + c0, o);
                tmem_load_wait();
                if (folded) {
                    const float *before = sums_so_far() + c0 * 256;
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(fmaf(before[c * 256], g, __uint_as_float(o[c])));
                }
                const bool nan = nan_blocks >> ((dim0 + c0) / 32) & 1u;
#pragma unroll
                for (int c = 0; c < 32; ++c) o[c] = nan ? 0x7fffffffu : __float_as_uint(__uint_as_float(o[c]) * up);
                if (!whole) {
                    float4 *dst = (float4 *)(partial + (size_t)(q * 128 + row) * W + dim0 + c0);
#pragma unroll
                    for (int c = 0; c < 8; ++c) dst[c] = make_float4(__uint_as_float(o[c * 4]), __uint_as_float(o[c * 4 + 1]), __uint_as_float(o[c * 4 + 2]), __uint_as_float(o[c * 4 + 3]));
                } else {  // to this warp's rows of the queries' place: no product reads them any more
                    uint32_t pk[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        const __nv_bfloat162 pair = __floats2bfloat162_rn(__uint_as_float(o[2 * c]), __uint_as_float(o[2 * c + 1]));
                        pk[c] = *(const uint32_t *)&pair;
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        *(uint4 *)(smem + T::Q + q * T::Q_TILE + swizzled(128, row, (dim0 + c0) / 8 + c)) = make_uint4(pk[c * 4], pk[c * 4 + 1], pk[c * 4 + 2], pk[c * 4 + 3]);
                }
            }
            if (whole) {  // and on, whole runs of a row at a time
                __syncwarp();
                constexpr uint32_t CHUNKS = OCOLS / 8;
                const bool aligned = ((uintptr_t)p.out | p.out_stride * 2) % 16 == 0;
#pragma unroll 4
                for (uint32_t i = lane; i < 32 * CHUNKS; i += 32) {
                    const uint32_t r = warp % 4 * 32 + i / CHUNKS, chunk = dim0 / 8 + i % CHUNKS, to = tile_row0 + q * 128 + r;
                    if (to >= live_rows) continue;
                    const uint4 x = *(const uint4 *)(smem + T::Q + q * T::Q_TILE + swizzled(128, r, chunk));
                    __nv_bfloat16 *dst = (__nv_bfloat16 *)p.out + (rows0 + to / p.group) * p.out_stride + (size_t)(sg.head * p.group + to % p.group) * W + chunk * 8;
                    if (aligned) {
                        *(uint4 *)dst = x;
                    } else {
                        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int c = 0; c < 8; ++c) dst[c] = __ushort_as_bfloat16((unsigned short)(w[c / 2] >> (c % 2 * 16)));
                    }
                }
                if (QT == 1) named_barrier<1, 256>();  // a row's next queries are written by either half
                else __syncwarp();
            }
            if (!whole) {
                if (QT == 2 || group == 0) {
                    partial[ROWS * W + q * 128 + row] = m;
                    partial[ROWS * W + ROWS + q * 128 + row] = l;
                }
                __threadfence();
                named_barrier<1, 256>();
                if (tid == 0) *last = atomicAdd(p.counters + sg.c0, 1u) == sg.c1 - sg.c0;
                named_barrier<1, 256>();
                if (*last) {  // this block arrived last: the parts of all blocks, in their order
                    __threadfence();
                    const uint32_t parts = sg.c1 - sg.c0 + 1;
                    auto part = [&](uint32_t c) { return p.partials + ((size_t)(sg.c0 + c) * 2 + (c == 0)) * T::PARTIAL; };
                    // a thread a row finds the parts' weights, 2^(their maximum - the row's) over the row's sum (KEPT parts' into the queries' place);
                    // then a warp adds up ROWS_AT rows at a time, so that many loads are on their way
                    constexpr uint32_t KEPT = 32, ROWS_AT = 4, EACH = W / 32;
                    static_assert(KEPT * ROWS * 4 <= QT * T::Q_TILE, "the weights take the queries' place");
                    float *weight = (float *)(smem + T::Q);  // [KEPT][ROWS]
                    // a part that the row does not see (its maximum is minus infinity) has weight 0 and stays out, whatever it holds
                    auto weigh = [](float m, float mm, float inv) {
                        const float f = exp2_approx(m - mm);
                        return f == 0.0f ? 0.0f : f * inv;
                    };
                    if (tid < (uint32_t)ROWS) {
                        float mm = -INFINITY, ll = 0.0f;
                        for (uint32_t c = 0; c < parts; ++c) mm = fmaxf(mm, __ldcg(part(c) + ROWS * W + tid));
                        mm = mm == -INFINITY ? 0.0f : mm;
                        for (uint32_t c = 0; c < parts; ++c) ll += __ldcg(part(c) + ROWS * W + ROWS + tid) * exp2_approx(__ldcg(part(c) + ROWS * W + tid) - mm);
                        ll = 1.0f / ll;
                        for (uint32_t c = 0; c < min(parts, KEPT); ++c) weight[c * ROWS + tid] = weigh(__ldcg(part(c) + ROWS * W + tid), mm, ll);
                        exchange[tid] = mm;
                        exchange[256 + tid] = ll;
                    }
                    named_barrier<1, 256>();
                    for (uint32_t r0 = warp * ROWS_AT; r0 < (uint32_t)ROWS; r0 += T::SOFT * ROWS_AT) {
                        float acc[ROWS_AT][EACH] = {};
#pragma unroll 2
                        for (uint32_t c = 0; c < parts; ++c)
#pragma unroll
                            for (uint32_t i = 0; i < ROWS_AT; ++i) {
                                const float f = c < KEPT ? weight[c * ROWS + r0 + i] : weigh(__ldcg(part(c) + ROWS * W + r0 + i), exchange[r0 + i], exchange[256 + r0 + i]);
                                float x[EACH];
                                const float *src = part(c) + (size_t)(r0 + i) * W + lane * EACH;
                                if (EACH == 2) {
                                    const float2 y = __ldcg((const float2 *)src);
                                    x[0] = y.x; x[EACH - 1] = y.y;
                                } else {
#pragma unroll
                                    for (uint32_t k = 0; k < EACH; k += 4) {
                                        const float4 y = __ldcg((const float4 *)(src + k));
                                        x[k] = y.x; x[(k + 1) % EACH] = y.y; x[(k + 2) % EACH] = y.z; x[(k + 3) % EACH] = y.w;
                                    }
                                }
#pragma unroll
                                for (uint32_t k = 0; k < EACH; ++k) acc[i][k] = f != 0.0f ? fmaf(x[k], f, acc[i][k]) : acc[i][k];
                            }
#pragma unroll
                        for (uint32_t i = 0; i < ROWS_AT; ++i) {
                            const uint32_t to = tile_row0 + r0 + i;
                            if (to >= live_rows) continue;
                            __nv_bfloat16 *dst = (__nv_bfloat16 *)p.out + (rows0 + to / p.group) * p.out_stride + (size_t)(sg.head * p.group + to % p.group) * W + lane * EACH;
#pragma unroll
                            for (uint32_t k = 0; k < EACH; ++k) dst[k] = __float2bfloat16_rn(acc[i][k]);
                        }
                    }
                    named_barrier<1, 256>();
                    if (tid == 0) p.counters[sg.c0] = 0;
                }
            }
        }
        fence_before();
    } else if (warp < T::SOFT + T::PROD) {
        fewer_registers<T::PROD_REGS>();
        // ---- decoding: a warp has TILES tiles of eight keys of a step, and the values of as many positions. Keys: lane (g, t) its own
        // vectors of a tile; values: lane (half, words w, g) the four lanes' words of two neighbouring words, which are eight positions each of a
        // dimension and (Q4_0) the one eight on ----
        const uint32_t pw = warp - T::SOFT, g8 = lane / 4, t4 = lane % 4;
        constexpr int TILES = KT / 8 / T::PROD;
        constexpr int KVEC = L.k_vec, KWORDS = KVEC / 4;                        // words of a vector
        constexpr int KVECS = (K8 ? 2 : 1) * NB / KWORDS, KITEMS = TILES * KVECS;  // vectors of a tile; of a warp in a step
        constexpr int VVECS = W / (V8 ? 8 : 16) / 4;                            // vectors of a granule
        constexpr int VTURN = 4 / TILES, VITEMS = VVECS < VTURN ? 1 : VVECS / VTURN;  // a half warp has every VTURN-th of a granule's
        const uint32_t half = lane / 16, vpair = lane / 8 % 2, vg = lane % 8;
        const uint32_t kgran = pw * TILES / 2, vgran = TILES == 4 ? pw * 2 + half : pw * TILES / 2, v0 = TILES == 4 ? 0 : TILES == 2 ? half : pw % 2 * 2 + half;
        const bool valued = VVECS >= VTURN || v0 < (uint32_t)VVECS;             // (one vector a granule: half a warp)
        uint32_t k1024 = 0x64006400u;
        asm volatile("" : "+r"(k1024));
        uint32_t step = 0;
        while (walk.next(p, pl, sg)) {
            const uint32_t live_rows = sg.span.count * p.group;
            const uint32_t high = sg.span.first + (min(live_rows, sg.tile * ROWS + ROWS) - 1) / p.group;
            const uint8_t *base = kv_head(p.c, sg.span.slot, sg.head);
            const uint32_t last_granule = high / KV_GRANULE;  // what is behind it may lie past the slot's end: it is not read
            uint32_t kw[KITEMS][KWORDS], vw[VITEMS][4][2];
            auto load_keys = [&](uint32_t key0) {
                const uint32_t gran = key0 / KV_GRANULE + kgran;
                const uint8_t *g = base + (size_t)gran * L.bytes + (TILES == 1 ? pw % 2 * (L.k_scales / 2) : 0) + lane * KVEC;
#pragma unroll
                for (int i = 0; i < KITEMS; ++i) {
                    const uint8_t *src = g + i / KVECS / 2 * L.bytes + i / KVECS % 2 * (L.k_scales / 2) + i % KVECS * 32 * KVEC;
                    const bool in = gran + i / KVECS / 2 <= last_granule;
                    if (KVEC == 16) {
                        const uint4 x = in ? __ldg((const uint4 *)src) : make_uint4(0u, 0u, 0u, 0u);
                        kw[i][0] = x.x; kw[i][1] = x.y; kw[i][KWORDS - 2] = x.z; kw[i][KWORDS - 1] = x.w;
                    } else {
                        const uint2 x = in ? __ldg((const uint2 *)src) : make_uint2(0u, 0u);
                        kw[i][0] = x.x; kw[i][1] = x.y;
                    }
                }
            };
            auto load_values = [&](uint32_t key0) {
                const uint32_t gran = key0 / KV_GRANULE + vgran;
                const bool in = gran <= last_granule && valued;
                const uint8_t *g = base + (size_t)gran * L.bytes + L.v_codes + v0 * 512 + vg * 64 + vpair * 8;
#pragma unroll
                for (int i = 0; i < VITEMS; ++i)
#pragma unroll
                    for (int tt = 0; tt < 4; ++tt) {
                        const uint2 x = in ? __ldg((const uint2 *)(g + i * VTURN * 512 + tt * 16)) : make_uint2(0u, 0u);
                        vw[i][tt][0] = x.x; vw[i][tt][1] = x.y;
                    }
            };
            const uint32_t begin = (sg.first + sg.skip) * KT;
            load_keys(begin);
            load_values(begin);
            for (uint32_t i = 0; i < sg.n; ++i, ++step) {
                const uint32_t key0 = begin + i * KT, stage = step & 1u, parity = (step >> 1) & 1u;
                const bool more = i + 1 < sg.n;
                // keys
                wait_or_give_up(bar(SCALES_FULL + stage), parity, abort_flag);
                if (step >= 2) wait_or_give_up(bar(K_EMPTY + stage), parity ^ 1u, abort_flag);
                uint8_t *kt = smem + T::K + stage * T::K_BYTES;
#pragma unroll
                for (int j = 0; j < KITEMS; ++j) {
                    const uint32_t row = (pw * TILES + j / KVECS) * 8 + g8, v = j % KVECS;
                    constexpr int BLOCKS = KWORDS / (K8 ? 2 : 1);
                    const uint32_t b0 = v * BLOCKS;
                    uint32_t pairs[BLOCKS / 2];
                    const __half *d16 = key_scales + (stage * KT + row) * NB + b0;
                    if (BLOCKS == 4) {
                        const uint2 x = *(const uint2 *)d16;
                        pairs[0] = x.x; pairs[BLOCKS / 2 - 1] = x.y;
                    } else {
                        pairs[0] = *(const uint32_t *)d16;
                    }
#pragma unroll
                    for (int b = 0; b < BLOCKS; ++b) {
                        const uint32_t d = __byte_perm(pairs[b / 2], 0u, b % 2 ? 0x3232 : 0x1010);
                        uint4 x;
                        if (K8) {
                            const uint32_t w0 = kw[j][2 * b % KWORDS], w1 = kw[j][(2 * b + 1) % KWORDS];
                            x = make_uint4(value2(byte_codes(w0, 0x4140), d), value2(byte_codes(w0, 0x4342), d), value2(byte_codes(w1, 0x4140), d),
                                           value2(byte_codes(w1, 0x4342), d));
                        } else {
                            const uint32_t w = kw[j][b], w8 = w >> 8;
                            x = make_uint4(value2(low_codes(w, k1024), d), value2(high_codes(w, k1024), d), value2(low_codes(w8, k1024), d), value2(high_codes(w8, k1024), d));
                        }
                        *(uint4 *)(kt + swizzled(KT, row, chunk_of(b0 + b, t4))) = x;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(K_FULL + stage));
                if (more) load_keys(key0 + KT);

                // values
                if (step >= 2) wait_or_give_up(bar(V_EMPTY + stage), parity ^ 1u, abort_flag);
                uint8_t *vt = smem + T::V + stage * T::K_BYTES;
#pragma unroll
                for (int j = 0; j < VITEMS; ++j) {
                    if (!valued) break;
                    const uint32_t v = j * VTURN + v0, gran = vgran, word = v * 4 + vpair * 2, block = word / (V8 ? 4 : 2);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // eight positions of the granule: 2t, 2t + 1 of every t
                        const uint4 d4 = *(const uint4 *)(value_scales + (stage * NB + block) * KT + gran * 16 + h * 8);
                        const uint32_t d[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            uint32_t x[4], y[4];  // a dimension's eight positions; Q4_0: the dimension eight on
#pragma unroll
                            for (int tt = 0; tt < 4; ++tt) {
                                const uint32_t z = vw[j][tt][w];
                                if (V8) {
                                    x[tt] = value2(byte_codes(z, h ? 0x4342 : 0x4140), d[tt]);
                                } else {
                                    const uint32_t z8 = h ? z >> 8 : z;
                                    x[tt] = value2(low_codes(z8, k1024), d[tt]);
                                    y[tt] = value2(high_codes(z8, k1024), d[tt]);
                                }
                            }
                            const uint32_t dim = (word + w) * (V8 ? 8 : 16) + vg;
                            *(uint4 *)(vt + swizzled(W, dim, gran * 2 + h)) = make_uint4(x[0], x[1], x[2], x[3]);
                            if (!V8) *(uint4 *)(vt + swizzled(W, dim + 8, gran * 2 + h)) = make_uint4(y[0], y[1], y[2], y[3]);
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(V_FULL + stage));
                    mbar_arrive(bar(SCALES_EMPTY + stage));
                }
                if (more) load_values(key0 + KT);
            }
        }
    } else {
        // ---- the products: the first warp of the last warpgroup ----
        fewer_registers<T::MMA_REGS>();
        constexpr uint32_t s_desc = instruction(128, KT), o_desc = instruction(128, W);
        uint32_t step = 0, segment = 0;
        const uint32_t base = __reduce_max_sync(0xffffffffu, tmem);  // (a uniform register)
        const uint32_t q_desc = descriptor(smem_u32(smem + T::Q)), k_desc = descriptor(smem_u32(smem + T::K)), v_desc = descriptor(smem_u32(smem + T::V));
        auto scores = [&](uint32_t q, uint32_t at) {  // S of step `at`
            const uint32_t buffer = QT == 2 ? q : at & 1u, k = k_desc + (at & 1u) * (T::K_BYTES / 16);
#pragma unroll
            for (int s = 0; s < W / 64; ++s) mma_ss4(base + buffer * T::S_COLS, q_desc + (q * T::Q_TILE + s * 128 * 128) / 16, k + s * KT * 128 / 16, s_desc, s != 0);
            commit(bar(S_FULL + buffer));
        };
        while (warp == T::SOFT + T::PROD && walk.next(p, pl, sg)) {
            const uint32_t n = __reduce_max_sync(0xffffffffu, sg.n);
            wait_or_give_up(bar(Q_FULL), segment & 1u, abort_flag);
            wait_or_give_up(bar(K_FULL + (step & 1u)), (step >> 1) & 1u, abort_flag);
            fence_after();
#pragma unroll
            for (uint32_t q = 0; q < QT; ++q) scores(q, step);
            commit(bar(K_EMPTY + (step & 1u)));
            for (uint32_t i = 0; i < n; ++i, ++step) {
                const uint32_t next = step + 1;
                const bool more = i + 1 < n;
                if (more) {
                    wait_or_give_up(bar(K_FULL + (next & 1u)), (next >> 1) & 1u, abort_flag);
                    fence_after();
                    if (QT == 1) {
                        scores(0, next);
                        commit(bar(K_EMPTY + (next & 1u)));
                    }
                }
#pragma unroll
                for (uint32_t q = 0; q < QT; ++q) {
                    wait_or_give_up(bar(P_FULL + q), step & 1u, abort_flag);
                    if (q == 0) wait_or_give_up(bar(V_FULL + (step & 1u)), (step >> 1) & 1u, abort_flag);
                    fence_after();
                    const uint32_t pcol = base + (QT == 2 ? q : step & 1u) * T::S_COLS, v = v_desc + (step & 1u) * (T::K_BYTES / 16);
#pragma unroll
                    for (int s = 0; s < KT / 64; ++s) mma_ts4(base + T::O_COL + q * W, pcol + s * 32, v + s * W * 128 / 16, o_desc, i != 0 || s != 0);
                    commit(bar(PV_DONE + q));
                    if (QT == 2 && more) scores(q, next);
                }
                commit(bar(V_EMPTY + (step & 1u)));
                if (QT == 2 && more) commit(bar(K_EMPTY + (next & 1u)));
            }
            ++segment;
        }
        // ---- the scales, by the next two warps, a step or two ahead of the decoding: a thread has KT / 64 keys. What no row of the tile
        // sees counts as zero; the largest of all sets the step's power of two ----
        if (warp == T::SOFT + T::PROD + 1 || warp == T::SOFT + T::PROD + 2) {
            constexpr int KEYS = KT / 64;
            const uint32_t rw = warp - (T::SOFT + T::PROD + 1), t = rw * 32 + lane;
            while (walk.next(p, pl, sg)) {
                const uint32_t live_rows = sg.span.count * p.group, first_row = sg.tile * ROWS;
                const uint32_t first_pos = sg.span.first + first_row / p.group, high = sg.span.first + (min(live_rows, first_row + ROWS) - 1) / p.group;
                const uint32_t low = p.window && first_pos >= p.window ? first_pos - p.window + 1 : 0;   // some row sees [low, high]
                const uint8_t *head = kv_head(p.c, sg.span.slot, sg.head);
                uint32_t ks[KEYS][NB / 2], vs[KEYS][NB / 2];
                auto load = [&](uint32_t key0) {
#pragma unroll
                    for (int j = 0; j < KEYS; ++j) {
                        const uint32_t at = key0 + t + j * 64;
                        const bool seen = at >= low && at <= high;
                        const uint8_t *g = head + (size_t)(at / KV_GRANULE) * L.bytes + at % KV_GRANULE * NB * 2;
#pragma unroll
                        for (int i = 0; i < NB / 2; ++i) {
                            ks[j][i] = seen ? *(const uint32_t *)(g + L.k_scales + i * 4) : 0u;
                            vs[j][i] = seen ? *(const uint32_t *)(g + L.v_scales + i * 4) : 0u;
                        }
                    }
                };
                const uint32_t begin = (sg.first + sg.skip) * KT;
                load(begin);
                for (uint32_t i = 0; i < sg.n; ++i, ++step) {
                    const uint32_t stage = step & 1u, ring = step & 3u;
                    __half2 kmax = __float2half2_rn(0.0f), vmax = kmax;  // (a NaN loses)
                    uint32_t masks[KEYS], any = 0;
#pragma unroll
                    for (int j = 0; j < KEYS; ++j) {
                        masks[j] = 0;
#pragma unroll
                        for (int k = 0; k < NB / 2; ++k) {
                            const uint32_t x = vs[j][k];
                            if ((x & 0x7fffu) > 0x7c00u) { masks[j] |= 1u << (2 * k); vs[j][k] &= 0xffff0000u; }
                            if ((x >> 16 & 0x7fffu) > 0x7c00u) { masks[j] |= 2u << (2 * k); vs[j][k] &= 0x0000ffffu; }
                            kmax = __hmax2(kmax, __habs2(as_h2(ks[j][k])));
                            vmax = __hmax2(vmax, __habs2(as_h2(vs[j][k])));
                        }
                        any |= masks[j];
                    }
                    const float2 k2 = __half22float2(kmax), v2 = __half22float2(vmax);
                    uint32_t kbits = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(k2.x, k2.y))), vbits = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(v2.x, v2.y)));
                    any = __reduce_or_sync(0xffffffffu, any);
                    if (lane == 0) {
                        largest[stage * 4 + rw * 2] = kbits;
                        largest[stage * 4 + rw * 2 + 1] = vbits;
                        rated_nan[stage * 2 + rw] = any;
                    }
                    named_barrier<3, 64>();
                    kbits = max(largest[stage * 4], largest[stage * 4 + 2]);
                    vbits = max(largest[stage * 4 + 1], largest[stage * 4 + 3]);
                    any = rated_nan[stage * 2] | rated_nan[stage * 2 + 1];
                    const int xk = (int)max(kbits >> 23, 64u) - 127, xv = (int)max(vbits >> 23, 64u) - 127;
                    const float fk = power_of_two(T::K_TOP - xk), fv = power_of_two(T::V_TOP - xv);
                    // the tables of two steps ago have been read, and with them (the values' stage was free) that softmax's four steps ago
                    if (step >= 2) wait_or_give_up(bar(SCALES_EMPTY + stage), ((step >> 1) & 1u) ^ 1u, abort_flag);
#pragma unroll
                    for (int j = 0; j < KEYS; ++j) {
                        const uint32_t key = t + j * 64;
                        nans[ring * 128 + key] = (uint8_t)masks[j];
#pragma unroll
                        for (int k = 0; k < NB / 2; ++k) {
                            const float2 dk = __half22float2(as_h2(ks[j][k])), dv = __half22float2(as_h2(vs[j][k]));
                            *(__half2 *)(key_scales + (stage * KT + key) * NB + 2 * k) = __floats2half2_rn(dk.x * fk, dk.y * fk);
                            value_scales[(stage * NB + 2 * k) * KT + key] = __float2half_rn(dv.x * fv);
                            value_scales[(stage * NB + 2 * k + 1) * KT + key] = __float2half_rn(dv.y * fv);
                        }
                    }
                    if (t == 0) {
                        exponents[ring * 2] = xk - T::K_TOP;
                        exponents[ring * 2 + 1] = vbits ? xv - T::V_TOP : T::NO_VALUES;
                        any_nan[ring] = any;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(SCALES_FULL + stage));
                    if (i + 1 < sg.n) load(begin + (i + 1) * KT);
                }
            }
        }
    }
    __syncwarp();
    __syncthreads();
    if (warp == T::SOFT + T::PROD) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (tid == 0 && *abort_flag) *(volatile uint32_t *)(p.c.status + STATUS_WAIT) = 1u;
}

template <int W, bool K8, bool V8>
bool configure() {
    return cudaFuncSetAttribute(tile_kernel<W, K8, V8, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<W, K8, V8>::BYTES) == cudaSuccess &&
           cudaFuncSetAttribute(tile_kernel<W, K8, V8, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<W, K8, V8>::BYTES) == cudaSuccess;
}
template <int W, bool K8, bool V8>
int launch(cudaStream_t s, AttentionParams p, int sm_count) {
    using T = Tile<W, K8, V8>;
    p.tiles = (uint32_t)(((uint64_t)p.tokens * p.group + T::ROWS - 1) / T::ROWS);
    // What a row sees is at most the cache's capacity, and the window. Sums of values of one sign were up to 4e-4 too small over 100,000 positions (400,000 1.6e-3,
    // 1,500,000 1.1e-2; with the sums elsewhere 4e-4 over any number), a tenth of BF16's half step, and the loop without them is the faster one (2,048 rows of 40 heads on 8, width 128, at
    // 100,000 6,275 against 6,345 us, 20 on 4 of width 256 5,510 / 5,555; 1,024 rows at 400,000, width 64, 10,390 / 11,090).
    const uint64_t capacity = (uint64_t)p.c.granules * KV_GRANULE, seen = p.window ? std::min(capacity, (uint64_t)p.window + T::ROWS) : capacity;
    if (seen > 1u << 17) launch_after_previous_smem(tile_kernel<W, K8, V8, true>, dim3(sm_count), dim3(T::THREADS), T::BYTES, s, p);
    else launch_after_previous_smem(tile_kernel<W, K8, V8, false>, dim3(sm_count), dim3(T::THREADS), T::BYTES, s, p);
    return 1;
}
#define NU_EVERY(F, W, ...) (k8 ? (v8 ? F<W, true, true>(__VA_ARGS__) : F<W, true, false>(__VA_ARGS__)) : (v8 ? F<W, false, true>(__VA_ARGS__) : F<W, false, false>(__VA_ARGS__)))

}  // namespace

bool attention_tile_configure() {
    bool ok = true;
    for (int i = 0; i < 4; ++i) {
        const bool k8 = i & 1, v8 = i & 2;
        ok = ok && NU_EVERY(configure, 64) && NU_EVERY(configure, 128) && NU_EVERY(configure, 256);
    }
    return ok;
}

// From 128 query rows a key/value head, whatever the position. The kernel for few rows has a smaller fixed cost and takes time with rows x positions x heads; this
// one hardly does. Measured (few rows / this one, us; Q8_0 keys, Q4_0 values, rows a head at a position):
//   8 heads of width 128: 128 rows at 300 17 / 37, at 2,000 29 / 51, at 8,000 66 / 75; 256 rows 16 / 41, 38 / 53, 109 / 78; 512 rows 23 / 41, 70 / 55, 201 / 79;
//     1,024 rows 35 / 43, 123 / 55, 383 / 102
//   4 heads of width 256: 128 rows 23 / 39, 33 / 57, 68 / 86; 256 rows 23 / 40, 43 / 58, 107 / 87; 1,024 rows 29 / 40, 114 / 53, 358 / 84
//   8 heads of width 64: 128 rows 14 / 33, 21 / 45, 39 / 66; 512 rows 18 / 35, 39 / 49, 111 / 68; 1,024 rows 28 / 37, 75 / 47, 205 / 88
//   32 heads of width 128: 128 rows 23 / 41, 70 / 54, 201 / 99; 512 rows 86 / 49, 201 / 70, 738 / 164
// So they meet near rows x positions x heads x width = 2^29, and this rule is 20 to 28 us slower than the better kernel for a short prompt at the start of a
// session (up to 2.6 times), for up to ten times that gained on a long one. What it would take to do better, the positions, is in the spans on the device; all
// that the host has is the capacity, which in a session's cache is far above them.
bool attention_tile_supported(const AttentionJob &j) {
    const uint32_t w = j.cache.width;
    return j.bf16 && (w == 64 || w == 128 || w == 256) && (uint64_t)j.tokens * (j.heads / j.cache.heads) >= 128;
}

int launch_attention_tile(cudaStream_t s, const AttentionJob &j, AttentionParams p) {
    const bool k8 = j.cache.k8, v8 = j.cache.v8;
    const uint32_t w = j.cache.width;
    if (w == 64) return NU_EVERY(launch, 64, s, p, j.sm_count);
    if (w == 128) return NU_EVERY(launch, 128, s, p, j.sm_count);
    return NU_EVERY(launch, 256, s, p, j.sm_count);
}

}  // namespace nu
