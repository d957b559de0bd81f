// Log probabilities of given tokens, the entropy of each row's distribution and its most likely alternatives, in one pass
// over the logits:
//
//     m = max_i x_i,  Z = sum_i e^(x_i - m),  log p_t = (x_t - m) - ln Z,  H = ln Z - (sum_i (x_i - m) e^(x_i - m)) / Z
//
// Every thread keeps (m, Z, sum) of its share online, raising m once per batch of 16 values, whose sums join the share's as one term each: term
// by term those of the bulk are lost next to a clear candidate's one (results of 509 rows 2.6e-7 off 64 bits; so it is 6e-8, and as fast). ex2.approx of the
// rounded product with log2(e) is off by 2^-22 and up to 2^-24 |x - m|, of random sign over the values: less than F32's own rounding of the result. The alternatives are kept
// by each warp on its own, so that no barrier stands in the loop: after its first 512 values the k-th largest of the lanes' maxima
// bounds the k-th largest value from below, so only the few values above it become candidates (64-bit keys: the
// value's order, then the lower index), and later only what passes the k-th candidate kept; the candidates are cut back to k when
// eight more have come (each cut raises the bar, and what passes it costs the whole warp a look at its values).
//
// The rounds of 4096 values of all rows are laid end to end and every block takes the same number of them, so that all end
// together; a row that several blocks share is joined by the one that arrives last, in block order.
//
// Bound by memory where there are many rows: 509 rows of 248,320 107 us, 4.7 TB/s, 73 % of a copy (127 us before
// the equal shares and with a longer round, 111 with a bar of each warp's own instead of a shared one). One row of 248,320 is 61 blocks of one round, the ranking and the join: 16.6 us.
#include "kernels.hpp"
#include "launch.cuh"

namespace nu {

namespace {

constexpr int MAX_K = (int)LOGPROB_ALTERNATIVES;
constexpr int THREADS = 256, WARPS = THREADS / 32, EACH = 16, ROUND = THREADS * EACH;
constexpr int RESIDENT = 3;                 // blocks a multiprocessor: 85 registers a thread, for two rounds of values
constexpr int WARP_ROUND = 32 * EACH, CUT = 8, WARP_CANDIDATES = WARP_ROUND + MAX_K + CUT;  // a round on top of what is not yet cut back
constexpr int CANDIDATES = WARPS * WARP_CANDIDATES;
constexpr uint32_t PARTS_MAX = 128;         // blocks that share a row: what the joining block ranks
static_assert(PARTS_MAX * MAX_K <= (uint32_t)CANDIDATES && PARTS_MAX <= (uint32_t)THREADS, "the joining block holds every part's candidates");
constexpr int FEW = 256;                    // candidates that are ranked by counting
constexpr int RECORD = 4 + 2 * MAX_K;       // floats a block leaves: m, Z, sum, bad, then the keys

static_assert(SCRATCH_SMS * RESIDENT * 2 * RECORD <= SCRATCH_FLOATS && SCRATCH_SMS * RESIDENT <= SCRATCH_COUNTERS, "the handle's scratch");

struct Params {
    LogprobJob j;
    uint32_t rounds, share;  // rounds a row, rounds a block
};

__device__ __forceinline__ uint32_t order(float x) {  // larger floats have larger keys; both zeros the same
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t LOWEST = 0x00800000u;  // the order of the lowest finite value (minus infinity's is one less)
__device__ __forceinline__ float unorder(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ unsigned long long key_of(uint32_t ord, uint32_t index) { return (unsigned long long)ord << 32 | (0xffffffffu - index); }

struct Stats {
    float m, z, w;
    uint32_t bad;
    __device__ __forceinline__ void raise(float next) {  // to a maximum next > m
        if (z > 0.0f) {
            const float d = m - next, f = expf(d);
            w = f > 0.0f ? (w + d * z) * f : 0.0f;  // d z overflows where f is long zero
            z *= f;
        }
        m = next;
    }
};

struct Shared {
    unsigned long long candidates[CANDIDATES];
    unsigned long long kept[MAX_K];
    unsigned long long best[WARPS];
    uint32_t counts[WARPS];
    uint32_t maxima[THREADS];
    Stats stats[WARPS];
    uint32_t count, bound, last;
    uint32_t bar;  // what the k-th value of some warp lies above: the others look no lower
};

__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == high ? (uint32_t)v : 0u);
    return (unsigned long long)high << 32 | low;
}

// The k largest of a warp's candidates c[0..n), n >= k, to the front in falling order. One warp.
__device__ __forceinline__ void cut_back(unsigned long long *c, uint32_t n, uint32_t k) {
    const uint32_t lane = threadIdx.x & 31;
    if (n <= 64) {  // by counting what is larger
        const unsigned long long x = lane < n ? c[lane] : 0, y = lane + 32 < n ? c[lane + 32] : 0;
        uint32_t above_x = 0, above_y = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < n; ++i) {
            const unsigned long long z = c[i];
            above_x += z > x;
            above_y += z > y;
        }
        __syncwarp();
        if (x && above_x < k) c[above_x] = x;
        if (y && above_y < k) c[above_y] = y;
        __syncwarp();
        return;
    }
    unsigned long long mine = 0, kept = 0;
    for (uint32_t i = lane; i < n; i += 32) mine = max(mine, c[i]);
    for (uint32_t r = 0; r < k; ++r) {
        const unsigned long long top = warp_max(mine);
        if (lane == r) kept = top;
        if (mine == top) {  // keys are distinct: one lane
            unsigned long long next = 0;
            for (uint32_t i = lane; i < n; i += 32)
                if (c[i] < top) next = max(next, c[i]);
            mine = next;
        }
    }
    __syncwarp();
    if (lane < k) c[lane] = kept;
    __syncwarp();
}

// The k largest of sh.candidates[0..n) into sh.kept, in falling order; zero where there are fewer. All threads; n is uniform.
__device__ __forceinline__ void select(Shared &sh, uint32_t n, uint32_t k) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    if (n <= FEW) {
        const unsigned long long mine = tid < n ? sh.candidates[tid] : 0;
        uint32_t above = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < n; ++i) above += sh.candidates[i] > mine;
        if (tid < k) sh.kept[tid] = 0;
        __syncthreads();
        if (mine && above < k) sh.kept[above] = mine;
        __syncthreads();
        return;
    }
    unsigned long long mine = 0;
    for (uint32_t i = tid; i < n; i += THREADS) mine = max(mine, sh.candidates[i]);
    for (uint32_t r = 0; r < k; ++r) {
        const unsigned long long w = warp_max(mine);
        if (lane == 0) sh.best[warp] = w;
        __syncthreads();
        unsigned long long top = sh.best[0];
#pragma unroll
        for (int i = 1; i < WARPS; ++i) top = max(top, sh.best[i]);
        if (tid == 0) sh.kept[r] = top;
        if (mine == top) {  // keys are distinct: one thread
            unsigned long long next = 0;
            for (uint32_t i = tid; i < n; i += THREADS)
                if (sh.candidates[i] < top) next = max(next, sh.candidates[i]);
            mine = next;
        }
        __syncthreads();
    }
}

// The block's, in every thread: the largest m of all first, so that each part is scaled once.
__device__ __forceinline__ Stats block_stats(Shared &sh, Stats s) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    auto all = [&](Stats x, float m) {  // x brought to the maximum m, summed over the warp
        const uint32_t bad = __reduce_or_sync(0xffffffffu, x.bad);
        const float d = x.m - m, f = x.z > 0.0f ? expf(d) : 0.0f;
        float w = f > 0.0f ? (x.w + d * x.z) * f : 0.0f, z = f > 0.0f ? x.z * f : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            z += __shfl_xor_sync(0xffffffffu, z, o);
            w += __shfl_xor_sync(0xffffffffu, w, o);
        }
        return Stats{m, z, w, bad};
    };
    s = all(s, unorder(__reduce_max_sync(0xffffffffu, order(s.m))));
    if (lane == 0) sh.stats[warp] = s;
    __syncthreads();
    s = lane < WARPS ? sh.stats[lane] : Stats{-INFINITY, 0.0f, 0.0f, 0u};
    return all(s, unorder(__reduce_max_sync(0xffffffffu, order(s.m))));
}

__device__ __forceinline__ void write_row(const LogprobJob &j, const Shared &sh, const Stats &s, uint32_t row) {
    const uint32_t tid = threadIdx.x;
    const float ln = logf(s.z);
    const bool empty = !(s.z > 0.0f);  // nothing above minus infinity
    if (tid == 0) {
        const uint32_t token = j.tokens[row];
        const float x = token < j.count ? j.logits[(size_t)row * j.stride + token] : NAN;
        j.logprobs[row] = s.bad ? NAN : empty && token < j.count ? -INFINITY : (x - s.m) - ln;
        j.entropies[row] = s.bad ? NAN : empty ? 0.0f : fmaxf(ln - s.w / s.z, 0.0f);
    }
    if (tid < j.k) {
        const unsigned long long key = sh.kept[tid];
        j.top[(size_t)row * j.k + tid] = s.bad ? 0xffffffffu : 0xffffffffu - (uint32_t)key;
        j.top_logprobs[(size_t)row * j.k + tid] = s.bad ? NAN : empty ? -INFINITY : (unorder((uint32_t)(key >> 32)) - s.m) - ln;
    }
}

__global__ void __launch_bounds__(THREADS, RESIDENT) token_logprobs_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(16) uint8_t raw[];
    Shared &sh = *(Shared *)raw;
    const LogprobJob &j = p.j;
    const uint32_t tid = threadIdx.x, k = j.k, lane = tid & 31, warp = tid / 32;
    unsigned long long *own = sh.candidates + warp * WARP_CANDIDATES;
    wait_for_previous_operator();
    const unsigned long long total = (unsigned long long)j.rows * p.rounds, last_round = min(total, (blockIdx.x + 1ull) * p.share);
    for (unsigned long long at_round = (unsigned long long)blockIdx.x * p.share; at_round < last_round;) {
    // this block's part of the row: rounds [r_begin, r_end); the row is that of blocks c0 .. c1
    const uint32_t row = (uint32_t)(at_round / p.rounds), r_begin = (uint32_t)(at_round % p.rounds);
    const uint32_t r_end = (uint32_t)min((unsigned long long)p.rounds, r_begin + (last_round - at_round));
    const uint32_t c0 = (uint32_t)((unsigned long long)row * p.rounds / p.share), c1 = (uint32_t)(((unsigned long long)(row + 1) * p.rounds - 1) / p.share);
    at_round += r_end - r_begin;
    const float *x = j.logits + (size_t)row * j.stride;
    // a part starts on a 16-byte boundary: the first also has the values ahead of it
    const uint32_t ahead = (uint32_t)((16 - ((uintptr_t)x & 15)) & 15) / 4;
    const uint32_t begin = r_begin == 0 ? 0 : min(j.count, ahead + r_begin * ROUND), end = r_end == p.rounds ? j.count : min(j.count, ahead + r_end * ROUND);
    const uint32_t shift = r_begin == 0 ? (4 - ahead) % 4 : 0;  // values of the first vector that lie before the row
    if (lane == 0) sh.counts[warp] = 0;
    if (tid == 0) sh.bar = 0;
    __syncthreads();

    Stats s{-INFINITY, 0.0f, 0.0f, 0u};
    uint32_t floor = 0;      // order of the k-th value this warp has kept: later equals have higher indexes and lose
    const int n = (int)(end - begin + shift);  // of the piece, from the vector that holds its first value
    const float *v = x + begin - shift;
    auto load = [&](float (&to)[EACH], int r0) {
        if (r0 >= n) return;
        const float *src = v + r0 + (int)tid * 4;
        if (r0 >= (int)shift && r0 + ROUND <= n) {
#pragma unroll
            for (int q = 0; q < EACH / 4; ++q) {
                const float4 f = __ldcs((const float4 *)(src + q * THREADS * 4));
                to[q * 4] = f.x; to[q * 4 + 1] = f.y; to[q * 4 + 2] = f.z; to[q * 4 + 3] = f.w;
            }
        } else {  // a part's first or last round
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int at = r0 + (i / 4 * THREADS + (int)tid) * 4 + i % 4;
                to[i] = at >= (int)shift && at < n ? v[at] : -INFINITY;
            }
        }
    };
    auto work = [&](const float (&a)[EACH], int r0) {
        float top = a[0];
#pragma unroll
        for (int i = 1; i < EACH; ++i) top = fmaxf(top, a[i]);  // (a NaN shows in the sum)
        if (top == INFINITY) s.bad = 1;
        if (top > s.m) s.raise(top);
        const float m = s.m == -INFINITY ? 0.0f : s.m;
        float z = 0.0f, w = 0.0f;  // of the batch
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const float d = a[i] - m;
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * 1.4426950408889634f));
            z += e;
            w = fmaf(fmaxf(d, -1000.0f), e, w);  // the bound only meets terms whose e is zero
        }
        s.z += z;
        s.w += w;
        if (k == 0) return;
        const uint32_t mine = order(top), least = max(floor, *(volatile uint32_t *)&sh.bar);
        const uint32_t hopeful = __ballot_sync(0xffffffffu, mine > least);
        if (hopeful == 0) return;
        uint32_t bound = __reduce_max_sync(0xffffffffu, least);
        if (__popc(hopeful) >= (int)k) {  // only what reaches the k-th largest of the lanes' maxima can be among the k largest
            uint32_t above = 0;  // lanes ahead of this one, equals by number
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t o = __shfl_sync(0xffffffffu, mine, i);
                above += o > mine || (o == mine && i < (int)lane);
            }
            bound = max(bound, __reduce_max_sync(0xffffffffu, above == k - 1 ? mine - 1 : 0u));  // (an order is never zero)
        }
        // which of the lane's values pass: compared as floats, unless minus infinities count too (the row has had fewer than k others)
        uint32_t passed = 0;
        if (bound >= LOWEST) {
            const float limit = unorder(bound == 0x7fffffffu ? bound - 1 : bound);  // (just below zero is not minus zero, which equals it)
#pragma unroll
            for (int i = 0; i < EACH; ++i) passed |= (uint32_t)(a[i] > limit) << i;
        } else {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int at = r0 + (i / 4 * THREADS + (int)tid) * 4 + i % 4;
                passed |= (uint32_t)(order(a[i]) > bound && at >= (int)shift && at < n) << i;
            }
        }
        while (passed) {  // few
            const int i = __ffs(passed) - 1;
            passed &= passed - 1;
            const int at = r0 + (i / 4 * THREADS + (int)tid) * 4 + i % 4;
            float x_i = a[0];
#pragma unroll
            for (int j = 1; j < EACH; ++j) x_i = j == i ? a[j] : x_i;
            own[atomicAdd(&sh.counts[warp], 1u)] = key_of(order(x_i), begin + (uint32_t)at - shift);
        }
        __syncwarp();
        const uint32_t c = sh.counts[warp];
        if (c >= k && (floor == 0 || c > k + CUT)) {
            cut_back(own, c, k);
            floor = (uint32_t)(own[k - 1] >> 32);
            if (lane == 0) {
                sh.counts[warp] = k;
                atomicMax(&sh.bar, floor - 1);  // equals elsewhere may have lower indexes
            }
        }
        __syncwarp();
    };
    float next[EACH];  // the round after is on its way while one is worked on
    load(next, 0);
#pragma unroll 1
    for (int r0 = 0; r0 < n; r0 += ROUND) {
        float a[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) a[i] = next[i];
        load(next, r0 + ROUND);
        work(a, r0);
    }
    if (s.z != s.z) s.bad = 1;
    if (k) {  // the warps' candidates together: what one has at most between cuts, or its k where that is too many to rank
        const uint32_t each = WARPS * (k + CUT) <= (uint32_t)FEW ? k + CUT : k;
        if (sh.counts[warp] > each) {
            cut_back(own, sh.counts[warp], k);
            if (lane == 0) sh.counts[warp] = k;
            __syncwarp();
        }
        const uint32_t c = sh.counts[warp];
        const unsigned long long key = lane < c ? own[lane] : 0, more = lane + 32 < c ? own[lane + 32] : 0;
        __syncthreads();
        if (lane < each) sh.candidates[warp * each + lane] = key;
        if (lane + 32 < each) sh.candidates[warp * each + lane + 32] = more;
        __syncthreads();
        select(sh, WARPS * each, k);
    }
    s = block_stats(sh, s);
    if (c0 == c1) {
        write_row(j, sh, s, row);
        __syncthreads();
        continue;
    }

    // ---- several blocks a row: the last one joins ----
    const uint32_t parts = c1 - c0 + 1;
    auto record = [&](uint32_t c) { return j.partials + ((size_t)(c0 + c) * 2 + (c == 0)) * RECORD; };  // a block's second place: the row that starts in it
    float *mine = record(blockIdx.x - c0);
    if (tid == 0) { mine[0] = s.m; mine[1] = s.z; mine[2] = s.w; mine[3] = __uint_as_float(s.bad); }
    if (tid < k) ((unsigned long long *)(mine + 4))[tid] = sh.kept[tid];
    __threadfence();
    __syncthreads();
    if (tid == 0) sh.last = atomicAdd(j.counters + c0, 1u) == parts - 1;
    __syncthreads();
    if (!sh.last) continue;  // (uniform; the next part's first barrier is behind this read)
    __threadfence();
    Stats all{-INFINITY, 0.0f, 0.0f, 0u};
    if (tid < parts) {
        const float *r = record(tid);
        all = {__ldcg(r), __ldcg(r + 1), __ldcg(r + 2), __float_as_uint(__ldcg(r + 3))};
    }
    __syncthreads();
    all = block_stats(sh, all);
    if (k) {
        // the k-th largest of the pieces' first candidates bounds what can be among the k largest, as above
        uint32_t bound = 0;
        sh.maxima[tid] = tid < parts ? (uint32_t)(__ldcg((const unsigned long long *)(record(tid) + 4)) >> 32) : 0u;
        if (tid == 0) { sh.bound = 0; sh.count = 0; }
        __syncthreads();
        if (parts > k) {
            uint32_t above = 0;
            for (uint32_t i = 0; i < THREADS; ++i) above += sh.maxima[i] > sh.maxima[tid] || (sh.maxima[i] == sh.maxima[tid] && i < tid);
            if (above == k - 1) sh.bound = sh.maxima[tid];
            __syncthreads();
            bound = sh.bound;
        }
        for (uint32_t i = tid; i < parts * k; i += THREADS) {
            const unsigned long long key = __ldcg((const unsigned long long *)(record(i / k) + 4) + i % k);
            if (key && (uint32_t)(key >> 32) >= bound) {
                const uint32_t at = atomicAdd(&sh.count, 1u);
                if (at < (uint32_t)CANDIDATES) sh.candidates[at] = key;
            }
        }
        __syncthreads();
        const uint32_t c = sh.count;
        select(sh, c, k);
    }
    write_row(j, sh, all, row);
    if (tid == 0) j.counters[c0] = 0;
    __syncthreads();
    }
}

}  // namespace

int launch_token_logprobs(cudaStream_t s, const LogprobJob &j) {
    // A block for every place on the multiprocessors, less when there are fewer rounds; no row over more than PARTS_MAX blocks.
    Params p{j, (j.count + ROUND - 1) / ROUND, 0};
    const unsigned long long total = (unsigned long long)j.rows * p.rounds, slots = (unsigned long long)j.sm_count * RESIDENT;
    const unsigned long long least = (p.rounds + PARTS_MAX - 2) / (PARTS_MAX - 1), even = (total + slots - 1) / slots;
    p.share = (uint32_t)(even > least ? even : least);
    launch_after_previous_smem(token_logprobs_kernel, dim3((unsigned)((total + p.share - 1) / p.share)), dim3(THREADS), sizeof(Shared), s, p);
    return 1;
}

}  // namespace nu
