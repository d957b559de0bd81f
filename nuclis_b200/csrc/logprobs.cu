// Log probabilities of given tokens, the entropy of each row's distribution and its most likely alternatives, in one pass
// over the logits:
//
//     m = max_i x_i,  Z = sum_i e^(x_i - m),  log p_t = (x_t - m) - ln Z,  H = ln Z - (sum_i (x_i - m) e^(x_i - m)) / Z
//
// Every thread keeps (m, Z, sum) of its share online, raising m once per batch of 16 values. The alternatives are kept
// by each warp on its own, so that no barrier stands in the loop: after its first 512 values the k-th largest of the lanes' maxima
// bounds the k-th largest value from below, so only the few values above it become candidates (64-bit keys: the
// value's order, then the lower index), and later only what passes the k-th candidate kept; the candidates are cut back to k when
// eight more have come (each cut raises the bar, and what passes it costs the whole warp a look at its values). A row is cut over several blocks when there are few rows; the block that arrives last joins them in block order.
#include "kernels.hpp"
#include "launch.cuh"

namespace nu {

namespace {

constexpr int MAX_K = (int)LOGPROB_ALTERNATIVES;
constexpr int THREADS = 256, WARPS = THREADS / 32, EACH = 16, ROUND = THREADS * EACH;
constexpr int RESIDENT = 4;                 // blocks a multiprocessor: 64 registers a thread, for two rounds of values
constexpr int WARP_ROUND = 32 * EACH, CUT = 8, WARP_CANDIDATES = WARP_ROUND + MAX_K + CUT;  // a round on top of what is not yet cut back
constexpr int CANDIDATES = WARPS * WARP_CANDIDATES;
constexpr uint32_t SPLITS_MAX = 256;
constexpr int FEW = 256;                    // candidates that are ranked by counting
constexpr int RECORD = 4 + 2 * MAX_K;       // floats a block leaves: m, Z, sum, bad, then the keys

struct Params {
    LogprobJob j;
    uint32_t splits, piece;  // blocks a row, logits a block
};

__device__ __forceinline__ uint32_t order(float x) {  // larger floats have larger keys; both zeros the same
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
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
    const uint32_t tid = threadIdx.x, row = blockIdx.x / p.splits, split = blockIdx.x % p.splits, k = j.k;
    wait_for_previous_operator();
    const float *x = j.logits + (size_t)row * j.stride;
    // a block's piece starts on a 16-byte boundary: the first also has the values ahead of it
    const uint32_t ahead = (uint32_t)((16 - ((uintptr_t)x & 15)) & 15) / 4;
    const uint32_t begin = split == 0 ? 0 : min(j.count, ahead + split * p.piece), end = split + 1 == p.splits ? j.count : min(j.count, ahead + (split + 1) * p.piece);
    const uint32_t shift = split == 0 ? (4 - ahead) % 4 : 0;  // values of the first vector that lie before the row
    const uint32_t lane = tid & 31, warp = tid / 32;
    unsigned long long *own = sh.candidates + warp * WARP_CANDIDATES;
    if (lane == 0) sh.counts[warp] = 0;
    __syncwarp();

    Stats s{-INFINITY, 0.0f, 0.0f, 0u};
    uint32_t floor = 0;      // order of the k-th value this warp has kept: later equals have higher indexes and lose
    const int n = (int)(end - begin + shift);  // of the piece, from the vector that holds its first value
    const float *v = x + begin - shift;
    auto load = [&](float (&to)[EACH], int r0) {
#pragma unroll
        for (int q = 0; q < EACH / 4; ++q) {
            const int i = r0 + (q * THREADS + (int)tid) * 4;
            if (i >= (int)shift && i + 4 <= n) {
                const float4 f = __ldcs((const float4 *)(v + i));
                to[q * 4] = f.x; to[q * 4 + 1] = f.y; to[q * 4 + 2] = f.z; to[q * 4 + 3] = f.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) to[q * 4 + c] = i + c >= (int)shift && i + c < n ? v[i + c] : -INFINITY;
            }
        }
    };
    float next[EACH];  // the round after is on its way while one is worked on
    load(next, 0);
    for (int r0 = 0; r0 < n; r0 += ROUND) {
        float a[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) a[i] = next[i];
        if (r0 + ROUND < n) load(next, r0 + ROUND);
        float top = a[0];
        bool nan = false;
#pragma unroll
        for (int i = 0; i < EACH; ++i) { top = fmaxf(top, a[i]); nan |= a[i] != a[i]; }
        if (nan || top == INFINITY) s.bad = 1;
        if (top > s.m) s.raise(top);
        const float m = s.m == -INFINITY ? 0.0f : s.m;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const float d = a[i] - m;
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * 1.4426950408889634f));
            s.z += e;
            s.w = fmaf(fmaxf(d, -1000.0f), e, s.w);  // the bound only meets terms whose e is zero
        }
        if (k == 0) continue;
        const uint32_t mine = order(top);
        const uint32_t hopeful = __ballot_sync(0xffffffffu, mine > floor);
        if (hopeful == 0) continue;
        uint32_t bound = floor;
        if (__popc(hopeful) >= (int)k) {  // only what reaches the k-th largest of the lanes' maxima can be among the k largest
            uint32_t above = 0;  // lanes ahead of this one, equals by number
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t o = __shfl_sync(0xffffffffu, mine, i);
                above += o > mine || (o == mine && i < (int)lane);
            }
            bound = max(floor, __reduce_max_sync(0xffffffffu, above == k - 1 ? mine - 1 : 0u));  // (an order is never zero)
        }
        if (mine > bound) {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int at = r0 + ((i / 4) * THREADS + (int)tid) * 4 + i % 4;
                const uint32_t o = order(a[i]);
                if (o > bound && at >= (int)shift && at < n) own[atomicAdd(&sh.counts[warp], 1u)] = key_of(o, begin + (uint32_t)at - shift);
            }
        }
        __syncwarp();
        const uint32_t c = sh.counts[warp];
        if (c >= k && (floor == 0 || c > k + CUT)) {
            cut_back(own, c, k);
            if (lane == 0) sh.counts[warp] = k;
            floor = (uint32_t)(own[k - 1] >> 32);
        }
        __syncwarp();
    }
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
    if (p.splits == 1) {
        write_row(j, sh, s, row);
        return;
    }

    // ---- several blocks a row: the last one joins ----
    float *records = j.partials + (size_t)row * p.splits * RECORD;
    float *mine = records + (size_t)split * RECORD;
    if (tid == 0) { mine[0] = s.m; mine[1] = s.z; mine[2] = s.w; mine[3] = __uint_as_float(s.bad); }
    if (tid < k) ((unsigned long long *)(mine + 4))[tid] = sh.kept[tid];
    __threadfence();
    __syncthreads();
    if (tid == 0) sh.last = atomicAdd(j.counters + row, 1u) == p.splits - 1;
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    Stats all{-INFINITY, 0.0f, 0.0f, 0u};
    if (tid < p.splits) {
        const float *r = records + (size_t)tid * RECORD;
        all = {__ldcg(r), __ldcg(r + 1), __ldcg(r + 2), __float_as_uint(__ldcg(r + 3))};
    }
    __syncthreads();
    all = block_stats(sh, all);
    if (k) {
        // the k-th largest of the pieces' first candidates bounds what can be among the k largest, as above
        uint32_t bound = 0;
        sh.maxima[tid] = tid < p.splits ? (uint32_t)(__ldcg((const unsigned long long *)(records + (size_t)tid * RECORD + 4)) >> 32) : 0u;
        if (tid == 0) { sh.bound = 0; sh.count = 0; }
        __syncthreads();
        if (p.splits > k) {
            uint32_t above = 0;
            for (uint32_t i = 0; i < THREADS; ++i) above += sh.maxima[i] > sh.maxima[tid] || (sh.maxima[i] == sh.maxima[tid] && i < tid);
            if (above == k - 1) sh.bound = sh.maxima[tid];
            __syncthreads();
            bound = sh.bound;
        }
        for (uint32_t i = tid; i < p.splits * k; i += THREADS) {
            const unsigned long long key = __ldcg((const unsigned long long *)(records + (size_t)(i / k) * RECORD + 4) + i % k);
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
    if (tid == 0) j.counters[row] = 0;
}

}  // namespace

int launch_token_logprobs(cudaStream_t s, const LogprobJob &j) {
    // Cuts of a row: the ones whose blocks fill whole waves best, a block's start and join counted as five rounds; never less than a
    // round a block.
    Params p{j, 1, j.count};
    const uint32_t slots = (uint32_t)j.sm_count * RESIDENT, rounds = (j.count + ROUND - 1) / ROUND;
    const uint32_t join = CANDIDATES / (j.k ? j.k : 1);  // the joining block holds every piece's candidates
    uint32_t most = rounds < SPLITS_MAX ? rounds : SPLITS_MAX, splits = 1;
    if (most > join) most = join;
    unsigned long long best = ~0ull;
    for (uint32_t c = 1; c <= most; ++c) {
        const unsigned long long waves = ((unsigned long long)j.rows * c + slots - 1) / slots, cost = waves * ((rounds + c - 1) / c + 5) + (c > 1);
        if (cost < best) { best = cost; splits = c; }
    }
    if (splits > 1 && j.rows <= j.counters_len && (size_t)j.rows * splits * RECORD <= j.partials_floats) {
        p.piece = ((j.count + splits - 1) / splits + 3) / 4 * 4;
        p.splits = (j.count + p.piece - 1) / p.piece;
    }
    launch_after_previous_smem(token_logprobs_kernel, dim3(j.rows * p.splits), dim3(THREADS), sizeof(Shared), s, p);
    return 1;
}

}  // namespace nu
