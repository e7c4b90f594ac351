// Token ids from logits and random numbers (the host loop of mygrad/llama/llama_model.py:144-160, on the device).
//
// For a row x of logits, with T, k, p and r the row's temperature, top-k, top-p and min-p and u its random number in [0, 1):
//     w_i = exp((x_i - max x) / T);  order by value, the lower index first among equals
//     1. the first k                       2. of these, those before which less than p of their sum lies (the first always)
//     3. of these, those with w >= r (the first always)
//     the id: the lowest index i for which the sum of what is kept up to and with i is above u times the sum of all that is kept
// What is kept is always a prefix of the order, so that it is named by its last element.
//
// Sums decide which side of a border a token falls on, so they have to come out the same however the row is divided: weights are
// computed in fp64 (2^(i / 32) from a table, and 2^f for |f| <= 1/64 by seven terms of the exponential series, whose rest is below 4e-18)
// and summed as 64-bit whole numbers of 2^-s, s the largest up to 50 for which a row's sum fits in 62 bits (47 for 32000 tokens, 44 for 262144).  A weight
// above 0 counts at least one such unit.
//
// A cluster of CTAs per row, each with a part of the row in shared memory: read once.  The border of top-k is found by a histogram of
// counts over 512 steps of the value below the maximum, which every CTA joins for itself through distributed shared memory.  For top-p the
// same counts, with the largest and the smallest weight of each step, tell between which two steps the border must lie.  Every token is
// then weighed once: those above and below only go into sums, those between into a second histogram, of weights as three 16-bit limbs
// (whose sums over a CTA's part, 32768 tokens at most, fit the 32-bit atomics that shared memory has, where 64-bit ones take 50 times as
// long; over the cluster they are added in 64 bits), and the places of all that may be kept are put side by side for the choice.
// Where few tokens lie in the steps down to the border, all that is left is done with a list of them, by the cluster's first CTA: ranks,
// sums, choice.  Otherwise the few elements of the border's step are ranked among each other, and what is kept is passed over once
// more for the choice.  A step with too many (equal logits, far outliers) is divided again by (value, index) until it has not.
// A batch pays for the instructions per token: 256 rows of 32000 with top-p of 0.9 take 74 us, 0.44 TB/s: 115 instructions per token and
// 2300 per warp, at 62% of what the SMs can issue, in 1.7 waves (107 with every weight through the histogram, 155 with the tokens that cannot
// matter left out by a bound on their number alone, 83 with twelve terms of the series and no table).  Few rows pay for barriers of the
// cluster, about 1 us each, three with a short list and six without: a row of 32000 with top-k 50 takes 10.1 us, without any limit 5.7.
#include <math.h>

#include "hybrid.cuh"

namespace bn {

using namespace ptx;

constexpr int SMP_THREADS = 512;
constexpr int SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_BINS = SMP_THREADS;                 // a thread has one
constexpr int SMP_LIST = SMP_THREADS;                 // elements that are ranked among each other, a thread each
// Up to so many elements the row's choice is made with them alone: ranking m costs m^2 / 512 comparisons a thread, and saves other passes
// and barriers.  By top-k alone (16 x 4000, us with the list and without, k of 100: 8.8, 9.2; 150: 10.3, 9.2; 300: 14.3, 9.3), by top-p
// alone (what is kept up to 99: 11.4, 14.3; 291: 17.2, 14.2), and by top-k before top-p, which the list then does as well (k of 200: 10.3,
// 19.0; 300: 12.6, 19.1; 480: 17.3, 19.2).
constexpr int SMP_FEW_BY_COUNT = 128, SMP_FEW_BY_WEIGHT = 256;
constexpr int SMP_LOG_STEPS = 5, SMP_STEPS = 1 << SMP_LOG_STEPS;      // of a power of two, in a table
constexpr int SMP_CLUSTER = 8;                        // CTAs per row at most
constexpr int SMP_MOST = 32768;                       // tokens per CTA: 5 bytes of shared memory each
constexpr int SMP_TWO = 16384;                        // tokens per CTA of which an SM takes two
constexpr size_t SMP_MOST_SMEM = (size_t)SMP_MOST * 5;
constexpr int SMP_MOST_COLS = SMP_MOST * SMP_CLUSTER;

struct SampleParams {
    const void* x;
    int64_t row_stride;
    const float *u, *temperature, *top_p, *min_p;      // per row, or null: the numbers below
    const int32_t* top_k;
    float temperature1, top_p1, min_p1;
    int top_k1;
    int32_t* out;
    int bf16, cols, slice, unit_bits;                        // slice: tokens per CTA, a multiple of 4
};

// a logit as it is kept: NaN is -inf, -0 is 0
__device__ __forceinline__ float plain_logit(float v) { return v > -INFINITY ? v + 0.f : -INFINITY; }
// 32 bits in the order of the values, and back
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }

struct SampleShared {
    uint32_t hist[4][SMP_BINS];                        // counts, and the limbs of weights
    uint32_t coarse[SMP_BINS];                         // counts that say where to look
    uint64_t list_key[SMP_LIST];                       // this CTA's elements
    uint64_t all_key[SMP_LIST];                        // the cluster's
    uint32_t index[SMP_LIST];                          // of what is kept of it
    uint64_t from[2][SMP_CLUSTER * SMP_WARPS][2];      // what all warps of the cluster tell each other
    uint64_t warp_sum[2][SMP_WARPS];
    uint32_t warp_cnt[2][SMP_WARPS];
    struct { uint64_t above; uint32_t lane1, count, upto; } border[SMP_WARPS];
    struct { uint32_t lane1, lane2, upto; } between[SMP_WARPS];
    uint64_t sums[SMP_WARPS][2];
    uint64_t kept_sum;
    double exp2[SMP_STEPS];                            // 2^(i / SMP_STEPS)
    uint32_t rank[SMP_LIST];
    int list_n;
};

__device__ __forceinline__ uint64_t warp_total(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The part's logits into shared memory; f sees each
template <typename T, typename F> __device__ __forceinline__ void load_logits(const T* x, float* sx, int n, F f) {
    const bool wide = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0;
    if (wide) {
#pragma unroll 4
        for (int i = 4 * threadIdx.x; i + 4 <= n; i += 4 * SMP_THREADS) {
            float v[4];
            load4(x + i, v);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = plain_logit(v[e]);
                f(v[e], i + e);
            }
            *reinterpret_cast<float4*>(sx + i) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
#pragma unroll 4
    for (int i = (wide ? n / 4 * 4 : 0) + threadIdx.x; i < n; i += SMP_THREADS) {
        const float v = plain_logit(to_f(x[i]));
        sx[i] = v;
        f(v, i);
    }
}

__global__ void __launch_bounds__(SMP_THREADS, 2) sample_rows_kernel(const SampleParams p) {
    extern __shared__ __align__(16) float sx[];        // the part's logits, and 16-bit places of up to half of them
    __shared__ SampleShared sh;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    uint32_t ncta;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ncta));
    const int C = (int)ncta, rank = (int)cluster_rank(), r = blockIdx.x / C;
    const int first = rank * p.slice, n = max(0, min(p.slice, p.cols - first)), n4 = (n + 3) / 4;
    // a warp has a run of the part, so that its sum is one of neighbours; in pieces of four
    const int run = (n4 + SMP_WARPS * 32 - 1) / (SMP_WARPS * 32) * 32, begin = warp * run, end = min(n4, begin + run);
    uint16_t* places = reinterpret_cast<uint16_t*>(sx + p.slice) + 2 * begin;      // of the warp's run, from its start
    cluster_arrive();                                  // waited for before the first number that goes to another CTA: all have started then
    if (tid < SMP_STEPS) sh.exp2[tid] = exp2((double)tid / SMP_STEPS);
    grid_dependency_wait();
    grid_launch_dependents();

    // every warp of the cluster tells all CTAs two numbers; in sh.from[turn ^ 1] behind the barrier
    int turn = 0, turn2 = 0;
    auto tell_and_go_on = [&](uint64_t a, uint64_t b) {
        if (lane < C) {
            const uint32_t at = in_rank(smem_u32(&sh.from[turn][rank * SMP_WARPS + warp][0]), lane);
            st_cluster_u64(at, a);
            st_cluster_u64(at + 8, b);
        }
        cluster_arrive();
        turn ^= 1;
    };
    auto tell = [&](uint64_t a, uint64_t b) {
        tell_and_go_on(a, b);
        cluster_wait();
    };
    // sums over the lower threads of the block, of a wide number and a narrow one, and over all
    auto block_scan = [&](uint64_t v, uint32_t w, uint64_t& total, uint32_t& below_w) -> uint64_t {
        uint64_t sum = v;
        uint32_t sumw = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, sum, o);
            const uint32_t tw = __shfl_up_sync(0xffffffffu, sumw, o);
            if (lane >= o) { sum += t; sumw += tw; }
        }
        if (lane == 31) { sh.warp_sum[turn2][warp] = sum; sh.warp_cnt[turn2][warp] = sumw; }
        __syncthreads();
        uint64_t s = lane < SMP_WARPS ? sh.warp_sum[turn2][lane] : 0;
        uint32_t sw = lane < SMP_WARPS ? sh.warp_cnt[turn2][lane] : 0;
        turn2 ^= 1;
#pragma unroll
        for (int o = 1; o < SMP_WARPS; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, s, o);
            const uint32_t tw = __shfl_up_sync(0xffffffffu, sw, o);
            if (lane >= o) { s += t; sw += tw; }
        }
        total = __shfl_sync(0xffffffffu, s, SMP_WARPS - 1);
        const uint64_t below = __shfl_sync(0xffffffffu, s, max(warp - 1, 0));
        const uint32_t belowc = __shfl_sync(0xffffffffu, sw, max(warp - 1, 0));
        below_w = sumw - w + (warp ? belowc : 0);
        return sum - v + (warp ? below : 0);
    };

    // ------------------------------------------------------------------ the row's part, its largest and its smallest element
    float top = -INFINITY, low = INFINITY;
    uint32_t top_at = 0xffffffffu;
    {
        auto see = [&](float v, int i) {
            if (v > top) { top = v; top_at = first + i; }          // (a thread's indices ascend: the first of equals stays)
            low = fminf(low, v > -INFINITY ? v : INFINITY);
        };
        if (tid < n4 * 4 - n) sx[n + tid] = -INFINITY; // (behind the last one: whole pieces of four)
        const int64_t at = r * p.row_stride + first;
        if (p.bf16) load_logits(static_cast<const __nv_bfloat16*>(p.x) + at, sx, n, see);
        else load_logits(static_cast<const float*>(p.x) + at, sx, n, see);
    }
    // over a warp: the largest, the lowest index that has it, the smallest
    auto join = [&](uint32_t& top_order, uint32_t& low_order) {
        const uint32_t all = __reduce_max_sync(0xffffffffu, top_order);
        top_at = __reduce_min_sync(0xffffffffu, top_order == all ? top_at : 0xffffffffu);
        top_order = all;
        low_order = __reduce_min_sync(0xffffffffu, low_order);
    };
    uint32_t top_order = order_of(top), low_order = order_of(low);
    join(top_order, low_order);
    cluster_wait();
    tell_and_go_on((uint64_t)top_order << 32 | top_at, low_order);
    // (what the row's numbers alone say is worked out while the barrier is waited for; a temperature above 0 is one from 1e-30 to 3e38, for
    // which the steps of the value are finite: beyond, the weights are those at the end, but for logits less than 1e-27 apart)
    const float temp_given = p.temperature ? p.temperature[r] : p.temperature1, temp = temp_given > 0.f ? fminf(fmaxf(temp_given, 1e-30f), 3e38f) : 0.f;
    const int top_k = p.top_k ? p.top_k[r] : p.top_k1;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p1, min_p = p.min_p ? p.min_p[r] : p.min_p1;
    const double u = fmin(fmax((double)p.u[r], 0.0), 1.0);
    const double per = 1.4426950408889634 / (double)temp;
    const double per_step = per * SMP_STEPS;
    const int unit = p.unit_bits;
    const uint64_t floor_w = min_p > 0.f ? (uint64_t)ceil((double)fminf(min_p, 1.f) * (double)(1ull << unit)) : 0;      // least weight that min-p keeps
    cluster_wait();
    top_order = order_of(-INFINITY);
    for (int i = lane; i < C * SMP_WARPS; i += 32) {
        const uint64_t a = sh.from[turn ^ 1][i][0];
        const uint32_t o = (uint32_t)(a >> 32);
        if (o > top_order || (o == top_order && (uint32_t)a < top_at)) { top_order = o; top_at = (uint32_t)a; }
        low_order = min(low_order, (uint32_t)sh.from[turn ^ 1][i][1]);
    }
    join(top_order, low_order);
    float peak = value_of(top_order), depth = peak - value_of(low_order);
    if (peak == -INFINITY || !(temp > 0.f) || top_k == 1) {
        if (rank == 0 && tid == 0) p.out[r] = peak == -INFINITY ? 0 : (int)top_at;
        return;                                        // (nothing reaches into another CTA behind the last barrier)
    }
    if (peak == INFINITY) {                            // infinities share the weight
        __syncthreads();
        for (int i = tid; i < 4 * n4; i += SMP_THREADS) sx[i] = sx[i] == INFINITY ? 0.f : -INFINITY;
        peak = depth = 0.f;
        __syncthreads();
    }

    // 2^((v - peak) / T * log2 e) in units of 2^-unit, to the nearest whole number, at least 1; 0 where fp64 has none.  No branches: a
    // warp weighs different values.  The smallest values above one unit and above nothing are rounded up, so that they part exactly.
    const float one_unit = __double2float_ru((double)peak - unit / per), nothing = __double2float_ru((double)peak - 1074.5 / per);
    auto weigh = [&](float v) -> uint64_t {
        const double d = (double)v - (double)peak;
        const double rounded = fma(d, per_step, 0x1.8p52 + SMP_STEPS * unit);      // to a whole number of steps: with the unit's, the low word
        const double f = fma(d, per_step, (0x1.8p52 + SMP_STEPS * unit) - rounded);
        const int steps = __double2loint(rounded);
        const double power = sh.exp2[steps & (SMP_STEPS - 1)];
        // (ln 2 / 32)^i / i!
        double w = 1.4345655584131934e-13;
        w = fma(w, f, 3.973709984549416e-11);
        w = fma(w, f, 9.172562701824643e-09);
        w = fma(w, f, 1.693850972437182e-06);
        w = fma(w, f, 0.0002345961982022468);
        w = fma(w, f, 0.02166084939249829);
        w = fma(w, f, 1.0);
        // (what is left behind 2^52 are the low bits)
        w = fma(w, __hiloint2double(__double2hiint(power) + (steps >> SMP_LOG_STEPS << 20), __double2loint(power)), 0x1p52);
        const uint32_t hi = v >= one_unit ? (uint32_t)__double2hiint(w) - 0x43300000u : 0u;
        const uint32_t lo = v >= one_unit ? (uint32_t)__double2loint(w) : v >= nothing ? 1u : 0u;
        return (uint64_t)hi << 32 | lo;
    };

    // kept: above `last` in the order, or `last` itself
    float last = -INFINITY;
    int last_at = -1;
    auto kept = [&](float v, int i) { return v > last || (v == last && first + i <= last_at); };
    auto key_of = [&](float v, int i) { return (uint64_t)order_of(v) << 32 | (uint32_t)~(first + i); };

    // What `which` says of the warp's run is put side by side, its places in the order of the index, if that is half of it at most
    int held = -1;                                     // of the warp's run; -1: all of it is looked at
    auto compact = [&](auto which) {
        int at = 0;
        const uint32_t lower = (1u << lane) - 1;
        for (int q0 = begin; q0 < end; q0 += 32) {
            const int q = q0 + lane;
            const float4 four = q < end ? *reinterpret_cast<const float4*>(sx + 4 * q) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            const float v[4] = {four.x, four.y, four.z, four.w};
            bool in[4];
            int before = at, own = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) in[e] = which(v[e], 4 * q + e);
#pragma unroll
            for (int e = 0; e < 4; ++e) {              // (not in turn with the weights: their chains overlap)
                const uint32_t who = __ballot_sync(0xffffffffu, in[e]);
                before += __popc(who & lower);
                at += __popc(who);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (in[e]) {
                    if (before + own < 2 * (end - begin)) places[before + own] = (uint16_t)(4 * (q - begin) + e);
                    ++own;
                }
        }
        __syncwarp();
        held = at <= 2 * (end - begin) ? at : -1;
    };
    // calls f(value, index in the part) for what the thread looks at
    auto each = [&](auto f) {
        if (held >= 0) {
#pragma unroll 2
            for (int j = lane; j < held; j += 32) {
                const int i = 4 * begin + places[j];
                f(sx[i], i);
            }
        } else {
            for (int q = begin + lane; q < end; q += 32) {
                const float4 four = *reinterpret_cast<const float4*>(sx + 4 * q);
                f(four.x, 4 * q);
                f(four.y, 4 * q + 1);
                f(four.z, 4 * q + 2);
                f(four.w, 4 * q + 3);
            }
        }
    };

    // the same, and may leave out what is below `near`
    auto each_from = [&](float near, auto f) {
        if (held >= 0 || near == -INFINITY) return each(f);
        for (int q = begin + lane; q < end; q += 32) {
            const float4 four = *reinterpret_cast<const float4*>(sx + 4 * q);
            if (fmaxf(fmaxf(four.x, four.y), fmaxf(four.z, four.w)) < near) continue;
            f(four.x, 4 * q);
            f(four.y, 4 * q + 1);
            f(four.z, 4 * q + 2);
            f(four.w, 4 * q + 3);
        }
    };

    // The last element before which there is less than a limit: top_k by count, top_p times their sum by weight.  True: the choice has
    // been made with the list.
    auto cut = [&](bool by_weight, float range) -> bool {
        uint64_t above = 0, hi = 0, lo = 0;            // what lies above the steps; their range of keys, where they divide one
        int shift = -1, step = 0, m = 0, step1 = 0, step2 = SMP_BINS - 1;
        double limit = (double)top_k;
        bool listed = false;
        const float scale = range > 0.f ? fminf(SMP_BINS / range, 3e38f) : 0.f;      // (finite: what equals the maximum is in step 0)
        float edge = peak, scale2 = scale;             // of the steps between step1 and step2
        // (the rounding is to the nearest step: any will do that never puts the larger value behind the smaller)
        auto step_below = [&](float d) -> int { return (int)(__float_as_uint(fminf(d, SMP_BINS - 1.f) + 8388608.f) & (SMP_BINS - 1)); };
        auto coarse = [&](float v) -> int { return step_below((peak - v) * scale); };
        auto in_step = [&](float v, int i) -> int {    // -1: not in the range
            if (!kept(v, i)) return -1;
            if (shift < 0) {
                const int b = coarse(v);
                return !by_weight ? b : b < step1 || b > step2 ? -1 : step_below(fmaxf((edge - v) * scale2, 0.f));
            }
            const uint64_t key = key_of(v, i);
            return key > hi || key < lo ? -1 : (int)((hi - key) >> shift);
        };
        auto clear = [&]() {
            sh.hist[0][tid] = 0;
            if (by_weight) sh.coarse[tid] = sh.hist[1][tid] = sh.hist[2][tid] = sh.hist[3][tid] = 0;
            if (tid == 0) sh.list_n = 0;
            __syncthreads();
        };
        auto add = [&](int b, uint64_t w) {
            atomicAdd(&sh.hist[0][b], 1u);
            if (by_weight) {
                atomicAdd(&sh.hist[1][b], (uint32_t)w & 0xffffu);
                if (w >> 16) {
                    atomicAdd(&sh.hist[2][b], (uint32_t)(w >> 16) & 0xffffu);
                    if (w >> 32) atomicAdd(&sh.hist[3][b], (uint32_t)(w >> 32));
                }
            }
        };
        auto put = [&](float v, int i) {
            const int at = min(atomicAdd(&sh.list_n, 1), SMP_LIST - 1);      // (m of them in the whole cluster)
            sh.list_key[at] = key_of(v, i);
        };
        auto joined = [&](const uint32_t* row) -> uint64_t {       // the cluster's histogram at the thread's step
            uint64_t sum = 0;                          // (eight CTAs' sums of limbs have up to 34 bits)
#pragma unroll
            for (int c = 0; c < SMP_CLUSTER; ++c)
                if (c < C) sum += ld_cluster_u32(in_rank(smem_u32(row + tid), c));
            return sum;
        };

        clear();
        if (by_weight) {
            if (last == -INFINITY) {
                each([&](float v, int) {
                    if (v > -INFINITY) atomicAdd(&sh.coarse[coarse(v)], 1u);
                });
            } else {
                each([&](float v, int i) {
                    if (kept(v, i)) atomicAdd(&sh.coarse[coarse(v)], 1u);
                });
            }
            cluster_sync();
            const uint32_t cnt = (uint32_t)joined(sh.coarse);
            // the step's weights lie between these, its sums between theirs (a thousandth of a step and 1e-4 for the roundings)
            const float wide = range / SMP_BINS / temp, most = tid == 0 ? 1.f : __expf(-(tid - 0.501f) * wide), least = tid == SMP_BINS - 1 ? 0.f : __expf(-(tid + 0.501f) * wide);
            float a = cnt * most, b = cnt ? cnt * least : 0.f;
            uint32_t upto = cnt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const float ta = __shfl_up_sync(0xffffffffu, a, o), tb = __shfl_up_sync(0xffffffffu, b, o);
                const uint32_t tc = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) { a += ta; b += tb; upto += tc; }
            }
            if (lane == 31) { sh.sums[warp][0] = (uint64_t)__float_as_uint(a) << 32 | __float_as_uint(b); sh.sums[warp][1] = upto; }
            __syncthreads();
            const uint64_t ab = sh.sums[lane % SMP_WARPS][0];
            float all_a = __uint_as_float((uint32_t)(ab >> 32)), all_b = __uint_as_float((uint32_t)ab);
            uint32_t all_c = (uint32_t)sh.sums[lane % SMP_WARPS][1];
#pragma unroll
            for (int o = 1; o < SMP_WARPS; o <<= 1) {
                const float ta = __shfl_up_sync(0xffffffffu, all_a, o), tb = __shfl_up_sync(0xffffffffu, all_b, o);
                const uint32_t tc = __shfl_up_sync(0xffffffffu, all_c, o);
                if (lane >= o) { all_a += ta; all_b += tb; all_c += tc; }
            }
            const float low_a = warp ? __shfl_sync(0xffffffffu, all_a, warp - 1) : 0.f, low_b = warp ? __shfl_sync(0xffffffffu, all_b, warp - 1) : 0.f;
            // of the steps before this one.  (Not the sum less the step's own part: of 1e5 tokens in a step nothing would be left of 1e-4.)
            const float ta = __shfl_up_sync(0xffffffffu, a, 1), tb = __shfl_up_sync(0xffffffffu, b, 1);
            const float before_a = low_a + (lane ? ta : 0.f), before_b = low_b + (lane ? tb : 0.f);
            upto += warp ? __shfl_sync(0xffffffffu, all_c, warp - 1) : 0;
            all_a = __shfl_sync(0xffffffffu, all_a, SMP_WARPS - 1);
            all_b = __shfl_sync(0xffffffffu, all_b, SMP_WARPS - 1);
            const uint32_t first_ok = __ballot_sync(0xffffffffu, cnt && before_a * 1.0001f < top_p * all_b * 0.9999f);
            const uint32_t last_ok = __ballot_sync(0xffffffffu, cnt && before_b * 0.9999f <= top_p * all_a * 1.0001f);
            if (lane == (last_ok ? 31 - __clz(last_ok) : 0)) {
                sh.between[warp].lane1 = first_ok ? 32 - __clz(first_ok) : 0;
                sh.between[warp].lane2 = last_ok ? 32 - __clz(last_ok) : 0;
                sh.between[warp].upto = upto;
            }
            __syncthreads();
            const uint32_t w1 = __ballot_sync(0xffffffffu, lane < SMP_WARPS && sh.between[lane % SMP_WARPS].lane1 != 0);
            const uint32_t w2 = __ballot_sync(0xffffffffu, lane < SMP_WARPS && sh.between[lane % SMP_WARPS].lane2 != 0);
            step1 = w1 ? (31 - __clz(w1)) * 32 + (int)sh.between[31 - __clz(w1)].lane1 - 1 : 0;
            step2 = w2 ? (31 - __clz(w2)) * 32 + (int)sh.between[31 - __clz(w2)].lane2 - 1 : 0;
            m = w2 ? (int)sh.between[31 - __clz(w2)].upto : SMP_LIST + 1;
            step1 = min(step1, step2);
            listed = m <= SMP_FEW_BY_WEIGHT;
            edge = step1 == 0 ? peak : peak - (step1 - 0.5f) / scale;
            scale2 = scale * SMP_BINS / (step2 - step1 + 1);
            // the smallest value of the steps up to step2: a warp looks at 32 at once
            uint32_t from = order_of(-INFINITY) + 1, to = order_of(peak);
            if (step2 < SMP_BINS - 1 && scale > 0.f) { // (whatever is rounded: a whole step lower none is in step2, half a step higher all)
                from = max(from, order_of(__fsub_rd(peak, __fdiv_ru(step2 + 1.f, scale))));
                to = min(to, order_of(__fsub_ru(peak, __fdiv_rd((float)step2, scale))));
            }
            while (from < to) {
                const uint32_t apart = (to - from) / 32 + 1, at = from + lane * apart;
                const uint32_t who = __ballot_sync(0xffffffffu, at >= to || coarse(value_of(at)) <= step2);
                if (who == 0) { from += 31 * apart + 1; continue; }
                const int f = __ffs(who) - 1;
                to = min(to, from + f * apart);
                if (f) from += (f - 1) * apart + 1;
            }
            const float lowest = value_of(to);
            // every token is weighed, once: what lies below the steps, and all
            uint64_t all = 0, below = 0;
            if (last == -INFINITY) {
                compact([&](float v, int i) {
                    const uint64_t w = weigh(v);
                    all += w;
                    if (v < lowest) below += w;
                    return v >= lowest;
                });
            } else {
                compact([&](float v, int i) {
                    const bool k = kept(v, i);
                    const uint64_t w = k ? weigh(v) : 0;
                    all += w;
                    if (v < lowest) below += w;
                    return k && v >= lowest;
                });
            }
            each([&](float v, int i) {
                if (listed) {
                    if (kept(v, i) && v >= lowest) put(v, i);
                } else {
                    const int b = in_step(v, i);
                    if (b >= 0) add(b, weigh(v));
                }
            });
            all = warp_total(all);
            below = warp_total(below);
            tell(all, below);
            all = below = 0;
            for (int i = lane; i < C * SMP_WARPS; i += 32) {
                all += sh.from[turn ^ 1][i][0];
                below += sh.from[turn ^ 1][i][1];
            }
            all = warp_total(all);
            limit = fmax((double)top_p * (double)all, 0.5);
            above = all - warp_total(below);           // (and less by what the steps hold)
        } else {
            each([&](float v, int) {
                if (v > -INFINITY) add(coarse(v), 0);
            });
            cluster_sync();
        }
        for (bool again = false; !(by_weight && listed); again = true) {
            if (again) {
                clear();
                each([&](float v, int i) {
                    const int b = in_step(v, i);
                    if (b >= 0) add(b, by_weight ? weigh(v) : 0);
                });
                cluster_sync();
            }
            const uint32_t cnt = (uint32_t)joined(sh.hist[0]);
            uint64_t total;
            uint32_t upto;
            const uint64_t sum = by_weight ? joined(sh.hist[1]) + (joined(sh.hist[2]) << 16) + (joined(sh.hist[3]) << 32) : cnt;
            const uint64_t earlier = block_scan(sum, cnt, total, upto);
            if (by_weight && !again) above -= total;
            const uint64_t before = earlier + above;
            // the last step that has elements and less than the limit above it; the first that has any qualifies, whatever was rounded
            const uint32_t here = __ballot_sync(0xffffffffu, cnt > 0 && (earlier == 0 || (double)before < limit));
            if (lane == (here ? 31 - __clz(here) : 0)) {
                sh.border[warp].above = before;
                sh.border[warp].lane1 = here ? lane + 1 : 0;
                sh.border[warp].count = cnt;
                sh.border[warp].upto = upto + cnt;
            }
            __syncthreads();
            const uint32_t warps = __ballot_sync(0xffffffffu, lane < SMP_WARPS && sh.border[lane % SMP_WARPS].lane1 != 0);
            const int w = 31 - __clz(warps);
            above = sh.border[w].above;
            step = w * 32 + sh.border[w].lane1 - 1;
            m = sh.border[w].count;
            if (!by_weight && !again && (int)sh.border[w].upto <= (top_p < 1.f ? SMP_LIST : SMP_FEW_BY_COUNT)) { m = sh.border[w].upto; listed = true; }
            if (m <= SMP_LIST) break;
            // too many to be ranked: the step's range of keys, to be divided
            if (shift < 0) {
                uint64_t most = 0, least = 0;          // (least: of the complement)
                each([&](float v, int i) {
                    if (in_step(v, i) != step) return;
                    most = max(most, key_of(v, i));
                    least = max(least, ~key_of(v, i));
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                    least = max(least, __shfl_xor_sync(0xffffffffu, least, o));
                }
                tell(most, least);
                for (int i = 0; i < C * SMP_WARPS; ++i) {
                    most = max(most, sh.from[turn ^ 1][i][0]);
                    least = max(least, sh.from[turn ^ 1][i][1]);
                }
                hi = most;
                lo = ~least;
            } else {
                hi -= (uint64_t)step << shift;
                lo = max(lo, hi - (((uint64_t)1 << shift) - 1));
                cluster_sync();                        // the others have read this CTA's histogram
            }
            shift = max(0, 64 - __clzll((long long)(hi - lo)) - 9);
        }
        if (by_weight && listed) {
            above = 0;
        } else {
            // the list: the step's elements, or all down to it.  (What is smaller than this lies in a later step, whatever was rounded.)
            const float near = !by_weight && shift < 0 && step < SMP_BINS - 1 ? __fsub_rd(peak, __fdiv_ru(step + 1.f, scale)) : -INFINITY;
            each_from(near, [&](float v, int i) {
                const int b = in_step(v, i);
                if (b >= 0 && b <= step && (b == step || listed)) put(v, i);
            });
            cluster_sync();
        }
        if (!listed || rank == 0) {
            // the thread's element of the cluster's list: which CTA's, and which there
            uint32_t here = lane < C ? ld_cluster_u32(in_rank(smem_u32(&sh.list_n), min(lane, C - 1))) : 0;
            int c = 0, at = tid;
            for (int i = 0; i < C; ++i) {
                const int k = (int)__shfl_sync(0xffffffffu, here, i);
                if (c == i && at >= k) { at -= k; ++c; }
            }
            if (tid < m) sh.all_key[tid] = ld_cluster_u64(in_rank(smem_u32(&sh.list_key[at]), c));
        }
        if (listed) {                                  // the first CTA goes on alone; the others stay until it has read their lists
            cluster_arrive();
            if (rank) {
                cluster_wait();
                return true;
            }
        }
        __syncthreads();
        // How many of m keys are larger than the thread's.  All warps share the comparisons: a lane has four keys to count for, so that what
        // it reads of shared memory is compared four times.
        auto rank_among = [&](const auto* keys, int m) -> int {
            sh.rank[tid] = 0;
            __syncthreads();
            // 1 to 4 groups of 128 keys, 16, 8, 5 or 4 parts of what they are compared to; the quotients by multiplication
            const int groups = (m + 127) / 128, shares = groups == 1 ? 16 : groups == 2 ? 8 : groups == 3 ? 5 : 4;
            const int share = warp * (groups == 3 ? 11 : groups == 1 ? 32 : groups == 2 ? 16 : 8) >> 5, t = (warp - share * groups) * 128 + lane;
            const int part = m * (groups == 3 ? 13108 : groups == 1 ? 4096 : groups == 2 ? 8192 : 16384);
            if (share < shares) {
                const int end = part * (share + 1) >> 16;
                const auto a = keys[min(t, m - 1)], b = keys[min(t + 32, m - 1)], c = keys[min(t + 64, m - 1)], d = keys[min(t + 96, m - 1)];
                uint32_t la = 0, lb = 0, lc = 0, ld = 0;
#pragma unroll 4
                for (int i = part * share >> 16; i < end; ++i) {
                    const auto k = keys[i];
                    la += k > a;
                    lb += k > b;
                    lc += k > c;
                    ld += k > d;
                }
                if (t < m) atomicAdd(&sh.rank[t], la);
                if (t + 32 < m) atomicAdd(&sh.rank[t + 32], lb);
                if (t + 64 < m) atomicAdd(&sh.rank[t + 64], lc);
                if (t + 96 < m) atomicAdd(&sh.rank[t + 96], ld);
            }
            __syncthreads();
            return (int)sh.rank[tid];
        };
        const uint64_t key = tid < m ? sh.all_key[tid] : 0;
        const uint64_t weight = tid >= m ? 0 : by_weight || listed ? weigh(value_of((uint32_t)(key >> 32))) : 1;
        const int rank_of = rank_among(sh.all_key, m);
        // in order, where the histogram was
        uint64_t* in_key = reinterpret_cast<uint64_t*>(sh.hist[0]);
        uint64_t* in_w = in_key + SMP_LIST;
        if (tid < m) { in_key[rank_of] = key; in_w[rank_of] = weight; }
        __syncthreads();
        const uint64_t w = tid < m ? in_w[tid] : 0;
        uint64_t total;
        uint32_t unused;
        if (!listed) {
            const uint64_t before = block_scan(w, 0, total, unused) + above;
            const int stay = __syncthreads_count(tid < m && (tid == 0 || (double)before < limit));
            const uint64_t k = in_key[stay - 1];
            last = value_of((uint32_t)(k >> 32));
            last_at = (int)~(uint32_t)k;
            cluster_sync();                            // the others have read this CTA's list (and histogram)
            return false;
        }
        const int few = !by_weight && top_k < m ? top_k : m;
        const uint64_t before = block_scan(tid < few ? w : 0, 0, total, unused);
        if (!by_weight) limit = fmax((double)top_p * (double)total, 0.5);
        const int stay = __syncthreads_count(tid < few && (tid == 0 || ((!(top_p < 1.f) || (double)before < limit) && w >= floor_w)));
        if (tid == stay - 1) sh.kept_sum = before + w;
        __syncthreads();
        const uint64_t all = sh.kept_sum, reach = min((uint64_t)(u * (double)all), all - 1);
        // in the order of the index (whose complement the key has), for the sums up to each
        uint32_t* index = sh.index;
        uint64_t* by_index = sh.all_key;
        if (tid < stay) index[tid] = (uint32_t)in_key[tid];
        const int place = rank_among(index, stay);
        const uint32_t mine = tid < stay ? index[tid] : 0;
        __syncthreads();
        if (tid < stay) {
            by_index[place] = w;
            index[place] = mine;
        }
        __syncthreads();
        const uint64_t w2 = tid < stay ? by_index[tid] : 0, earlier = block_scan(w2, 0, total, unused);
        if (tid < stay && earlier <= reach && reach < earlier + w2) p.out[r] = (int)~index[tid];
        cluster_wait();
        return true;
    };

    bool chosen = false;
    if (top_k > 0 && top_k < p.cols) chosen = cut(false, fminf(depth, 128.f));
    if (!chosen && top_p < 1.f) chosen = cut(true, fminf(fminf(depth, 64.f * temp), 3e38f));
    if (chosen) return;
    if (held < 0 && last > -INFINITY) compact(kept);

    // ---------------------------------------------------------------------------------------- the choice from all that is kept
    auto counted = [&](float v, int i) -> uint64_t {
        const uint64_t w = kept(v, i) ? weigh(v) : 0;
        return w < floor_w && (uint32_t)(first + i) != top_at ? 0 : w;
    };
    uint64_t mine = 0;
    each([&](float v, int i) { mine += counted(v, i); });
    mine = warp_total(mine);
    tell(mine, 0);
    uint64_t all = 0, below = 0;
    for (int i = lane; i < C * SMP_WARPS; i += 32) {
        const uint64_t v = sh.from[turn ^ 1][i][0];
        all += v;
        if (i < rank * SMP_WARPS + warp) below += v;
    }
    all = warp_total(all);
    below = warp_total(below);
    const uint64_t reach = min((uint64_t)(u * (double)all), all - 1);
    if (reach < below || reach >= below + mine) return;
    // one warp finds it in its run: of many tokens the lane whose share of them it is in first, then 32 at a time
    auto value_at = [&](int j, uint64_t& w) -> int {
        const int i = 4 * begin + (held < 0 ? j : places[j]);
        w = counted(sx[i], i);
        return first + i;
    };
    auto scan = [&](uint64_t sum) -> uint64_t {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += t;
        }
        return sum;
    };
    int from = 0, to = held >= 0 ? held : 4 * (end - begin);
    if (to > 4 * 32) {
        const int share = (to + 31) / 32, stop = min(to, share * (lane + 1));
        uint64_t own = 0, w;
#pragma unroll 4
        for (int j = share * lane; j < stop; ++j) {
            value_at(j, w);
            own += w;
        }
        const uint64_t sum = scan(own);
        const int lane_of = __ffs(__ballot_sync(0xffffffffu, below + sum > reach)) - 1;
        below += __shfl_sync(0xffffffffu, sum - own, lane_of);
        from = share * lane_of;
        to = min(to, from + share);
    }
    for (int j = from + lane; j - lane < to; j += 32) {
        uint64_t w = 0;
        const int id = j < to ? value_at(j, w) : 0;
        const uint64_t sum = scan(w);
        const uint32_t over = __ballot_sync(0xffffffffu, below + sum > reach);
        if (over) {
            if (lane == __ffs(over) - 1) p.out[r] = id;
            return;
        }
        below += __shfl_sync(0xffffffffu, sum, 31);
    }
}

}  // namespace bn

using namespace bn;

extern "C" int bn_sample_rows(const void* logits, int64_t row_stride, int dtype, const float* uniform, const float* temperature, float temperature_all,
                              const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all, int32_t* out,
                              int rows, int cols, bn_stream_t stream) {
    const char* what = "bn_sample_rows";
    if (!logits || !uniform || !out) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (rows < 0 || rows > 0x7fffffff / SMP_CLUSTER || cols <= 0 || row_stride < cols) return fail(BN_ERR_INVALID_ARG, "%s: bad shape rows=%d cols=%d row_stride=%lld", what, rows, cols, (long long)row_stride);
    if (cols > SMP_MOST_COLS) return fail(BN_ERR_UNSUPPORTED, "%s: %d columns (<= %d supported)", what, cols, SMP_MOST_COLS);
    if (dtype != 0 && dtype != 1) return fail(BN_ERR_INVALID_ARG, "%s: dtype=%d (0 = fp32, 1 = bf16)", what, dtype);
    if (!temperature && !(temperature_all >= 0.f && temperature_all < INFINITY)) return fail(BN_ERR_INVALID_ARG, "%s: temperature=%g", what, temperature_all);
    if (!top_p && !(top_p_all >= 0.f && top_p_all <= 1.f)) return fail(BN_ERR_INVALID_ARG, "%s: top_p=%g", what, top_p_all);
    if (!min_p && !(min_p_all >= 0.f && min_p_all <= 1.f)) return fail(BN_ERR_INVALID_ARG, "%s: min_p=%g", what, min_p_all);
    if (!top_k && top_k_all < 0) return fail(BN_ERR_INVALID_ARG, "%s: top_k=%d", what, top_k_all);
    if (int rc = require_sm100()) return rc;
    if (rows == 0) return BN_OK;
    SampleParams p;
    p.x = logits; p.row_stride = row_stride; p.u = uniform;
    p.temperature = temperature; p.top_p = top_p; p.min_p = min_p; p.top_k = top_k;
    p.temperature1 = temperature_all; p.top_p1 = top_p_all; p.min_p1 = min_p_all; p.top_k1 = top_k_all;
    p.out = out; p.cols = cols;
    p.unit_bits = 50;
    while ((1ll << (62 - p.unit_bits)) < cols) --p.unit_bits;
    // As many CTAs for a row as there are SMs for, but no fewer than its tokens need: of more than 1024 tokens
    // while half of the SMs are left over, of more than 6144 up to all SMs (us with top-k 50 by 1, 2, 4, 8 CTAs: 1 x 10007 11.4, 9.4, 9.0, 8.5; 32 x 10007 12.6, 10.1, 10.5, 12.5;
    // 32 x 32000 21.7, 14.8, 12.6, 13.9; 64 x 32000 21.7, 14.8, 14.6, 26.8)
    int c = 1;
    while (c < SMP_CLUSTER) {
        const int64_t ctas = (int64_t)rows * 2 * c;
        if (!(cols > c * SMP_MOST || (rows > 8 && cols > c * SMP_TWO) || (ctas <= sm_count() && cols > c * (2 * ctas <= sm_count() ? 1024 : 6144)))) break;
        c *= 2;
    }
    p.slice = ((cols + c - 1) / c + 3) / 4 * 4;
    const size_t smem = (size_t)p.slice * 5;
    p.bf16 = dtype;
    if (int rc = allow_smem(sample_rows_kernel, smem, what, SMP_MOST_SMEM, sizeof(SampleShared))) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * c));
    cfg.blockDim = dim3(SMP_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = as_stream(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    (void)launch_config(cfg, 1, sample_rows_kernel, p);
    return launch_status(what);
}
