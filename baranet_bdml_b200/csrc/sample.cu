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
// computed in fp64 (2^f for |f| <= 1/2 by twelve terms of the exponential series, whose rest is below 2e-16) and summed as 64-bit whole numbers of
// 2^-s, s the largest up to 50 for which a row's sum fits in 62 bits (47 for 32000 tokens).  A weight above 0 counts at least one such unit.
//
// A cluster of CTAs per row, each with a part of the row in shared memory (as integers in the values' order): read once.  The border of
// top-k or top-p is found by a histogram of 512 steps of the value below the maximum (counts, or counts and weights as three 16-bit
// limbs, whose sums fit the 32-bit atomics that shared memory has), which every CTA joins for itself through distributed shared memory.
// Where no more than 512 tokens lie in the steps down to the border, all that is left is done with a list of them, in every CTA alike:
// ranks, sums, choice.  Otherwise the few elements of the border's step are ranked among each other, and the row is passed over once
// more for the choice.  A step with too many (equal logits, far outliers) is divided again by (value, index) until it has not.  Fp64 is
// only spent on what top-k has left.  What bounds it: a cluster's barriers, about 1 us each, of which there are three with a short list
// and five without, and, for many rows, fp64 and the histogram's atomics.
#include <math.h>

#include "hybrid.cuh"

namespace bn {

using namespace ptx;

constexpr int SMP_THREADS = 512;
constexpr int SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_BINS = SMP_THREADS;                 // a thread has one
constexpr int SMP_LIST = SMP_THREADS;                 // elements that are ranked among each other, a thread each
constexpr int SMP_CLUSTER = 8;                        // CTAs per row at most
constexpr int SMP_MOST = 49152;                       // tokens per CTA
constexpr int SMP_TWO = 20480;                        // tokens per CTA of which an SM takes two
constexpr size_t SMP_MOST_SMEM = (size_t)SMP_MOST * 4;
constexpr int SMP_MOST_COLS = SMP_MOST * SMP_CLUSTER;

struct SampleParams {
    const void* x;
    int64_t row_stride;
    const float *u, *temperature, *top_p, *min_p;      // per row, or null: the numbers below
    const int32_t* top_k;
    float temperature1, top_p1, min_p1;
    int top_k1;
    int32_t* out;
    int cols, slice, unit_bits;                        // slice: tokens per CTA, a multiple of 4
};

// 32 bits in the order of the values; NaN and -inf: 0, which nothing else is
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);          // (-0 is 0)
    const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return v > -INFINITY ? o : 0u;
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }

struct SampleShared {
    uint32_t hist[4][SMP_BINS];                        // counts, and the limbs of weights
    uint64_t list_key[SMP_LIST];                       // this CTA's elements
    uint64_t all_key[SMP_LIST], all_w[SMP_LIST];       // the cluster's
    uint64_t from[2][SMP_CLUSTER * SMP_WARPS][2];      // what all warps of the cluster tell each other
    uint64_t warp_sum[2][SMP_WARPS];
    uint32_t warp_cnt[2][SMP_WARPS];
    struct { uint64_t above; uint32_t lane1, count, upto; } border[SMP_WARPS];
    uint64_t kept_sum;
    uint32_t rank[SMP_LIST];
    int list_n;
};

__device__ __forceinline__ uint64_t warp_total(uint64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T> __global__ void __launch_bounds__(SMP_THREADS, 2) sample_rows_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint32_t so[];     // the part's orders
    __shared__ SampleShared sh;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    uint32_t ncta;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ncta));
    const int C = (int)ncta, rank = (int)cluster_rank(), r = blockIdx.x / C;
    const int first = rank * p.slice, n = max(0, min(p.slice, p.cols - first)), n4 = (n + 3) / 4;
    grid_dependency_wait();
    grid_launch_dependents();

    // every warp of the cluster tells all CTAs two numbers; in sh.from[turn ^ 1] behind the barrier
    int turn = 0, turn2 = 0;
    auto cluster_arrive_tell = [&](uint64_t a, uint64_t b) {
        if (lane < C) {
            const uint32_t at = in_rank(smem_u32(&sh.from[turn][rank * SMP_WARPS + warp][0]), lane);
            st_cluster_u64(at, a);
            st_cluster_u64(at + 8, b);
        }
        cluster_arrive();
        turn ^= 1;
    };
    auto tell = [&](uint64_t a, uint64_t b) {
        cluster_arrive_tell(a, b);
        cluster_wait();
    };
    // sums over the lower threads of the block, of a wide number and a narrow one, and over all
    auto block_scan = [&](uint64_t v, uint32_t w, uint64_t& total, uint32_t& below_w) -> uint64_t {
        uint64_t run = v;
        uint32_t runw = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, run, o);
            const uint32_t tw = __shfl_up_sync(0xffffffffu, runw, o);
            if (lane >= o) { run += t; runw += tw; }
        }
        if (lane == 31) { sh.warp_sum[turn2][warp] = run; sh.warp_cnt[turn2][warp] = runw; }
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
        below_w = runw - w + (warp ? belowc : 0);
        return run - v + (warp ? below : 0);
    };

    // ------------------------------------------------------------------ the row's part, its largest and its smallest element
    uint32_t top = 0, top_at = 0xffffffffu, low = 0xffffffffu;
    {
        const T* x = static_cast<const T*>(p.x) + r * p.row_stride + first;
        auto see = [&](uint32_t o, int i) {
            if (o > top) { top = o; top_at = first + i; }          // (a thread's indices ascend: the first of equals stays)
            if (o) low = min(low, o);
        };
        if (tid < n4 * 4 - n) so[n + tid] = 0;         // (behind the last one: whole pieces of four)
        const bool wide = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0;
        if (wide) {
#pragma unroll 4
            for (int i = 4 * tid; i + 4 <= n; i += 4 * SMP_THREADS) {
                float v[4];
                load4(x + i, v);
                const uint4 o = make_uint4(order_of(v[0]), order_of(v[1]), order_of(v[2]), order_of(v[3]));
                *reinterpret_cast<uint4*>(so + i) = o;
                see(o.x, i); see(o.y, i + 1); see(o.z, i + 2); see(o.w, i + 3);
            }
        }
#pragma unroll 4
        for (int i = (wide ? n / 4 * 4 : 0) + tid; i < n; i += SMP_THREADS) {
            const uint32_t o = order_of(to_f(x[i]));
            so[i] = o;
            see(o, i);
        }
        const uint32_t all = __reduce_max_sync(0xffffffffu, top);
        top_at = __reduce_min_sync(0xffffffffu, top == all ? top_at : 0xffffffffu);
        top = all;
        low = __reduce_min_sync(0xffffffffu, low);
    }
    // (what the row's numbers alone say is worked out while the barrier is waited for)
    cluster_arrive_tell((uint64_t)top << 32 | top_at, low);
    const float temp = p.temperature ? p.temperature[r] : p.temperature1;
    const int top_k = p.top_k ? p.top_k[r] : p.top_k1;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p1, min_p = p.min_p ? p.min_p[r] : p.min_p1;
    const double u = fmin(fmax((double)p.u[r], 0.0), 1.0);
    const double per = 1.4426950408889634 / (double)temp;
    const int unit = p.unit_bits;
    const double floor_w = (min_p > 1.f ? 1.0 : (double)min_p) * (double)(1ull << unit);
    // Further below the maximum than `deep` the weights of all the row's tokens together are less than 1 - top_p of the largest: the
    // border of top-p lies above
    const float deep = temp * (logf((float)p.cols) - logf(1.f - top_p) + 1.f);
    cluster_wait();
    top = 0;
    for (int i = lane; i < C * SMP_WARPS; i += 32) {
        const uint64_t a = sh.from[turn ^ 1][i][0];
        const uint32_t o = (uint32_t)(a >> 32);
        if (o > top || (o == top && (uint32_t)a < top_at)) { top = o; top_at = (uint32_t)a; }
        low = min(low, (uint32_t)sh.from[turn ^ 1][i][1]);
    }
    {
        const uint32_t all = __reduce_max_sync(0xffffffffu, top);
        top_at = __reduce_min_sync(0xffffffffu, top == all ? top_at : 0xffffffffu);
        top = all;
        low = __reduce_min_sync(0xffffffffu, low);
    }
    if (top == 0 || !(temp > 0.f) || top_k == 1) {
        if (rank == 0 && tid == 0) p.out[r] = top == 0 ? 0 : (int)top_at;
        return;                                        // (nothing reaches into another CTA behind the last barrier)
    }
    const float peak = value_of(top), depth = peak - value_of(low);

    // 2^((v - peak) / T * log2 e + unit), whole and at least 1; 0 where fp64 has none.  No branches: a warp weighs different values, and
    // a thread's four at a time are worked out side by side
    auto weigh = [&](uint32_t order) -> uint64_t {
        const double t = ((double)value_of(order) - (double)peak) * per;
        const double near = fmax(t, -(double)(unit + 1));          // (a NaN, infinity less infinity, comes out as the bound)
        const double rounded = near + 0x1.8p52;                    // to a whole number, which is the low word
        const double f = near - (rounded - 0x1.8p52);
        // (ln 2)^i / i!
        double w = 2.5678435993488196e-11;
        w = fma(w, f, 4.4455382718708101e-10);
        w = fma(w, f, 7.0549116208011209e-09);
        w = fma(w, f, 1.0178086009239696e-07);
        w = fma(w, f, 1.3215486790144305e-06);
        w = fma(w, f, 1.5252733804059838e-05);
        w = fma(w, f, 1.5403530393381606e-04);
        w = fma(w, f, 1.3333558146428441e-03);
        w = fma(w, f, 9.6181291076284769e-03);
        w = fma(w, f, 5.5504108664821576e-02);
        w = fma(w, f, 2.4022650695910069e-01);
        w = fma(w, f, 6.9314718055994529e-01);
        w = fma(w, f, 1.0);
        w = __hiloint2double(__double2hiint(w) + ((__double2loint(rounded) + unit) << 20), __double2loint(w));
        const uint64_t m = max((uint64_t)(__double_as_longlong(w + 0x1p52) - 0x4330000000000000ll), (uint64_t)1);
        return order == top ? 1ull << unit : t >= -1074.5 ? m : 0;
    };

    // kept: above `last` in the order, or `last` itself
    uint32_t last_order = 1, last_at = 0xffffffffu;
    auto kept = [&](uint32_t o, int i) { return o > last_order || (o == last_order && (uint32_t)(first + i) <= last_at); };
    auto key_of = [&](uint32_t o, int i) { return (uint64_t)o << 32 | (uint32_t)~(first + i); };

    // The last element before which there is less than a limit: top_k by count, top_p times their sum by weight.  True: the choice has
    // been made with the list.
    auto cut = [&](bool by_weight, float range) -> bool {
        uint64_t above = 0, hi = 0, lo = 0;            // what lies above the step; the step as a range of keys, once it is one
        int shift = -1, step = 0, m = 0;
        double limit = (double)top_k;
        bool listed = false;
        // (an order below that of the rounded edge is below the edge itself)
        const uint32_t deep_order = by_weight && range < depth ? order_of(peak - range) : 0;
        const float scale = range > 0.f ? SMP_BINS / range : 0.f;
        auto in_range = [&](uint32_t o, int i) { return kept(o, i) && (shift < 0 || (key_of(o, i) <= hi && key_of(o, i) >= lo)); };
        // (the rounding is to the nearest step: any will do that never puts the larger value behind the smaller)
        auto step_of_order = [&](uint32_t o) -> int {
            return o == top ? 0 : (int)(__float_as_uint(fminf((peak - value_of(o)) * scale, SMP_BINS - 1.f) + 8388608.f) & (SMP_BINS - 1));
        };
        auto step_of = [&](uint32_t o, int i) -> int { return shift >= 0 ? (int)((hi - key_of(o, i)) >> shift) : step_of_order(o); };
        for (;;) {
            sh.hist[0][tid] = 0;
            if (by_weight) sh.hist[1][tid] = sh.hist[2][tid] = sh.hist[3][tid] = 0;
            if (tid == 0) sh.list_n = 0;
            __syncthreads();
            uint64_t rest = 0;
            for (int q = tid; q < n4; q += SMP_THREADS) {
                const uint4 four = *reinterpret_cast<const uint4*>(so + 4 * q);
                const uint32_t os[4] = {four.x, four.y, four.z, four.w};
                uint64_t ws[4];
                if (by_weight) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint64_t w = weigh(os[e]);
                        ws[e] = in_range(os[e], 4 * q + e) ? w : 0;
                        rest += os[e] < deep_order ? ws[e] : 0;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t o = os[e];
                    if (o < deep_order || !in_range(o, 4 * q + e)) continue;
                    const int b = step_of(o, 4 * q + e);
                    atomicAdd(&sh.hist[0][b], 1u);
                    if (by_weight) {
                        const uint64_t w = ws[e];
                        atomicAdd(&sh.hist[1][b], (uint32_t)w & 0xffffu);
                        if (w >> 16) {
                            atomicAdd(&sh.hist[2][b], (uint32_t)(w >> 16) & 0xffffu);
                            if (w >> 32) atomicAdd(&sh.hist[3][b], (uint32_t)(w >> 32));
                        }
                    }
                }
            }
            if (by_weight && deep_order > 1) {         // what lies deep counts in the sum alone
                rest = warp_total(rest);
                if (lane < 3) atomicAdd(&sh.hist[lane + 1][SMP_BINS - 1], lane == 0 ? (uint32_t)rest & 0xffffu : lane == 1 ? (uint32_t)(rest >> 16) & 0xffffu : (uint32_t)(rest >> 32));
            }
            cluster_sync();
            uint32_t cnt = 0;
            uint64_t sum = 0;
#pragma unroll
            for (int c = 0; c < SMP_CLUSTER; ++c) {
                if (c >= C) break;
                const uint32_t at = in_rank(smem_u32(&sh.hist[0][tid]), c);
                cnt += ld_cluster_u32(at);
                if (by_weight)
                    sum += ld_cluster_u32(at + SMP_BINS * 4) + ((uint64_t)ld_cluster_u32(at + SMP_BINS * 8) << 16) +
                           ((uint64_t)ld_cluster_u32(at + SMP_BINS * 12) << 32);
            }
            if (!by_weight) sum = cnt;
            uint64_t total;
            uint32_t upto;
            const uint64_t before = block_scan(sum, cnt, total, upto) + above;
            if (by_weight && shift < 0) limit = fmax((double)top_p * (double)total, 0.5);
            // the last step that has elements and less than the limit above it
            const uint32_t here = __ballot_sync(0xffffffffu, cnt > 0 && (double)before < limit);
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
            if (shift < 0 && sh.border[w].upto <= SMP_LIST) { m = sh.border[w].upto; listed = true; }
            if (m <= SMP_LIST) break;
            // too many to be ranked: the step's range of keys, to be divided
            if (shift < 0) {
                uint64_t most = 0, least = 0;          // (least: of the complement)
                for (int i = tid; i < n; i += SMP_THREADS) {
                    const uint32_t o = so[i];
                    if (in_range(o, i) && step_of(o, i) == step) { most = max(most, key_of(o, i)); least = max(least, ~key_of(o, i)); }
                }
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
        // the list: the step's elements, or all down to it
        for (int q = tid; q < n4; q += SMP_THREADS) {
            const uint4 four = *reinterpret_cast<const uint4*>(so + 4 * q);
            const uint32_t os[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (os[e] < deep_order || !in_range(os[e], 4 * q + e)) continue;
                const int b = step_of(os[e], 4 * q + e);
                if (b > step || (b < step && !listed)) continue;
                const int at = min(atomicAdd(&sh.list_n, 1), SMP_LIST - 1);      // (m of them in the whole cluster)
                sh.list_key[at] = key_of(os[e], 4 * q + e);
            }
        }
        cluster_sync();
        {
            // the thread's element of the cluster's list: which CTA's, and which there
            uint32_t here = lane < C ? ld_cluster_u32(in_rank(smem_u32(&sh.list_n), min(lane, C - 1))) : 0;
            int c = 0, at = tid;
            for (int i = 0; i < C; ++i) {
                const int k = (int)__shfl_sync(0xffffffffu, here, i);
                if (c == i && at >= k) { at -= k; ++c; }
            }
            if (tid < m) sh.all_key[tid] = ld_cluster_u64(in_rank(smem_u32(&sh.list_key[at]), c));
        }
        __syncthreads();
        // how many of m keys are larger than the thread's: all threads share the comparisons
        auto rank_among = [&](const auto* keys, int m) -> int {
            sh.rank[tid] = 0;
            __syncthreads();
            const int wide = (m + 31) / 32 * 32, shares = SMP_THREADS / wide, share = tid / wide, t = tid % wide;
            if (share < shares && t < m) {
                const int end = m * (share + 1) / shares;
                const auto mine = keys[t];
                uint32_t larger = 0;
#pragma unroll 4
                for (int i = m * share / shares; i < end; ++i) larger += keys[i] > mine;
                atomicAdd(&sh.rank[t], larger);
            }
            __syncthreads();
            return (int)sh.rank[tid];
        };
        const uint64_t key = tid < m ? sh.all_key[tid] : 0;
        const uint64_t weight = tid >= m ? 0 : by_weight || listed ? weigh((uint32_t)(key >> 32)) : 1;
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
            const int stay = __syncthreads_count(tid < m && (double)before < limit);
            const uint64_t k = in_key[stay - 1];
            last_order = (uint32_t)(k >> 32);
            last_at = ~(uint32_t)k;
            cluster_sync();                            // the others have read this CTA's list (and histogram)
            return false;
        }
        const int few = !by_weight && top_k < m ? top_k : m;
        const uint64_t before = block_scan(tid < few ? w : 0, 0, total, unused);
        if (!by_weight) limit = fmax((double)top_p * (double)total, 0.5);
        const int stay = __syncthreads_count(tid < few && (tid == 0 || ((!(top_p < 1.f) || (double)before < limit) && !((double)w < floor_w))));
        if (tid == stay - 1) sh.kept_sum = before + w;
        __syncthreads();
        const uint64_t all = sh.kept_sum, reach = min((uint64_t)(u * (double)all), all - 1);
        // in the order of the index (whose complement the key has), for the sums up to each
        uint32_t* index = reinterpret_cast<uint32_t*>(sh.all_w);
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
        if (rank == 0 && tid < stay && earlier <= reach && reach < earlier + w2) p.out[r] = (int)~index[tid];
        return true;
    };

    bool chosen = false;
    if (top_k > 0 && top_k < p.cols) chosen = cut(false, fminf(depth, 128.f));
    if (!chosen && top_p < 1.f) chosen = cut(true, fminf(depth, deep));
    if (chosen) {
        cluster_sync();                                // the others have read this CTA's list
        return;
    }

    // ------------------------------------------------------------------------------------------- the choice from the whole row
    auto counted = [&](uint32_t o, int i) -> uint64_t {
        if (!kept(o, i)) return 0;
        const uint64_t w = weigh(o);
        return (double)w < floor_w && (uint32_t)(first + i) != top_at ? 0 : w;
    };
    // a warp has a run of its CTA's part, so that its sum is one of neighbours
    const int run = (n4 + SMP_WARPS * 32 - 1) / (SMP_WARPS * 32) * 32, begin = warp * run, end = min(n4, begin + run);      // in pieces of four
    uint64_t mine = 0;
    if (last_order == 1) {
        for (int q = begin + lane; q < end; q += 32) {
            const uint4 four = *reinterpret_cast<const uint4*>(so + 4 * q);
            mine += counted(four.x, 4 * q) + counted(four.y, 4 * q + 1) + counted(four.z, 4 * q + 2) + counted(four.w, 4 * q + 3);
        }
    } else {
        // few are kept: they are put side by side, so that 32 at a time are weighed
        uint32_t* queue = sh.hist[0] + warp * 64;
        int held = 0;
        auto weigh_queued = [&](int k) {               // the top's weight is above any floor
            const uint64_t w = lane < k ? weigh(queue[lane]) : 0;
            if (lane < k && (!((double)w < floor_w))) mine += w;
            __syncwarp();
        };
        for (int q = begin; q < end; q += 32) {
            const uint4 four = q + lane < end ? *reinterpret_cast<const uint4*>(so + 4 * (q + lane)) : make_uint4(0u, 0u, 0u, 0u);
            if (!__any_sync(0xffffffffu, max(max(four.x, four.y), max(four.z, four.w)) >= last_order)) continue;
            const uint32_t os[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = kept(os[e], 4 * (q + lane) + e);
                const uint32_t who = __ballot_sync(0xffffffffu, in);
                if (in) queue[held + __popc(who & ((1u << lane) - 1))] = os[e];
                held += __popc(who);
                __syncwarp();
                if (held >= 32) {
                    weigh_queued(32);
                    held -= 32;
                    const uint32_t o = lane < held ? queue[32 + lane] : 0;
                    __syncwarp();
                    if (lane < held) queue[lane] = o;
                    __syncwarp();
                }
            }
        }
        weigh_queued(held);
    }
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
    for (int q = begin + lane; q - lane < end; q += 32) {
        const uint4 four = q < end ? *reinterpret_cast<const uint4*>(so + 4 * q) : make_uint4(0u, 0u, 0u, 0u);
        const uint64_t w[4] = {counted(four.x, 4 * q), counted(four.y, 4 * q + 1), counted(four.z, 4 * q + 2), counted(four.w, 4 * q + 3)};
        uint64_t sum = w[0] + w[1] + w[2] + w[3];
        const uint64_t own = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += t;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, below + sum > reach);
        if (over) {
            if (lane == __ffs(over) - 1) {
                below += sum - own;
                int e = 0;
                while (e < 3 && below + w[e] <= reach) below += w[e++];
                p.out[r] = first + 4 * q + e;
            }
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
    // as many CTAs for a row as there are SMs for, but no fewer than its tokens need, and parts of 1024 tokens at least
    int c = 1;
    while (c < SMP_CLUSTER && (cols > c * SMP_MOST || (rows > 8 && cols > c * SMP_TWO) || ((int64_t)rows * 2 * c <= sm_count() && cols > c * 1024))) c *= 2;
    p.slice = ((cols + c - 1) / c + 3) / 4 * 4;
    const size_t smem = (size_t)p.slice * 4;
    auto* kernel = dtype == 0 ? sample_rows_kernel<float> : sample_rows_kernel<__nv_bfloat16>;
    if (int rc = allow_smem(kernel, smem, what, SMP_MOST_SMEM, sizeof(SampleShared))) return rc;
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
    (void)launch_config(cfg, 1, kernel, p);
    return launch_status(what);
}
