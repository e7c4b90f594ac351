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
// computed in fp64 (2^f by a table of 32 and five terms of the exponential series, |error| < 3e-15) and summed as 64-bit whole numbers of
// 2^-s, s the largest up to 50 for which a row's sum fits in 62 bits (47 for 32000 tokens).  A weight above 0 counts at least one such unit.
//
// A cluster of CTAs per row, each with a part of the row in shared memory: read once, 4 bytes a token.  The last element that is kept is
// found by a histogram of 1024 steps of the value below the maximum (counts for top-k, weights as three 16-bit limbs for top-p, whose
// sums fit the 32-bit atomics that shared memory has), each CTA joining a part of the steps through distributed shared memory; the few
// elements of the step that the border falls into are ranked among each other.  Where they are many (equal logits, far outliers), the step
// is divided again by (value, index) until they are not.  Fp64 is only spent on what top-k has left.
#include <math.h>

#include "hybrid.cuh"

namespace bn {

using namespace ptx;

constexpr int SMP_THREADS = 1024;
constexpr int SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_BINS = 1024;
constexpr int SMP_CLUSTER = 8;                        // CTAs per row at most
constexpr int SMP_LIST = 512;                         // elements that are ranked among each other
constexpr int SMP_KEPT = 16384;                       // tokens per CTA whose weights fit into shared memory beside the logits
constexpr int SMP_MOST = 49152;                       // tokens per CTA
constexpr size_t SMP_MOST_SMEM = (size_t)SMP_KEPT * 12;
static_assert(SMP_MOST_SMEM >= (size_t)SMP_MOST * 4, "either form of a part fits");
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
    const uint32_t b = __float_as_uint(v);
    if (!(v > -INFINITY)) return 0u;
    if (b == 0x80000000u) return 0x80000000u;             // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order); }
__device__ __forceinline__ uint64_t key_of(float v, int i) { return (uint64_t)order_of(v) << 32 | (uint32_t)~i; }

struct SampleShared {
    uint32_t hist[4][SMP_BINS];                        // counts, and the limbs of weights
    uint64_t list_key[SMP_LIST], list_w[SMP_LIST];     // this CTA's elements of the step
    uint64_t all_key[SMP_LIST], all_w[SMP_LIST];       // the cluster's
    uint64_t from[2][SMP_CLUSTER][4];                  // what the CTAs tell each other
    uint64_t red[2][2][SMP_WARPS];
    double table[32];                                  // 2^(j / 32)
    uint64_t found[3];
    int list_n;
};

template <typename T, bool KEEP> __global__ void __launch_bounds__(SMP_THREADS, 1) sample_rows_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ SampleShared sh;
    float* sx = reinterpret_cast<float*>(smem_raw);
    uint64_t* sw = reinterpret_cast<uint64_t*>(smem_raw + (size_t)p.slice * 4);      // KEEP: weights
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    uint32_t ncta;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ncta));
    const int C = (int)ncta, rank = (int)cluster_rank(), r = blockIdx.x / C;
    const int first = rank * p.slice, n = max(0, min(p.slice, p.cols - first));
    if (tid < 32) sh.table[tid] = exp2(tid / 32.0);
    grid_dependency_wait();
    grid_launch_dependents();

    int turn = 0, rturn = 0;
    // tells every CTA of the cluster up to three numbers; they are in sh.from[turn ^ 1] afterwards
    auto tell = [&](uint64_t a, uint64_t b, uint64_t c) {
        if (tid < C) {
            const uint32_t at = in_rank(smem_u32(&sh.from[turn][rank][0]), tid);
            st_cluster_u64(at, a);
            st_cluster_u64(at + 8, b);
            st_cluster_u64(at + 16, c);
        }
        cluster_sync();
        turn ^= 1;
    };
    // over the block, in every thread
    auto block_max2 = [&](uint64_t& a, uint64_t& b) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
            b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
        }
        if (lane == 0) { sh.red[rturn][0][warp] = a; sh.red[rturn][1][warp] = b; }
        __syncthreads();
        a = sh.red[rturn][0][lane];
        b = sh.red[rturn][1][lane];
        rturn ^= 1;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
            b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
        }
    };
    // sum of what the lower threads have, and of all
    auto block_scan = [&](uint64_t v, uint64_t& total) -> uint64_t {
        uint64_t run = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += t;
        }
        if (lane == 31) sh.red[rturn][0][warp] = run;
        __syncthreads();
        uint64_t w = sh.red[rturn][0][lane];
        rturn ^= 1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += t;
        }
        total = __shfl_sync(0xffffffffu, w, 31);
        const uint64_t below = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
        return run - v + (warp ? below : 0);
    };

    // ------------------------------------------------------------------ the row's part, its largest and its smallest element
    uint64_t best = 0, least = 0;                      // least: of the complement of the order
    {
        const T* x = static_cast<const T*>(p.x) + r * p.row_stride + first;
        auto see = [&](float v, int i) {
            const uint32_t o = order_of(v);
            if (o) {
                best = max(best, (uint64_t)o << 32 | (uint32_t)~(first + i));
                least = max(least, (uint64_t)(uint32_t)~o);
            }
        };
        const bool wide = (reinterpret_cast<uintptr_t>(x) & (4 * sizeof(T) - 1)) == 0;
        if (wide) {
            for (int i = 4 * tid; i + 4 <= n; i += 4 * SMP_THREADS) {
                float v[4];
                load4(x + i, v);
                *reinterpret_cast<float4*>(sx + i) = make_float4(v[0], v[1], v[2], v[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) see(v[e], i + e);
            }
        }
        for (int i = (wide ? n / 4 * 4 : 0) + tid; i < n; i += SMP_THREADS) {
            const float v = to_f(x[i]);
            sx[i] = v;
            see(v, i);
        }
    }
    block_max2(best, least);
    tell(best, least, 0);
    for (int c = 0; c < C; ++c) {
        best = max(best, sh.from[turn ^ 1][c][0]);
        least = max(least, sh.from[turn ^ 1][c][1]);
    }
    const float temp = p.temperature ? p.temperature[r] : p.temperature1;
    if (best == 0 || !(temp > 0.f)) {
        if (rank == 0 && tid == 0) p.out[r] = best == 0 ? 0 : (int)~(uint32_t)best;
        return;                                        // (nothing reaches into another CTA behind the last barrier)
    }
    const float peak = value_of((uint32_t)(best >> 32)), depth = peak - value_of(~(uint32_t)least);
    const double per = 1.4426950408889634 / (double)temp;
    const int unit = p.unit_bits;
    const int top_k = p.top_k ? p.top_k[r] : p.top_k1;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p1, min_p = p.min_p ? p.min_p[r] : p.min_p1;

    // 2^((v - peak) / T * log2 e + unit), whole and at least 1; 0 where fp64 has none
    auto weigh = [&](float v) -> uint64_t {
        if (v == peak) return 1ull << unit;
        const double t = ((double)v - (double)peak) * per;
        if (!(t >= -1074.5)) return 0;
        if (t < -(double)(unit + 1)) return 1;
        const double rounded = t + 0x1.8p47;           // to a multiple of 1 / 32, which is the low word
        const int k = __double2loint(rounded);
        const double f = t - (rounded - 0x1.8p47);
        // (ln 2)^i / i!
        double w = fma(f, fma(f, fma(f, fma(f, fma(f, 1.3333558146428443e-3, 9.6181291076284772e-3), 5.5504108664821580e-2), 0.24022650695910072),
                              0.69314718055994531), 1.0);
        w *= sh.table[k & 31];
        w = __hiloint2double(__double2hiint(w) + (((k >> 5) + unit) << 20), __double2loint(w));
        const uint64_t m = (uint64_t)__double_as_longlong(w + 0x1p52) - 0x4330000000000000ull;
        return max(m, (uint64_t)1);
    };

    uint64_t last = 0;                                 // all with a key of at least this are kept
    bool weighed = false;
    auto key_at = [&](int i) { return key_of(sx[i], first + i); };
    auto kept = [&](uint64_t key) { return key >> 32 != 0 && key >= last; };
    auto weight_at = [&](int i) -> uint64_t { return KEEP && weighed ? sw[i] : weigh(sx[i]); };
    // a warp has a run of its CTA's part, so that its sum is one of neighbours
    const int run = (n + SMP_WARPS * 32 - 1) / (SMP_WARPS * 32) * 32, begin = warp * run, end = min(n, begin + run);

    // `last` becomes the key of the last element before which there is less than `limit`
    auto cut = [&](bool by_weight, double limit, float range) {
        uint64_t above = 0, hi = 0, lo = 0;            // what lies above the step; the step as a range of keys, once it is one
        int shift = -1, step = 0;
        const float scale = range > 0.f ? SMP_BINS / range : 0.f;
        auto step_of = [&](uint64_t key, float v) -> int {
            if (shift >= 0) return (int)((hi - key) >> shift);
            return v == peak ? 0 : min(SMP_BINS - 1, __float2int_rd((peak - v) * scale));
        };
        auto in_range = [&](uint64_t key) { return kept(key) && (shift < 0 || (key <= hi && key >= lo)); };
        uint64_t count = 0;
        for (;;) {
            for (int i = tid; i < SMP_BINS; i += SMP_THREADS) {
                sh.hist[0][i] = 0;
                if (by_weight) sh.hist[1][i] = sh.hist[2][i] = sh.hist[3][i] = 0;
            }
            if (tid == 0) sh.list_n = 0;
            __syncthreads();
            for (int i = tid; i < n; i += SMP_THREADS) {
                const uint64_t key = key_at(i);
                if (!in_range(key)) continue;
                const int b = step_of(key, sx[i]);
                atomicAdd(&sh.hist[0][b], 1u);
                if (by_weight) {
                    const uint64_t w = weight_at(i);
                    atomicAdd(&sh.hist[1][b], (uint32_t)w & 0xffffu);
                    if (w >> 16) {
                        atomicAdd(&sh.hist[2][b], (uint32_t)(w >> 16) & 0xffffu);
                        if (w >> 32) atomicAdd(&sh.hist[3][b], (uint32_t)(w >> 32));
                    }
                }
            }
            cluster_sync();
            // a part of the steps for each CTA, a step a thread
            const int steps = SMP_BINS / C;
            uint64_t cnt = 0, sum = 0;
            if (tid < steps) {
                for (int c = 0; c < C; ++c) {
                    const uint32_t at = in_rank(smem_u32(&sh.hist[0][rank * steps + tid]), c);
                    cnt += ld_cluster_u32(at);
                    if (by_weight)
                        sum += ld_cluster_u32(at + SMP_BINS * 4) + ((uint64_t)ld_cluster_u32(at + SMP_BINS * 8) << 16) +
                               ((uint64_t)ld_cluster_u32(at + SMP_BINS * 12) << 32);
                }
                if (!by_weight) sum = cnt;
            }
            uint64_t total, before = block_scan(sum, total);
            tell(total, 0, 0);
            for (int c = 0; c < rank; ++c) before += sh.from[turn ^ 1][c][0];
            before += above;
            // the last step of the part that has elements and less than the limit above it
            uint64_t mine = tid < steps && cnt > 0 && (double)before < limit ? (uint64_t)(rank * steps + tid + 1) : 0, none = 0;
            const uint64_t own = mine;
            if (tid == 0) sh.found[1] = sh.found[2] = 0;
            block_max2(mine, none);
            if (mine != 0 && own == mine) { sh.found[1] = before; sh.found[2] = cnt; }
            __syncthreads();
            tell(mine, sh.found[1], sh.found[2]);
            uint64_t at = 0;
            for (int c = 0; c < C; ++c)
                if (sh.from[turn ^ 1][c][0] > at) {
                    at = sh.from[turn ^ 1][c][0];
                    above = sh.from[turn ^ 1][c][1];
                    count = sh.from[turn ^ 1][c][2];
                }
            step = (int)at - 1;
            if (count <= SMP_LIST) break;
            // too many to be ranked: the step's range of keys, to be divided
            if (shift < 0) {
                uint64_t top = 0, bottom = 0;
                for (int i = tid; i < n; i += SMP_THREADS) {
                    const uint64_t key = key_at(i);
                    if (in_range(key) && step_of(key, sx[i]) == step) { top = max(top, key); bottom = max(bottom, ~key); }
                }
                block_max2(top, bottom);
                tell(top, bottom, 0);
                for (int c = 0; c < C; ++c) {
                    top = max(top, sh.from[turn ^ 1][c][0]);
                    bottom = max(bottom, sh.from[turn ^ 1][c][1]);
                }
                hi = top;
                lo = ~bottom;
            } else {
                hi -= (uint64_t)step << shift;
                lo = max(lo, hi - (((uint64_t)1 << shift) - 1));
            }
            shift = max(0, 64 - __clzll((long long)(hi - lo)) - 10);
        }
        // rank them among each other
        for (int i = tid; i < n; i += SMP_THREADS) {
            const uint64_t key = key_at(i);
            if (!in_range(key) || step_of(key, sx[i]) != step) continue;
            const int at = atomicAdd(&sh.list_n, 1);
            sh.list_key[at] = key;
            sh.list_w[at] = by_weight ? weight_at(i) : 1;
        }
        cluster_sync();
        int m = 0;
        for (int c = 0; c < C; ++c) {
            const int here = (int)ld_cluster_u32(in_rank(smem_u32(&sh.list_n), c));
            for (int i = tid; i < here; i += SMP_THREADS) {
                sh.all_key[m + i] = ld_cluster_u64(in_rank(smem_u32(&sh.list_key[i]), c));
                sh.all_w[m + i] = ld_cluster_u64(in_rank(smem_u32(&sh.list_w[i]), c));
            }
            m += here;
        }
        __syncthreads();
        uint64_t low = 0, none = 0;
        if (tid < m) {
            const uint64_t key = sh.all_key[tid];
            uint64_t before = above;
            for (int i = 0; i < m; ++i)
                if (sh.all_key[i] > key) before += sh.all_w[i];
            if ((double)before < limit) low = ~key;
        }
        block_max2(low, none);
        last = ~low;
    };

    if (top_k > 0 && top_k < p.cols) cut(false, (double)top_k, fminf(depth, 128.f));
    if (top_p < 1.f) {
        uint64_t sum = 0, total;
        for (int i = tid; i < n; i += SMP_THREADS) {
            const uint64_t w = kept(key_at(i)) ? weigh(sx[i]) : 0;
            if (KEEP) sw[i] = w;
            sum += w;
        }
        weighed = true;                                // (read by other threads behind the barriers of the sums)
        block_scan(sum, total);
        tell(total, 0, 0);
        total = 0;
        for (int c = 0; c < C; ++c) total += sh.from[turn ^ 1][c][0];
        cut(true, fmax((double)top_p * (double)total, 0.5), fminf(depth, 64.f * temp));
    }

    // ------------------------------------------------------------------------------------------------------------- the choice
    const double floor_w = (double)min_p * (double)(1ull << unit);
    auto counted = [&](int i) -> uint64_t {
        const uint64_t key = key_at(i);
        if (!kept(key)) return 0;
        const uint64_t w = weight_at(i);
        return (double)w < floor_w && key != best ? 0 : w;
    };
    uint64_t mine = 0, total;
    for (int i = begin + lane; i < end; i += 32) mine += counted(i);
    uint64_t below = block_scan(mine, total);
    tell(total, 0, 0);
    uint64_t all = 0, before = 0;
    for (int c = 0; c < C; ++c) {
        if (c == rank) before = all;
        all += sh.from[turn ^ 1][c][0];
    }
    const double u = fmin(fmax((double)p.u[r], 0.0), 1.0);
    const uint64_t reach = min((uint64_t)(u * (double)all), all - 1);
    // sums before the warp and up to its end
    below = __shfl_sync(0xffffffffu, below, 0) + before;
    uint64_t own = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
    if (reach < below || reach >= below + own) return;
    for (int i = begin + lane; i - lane < end; i += 32) {
        uint64_t sum = i < end ? counted(i) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += t;
        }
        const uint32_t over = __ballot_sync(0xffffffffu, below + sum > reach);
        if (over) {
            if (lane == __ffs(over) - 1) p.out[r] = first + i;
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
    while (c < SMP_CLUSTER && (cols > c * SMP_KEPT || ((int64_t)rows * 2 * c <= sm_count() && cols > c * 1024))) c *= 2;
    p.slice = ((cols + c - 1) / c + 3) / 4 * 4;
    const bool keep = p.slice <= SMP_KEPT;
    const size_t smem = (size_t)p.slice * (keep ? 12 : 4);
    auto* kernel = dtype == 0 ? (keep ? sample_rows_kernel<float, true> : sample_rows_kernel<float, false>)
                              : (keep ? sample_rows_kernel<__nv_bfloat16, true> : sample_rows_kernel<__nv_bfloat16, false>);
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
