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
// computed in fp64 and summed as 64-bit whole numbers of 2^-s, s the largest for which a row's sum fits in 62 bits (46 for 32000
// tokens).  A weight above 0 counts at least one such unit.
//
// A block per row; the last element that is kept is found by bisection over (value, index) pairs as 64-bit keys.
#include <math.h>

#include "hybrid.cuh"

namespace bn {

constexpr int SMP_THREADS = 1024;

struct SampleParams {
    const void* x;
    int64_t row_stride;
    const float *u, *temperature, *top_p, *min_p;      // per row, or null: the numbers below
    const int32_t* top_k;
    float temperature1, top_p1, min_p1;
    int top_k1;
    int32_t* out;
    int cols, unit_bits;
};

// 32 bits in the order of the values; NaN and -inf: 0, which nothing else is
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v);
    if (!(v > -INFINITY)) return 0u;
    if (b == 0x80000000u) return 0x80000000u;             // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float v, int i) { return (uint64_t)order_of(v) << 32 | (uint32_t)~i; }

template <typename V> __device__ __forceinline__ V block_total(V v, V* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
    __syncthreads();
    V t = 0;
    for (int w = 0; w < SMP_THREADS / 32; ++w) t += sh[w];
    return t;
}

template <typename T> __global__ void __launch_bounds__(SMP_THREADS) sample_rows_kernel(const SampleParams p) {
    __shared__ uint64_t sh[SMP_THREADS / 32];
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int r = blockIdx.x, n = p.cols, tid = threadIdx.x;
    const T* x = static_cast<const T*>(p.x) + r * p.row_stride;
    const float temp = p.temperature ? p.temperature[r] : p.temperature1, top_p = p.top_p ? p.top_p[r] : p.top_p1,
                min_p = p.min_p ? p.min_p[r] : p.min_p1;
    const int top_k = p.top_k ? p.top_k[r] : p.top_k1;
    uint64_t best = 0;
    for (int i = tid; i < n; i += SMP_THREADS) best = max(best, key_of(to_f(x[i]), i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (tid % 32 == 0) sh[tid / 32] = best;
    __syncthreads();
    for (int w = 0; w < SMP_THREADS / 32; ++w) best = max(best, sh[w]);
    const int first = (int)~(uint32_t)best;
    if (best >> 32 == 0 || !(temp > 0.f)) {
        if (tid == 0) p.out[r] = best >> 32 == 0 ? 0 : first;
        return;
    }
    const double peak = to_f(x[first]), per = 1.0 / temp, units = (double)(1ull << p.unit_bits);
    auto weight = [&](float v) { return order_of(v) == 0u ? 0.0 : v == (float)peak ? 1.0 : exp(((double)v - peak) * per); };
    auto mass = [&](float v) {
        const double w = weight(v);
        return w > 0.0 ? max((uint64_t)__double2ull_rn(w * units), (uint64_t)1) : (uint64_t)0;
    };
    // the smallest key for which what lies above it is less than `limit`
    uint64_t last = 0;                                    // all with a key of at least this are kept
    auto cut = [&](bool by_mass, double limit) {
        uint64_t lo = last, hi = best;
        while (lo < hi) {
            const uint64_t mid = lo + (hi - lo) / 2;
            uint64_t above = 0;
            for (int i = tid; i < n; i += SMP_THREADS) {
                const float v = to_f(x[i]);
                if (order_of(v) != 0u && key_of(v, i) > mid) above += by_mass ? mass(v) : 1;
            }
            if ((double)block_total(above, sh) < limit) hi = mid; else lo = mid + 1;
        }
        last = lo;
    };
    auto kept = [&](float v, int i) { return order_of(v) != 0u && key_of(v, i) >= last; };
    if (top_k > 0 && top_k < n) cut(false, top_k);
    if (top_p < 1.f) {
        uint64_t sum = 0;
        for (int i = tid; i < n; i += SMP_THREADS) {
            const float v = to_f(x[i]);
            if (kept(v, i)) sum += mass(v);
        }
        cut(true, fmax((double)top_p * (double)block_total(sum, sh), 0.5));
    }
    // a thread's own run of columns, so that sums are in the order of the index
    const int per_thread = (n + SMP_THREADS - 1) / SMP_THREADS, begin = tid * per_thread, end = min(n, begin + per_thread);
    auto counted = [&](int i) -> uint64_t {
        const float v = to_f(x[i]);
        if (!kept(v, i) || (weight(v) < (double)min_p && key_of(v, i) != best)) return 0;
        return mass(v);
    };
    uint64_t mine = 0;
    for (int i = begin; i < end; ++i) mine += counted(i);
    uint64_t run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t t = __shfl_up_sync(0xffffffffu, run, o);
        if (tid % 32 >= o) run += t;
    }
    __syncthreads();
    if (tid % 32 == 31) sh[tid / 32] = run;
    __syncthreads();
    uint64_t before = run - mine, total = 0;
    for (int w = 0; w < SMP_THREADS / 32; ++w) {
        if (w < tid / 32) before += sh[w];
        total += sh[w];
    }
    const double u = fmin(fmax((double)p.u[r], 0.0), 1.0);
    const uint64_t reach = min((uint64_t)(u * (double)total), total - 1);
    if (before <= reach && reach < before + mine)
        for (int i = begin; i < end; ++i) {
            before += counted(i);
            if (before > reach) {
                p.out[r] = i;
                break;
            }
        }
}

}  // namespace bn

using namespace bn;

extern "C" int bn_sample_rows(const void* logits, int64_t row_stride, int dtype, const float* uniform, const float* temperature, float temperature_all,
                              const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all, int32_t* out,
                              int rows, int cols, bn_stream_t stream) {
    const char* what = "bn_sample_rows";
    if (!logits || !uniform || !out) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (rows < 0 || cols <= 0 || row_stride < cols) return fail(BN_ERR_INVALID_ARG, "%s: bad shape rows=%d cols=%d row_stride=%lld", what, rows, cols, (long long)row_stride);
    if (cols > (1 << 20)) return fail(BN_ERR_UNSUPPORTED, "%s: %d columns (<= 1048576 supported)", what, cols);
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
    p.unit_bits = 62;
    while ((1ll << (62 - p.unit_bits)) < cols) --p.unit_bits;
    if (dtype == 0) launch_dependent(sample_rows_kernel<float>, (unsigned)rows, SMP_THREADS, 0, as_stream(stream), p);
    else launch_dependent(sample_rows_kernel<__nv_bfloat16>, (unsigned)rows, SMP_THREADS, 0, as_stream(stream), p);
    return launch_status(what);
}
