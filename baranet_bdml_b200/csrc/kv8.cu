// The 8-bit paged cache (kv8.cuh): new tokens are rotated, scaled and rounded as they are written, and read back as bf16 or fp32.
// The reference keeps no cache (mygrad/llama/llama_model.py:136-144); this one holds twice the tokens of the bf16 cache (kv_cache.cu).
#include "kv8.cuh"

namespace bn {

constexpr int KV8_LANES = 8;                  // lanes that share one token's 64 numbers of a head: 8 each, 16 bytes of bf16
constexpr int KV8_PER = KV8_D / KV8_LANES;

template <typename T> __device__ __forceinline__ void load8(const T* p, bool wide, float (&x)[8]) {
    if (wide) {
        float a[4], b[4];
        load4(p, a);
        load4(p + 4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[i + 4] = b[i]; }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f(p[i]);
    }
}

// n / d of whole numbers by a multiplication: 2^(31 + s) / d rounded up, 2^s >= d, is exact for n < 2^31 (an instruction or two where a
// division takes 20, and one of 64 bits 100)
struct Divisor {
    uint32_t d, mul, shift;
    explicit Divisor(int by = 1) : d((uint32_t)by), mul(0), shift(31) {
        while ((1ull << (shift - 31)) < d) ++shift;
        mul = (uint32_t)(((1ull << shift) + d - 1) / d);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return (uint32_t)((uint64_t)n * mul >> shift); }
};

// the largest magnitude of the lanes of a group, as bits (so that a NaN is larger than all numbers)
__device__ __forceinline__ uint32_t group_most(const float (&x)[8]) {
    auto larger = [](float a, float b) {
        float m;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)));
        return m;
    };
    float m = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = larger(m, x[i]);
#pragma unroll
    for (int o = 1; o < KV8_LANES; o <<= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, o));
    return __float_as_uint(m);
}

struct Kv8AppendParams {
    uint8_t* pool;
    int64_t pool_pages;
    const int32_t *page_table, *seq_ids, *positions;
    const void *k, *v;
    int64_t k_stride, v_stride;
    int num_seqs, max_pages, T, Hkv, rotate, wide;
    Divisor heads;
    RotationFreqs freqs;
};

// A group of lanes per (token, key head).  Where the four groups of a warp have the same token (a multiple of four heads), each works out
// a quarter of its cosines and sines.  Bound by instructions: 371 a warp (e4m3; int8 514), 87 of them for the rotation, at 63 % of the issue
// slots.  16384 tokens, e4m3, bf16 in: 4 heads 8.3 us, 6.8 where keys come rotated; 8 heads 14.8 and 12.0; with all four pairs a lane
// 1 head 4.9 and 3.7, 2 heads 6.0 and 4.5, 5 heads 12.3 and 8.2, 6 heads 14.1 and 9.4.  int8, 4 heads 10.9 and 9.6.
template <typename T, int VALUES> __global__ void __launch_bounds__(256) kv8_append_kernel(const __grid_constant__ Kv8AppendParams p) {
    __shared__ double freq[KV8_D / 2];                 // (32 lanes that read 32 parameters take 32 turns: once a block, not once a warp)
    if (threadIdx.x < KV8_D / 2) freq[threadIdx.x] = p.freqs.f[threadIdx.x];
    __syncthreads();
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const uint32_t unit = blockIdx.x * (blockDim.x / KV8_LANES) + threadIdx.x / KV8_LANES;
    const int part = threadIdx.x % KV8_LANES, group = threadIdx.x % 32 / KV8_LANES;
    const bool there = unit < (uint32_t)p.T * (uint32_t)p.Hkv;
    const int t = there ? (int)p.heads.of(unit) : 0, g = there ? (int)(unit - (uint32_t)t * (uint32_t)p.Hkv) : 0;
    const int pos = p.positions[t], seq = p.seq_ids[t], slot = pos % BN_PAGE_TOKENS;
    int page = -1;
    if (there && pos >= 0 && pos / BN_PAGE_TOKENS < p.max_pages && seq >= 0 && seq < p.num_seqs)
        page = p.page_table[(int64_t)seq * p.max_pages + pos / BN_PAGE_TOKENS];
    float k[8], v[8];
    load8(static_cast<const T*>(p.k) + t * p.k_stride + g * KV8_D + part * KV8_PER, p.wide, k);
    load8(static_cast<const T*>(p.v) + t * p.v_stride + g * KV8_D + part * KV8_PER, p.wide, v);
    if (p.rotate) {
        float c[4], s[4];
        if (p.Hkv % 4 == 0) {
            float c1, s1;
            kv8_rotation(pos, freq[part * 4 + group], &c1, &s1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] = __shfl_sync(0xffffffffu, c1, i * KV8_LANES + part);
                s[i] = __shfl_sync(0xffffffffu, s1, i * KV8_LANES + part);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) kv8_rotation(pos, freq[part * 4 + i], &c[i], &s[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = k[2 * i], b = k[2 * i + 1];
            k[2 * i] = a * c[i] - b * s[i];
            k[2 * i + 1] = a * s[i] + b * c[i];
        }
    }
    const float ks = kv8_scale<VALUES>(group_most(k)), vs = kv8_scale<VALUES>(group_most(v));
    if (page < 0 || page >= p.pool_pages) return;
    uint8_t* block = p.pool + ((int64_t)page * p.Hkv + g) * BN_KV8_BLOCK;
    auto pack = [](const float (&x)[8], float s) {
        return make_uint2(kv8_pack<VALUES>(x[0], x[1], x[2], x[3], s), kv8_pack<VALUES>(x[4], x[5], x[6], x[7], s));
    };
    *reinterpret_cast<uint2*>(block + slot * KV8_D + part * KV8_PER) = pack(k, ks);
    *reinterpret_cast<uint2*>(block + KV8_V + slot * KV8_D + kv8_v_place(slot, part * KV8_PER)) = pack(v, vs);
    if (part == 0) *reinterpret_cast<uint32_t*>(block + KV8_SCALES + slot * 4) = __float_as_uint(ks) >> 16 | (__float_as_uint(vs) & 0xffff0000u);
}

struct Kv8GatherParams {
    const uint8_t* pool;
    int64_t pool_pages;
    const int32_t *page_table, *seq_lens, *seq_ids, *starts;
    void *k, *v;
    int64_t units;
    int num_seqs, max_pages, n_tokens, Hkv;
    Divisor heads, tokens;
};

// Four lanes per (row of the result, key head), bytes 8 part .. and 32 + 8 part .. of K and of V each: what the four read or store at once lies
// side by side
constexpr int KV8_GLANES = 4;
template <typename T, int VALUES> __global__ void __launch_bounds__(256) kv8_gather_kernel(const Kv8GatherParams p) {
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / KV8_GLANES;
    const int part = threadIdx.x % KV8_GLANES;
    if (unit >= p.units) return;
    int64_t row;
    int i, j;
    if (p.units < 0x7fffffffLL) {
        row = p.heads.of((uint32_t)unit);
        i = (int)p.tokens.of((uint32_t)row);
        j = (int)row - i * p.n_tokens;
    } else {
        row = unit / p.Hkv;
        i = (int)(row / p.n_tokens);
        j = (int)(row % p.n_tokens);
    }
    const int g = (int)(unit - row * p.Hkv);
    const int64_t pos = (int64_t)p.starts[i] + j;
    const int seq = p.seq_ids[i];
    int page = -1;
    if (seq >= 0 && seq < p.num_seqs && pos >= 0 && pos < p.seq_lens[seq] && pos / BN_PAGE_TOKENS < p.max_pages)
        page = p.page_table[(int64_t)seq * p.max_pages + pos / BN_PAGE_TOKENS];
    const bool there = page >= 0 && page < p.pool_pages;
    const int slot = there ? (int)(pos % BN_PAGE_TOKENS) : 0;
    uint4 kb = make_uint4(0u, 0u, 0u, 0u), vb = kb;
    uint32_t scales = 0u;
    if (there) {
        const uint8_t* block = p.pool + ((int64_t)page * p.Hkv + g) * BN_KV8_BLOCK;
        const uint2 k0 = *reinterpret_cast<const uint2*>(block + slot * KV8_D + part * 8), k1 = *reinterpret_cast<const uint2*>(block + slot * KV8_D + 32 + part * 8);
        const uint8_t* v = block + KV8_V + slot * KV8_D;
        const uint2 v0 = *reinterpret_cast<const uint2*>(v + kv8_v_place(slot, part * 8)), v1 = *reinterpret_cast<const uint2*>(v + kv8_v_place(slot, 32 + part * 8));
        kb = make_uint4(k0.x, k0.y, k1.x, k1.y);
        vb = make_uint4(v0.x, v0.y, v1.x, v1.y);
        scales = *reinterpret_cast<const uint32_t*>(block + KV8_SCALES + slot * 4);
    }
    auto put = [&](void* out, uint4 b, float scale) {
        T* dst = static_cast<T*>(out) + unit * KV8_D + part * 8;
        const uint32_t words[4] = {b.x, b.y, b.z, b.w};
        float o[16];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t lo, hi;
            kv8_halves<VALUES>(words[w], lo, hi);
            const float2 x = halves_to_floats(lo), y = halves_to_floats(hi);
            o[4 * w] = x.x * scale; o[4 * w + 1] = x.y * scale; o[4 * w + 2] = y.x * scale; o[4 * w + 3] = y.y * scale;
        }
        if (sizeof(T) == 2) {
#pragma unroll
            for (int w = 0; w < 2; ++w)
                *reinterpret_cast<uint4*>(dst + 32 * w) = make_uint4(ptx::pack_bf16(o[8 * w], o[8 * w + 1]), ptx::pack_bf16(o[8 * w + 2], o[8 * w + 3]),
                                                              ptx::pack_bf16(o[8 * w + 4], o[8 * w + 5]), ptx::pack_bf16(o[8 * w + 6], o[8 * w + 7]));
        } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) *reinterpret_cast<float4*>(dst + 32 * (w / 2) + 4 * (w % 2)) = make_float4(o[4 * w], o[4 * w + 1], o[4 * w + 2], o[4 * w + 3]);
        }
    };
    put(p.k, kb, ptx::bf16_lo(scales));
    put(p.v, vb, ptx::bf16_hi(scales));
}

}  // namespace bn

using namespace bn;

static int kv8_shape(const char* what, const void* pool, int64_t pool_pages, const int32_t* page_table, int num_seqs, int max_pages, int Hkv, int D,
                     int values) {
    if (!pool || !page_table) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (pool_pages <= 0 || num_seqs <= 0 || max_pages <= 0 || Hkv <= 0)
        return fail(BN_ERR_INVALID_ARG, "%s: bad sizes pool_pages=%lld num_seqs=%d max_pages=%d Hkv=%d", what, (long long)pool_pages, num_seqs, max_pages,
                    Hkv);
    if (D != KV8_D) return fail(BN_ERR_UNSUPPORTED, "%s: head_dim=%d (64 supported)", what, D);
    if (values != BN_KV8_E4M3 && values != BN_KV8_INT8) return fail(BN_ERR_INVALID_ARG, "%s: values=%d (0 = e4m3, 1 = int8)", what, values);
    if (reinterpret_cast<uintptr_t>(pool) & 15) return fail(BN_ERR_INVALID_ARG, "%s: the pool must be 16-byte aligned", what);
    return BN_OK;
}

extern "C" int bn_kv8_append(void* pool, int64_t pool_pages, const int32_t* page_table, int num_seqs, int max_pages, const int32_t* seq_ids,
                             const int32_t* positions, int T, const void* k_new, int64_t k_row_stride, const void* v_new, int64_t v_row_stride,
                             int dtype, int values, int rotate, int Hkv, int D, float theta, bn_stream_t stream) {
    const char* what = "bn_kv8_append";
    if (int rc = kv8_shape(what, pool, pool_pages, page_table, num_seqs, max_pages, Hkv, D, values)) return rc;
    if (!seq_ids || !positions || !k_new || !v_new) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (T < 0 || (int64_t)T * Hkv >= 0x7fffffffLL) return fail(BN_ERR_INVALID_ARG, "%s: T=%d tokens of %d heads", what, T, Hkv);
    if (dtype != 0 && dtype != 1) return fail(BN_ERR_INVALID_ARG, "%s: dtype=%d (0 = fp32, 1 = bf16)", what, dtype);
    if (rotate && !(theta > 0.f)) return fail(BN_ERR_INVALID_ARG, "%s: theta=%g", what, theta);
    if (int rc = require_sm100()) return rc;
    if (T == 0) return BN_OK;
    Kv8AppendParams p;
    p.pool = static_cast<uint8_t*>(pool);
    p.pool_pages = pool_pages;
    p.page_table = page_table; p.seq_ids = seq_ids; p.positions = positions;
    p.k = k_new; p.v = v_new; p.k_stride = k_row_stride; p.v_stride = v_row_stride;
    p.num_seqs = num_seqs; p.max_pages = max_pages; p.T = T; p.Hkv = Hkv; p.rotate = rotate;
    p.wide = ((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) & 15) == 0 && ((k_row_stride | v_row_stride) % 8) == 0;
    p.heads = Divisor(Hkv);
    if (rotate) p.freqs = rotation_freqs(theta);
    auto* kernel = dtype == 0 ? (values == BN_KV8_E4M3 ? kv8_append_kernel<float, BN_KV8_E4M3> : kv8_append_kernel<float, BN_KV8_INT8>)
                              : (values == BN_KV8_E4M3 ? kv8_append_kernel<__nv_bfloat16, BN_KV8_E4M3> : kv8_append_kernel<__nv_bfloat16, BN_KV8_INT8>);
    launch_dependent(kernel, (unsigned)(((int64_t)T * Hkv * KV8_LANES + 255) / 256), 256, 0, as_stream(stream), p);
    return launch_status(what);
}

extern "C" int bn_kv8_gather(const void* pool, int64_t pool_pages, const int32_t* page_table, int num_seqs, int max_pages, const int32_t* seq_lens,
                             const int32_t* seq_ids, const int32_t* starts, int n_seqs, int n_tokens, void* k_out, void* v_out, int out_dtype,
                             int values, int Hkv, int D, bn_stream_t stream) {
    const char* what = "bn_kv8_gather";
    if (int rc = kv8_shape(what, pool, pool_pages, page_table, num_seqs, max_pages, Hkv, D, values)) return rc;
    if (!seq_lens || !seq_ids || !starts || !k_out || !v_out) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    const int64_t units = (int64_t)n_seqs * n_tokens * Hkv;
    if (n_seqs < 0 || n_tokens < 0 || (int64_t)n_seqs * n_tokens > 0x7fffffffLL * 16 / Hkv) return fail(BN_ERR_INVALID_ARG, "%s: bad sizes n_seqs=%d n_tokens=%d", what, n_seqs, n_tokens);
    if (out_dtype != 0 && out_dtype != 1) return fail(BN_ERR_INVALID_ARG, "%s: out_dtype=%d (0 = fp32, 1 = bf16)", what, out_dtype);
    if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15)
        return fail(BN_ERR_INVALID_ARG, "%s: the outputs must be 16-byte aligned", what);
    if (int rc = require_sm100()) return rc;
    if (units == 0) return BN_OK;
    Kv8GatherParams p;
    p.pool = static_cast<const uint8_t*>(pool);
    p.pool_pages = pool_pages;
    p.page_table = page_table; p.seq_lens = seq_lens; p.seq_ids = seq_ids; p.starts = starts;
    p.k = k_out; p.v = v_out; p.units = units;
    p.num_seqs = num_seqs; p.max_pages = max_pages; p.n_tokens = n_tokens; p.Hkv = Hkv;
    p.heads = Divisor(Hkv); p.tokens = Divisor(n_tokens);
    auto* kernel = out_dtype == 0 ? (values == BN_KV8_E4M3 ? kv8_gather_kernel<float, BN_KV8_E4M3> : kv8_gather_kernel<float, BN_KV8_INT8>)
                                  : (values == BN_KV8_E4M3 ? kv8_gather_kernel<__nv_bfloat16, BN_KV8_E4M3> : kv8_gather_kernel<__nv_bfloat16, BN_KV8_INT8>);
    launch_dependent(kernel, (unsigned)((units * KV8_GLANES + 255) / 256), 256, 0, as_stream(stream), p);
    return launch_status(what);
}
