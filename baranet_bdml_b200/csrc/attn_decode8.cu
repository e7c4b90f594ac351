// Single-token decode attention over the 8-bit paged cache (kv8.cuh):
//     s_t = scale <RoPE(q), K_t> ks_t,   p = softmax(s),   out = sum_t p_t vs_t V_t,   lse = log sum exp s
// A block per (sequence, key head); a warp takes every eighth token, a lane two of the 64 dimensions, for all query heads of the group.
#include <math.h>

#include "kv8.cuh"

namespace bn {

constexpr int DEC8_G = 8;
constexpr int DEC8_WARPS = 8;

struct Decode8Params {
    const __nv_bfloat16* q;
    const uint8_t* pool;
    int64_t pool_pages;
    const int32_t *page_table, *seq_lens, *q_positions;
    __nv_bfloat16* out;
    float *out_f32, *lse;
    int* error;
    int Hq, Hkv, n_rep, max_pages, max_seq_len, rope_q;
    float scale;
    RotationFreqs freqs;
};

template <int VALUES> __global__ void __launch_bounds__(DEC8_WARPS * 32) decode8_kernel(const Decode8Params p) {
    __shared__ float s_m[DEC8_WARPS][DEC8_G], s_l[DEC8_WARPS][DEC8_G], s_o[DEC8_WARPS][DEC8_G][KV8_D];
    ptx::grid_dependency_wait();
    ptx::grid_launch_dependents();
    const int b = blockIdx.x / p.Hkv, g = blockIdx.x % p.Hkv, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int L = max(0, min(p.seq_lens[b], p.max_seq_len));
    float q[DEC8_G][2], m[DEC8_G], l[DEC8_G], o[DEC8_G][2];
    float c = 1.f, s = 0.f;
    if (p.rope_q) rotation(p.q_positions ? p.q_positions[b] : L - 1, p.freqs.f[lane], &c, &s);
#pragma unroll
    for (int h = 0; h < DEC8_G; ++h) {
        float x = 0.f, y = 0.f;
        if (h < p.n_rep) {
            const __nv_bfloat16* src = p.q + ((int64_t)b * p.Hq + g * p.n_rep + h) * KV8_D + 2 * lane;
            x = to_f(src[0]);
            y = to_f(src[1]);
        }
        q[h][0] = (x * c - y * s) * p.scale;
        q[h][1] = (x * s + y * c) * p.scale;
        m[h] = -INFINITY;
        l[h] = o[h][0] = o[h][1] = 0.f;
    }
    for (int t = warp; t < L; t += DEC8_WARPS) {
        int page = p.page_table[(int64_t)b * p.max_pages + t / BN_PAGE_TOKENS];
        if (page < 0 || page >= p.pool_pages) {
            if (lane == 0) atomicExch(p.error, BN_ERR_INVALID_ARG);
            page = 0;
        }
        const int slot = t % BN_PAGE_TOKENS;
        const uint8_t* block = p.pool + ((int64_t)page * p.Hkv + g) * BN_KV8_BLOCK;
        uint32_t lo, hi;
        kv8_halves<VALUES>(*reinterpret_cast<const uint16_t*>(block + slot * KV8_D + 2 * lane), lo, hi);
        const float2 k = halves_to_floats(lo);
        kv8_halves<VALUES>(*reinterpret_cast<const uint16_t*>(block + KV8_V + slot * KV8_D + kv8_v_place(slot, 2 * lane)), lo, hi);
        const float2 v = halves_to_floats(lo);
        const uint32_t scales = *reinterpret_cast<const uint32_t*>(block + KV8_SCALES + slot * 4);
        const float ks = ptx::bf16_lo(scales), vs = ptx::bf16_hi(scales);
#pragma unroll
        for (int h = 0; h < DEC8_G; ++h) {
            float z = q[h][0] * k.x + q[h][1] * k.y;
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) z += __shfl_xor_sync(0xffffffffu, z, w);
            z *= ks;
            const float top = fmaxf(m[h], z), keep = expf(m[h] - top), e = expf(z - top);
            m[h] = top;
            l[h] = l[h] * keep + e;
            o[h][0] = o[h][0] * keep + e * vs * v.x;
            o[h][1] = o[h][1] * keep + e * vs * v.y;
        }
    }
#pragma unroll
    for (int h = 0; h < DEC8_G; ++h) {
        s_m[warp][h] = m[h];
        s_l[warp][h] = l[h];
        s_o[warp][h][2 * lane] = o[h][0];
        s_o[warp][h][2 * lane + 1] = o[h][1];
    }
    __syncthreads();
    const int h = warp;
    if (h >= p.n_rep) return;
    float top = -INFINITY, sum = 0.f, a = 0.f, d = 0.f;
    for (int w = 0; w < DEC8_WARPS; ++w) top = fmaxf(top, s_m[w][h]);
    for (int w = 0; w < DEC8_WARPS && L > 0; ++w) {
        const float f = s_l[w][h] == 0.f ? 0.f : expf(s_m[w][h] - top);
        sum += s_l[w][h] * f;
        a += s_o[w][h][2 * lane] * f;
        d += s_o[w][h][2 * lane + 1] * f;
    }
    const float inv = L > 0 ? 1.f / sum : 0.f;
    const int64_t row = (int64_t)b * p.Hq + g * p.n_rep + h;
    if (p.out) *reinterpret_cast<uint32_t*>(p.out + row * KV8_D + 2 * lane) = ptx::pack_bf16(a * inv, d * inv);
    if (p.out_f32) *reinterpret_cast<float2*>(p.out_f32 + row * KV8_D + 2 * lane) = make_float2(a * inv, d * inv);
    if (p.lse && lane == 0) p.lse[row] = L > 0 ? top + logf(sum) : -INFINITY;
}

}  // namespace bn

using namespace bn;

extern "C" size_t bn_attn_decode_kv8_workspace_bytes(int B, int Hq, int Hkv, int D, int max_seq_len, int chunk_tokens) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || D != KV8_D || max_seq_len < 0 || chunk_tokens < 0 || chunk_tokens % 128) return 0;
    return 256;
}

extern "C" int bn_attn_decode_kv8(const void* q, const void* pool, int64_t pool_pages, const int32_t* page_table, int max_pages,
                                  const int32_t* seq_lens, const int32_t* q_positions, void* out, float* out_f32, float* lse, int values, int B, int Hq,
                                  int Hkv, int D, float scale, float theta, int rope_q, int max_seq_len, int chunk_tokens, void* workspace,
                                  size_t workspace_bytes, bn_stream_t stream) {
    const char* what = "bn_attn_decode_kv8";
    if (!q || !pool || !page_table || !seq_lens) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (!out && !out_f32) return fail(BN_ERR_INVALID_ARG, "%s: no output buffer", what);
    if (B < 0 || Hq <= 0 || Hkv <= 0 || max_pages < 0 || max_seq_len < 0 || pool_pages <= 0)
        return fail(BN_ERR_INVALID_ARG, "%s: bad sizes B=%d Hq=%d Hkv=%d max_pages=%d", what, B, Hq, Hkv, max_pages);
    if (D != KV8_D) return fail(BN_ERR_UNSUPPORTED, "%s: head_dim=%d (64 supported)", what, D);
    if (values != BN_KV8_E4M3 && values != BN_KV8_INT8) return fail(BN_ERR_INVALID_ARG, "%s: values=%d (0 = e4m3, 1 = int8)", what, values);
    if (Hq % Hkv != 0 || Hq / Hkv > DEC8_G) return fail(BN_ERR_UNSUPPORTED, "%s: Hq/Hkv=%d/%d (group of 1..8 supported)", what, Hq, Hkv);
    if (B > 1024) return fail(BN_ERR_UNSUPPORTED, "%s: %d sequences in one launch (<= 1024 supported)", what, B);
    if (chunk_tokens < 0 || chunk_tokens % 128) return fail(BN_ERR_INVALID_ARG, "%s: chunk_tokens=%d must be 0 or a multiple of 128", what, chunk_tokens);
    if ((int64_t)max_pages * BN_PAGE_TOKENS < max_seq_len)
        return fail(BN_ERR_INVALID_ARG, "%s: max_pages=%d cannot hold max_seq_len=%d", what, max_pages, max_seq_len);
    if (rope_q && !(theta > 0.f)) return fail(BN_ERR_INVALID_ARG, "%s: theta=%g", what, theta);
    if ((reinterpret_cast<uintptr_t>(pool) & 15) || (reinterpret_cast<uintptr_t>(q) & 7) || (out && (reinterpret_cast<uintptr_t>(out) & 7)) ||
        (out_f32 && (reinterpret_cast<uintptr_t>(out_f32) & 15)))
        return fail(BN_ERR_INVALID_ARG, "%s: pool/q/out buffers must be 16/8/8/16-byte aligned", what);
    if (int rc = require_sm100()) return rc;
    if (B == 0) return BN_OK;
    const size_t need = bn_attn_decode_kv8_workspace_bytes(B, Hq, Hkv, D, max_seq_len, chunk_tokens);
    if (!workspace || workspace_bytes < need) return fail(BN_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", what, workspace_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(BN_ERR_INVALID_ARG, "%s: workspace must be 256-byte aligned", what);
    Decode8Params p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.pool = static_cast<const uint8_t*>(pool);
    p.pool_pages = pool_pages;
    p.page_table = page_table; p.seq_lens = seq_lens; p.q_positions = q_positions;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.out_f32 = out_f32; p.lse = lse;
    p.error = static_cast<int*>(workspace);
    p.Hq = Hq; p.Hkv = Hkv; p.n_rep = Hq / Hkv; p.max_pages = max_pages; p.max_seq_len = max_seq_len; p.rope_q = rope_q;
    p.scale = scale;
    if (rope_q) p.freqs = rotation_freqs(theta);
    auto* kernel = values == BN_KV8_E4M3 ? decode8_kernel<BN_KV8_E4M3> : decode8_kernel<BN_KV8_INT8>;
    launch_dependent(kernel, (unsigned)(B * Hkv), DEC8_WARPS * 32, 0, as_stream(stream), p);
    return launch_status(what);
}
