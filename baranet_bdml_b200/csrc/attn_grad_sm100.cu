// Gradients of bn_attn_prefill_bf16 for sm_100a: rotated grouped-query attention by q, k and v (in the reference the chain of
// op_softmax_backward, src/ops/op_softmax.cuh:185-246, op_rope_backward, src/ops/op_rope.cuh:130-193, and two products of op_mm).
//
// With S = scale Q K^T on rotated q and k, P = exp(S - lse) and d_i = sum_c dO_ic O_ic:
//     dV = P^T dO    dP = dO V^T    dS = P (dP - d)    dQ = scale dS K    dK = scale dS^T Q
// and dQ, dK are turned back by the rows' angles.  P is computed again from lse, so nothing of size S x S is ever in memory.
//
// Launch 1 (prepare): q and k rotated once (each is read by many tiles), d and lse * log2(e) side by side per query.
// Launch 2: blocks of two kinds in one grid.  A KEY block holds 128 keys of one key head (K and V) and walks the query tiles of its heads
// that see them: dK and dV stay in tensor memory.  A QUERY block holds 128 queries of one head (Q and dO) and walks the key tiles: dQ stays
// in tensor memory.  P and dP are computed by both, 7 products of a tile instead of 5, and no gradient is summed by atomics: the
// same bits in every run, and no fp32 copy of dQ in memory.
// Both kinds are one program: F1, F2 are held and X1, X2 come in tiles of 64 rows,
//     S = F1 X1^T,  dP = F2 X2^T,  acc2 += dS X1,  and for keys acc1 += P X2        (keys: F = K, V, X = Q, dO; queries: F = Q, dO, X = K, V)
// P and dS are written as bf16 over the scores they came from and are the A operands of the second products (from tensor memory); X1 and X2
// are B operands twice, along both of their dimensions.  256 columns of tensor memory and 101 KB of shared memory: two blocks to an SM,
// so one block's softmax runs beside the other's products.
// Ten warps: 0-7 softmax (two threads a row, 32 columns each), 8 issues the MMAs, 9 loads by TMA.  S of the next tile is computed while
// dS of this one is.
// Launch 3, where the heads of a group are shared by several blocks: their fp32 sums of dK and dV are added in order.
// Every mbarrier wait is bounded; on expiry the kernel raises the caller's error word, frees TMEM and returns.
#include "common.cuh"
#include "ptx.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace bn {

using namespace ptx;

constexpr int AG_D = 64, AG_BF = 128, AG_BX = 64, AG_STAGES = 4, AG_THREADS = 320;
constexpr int AG_F_BYTES = AG_BF * AG_D * 2, AG_X_BYTES = AG_BX * AG_D * 2, AG_STAT_BYTES = AG_BX * 8;
constexpr int AG_STAGE_BYTES = 2 * AG_X_BYTES;
constexpr int AG_SMEM_BYTES = 1024 + 2 * AG_F_BYTES + AG_STAGES * (AG_STAGE_BYTES + AG_STAT_BYTES);
constexpr uint32_t AG_TMEM = 256, AG_S = 0, AG_DP = 64, AG_ACC1 = 128, AG_ACC2 = 192;

struct AttnGradParams {
    const float* stats;                  // [B][Hq][-lse * log2(e), -d][padded S]; rows behind S: -inf, 0
    const float2* table;                 // [S][32] cos, sin
    __nv_bfloat16 *dq, *dk, *dv;
    float* partial;                      // [part][dv, dk][B][S][Hkv][64]
    int* error_word;
    int B, S, padded, Hq, Hkv, rep, tiles, parts, key_blocks, offset, causal;
    float scale, scale_log2;
};

// 32 columns of a gradient row, `col` on: scaled, turned back by the row's angles where `table` is given, stored as bf16
__device__ __forceinline__ void store_gradient(__nv_bfloat16* row, const float2* table, int col, float scale, const float (&v)[32]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = v[q * 8 + 2 * e] * scale, b = v[q * 8 + 2 * e + 1] * scale;
            if (table) {
                const float2 t = table[col / 2 + q * 4 + e];
                w[e] = pack_bf16(a * t.x + b * t.y, b * t.x - a * t.y);
            } else {
                w[e] = pack_bf16(a, b);
            }
        }
        *reinterpret_cast<uint4*>(row + col + q * 8) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Rotated copies of q and k, the table of cos and sin, and a query's lse and d side by side.  A block has 16 positions and a share of the
// heads; 8 neighbouring lanes have a head's 64 values.
constexpr int AP_POS = 16, AP_THREADS = 256;
__global__ void __launch_bounds__(AP_THREADS)
attn_grad_prepare_kernel(const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* out, const __nv_bfloat16* dout, const float* lse, __nv_bfloat16* qrot,
                         __nv_bfloat16* krot, float2* table, float* stats, int S, int padded, int Hq, int Hkv, float theta, int offset) {
    __shared__ float2 cs[AP_POS][AG_D / 2];
    grid_dependency_wait();
    const int s0 = blockIdx.x * AP_POS, b = blockIdx.y, share = blockIdx.z, shares = gridDim.z;
    for (int e = threadIdx.x; e < AP_POS * (AG_D / 2); e += AP_THREADS) {
        const int s = e / (AG_D / 2), i = e % (AG_D / 2);
        const float angle = (s0 + s + offset) * rope_inv_freq(i, AG_D, theta);
        const float2 v = make_float2(cosf(angle), sinf(angle));
        cs[s][i] = v;
        if (b == 0 && share == 0 && s0 + s < S) table[(size_t)(s0 + s) * (AG_D / 2) + i] = v;
    }
    __syncthreads();
    auto rotate = [&](uint4 x, int s, int c) {
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const float2 v = cs[s][c * 4 + t];
            const float x0 = bf16_lo(w[t]), x1 = bf16_hi(w[t]);
            w[t] = pack_bf16(x0 * v.x - x1 * v.y, x0 * v.y + x1 * v.x);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    const int h0 = (int)((long long)Hq * share / shares), heads = (int)((long long)Hq * (share + 1) / shares) - h0;
#pragma unroll 2
    for (int e = threadIdx.x; e < AP_POS * heads * 8; e += AP_THREADS) {              // (a multiple of 32: whole warps)
        const int c = e % 8, h = h0 + e / 8 % heads, s = e / 8 / heads, pos = s0 + s;
        float sum = 0.f;
        if (pos < S) {
            const size_t at = (((size_t)b * S + pos) * Hq + h) * 8 + c;
            const uint4 x = reinterpret_cast<const uint4*>(q)[at], o = reinterpret_cast<const uint4*>(out)[at], d = reinterpret_cast<const uint4*>(dout)[at];
            reinterpret_cast<uint4*>(qrot)[at] = rotate(x, s, c);
            const uint32_t ow[4] = {o.x, o.y, o.z, o.w}, dw[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int t = 0; t < 4; ++t) sum = fmaf(bf16_lo(ow[t]), bf16_lo(dw[t]), fmaf(bf16_hi(ow[t]), bf16_hi(dw[t]), sum));
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        if (c == 0 && pos < padded) {
            float* to = stats + ((size_t)b * Hq + h) * 2 * padded + pos;
            to[0] = pos < S ? lse[((size_t)b * Hq + h) * S + pos] * -1.4426950408889634f : -INFINITY;
            to[padded] = pos < S ? -sum : 0.f;
        }
    }
    const int g0 = (int)((long long)Hkv * share / shares), groups = (int)((long long)Hkv * (share + 1) / shares) - g0;
    for (int e = threadIdx.x; e < AP_POS * groups * 8; e += AP_THREADS) {
        const int c = e % 8, g = g0 + e / 8 % groups, s = e / 8 / groups, pos = s0 + s;
        if (pos >= S) continue;
        const size_t at = (((size_t)b * S + pos) * Hkv + g) * 8 + c;
        reinterpret_cast<uint4*>(krot)[at] = rotate(reinterpret_cast<const uint4*>(k)[at], s, c);
    }
}

struct AttnGradShared {
    uint64_t bar_full[AG_STAGES], bar_empty[AG_STAGES], bar_fixed, bar_s, bar_dp, bar_p, bar_ds, bar_done;
    uint32_t tmem_base;
    int abort;
};

template <bool KEYS>
__device__ __forceinline__ void attn_grad_block(const CUtensorMap* map_f1, const CUtensorMap* map_f2, const CUtensorMap* map_x1, const CUtensorMap* map_x2,
                                                const AttnGradParams& p, AttnGradShared& sh, uint32_t smem0, int unit) {
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t sF1 = smem0, sF2 = smem0 + AG_F_BYTES, sX = smem0 + 2 * AG_F_BYTES, sStat = sX + AG_STAGES * AG_STAGE_BYTES;
    const uint32_t tmem = sh.tmem_base;
    // the block's rows f0 .. f0 + 127 of head hf of sequence b; its tiles of 64 rows: x tile x_lo .. x_hi - 1 of heads hx .. hx + heads - 1
    int b, hf, f0, hx, heads, x_lo, x_hi, part = 0;
    if (KEYS) {                                          // the first key tiles, which most queries see, come first
        part = unit % p.parts;
        const int bg = unit / p.parts % (p.B * p.Hkv), tile = unit / p.parts / (p.B * p.Hkv);
        b = bg / p.Hkv;
        hf = bg % p.Hkv;
        f0 = tile * AG_BF;
        hx = hf * p.rep + p.rep * part / p.parts;
        heads = hf * p.rep + p.rep * (part + 1) / p.parts - hx;
        x_lo = p.causal ? max(0, f0 - p.offset) / AG_BX : 0;
        x_hi = (p.S + AG_BX - 1) / AG_BX;
    } else {                                             // the last query tiles, which see most keys, come first
        const int bh = unit % (p.B * p.Hq), tile = p.tiles - 1 - unit / (p.B * p.Hq);
        b = bh / p.Hq;
        hf = bh % p.Hq;
        f0 = tile * AG_BF;
        hx = hf / p.rep;
        heads = 1;
        x_lo = 0;
        x_hi = (p.causal ? (int)min((long long)p.S - 1, (long long)f0 + AG_BF - 1 + p.offset) : p.S - 1) / AG_BX + 1;
    }
    const int per_head = x_hi - x_lo, steps = heads * per_head;

    if (warp == 9) {
        // ---------------------------------------------------------- TMA producer
        if (lane == 0) {
            mbar_arrive_expect_tx(smem_u32(&sh.bar_fixed), 2 * AG_F_BYTES);
            tma_load_4d(sF1, map_f1, 0, hf, f0, b, smem_u32(&sh.bar_fixed));
            tma_load_4d(sF2, map_f2, 0, hf, f0, b, smem_u32(&sh.bar_fixed));
            int h = hx, x = x_lo;
            for (int i = 0; i < steps; ++i) {
                const int st = i % AG_STAGES;
                if (!mbar_wait(smem_u32(&sh.bar_empty[st]), ((i / AG_STAGES) & 1u) ^ 1u, &sh.abort)) break;
                const uint32_t full = smem_u32(&sh.bar_full[st]), dst = sX + st * AG_STAGE_BYTES;
                mbar_arrive_expect_tx(full, AG_STAGE_BYTES + (KEYS ? AG_STAT_BYTES : 0));
                tma_load_4d(dst, map_x1, 0, h, x * AG_BX, b, full);
                tma_load_4d(dst + AG_X_BYTES, map_x2, 0, h, x * AG_BX, b, full);
                if (KEYS) {
                    const float* from = p.stats + ((size_t)b * p.Hq + h) * 2 * p.padded + x * AG_BX;
                    bulk_load(sStat + st * AG_STAT_BYTES, from, AG_STAT_BYTES / 2, full);
                    bulk_load(sStat + st * AG_STAT_BYTES + AG_STAT_BYTES / 2, from + p.padded, AG_STAT_BYTES / 2, full);
                }
                if (++x == x_hi) { x = x_lo; ++h; }
            }
        }
    } else if (warp == 8) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t I_SCORE = tc::idesc_bf16(AG_BF, AG_BX, 0), I_GRAD = tc::idesc_bf16(AG_BF, AG_D, 1);
        const uint64_t d0 = tc::smem_desc_sw128(0);
        auto at = [&](uint32_t addr) { return d0 + (uint64_t)(addr >> 4); };
        auto score = [&](uint32_t column, uint32_t sF, uint32_t sXi, uint32_t bar) {          // F X^T
#pragma unroll
            for (int kk = 0; kk < AG_D / 16; ++kk) tc::mma_ss(tmem + column, at(sF + kk * 32), at(sXi + kk * 32), I_SCORE, kk > 0);
            tc::commit(bar);
        };
        auto grad = [&](uint32_t column, uint32_t from, uint32_t sXi, bool first) {           // (P or dS) X; the halves of a row lie 32 columns apart
#pragma unroll
            for (int kk = 0; kk < AG_BX / 16; ++kk)
                tc::mma_ts(tmem + column, tmem + from + kk / 2 * 32 + kk % 2 * 8, at(sXi + kk * 2048), I_GRAD, !first || kk > 0);
        };
        bool ok = mbar_wait_warp(smem_u32(&sh.bar_fixed), 0, &sh.abort) && mbar_wait_warp(smem_u32(&sh.bar_full[0]), 0, &sh.abort);
        if (ok && elect_one()) {
            tc::fence_after_sync();
            score(AG_S, sF1, sX, smem_u32(&sh.bar_s));
            score(AG_DP, sF2, sX + AG_X_BYTES, smem_u32(&sh.bar_dp));
        }
        __syncwarp();
        for (int i = 0; ok && i < steps; ++i) {
            const int st = i % AG_STAGES, nx = (i + 1) % AG_STAGES;
            const uint32_t here = sX + st * AG_STAGE_BYTES, next = sX + nx * AG_STAGE_BYTES;
            const bool more = i + 1 < steps;
            // the scores have been read (and P lies over them): P X2, then the next tile's scores into their place (MMAs run in order)
            ok = mbar_wait_warp(smem_u32(&sh.bar_p), i & 1, &sh.abort);
            if (ok && more) ok = mbar_wait_warp(smem_u32(&sh.bar_full[nx]), ((i + 1) / AG_STAGES) & 1u, &sh.abort);
            if (!ok) break;
            if (elect_one()) {
                tc::fence_after_sync();
                if (KEYS) grad(AG_ACC1, AG_S, here + AG_X_BYTES, i == 0);
                if (more) score(AG_S, sF1, next, smem_u32(&sh.bar_s));
            }
            __syncwarp();
            ok = mbar_wait_warp(smem_u32(&sh.bar_ds), i & 1, &sh.abort);
            if (!ok) break;
            if (elect_one()) {
                tc::fence_after_sync();
                grad(AG_ACC2, AG_DP, here, i == 0);
                tc::commit(smem_u32(&sh.bar_empty[st]));
                if (more) score(AG_DP, sF2, next + AG_X_BYTES, smem_u32(&sh.bar_dp));
                else tc::commit(smem_u32(&sh.bar_done));
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------ softmax warps: thread = (row = TMEM lane, half of the tile's 64 columns)
        const int half = warp / 4, row = tid % 128, f = f0 + row;
        const uint32_t mine = tmem + ((uint32_t)(warp % 4 * 32) << 16) + half * 32;
        uint64_t lse2 = 0, d2 = 0;                                                 // -lse * log2(e) and -d of the row, twice
        if (!KEYS) {
            const float* of = p.stats + ((size_t)b * p.Hq + hf) * 2 * p.padded + f;    // (rows behind S are padded)
            lse2 = pack_f32x2(of[0], of[0]);
            d2 = pack_f32x2(of[p.padded], of[p.padded]);
        }
        const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
        // which columns of a tile a row sees: keys from x >= first on, queries up to x <= last
        const int first = KEYS && p.causal ? f - p.offset : 0, last = KEYS ? INT32_MAX : (p.causal ? (int)min((long long)p.S - 1, (long long)f + p.offset) : p.S - 1);
        const int all_first = KEYS && p.causal ? f0 + AG_BF - 1 - p.offset : 0, all_last = KEYS ? INT32_MAX : (p.causal ? (int)min((long long)p.S - 1, (long long)f0 + p.offset) : p.S - 1);
        int x = x_lo;
        bool ok = true;
        for (int i = 0; i < steps; ++i) {
            const int st = i % AG_STAGES, x0 = x * AG_BX;
            if (++x == x_hi) x = x_lo;
            const bool masked = x0 < all_first || x0 + AG_BX - 1 > all_last;       // (the same for the whole block)
            const uint32_t stat = sStat + st * AG_STAT_BYTES + half * (AG_STAT_BYTES / 4);      // of the half's 32 columns
            // four columns' values of one kind; for a row of queries the row's own
            auto of_columns = [&](uint32_t from, int e, uint64_t own, uint64_t& lo, uint64_t& hi) {
                if (KEYS) asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];" : "=l"(lo), "=l"(hi) : "r"(from + e * 4));
                else lo = hi = own;
            };
            ok = mbar_wait_warp(smem_u32(&sh.bar_s), i & 1, &sh.abort);          // (the tile and its statistics came before)
            if (KEYS && ok) ok = mbar_wait_warp(smem_u32(&sh.bar_full[st]), (i / AG_STAGES) & 1u, &sh.abort);
            if (!ok) break;
            tc::fence_after_sync();
            uint32_t s[32];
            tc::ld32(mine + AG_S, s);
            tc::wait_ld(s);
            uint64_t pr[16];
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                uint64_t l[2];
                of_columns(stat, e, lse2, l[0], l[1]);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float a, c;
                    unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[e + 2 * j]), __uint_as_float(s[e + 2 * j + 1])), scale2, l[j]), a, c);
                    pr[e / 2 + j] = pack_f32x2(ex2(a), ex2(c));
                }
            }
            if (masked) {                                // (dS has the factor P, so one mask is enough)
                const int c0 = x0 + half * 32;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float a, c;
                    unpack_f32x2(pr[e], a, c);
                    if (c0 + 2 * e < first || c0 + 2 * e > last) a = 0.f;
                    if (c0 + 2 * e + 1 < first || c0 + 2 * e + 1 > last) c = 0.f;
                    pr[e] = pack_f32x2(a, c);
                }
            }
            auto packed = [](uint64_t v) {
                float a, c;
                unpack_f32x2(v, a, c);
                return pack_bf16(a, c);
            };
            uint32_t pk[16];
            if (KEYS) {
#pragma unroll
                for (int e = 0; e < 16; ++e) pk[e] = packed(pr[e]);
                tc::st16(mine + AG_S, pk);
                tc::wait_st();
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.bar_p));
            ok = mbar_wait_warp(smem_u32(&sh.bar_dp), i & 1, &sh.abort);
            if (!ok) break;
            tc::fence_after_sync();
            tc::ld32(mine + AG_DP, s);
            tc::wait_ld(s);
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
                uint64_t l[2];
                of_columns(stat + AG_STAT_BYTES / 2, e, d2, l[0], l[1]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    pk[e / 2 + j] = packed(mul_f32x2(pr[e / 2 + j], add_f32x2(pack_f32x2(__uint_as_float(s[e + 2 * j]), __uint_as_float(s[e + 2 * j + 1])), l[j])));
            }
            tc::st16(mine + AG_DP, pk);
            tc::wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.bar_ds));
        }
        // ------------------------------------------------ the block's gradients
        if (ok) ok = mbar_wait_warp(smem_u32(&sh.bar_done), 0, &sh.abort);
        if (ok) {
            tc::fence_after_sync();
            // keys: the first four warps have dV, the others dK; queries: each half of dQ's columns
            const int n = KEYS ? 2 : 1;
#pragma unroll
            for (int c = 0; c < n; ++c) {
                const int col = KEYS ? c * 32 : half * 32;
                uint32_t r[32];
                tc::ld32(tmem + ((uint32_t)(warp % 4 * 32) << 16) + (KEYS && half == 0 ? AG_ACC1 : AG_ACC2) + col, r);
                tc::wait_ld(r);
                if (f < p.S) {
                    float v[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = __uint_as_float(r[e]);
                    const float2* table = p.table + (size_t)f * (AG_D / 2);
                    if (!KEYS) {
                        store_gradient(p.dq + (((size_t)b * p.S + f) * p.Hq + hf) * AG_D, table, col, p.scale, v);
                    } else if (p.parts == 1) {
                        const size_t at = (((size_t)b * p.S + f) * p.Hkv + hf) * AG_D;
                        store_gradient((half ? p.dk : p.dv) + at, half ? table : nullptr, col, half ? p.scale : 1.f, v);
                    } else {
                        float* to = p.partial + ((((size_t)(part * 2 + half) * p.B + b) * p.S + f) * p.Hkv + hf) * AG_D + col;
#pragma unroll
                        for (int e = 0; e < 8; ++e) reinterpret_cast<float4*>(to)[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
                    }
                }
            }
        }
    }
}

__global__ void __launch_bounds__(AG_THREADS, 2)
attn_grad_kernel(const __grid_constant__ CUtensorMap q_tile, const __grid_constant__ CUtensorMap do_tile, const __grid_constant__ CUtensorMap k_tile,
                 const __grid_constant__ CUtensorMap v_tile, const __grid_constant__ CUtensorMap q_rows, const __grid_constant__ CUtensorMap do_rows,
                 const __grid_constant__ CUtensorMap k_rows, const __grid_constant__ CUtensorMap v_rows, const AttnGradParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) AttnGradShared sh;
    const int warp = threadIdx.x / 32;
    if (threadIdx.x == 0) {
        for (int s = 0; s < AG_STAGES; ++s) {
            mbar_init(smem_u32(&sh.bar_full[s]), 1);
            mbar_init(smem_u32(&sh.bar_empty[s]), 1);
        }
        mbar_init(smem_u32(&sh.bar_fixed), 1);
        mbar_init(smem_u32(&sh.bar_s), 1);
        mbar_init(smem_u32(&sh.bar_dp), 1);
        mbar_init(smem_u32(&sh.bar_p), 8);                // one arrive per softmax warp
        mbar_init(smem_u32(&sh.bar_ds), 8);
        mbar_init(smem_u32(&sh.bar_done), 1);
        sh.abort = 0;
        fence_mbar_init();
    }
    if (warp == 8) {
        tc::tmem_alloc(smem_u32(&sh.tmem_base), AG_TMEM);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    grid_dependency_wait();
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    if ((int)blockIdx.x < p.key_blocks) attn_grad_block<true>(&k_tile, &v_tile, &q_rows, &do_rows, p, sh, smem0, blockIdx.x);
    else attn_grad_block<false>(&q_tile, &do_tile, &k_rows, &v_rows, p, sh, smem0, blockIdx.x - p.key_blocks);
    // common exit: everybody arrives here (bounded waits), then TMEM is freed
    tc::fence_before_sync();
    __syncthreads();
    if (threadIdx.x == 0 && sh.abort && p.error_word) atomicExch(p.error_word, BN_ERR_TIMEOUT);
    if (warp == 8) {
        tc::fence_after_sync();
        tc::tmem_dealloc(sh.tmem_base, AG_TMEM);
    }
}

// dV and dK of the blocks that share a group's heads, added in their order; a thread has 32 columns of a row
__global__ void __launch_bounds__(128) attn_grad_sum_kernel(const AttnGradParams p) {
    grid_dependency_wait();
    const long long rows = (long long)p.B * p.S * p.Hkv, e = (long long)blockIdx.x * 128 + threadIdx.x, row = e / 2;
    if (row >= rows) return;
    const int col = (int)(e % 2) * 32, which = blockIdx.y;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0.f;
    for (int part = 0; part < p.parts; ++part) {
        const float4* from = reinterpret_cast<const float4*>(p.partial + ((size_t)(part * 2 + which) * rows + row) * AG_D + col);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 t = __ldcg(from + i);
            v[4 * i] += t.x; v[4 * i + 1] += t.y; v[4 * i + 2] += t.z; v[4 * i + 3] += t.w;
        }
    }
    store_gradient((which ? p.dk : p.dv) + (size_t)row * AG_D, which ? p.table + (size_t)(row / p.Hkv % p.S) * (AG_D / 2) : nullptr, col, which ? p.scale : 1.f, v);
}

}  // namespace bn

using namespace bn;

namespace {

struct AttnGradLayout { size_t table, stats, qrot, krot, partial, total; int parts, padded; };

// How many blocks share the heads of a group: the longest block should not take longer than all blocks' work spread over the GPU
// (two blocks to an SM), or it is what the launch waits for; each further part is written and read again in fp32.
AttnGradLayout attn_grad_layout(int B, int S, int Hq, int Hkv, int causal) {
    AttnGradLayout L;
    const long long tiles = (S + AG_BF - 1) / AG_BF, n = (S + AG_BX - 1) / AG_BX, rep = Hq / Hkv;
    const long long all = 2 * (long long)B * Hq * tiles * n / (causal ? 2 : 1), slots = 2 * sm_count();
    int parts = 1;
    while (parts < rep && (rep + parts - 1) / parts * n * slots > all) ++parts;
    L.parts = parts;
    L.padded = (int)(tiles * AG_BF);
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    L.table = 0;
    L.stats = up((size_t)S * (AG_D / 2) * sizeof(float2));
    L.qrot = L.stats + up((size_t)B * Hq * 2 * L.padded * sizeof(float));
    L.krot = L.qrot + up((size_t)B * S * Hq * AG_D * 2);
    L.partial = L.krot + up((size_t)B * S * Hkv * AG_D * 2);
    L.total = L.partial + (parts > 1 ? up((size_t)parts * 2 * B * S * Hkv * AG_D * sizeof(float)) : 0);
    return L;
}

}  // namespace

extern "C" size_t bn_attn_prefill_bf16_backward_workspace_bytes(int B, int S, int Hq, int Hkv, int D, int causal) {
    if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D != AG_D) return 0;
    return attn_grad_layout(B, S, Hq, Hkv, causal).total;
}

extern "C" int bn_attn_prefill_bf16_backward(const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse, void* dq,
                                             void* dk, void* dv, int B, int S, int Hq, int Hkv, int D, float scale, float theta, int position_offset,
                                             int causal, void* workspace, size_t workspace_bytes, int* error_word, bn_stream_t stream) {
    const char* what = "bn_attn_prefill_bf16_backward";
    if (!dout || !q || !k || !v || !out || !lse || !dq || !dk || !dv) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (B < 0 || S < 0 || Hq <= 0 || Hkv <= 0) return fail(BN_ERR_INVALID_ARG, "%s: bad shape B=%d S=%d Hq=%d Hkv=%d", what, B, S, Hq, Hkv);
    if (Hq % Hkv) return fail(BN_ERR_INVALID_ARG, "%s: Hq=%d not a multiple of Hkv=%d", what, Hq, Hkv);
    if (D != AG_D) return fail(BN_ERR_UNSUPPORTED, "%s: head_dim=%d (64 supported)", what, D);
    if (position_offset < 0) return fail(BN_ERR_INVALID_ARG, "%s: position_offset=%d < 0", what, position_offset);
    for (const void* t : {dout, q, k, v, out, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
        if (reinterpret_cast<uintptr_t>(t) & 15) return fail(BN_ERR_INVALID_ARG, "%s: tensors must be 16-byte aligned", what);
    if (int rc = require_sm100()) return rc;
    if (B == 0 || S == 0) return BN_OK;
    const AttnGradLayout L = attn_grad_layout(B, S, Hq, Hkv, causal);
    if (!workspace || workspace_bytes < L.total) return fail(BN_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", what, workspace_bytes, L.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(BN_ERR_INVALID_ARG, "%s: workspace must be 256-byte aligned", what);
    const long long tiles = (S + AG_BF - 1) / AG_BF, key_blocks = tiles * B * Hkv * L.parts, blocks = key_blocks + tiles * B * Hq;
    const long long sum_blocks = ((long long)B * S * Hkv * 2 + 127) / 128;
    if (blocks > INT32_MAX || sum_blocks > INT32_MAX || B > 65535 || S > INT32_MAX - 256 || position_offset > INT32_MAX - S - 256)
        return fail(BN_ERR_UNSUPPORTED, "%s: problem too large for one launch", what);

    uint8_t* ws = static_cast<uint8_t*>(workspace);
    cudaStream_t st = as_stream(stream);
    AttnGradParams p{};
    p.stats = reinterpret_cast<const float*>(ws + L.stats);
    p.table = reinterpret_cast<const float2*>(ws + L.table);
    p.dq = static_cast<__nv_bfloat16*>(dq);
    p.dk = static_cast<__nv_bfloat16*>(dk);
    p.dv = static_cast<__nv_bfloat16*>(dv);
    p.partial = reinterpret_cast<float*>(ws + L.partial);
    p.error_word = error_word;
    p.B = B; p.S = S; p.padded = L.padded; p.Hq = Hq; p.Hkv = Hkv; p.rep = Hq / Hkv; p.tiles = (int)tiles; p.parts = L.parts;
    p.key_blocks = (int)key_blocks;
    p.offset = position_offset;
    p.causal = causal != 0;
    p.scale = scale;
    p.scale_log2 = scale * 1.4426950408889634f;
    __nv_bfloat16 *qrot = reinterpret_cast<__nv_bfloat16*>(ws + L.qrot), *krot = reinterpret_cast<__nv_bfloat16*>(ws + L.krot);

    CUtensorMap maps[8];
    {
        const void* base[4] = {qrot, dout, krot, v};
        for (int i = 0; i < 8; ++i) {
            const uint64_t heads = i % 4 < 2 ? Hq : Hkv;
            const uint64_t dims[4] = {AG_D, heads, (uint64_t)S, (uint64_t)B}, strides[3] = {AG_D * 2, heads * AG_D * 2, (uint64_t)S * heads * AG_D * 2};
            const uint32_t box[4] = {AG_D, 1, (uint32_t)(i < 4 ? AG_BF : AG_BX), 1};
            if (int rc = make_tensor_map(&maps[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base[i % 4], dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
        }
    }
    // enough blocks for the GPU, by positions and, where those are few, by heads too
    const unsigned pos_blocks = (unsigned)(L.padded / AP_POS);
    long long shares = 4 * sm_count() / ((long long)pos_blocks * B);
    shares = shares < 1 ? 1 : shares > Hq ? Hq : shares;
    launch_dependent(attn_grad_prepare_kernel, dim3(pos_blocks, (unsigned)B, (unsigned)shares), AP_THREADS, 0, st, static_cast<const __nv_bfloat16*>(q),
                     static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(dout), lse, qrot, krot,
                     reinterpret_cast<float2*>(ws + L.table), reinterpret_cast<float*>(ws + L.stats), S, L.padded, Hq, Hkv, theta, position_offset);
    if (int rc = launch_status(what)) return rc;
    if (int rc = allow_smem(attn_grad_kernel, AG_SMEM_BYTES, what, AG_SMEM_BYTES)) return rc;
    launch_dependent(attn_grad_kernel, dim3((unsigned)blocks), AG_THREADS, AG_SMEM_BYTES, st, maps[0], maps[1], maps[2], maps[3], maps[4], maps[5], maps[6],
                     maps[7], p);
    if (int rc = launch_status(what)) return rc;
    if (L.parts > 1) {
        launch_dependent(attn_grad_sum_kernel, dim3((unsigned)sum_blocks, 2), 128, 0, st, p);
        return launch_status(what);
    }
    return BN_OK;
}
