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
// are B operands twice, along both of their dimensions.
// One CTA per SM takes blocks from a counter, the longest first, and goes on to the next without a pause: three F are kept, tiles of X
// come through a ring.  Tensor memory: three slots of S and dP (128 columns) and 128 columns of gradients, so three tiles are under way:
// warps 0-15 are two groups that take tiles in turn (thread = row and half of the columns; three groups of four warps with a row's 64 columns
// each: 544 instead of 538 us at 8 x 2048; three of eight, whose 72 registers a thread are too few, 560); warp 17 loads by TMA; warps 16, 18
// and 19 have a thread each that issues the products of S, of the gradients and of dP; warps 20-23 store a block's gradients under the tiles of
// the next.  (One thread for all products took 1950 cycles a tile for its waits and commits of 100 to 200 cycles each, where the products take
// 530 to 690.)
// A slot's S is free for the next tile as soon as P X2 has been computed, or a query block's group has read it, so S of a tile is there
// before its group is.
// A block's gradients need warps of their own: groups that stored them, 16 columns at a time behind their first tile of the next block, were
// late for their tiles by 3000 cycles a block, most of it code that had left the instruction cache (8 x 2048 591 -> 562 us).  Registers are
// shared out by role, so that no warp spills (softmax warps of eight registers fewer: 571).
// Launch 3, where the heads of a group are shared by several blocks: their fp32 sums of dK and dV are added in order.
// Every mbarrier wait is bounded; on expiry the kernel raises the caller's error word, frees TMEM and returns.
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace bn {

using namespace ptx;

constexpr int AG_D = 64, AG_BF = 128, AG_BX = 64, AG_STAGES = 6, AG_SLOTS = 3, AG_F = 3, AG_UNITS = 8;
constexpr int AG_COLS = AG_BX / 2, AG_GROUPS = 2, AG_SOFT = 8 * AG_GROUPS, AG_THREADS = (AG_SOFT + 8) * 32;      // a thread's columns; groups, their warps
constexpr int AG_F_BYTES = AG_BF * AG_D * 2, AG_X_BYTES = AG_BX * AG_D * 2, AG_STAT_BYTES = AG_BX * 8, AG_F_STAT_BYTES = AG_BF * 8;
constexpr int AG_STAGE_BYTES = 2 * AG_X_BYTES;
constexpr int AG_SMEM_BYTES = 1024 + AG_F * (2 * AG_F_BYTES + AG_F_STAT_BYTES) + AG_STAGES * (AG_STAGE_BYTES + AG_STAT_BYTES);
constexpr uint32_t AG_TMEM = 512, AG_DP = 64, AG_ACC = 384;               // slot: S, then dP; behind the slots two gradients of 64 columns

struct AttnGradParams {
    const float* stats;                  // [B][Hq][-lse * log2(e), -d][padded S]; rows behind S: -inf, 0
    const float2* table;                 // [S][32] cos, sin
    __nv_bfloat16 *dq, *dk, *dv;
    float* partial;                      // [part][dv, dk][B][S][Hkv][64]
    int *error_word, *counter;           // the next block that nobody has
    int blocks, B, S, padded, Hq, Hkv, rep, tiles, parts, key_blocks, offset, causal;
    float scale, scale_log2;
};

// a pair of a gradient by a rotated row, by the row itself
__device__ __forceinline__ uint32_t turned_back(float a, float b, float cos, float sin) { return pack_bf16(a * cos + b * sin, b * cos - a * sin); }

// Rotated copies of q and k, the table of cos and sin, and a query's lse and d side by side.  A block has 4 positions and a share of the
// heads, a warp one position: 8 lanes have a head's 64 values, 4 heads at a time, and their angles in registers; 12 loads of 16 bytes
// under way, the first while the angles are computed.  Memory bounds it: 55 us at 8 x 2048, 4.9 TB/s (16 positions and angles in shared
// memory 73; 8 positions 59, 8 heads more under way 78, loads behind the angles 57).
constexpr int AP_POS = 4, AP_HEADS = 32, AP_THREADS = 32 * AP_POS, AP_BATCH = 4;
__global__ void __launch_bounds__(AP_THREADS)
attn_grad_prepare_kernel(const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* out, const __nv_bfloat16* dout, const float* lse, __nv_bfloat16* qrot,
                         __nv_bfloat16* krot, float2* table, float* stats, int* counter, int taken, int S, int padded, int Hq, int Hkv, float theta, int offset) {
    __shared__ float sums[AP_HEADS][AP_POS + 1];
    grid_dependency_wait();
    if (blockIdx.x + blockIdx.y + blockIdx.z + threadIdx.x == 0) *counter = taken;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, c = lane % 8;
    const int s0 = blockIdx.x * AP_POS, pos = s0 + warp, b = blockIdx.y, share = blockIdx.z, shares = gridDim.z;
    const bool live = pos < S;                            // (of the warp)
    const int h0 = (int)((long long)Hq * share / shares), h1 = (int)((long long)Hq * (share + 1) / shares);
    uint4 x[AP_BATCH], o[AP_BATCH], d[AP_BATCH];
    auto load = [&](int hc, int i) {                      // heads hc + i, hc + i + 4, ..
        const size_t at = (((size_t)b * S + pos) * Hq + hc + i) * 8 + c;
#pragma unroll
        for (int j = 0; j < AP_BATCH; ++j)
            if (live && i + 4 * j < AP_HEADS && hc + i + 4 * j < h1) {
                x[j] = reinterpret_cast<const uint4*>(q)[at + j * 32];
                o[j] = reinterpret_cast<const uint4*>(out)[at + j * 32];
                d[j] = reinterpret_cast<const uint4*>(dout)[at + j * 32];
            } else {
                x[j] = o[j] = d[j] = make_uint4(0, 0, 0, 0);
            }
    };
    load(h0, lane / 8);                                   // (under way while the angles are computed)
    float2 cs[4];
    {
        const float angle = (pos + offset) * rope_inv_freq(lane, AG_D, theta);
        const float2 mine = make_float2(cosf(angle), sinf(angle));
        if (b == 0 && share == 0 && live) table[(size_t)pos * (AG_D / 2) + lane] = mine;
#pragma unroll
        for (int t = 0; t < 4; ++t) cs[t] = make_float2(__shfl_sync(0xffffffffu, mine.x, c * 4 + t), __shfl_sync(0xffffffffu, mine.y, c * 4 + t));
    }
    auto rotate = [&](uint4 x) {
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const float x0 = bf16_lo(w[t]), x1 = bf16_hi(w[t]);
            w[t] = pack_bf16(x0 * cs[t].x - x1 * cs[t].y, x0 * cs[t].y + x1 * cs[t].x);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    for (int hc = h0; hc < h1; hc += AP_HEADS) {
        const int heads = min(AP_HEADS, h1 - hc);
        for (int i = lane / 8; live && i - lane / 8 < heads; i += 4 * AP_BATCH) {
            const size_t at = (((size_t)b * S + pos) * Hq + hc + i) * 8 + c;
#pragma unroll
            for (int j = 0; j < AP_BATCH; ++j) {
                if (i + 4 * j < heads) reinterpret_cast<uint4*>(qrot)[at + j * 32] = rotate(x[j]);
                const uint32_t ow[4] = {o[j].x, o[j].y, o[j].z, o[j].w}, dw[4] = {d[j].x, d[j].y, d[j].z, d[j].w};
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 4; ++t) sum = fmaf(bf16_lo(ow[t]), bf16_lo(dw[t]), fmaf(bf16_hi(ow[t]), bf16_hi(dw[t]), sum));
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                if (c == 0 && i + 4 * j < heads) sums[i + 4 * j][warp] = sum;
            }
            if (i - lane / 8 + 4 * AP_BATCH < heads) load(hc, i + 4 * AP_BATCH);
            else if (hc + AP_HEADS < h1) load(hc + AP_HEADS, lane / 8);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < AP_POS * heads; e += AP_THREADS) {              // positions side by side, as lse and stats have them
            const int s = e % AP_POS, h = e / AP_POS, at = s0 + s;
            float* to = stats + ((size_t)b * Hq + hc + h) * 2 * padded + at;
            to[0] = at < S ? lse[((size_t)b * Hq + hc + h) * S + at] * -1.4426950408889634f : -INFINITY;
            to[padded] = at < S ? -sums[h][s] : 0.f;
        }
        __syncthreads();
    }
    const int g0 = (int)((long long)Hkv * share / shares), g1 = (int)((long long)Hkv * (share + 1) / shares);
    for (int g = g0 + lane / 8; live && g < g1; g += 4) {
        const size_t at = (((size_t)b * S + pos) * Hkv + g) * 8 + c;
        reinterpret_cast<uint4*>(krot)[at] = rotate(reinterpret_cast<const uint4*>(k)[at]);
    }
}

// A block: rows f0 .. f0 + 127 of head hf of sequence b, and `steps` tiles: x_lo .. x_hi - 1 of heads hx, hx + 1, ..  (steps 0: there is none)
struct AttnGradUnit { int keys, b, hf, f0, hx, x_lo, x_hi, part, steps; };

struct AttnGradShared {
    uint64_t full[AG_STAGES], tile_done[AG_STAGES], f_full[AG_F], f_empty[AG_F], s[AG_SLOTS], dp[AG_SLOTS], p[AG_SLOTS], ds[AG_SLOTS], s_free[AG_SLOTS], done[2], acc_free[2], unit[AG_UNITS];
    AttnGradUnit units[AG_UNITS];        // (decoded once: the divisions take 1400 cycles)
    uint32_t tmem_base;
    int abort;
};

__device__ __forceinline__ AttnGradUnit attn_grad_unit(const AttnGradParams& p, int unit) {
    AttnGradUnit w;
    w.keys = unit < p.key_blocks;
    w.part = w.x_lo = 0;
    int heads = 1;
    if (unit >= p.blocks) {
        heads = w.b = w.hf = w.f0 = w.hx = w.x_hi = 0;
    } else if (w.keys) {                                 // the first key tiles, which most queries see, come first
        w.part = unit % p.parts;
        const int bg = unit / p.parts % (p.B * p.Hkv);
        w.b = bg / p.Hkv;
        w.hf = bg % p.Hkv;
        w.f0 = unit / p.parts / (p.B * p.Hkv) * AG_BF;
        w.hx = w.hf * p.rep + p.rep * w.part / p.parts;
        heads = w.hf * p.rep + p.rep * (w.part + 1) / p.parts - w.hx;
        w.x_lo = p.causal ? max(0, w.f0 - p.offset) / AG_BX : 0;
        w.x_hi = (p.S + AG_BX - 1) / AG_BX;
    } else {                                             // the last query tiles, which see most keys, come first
        unit -= p.key_blocks;
        const int bh = unit % (p.B * p.Hq);
        w.b = bh / p.Hq;
        w.hf = bh % p.Hq;
        w.f0 = (p.tiles - 1 - unit / (p.B * p.Hq)) * AG_BF;
        w.hx = w.hf / p.rep;
        w.x_hi = (p.causal ? (int)min((long long)p.S - 1, (long long)w.f0 + AG_BF - 1 + p.offset) : p.S - 1) / AG_BX + 1;
    }
    w.steps = heads * (w.x_hi - w.x_lo);
    return w;
}

// The waits of the softmax warps: mostly over before they begin, so the loop is kept out of the tiles' code (3 x 1371 tokens 147 -> 142 us)
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* abort_flag) { return mbar_wait_warp(bar, parity, abort_flag); }
__device__ __forceinline__ bool wait_quick(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || wait_on(bar, parity, abort_flag);
}

__device__ __forceinline__ uint32_t packed_bf16(uint64_t v) {
    float a, c;
    unpack_f32x2(v, a, c);
    return pack_bf16(a, c);
}

// The block is launched with 80 registers a thread; the warps that issue and store give some to the softmax warps
template <int N> __device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr int AG_REGS = 80, AG_REG_SOFTMAX = 88, AG_REG_ISSUE = 56, AG_REG_STORE = 72;
static_assert(128 * (AG_SOFT / 4 * AG_REG_SOFTMAX + AG_REG_ISSUE + AG_REG_STORE) <= AG_THREADS * AG_REGS, "more registers than the block is launched with");

// A thread's share of a tile, `edge`: the first of its columns (of queries) or the last (of keys) that its row sees: scores -> P (bf16, over
// them) -> with dP, dS (bf16, over that).  `mine`: the thread's columns of the slot, in its warp's lanes; `stat`: of them too.
template <bool KEYS>
__device__ __forceinline__ bool attn_grad_tile(AttnGradShared& sh, int slot, uint32_t parity, uint32_t mine, uint32_t stat, int stage, uint32_t stage_parity,
                                               uint64_t lse2, uint64_t d2, uint64_t scale2, bool masked, int edge, int lane) {
    // four columns' values of one kind; for a row of queries the row's own
    auto of_columns = [&](uint32_t from, int e, uint64_t own, uint64_t& lo, uint64_t& hi) {
        if (KEYS) asm volatile("ld.shared.v2.b64 {%0,%1}, [%2];" : "=l"(lo), "=l"(hi) : "r"(from + e * 4));
        else lo = hi = own;
    };
    if (!wait_quick(smem_u32(&sh.s[slot]), parity, &sh.abort)) return false;
    if (KEYS && !wait_quick(smem_u32(&sh.full[stage]), stage_parity, &sh.abort)) return false;      // (the statistics; they came before)
    tc::fence_after_sync();
    uint64_t pr[AG_COLS / 2];
    {
        uint32_t s[AG_COLS];
        tc::ld32(mine, s);
        tc::wait_ld(s);
        if (!KEYS) {
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.p[slot]));
        }
#pragma unroll
        for (int e = 0; e < AG_COLS; e += 4) {
            uint64_t l[2];
            of_columns(stat, e, lse2, l[0], l[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float a, c;
                unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[e + 2 * j]), __uint_as_float(s[e + 2 * j + 1])), scale2, l[j]), a, c);
                pr[e / 2 + j] = pack_f32x2(ex2(a), ex2(c));
            }
        }
    }
    if (masked) {                                        // (dS has the factor P, so one mask is enough)
#pragma unroll
        for (int e = 0; e < AG_COLS / 2; ++e) {
            float a, c;
            unpack_f32x2(pr[e], a, c);
            if (KEYS ? 2 * e < edge : 2 * e > edge) a = 0.f;
            if (KEYS ? 2 * e + 1 < edge : 2 * e + 1 > edge) c = 0.f;
            pr[e] = pack_f32x2(a, c);
        }
    }
    uint32_t pk[AG_COLS / 2];
    if (KEYS) {
#pragma unroll
        for (int e = 0; e < AG_COLS / 2; ++e) pk[e] = packed_bf16(pr[e]);
        tc::st16(mine, pk);
        tc::wait_st();
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.p[slot]));
    }
    if (!wait_quick(smem_u32(&sh.dp[slot]), parity, &sh.abort)) return false;
    tc::fence_after_sync();
    uint32_t dp[2][16];                                  // (the second half on its way while the first is used)
    tc::ld16(mine + AG_DP, dp[0]);
    tc::wait_ld(dp[0]);
    tc::ld16(mine + AG_DP + 16, dp[1]);
#pragma unroll
    for (int e = 0; e < AG_COLS; e += 4) {
        if (e == 16) tc::wait_ld(dp[1]);
        uint64_t l[2];
        of_columns(stat + AG_STAT_BYTES / 2, e, d2, l[0], l[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
            pk[e / 2 + j] = packed_bf16(mul_f32x2(
                pr[e / 2 + j], add_f32x2(pack_f32x2(__uint_as_float(dp[e / 16][e % 16 + 2 * j]), __uint_as_float(dp[e / 16][e % 16 + 2 * j + 1])), l[j])));
    }
    tc::st16(mine + AG_DP, pk);
    tc::wait_st();
    tc::fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&sh.ds[slot]));
    return true;
}

__global__ void __launch_bounds__(AG_THREADS, 1)
attn_grad_kernel(const __grid_constant__ CUtensorMap q_rows, const __grid_constant__ CUtensorMap do_rows, const __grid_constant__ CUtensorMap k_rows,
                 const __grid_constant__ CUtensorMap v_rows, const AttnGradParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) AttnGradShared sh;
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sF = smem0, sX = smem0 + AG_F * 2 * AG_F_BYTES, sStat = sX + AG_STAGES * AG_STAGE_BYTES, sFStat = sStat + AG_STAGES * AG_STAT_BYTES;
    if (tid == 0) {
        for (int i = 0; i < AG_STAGES; ++i) {
            mbar_init(smem_u32(&sh.full[i]), 1);
            mbar_init(smem_u32(&sh.tile_done[i]), 1);
        }
        for (int i = 0; i < AG_F; ++i) {
            mbar_init(smem_u32(&sh.f_full[i]), 1);
            mbar_init(smem_u32(&sh.f_empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.done[i]), 1);
            mbar_init(smem_u32(&sh.acc_free[i]), 4);      // one arrive per warp that stores gradients
        }
        for (int i = 0; i < AG_SLOTS; ++i) {
            mbar_init(smem_u32(&sh.s[i]), 1);
            mbar_init(smem_u32(&sh.dp[i]), 1);
            mbar_init(smem_u32(&sh.p[i]), 8);
            mbar_init(smem_u32(&sh.ds[i]), 8);
            mbar_init(smem_u32(&sh.s_free[i]), 1);
        }
        for (int i = 0; i < AG_UNITS; ++i) mbar_init(smem_u32(&sh.unit[i]), 1);
        sh.abort = 0;
        fence_mbar_init();
    }
    if (warp == AG_SOFT) {
        tc::tmem_alloc(smem_u32(&sh.tmem_base), AG_TMEM);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sh.tmem_base;
    grid_dependency_wait();

    // number `u` of this CTA's blocks.  The ring is long enough: the loader is at most AG_F blocks ahead of the MMAs, of any two tiles that
    // follow one another each group has had one, and the products of a block wait until the gradients two blocks before are stored.  (Three
    // tiles may belong to three blocks: so many F are kept.)
    auto unit_at = [&](uint32_t u, bool& ok) -> const AttnGradUnit& {
        ok = mbar_wait(smem_u32(&sh.unit[u % AG_UNITS]), u / AG_UNITS & 1u, &sh.abort);
        return sh.units[u % AG_UNITS];
    };

    if (warp >= AG_SOFT && warp < AG_SOFT + 4) registers_down<AG_REG_ISSUE>();
    if (warp == AG_SOFT + 1) {
        // ---------------------------------------------------------- blocks, TMA producer
        if (elect_one()) {
            int unit = blockIdx.x;
            uint32_t n = 0;
            bool ok = true;
            for (uint32_t u = 0; ok; ++u) {
                const AttnGradUnit w = attn_grad_unit(p, unit);
                sh.units[u % AG_UNITS] = w;
                mbar_arrive(smem_u32(&sh.unit[u % AG_UNITS]));
                if (w.steps == 0) break;
                unit = atomicAdd(p.counter, 1);           // (asked for ahead of the loads)
                const CUtensorMap *f1 = w.keys ? &k_rows : &q_rows, *f2 = w.keys ? &v_rows : &do_rows, *x1 = w.keys ? &q_rows : &k_rows, *x2 = w.keys ? &do_rows : &v_rows;
                ok = mbar_wait(smem_u32(&sh.f_empty[u % AG_F]), (u / AG_F & 1u) ^ 1u, &sh.abort);
                if (!ok) break;
                const uint32_t f_full = smem_u32(&sh.f_full[u % AG_F]), f_dst = sF + u % AG_F * 2 * AG_F_BYTES;
                mbar_arrive_expect_tx(f_full, 2 * AG_F_BYTES + (w.keys ? 0 : AG_F_STAT_BYTES));
                if (!w.keys) {                            // the rows' own statistics (asked for by each thread they took 700 cycles: 563 -> 559 us)
                    const float* from = p.stats + ((size_t)w.b * p.Hq + w.hf) * 2 * p.padded + w.f0;
                    const uint32_t to = sFStat + u % AG_F * AG_F_STAT_BYTES;
                    bulk_load(to, from, AG_F_STAT_BYTES / 2, f_full);
                    bulk_load(to + AG_F_STAT_BYTES / 2, from + p.padded, AG_F_STAT_BYTES / 2, f_full);
                }
#pragma unroll
                for (int j = 0; j < AG_BF / AG_BX; ++j) {
                    tma_load_4d(f_dst + j * AG_X_BYTES, f1, 0, w.hf, w.f0 + j * AG_BX, w.b, f_full);
                    tma_load_4d(f_dst + AG_F_BYTES + j * AG_X_BYTES, f2, 0, w.hf, w.f0 + j * AG_BX, w.b, f_full);
                }
                int h = w.hx, x = w.x_lo;
                for (int i = 0; i < w.steps; ++i, ++n) {
                    const uint32_t st = n % AG_STAGES;
                    ok = mbar_wait(smem_u32(&sh.tile_done[st]), (n / AG_STAGES & 1u) ^ 1u, &sh.abort);
                    if (!ok) break;
                    const uint32_t full = smem_u32(&sh.full[st]), dst = sX + st * AG_STAGE_BYTES;
                    mbar_arrive_expect_tx(full, AG_STAGE_BYTES + (w.keys ? AG_STAT_BYTES : 0));
                    tma_load_4d(dst, x1, 0, h, x * AG_BX, w.b, full);
                    tma_load_4d(dst + AG_X_BYTES, x2, 0, h, x * AG_BX, w.b, full);
                    if (w.keys) {
                        const float* from = p.stats + ((size_t)w.b * p.Hq + h) * 2 * p.padded + x * AG_BX;
                        bulk_load(sStat + st * AG_STAT_BYTES, from, AG_STAT_BYTES / 2, full);
                        bulk_load(sStat + st * AG_STAT_BYTES + AG_STAT_BYTES / 2, from + p.padded, AG_STAT_BYTES / 2, full);
                    }
                    if (++x == w.x_hi) { x = w.x_lo; ++h; }
                }
            }
        }
    } else if (warp == AG_SOFT || warp == AG_SOFT + 3) {
        // ------------------------------------------------------------ products of the scores: S (the first of these warps), dP
        constexpr uint32_t I_SCORE = tc::idesc_bf16(AG_BF, AG_BX, 0);
        const uint64_t d0 = tc::smem_desc_sw128(0);
        auto at = [&](uint32_t addr) { return d0 + (uint64_t)(addr >> 4); };
        const uint32_t second = warp == AG_SOFT + 3;
        if (elect_one()) {
            uint32_t n = 0, was_keys = 0, freed = 0;      // per slot: whether its last tile was one of keys; the parity of s_free
            bool ok = true;
            for (uint32_t u = 0; ok; ++u) {
                const AttnGradUnit& w = unit_at(u, ok);
                if (!ok || w.steps == 0) break;
                const int steps = w.steps, keys = w.keys;
                ok = mbar_wait(smem_u32(&sh.f_full[u % AG_F]), u / AG_F & 1u, &sh.abort);
                const uint32_t f = sF + (u % AG_F * 2 + second) * AG_F_BYTES;
                for (int i = 0; ok && i < steps; ++i, ++n) {
                    const uint32_t st = n % AG_STAGES, slot = n % AG_SLOTS, x = sX + st * AG_STAGE_BYTES + second * AG_X_BYTES;
                    const uint32_t col = tmem + slot * 128 + second * AG_DP;
                    if (n >= AG_SLOTS) {                  // what the tile before in this slot had here has been used
                        const uint32_t before = n - AG_SLOTS;
                        if (second) {
                            ok = mbar_wait(smem_u32(&sh.tile_done[before % AG_STAGES]), before / AG_STAGES & 1u, &sh.abort);
                        } else if (was_keys >> slot & 1u) {
                            ok = mbar_wait(smem_u32(&sh.s_free[slot]), freed >> slot & 1u, &sh.abort);
                            freed ^= 1u << slot;
                        } else {
                            ok = mbar_wait(smem_u32(&sh.p[slot]), before / AG_SLOTS & 1u, &sh.abort);
                        }
                    }
                    was_keys = (was_keys & ~(1u << slot)) | (uint32_t)keys << slot;
                    ok = ok && mbar_wait(smem_u32(&sh.full[st]), n / AG_STAGES & 1u, &sh.abort);
                    if (!ok) break;
                    tc::fence_after_sync();
#pragma unroll
                    for (int kk = 0; kk < AG_D / 16; ++kk) tc::mma_ss(col, at(f + kk * 32), at(x + kk * 32), I_SCORE, kk > 0);
                    tc::commit(second ? smem_u32(&sh.dp[slot]) : smem_u32(&sh.s[slot]));
                }
            }
        }
    } else if (warp == AG_SOFT + 2) {
        // ------------------------------------------------------------ products of the gradients
        constexpr uint32_t I_GRAD = tc::idesc_bf16(AG_BF, AG_D, 1);
        const uint64_t d0 = tc::smem_desc_sw128(0);
        auto grad = [&](uint32_t column, uint32_t from, uint32_t sXi, bool first) {           // (P or dS) X: each half of P where its scores began
#pragma unroll
            for (int kk = 0; kk < AG_BX / 16; ++kk)
                tc::mma_ts(tmem + column, tmem + from + kk / 2 * AG_COLS + kk % 2 * 8, d0 + (uint64_t)((sXi + kk * 2048) >> 4), I_GRAD, !first || kk > 0);
        };
        if (elect_one()) {
            uint32_t n = 0, uses0 = 0, uses1 = 0;
            bool ok = true;
            for (uint32_t u = 0; ok; ++u) {
                const AttnGradUnit& w = unit_at(u, ok);
                if (!ok || w.steps == 0) break;
                const int steps = w.steps, keys = w.keys;
                // keys: dV and dK in both gradients; queries: dQ in one of them
                const uint32_t acc2 = keys ? 1u : u & 1u;
                if (keys || acc2 == 0) ok = mbar_wait(smem_u32(&sh.acc_free[0]), (uses0++ & 1u) ^ 1u, &sh.abort);
                if (ok && (keys || acc2 == 1)) ok = mbar_wait(smem_u32(&sh.acc_free[1]), (uses1++ & 1u) ^ 1u, &sh.abort);
                for (int i = 0; ok && i < steps; ++i, ++n) {
                    const uint32_t st = n % AG_STAGES, slot = n % AG_SLOTS, here = sX + st * AG_STAGE_BYTES;
                    if (keys) {
                        ok = mbar_wait(smem_u32(&sh.p[slot]), n / AG_SLOTS & 1u, &sh.abort);
                        if (!ok) break;
                        tc::fence_after_sync();
                        grad(AG_ACC, slot * 128, here + AG_X_BYTES, i == 0);
                        tc::commit(smem_u32(&sh.s_free[slot]));
                    }
                    ok = mbar_wait(smem_u32(&sh.ds[slot]), n / AG_SLOTS & 1u, &sh.abort);     // (behind p)
                    if (!ok) break;
                    tc::fence_after_sync();
                    grad(AG_ACC + acc2 * 64, slot * 128 + AG_DP, here, i == 0);
                    tc::commit(smem_u32(&sh.tile_done[st]));
                    if (i == steps - 1) {
                        tc::commit(smem_u32(&sh.done[u & 1]));
                        tc::commit(smem_u32(&sh.f_empty[u % AG_F]));
                    }
                }
            }
        }
    } else if (warp >= AG_SOFT + 4) {
        // ------------------------------------------------ gradients: thread = row
        registers_down<AG_REG_STORE>();
        const int row = tid % 128;
        const uint32_t lanes = tmem + ((uint32_t)(warp % 4 * 32) << 16);
        for (uint32_t u = 0;; ++u) {
            bool ok = true;
            const AttnGradUnit& w = unit_at(u, ok);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok || w.steps == 0) break;
            const bool keys = w.keys;
            const int f = w.f0 + row, heads = keys ? p.Hkv : p.Hq;
            const size_t at = (((size_t)w.b * p.S + f) * heads + w.hf) * AG_D, all = (size_t)p.B * p.S * p.Hkv * AG_D;
            const float4* table = reinterpret_cast<const float4*>(p.table + (size_t)min(f, p.S - 1) * (AG_D / 2));
            float4 angle[4], next[4];
            auto ask = [&](int c, float4 (&to)[4]) {      // (dV is not turned)
#pragma unroll
                for (int e = 0; e < 4; ++e) to[e] = c >= 4 && c < 8 ? table[c % 4 * 4 + e] : make_float4(1.f, 0.f, 1.f, 0.f);
            };
            ask(keys ? 0 : 4, next);
            if (!mbar_wait_warp(smem_u32(&sh.done[u & 1]), u >> 1 & 1u, &sh.abort)) break;
            tc::fence_after_sync();
#pragma unroll 1
            for (int c = keys ? 0 : 4; c < 8; ++c) {
                const int col = c % 4 * 16;
                const uint32_t acc = keys ? c / 4 : u & 1u;
                const bool dv = c < 4;
                uint32_t r[16];
                tc::ld16(lanes + AG_ACC + acc * 64 + col, r);
#pragma unroll
                for (int e = 0; e < 4; ++e) angle[e] = next[e];
                ask(c + 1, next);
                tc::wait_ld(r);
                if (c % 4 == 3) {                         // the next block may have this gradient's columns (both at the end: 3 x 1371 124 -> 121 us)
                    tc::fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.acc_free[acc]));
                }
                if (f < p.S) {
                    if (keys && p.parts > 1) {
                        float4* to = reinterpret_cast<float4*>(p.partial + (w.part * 2 + (dv ? 0 : 1)) * all + at + col);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            to[e] = make_float4(__uint_as_float(r[4 * e]), __uint_as_float(r[4 * e + 1]), __uint_as_float(r[4 * e + 2]), __uint_as_float(r[4 * e + 3]));
                    } else {
                        const float scale = dv ? 1.f : p.scale;
                        uint32_t o[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float4 t = angle[e / 2];
                            o[e] = turned_back(__uint_as_float(r[2 * e]) * scale, __uint_as_float(r[2 * e + 1]) * scale, e % 2 ? t.z : t.x, e % 2 ? t.w : t.y);
                        }
                        uint4* to = reinterpret_cast<uint4*>((keys ? dv ? p.dv : p.dk : p.dq) + at + col);
                        to[0] = make_uint4(o[0], o[1], o[2], o[3]);
                        to[1] = make_uint4(o[4], o[5], o[6], o[7]);
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------ softmax groups
        registers_up<AG_REG_SOFTMAX>();
        const int group = warp / 8, row = tid % 128, half = warp / 4 % 2 * AG_COLS;
        const uint32_t lanes = tmem + ((uint32_t)(warp % 4 * 32) << 16) + half;
        const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
        uint32_t n0 = 0;                                  // the block's first tile among all of this CTA's
        bool ok = true;
        for (uint32_t u = 0; ok; ++u) {
            const AttnGradUnit& w = unit_at(u, ok);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int steps = w.steps, f0 = w.f0, f = f0 + row, x_lo = w.x_lo, width = w.x_hi - x_lo;
            const int i0 = (int)((group + AG_GROUPS - n0 % AG_GROUPS) % AG_GROUPS);
            // the group's tiles; from which column on (queries) or up to which (keys) its rows see everything
            auto tiles = [&](auto keys, uint64_t lse2, uint64_t d2, int mine_sees, int all_see) {
                constexpr bool KEYS = decltype(keys)::value;
                uint32_t n = n0 + i0;
                int x0 = (x_lo + (i0 < width ? i0 : 0)) * AG_BX;              // (i0 is 0 or 1)
                const int behind = (x_lo + width) * AG_BX;
                for (int i = i0; i < steps; i += AG_GROUPS, n += AG_GROUPS) {
                    const uint32_t st = n % AG_STAGES;
                    const bool masked = KEYS ? x0 < all_see : x0 + AG_BX - 1 > all_see;
                    if (!attn_grad_tile<KEYS>(sh, n % AG_SLOTS, n / AG_SLOTS & 1u, lanes + n % AG_SLOTS * 128, sStat + st * AG_STAT_BYTES + half * 4, st,
                                              n / AG_STAGES & 1u, lse2, d2, scale2, masked, mine_sees - x0 - half, lane))
                        return false;
                    x0 += AG_GROUPS * AG_BX;
                    while (x0 >= behind) x0 -= width * AG_BX;
                }
                return true;
            };
            if (i0 >= steps) {
            } else if (w.keys) {
                ok = tiles(std::true_type{}, 0, 0, p.causal ? f - p.offset : 0, p.causal ? f0 + AG_BF - 1 - p.offset : 0);
            } else {                                      // -lse * log2(e) and -d of the row, twice (rows behind S are padded)
                ok = wait_quick(smem_u32(&sh.f_full[u % AG_F]), u / AG_F & 1u, &sh.abort);
                if (!ok) break;
                float lse, d;
                const uint32_t of = sFStat + u % AG_F * AG_F_STAT_BYTES + row * 4;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(lse) : "r"(of));
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(d) : "r"(of + AG_F_STAT_BYTES / 2));
                const long long sees = p.causal ? p.offset : p.S;
                ok = tiles(std::false_type{}, pack_f32x2(lse, lse), pack_f32x2(d, d), (int)min((long long)p.S - 1, f + sees), (int)min((long long)p.S - 1, f0 + sees));
            }
            if (steps == 0) break;
            n0 += steps;
        }
    }
    // common exit: everybody arrives here (bounded waits), then TMEM is freed
    tc::fence_before_sync();
    __syncthreads();
    if (tid == 0 && sh.abort && p.error_word) atomicExch(p.error_word, BN_ERR_TIMEOUT);
    if (warp == AG_SOFT) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, AG_TMEM);
    }
}

// dV and dK of the blocks that share a group's heads, added in their order; a thread has 8 columns of a row
__global__ void __launch_bounds__(256) attn_grad_sum_kernel(const AttnGradParams p) {
    grid_dependency_wait();
    const long long rows = (long long)p.B * p.S * p.Hkv, e = (long long)blockIdx.x * 256 + threadIdx.x, row = e / 8;
    if (row >= rows) return;
    const int col = (int)(e % 8) * 8, which = blockIdx.y;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const float4* from = reinterpret_cast<const float4*>(p.partial + ((size_t)which * rows + row) * AG_D + col);
    for (int part = 0; part < p.parts; ++part) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float4 t = __ldcg(from + (size_t)part * 2 * rows * (AG_D / 4) + i);
            v[4 * i] += t.x; v[4 * i + 1] += t.y; v[4 * i + 2] += t.z; v[4 * i + 3] += t.w;
        }
    }
    const float2* table = p.table + (size_t)(row / p.Hkv % p.S) * (AG_D / 2) + col / 2;
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = which ? table[i] : make_float2(1.f, 0.f);
        const float scale = which ? p.scale : 1.f;
        o[i] = turned_back(v[2 * i] * scale, v[2 * i + 1] * scale, t.x, t.y);
    }
    reinterpret_cast<uint4*>((which ? p.dk : p.dv) + (size_t)row * AG_D)[col / 8] = make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace bn

using namespace bn;

namespace {

struct AttnGradLayout { size_t counter, table, stats, qrot, krot, partial, total; int parts, padded; };

// How many blocks share the heads of a group: the longest block should not take longer than all blocks' work spread over the GPU, or it
// is what the launch waits for; each further part is written and read again in fp32.
AttnGradLayout attn_grad_layout(int B, int S, int Hq, int Hkv, int causal) {
    AttnGradLayout L;
    const long long tiles = (S + AG_BF - 1) / AG_BF, n = (S + AG_BX - 1) / AG_BX, rep = Hq / Hkv;
    const long long all = 2 * (long long)B * Hq * tiles * n / (causal ? 2 : 1), slots = sm_count();
    int parts = 1;
    while (parts < rep && (rep + parts - 1) / parts * n * slots > all) ++parts;
    L.parts = parts;
    L.padded = (int)(tiles * AG_BF);
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    L.counter = 0;
    L.table = 256;
    L.stats = L.table + up((size_t)S * (AG_D / 2) * sizeof(float2));
    L.qrot = L.stats + up((size_t)B * Hq * 2 * L.padded * sizeof(float));
    L.krot = L.qrot + up((size_t)B * S * Hq * AG_D * 2);
    L.partial = L.krot + up((size_t)B * S * Hkv * AG_D * 2);
    L.total = L.partial + (parts > 1 ? up((size_t)parts * 2 * B * S * Hkv * AG_D * sizeof(float)) : 0);
    return L;
}

}  // namespace

extern "C" size_t bn_attn_prefill_bf16_backward_workspace_bytes(int B, int S, int Hq, int Hkv, int D, int causal) {
    if (B <= 0 || S <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D != AG_D || B > 65535 || S > INT32_MAX - 256) return 0;
    return attn_grad_layout(B, S, Hq, Hkv, causal).total;
}

extern "C" int bn_attn_prefill_bf16_backward(const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse, void* dq,
                                             void* dk, void* dv, int B, int S, int Hq, int Hkv, int D, float scale, float theta, int position_offset,
                                             int causal, void* workspace, size_t workspace_bytes, int* error_word, bn_stream_t stream) {
    const char* what = "bn_attn_prefill_bf16_backward";
    if (B > 0 && S > 0 && (!dout || !q || !k || !v || !out || !lse || !dq || !dk || !dv)) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (B < 0 || S < 0 || Hq <= 0 || Hkv <= 0) return fail(BN_ERR_INVALID_ARG, "%s: bad shape B=%d S=%d Hq=%d Hkv=%d", what, B, S, Hq, Hkv);
    if (Hq % Hkv) return fail(BN_ERR_INVALID_ARG, "%s: Hq=%d not a multiple of Hkv=%d", what, Hq, Hkv);
    if (D != AG_D) return fail(BN_ERR_UNSUPPORTED, "%s: head_dim=%d (64 supported)", what, D);
    if (B > 65535 || S > INT32_MAX - 256 || position_offset > INT32_MAX - S - 256) return fail(BN_ERR_UNSUPPORTED, "%s: B=%d S=%d offset=%d too large", what, B, S, position_offset);
    if (position_offset < 0) return fail(BN_ERR_INVALID_ARG, "%s: position_offset=%d < 0", what, position_offset);
    for (const void* t : {dout, q, k, v, out, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
        if (reinterpret_cast<uintptr_t>(t) & 15) return fail(BN_ERR_INVALID_ARG, "%s: tensors must be 16-byte aligned", what);
    if (int rc = require_sm100()) return rc;
    if (B == 0 || S == 0) return BN_OK;
    const AttnGradLayout L = attn_grad_layout(B, S, Hq, Hkv, causal);
    if (!workspace || workspace_bytes < L.total) return fail(BN_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", what, workspace_bytes, L.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(BN_ERR_INVALID_ARG, "%s: workspace must be 256-byte aligned", what);
    const long long tiles = (S + AG_BF - 1) / AG_BF, key_blocks = tiles * B * Hkv * L.parts, blocks = key_blocks + tiles * B * Hq;
    const long long sum_blocks = ((long long)B * S * Hkv * 8 + 255) / 256;
    if (blocks > INT32_MAX / 2 || sum_blocks > INT32_MAX)
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
    p.counter = reinterpret_cast<int*>(ws + L.counter);
    p.blocks = (int)blocks;
    const unsigned grid = (unsigned)(blocks < sm_count() ? blocks : sm_count());
    p.B = B; p.S = S; p.padded = L.padded; p.Hq = Hq; p.Hkv = Hkv; p.rep = Hq / Hkv; p.tiles = (int)tiles; p.parts = L.parts;
    p.key_blocks = (int)key_blocks;
    p.offset = position_offset;
    p.causal = causal != 0;
    p.scale = scale;
    p.scale_log2 = scale * 1.4426950408889634f;
    __nv_bfloat16 *qrot = reinterpret_cast<__nv_bfloat16*>(ws + L.qrot), *krot = reinterpret_cast<__nv_bfloat16*>(ws + L.krot);

    CUtensorMap maps[4];                                                       // one box: 64 rows of a head
    {
        const void* base[4] = {qrot, dout, krot, v};
        for (int i = 0; i < 4; ++i) {
            const uint64_t heads = i < 2 ? Hq : Hkv;
            const uint64_t dims[4] = {AG_D, heads, (uint64_t)S, (uint64_t)B}, strides[3] = {AG_D * 2, heads * AG_D * 2, (uint64_t)S * heads * AG_D * 2};
            const uint32_t box[4] = {AG_D, 1, AG_BX, 1};
            if (int rc = make_tensor_map(&maps[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base[i], dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
        }
    }
    // enough blocks for the GPU, by positions and, where those are few, by heads too
    const unsigned pos_blocks = (unsigned)(L.padded / AP_POS);
    long long shares = 4 * sm_count() / ((long long)pos_blocks * B);
    shares = shares < 1 ? 1 : shares > Hq ? Hq : shares;
    launch_dependent(attn_grad_prepare_kernel, dim3(pos_blocks, (unsigned)B, (unsigned)shares), AP_THREADS, 0, st, static_cast<const __nv_bfloat16*>(q),
                     static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(dout), lse, qrot, krot,
                     reinterpret_cast<float2*>(ws + L.table), reinterpret_cast<float*>(ws + L.stats), p.counter, (int)grid, S, L.padded, Hq, Hkv, theta, position_offset);
    if (int rc = launch_status(what)) return rc;
    static thread_local int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        cudaFuncAttributes attr;                                               // (with fewer registers at launch the softmax warps would wait for theirs)
        if (cudaFuncGetAttributes(&attr, attn_grad_kernel) != cudaSuccess || attr.numRegs < AG_REGS)
            return fail(BN_ERR_CUDA, "%s: the kernel is launched with fewer registers than it shares out", what);
        if (int rc = allow_smem(attn_grad_kernel, AG_SMEM_BYTES, what, AG_SMEM_BYTES)) return rc;
        configured_dev = dev;
    }
    launch_dependent(attn_grad_kernel, dim3(grid), AG_THREADS, AG_SMEM_BYTES, st, maps[0], maps[1], maps[2], maps[3], p);
    if (int rc = launch_status(what)) return rc;
    if (L.parts > 1) {
        launch_dependent(attn_grad_sum_kernel, dim3((unsigned)sum_blocks, 2), 256, 0, st, p);
        return launch_status(what);
    }
    return BN_OK;
}
