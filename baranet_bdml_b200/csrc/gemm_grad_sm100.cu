// The products of a backward pass, bf16 with fp32 accumulation in tensor memory, for sm_100a, and the two operators of a training step
// that are made of them: softmax cross entropy over a large vocabulary (op_cross_entropy, src/ops/op_cross_entropy.cuh:5-45, and the
// lm_head product before it) and the gradients of the gated feed-forward block (MLP.__call__, mygrad/llama/llama_layers.py:194-235;
// op_silu_backward, src/ops/op_silu.cuh).
//
// One kernel, three operand orders, several products in a launch.  y = x W^T reads both operands along K (NT).  Its gradients do not: dx =
// dy W reads W across its rows (NN), dW = dy^T x reads both across (TN).  tcgen05 takes either order from shared memory (MN-major operands:
// tiles of 64 k rows of 64 contiguous m or n), so nothing is transposed in memory.
// Persistent kernel: four epilogue warps (GLU: eight, thread = row and half of the columns, for its arithmetic: 16384 x 5632 x 2048 613 us,
// 588 with eight), one that issues the MMAs, one that loads by TMA (an elected thread: with lane == 0, for which the compiler keeps a tensor
// map's address and coordinates in ordinary registers, four loads a step took longer than its MMAs; 1490 -> 1376 us for the gradients of
// that block).  Output tile 128 x 256, or (PAIR) 256 x 256 shared by a cluster of two CTAs (tcgen05.mma.cta_group::2); fp32 accumulators
// double buffered in tensor memory, so that the epilogue of a tile runs under the products of the next.  Tiles may have 128 columns, where
// there are few (tile_columns).  They go in bands of 16 tile rows, n outside, so that what runs at one time shares both operands in L2.
//
// Results leave through shared memory: a warp writes 32 rows of 128 bytes and one thread has TMA store them (a thread that stores its own
// row takes 32 places in memory for every 16 bytes: 32000 x 2048 of K = 200 71 -> 46 us, and 39 since the elected thread loads, of which 32
// without the stores; eight epilogue warps instead of four made no difference there, and 2 - 5 % more for long K).
//
// Gradients that wait for the same operand are one launch: the tiles of up to three products (NN and TN) follow one another, those of the
// longest K first, so that one's last wave is filled by the next.
//
// Epilogues
//   PRODUCTS  the result as bf16, or, PARTIAL, fp32 sums of a range of K, kept or added to what an earlier launch left: few tiles share K,
//             pieces of the vocabulary follow one another.  An element gets one sum from a launch, and grad_sum_kernel adds the ranges in
//             order: the same bits in every run
//   LOSS      logits: of every row's columns in a tile the maximum and the sum of exponentials, and the target's logit: the logits stay in
//             tensor memory
//   DLOGITS   logits again -> g (exp(z - lse) - [v = target]) over the first row's g (its significand), as bf16
//   GLU       columns [0,128) gate, [128,256) up of the same indices, and dh, fp32 -> dgate, dup and the product that the forward pass had
// Every mbarrier wait is bounded; on expiry the kernel raises the caller's error word, frees TMEM and returns.
#include <type_traits>

#include "common.cuh"
#include "hybrid.cuh"
#include "ptx.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace bn {

using namespace ptx;

constexpr int GG_BM = 128, GG_BN = 256, GG_BK = 64, GG_BAND = 16;
constexpr int GG_A_BYTES = GG_BM * GG_BK * 2;
constexpr int GG_OUT_BYTES = 32 * 128;                                     // what a warp stores at a time (GLU: half of that, of three results)
// Shared memory: as many stages of operands as fit beside the epilogue warps' buffers (GLU: one for each of three results, else two in turn)
constexpr int GG_MAX_STAGES = 6;
struct GradRing { int stage_bytes, stages; };
constexpr int grad_out_bytes(bool glu) { return glu ? 8 * 3 * GG_OUT_BYTES / 2 : 4 * 2 * GG_OUT_BYTES; }
constexpr GradRing grad_ring(bool pair, bool glu, int bn) {
    const int stage = GG_A_BYTES + (pair ? bn / 2 : bn) * GG_BK * 2, room = 225 * 1024 - grad_out_bytes(glu);
    return {stage, room / stage < GG_MAX_STAGES ? room / stage : GG_MAX_STAGES};
}

constexpr int GE_PRODUCTS = 0, GE_LOSS = 1, GE_DLOGITS = 2, GE_GLU = 3;
// what the second pair of operands is: none, the second half of K (NN), further rows of the result (TN), the upper half of every tile's
// columns (NT, GLU)
constexpr int SECOND_NONE = 0, SECOND_K = 1, SECOND_M = 2;

struct GradJob {
    int M, N, K;                       // of one pair of operands
    int second;
    int a_mn;                          // PRODUCTS: A is (K, M)
    int partial, add;                  // PRODUCTS: fp32 sums of ranges of K, added to what is there
    int splits, k_per_split;
    const float* factor;               // PRODUCTS: what common_factor makes of it is a factor of the result
    int tiles_m0, tiles_m, tiles_n, tiles;      // of one pair of operands' rows, all, columns, rows x columns
    int first;                         // number of the job's first item: a tile and a range of K
};
constexpr int GG_JOBS = 3;
struct GradParams {
    GradJob job[GG_JOBS];              // those behind the last begin at `items`
    int items;
    int bn;                            // columns of a tile (GLU: of gate and up together)
    GradRing ring;
    int* error_word;
    const int32_t* targets;            // LOSS, DLOGITS: (M), minus first_column is the column here
    int first_column, vocab;
    float2* stats;                     // LOSS: [tile][M] maximum, sum of exponentials of the distances to it
    float* picked;                     // LOSS: (M) the target's logit
    const float *lse, *grad;           // DLOGITS: (M)
    const float* dh;                   // GLU: [dh_parts][M][N], to be added up
    int dh_parts;
};

// Tensor maps of a job's operands and of what is stored: PRODUCTS c0 and (of the second rows) c1, bf16, or c0, fp32 (N, M, range); DLOGITS
// c0; GLU c0 = h, c1 = dgate, c2 = dup
struct GradMaps { CUtensorMap a0, a1, b0, b1, c0, c1, c2; };
struct AllMaps { GradMaps job[GG_JOBS]; };

// What the logits' gradients are divided by before they are rounded, and their products multiplied by: the first row's gradient without its
// power of two, 1 <= |factor| < 2, so that a mean's 1 / rows, which all rows have, is not rounded to bf16 in every one of them alike
// (errors of 1.9 - 2.2e-3 instead of 1.66e-3, which the last rounding alone makes), and no other row's gradient leaves the range that it
// has itself.  0, subnormal numbers, infinities and NaN: 1.
__device__ __forceinline__ float common_factor(const float* grad) {
    const uint32_t bits = grad ? __float_as_uint(*grad) : 0u, exponent = bits & 0x7f800000u;
    return exponent == 0 || exponent == 0x7f800000u ? 1.f : __uint_as_float((bits & 0x807fffffu) | 0x3f800000u);
}

__device__ __forceinline__ float log2e() { return 1.4426950408889634f; }

// a and da/dz of a gated unit's activation.  silu: z s with s = 1 / (1 + e^-z), slope s + z s (1 - s).  gelu_tanh(z) = z s(2u), u =
// sqrt(2/pi) (z + 0.044715 z^3): slope s + z s (1 - s) 2u'.  The results are rounded to bf16, so the fast exponential suffices.
template <int ACT> __device__ __forceinline__ void act_and_slope(float z, float& a, float& slope) {
    const float t = ACT == BN_ACT_GELU_TANH ? 1.5957691216057308f * fmaf(0.044715f * z * z, z, z) : z;
    const float dt = ACT == BN_ACT_GELU_TANH ? fmaf(0.2140644488f * z, z, 1.5957691216057308f) : 1.f;
    const float s = sigmoid_fast(t);
    a = z * s;
    slope = fmaf(a * (1.f - s), dt, s);
}

template <int EPI, int ACT, bool PAIR>
__global__ void __launch_bounds__(EPI == GE_GLU ? 320 : 192, 1)
gemm_grad_kernel(const __grid_constant__ AllMaps all, const __grid_constant__ GradParams p) {
    constexpr bool PRODUCTS = EPI == GE_PRODUCTS;
    constexpr int TILE_M = PAIR ? 2 * GG_BM : GG_BM, EW = EPI == GE_GLU ? 8 : 4;      // epilogue warps
    const int n_stages = p.ring.stages;
    const int n_here = PAIR ? p.bn / 2 : p.bn;                             // columns of the tile that this CTA loads
    const int columns = EPI == GE_GLU ? p.bn / 2 : p.bn;                   // columns of the result that a tile covers
    constexpr uint32_t TMEM_COLS = 2 * GG_BN;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[GG_MAX_STAGES], bar_empty[GG_MAX_STAGES], bar_acc_full[2], bar_acc_empty[2];
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort;

    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t rank = PAIR ? cluster_rank() : 0;
    const int first = PAIR ? blockIdx.x / 2 : blockIdx.x, stride = PAIR ? gridDim.x / 2 : gridDim.x;
    struct Item { int m, n, part, split, ks0, ks1; };                      // tile row and column; which operands; K steps
    auto item = [&](const GradJob& q, int t) {
        Item w;
        t -= q.first;
        w.split = PRODUCTS ? t / q.tiles : 0;
        t -= w.split * q.tiles;
        const int band = t / (GG_BAND * q.tiles_n), in_band = t - band * GG_BAND * q.tiles_n;
        const int height = min(GG_BAND, q.tiles_m - band * GG_BAND);
        w.n = in_band / height;
        w.m = band * GG_BAND + in_band - w.n * height;
        w.part = w.m >= q.tiles_m0;
        if (w.part) w.m -= q.tiles_m0;
        const int steps = (q.K + GG_BK - 1) / GG_BK * (q.second == SECOND_K ? 2 : 1);
        w.ks0 = PRODUCTS ? w.split * q.k_per_split : 0;
        w.ks1 = PRODUCTS ? min(steps, w.ks0 + q.k_per_split) : steps;
        return w;
    };
    if (tid == 0) {
        for (int s = 0; s < n_stages; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&bar_acc_full[i]), 1);
            mbar_init(smem_u32(&bar_acc_empty[i]), PAIR ? 2 * EW : EW);          // one arrive per epilogue warp
        }
        s_abort = 0;
        fence_mbar_init();
    }
    if (warp == EW) {
        if (PAIR) {
            tc::pair_tmem_alloc(smem_u32(&s_tmem_base), TMEM_COLS);
            tc::pair_tmem_relinquish();
        } else {
            tc::tmem_alloc(smem_u32(&s_tmem_base), TMEM_COLS);
            tc::tmem_relinquish();
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync();                                              // the other CTA's barriers are there
    tc::fence_after_sync();
    const uint32_t tmem = s_tmem_base;
    grid_dependency_wait();

    // a CTA's items, job by job; the body is unrolled by jobs, so that what it reads of one is uniform (MMAs take their operands from uniform
    // registers: with a job's number in a register 16384 x 5632 x 2048 took 323 us instead of 271), and once for each order of A
    auto each_item = [&](auto&& body) {
        int t = first;
#pragma unroll
        for (int j = 0; j < (PRODUCTS ? GG_JOBS : 1); ++j) {
            const int end = PRODUCTS && j + 1 < GG_JOBS ? p.job[j + 1].first : p.items;
            if (PRODUCTS && p.job[j].a_mn) {
                for (; t < end; t += stride)
                    if (!body(std::true_type{}, j, t)) return;
            } else {
                for (; t < end; t += stride)
                    if (!body(std::false_type{}, j, t)) return;
            }
        }
    };

    if (warp == EW + 1) {
        // ---------------------------------------------------------- TMA producer
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            each_item([&](auto mn, int job, int t) {
                constexpr bool a_mn = decltype(mn)::value;
                const GradJob& q = p.job[job];
                const GradMaps& maps = all.job[job];
                const Item w = item(q, t);
                const bool second_k = q.second == SECOND_K;
                const int steps0 = (q.K + GG_BK - 1) / GG_BK;
                const int m0 = w.m * TILE_M + rank * GG_BM, n0 = w.n * columns + (EPI == GE_GLU ? 0 : rank * n_here);
                const uint32_t bytes = (PAIR ? 2 : 1) * (GG_A_BYTES + n_here * GG_BK * 2);
                for (int ks = w.ks0; ks < w.ks1; ++ks) {
                    if (!mbar_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, &s_abort)) return false;
                    const bool half2 = second_k && ks >= steps0;
                    const int k0 = (half2 ? ks - steps0 : ks) * GG_BK;
                    const CUtensorMap* ma = half2 || w.part ? &maps.a1 : &maps.a0;
                    const CUtensorMap* mb = half2 ? &maps.b1 : &maps.b0;
                    const uint32_t sA = smem0 + stage * p.ring.stage_bytes, sB = sA + GG_A_BYTES;
                    const uint32_t full = PAIR ? in_rank(smem_u32(&bar_full[stage]), 0) : smem_u32(&bar_full[stage]);
                    if (rank == 0) mbar_arrive_expect_tx(smem_u32(&bar_full[stage]), bytes);
                    auto load = [&](uint32_t dst, const CUtensorMap* m, int x, int y) {
                        if (PAIR) tma_load_2d_pair(dst, m, x, y, full);
                        else tma_load_2d(dst, m, x, y, full);
                    };
                    if (a_mn) {
#pragma unroll
                        for (int j = 0; j < GG_BM / 64; ++j) load(sA + j * 8192, ma, m0 + j * 64, k0);
                    } else {
                        load(sA, ma, k0, m0);
                    }
                    if (EPI == GE_GLU) {                                   // 128 gate rows, 128 up rows
                        if (PAIR) {
                            load(sB, rank ? &maps.b1 : &maps.b0, k0, n0);
                        } else {
                            load(sB, &maps.b0, k0, n0);
                            load(sB + p.bn / 2 * GG_BK * 2, &maps.b1, k0, n0);
                        }
                    } else if (PRODUCTS) {
                        for (int j = 0; j < n_here / 64; ++j) load(sB + j * 8192, mb, n0 + j * 64, k0);
                    } else {
                        load(sB, mb, k0, n0);
                    }
                    if (++stage == n_stages) stage = 0, phase ^= 1u;
                }
                return true;
            });
        }
    } else if (warp == EW) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t idesc = tc::idesc_bf16(TILE_M, p.bn, PRODUCTS ? 1 : 0);
        const uint64_t dK = tc::smem_desc_sw128(0);                        // descriptor = this + (address >> 4)
        const uint64_t dMN = (dK & ~((uint64_t)0x3fff << 16)) | (uint64_t)(8192 >> 4) << 16;      // the next 64 m or n lie 8 KB on
        constexpr uint32_t B_STEP = PRODUCTS ? 128 : 2;                                           // 16 k further, in 16 bytes
        uint32_t local = 0, phase = 0;
        int stage = 0;
        if (rank == 0) each_item([&](auto mn, int job, int t) {
            constexpr bool a_mn = decltype(mn)::value;
            const uint32_t acc = local & 1u;
            if (!mbar_wait_warp(smem_u32(&bar_acc_empty[acc]), ((local >> 1) & 1u) ^ 1u, &s_abort)) return false;       // drained two tiles ago
            ++local;
            tc::fence_after_sync();
            const GradJob& q = p.job[job];
            const Item w = item(q, t);
            const uint32_t i_desc = idesc | (a_mn ? 1u << 15 : 0u);
            constexpr uint32_t a_step = a_mn ? 128 : 2;
            for (int ks = w.ks0; ks < w.ks1; ++ks) {
                if (!mbar_wait_warp(smem_u32(&bar_full[stage]), phase, &s_abort)) return false;
                if (elect_one()) {
                    tc::fence_after_sync();
                    const uint32_t sA = smem0 + stage * p.ring.stage_bytes, sB = sA + GG_A_BYTES;
#pragma unroll
                    for (int kk = 0; kk < GG_BK / 16; ++kk) {
                        const uint64_t da = (a_mn ? dMN : dK) + (uint64_t)((sA >> 4) + kk * a_step);
                        const uint64_t db = (PRODUCTS ? dMN : dK) + (uint64_t)((sB >> 4) + kk * B_STEP);
                        if (PAIR) tc::pair_mma_ss(tmem + acc * GG_BN, da, db, i_desc, (ks > w.ks0) || (kk > 0));
                        else tc::mma_ss(tmem + acc * GG_BN, da, db, i_desc, (ks > w.ks0) || (kk > 0));
                    }
                    const uint32_t empty = smem_u32(&bar_empty[stage]), full = smem_u32(&bar_acc_full[acc]);
                    if (PAIR) {
                        tc::pair_commit(empty);
                        if (ks == w.ks1 - 1) tc::pair_commit(full);
                    } else {
                        tc::commit(empty);
                        if (ks == w.ks1 - 1) tc::commit(full);
                    }
                }
                __syncwarp();
                if (++stage == n_stages) stage = 0, phase ^= 1u;
            }
            return true;
        });
    } else {
        // ------------------------------------------------------ epilogue: thread = row of the tile = TMEM lane
        const int half = EW == 8 ? warp / 4 : 0, row = tid % GG_BM;
        const uint32_t lane_base = ((uint32_t)(warp % 4 * 32)) << 16;
        const uint32_t out0 = smem0 + n_stages * p.ring.stage_bytes + warp * (grad_out_bytes(EPI == GE_GLU) / EW);
        int out_turn = 0;
        // the warp's next buffer, when what was sent from it before has been read: all but the newest group have been, and the newest is the
        // other buffer's, so every buffer that is taken has to be sent
        auto out_buffer = [&] {
            if (lane == 0) bulk_wait_group_read<1>();
            __syncwarp();
            out_turn ^= 1;
            return out0 + out_turn * GG_OUT_BYTES;
        };
        auto put_at = [&](uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
        };
        auto put16 = [&](uint32_t buf, int chunk, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {      // 16 bytes of the thread's row of 128, swizzled
            put_at(buf + lane * 128 + ((chunk ^ (lane & 7)) << 4), a, b, c, d);
        };
        auto put_row = [&](uint32_t buf, int hf, const uint32_t (&r)[32]) {
#pragma unroll
            for (int v = 0; v < 4; ++v)
                put16(buf, hf * 4 + v, pack_bf16(__uint_as_float(r[v * 8]), __uint_as_float(r[v * 8 + 1])),
                      pack_bf16(__uint_as_float(r[v * 8 + 2]), __uint_as_float(r[v * 8 + 3])), pack_bf16(__uint_as_float(r[v * 8 + 4]), __uint_as_float(r[v * 8 + 5])),
                      pack_bf16(__uint_as_float(r[v * 8 + 6]), __uint_as_float(r[v * 8 + 7])));
        };
        auto send = [&](auto&& stores) {                                   // one thread, when the warp has written
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                stores();
                bulk_commit_group();
            }
        };
        uint32_t local = 0;
        bool ok = true;
        for (int t = first; ok && t < p.items; t += stride, ++local) {
            const uint32_t acc = local & 1u;
            const int job = !PRODUCTS ? 0 : t >= p.job[2].first ? 2 : t >= p.job[1].first ? 1 : 0;
            const GradJob& q = p.job[job];
            const GradMaps& maps = all.job[job];
            const Item w = item(q, t);
            const int M = q.M, N = q.N;
            const int gm = w.m * TILE_M + rank * GG_BM + row, n0 = w.n * columns + half * (columns / 2);
            const int y = w.m * TILE_M + rank * GG_BM + warp % 4 * 32;          // the warp's first row
            const bool live = gm < M;
            // what a row needs beside its products, fetched while those run
            int target = -1;
            float lse2 = 0.f, grad = 0.f;
            if ((EPI == GE_LOSS || EPI == GE_DLOGITS) && live) {
                const int v = p.targets[gm];
                target = v < 0 ? -1 : v - p.first_column;
                if (EPI == GE_DLOGITS && v >= 0 && v < p.vocab) {
                    lse2 = p.lse[gm] * log2e();
                    grad = p.grad[gm] / common_factor(p.grad);
                } else if (EPI == GE_DLOGITS) {
                    target = INT32_MIN;                                    // no loss, no gradient
                }
            }
            float d[EPI == GE_GLU ? 32 : 1];                               // 32 columns of dh
            auto load_dh = [&](int col0) {
                if (EPI != GE_GLU || col0 >= N) return;
                const float4* from = reinterpret_cast<const float4*>(p.dh + (size_t)(live ? gm : 0) * N + col0);
                const size_t part = (size_t)M * N / 4;
#pragma unroll
                for (int v = 0; v < 8; ++v) {                              // (columns are a multiple of 8)
                    const float4 f = col0 + v * 4 < N ? __ldcg(from + v) : make_float4(0.f, 0.f, 0.f, 0.f);
                    d[v * 4] = f.x; d[v * 4 + 1] = f.y; d[v * 4 + 2] = f.z; d[v * 4 + 3] = f.w;
                }
#pragma unroll 2
                for (int k = 1; k < p.dh_parts; ++k) {                     // (eight loads under way, or sixteen)
#pragma unroll
                    for (int v = 0; v < 8; ++v) {
                        const float4 f = col0 + v * 4 < N ? __ldcg(from + k * part + v) : make_float4(0.f, 0.f, 0.f, 0.f);
                        d[v * 4] += f.x; d[v * 4 + 1] += f.y; d[v * 4 + 2] += f.z; d[v * 4 + 3] += f.w;
                    }
                }
            };
            load_dh(n0);
            ok = mbar_wait_warp(smem_u32(&bar_acc_full[acc]), (local >> 1) & 1u, &s_abort);
            if (!ok) break;
            tc::fence_after_sync();
            const uint32_t tacc = tmem + lane_base + acc * GG_BN + half * (columns / 2);
            if (y >= M) {
                // no row of this warp is one of the result's: nothing to take from tensor memory, nothing to send
            } else if (EPI == GE_DLOGITS || (PRODUCTS && !q.partial)) {
                const float factor = PRODUCTS ? common_factor(q.factor) : 1.f;
#pragma unroll 1
                for (int c = 0; c < p.bn / 64; ++c) {
                    if (n0 + c * 64 >= N) break;                         // (uniform)
                    const uint32_t buf = out_buffer();
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        uint32_t r[32];
                        tc::ld32(tacc + c * 64 + hf * 32, r);
                        tc::wait_ld(r);
                        if (PRODUCTS) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * factor);
                        }
                        if (EPI == GE_DLOGITS) {
                            const int at = target - (n0 + c * 64 + hf * 32);
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float dz = ex2(fmaf(__uint_as_float(r[e]), log2e(), -lse2)) - (e == at ? 1.f : 0.f);
                                r[e] = __float_as_uint(target == INT32_MIN ? 0.f : grad * dz);
                            }
                        }
                        put_row(buf, hf, r);
                    }
                    send([&] { tma_store_2d(w.part ? &maps.c1 : &maps.c0, buf, n0 + c * 64, y); });
                }
            } else if (PRODUCTS) {
                const bool add = q.add;
#pragma unroll 1
                for (int c = 0; c < p.bn / 32; ++c) {
                    if (n0 + c * 32 >= N) break;
                    const uint32_t buf = out_buffer();
                    uint32_t r[32];
                    tc::ld32(tacc + c * 32, r);
                    tc::wait_ld(r);
#pragma unroll
                    for (int v = 0; v < 8; ++v) put16(buf, v, r[v * 4], r[v * 4 + 1], r[v * 4 + 2], r[v * 4 + 3]);
                    send([&] {
                        if (add) tma_add_3d(&maps.c0, buf, n0 + c * 32, y, w.split);
                        else tma_store_3d(&maps.c0, buf, n0 + c * 32, y, w.split);
                    });
                }
            } else if (EPI == GE_LOSS) {
                // one pass: the sum is kept relative to the largest logit so far
                float top = -INFINITY, sum = 0.f;
#pragma unroll 1
                for (int c = 0; c < p.bn / 32; ++c) {
                    uint32_t r[32];
                    tc::ld32(tacc + c * 32, r);
                    tc::wait_ld(r);
                    const int col = n0 + c * 32;
                    if (col >= N) continue;                              // (uniform)
                    if (col + 32 > N) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (col + e >= N) r[e] = __float_as_uint(-INFINITY);
                    }
                    float m = top;
#pragma unroll
                    for (int e = 0; e < 32; ++e) m = fmaxf(m, __uint_as_float(r[e]));
                    const float shift = m == -INFINITY ? 0.f : -m * log2e();
                    sum *= ex2(fmaf(top, log2e(), shift));
                    float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < 32; ++e) s4[e & 3] += ex2(fmaf(__uint_as_float(r[e]), log2e(), shift));
                    sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
                    top = m;
                    const int at = target - col;
                    if (__any_sync(0xffffffffu, at >= 0 && at < 32)) {
                        float z = 0.f;
#pragma unroll
                        for (int e = 0; e < 32; ++e) z = e == at ? __uint_as_float(r[e]) : z;
                        if (at >= 0 && at < 32 && target < N) p.picked[gm] = z;
                    }
                }
                if (live) p.stats[(size_t)w.n * M + gm] = make_float2(top, sum);
            } else {
                const uint32_t h_buf = out0, g_buf = out0 + GG_OUT_BYTES / 2, u_buf = out0 + GG_OUT_BYTES;
#pragma unroll 1
                for (int c = 0; c < p.bn / 128; ++c) {                     // 32 columns of the half
                    const int col0 = n0 + c * 32;
                    if (col0 >= N) break;
                    uint32_t g[32], u[32];
                    tc::ld32(tacc + c * 32, g);
                    tc::ld32(tacc + p.bn / 2 + c * 32, u);
                    tc::wait_ld(g);
                    tc::wait_ld(u);
                    if (lane == 0) bulk_wait_group_read<0>();              // the buffers have been read
                    __syncwarp();
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        uint32_t h4[4], g4[4], u4[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float h[2], dgate[2], dup[2];
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                const int i = v * 8 + 2 * e + s;
                                const float uv = __uint_as_float(u[i]);
                                float a, slope;
                                act_and_slope<ACT>(__uint_as_float(g[i]), a, slope);
                                h[s] = a * uv;
                                dgate[s] = d[i] * uv * slope;
                                dup[s] = d[i] * a;
                            }
                            h4[e] = pack_bf16(h[0], h[1]);
                            g4[e] = pack_bf16(dgate[0], dgate[1]);
                            u4[e] = pack_bf16(dup[0], dup[1]);
                        }
                        const uint32_t at = lane * 64 + ((v ^ (lane >> 1 & 3)) << 4);       // (64-byte swizzle)
                        put_at(h_buf + at, h4[0], h4[1], h4[2], h4[3]);
                        put_at(g_buf + at, g4[0], g4[1], g4[2], g4[3]);
                        put_at(u_buf + at, u4[0], u4[1], u4[2], u4[3]);
                    }
                    if (c + 1 < p.bn / 128) load_dh(col0 + 32);            // (the next tile's: before its products are waited for)
                    send([&] {
                        tma_store_2d(&maps.c0, h_buf, col0, y);
                        tma_store_2d(&maps.c1, g_buf, col0, y);
                        tma_store_2d(&maps.c2, u_buf, col0, y);
                    });
                }
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) mbar_arrive_cluster(in_rank(smem_u32(&bar_acc_empty[acc]), 0));
                else mbar_arrive(smem_u32(&bar_acc_empty[acc]));
            }
        }
        if (EPI != GE_LOSS && lane == 0) bulk_wait_group0();
    }

    // common exit: everybody arrives here (all waits are bounded), then TMEM is freed
    tc::fence_before_sync();
    __syncthreads();
    if (PAIR) cluster_sync();                                              // nothing more is on its way from one CTA to the other
    if (tid == 0 && s_abort && p.error_word) atomicExch(p.error_word, BN_ERR_TIMEOUT);
    if (warp == EW) {
        tc::fence_after_sync();
        if (PAIR) tc::pair_tmem_dealloc(tmem, TMEM_COLS);
        else tc::tmem_dealloc(tmem, TMEM_COLS);
    }
}

// the ranges' sums, added in their order, rounded once
__global__ void __launch_bounds__(128) grad_sum_kernel(const float* partial, __nv_bfloat16* c, long long groups, int splits, const float* factor) {
    grid_dependency_wait();
    const long long i = (long long)blockIdx.x * 128 + threadIdx.x;         // of 4 elements
    if (i >= groups) return;
    const float4* p4 = reinterpret_cast<const float4*>(partial);
    float4 s = __ldcg(p4 + i);
#pragma unroll 8
    for (int k = 1; k < splits; ++k) {
        const float4 v = __ldcg(p4 + (long long)k * groups + i);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float f = common_factor(factor);
    reinterpret_cast<uint2*>(c)[i] = make_uint2(pack_bf16(s.x * f, s.y * f), pack_bf16(s.z * f, s.w * f));
}

// the tiles' maxima and sums of 32 rows: 32 warps take the tiles in turn, the first warp joins theirs
constexpr int GG_JOIN = 32;
__global__ void __launch_bounds__(32 * GG_JOIN)
loss_join_kernel(const float2* stats, const float* picked, const int32_t* targets, float* loss, float* lse, int* id_error, int rows, int tiles, int vocab) {
    __shared__ float2 part[GG_JOIN][32];
    grid_dependency_wait();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, row = blockIdx.x * 32 + lane;
    float top = -INFINITY, sum = 0.f;
    auto join = [&](float2 v) {
        const float m = fmaxf(top, v.x), ref = m == -INFINITY ? 0.f : m;
        sum = sum * ex2((top - ref) * log2e()) + v.y * ex2((v.x - ref) * log2e());
        top = m;
    };
    if (row < rows) {
        for (int t = warp; t < tiles; t += 4 * GG_JOIN) {                  // four loads under way
            float2 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = t + k * GG_JOIN < tiles ? __ldcg(stats + (size_t)(t + k * GG_JOIN) * rows + row) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int k = 0; k < 4; ++k) join(v[k]);
        }
    }
    part[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (warp || row >= rows) return;
    const int target = targets[row];
    const float z = target >= 0 && target < vocab ? __ldcg(picked + row) : 0.f;
    for (int k = 1; k < min(tiles, GG_JOIN); ++k) join(part[k][lane]);
    const float total = top + logf(sum);
    if (lse) lse[row] = total;
    loss[row] = target >= 0 && target < vocab ? total - z : 0.f;
    if (target >= vocab && id_error) atomicExch(id_error, 1);
}

}  // namespace bn

using namespace bn;

namespace {

struct Operand {
    const void *p0, *p1;
    long long ld;
};
// A product to be launched: bf16 results (M, N) with rows of ldc elements, up to three of them, or `partial`: fp32, [range][M][N]
struct Product {
    int M, N, K, second;
    bool a_mn;
    Operand a, b;
    void *c0, *c1, *c2;
    long long ldc;
    bool sums;                                                             // fp32 sums are kept in any case (pieces, or a reader of sums)
    float* partial;
    int add;
    const float* factor;
    int splits, per;                                                       // from a plan
    int steps() const { return (K + GG_BK - 1) / GG_BK * (second == SECOND_K ? 2 : 1); }
};

// Whether two CTAs share a tile of 256 x 256 (NT): not where one wave of single tiles is all there is, nor where tiles of twice the rows
// make a wave more than they save (an eighth).  Single tiles that would leave half of the SMs without one have 128 columns: what few rows
// wait for is the weight, and more SMs ask for it (gradients of a gated block of 64 rows, 2048 x 5632: 84 us with 44 tiles for gate and up,
// 79 with 88, 75 with the stages that the narrower tiles leave room for).
struct Cut { bool pair; int bn; };
Cut tile_columns(int M, int N, bool glu) {
    const long long sms = sm_count(), columns = (N + (glu ? GG_BN / 2 : GG_BN) - 1) / (glu ? GG_BN / 2 : GG_BN);
    const long long single = ((M + GG_BM - 1) / GG_BM) * columns, pairs = ((M + 2 * GG_BM - 1) / (2 * GG_BM)) * columns;
    const long long waves = (single + sms - 1) / sms, waves_of_pairs = (pairs + sms / 2 - 1) / (sms / 2);
    return {waves > 1 && waves_of_pairs * 7 <= waves * 8, 2 * single <= sms ? GG_BN / 2 : GG_BN};
}

long long tiles_of(const Product& p, bool pair) {
    const int rows = pair ? 2 * GG_BM : GG_BM;
    return (long long)((p.M + rows - 1) / rows) * ((p.N + GG_BN - 1) / GG_BN) * (p.second == SECOND_M ? 2 : 1);
}

// How products that share a launch are cut: all in pairs of CTAs or none, and the first of them (NN) into ranges of K, by the time until the
// last CTA is done.  Its unit is a pair's step of 64 k, 0.38 us; a single CTA's, of half the rows, half as long again (768
// cycles for its shared memory instead of 512).  An item takes its steps, or 6 for its epilogue where those are fewer, and 1.  CTAs take items in turn, the longest
// first.  A range of K is at least 4 steps, and its sums are written and read once more (0.75 MB a unit, and a launch).
struct Plan { bool pair; };
Plan plan_products(Product* p, int n) {
    const int sms = sm_count();
    double least = 1e30;
    Plan best{false};
    int best_splits = 1;
    const int most = p[0].a_mn ? 1 : p[0].steps() / 4 < 1 ? 1 : p[0].steps() / 4 > 32 ? 32 : p[0].steps() / 4;
    for (int pair = 0; pair < 2; ++pair)
        for (int s = 1; s <= most; ++s) {
            const int places = pair ? sms / 2 : sms, per = (p[0].steps() + s - 1) / s;
            if ((p[0].steps() + per - 1) / per != s) continue;
            double cost[GG_JOBS];
            long long count[GG_JOBS];
            int order[GG_JOBS];
            for (int i = 0; i < n; ++i) {
                const double steps = (i ? p[i].steps() : per) * (pair ? 1. : 1.5);
                cost[i] = (steps < 6 ? 6 : steps) + 1;
                count[i] = tiles_of(p[i], pair) * (i ? 1 : s);
                order[i] = i;
                for (int j = i; j > 0 && cost[order[j]] > cost[order[j - 1]]; --j) { const int t = order[j]; order[j] = order[j - 1]; order[j - 1] = t; }
            }
            // a round of all CTAs takes as long as its first item
            double time = 0;
            long long at = 0, end = 0;
            for (int k = 0; k < n; ++k) {
                end += count[order[k]];
                const long long rounds = end > at ? (end - at + places - 1) / places : 0;
                time += rounds * cost[order[k]];
                at += rounds * places;
            }
            if (s > 1) time += (double)s * p[0].M * p[0].N * 4 / 0.75e6 + (p[0].sums ? 0 : 8);
            if (time < least) least = time, best.pair = pair, best_splits = s;
        }
    for (int i = 0; i < n; ++i) {
        p[i].splits = i ? 1 : best_splits;
        p[i].per = i ? p[i].steps() : (p[0].steps() + best_splits - 1) / best_splits;
    }
    return best;
}

template <int EPI, int ACT, bool PAIR>
int grad_run(const AllMaps& m, const GradParams& p, unsigned grid, cudaStream_t st, const char* what) {
    const size_t smem = 1024 + (size_t)p.ring.stages * p.ring.stage_bytes + grad_out_bytes(EPI == GE_GLU);
    auto kernel = gemm_grad_kernel<EPI, ACT, PAIR>;
    static thread_local int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        if (int rc = allow_smem(kernel, smem, what, 226 * 1024)) return rc;
        configured_dev = dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(EPI == GE_GLU ? 320 : 192);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (PAIR) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 2;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaError_t e = launch_config(cfg, PAIR ? 1 : 0, kernel, m, p);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return fail(BN_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    }
    return BN_OK;
}

// n products in one launch (EPI other than PRODUCTS: one); sizes > 0, sizes and addresses are ones that a tensor map takes
template <int EPI, int ACT = 0>
int grad_gemm(const Product* products, int n, Cut cut, GradParams p, cudaStream_t st, const char* what) {
    constexpr bool MANY = EPI == GE_PRODUCTS;
    const int sms = sm_count();
    const bool pair = cut.pair;
    p.bn = cut.bn;
    p.ring = grad_ring(pair, EPI == GE_GLU, p.bn);
    const int columns = EPI == GE_GLU ? p.bn / 2 : p.bn, rows = pair ? 2 * GG_BM : GG_BM, places = pair ? sms / 2 : sms;
    const uint32_t n_box = EPI == GE_GLU || pair ? p.bn / 2 : p.bn;
    AllMaps all;
    long long items = 0;
    for (int i = 0; i < GG_JOBS; ++i) {
        GradJob& q = p.job[i];
        q.first = (int)items;
        if (i >= n) {
            all.job[i] = all.job[0];
            q.tiles = q.tiles_n = 1;
            continue;
        }
        // the longest items first
        const Product* o = &products[i];
        if (MANY) {
            const Product* order[GG_JOBS];
            for (int k = 0; k < n; ++k) {
                order[k] = &products[k];
                for (int j = k; j > 0 && order[j]->per > order[j - 1]->per; --j) { const Product* t = order[j]; order[j] = order[j - 1]; order[j - 1] = t; }
            }
            o = order[i];
        }
        const bool partial = MANY && (o->sums || o->splits > 1);
        q.M = o->M; q.N = o->N; q.K = o->K; q.second = o->second; q.a_mn = o->a_mn;
        q.partial = partial;
        q.add = o->add;
        q.splits = MANY ? (o->steps() + o->per - 1) / o->per : 1;
        q.k_per_split = o->per;
        q.factor = o->factor;
        q.tiles_m0 = (o->M + rows - 1) / rows;
        q.tiles_m = q.tiles_m0 * (o->second == SECOND_M ? 2 : 1);
        q.tiles_n = (o->N + columns - 1) / columns;
        const long long tiles = (long long)q.tiles_m * q.tiles_n;
        items += tiles * q.splits;
        if (items > INT32_MAX / 2) return fail(BN_ERR_UNSUPPORTED, "%s: more than 2^30 tiles", what);
        q.tiles = (int)tiles;
        GradMaps& m = all.job[i];
        auto map = [&](CUtensorMap* out, const void* base, long long ld, bool mn, int extent, uint32_t box_rows) {
            const uint64_t dims[2] = {(uint64_t)(mn ? extent : o->K), (uint64_t)(mn ? o->K : extent)}, strides[1] = {(uint64_t)ld * 2};
            const uint32_t box[2] = {64, mn ? 64 : box_rows};
            return make_tensor_map(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
        };
        if (int rc = map(&m.a0, o->a.p0, o->a.ld, o->a_mn, o->M, GG_BM)) return rc;
        if (int rc = map(&m.b0, o->b.p0, o->b.ld, MANY, o->N, n_box)) return rc;
        m.a1 = m.c0 = m.c1 = m.c2 = m.a0;
        m.b1 = m.b0;
        if (o->a.p1)
            if (int rc = map(&m.a1, o->a.p1, o->a.ld, o->a_mn, o->M, GG_BM)) return rc;
        if (o->b.p1)
            if (int rc = map(&m.b1, o->b.p1, o->b.ld, MANY, o->N, n_box)) return rc;
        if (partial) {
            const uint64_t dims[3] = {(uint64_t)o->N, (uint64_t)o->M, (uint64_t)q.splits}, strides[2] = {(uint64_t)o->N * 4, (uint64_t)o->M * o->N * 4};
            const uint32_t box[3] = {32, 32, 1};
            if (int rc = make_tensor_map(&m.c0, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, o->partial, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
            continue;
        }
        CUtensorMap* to[3] = {&m.c0, &m.c1, &m.c2};
        void* const base[3] = {o->c0, o->c1, o->c2};
        for (int k = 0; k < 3; ++k) {
            if (!base[k]) continue;
            const uint64_t dims[2] = {(uint64_t)o->N, (uint64_t)o->M}, strides[1] = {(uint64_t)o->ldc * 2};
            const uint32_t box[2] = {EPI == GE_GLU ? 32u : 64u, 32};
            if (int rc = make_tensor_map(to[k], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base[k], dims, strides, box,
                                         EPI == GE_GLU ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B))
                return rc;
        }
    }
    p.items = (int)items;
    const unsigned grid = (unsigned)(items < places ? items : places) * (pair ? 2 : 1);
    return pair ? grad_run<EPI, ACT, true>(all, p, grid, st, what) : grad_run<EPI, ACT, false>(all, p, grid, st, what);
}

int products(const Product* p, int n, Plan plan, int* error_word, cudaStream_t st, const char* what) {
    GradParams g{};
    g.error_word = error_word;
    return grad_gemm<GE_PRODUCTS>(p, n, {plan.pair, GG_BN}, g, st, what);
}

// sizes that stay 32-bit numbers when they are rounded up to tiles
constexpr int GG_LONGEST = INT32_MAX - 256;
bool longer(int a, int b, int c) { return a > GG_LONGEST || b > GG_LONGEST || c > GG_LONGEST; }

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

Product nn(int M, int N, int K, int second, bool sums) {
    Product p{};
    p.M = M; p.N = N; p.K = K; p.second = second; p.sums = sums;
    return p;
}
Product tn(int M, int N, int K, int second) {
    Product p{};
    p.M = M; p.N = N; p.K = K; p.second = second; p.a_mn = true;
    return p;
}
// the fp32 sums that a planned product leaves
size_t sum_bytes(const Product& p) { return p.sums || p.splits > 1 ? up256((size_t)p.splits * p.M * p.N * 4) : 0; }
// adds them, where it has left any
int add_sums(const Product& p, void* c, int splits, cudaStream_t st, const char* what) {
    if (!p.sums && splits == 1) return BN_OK;
    const long long groups = (long long)p.M * p.N / 4;
    launch_dependent(grad_sum_kernel, (unsigned)((groups + 127) / 128), 128, 0, st, (const float*)p.partial, static_cast<__nv_bfloat16*>(c), groups, splits, p.factor);
    return launch_status(what);
}

bool misaligned(std::initializer_list<const void*> all) {
    for (const void* p : all)
        if (reinterpret_cast<uintptr_t>(p) & 15) return true;
    return false;
}

int zero(void* p, size_t bytes, cudaStream_t st, const char* what) {
    if (!p || !bytes) return BN_OK;
    cudaError_t e = cudaMemsetAsync(p, 0, bytes, st);
    return e == cudaSuccess ? BN_OK : fail(BN_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Columns of the vocabulary that a piece of the backward pass takes: the piece's logit gradients, 2 bytes each, stay at 128 MB, about what
// L2 holds, or at 4096 columns where that is more (above 16384 rows): every piece reads and writes the rows' fp32 gradients again (rows x
// hidden x 8 bytes against 6 x rows x columns x hidden operations: of 4096 columns a tenth of the products' time).  Pieces are of equal
// size, so they have more than half as many columns: 4500 of 16500 rows are two of 2304, whose traffic is then a fifth.
int piece_columns(int rows, int vocab) {
    long long want = (64LL << 20) / rows / 256 * 256;
    if (want < 4096) want = 4096;
    const long long all = ((long long)vocab + 255) / 256 * 256;
    if (want >= all) return (int)all;
    const long long pieces = (all + want - 1) / want;                      // of equal size
    return (int)(((all + pieces - 1) / pieces + 255) / 256 * 256);
}

int check_loss(const char* what, const void* x, const void* w, const void* targets, int rows, int vocab, int hidden) {
    if (!w || (rows > 0 && (!x || !targets))) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (rows < 0 || vocab <= 0 || hidden <= 0) return fail(BN_ERR_INVALID_ARG, "%s: bad shape rows=%d vocab=%d hidden=%d", what, rows, vocab, hidden);
    if (hidden % 8) return fail(BN_ERR_UNSUPPORTED, "%s: hidden=%d must be a multiple of 8 (16-byte rows)", what, hidden);
    if (longer(rows, vocab, hidden)) return fail(BN_ERR_UNSUPPORTED, "%s: rows=%d vocab=%d hidden=%d too large", what, rows, vocab, hidden);
    if (misaligned({x, w})) return fail(BN_ERR_INVALID_ARG, "%s: x and the weight must be 16-byte aligned", what);
    return BN_OK;
}

int check_ws(const char* what, const void* ws, size_t given, size_t needed) {
    if (given < needed || (needed && !ws)) return fail(BN_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", what, given, needed);
    if (reinterpret_cast<uintptr_t>(ws) & 255) return fail(BN_ERR_INVALID_ARG, "%s: workspace must be 256-byte aligned", what);
    return BN_OK;
}

}  // namespace

// ------------------------------------------------------------------------------------------------------------- products
extern "C" size_t bn_gemm_bf16_nn_workspace_bytes(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || longer(M, N, K)) return 0;
    Product p = nn(M, N, K, SECOND_NONE, false);
    plan_products(&p, 1);
    return sum_bytes(p);
}

static int check_product(const char* what, const void* a, const void* b, const void* c, int M, int N, int K, int inner_a) {
    if ((M > 0 && N > 0 && !c) || (M > 0 && K > 0 && !a) || (N > 0 && K > 0 && !b)) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (M < 0 || N < 0 || K < 0) return fail(BN_ERR_INVALID_ARG, "%s: bad shape M=%d N=%d K=%d", what, M, N, K);
    if (longer(M, N, K)) return fail(BN_ERR_UNSUPPORTED, "%s: M=%d N=%d K=%d too large", what, M, N, K);
    if (N % 8 || inner_a % 8) return fail(BN_ERR_UNSUPPORTED, "%s: rows of %d and %d elements must be multiples of 8 (16 bytes)", what, inner_a, N);
    if (misaligned({a, b, c})) return fail(BN_ERR_INVALID_ARG, "%s: a/b/c must be 16-byte aligned", what);
    return require_sm100();
}

extern "C" int bn_gemm_bf16_nn(const void* a, const void* b, void* c, int M, int N, int K, void* workspace, size_t workspace_bytes, int* error_word,
                               bn_stream_t stream) {
    const char* what = "bn_gemm_bf16_nn";
    if (int rc = check_product(what, a, b, c, M, N, K, K)) return rc;
    if (M == 0 || N == 0) return BN_OK;
    if (K == 0) return zero(c, (size_t)M * N * 2, as_stream(stream), what);
    if (int rc = check_ws(what, workspace, workspace_bytes, bn_gemm_bf16_nn_workspace_bytes(M, N, K))) return rc;
    Product p = nn(M, N, K, SECOND_NONE, false);
    p.a = {a, nullptr, K};
    p.b = {b, nullptr, N};
    p.c0 = c;
    p.ldc = N;
    p.partial = static_cast<float*>(workspace);
    const Plan plan = plan_products(&p, 1);
    if (int rc = products(&p, 1, plan, error_word, as_stream(stream), what)) return rc;
    return add_sums(p, c, p.splits, as_stream(stream), what);
}

extern "C" int bn_gemm_bf16_tn(const void* a, const void* b, void* c, int M, int N, int K, int* error_word, bn_stream_t stream) {
    const char* what = "bn_gemm_bf16_tn";
    if (int rc = check_product(what, a, b, c, M, N, K, M)) return rc;
    if (M == 0 || N == 0) return BN_OK;
    if (K == 0) return zero(c, (size_t)M * N * 2, as_stream(stream), what);
    Product p = tn(M, N, K, SECOND_NONE);
    p.a = {a, nullptr, M};
    p.b = {b, nullptr, N};
    p.c0 = c;
    p.ldc = N;
    const Plan plan = plan_products(&p, 1);
    return products(&p, 1, plan, error_word, as_stream(stream), what);
}

// ------------------------------------------------------------------------------------------------- loss over the vocabulary
extern "C" size_t bn_linear_cross_entropy_bf16_workspace_bytes(int rows, int vocab, int hidden) {
    if (rows <= 0 || vocab <= 0 || hidden <= 0 || longer(rows, vocab, hidden)) return 0;
    const int columns = tile_columns(rows, vocab, false).bn;
    const size_t tiles = ((size_t)vocab + columns - 1) / columns;
    return up256(tiles * rows * sizeof(float2)) + up256((size_t)rows * sizeof(float));
}

extern "C" int bn_linear_cross_entropy_bf16(const void* x, const void* weight_t, const int32_t* targets, float* loss, float* lse, int rows, int vocab,
                                            int hidden, void* workspace, size_t workspace_bytes, int* id_error, int* error_word, bn_stream_t stream) {
    const char* what = "bn_linear_cross_entropy_bf16";
    if (int rc = check_loss(what, x, weight_t, targets, rows, vocab, hidden)) return rc;
    if (rows > 0 && !loss) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (int rc = require_sm100()) return rc;
    if (rows == 0) return BN_OK;
    if (int rc = check_ws(what, workspace, workspace_bytes, bn_linear_cross_entropy_bf16_workspace_bytes(rows, vocab, hidden))) return rc;
    const Cut cut = tile_columns(rows, vocab, false);
    const int tiles = (vocab + cut.bn - 1) / cut.bn;
    Product z = nn(rows, vocab, hidden, SECOND_NONE, false);               // (logits: along K on both sides)
    z.a = {x, nullptr, hidden};
    z.b = {weight_t, nullptr, hidden};
    z.per = z.steps();
    GradParams p{};
    p.error_word = error_word;
    p.targets = targets;
    p.stats = static_cast<float2*>(workspace);
    p.picked = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + up256((size_t)tiles * rows * sizeof(float2)));
    cudaStream_t st = as_stream(stream);
    if (int rc = grad_gemm<GE_LOSS>(&z, 1, cut, p, st, what)) return rc;
    launch_dependent(loss_join_kernel, (unsigned)((rows + 31) / 32), 32 * GG_JOIN, 0, st, (const float2*)p.stats, (const float*)p.picked, targets, loss, lse, id_error,
                     rows, tiles, vocab);
    return launch_status(what);
}

// a piece's two products
static Plan plan_piece(Product (&p)[2], int rows, int vocab, int hidden) {
    const int columns = piece_columns(rows, vocab), n = columns < vocab ? columns : vocab;
    p[0] = nn(rows, hidden, n, SECOND_NONE, columns < vocab);
    p[1] = tn(n, hidden, rows, SECOND_NONE);
    return plan_products(p, 2);
}

extern "C" size_t bn_linear_cross_entropy_backward_bf16_workspace_bytes(int rows, int vocab, int hidden) {
    if (rows <= 0 || vocab <= 0 || hidden <= 0 || longer(rows, vocab, hidden)) return 0;
    Product p[2];
    plan_piece(p, rows, vocab, hidden);
    return up256((size_t)rows * piece_columns(rows, vocab) * 2) + sum_bytes(p[0]);
}

extern "C" int bn_linear_cross_entropy_backward_bf16(const void* x, const void* weight_t, const int32_t* targets, const float* lse, const float* grad_loss,
                                                     void* dx, void* dweight_t, int rows, int vocab, int hidden, void* workspace, size_t workspace_bytes,
                                                     int* error_word, bn_stream_t stream) {
    const char* what = "bn_linear_cross_entropy_backward_bf16";
    if (int rc = check_loss(what, x, weight_t, targets, rows, vocab, hidden)) return rc;
    if (rows > 0 && (!lse || !grad_loss || (!dx && !dweight_t))) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (misaligned({dx, dweight_t})) return fail(BN_ERR_INVALID_ARG, "%s: gradients must be 16-byte aligned", what);
    if (int rc = require_sm100()) return rc;
    cudaStream_t st = as_stream(stream);
    if (rows == 0) return zero(dweight_t, (size_t)vocab * hidden * 2, st, what);
    if (int rc = check_ws(what, workspace, workspace_bytes, bn_linear_cross_entropy_backward_bf16_workspace_bytes(rows, vocab, hidden))) return rc;
    const int columns = piece_columns(rows, vocab);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    Product p[2];                                                          // dx and dweight of a piece, in one launch
    const Plan plan = plan_piece(p, rows, vocab, hidden);
    const int splits = p[0].splits;
    p[0].a = p[1].a = {ws, nullptr, columns};
    p[0].c0 = dx;
    p[0].ldc = p[1].ldc = hidden;
    p[0].partial = reinterpret_cast<float*>(ws + up256((size_t)rows * columns * 2));
    p[0].factor = p[1].factor = grad_loss;
    p[1].b = {x, nullptr, hidden};
    for (int v0 = 0; v0 < vocab; v0 += columns) {
        const int n = vocab - v0 < columns ? vocab - v0 : columns;
        const void* w = static_cast<const __nv_bfloat16*>(weight_t) + (size_t)v0 * hidden;
        Product z = nn(rows, n, hidden, SECOND_NONE, false);
        z.a = {x, nullptr, hidden};
        z.b = {w, nullptr, hidden};
        z.c0 = ws;
        z.ldc = columns;
        z.per = z.steps();
        GradParams g{};
        g.error_word = error_word;
        g.targets = targets; g.first_column = v0; g.vocab = vocab; g.lse = lse; g.grad = grad_loss;
        if (int rc = grad_gemm<GE_DLOGITS>(&z, 1, tile_columns(rows, n, false), g, st, what)) return rc;
        // a last, shorter piece leaves ranges of K without a step: they are not launched, and what they have so far stays
        p[0].K = p[1].M = n;
        p[0].add = v0 > 0;
        p[0].b = {w, nullptr, hidden};
        p[1].c0 = dweight_t ? static_cast<__nv_bfloat16*>(dweight_t) + (size_t)v0 * hidden : nullptr;
        if (int rc = products(dx ? p : p + 1, (dx != nullptr) + (dweight_t != nullptr), plan, error_word, st, what)) return rc;
    }
    return dx ? add_sums(p[0], dx, splits, st, what) : BN_OK;
}

// --------------------------------------------------------------------------------------------- gated feed-forward block
// dh; then dx and the weights' gradients
static Plan plan_dh(Product& p, int rows, int hidden, int inter) {
    p = nn(rows, inter, hidden, SECOND_NONE, true);
    return plan_products(&p, 1);
}
static Plan plan_gradients(Product (&p)[3], int rows, int hidden, int inter) {
    p[0] = nn(rows, hidden, inter, SECOND_K, false);
    p[1] = tn(inter, hidden, rows, SECOND_M);
    p[2] = tn(hidden, inter, rows, SECOND_NONE);
    return plan_products(p, 3);
}

// h, dgate and dup (bf16); dh and, when that has been used, the sums of dx (fp32): dh rounded to bf16 would add half of the error that the
// gradients have from their own roundings (2.9e-3 instead of 2.35e-3), and its ranges of K are added where it is read
extern "C" size_t bn_gated_ff_backward_bf16_workspace_bytes(int rows, int hidden, int inter) {
    if (rows <= 0 || hidden <= 0 || inter <= 0 || longer(rows, hidden, inter)) return 0;
    Product dh, p[3];
    plan_dh(dh, rows, hidden, inter);
    plan_gradients(p, rows, hidden, inter);
    const size_t a = sum_bytes(dh), b = sum_bytes(p[0]);
    return 3 * up256((size_t)rows * inter * 2) + (a > b ? a : b);
}

extern "C" int bn_gated_ff_backward_bf16(const void* dy, const void* x, const void* gate_t, const void* up_t, const void* down_t, void* dx, void* dgate_t,
                                         void* dup_t, void* ddown_t, int rows, int hidden, int inter, int act, void* workspace, size_t workspace_bytes,
                                         int* error_word, bn_stream_t stream) {
    const char* what = "bn_gated_ff_backward_bf16";
    if (!gate_t || !up_t || !down_t || !dgate_t || !dup_t || !ddown_t || (rows > 0 && (!dy || !x || !dx))) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (rows < 0 || hidden <= 0 || inter <= 0) return fail(BN_ERR_INVALID_ARG, "%s: bad shape rows=%d hidden=%d inter=%d", what, rows, hidden, inter);
    if (longer(rows, hidden, inter)) return fail(BN_ERR_UNSUPPORTED, "%s: rows=%d hidden=%d inter=%d too large", what, rows, hidden, inter);
    if (hidden % 8 || inter % 8)
        return fail(BN_ERR_UNSUPPORTED, "%s: hidden=%d and inter=%d must be multiples of 8 (16-byte rows)", what, hidden, inter);
    if (act != BN_ACT_SILU && act != BN_ACT_GELU_TANH) return fail(BN_ERR_UNSUPPORTED, "%s: activation %d", what, act);
    if (misaligned({dy, x, gate_t, up_t, down_t, dx, dgate_t, dup_t, ddown_t}))
        return fail(BN_ERR_INVALID_ARG, "%s: operands must be 16-byte aligned", what);
    if (int rc = require_sm100()) return rc;
    cudaStream_t st = as_stream(stream);
    if (rows == 0) {
        const size_t bytes = (size_t)inter * hidden * 2;
        if (int rc = zero(dgate_t, bytes, st, what)) return rc;
        if (int rc = zero(dup_t, bytes, st, what)) return rc;
        return zero(ddown_t, bytes, st, what);
    }
    if (int rc = check_ws(what, workspace, workspace_bytes, bn_gated_ff_backward_bf16_workspace_bytes(rows, hidden, inter))) return rc;
    const size_t each = up256((size_t)rows * inter * 2);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    void *h = ws, *dg = ws + each, *du = ws + 2 * each;
    float* partial = reinterpret_cast<float*>(ws + 3 * each);
    // dh = dy Wdown
    Product d;
    const Plan first = plan_dh(d, rows, hidden, inter);
    d.a = {dy, nullptr, hidden};
    d.b = {down_t, nullptr, inter};
    d.partial = partial;
    if (int rc = products(&d, 1, first, error_word, st, what)) return rc;
    // gate and up again; their gradients, and the product of the forward pass
    Product gu = nn(rows, inter, hidden, SECOND_NONE, false);              // (along K on both sides)
    gu.a = {x, nullptr, hidden};
    gu.b = {gate_t, up_t, hidden};
    gu.c0 = h;
    gu.c1 = dg;
    gu.c2 = du;
    gu.ldc = inter;
    gu.per = gu.steps();
    GradParams g{};
    g.error_word = error_word;
    g.dh = partial;
    g.dh_parts = d.splits;
    const Cut cut = tile_columns(rows, inter, true);
    if (int rc = act == BN_ACT_SILU ? grad_gemm<GE_GLU, BN_ACT_SILU>(&gu, 1, cut, g, st, what) : grad_gemm<GE_GLU, BN_ACT_GELU_TANH>(&gu, 1, cut, g, st, what))
        return rc;
    // dx = dgate Wgate + dup Wup (one product of twice the K), dWgate and dWup = dgate^T x, dup^T x, dWdown = dy^T h
    Product p[3];
    const Plan plan = plan_gradients(p, rows, hidden, inter);
    p[0].a = p[1].a = {dg, du, inter};
    p[0].b = {gate_t, up_t, hidden};
    p[0].c0 = dx;
    p[0].partial = partial;
    p[1].b = {x, nullptr, hidden};
    p[1].c0 = dgate_t;
    p[1].c1 = dup_t;
    p[2].a = {dy, nullptr, hidden};
    p[2].b = {h, nullptr, inter};
    p[2].c0 = ddown_t;
    p[0].ldc = p[1].ldc = hidden;
    p[2].ldc = inter;
    if (int rc = products(p, 3, plan, error_word, st, what)) return rc;
    return add_sums(p[0], dx, p[0].splits, st, what);
}
