// The products of a backward pass, bf16 with fp32 accumulation in tensor memory, for sm_100a, and the two operators of a training step
// that are made of them: softmax cross entropy over a large vocabulary (op_cross_entropy, src/ops/op_cross_entropy.cuh:5-45, and the
// lm_head product before it) and the gradients of the gated feed-forward block (MLP.__call__, mygrad/llama/llama_layers.py:194-235;
// op_silu_backward, src/ops/op_silu.cuh).
//
// One kernel, three operand orders.  y = x W^T reads both operands along K (NT).  Its gradients do not: dx = dy W reads W across its
// rows (NN), dW = dy^T x reads both across (TN).  tcgen05 takes either order from shared memory (MN-major operands: tiles of 64 k rows of
// 64 contiguous m or n), so nothing is transposed in memory.
// Persistent kernel, 192 threads: warps 0-3 epilogue, warp 4 issues the MMAs, warp 5 loads by TMA.  Output tile 128 x 256, or (PAIR) 256 x
// 256 shared by a cluster of two CTAs (tcgen05.mma.cta_group::2); fp32 accumulators double buffered in tensor memory, so that the
// epilogue of a tile runs under the products of the next.  Tiles may have 128 columns, where there are few
// (tile_columns).  They go in bands of 16 tile rows, n outside, so that what runs at one time shares both operands in L2.
//
// Results leave through shared memory: a warp writes 32 rows of 128 bytes and one thread has TMA store them (a thread that stores its own
// row takes 32 places in memory for every 16 bytes: 32000 x 2048 of K = 200 71 -> 46 us; eight epilogue warps instead of four 46, and 2 - 5 %
// more for long K).
//
// Epilogues
//   STORE     the result as bf16
//   PARTIAL   fp32 sums of a range of K, kept or added to what an earlier launch left: few tiles share K, pieces of the vocabulary follow
//             one another.  An element gets one sum from a launch, and grad_sum_kernel adds the ranges in order: the same bits in every run
//   LOSS      logits: of every row's columns in a tile the maximum and the sum of exponentials, and the target's logit: the logits stay in
//             tensor memory
//   DLOGITS   logits again -> g (exp(z - lse) - [v = target]) over the first row's g, as bf16
//   GLU       columns [0,128) gate, [128,256) up of the same indices, and dh, fp32 -> dgate, dup and the product that the forward pass had
// Every mbarrier wait is bounded; on expiry the kernel raises the caller's error word, frees TMEM and returns.
#include "common.cuh"
#include "hybrid.cuh"
#include "ptx.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace bn {

using namespace ptx;

constexpr int GG_BM = 128, GG_BN = 256, GG_BK = 64, GG_THREADS = 192, GG_BAND = 16;
constexpr int GG_A_BYTES = GG_BM * GG_BK * 2;
constexpr int GG_OUT_BYTES = 32 * 128;                                     // what a warp stores at a time
// Shared memory: as many stages of operands as fit beside each epilogue warp's buffers (GLU: one for each of three results, else two in turn)
constexpr int GG_MAX_STAGES = 6;
struct GradRing { int stage_bytes, stages; };
constexpr GradRing grad_ring(bool pair, bool glu, int bn) {
    const int stage = GG_A_BYTES + (pair ? bn / 2 : bn) * GG_BK * 2, room = 225 * 1024 - 4 * (glu ? 3 : 2) * GG_OUT_BYTES;
    return {stage, room / stage < GG_MAX_STAGES ? room / stage : GG_MAX_STAGES};
}

constexpr int GE_STORE = 0, GE_PARTIAL = 1, GE_LOSS = 2, GE_DLOGITS = 3, GE_GLU = 4;
// what the second pair of operands is: none, the second half of K (NN), further rows of the result (TN), the upper 128 columns of every
// tile (NT, GLU)
constexpr int SECOND_NONE = 0, SECOND_K = 1, SECOND_M = 2;

struct GradParams {
    int M, N, K;                       // of one pair of operands
    int second;
    int bn;                            // columns of a tile (GLU: of gate and up together)
    GradRing ring;
    int splits, k_per_split;           // PARTIAL: ranges of K steps
    int* error_word;
    int add;                           // PARTIAL: added to what is there
    const int32_t* targets;            // LOSS, DLOGITS: (M), minus first_column is the column here
    int first_column, vocab;
    float2* stats;                     // LOSS: [tile][M] maximum, sum of exponentials of the distances to it
    float* picked;                     // LOSS: (M) the target's logit
    const float *lse, *grad;           // DLOGITS: (M)
    const float* factor;               // STORE: what common_factor makes of it is a factor of the result
    const float* dh;                   // GLU: [dh_parts][M][N], to be added up
    int dh_parts;
};

// Tensor maps of the operands and of what is stored: STORE c0 and (of the second rows) c1, bf16; PARTIAL c0, fp32 (N, M, split); DLOGITS c0;
// GLU c0 = h, c1 = dgate, c2 = dup
struct GradMaps { CUtensorMap a0, a1, b0, b1, c0, c1, c2; };

// What the logits' gradients are divided by before they are rounded, and their products multiplied by: the first row's gradient, so that a
// mean's 1 / rows, which all rows have, is not rounded to bf16 in every one of them alike (errors of 2.9e-3 instead of 2.4e-3)
__device__ __forceinline__ float common_factor(const float* grad) {
    const float g = grad ? *grad : 1.f, size = fabsf(g);
    return size >= 0x1p-40f && size <= 0x1p40f ? g : 1.f;
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

template <bool A_MN, bool B_MN, int EPI, int ACT, bool PAIR>
__global__ void __launch_bounds__(GG_THREADS, 1)
gemm_grad_kernel(const __grid_constant__ GradMaps maps, const GradParams p) {
    constexpr int TILE_M = PAIR ? 2 * GG_BM : GG_BM, OUT = EPI == GE_GLU ? 3 : 2;
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
    const int tiles_m0 = (p.M + TILE_M - 1) / TILE_M, tiles_m = p.second == SECOND_M ? 2 * tiles_m0 : tiles_m0;
    const int tiles_n = (p.N + columns - 1) / columns, tiles = tiles_m * tiles_n;
    const int steps0 = (p.K + GG_BK - 1) / GG_BK, steps = p.second == SECOND_K ? 2 * steps0 : steps0;
    const int items = tiles * (EPI == GE_PARTIAL ? p.splits : 1);
    struct Item { int m, n, part, ks0, ks1; };                             // tile row and column; which operands; K steps
    auto item = [&](int t) {
        Item w;
        const int split = EPI == GE_PARTIAL ? t / tiles : 0;
        t -= split * tiles;
        const int band = t / (GG_BAND * tiles_n), in_band = t - band * GG_BAND * tiles_n;
        const int height = min(GG_BAND, tiles_m - band * GG_BAND);
        w.n = in_band / height;
        w.m = band * GG_BAND + in_band - w.n * height;
        w.part = w.m >= tiles_m0;
        if (w.part) w.m -= tiles_m0;
        w.ks0 = EPI == GE_PARTIAL ? split * p.k_per_split : 0;
        w.ks1 = EPI == GE_PARTIAL ? min(steps, w.ks0 + p.k_per_split) : steps;
        return w;
    };

    if (tid == 0) {
        for (int s = 0; s < n_stages; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&bar_acc_full[i]), 1);
            mbar_init(smem_u32(&bar_acc_empty[i]), PAIR ? 8 : 4);          // one arrive per epilogue warp
        }
        s_abort = 0;
        fence_mbar_init();
    }
    if (warp == 4) {
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

    if (warp == 5) {
        // ---------------------------------------------------------- TMA producer
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = first; ok && t < items; t += stride) {
                const Item w = item(t);
                const int m0 = w.m * TILE_M + rank * GG_BM, n0 = w.n * columns + (EPI == GE_GLU ? 0 : rank * n_here);
                const uint32_t bytes = (PAIR ? 2 : 1) * (GG_A_BYTES + n_here * GG_BK * 2);
                for (int ks = w.ks0; ks < w.ks1; ++ks) {
                    ok = mbar_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, &s_abort);
                    if (!ok) break;
                    const bool half2 = p.second == SECOND_K && ks >= steps0;
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
                    if (A_MN) {
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
                    } else if (B_MN) {
                        for (int j = 0; j < n_here / 64; ++j) load(sB + j * 8192, mb, n0 + j * 64, k0);
                    } else {
                        load(sB, mb, k0, n0);
                    }
                    if (++stage == n_stages) stage = 0, phase ^= 1u;
                }
            }
        }
    } else if (warp == 4) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t IDESC = tc::idesc_bf16(TILE_M, p.bn, B_MN ? 1 : 0) | (A_MN ? 1u << 15 : 0u);
        const uint64_t dK = tc::smem_desc_sw128(0);                        // descriptor = this + (address >> 4)
        const uint64_t dMN = (dK & ~((uint64_t)0x3fff << 16)) | (uint64_t)(8192 >> 4) << 16;      // the next 64 m or n lie 8 KB on
        constexpr uint32_t A_STEP = A_MN ? 128 : 2, B_STEP = B_MN ? 128 : 2;                      // 16 k further, in 16 bytes
        uint32_t local = 0, phase = 0;
        int stage = 0;
        bool ok = rank == 0;
        for (int t = first; ok && t < items; t += stride, ++local) {
            const uint32_t acc = local & 1u;
            ok = mbar_wait_warp(smem_u32(&bar_acc_empty[acc]), ((local >> 1) & 1u) ^ 1u, &s_abort);    // drained two tiles ago
            if (!ok) break;
            tc::fence_after_sync();
            const Item w = item(t);
            for (int ks = w.ks0; ks < w.ks1; ++ks) {
                ok = mbar_wait_warp(smem_u32(&bar_full[stage]), phase, &s_abort);
                if (!ok) break;
                if (elect_one()) {
                    tc::fence_after_sync();
                    const uint32_t sA = smem0 + stage * p.ring.stage_bytes, sB = sA + GG_A_BYTES;
#pragma unroll
                    for (int kk = 0; kk < GG_BK / 16; ++kk) {
                        const uint64_t da = (A_MN ? dMN : dK) + (uint64_t)((sA >> 4) + kk * A_STEP);
                        const uint64_t db = (B_MN ? dMN : dK) + (uint64_t)((sB >> 4) + kk * B_STEP);
                        if (PAIR) tc::pair_mma_ss(tmem + acc * GG_BN, da, db, IDESC, (ks > w.ks0) || (kk > 0));
                        else tc::mma_ss(tmem + acc * GG_BN, da, db, IDESC, (ks > w.ks0) || (kk > 0));
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
        }
    } else {
        // ------------------------------------------------------ epilogue: thread = row of the tile = TMEM lane
        const uint32_t lane_base = ((uint32_t)(warp * 32)) << 16;
        const uint32_t out0 = smem0 + n_stages * p.ring.stage_bytes + warp * OUT * GG_OUT_BYTES;
        int out_turn = 0;
        // the warp's next buffer, when what was sent from it before has been read
        auto out_buffer = [&] {
            if (lane == 0) bulk_wait_group_read<1>();
            __syncwarp();
            out_turn ^= 1;
            return out0 + out_turn * GG_OUT_BYTES;
        };
        auto put16 = [&](uint32_t buf, int chunk, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {      // 16 bytes of the thread's row, swizzled
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(buf + lane * 128 + ((chunk ^ (lane & 7)) << 4)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
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
        for (int t = first; ok && t < items; t += stride, ++local) {
            const uint32_t acc = local & 1u;
            const Item w = item(t);
            const int gm = w.m * TILE_M + rank * GG_BM + tid, n0 = w.n * columns;
            const bool live = gm < p.M;
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
                if (EPI != GE_GLU || col0 >= p.N) return;
                const float4* from = reinterpret_cast<const float4*>(p.dh + (size_t)(live ? gm : 0) * p.N + col0);
                const size_t part = (size_t)p.M * p.N / 4;
#pragma unroll
                for (int v = 0; v < 8; ++v) {                              // (columns are a multiple of 8)
                    const float4 f = col0 + v * 4 < p.N ? __ldcg(from + v) : make_float4(0.f, 0.f, 0.f, 0.f);
                    d[v * 4] = f.x; d[v * 4 + 1] = f.y; d[v * 4 + 2] = f.z; d[v * 4 + 3] = f.w;
                }
#pragma unroll 2
                for (int k = 1; k < p.dh_parts; ++k) {                     // (eight loads under way, or sixteen)
#pragma unroll
                    for (int v = 0; v < 8; ++v) {
                        const float4 f = col0 + v * 4 < p.N ? __ldcg(from + k * part + v) : make_float4(0.f, 0.f, 0.f, 0.f);
                        d[v * 4] += f.x; d[v * 4 + 1] += f.y; d[v * 4 + 2] += f.z; d[v * 4 + 3] += f.w;
                    }
                }
            };
            load_dh(n0);
            ok = mbar_wait_warp(smem_u32(&bar_acc_full[acc]), (local >> 1) & 1u, &s_abort);
            if (!ok) break;
            tc::fence_after_sync();
            const uint32_t tacc = tmem + lane_base + acc * GG_BN;
            const int y = w.m * TILE_M + rank * GG_BM + warp * 32;          // the warp's first row
            if (EPI == GE_STORE || EPI == GE_DLOGITS) {
#pragma unroll 1
                for (int c = 0; c < p.bn / 64; ++c) {
                    if (n0 + c * 64 >= p.N) break;                         // (uniform)
                    const uint32_t buf = out_buffer();
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        uint32_t r[32];
                        tc::ld32(tacc + c * 64 + hf * 32, r);
                        tc::wait_ld(r);
                        if (EPI == GE_STORE && p.factor) {
                            const float factor = common_factor(p.factor);
#pragma unroll
                            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * factor);
                        }
                        if (EPI == GE_DLOGITS) {
                            const int at = target - (n0 + c * 64 + hf * 32);
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float q = ex2(fmaf(__uint_as_float(r[e]), log2e(), -lse2)) - (e == at ? 1.f : 0.f);
                                r[e] = __float_as_uint(target == INT32_MIN ? 0.f : grad * q);
                            }
                        }
                        put_row(buf, hf, r);
                    }
                    if (y < p.M) send([&] { tma_store_2d(w.part ? &maps.c1 : &maps.c0, buf, n0 + c * 64, y); });
                }
            } else if (EPI == GE_PARTIAL) {
#pragma unroll 1
                for (int c = 0; c < p.bn / 32; ++c) {
                    if (n0 + c * 32 >= p.N) break;
                    const uint32_t buf = out_buffer();
                    uint32_t r[32];
                    tc::ld32(tacc + c * 32, r);
                    tc::wait_ld(r);
#pragma unroll
                    for (int v = 0; v < 8; ++v) put16(buf, v, r[v * 4], r[v * 4 + 1], r[v * 4 + 2], r[v * 4 + 3]);
                    if (y < p.M)
                        send([&] {
                            if (p.add) tma_add_3d(&maps.c0, buf, n0 + c * 32, y, t / tiles);
                            else tma_store_3d(&maps.c0, buf, n0 + c * 32, y, t / tiles);
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
                    if (col >= p.N) continue;                              // (uniform)
                    if (col + 32 > p.N) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (col + e >= p.N) r[e] = __float_as_uint(-INFINITY);
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
                        if (at >= 0 && at < 32 && target < p.N) p.picked[gm] = z;
                    }
                }
                if (live) p.stats[(size_t)w.n * p.M + gm] = make_float2(top, sum);
            } else {
                const uint32_t h_buf = out0, g_buf = out0 + GG_OUT_BYTES, u_buf = out0 + 2 * GG_OUT_BYTES;
#pragma unroll 1
                for (int c = 0; c < p.bn / 64; ++c) {                      // 32 columns: half of what is stored at a time
                    const int col0 = n0 + c * 32;
                    if (col0 >= p.N) break;
                    uint32_t g[32], u[32];
                    tc::ld32(tacc + c * 32, g);
                    tc::ld32(tacc + p.bn / 2 + c * 32, u);
                    tc::wait_ld(g);
                    tc::wait_ld(u);
                    if (c % 2 == 0) {                                      // the buffers have been read
                        if (lane == 0) bulk_wait_group_read<0>();
                        __syncwarp();
                    }
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
                        const int chunk = c % 2 * 4 + v;
                        put16(h_buf, chunk, h4[0], h4[1], h4[2], h4[3]);
                        put16(g_buf, chunk, g4[0], g4[1], g4[2], g4[3]);
                        put16(u_buf, chunk, u4[0], u4[1], u4[2], u4[3]);
                    }
                    if (c + 1 < p.bn / 64) load_dh(col0 + 32);             // (the next tile's: before its products are waited for)
                    if ((c % 2 == 1 || col0 + 32 >= p.N) && y < p.M) {     // (what a last half does not fill lies behind the columns)
                        const int x = n0 + c / 2 * 64;
                        send([&] {
                            tma_store_2d(&maps.c0, h_buf, x, y);
                            tma_store_2d(&maps.c1, g_buf, x, y);
                            tma_store_2d(&maps.c2, u_buf, x, y);
                        });
                    }
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
    if (warp == 4) {
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
// What is stored: bf16 (M, N) with rows of ld elements, up to three of them, or `splits` fp32 (M, N)
struct Result {
    void *p0, *p1, *p2;
    long long ld;
};

// How a product is cut.  Two CTAs share a tile of 256 x 256, but not where one wave of single tiles is all there is, nor where tiles of twice
// the rows make a wave more than they save (an eighth).  Single tiles that would leave half of the SMs without one have 128 columns: what
// few rows wait for is the weight, and more SMs ask for it (gradients of a gated block of 64 rows, 2048 x 5632: 84 us with 44 tiles for gate
// and up, 79 with 88, 75 with the stages that the narrower tiles leave room for).
struct Cut { bool pair; int bn; };
Cut tile_columns(int M, int N, int second, bool glu) {
    const long long sms = sm_count(), twice = second == SECOND_M ? 2 : 1, columns = (N + (glu ? GG_BN / 2 : GG_BN) - 1) / (glu ? GG_BN / 2 : GG_BN);
    const long long single = twice * ((M + GG_BM - 1) / GG_BM) * columns, pairs = twice * ((M + 2 * GG_BM - 1) / (2 * GG_BM)) * columns;
    const long long waves = (single + sms - 1) / sms, waves_of_pairs = (pairs + sms / 2 - 1) / (sms / 2);
    return {waves > 1 && waves_of_pairs * 7 <= waves * 8, 2 * single <= sms ? GG_BN / 2 : GG_BN};
}

template <bool A_MN, bool B_MN, int EPI, int ACT, bool PAIR>
int grad_run(const GradMaps& m, const GradParams& p, unsigned grid, cudaStream_t st, const char* what) {
    const size_t smem = 1024 + (size_t)p.ring.stages * p.ring.stage_bytes + 4 * (EPI == GE_GLU ? 3 : 2) * GG_OUT_BYTES;
    auto kernel = gemm_grad_kernel<A_MN, B_MN, EPI, ACT, PAIR>;
    static thread_local int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        if (int rc = allow_smem(kernel, smem, what, 226 * 1024)) return rc;
        configured_dev = dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(GG_THREADS);
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

// M, N, K > 0; all sizes and addresses are ones that a tensor map takes
template <bool A_MN, bool B_MN, int EPI, int ACT = 0>
int grad_gemm(const Operand& a, const Operand& b, const Result& c, GradParams p, cudaStream_t st, const char* what) {
    const int sms = sm_count();
    const Cut cut = p.splits > 1 ? Cut{false, GG_BN} : tile_columns(p.M, p.N, p.second, EPI == GE_GLU);
    const bool pair = cut.pair;
    p.bn = cut.bn;
    p.ring = grad_ring(pair, EPI == GE_GLU, p.bn);
    const int columns = EPI == GE_GLU ? p.bn / 2 : p.bn, tiles_n = (p.N + columns - 1) / columns;
    const uint32_t n_box = EPI == GE_GLU || pair ? p.bn / 2 : p.bn;
    GradMaps m;
    auto map = [&](CUtensorMap* out, const void* base, long long ld, bool mn, int extent, uint32_t box_rows) {
        const uint64_t dims[2] = {(uint64_t)(mn ? extent : p.K), (uint64_t)(mn ? p.K : extent)}, strides[1] = {(uint64_t)ld * 2};
        const uint32_t box[2] = {64, mn ? 64 : box_rows};
        return make_tensor_map(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    if (int rc = map(&m.a0, a.p0, a.ld, A_MN, p.M, GG_BM)) return rc;
    if (int rc = map(&m.b0, b.p0, b.ld, B_MN, p.N, n_box)) return rc;
    m.a1 = m.a0;
    m.b1 = m.b0;
    if (a.p1)
        if (int rc = map(&m.a1, a.p1, a.ld, A_MN, p.M, GG_BM)) return rc;
    if (b.p1)
        if (int rc = map(&m.b1, b.p1, b.ld, B_MN, p.N, n_box)) return rc;
    if (p.splits < 1) p.splits = 1, p.k_per_split = 1 << 30;
    m.c0 = m.c1 = m.c2 = m.a0;
    if (EPI == GE_PARTIAL) {
        const uint64_t dims[3] = {(uint64_t)p.N, (uint64_t)p.M, (uint64_t)p.splits}, strides[2] = {(uint64_t)p.N * 4, (uint64_t)p.M * p.N * 4};
        const uint32_t box[3] = {32, 32, 1};
        if (int rc = make_tensor_map(&m.c0, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, c.p0, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    } else if (EPI != GE_LOSS) {
        CUtensorMap* to[3] = {&m.c0, &m.c1, &m.c2};
        void* const base[3] = {c.p0, c.p1, c.p2};
        for (int i = 0; i < 3; ++i) {
            if (!base[i]) continue;
            const uint64_t dims[2] = {(uint64_t)p.N, (uint64_t)p.M}, strides[1] = {(uint64_t)c.ld * 2};
            const uint32_t box[2] = {64, 32};
            if (int rc = make_tensor_map(to[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base[i], dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
        }
    }
    const int tile_m = pair ? 2 * GG_BM : GG_BM, places = pair ? sms / 2 : sms;
    const long long items = (long long)((p.M + tile_m - 1) / tile_m) * tiles_n * (p.second == SECOND_M ? 2 : 1) * p.splits;
    if (items > INT32_MAX / 2) return fail(BN_ERR_UNSUPPORTED, "%s: %lld tiles", what, items);
    const unsigned grid = (unsigned)(items < places ? items : places) * (pair ? 2 : 1);
    return pair ? grad_run<A_MN, B_MN, EPI, ACT, true>(m, p, grid, st, what) : grad_run<A_MN, B_MN, EPI, ACT, false>(m, p, grid, st, what);
}

// Ranges of K for a product of few tiles: about one work item for every SM, none shorter than 4 steps of 64
void grad_splits(int M, int N, int K_steps, int* splits, int* per) {
    const long long tiles = (long long)((M + GG_BM - 1) / GG_BM) * ((N + GG_BN - 1) / GG_BN), sms = sm_count();
    long long want = tiles * 2 > sms ? 1 : sms / tiles;
    if (want > K_steps / 4) want = K_steps / 4 > 0 ? K_steps / 4 : 1;
    *per = (int)((K_steps + want - 1) / want);
    *splits = (K_steps + *per - 1) / *per;
}

int steps_of(int K) { return (K + GG_BK - 1) / GG_BK; }
size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// c (M, N) = a0 (M, K) b0 (K, N) [+ a1 b1] in `pieces` launches that this is number `piece` of; partial: room for the ranges' sums
size_t nn_bytes(int M, int N, int K_steps, bool pieces) {
    int splits, per;
    grad_splits(M, N, K_steps, &splits, &per);
    return splits > 1 || pieces ? up256((size_t)splits * M * N * 4) : 0;
}
int nn_sum(const float* partial, void* c, int M, int N, int splits, const float* factor, cudaStream_t st, const char* what) {
    const long long groups = (long long)M * N / 4;
    launch_dependent(grad_sum_kernel, (unsigned)((groups + 127) / 128), 128, 0, st, partial, static_cast<__nv_bfloat16*>(c), groups, splits, factor);
    return launch_status(what);
}
int nn_product(const Operand& a, const Operand& b, void* c, int M, int N, int K, int second, float* partial, int* error_word, cudaStream_t st, const char* what) {
    GradParams p{};
    p.M = M; p.N = N; p.K = K; p.second = second; p.error_word = error_word;
    grad_splits(M, N, steps_of(K) * (second == SECOND_K ? 2 : 1), &p.splits, &p.k_per_split);
    if (p.splits == 1) return grad_gemm<false, true, GE_STORE>(a, b, {c, nullptr, nullptr, N}, p, st, what);
    if (int rc = grad_gemm<false, true, GE_PARTIAL>(a, b, {partial, nullptr, nullptr, N}, p, st, what)) return rc;
    return nn_sum(partial, c, M, N, p.splits, nullptr, st, what);
}

int tn_product(const Operand& a, const Operand& b, void* c0, void* c1, int M, int N, int K, int* error_word, cudaStream_t st, const char* what,
               const float* factor = nullptr) {
    GradParams p{};
    p.M = M; p.N = N; p.K = K; p.second = c1 ? SECOND_M : SECOND_NONE; p.error_word = error_word; p.factor = factor;
    return grad_gemm<true, true, GE_STORE>(a, b, {c0, c1, nullptr, N}, p, st, what);
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
// L2 holds, but never fewer than 4096 columns: every piece reads and writes the rows' fp32 gradients again (rows x hidden x 8 bytes
// against 6 x rows x 4096 x hidden operations: a tenth of the products' time).
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
    if (vocab > INT32_MAX - 256) return fail(BN_ERR_UNSUPPORTED, "%s: vocab=%d", what, vocab);
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
extern "C" size_t bn_gemm_bf16_nn_workspace_bytes(int M, int N, int K) { return M > 0 && N > 0 && K > 0 ? nn_bytes(M, N, steps_of(K), false) : 0; }

static int check_product(const char* what, const void* a, const void* b, const void* c, int M, int N, int K, int inner_a) {
    if ((M > 0 && N > 0 && !c) || (M > 0 && K > 0 && !a) || (N > 0 && K > 0 && !b)) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (M < 0 || N < 0 || K < 0) return fail(BN_ERR_INVALID_ARG, "%s: bad shape M=%d N=%d K=%d", what, M, N, K);
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
    return nn_product({a, nullptr, K}, {b, nullptr, N}, c, M, N, K, SECOND_NONE, static_cast<float*>(workspace), error_word,
                      as_stream(stream), what);
}

extern "C" int bn_gemm_bf16_tn(const void* a, const void* b, void* c, int M, int N, int K, int* error_word, bn_stream_t stream) {
    const char* what = "bn_gemm_bf16_tn";
    if (int rc = check_product(what, a, b, c, M, N, K, M)) return rc;
    if (M == 0 || N == 0) return BN_OK;
    if (K == 0) return zero(c, (size_t)M * N * 2, as_stream(stream), what);
    return tn_product({a, nullptr, M}, {b, nullptr, N}, c, nullptr, M, N, K, error_word, as_stream(stream), what);
}

// ------------------------------------------------------------------------------------------------- loss over the vocabulary
extern "C" size_t bn_linear_cross_entropy_bf16_workspace_bytes(int rows, int vocab, int hidden) {
    if (rows <= 0 || vocab <= 0 || hidden <= 0) return 0;
    const int columns = tile_columns(rows, vocab, SECOND_NONE, false).bn;
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
    const int columns = tile_columns(rows, vocab, SECOND_NONE, false).bn, tiles = (vocab + columns - 1) / columns;
    GradParams p{};
    p.M = rows; p.N = vocab; p.K = hidden; p.error_word = error_word;
    p.targets = targets;
    p.stats = static_cast<float2*>(workspace);
    p.picked = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + up256((size_t)tiles * rows * sizeof(float2)));
    cudaStream_t st = as_stream(stream);
    if (int rc = grad_gemm<false, false, GE_LOSS>({x, nullptr, hidden}, {weight_t, nullptr, hidden}, {}, p, st, what)) return rc;
    launch_dependent(loss_join_kernel, (unsigned)((rows + 31) / 32), 32 * GG_JOIN, 0, st, (const float2*)p.stats, (const float*)p.picked, targets, loss, lse, id_error,
                     rows, tiles, vocab);
    return launch_status(what);
}

extern "C" size_t bn_linear_cross_entropy_backward_bf16_workspace_bytes(int rows, int vocab, int hidden) {
    if (rows <= 0 || vocab <= 0 || hidden <= 0) return 0;
    const int columns = piece_columns(rows, vocab);
    return up256((size_t)rows * columns * 2) + nn_bytes(rows, hidden, steps_of(columns < vocab ? columns : vocab), columns < vocab);
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
    float* partial = reinterpret_cast<float*>(ws + up256((size_t)rows * columns * 2));
    int splits = 1, per = 1 << 30;
    grad_splits(rows, hidden, steps_of(columns < vocab ? columns : vocab), &splits, &per);
    const bool sums = splits > 1 || columns < vocab;
    for (int v0 = 0; v0 < vocab; v0 += columns) {
        const int n = vocab - v0 < columns ? vocab - v0 : columns;
        const void* w = static_cast<const __nv_bfloat16*>(weight_t) + (size_t)v0 * hidden;
        GradParams p{};
        p.M = rows; p.N = n; p.K = hidden; p.error_word = error_word;
        p.targets = targets; p.first_column = v0; p.vocab = vocab; p.lse = lse; p.grad = grad_loss;
        if (int rc = grad_gemm<false, false, GE_DLOGITS>({x, nullptr, hidden}, {w, nullptr, hidden}, {ws, nullptr, nullptr, columns}, p, st, what)) return rc;
        if (dx) {
            GradParams q{};
            q.M = rows; q.N = hidden; q.K = n; q.error_word = error_word; q.factor = grad_loss;
            const Operand dz{ws, nullptr, columns}, wt{w, nullptr, hidden};
            if (sums) {
                // a last, shorter piece leaves ranges without a step: they are not launched, and what they have so far stays
                q.k_per_split = per;
                q.splits = (steps_of(n) + per - 1) / per;
                q.add = v0 > 0;
                if (int rc = grad_gemm<false, true, GE_PARTIAL>(dz, wt, {partial, nullptr, nullptr, hidden}, q, st, what)) return rc;
            } else if (int rc = grad_gemm<false, true, GE_STORE>(dz, wt, {dx, nullptr, nullptr, hidden}, q, st, what)) {
                return rc;
            }
        }
        if (dweight_t)
            if (int rc = tn_product({ws, nullptr, columns}, {x, nullptr, hidden}, static_cast<__nv_bfloat16*>(dweight_t) + (size_t)v0 * hidden, nullptr, n,
                                    hidden, rows, error_word, st, what, grad_loss))
                return rc;
    }
    return dx && sums ? nn_sum(partial, dx, rows, hidden, splits, grad_loss, st, what) : BN_OK;
}

// --------------------------------------------------------------------------------------------- gated feed-forward block
// h, dgate and dup (bf16); dh and, when that has been used, the sums of dx (fp32): dh rounded to bf16 would add half of the error that the
// gradients have from their own roundings (2.9e-3 instead of 2.4e-3), and its ranges of K are added where it is read
extern "C" size_t bn_gated_ff_backward_bf16_workspace_bytes(int rows, int hidden, int inter) {
    if (rows <= 0 || hidden <= 0 || inter <= 0) return 0;
    const size_t a = nn_bytes(rows, inter, steps_of(hidden), true), b = nn_bytes(rows, hidden, 2 * steps_of(inter), false);
    return 3 * up256((size_t)rows * inter * 2) + (a > b ? a : b);
}

extern "C" int bn_gated_ff_backward_bf16(const void* dy, const void* x, const void* gate_t, const void* up_t, const void* down_t, void* dx, void* dgate_t,
                                         void* dup_t, void* ddown_t, int rows, int hidden, int inter, int act, void* workspace, size_t workspace_bytes,
                                         int* error_word, bn_stream_t stream) {
    const char* what = "bn_gated_ff_backward_bf16";
    if (!gate_t || !up_t || !down_t || !dgate_t || !dup_t || !ddown_t || (rows > 0 && (!dy || !x || !dx))) return fail(BN_ERR_INVALID_ARG, "%s: null pointer", what);
    if (rows < 0 || hidden <= 0 || inter <= 0) return fail(BN_ERR_INVALID_ARG, "%s: bad shape rows=%d hidden=%d inter=%d", what, rows, hidden, inter);
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
    GradParams q{};
    q.M = rows; q.N = inter; q.K = hidden; q.error_word = error_word;
    grad_splits(rows, inter, steps_of(hidden), &q.splits, &q.k_per_split);
    if (int rc = grad_gemm<false, true, GE_PARTIAL>({dy, nullptr, hidden}, {down_t, nullptr, inter}, {partial, nullptr, nullptr, inter}, q, st, what)) return rc;
    // gate and up again; their gradients, and the product of the forward pass
    GradParams p{};
    p.M = rows; p.N = inter; p.K = hidden; p.error_word = error_word;
    p.dh = partial;
    p.dh_parts = q.splits;
    const Operand xr{x, nullptr, hidden}, weights{gate_t, up_t, hidden};
    const Result three{h, dg, du, inter};
    if (int rc = act == BN_ACT_SILU ? grad_gemm<false, false, GE_GLU, BN_ACT_SILU>(xr, weights, three, p, st, what)
                                    : grad_gemm<false, false, GE_GLU, BN_ACT_GELU_TANH>(xr, weights, three, p, st, what))
        return rc;
    // dx = dgate Wgate + dup Wup, one product of twice the K
    if (int rc = nn_product({dg, du, inter}, {gate_t, up_t, hidden}, dx, rows, hidden, inter, SECOND_K, partial, error_word, st, what)) return rc;
    if (int rc = tn_product({dg, du, inter}, {x, nullptr, hidden}, dgate_t, dup_t, inter, hidden, rows, error_word, st, what)) return rc;
    return tn_product({dy, nullptr, hidden}, {h, nullptr, inter}, ddown_t, nullptr, hidden, inter, rows, error_word, st, what);
}
