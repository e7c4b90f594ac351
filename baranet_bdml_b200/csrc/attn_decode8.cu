// Single-token decode attention over the 8-bit paged cache (kv8.cuh), HBM bound:
//     s_t = scale <RoPE(q), K_t> ks_t,   p = softmax(s),   out = sum_t p_t vs_t V_t,   lse = log sum exp s
//
// The schedule, the ring of stages and the merge are those of attn_decode.cu (decode_schedule.cuh): one persistent CTA per SM takes an
// equal share of all 256-token stages, a producer warp fills a ring of shared memory, eight consumer warps take two pages of a stage
// each, a tenth warp merges what several CTAs hold.  What 8 bits change:
//   * A block (page, key head) is one bulk copy of 2112 bytes, scales included: no tensor map.
//   * Both products are m16n8k16 MMAs of fp16, which holds every e4m3 and int8 number exactly:
//       S^T (16 tokens x 8 heads) = K (16 x 64) Q^T,     O^T (64 x 8 heads) += V^T (64 x 16 tokens) P^T.
//     The sum over k may run in any order, so a lane reads 16 bytes of a key's row at once (dims 16 c .. 16 c + 15 are its k's of all
//     four MMAs) and q is laid out to match; V goes through ldmatrix.trans as pairs of bytes, which a byte permutation turns into
//     pairs of tokens.  Two bytes become two fp16 by one conversion (e4m3) or two operations (int8).
//   * q is rounded to fp16 as a multiple of a power of two that brings the head's largest element to 2^14 (a relative error of 2^-11; the
//     2^28 below that keep it).
//   * A token's value scale goes into its weight: p' = 2^(s - m) vs, with m the running maximum of s + log2 vs, not of s.  So p' is
//     never above 2^8 and the tokens that count most in the result have the most bits of fp16, however far scales and weights are
//     apart (2^-11 for 22 binades).  The sum of weights l runs in fp32 without vs; s - m + 8 is at most 98 (log2 vs counts as -90 at
//     least), so it leaves no room for an overflow below 2^29 tokens.
#include "decode_schedule.cuh"
#include "kv8.cuh"

namespace bn {

constexpr int DEC8_STAGE_TOKENS = 256;
constexpr int DEC8_PAGES = DEC8_STAGE_TOKENS / BN_PAGE_TOKENS;       // of a stage
constexpr int DEC8_STAGE_BYTES = DEC8_PAGES * BN_KV8_BLOCK;          // 33792
constexpr int DEC8_NSTAGES = 6;
constexpr int DEC8_CWARPS = 8;                                       // consumer warps
constexpr int DEC8_PPW = DEC8_PAGES / DEC8_CWARPS;                   // pages per warp and stage
constexpr int DEC8_CTHREADS = DEC8_CWARPS * 32;
constexpr int DEC8_PWARPS = 4;                                       // producer warps
constexpr int DEC8_PPP = DEC8_PAGES / DEC8_PWARPS;                   // pages per producer warp and stage
constexpr int DEC8_THREADS = (DEC8_CWARPS + DEC8_PWARPS + 1) * 32;   // + combine warp
constexpr int DEC8_SMEM_BYTES = DEC8_NSTAGES * DEC8_STAGE_BYTES + 128;
constexpr int DEC8_DEFAULT_MIN_TOKENS = 1024;                        // a CTA's range is never shorter than this
constexpr int DEC8_WHOLE_MAX_STAGES = 8;                             // sequences up to this many stages are never split (if there are enough)
constexpr float DEC8_HEADROOM = 8.f;                                 // p' <= 2^8
static_assert(DEC8_CTHREADS == DEC_G * DEC_D / 2, "a thread per head and two dimensions where warps are merged");

struct Decode8Params {
    const __nv_bfloat16* q;
    const uint8_t* pool;
    int64_t pool_pages;
    const int32_t *page_table, *seq_lens, *q_positions;
    __nv_bfloat16* out;
    float *out_f32, *lse;
    DecodeHeader* hdr;
    int* tickets;
    float *part_m, *part_l, *part_o;
    int B, Hq, Hkv, n_rep, max_pages, max_seq_len, min_stages, max_parts, rope_q;
    float scale_log2;
    RotationFreqs freqs;
};

template <int VALUES> __global__ void __launch_bounds__(DEC8_THREADS, 1) decode8_kernel(const __grid_constant__ Decode8Params p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[DEC8_NSTAGES];
    __shared__ __align__(8) uint64_t empty_bar[DEC8_NSTAGES];
    __shared__ __align__(8) uint64_t merge_bar, part_bar;
    __shared__ int s_prefix[DEC_MAX_SEQS + 1];
    __shared__ int s_len[DEC_MAX_SEQS];
    __shared__ int s_nmax;                      // stages of the longest sequence
    __shared__ float mrg_m[DEC8_CWARPS][DEC_G], mrg_l[DEC8_CWARPS][DEC_G];
    __shared__ __align__(16) float mrg_o[DEC8_CWARPS][DEC_G][DEC_D + 2];   // written and read as float2
    __shared__ __align__(16) uint32_t s_q[DEC_G][3 * DEC_D / 4]; // rotated query heads of the current segment: three e4m3 parts, or fp16
    constexpr uint32_t QUERY_TOP = VALUES == BN_KV8_E4M3 ? 7 : 14;
    __shared__ float s_factor[DEC_G];                           // scale * log2(e) * what q was divided by
    __shared__ int s_abort;

    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t ring = (smem_u32(smem_raw) + 127u) & ~127u;

    if (tid == 0) {
        for (int s = 0; s < DEC8_NSTAGES; ++s) {
            mbar_init(smem_u32(&full_bar[s]), DEC8_PWARPS);
            mbar_init(smem_u32(&empty_bar[s]), DEC8_CWARPS);
        }
        mbar_init(smem_u32(&merge_bar), DEC8_CWARPS);
        mbar_init(smem_u32(&part_bar), DEC8_CWARPS);
        s_abort = 0;
        fence_mbar_init();
    }
    grid_dependency_wait();
    grid_launch_dependents();
    decode_prefix<DEC8_THREADS, DEC8_STAGE_TOKENS>(p.seq_lens, p.B, p.max_seq_len, s_len, s_prefix, &s_nmax);

    Schedule sc;
    sc.prefix = s_prefix;
    sc.len = s_len;
    sc.Hkv = p.Hkv;
    sc.B = p.B;
    sc.T = p.Hkv * s_prefix[p.B];
    sc.whole = s_nmax <= DEC8_WHOLE_MAX_STAGES && p.B * p.Hkv >= 16;
    sc.G = sc.whole ? min((int)gridDim.x, p.B * p.Hkv) : max(1, min((int)gridDim.x, sc.T / p.min_stages));
    const bool active = sc.T > 0 && (int)blockIdx.x < sc.G;
    const int range_lo = active ? sc.range_begin(blockIdx.x) : 0;
    const int range_hi = active ? sc.range_begin(blockIdx.x + 1) : 0;

    if (warp >= DEC8_CWARPS && warp < DEC8_CWARPS + DEC8_PWARPS) {
        // ------------------------------------------------------------ producer
        // page numbers are read two stages (a 128-byte line of the table) at a time, one such group ahead of their use
        constexpr int GRP = 32 / DEC8_PAGES;
        const int mine = (warp - DEC8_CWARPS) * DEC8_PPP + lane % DEC8_PPP;      // the lane's page of a stage
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true, bad = false;
        SegmentIter iter;
        iter.init(range_lo, range_hi);
        Segment sg, sg_next;
        bool have = iter.next(sc, sg, false);
        auto load_group = [&](const Segment& sgm, int grp) {
            const int e = grp * 32 + lane;
            const int n_pages_seq = (sgm.L + BN_PAGE_TOKENS - 1) / BN_PAGE_TOKENS;
            return e < n_pages_seq ? p.page_table[(size_t)sgm.b * p.max_pages + e] : 0;
        };
        const uint64_t stream_policy = l2_policy_evict_first();     // every cache byte is read once per launch
        int ids = have ? load_group(sg, sg.s0 / GRP) : 0, ids_pref = 0;
        while (ok && have) {
            const bool have_next = iter.next(sc, sg_next, false);
            const int n_pages_seq = (sg.L + BN_PAGE_TOKENS - 1) / BN_PAGE_TOKENS;
            for (int s = sg.s0; s < sg.s1; ++s) {
                if (s == sg.s0 || s % GRP == 0) {
                    if (s != sg.s0) ids = ids_pref;
                    const int grp = s / GRP;
                    if ((grp + 1) * GRP < sg.s1) ids_pref = load_group(sg, grp + 1);
                    else if (have_next) ids_pref = load_group(sg_next, sg_next.s0 / GRP);
                }
                int page = __shfl_sync(0xffffffffu, ids, (s % GRP) * DEC8_PAGES + mine);
                if (page < 0 || page >= p.pool_pages) { page = 0; bad = true; }
                if (!mbar_wait(smem_u32(&empty_bar[stage]), phase ^ 1u, &s_abort)) { ok = false; break; }
                const int npages = max(0, min(DEC8_PPP, n_pages_seq - s * DEC8_PAGES - (warp - DEC8_CWARPS) * DEC8_PPP));
                const uint32_t fb = smem_u32(&full_bar[stage]);
                if (lane == 0) mbar_arrive_expect_tx(fb, (uint32_t)npages * BN_KV8_BLOCK);
                __syncwarp();
                if (lane < npages)
                    bulk_load_hint(ring + stage * DEC8_STAGE_BYTES + mine * BN_KV8_BLOCK,
                                   p.pool + ((int64_t)page * p.Hkv + sg.g) * BN_KV8_BLOCK, BN_KV8_BLOCK, fb, stream_policy);
                if (++stage == DEC8_NSTAGES) { stage = 0; phase ^= 1u; }
            }
            sg = sg_next;
            ids = ids_pref;
            have = have_next;
        }
        if (bad) atomicExch(&p.hdr->error, BN_ERR_INVALID_ARG);
        if (lane == 0 && s_abort) atomicExch(&p.hdr->error, BN_ERR_TIMEOUT);
        return;
    }

    if (warp == DEC8_CWARPS + DEC8_PWARPS) {
        // -------------------------------------------------------- combine warp
        SegmentIter iter;
        iter.init(range_lo, range_hi);
        Segment sg;
        uint32_t pphase = 0;
        while (iter.next(sc, sg)) {
            if (sg.n_parts == 1) continue;
            if (!mbar_wait(smem_u32(&part_bar), pphase, &s_abort)) break;
            pphase ^= 1u;
            decode_combine(p, sg, lane);
        }
        if (lane == 0 && s_abort) atomicExch(&p.hdr->error, BN_ERR_TIMEOUT);
        return;
    }

    // --------------------------------------------------------------- consumers
    // where the heads' 64 results are laid over the consumers: a warp has a head, a lane two dimensions
    const int td = 2 * lane;
    // sequences without tokens get a zero output from whoever passes by
    for (int bgi = blockIdx.x; bgi < p.B * p.Hkv; bgi += gridDim.x) {
        const int b = bgi / p.Hkv, g = bgi % p.Hkv;
        if (sc.nst(b) > 0 || warp >= p.n_rep) continue;
        const size_t row = (size_t)b * p.Hq + (size_t)g * p.n_rep + warp;
        if (p.out) *reinterpret_cast<uint32_t*>(p.out + row * DEC_D + td) = 0u;
        if (p.out_f32) *reinterpret_cast<float2*>(p.out_f32 + row * DEC_D + td) = make_float2(0.f, 0.f);
        if (p.lse && lane == 0) p.lse[row] = -INFINITY;
    }

    int stage = 0;
    uint32_t phase = 0, mphase = 0;
    const int hA = 2 * (lane % 4);       // the two heads whose softmax state this thread carries
    const uint32_t mb = smem_u32(&merge_bar);
    auto group_sync = [&]() -> bool {
        __syncwarp();
        if (lane == 0) mbar_arrive(mb);
        const bool ok = mbar_wait_warp(mb, mphase, &s_abort);
        mphase ^= 1u;
        return ok;
    };
    auto load_q_raw = [&](const Segment& sg) -> uint32_t {
        if (warp >= p.n_rep) return 0u;
        return *reinterpret_cast<const uint32_t*>(p.q + ((size_t)sg.b * p.Hq + (size_t)sg.g * p.n_rep + warp) * DEC_D + 2 * lane);
    };
    auto store_q = [&](const Segment& sgq, uint32_t raw) {
        float x0 = bf16_lo(raw), x1 = bf16_hi(raw);
        if (p.rope_q) {
            float c, s;
            rotation(p.q_positions ? p.q_positions[sgq.b] : sgq.L - 1, p.freqs.f[lane], &c, &s);
            const float y0 = x0 * c - x1 * s;
            const float y1 = x0 * s + x1 * c;
            x0 = y0; x1 = y1;
        }
        const uint32_t most = __reduce_max_sync(0xffffffffu, max(__float_as_uint(x0) & 0x7fffffffu, __float_as_uint(x1) & 0x7fffffffu));
        const uint32_t e = max(most >> 23, 30u);
        const float up = __uint_as_float((254u + QUERY_TOP - e) << 23);        // the head's largest magnitude to 2^QUERY_TOP and above
        x0 *= up;
        x1 *= up;
        if (VALUES == BN_KV8_E4M3) {
#pragma unroll
            for (int part = 0; part < 3; ++part) {
                uint16_t two;
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(x1), "f"(x0));
                reinterpret_cast<uint16_t*>(&s_q[warp][part * (DEC_D / 4)])[lane] = two;
                uint32_t back;
                asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(two));
                const float2 f = halves_to_floats(back);
                x0 -= f.x;
                x1 -= f.y;
            }
        } else {
            reinterpret_cast<uint32_t*>(s_q[warp])[lane] = pack_f16(x0, x1);
        }
        if (lane == 0) s_factor[warp] = p.scale_log2 * (e == 255u ? NAN : __uint_as_float((e - QUERY_TOP) << 23));     // (an infinity would saturate)
    };

    SegmentIter iter;
    iter.init(range_lo, range_hi);
    Segment sg, sg_next;
    bool have = iter.next(sc, sg);
    bool ok = true;
    if (have) {
        store_q(sg, load_q_raw(sg));
        ok = group_sync();
    }
    while (ok && have) {
        // look one segment ahead so that its query is already on the way
        const bool have_next = iter.next(sc, sg_next);
        const uint32_t q_raw_next = have_next ? load_q_raw(sg_next) : 0u;
        // Q^T fragments: dims 16 c .. 16 c + 15 of head lane / 4, c = lane % 4
        uint32_t qb[VALUES == BN_KV8_E4M3 ? 12 : 8];
#pragma unroll
        for (int i = 0; i < (VALUES == BN_KV8_E4M3 ? 3 : 2); ++i) {
            // (a part's 16 elements are one 16-byte piece of e4m3, or half of the two pieces of fp16)
            const uint4 a = VALUES == BN_KV8_E4M3 ? *reinterpret_cast<const uint4*>(&s_q[lane / 4][i * (DEC_D / 4) + 4 * (lane % 4)])
                                                  : *reinterpret_cast<const uint4*>(&s_q[lane / 4][8 * (lane % 4) + 4 * i]);
            qb[4 * i] = a.x; qb[4 * i + 1] = a.y; qb[4 * i + 2] = a.z; qb[4 * i + 3] = a.w;
        }
        const float fA = s_factor[hA], fB = s_factor[hA + 1];

        // weights are 2^(s - m_run) (times vs for the product): no larger than 2^8 where m_run is renewed, and it is renewed before
        // they pass 2^14
        float m_run[2] = {-INFINITY, -INFINITY}, less[2] = {0.f, 0.f}, l_run[2] = {0.f, 0.f};
        float o[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

        for (int s = sg.s0; s < sg.s1; ++s) {
            if (!mbar_wait_warp(smem_u32(&full_bar[stage]), phase, &s_abort)) { ok = false; break; }
            // tokens of the warp's pages
            const int mine = min(DEC8_STAGE_TOKENS, sg.L - s * DEC8_STAGE_TOKENS) - warp * DEC8_PPW * BN_PAGE_TOKENS;
            if (mine > 0) {
                const uint32_t sbase = ring + stage * DEC8_STAGE_BYTES + warp * DEC8_PPW * BN_KV8_BLOCK;
                // thread owns heads hA, hA + 1 and tokens lane / 4 (+ 8) of each page
                float sv[DEC8_PPW][4], pr[DEC8_PPW][4], vs[DEC8_PPW][2];
                bool renew = m_run[0] == -INFINITY || m_run[1] == -INFINITY;
                const bool ragged = mine < DEC8_PPW * BN_PAGE_TOKENS;
                if (VALUES == BN_KV8_E4M3 && ragged) {
                    // what lies behind the last token may be a NaN, and 0 * NaN must not reach O (whole pages may not have been loaded)
                    for (int e = mine * 4 + lane; e < DEC8_PPW * BN_PAGE_TOKENS * 4; e += 32)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(sbase + (e / 64) * BN_KV8_BLOCK + KV8_V + (e % 64) * 16), "r"(0) : "memory");
                    fence_proxy_async_smem();          // the next copy into this stage comes after
                    __syncwarp();
                }
#pragma unroll
                for (int pi = 0; pi < DEC8_PPW; ++pi) {
                    const uint32_t block = sbase + pi * BN_KV8_BLOCK;
                    const uint32_t row = block + (lane / 4) * KV8_D + (lane % 4) * 16, sc0 = block + KV8_SCALES + (lane / 4) * 4;
                    uint32_t a[4], b[4];
                    lds_v4(row, a);
                    lds_v4(row + 8 * KV8_D, b);
                    const uint32_t s0 = lds(sc0), s1 = lds(sc0 + 32);
#pragma unroll
                    for (int j = 0; j < 4; ++j) sv[pi][j] = 0.f;
                    if (VALUES == BN_KV8_E4M3) {
#pragma unroll
                        for (int part = 0; part < 3; ++part)
#pragma unroll
                            for (int kk = 0; kk < 2; ++kk)
                                mma_e4m3_16832(sv[pi], a[2 * kk], b[2 * kk], a[2 * kk + 1], b[2 * kk + 1], qb[4 * part + 2 * kk], qb[4 * part + 2 * kk + 1]);
                    } else {
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            uint32_t a0, a1, a2, a3;
                            kv8_halves<VALUES>(a[kk], a0, a2);
                            kv8_halves<VALUES>(b[kk], a1, a3);
                            mma_f16_16816(sv[pi], a0, a1, a2, a3, qb[2 * kk], qb[2 * kk + 1]);
                        }
                    }
                    const float k0 = bf16_lo(s0), k1 = bf16_lo(s1);
                    vs[pi][0] = bf16_hi(s0); vs[pi][1] = bf16_hi(s1);
                    sv[pi][0] *= k0 * fA; sv[pi][1] *= k0 * fB; sv[pi][2] *= k1 * fA; sv[pi][3] *= k1 * fB;
                }
                if (ragged) {
#pragma unroll
                    for (int i = 0; i < 2 * DEC8_PPW; ++i)
                        if (lane / 4 + 8 * i >= mine) { sv[i / 2][2 * (i % 2)] = sv[i / 2][2 * (i % 2) + 1] = -INFINITY; vs[i / 2][i % 2] = 0.f; }
                }
#pragma unroll
                for (int pi = 0; pi < DEC8_PPW; ++pi) {
                    float most = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        pr[pi][j] = ex2(sv[pi][j] - less[j & 1]);
                        most = fmaxf(most, pr[pi][j]);
                    }
                    // (2^-86: the sum of weights does without vs, and has to stay a number where vs is very small)
                    renew |= most * fmaxf(fmaxf(vs[pi][0], vs[pi][1]), 1.2924697e-26f) > 16384.f;
                }
                if (__any_sync(0xffffffffu, renew)) {
                    float tmax[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int pi = 0; pi < DEC8_PPW; ++pi)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            tmax[j & 1] = fmaxf(tmax[j & 1], sv[pi][j] + lg2(fmaxf(vs[pi][j >> 1], 8.0779357e-28f)));      // 2^-90
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        tmax[hh] = fmaxf(tmax[hh], __shfl_xor_sync(0xffffffffu, tmax[hh], 4));
                        tmax[hh] = fmaxf(tmax[hh], __shfl_xor_sync(0xffffffffu, tmax[hh], 8));
                        tmax[hh] = fmaxf(tmax[hh], __shfl_xor_sync(0xffffffffu, tmax[hh], 16));
                        const float m_new = fmaxf(m_run[hh], tmax[hh] - DEC8_HEADROOM);
                        less[hh] = m_new == -INFINITY ? 0.f : m_new;
                        const float alpha = ex2(m_run[hh] - less[hh]);
                        m_run[hh] = m_new;
                        l_run[hh] *= alpha;
#pragma unroll
                        for (int i = 0; i < 4; ++i) { o[i][hh] *= alpha; o[i][hh + 2] *= alpha; }
                    }
#pragma unroll
                    for (int pi = 0; pi < DEC8_PPW; ++pi)
#pragma unroll
                        for (int j = 0; j < 4; ++j) pr[pi][j] = ex2(sv[pi][j] - less[j & 1]);
                }
#pragma unroll
                for (int pi = 0; pi < DEC8_PPW; ++pi) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        l_run[j & 1] += pr[pi][j];
                        pr[pi][j] *= vs[pi][j >> 1];
                    }
                    const uint32_t b0 = movmatrix_trans(pack_f16(pr[pi][0], pr[pi][1]));
                    const uint32_t b1 = movmatrix_trans(pack_f16(pr[pi][2], pr[pi][3]));
                    const int tok = (lane % 8) + ((lane / 8) & 1) * 8;
                    const uint32_t vrow = sbase + pi * BN_KV8_BLOCK + KV8_V + tok * KV8_D;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        // matrices: tokens 0-7 and 8-15 of 16 dims, the same of the next 16
                        uint32_t r[4], a0, a1, a2, a3;
                        ldmatrix_x4_trans(vrow + (((half * 2 + (lane / 16)) ^ ((tok >> 1) & 3)) << 4), r[0], r[1], r[2], r[3]);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            kv8_token_pairs<VALUES>(r[2 * i], a0, a1);
                            kv8_token_pairs<VALUES>(r[2 * i + 1], a2, a3);
                            mma_f16_16816(o[half * 2 + i], a0, a1, a2, a3, b0, b1);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&empty_bar[stage]));
            if (++stage == DEC8_NSTAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;

        // ------------------------------------------------ merge the warps
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            l_run[hh] += __shfl_xor_sync(0xffffffffu, l_run[hh], 4);
            l_run[hh] += __shfl_xor_sync(0xffffffffu, l_run[hh], 8);
            l_run[hh] += __shfl_xor_sync(0xffffffffu, l_run[hh], 16);
        }
        if (lane < 4) {
            mrg_m[warp][hA] = m_run[0]; mrg_m[warp][hA + 1] = m_run[1];
            mrg_l[warp][hA] = l_run[0]; mrg_l[warp][hA + 1] = l_run[1];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = i * 16 + 2 * (lane / 4);
            *reinterpret_cast<float2*>(&mrg_o[warp][hA][d]) = make_float2(o[i][0], o[i][2]);
            *reinterpret_cast<float2*>(&mrg_o[warp][hA + 1][d]) = make_float2(o[i][1], o[i][3]);
        }
        if (!group_sync()) break;
        float mstar = -INFINITY;
#pragma unroll
        for (int w = 0; w < DEC8_CWARPS; ++w) mstar = fmaxf(mstar, mrg_m[w][warp]);
        const float ms = mstar == -INFINITY ? 0.f : mstar;
        float lsum = 0.f, acc[2] = {0.f, 0.f};
#pragma unroll
        for (int w = 0; w < DEC8_CWARPS; ++w) {
            const float scl = ex2(mrg_m[w][warp] - ms);
            lsum += mrg_l[w][warp] * scl;
            const float2 po = *reinterpret_cast<const float2*>(&mrg_o[w][warp][td]);
            acc[0] += po.x * scl; acc[1] += po.y * scl;
        }
        const int bgi = sg.b * p.Hkv + sg.g;
        if (sg.n_parts == 1) {
            if (warp < p.n_rep) {
                const size_t row = (size_t)sg.b * p.Hq + (size_t)sg.g * p.n_rep + warp;
                const float inv = lsum > 0.f ? 1.f / lsum : 0.f;
                const float r0 = acc[0] * inv, r1 = acc[1] * inv;
                if (p.out) *reinterpret_cast<uint32_t*>(p.out + row * DEC_D + td) = pack_bf16(r0, r1);
                if (p.out_f32) *reinterpret_cast<float2*>(p.out_f32 + row * DEC_D + td) = make_float2(r0, r1);
                if (p.lse && lane == 0) p.lse[row] = lsum > 0.f ? (mstar + log2f(lsum)) * LN2 : -INFINITY;
            }
        } else {
            const size_t slot = (size_t)bgi * p.max_parts + ((int)blockIdx.x - sg.c_first);
            if (lane == 0) {
                p.part_m[slot * DEC_G + warp] = mstar;
                p.part_l[slot * DEC_G + warp] = lsum;
            }
            *reinterpret_cast<float2*>(p.part_o + (slot * DEC_G + warp) * DEC_D + td) = make_float2(acc[0], acc[1]);
            // hand the partial to the combine warp and go on
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&part_bar));
        }
        // the next segment's query replaces this one's (every warp took its fragments long ago)
        if (have_next) store_q(sg_next, q_raw_next);
        if (!group_sync()) break;              // mrg_* free again, s_q visible
        sg = sg_next;
        have = have_next;
    }
    if (s_abort && lane == 0) atomicExch(&p.hdr->error, BN_ERR_TIMEOUT);
}

}  // namespace bn

using namespace bn;

static int dec8_min_tokens(int chunk_tokens) {
    const int t = chunk_tokens > 0 ? chunk_tokens : DEC8_DEFAULT_MIN_TOKENS;
    return (int)(((int64_t)t + DEC8_STAGE_TOKENS - 1) / DEC8_STAGE_TOKENS) * DEC8_STAGE_TOKENS;   // whole stages
}

extern "C" size_t bn_attn_decode_kv8_workspace_bytes(int B, int Hq, int Hkv, int D, int max_seq_len, int chunk_tokens) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || D != KV8_D || max_seq_len < 0 || chunk_tokens < 0 || chunk_tokens % 128) return 0;
    return decode_layout(B, Hkv, max_seq_len, dec8_min_tokens(chunk_tokens), regular_ticket_slots(Hkv)).total;
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
    if (Hq % Hkv != 0 || Hq / Hkv > DEC_G) return fail(BN_ERR_UNSUPPORTED, "%s: Hq/Hkv=%d/%d (group of 1..8 supported)", what, Hq, Hkv);
    if (B > DEC_MAX_SEQS) return fail(BN_ERR_UNSUPPORTED, "%s: %d sequences in one launch (<= %d supported)", what, B, DEC_MAX_SEQS);
    if ((long long)B * Hkv * (max_seq_len / DEC8_STAGE_TOKENS + 1) > 0x3fffffffLL || max_seq_len > 0x7fffffff - DEC8_STAGE_TOKENS ||
        chunk_tokens > 0x7fffffff - DEC8_STAGE_TOKENS)
        return fail(BN_ERR_UNSUPPORTED, "%s: B * Hkv * max_seq_len is too large for one launch", what);
    if (chunk_tokens < 0 || chunk_tokens % 128) return fail(BN_ERR_INVALID_ARG, "%s: chunk_tokens=%d must be 0 or a multiple of 128", what, chunk_tokens);
    if ((int64_t)max_pages * BN_PAGE_TOKENS < max_seq_len)
        return fail(BN_ERR_INVALID_ARG, "%s: max_pages=%d cannot hold max_seq_len=%d", what, max_pages, max_seq_len);
    if (rope_q && !(theta > 0.f)) return fail(BN_ERR_INVALID_ARG, "%s: theta=%g", what, theta);
    if ((reinterpret_cast<uintptr_t>(pool) & 15) || (reinterpret_cast<uintptr_t>(q) & 7) || (out && (reinterpret_cast<uintptr_t>(out) & 7)) ||
        (out_f32 && (reinterpret_cast<uintptr_t>(out_f32) & 15)))
        return fail(BN_ERR_INVALID_ARG, "%s: pool/q/out buffers must be 16/8/8/16-byte aligned", what);
    if (int rc = require_sm100()) return rc;
    if (B == 0) return BN_OK;
    const int min_tokens = dec8_min_tokens(chunk_tokens);
    const DecodeLayout L = decode_layout(B, Hkv, max_seq_len, min_tokens, regular_ticket_slots(Hkv));
    if (!workspace || workspace_bytes < L.total) return fail(BN_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", what, workspace_bytes, L.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(BN_ERR_INVALID_ARG, "%s: workspace must be 256-byte aligned", what);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    Decode8Params p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.pool = static_cast<const uint8_t*>(pool);
    p.pool_pages = pool_pages;
    p.page_table = page_table; p.seq_lens = seq_lens; p.q_positions = q_positions;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.out_f32 = out_f32; p.lse = lse;
    p.hdr = reinterpret_cast<DecodeHeader*>(ws);
    p.tickets = reinterpret_cast<int*>(ws + L.tickets);
    p.part_m = reinterpret_cast<float*>(ws + L.part_m);
    p.part_l = reinterpret_cast<float*>(ws + L.part_l);
    p.part_o = reinterpret_cast<float*>(ws + L.part_o);
    p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.n_rep = Hq / Hkv; p.max_pages = max_pages; p.max_seq_len = max_seq_len;
    p.min_stages = min_tokens / DEC8_STAGE_TOKENS;
    p.max_parts = L.max_parts;
    p.rope_q = rope_q;
    p.scale_log2 = scale * LOG2E;
    if (rope_q) p.freqs = rotation_freqs(theta);

    static thread_local int configured_dev = -1;
    int dev = 0;
    cudaGetDevice(&dev);
    if (configured_dev != dev) {
        cudaError_t e = cudaFuncSetAttribute(decode8_kernel<BN_KV8_E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, DEC8_SMEM_BYTES);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(decode8_kernel<BN_KV8_INT8>, cudaFuncAttributeMaxDynamicSharedMemorySize, DEC8_SMEM_BYTES);
        if (e != cudaSuccess) return fail(BN_ERR_CUDA, "cudaFuncSetAttribute(decode8): %s", cudaGetErrorString(e));
        configured_dev = dev;
    }
    // no more CTAs than ranges of the minimum length can exist
    const long long max_ranges = (long long)B * Hkv * ((max_seq_len + (long long)min_tokens - 1) / min_tokens + 1);
    const int grid = (int)(max_ranges < sm_count() ? (max_ranges > 0 ? max_ranges : 1) : sm_count());
    launch_dependent(values == BN_KV8_E4M3 ? decode8_kernel<BN_KV8_E4M3> : decode8_kernel<BN_KV8_INT8>, (unsigned)grid, DEC8_THREADS, DEC8_SMEM_BYTES,
                     as_stream(stream), p);
    return launch_status(what);
}
