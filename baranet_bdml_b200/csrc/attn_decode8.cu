// Single-token decode attention over the 8-bit paged cache (kv8.cuh), HBM bound:
//     s_t = scale <RoPE(q), K_t> ks_t,   p = softmax(s),   out = sum_t p_t vs_t V_t,   lse = log sum exp s
//
// The schedule is that of attn_decode.cu (decode_schedule.cuh): one persistent CTA per SM takes an equal share of all 256-token stages, as a
// list of segments = (sequence, key head, run of stages).  Half the bytes leave half the time per token, so that what the consumers
// do beside the two products has to go elsewhere:
//   * two producer warps keep a ring of stages filled.  A block (page, key head) is one bulk copy of 2112 bytes, scales included; one
//     warp issues one in 44 ns, two one in 30, and 52 is what DRAM needs for it (4 x 262144 tokens 115 us with one, 91 with two; finding the
//     next segment only behind the first copies starts 0.3 us sooner and streams 3 % slower);
//   * a query warp rotates and converts the next segment's queries while the consumers work on the one before;
//   * eight consumer warps, two groups of four that take stages in turn, four pages of a stage each: with two pages each, whose
//     instruction chains are as long, 95 us instead of 91;
//   * four merger warps, two heads each, join the consumers' (m, l, O) of a segment, write the result or a partial, and, where they hold
//     the last of a (sequence, head)'s partials, join those; buffers are double, so that nobody waits for them.
//     Partials are joined sixteen at a time, a lane having one's (m, l): one round of loads (1 x 16000 tokens 10.8 us; eight at a time 12.3).
//     (Two mergers of four heads: 24.1 -> 24.9 us for 64 sequences of 1024 to 4096 tokens.  Taking the segment that a range's end cuts first, so
//     that its partials are joined before the CTAs end, costs more at the start than it saves at the end: 22.9 -> 24.1 us.)
// Both products are m16n8k16 MMAs of fp16, which holds every e4m3 and int8 number exactly:
//     S^T (16 tokens x 8 heads) = K (16 x 64) Q^T,     O^T (64 x 8 heads) += V^T (64 x 16 tokens) P^T.
//   * The sum over k may run in any order, so a lane reads 16 bytes of a key's row at once (dims 16 c .. 16 c + 15 are its k's of all four
//     MMAs) and q is laid out to match; V goes through ldmatrix.trans as pairs of bytes, which a byte permutation turns into pairs of
//     tokens.  Two bytes become two fp16 by one conversion (e4m3) or two operations (int8).  (Scores by e4m3 MMAs, q in three parts, take
//     fewer instructions and longer: 105 us instead of 97.)
//   * q is rounded to fp16 as a multiple of a power of two that brings the head's largest element to 2^14 (a relative error of 2^-11; the
//     2^28 below that keep it).
//   * A token's value scale goes into its weight: p' = 2^(s - m) vs, with m the running maximum of s + log2 vs - 8, not of s.  So the
//     tokens that count most in the result have the most bits of fp16, however far scales and weights are apart.  m is only renewed
//     when a weight would pass 2^14 (a vote instead of a reduction in every stage).  The sum of weights l runs in fp32 without vs: log2 vs
//     counts as -90 at least there and a weight without vs renews m beyond 2^100, so l has room for 2^27 tokens.
//     fp16 ends at 2^-24: a share 2^-33 below the largest p' (zeros count with 2^-90 there) is lost, which shows only in elements to which
//     all larger tokens add a zero.
//   * Scales lie anywhere in 2^-100 .. 2^122 (zeros have the least), so m may be 98 below the largest score or 114 above it, and rise by far more than
//     126 over weights that still count: l is between 2^-114 and 2^127, but 2^-126 is the least single factor.  Whatever l is multiplied by
//     where m rises or sums are joined is therefore the square of a half power, one factor after the other, and so are the weights themselves
//     where m is renewed, and in every stage from a vs above 2^60 on: below that, a weight that is flushed to 0 is less than 2^-74 of l.  (A second
//     maximum for l alone took 2 to 8 % longer where sequences are short: code, which each launch fetches anew.)  The code has s and m in halves.
#include "decode_schedule.cuh"
#include "kv8.cuh"

namespace bn {

constexpr int DEC8_STAGE_TOKENS = 256;
constexpr int DEC8_PAGES = DEC8_STAGE_TOKENS / BN_PAGE_TOKENS;       // of a stage
constexpr int DEC8_STAGE_BYTES = DEC8_PAGES * BN_KV8_BLOCK;          // 33792
constexpr int DEC8_NSTAGES = 4;
constexpr int DEC8_GROUPS = 2;                                       // groups of consumer warps, which take stages in turn
constexpr int DEC8_GWARPS = 4;                                       // warps of a group
constexpr int DEC8_CWARPS = DEC8_GROUPS * DEC8_GWARPS;
constexpr int DEC8_PPW = DEC8_PAGES / DEC8_GWARPS;                   // pages per warp and stage
constexpr int DEC8_PWARPS = 2;                                       // producers
constexpr int DEC8_PPP = DEC8_PAGES / DEC8_PWARPS;                   // pages per producer warp and stage
constexpr int DEC8_MWARPS = 4;                                       // mergers
constexpr int DEC8_HPM = DEC_G / DEC8_MWARPS;                        // heads per merger
constexpr int DEC8_QUERY_WARP = DEC8_CWARPS + DEC8_PWARPS, DEC8_MERGER = DEC8_QUERY_WARP + 1;
constexpr int DEC8_THREADS = (DEC8_MERGER + DEC8_MWARPS) * 32;
constexpr int DEC8_SMEM_BYTES = DEC8_NSTAGES * DEC8_STAGE_BYTES + 128;
constexpr int DEC8_MAX_CTAS = 256;
constexpr int DEC8_CUT_STAGES = 4;                                   // what a cut segment costs, in stages
// a group has to have waited for every fill of the slots that it reads: with another's fills in between, the parity that it waits for
// may be that of the fill before the last
static_assert(DEC8_NSTAGES % DEC8_GROUPS == 0, "slots belong to groups");

struct Decode8Params {
    const __nv_bfloat16* q;
    const uint8_t* pool;
    int64_t pool_pages;
    const int32_t *page_table, *seq_lens, *q_positions;
    __nv_bfloat16* out;
    float *out_f32, *lse;
    DecodeHeader* hdr;
    int* tickets;                               // [merger][CTA that holds the segment's first part]
    float *part_m, *part_l, *part_o;            // [CTA][0: the segment began before its range, 1: it ends behind it][head] ([dim])
    int B, Hq, Hkv, n_rep, max_pages, max_seq_len, min_stages, rope_q;
    int most_heads;                             // (sequence, key head)s of a CTA that takes whole ones
    float half_scale_log2;
    RotationFreqs freqs;
};

// results of one head (m in halves): lane -> dims 2 * lane, + 1
__device__ __forceinline__ void decode8_store(const Decode8Params& p, size_t row, int lane, float m, float l, float a, float b) {
    const float inv = l > 0.f ? 1.f / l : 0.f;
    if (p.out) *reinterpret_cast<uint32_t*>(p.out + row * DEC_D + 2 * lane) = pack_bf16(a * inv, b * inv);
    if (p.out_f32) *reinterpret_cast<float2*>(p.out_f32 + row * DEC_D + 2 * lane) = make_float2(a * inv, b * inv);
    if (p.lse && lane == 0) p.lse[row] = l == 0.f ? -INFINITY : (2.f * m + log2f(l)) * LN2;
}

// the queries of a key head: lane -> dims 2 * lane, + 1, of each
__device__ __forceinline__ void decode8_query(const Decode8Params& p, int b, int g, int lane, uint32_t (&raw)[DEC_G]) {
    const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q) + ((size_t)b * p.Hq + (size_t)g * p.n_rep) * (DEC_D / 2) + lane;
#pragma unroll
    for (int h = 0; h < DEC_G; ++h) raw[h] = h < p.n_rep ? src[h * (DEC_D / 2)] : 0u;
}

template <int VALUES> __global__ void __launch_bounds__(DEC8_THREADS, 1) decode8_kernel(const __grid_constant__ Decode8Params p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[DEC8_NSTAGES], empty_bar[DEC8_NSTAGES];
    __shared__ __align__(8) uint64_t q_full[2], q_free[2], mrg_full[2], mrg_free[2];
    __shared__ int s_prefix[DEC_MAX_SEQS + 1];
    __shared__ int s_len[DEC_MAX_SEQS];
    __shared__ int s_nmax;                      // stages of the longest sequence
    __shared__ float mrg_m[2][DEC8_CWARPS][DEC_G], mrg_l[2][DEC8_CWARPS][DEC_G];
    __shared__ __align__(16) float mrg_o[2][DEC8_CWARPS][DEC_G][DEC_D + 2];   // written and read as float2
    __shared__ __align__(16) uint32_t s_q[2][DEC_G][DEC_D / 2]; // rotated query heads of a segment, pairs of fp16
    __shared__ float s_factor[2][DEC_G];                        // half of scale * log2(e) * what q was divided by
    __shared__ int s_abort;

    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    const uint32_t ring = (smem_u32(smem_raw) + 127u) & ~127u;

    if (tid == 0) {
        for (int s = 0; s < DEC8_NSTAGES; ++s) {
            mbar_init(smem_u32(&full_bar[s]), DEC8_PWARPS);
            mbar_init(smem_u32(&empty_bar[s]), DEC8_GWARPS);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&q_full[s]), 1);
            mbar_init(smem_u32(&q_free[s]), DEC8_CWARPS);
            mbar_init(smem_u32(&mrg_full[s]), DEC8_CWARPS);
            mbar_init(smem_u32(&mrg_free[s]), DEC8_MWARPS);
        }
        s_abort = 0;
        fence_mbar_init();
    }
    // Where this CTA begins (lane 1: and ends) if it takes whole (sequence, key head)s.  Its page numbers and queries are asked for before the
    // lengths that tell whether it does, and then neither divisions nor a search lie between them and the first copies.
    const int grid = gridDim.x, heads = p.B * p.Hkv, edge_of = (int)((blockIdx.x + lane % 2) * (unsigned)heads / (unsigned)min(grid, heads));
    const int edge_b = edge_of / p.Hkv, edge_g = edge_of - edge_b * p.Hkv, guess = min(__shfl_sync(0xffffffffu, edge_of, 0), heads - 1);
    const int guess_b = guess / p.Hkv, guess_g = guess - guess_b * p.Hkv;
    int guess_ids = 0;
    uint32_t guess_raw[DEC_G];
    grid_dependency_wait();
    grid_launch_dependents();
    if (warp >= DEC8_CWARPS && warp < DEC8_QUERY_WARP && lane < p.max_pages) guess_ids = p.page_table[(size_t)guess_b * p.max_pages + lane];
    if (warp == DEC8_QUERY_WARP) decode8_query(p, guess_b, guess_g, lane, guess_raw);
    decode_prefix<DEC8_THREADS, DEC8_STAGE_TOKENS>(p.seq_lens, p.B, p.max_seq_len, s_len, s_prefix, &s_nmax);

    Schedule sc;
    sc.prefix = s_prefix;
    sc.len = s_len;
    sc.Hkv = p.Hkv;
    sc.B = p.B;
    sc.T = p.Hkv * s_prefix[p.B];
    // whole (sequence, key head)s for every CTA where equal shares would save less than their cuts cost
    sc.whole = (int64_t)p.most_heads * s_nmax * grid <= sc.T + DEC8_CUT_STAGES * grid;
    sc.G = sc.whole ? min(grid, p.B * p.Hkv) : max(1, min(grid, p.min_stages == 1 ? sc.T : sc.T / p.min_stages));
    const bool active = sc.T > 0 && (int)blockIdx.x < sc.G;
    SegmentIter iter;
    int edge = 0;                                      // both ends by one run through the divisions
    if (active && sc.whole) edge = edge_of < heads ? p.Hkv * s_prefix[edge_b] + edge_g * sc.nst(edge_b) : sc.T;
    else if (active) edge = sc.range_begin(blockIdx.x + lane % 2);
    iter.init(__shfl_sync(0xffffffffu, edge, 0), __shfl_sync(0xffffffffu, edge, 1));
    if (sc.whole && sc.nst(guess_b) > 0) iter.start_at(guess_b, guess_g);
    else iter.search_warp(sc);
    Segment sg;

    if (warp >= DEC8_CWARPS && warp < DEC8_QUERY_WARP) {
        // ----------------------------------------------------------- producers
        // page numbers are read two stages (a 128-byte line of the table) at a time, one such group ahead of their use
        constexpr int GRP = 32 / DEC8_PAGES;
        const int first = (warp - DEC8_CWARPS) * DEC8_PPP, mine = first + lane % DEC8_PPP;      // of a stage's pages: the warp's and the lane's
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true, bad = false;
        Segment sg_next;
        bool have = iter.next(sc, sg, false);
        auto load_group = [&](const Segment& sgm, int grp) {
            const int e = grp * 32 + lane;
            const int n_pages_seq = (sgm.L + BN_PAGE_TOKENS - 1) / BN_PAGE_TOKENS;
            return e < n_pages_seq ? p.page_table[(size_t)sgm.b * p.max_pages + e] : 0;
        };
        const uint64_t stream_policy = l2_policy_evict_first();     // every cache byte is read once per launch
        int ids = 0, ids_pref = 0;
        if (have && sg.b == guess_b && sg.s0 < GRP) ids = lane < (sg.L + BN_PAGE_TOKENS - 1) / BN_PAGE_TOKENS ? guess_ids : 0;
        else if (have) ids = load_group(sg, sg.s0 / GRP);
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
                if (!mbar_wait_warp(smem_u32(&empty_bar[stage]), phase ^ 1u, &s_abort)) { ok = false; break; }
                const int npages = max(0, min(DEC8_PPP, n_pages_seq - s * DEC8_PAGES - first));
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

    if (warp == DEC8_QUERY_WARP) {
        // ---------------------------------------------------------- query warp: lane -> dims 2 * lane, + 1, of all heads
        const double freq = p.freqs.f[lane];           // (of 32 different parameters a warp reads one at a time: not in every segment)
        auto position = [&](const Segment& of) { return p.rope_q && p.q_positions ? p.q_positions[of.b] : of.L - 1; };
        uint32_t raw[DEC_G], raw_next[DEC_G];
        int pos = 0, pos_next = 0, known = -1;
        float c = 1.f, s = 0.f;
        bool have = iter.next(sc, sg, false);
        if (have) {
            pos = position(sg);
#pragma unroll
            for (int h = 0; h < DEC_G; ++h) raw[h] = guess_raw[h];
            if (sg.b != guess_b || sg.g != guess_g) decode8_query(p, sg.b, sg.g, lane, raw);
        }
        for (int n = 0; have; ++n) {
            const int buf = n % 2, b = sg.b;
            have = iter.next(sc, sg, false);
            if (have) {                                                // under way while this one is rotated
                pos_next = position(sg);
                decode8_query(p, sg.b, sg.g, lane, raw_next);
            }
            if (p.rope_q && b != known) kv8_rotation(pos, freq, &c, &s);
            known = b;
            if (!mbar_wait_warp(smem_u32(&q_free[buf]), (n / 2 & 1) ^ 1u, &s_abort)) break;
#pragma unroll
            for (int h = 0; h < DEC_G; ++h) {
                const float x0 = bf16_lo(raw[h]), x1 = bf16_hi(raw[h]);
                const float y0 = x0 * c - x1 * s, y1 = x0 * s + x1 * c;
                const uint32_t most = __reduce_max_sync(0xffffffffu, max(__float_as_uint(y0) & 0x7fffffffu, __float_as_uint(y1) & 0x7fffffffu));
                const uint32_t e = max(most >> 23, 30u);
                const float up = __uint_as_float((254u + 14u - e) << 23);              // the largest magnitude to 2^14 and above
                s_q[buf][h][lane] = pack_f16(y0 * up, y1 * up);
                if (lane == 0) s_factor[buf][h] = p.half_scale_log2 * __uint_as_float((e - 14u) << 23);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&q_full[buf]));
            pos = pos_next;
#pragma unroll
            for (int h = 0; h < DEC_G; ++h) raw[h] = raw_next[h];
        }
        if (lane == 0 && s_abort) atomicExch(&p.hdr->error, BN_ERR_TIMEOUT);
        return;
    }

    if (warp >= DEC8_MERGER) {
        // ------------------------------------------------------------- mergers
        const int h0 = (warp - DEC8_MERGER) * DEC8_HPM;
        // sequences without tokens get a zero output from whoever passes by
        for (int bgi = blockIdx.x; bgi < p.B * p.Hkv; bgi += gridDim.x) {
            const int b = bgi / p.Hkv, g = bgi % p.Hkv;
            if (sc.nst(b) > 0) continue;
#pragma unroll
            for (int h = h0; h < h0 + DEC8_HPM; ++h)
                if (h < p.n_rep) decode8_store(p, (size_t)b * p.Hq + (size_t)g * p.n_rep + h, lane, 0.f, 0.f, 0.f, 0.f);
        }
        for (int n = 0; iter.next(sc, sg, true); ++n) {
            const int buf = n % 2;
            if (!mbar_wait_warp(smem_u32(&mrg_full[buf]), n / 2 & 1, &s_abort)) break;
            float m[DEC8_HPM], l[DEC8_HPM], a[DEC8_HPM], b[DEC8_HPM];
#pragma unroll
            for (int i = 0; i < DEC8_HPM; ++i) {
                const int h = h0 + i;
                m[i] = -INFINITY;
#pragma unroll
                for (int w = 0; w < DEC8_CWARPS; ++w) m[i] = fmaxf(m[i], mrg_m[buf][w][h]);
                const float base = m[i] == -INFINITY ? 0.f : m[i];
                l[i] = a[i] = b[i] = 0.f;
#pragma unroll
                for (int w = 0; w < DEC8_CWARPS; ++w) {
                    const float half = ex2(mrg_m[buf][w][h] - base), scl = half * half;
                    const float2 o = *reinterpret_cast<const float2*>(&mrg_o[buf][w][h][2 * lane]);
                    l[i] += mrg_l[buf][w][h] * half * half;
                    a[i] += o.x * scl;
                    b[i] += o.y * scl;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&mrg_free[buf]));
            const size_t row = (size_t)sg.b * p.Hq + (size_t)sg.g * p.n_rep;
            if (sg.n_parts > 1) {
                const int part = ((int)blockIdx.x * 2 + ((int)blockIdx.x == sg.c_first)) * DEC_G;
#pragma unroll
                for (int i = 0; i < DEC8_HPM; ++i) {
                    if (lane == 0) { p.part_m[part + h0 + i] = m[i]; p.part_l[part + h0 + i] = l[i]; }
                    *reinterpret_cast<float2*>(p.part_o + (part + h0 + i) * DEC_D + 2 * lane) = make_float2(a[i], b[i]);
                }
                __threadfence();
                __syncwarp();
                int* ticket = p.tickets + (warp - DEC8_MERGER) * DEC8_MAX_CTAS + sg.c_first;
                int t = 0;
                if (lane == 0) t = atomicAdd(ticket, 1);
                if (__shfl_sync(0xffffffffu, t, 0) != sg.n_parts - 1) continue;
                __threadfence();
                if (lane == 0) *ticket = 0;            // leave the scratch clean for the next launch
                // this CTA stored the last part: joined in the order of the parts, whoever is last
#pragma unroll
                for (int i = 0; i < DEC8_HPM; ++i) { m[i] = -INFINITY; l[i] = a[i] = b[i] = 0.f; }
                constexpr int AHEAD = 16;              // parts whose loads are under way together; a lane has a part's m and l
                for (int c0 = 0; c0 < sg.n_parts; c0 += AHEAD) {
                    float pm[DEC8_HPM], pl[DEC8_HPM];
                    float2 po[AHEAD][DEC8_HPM];
                    const int own = c0 + lane;
                    const bool has = lane < AHEAD && own < sg.n_parts;
                    const int at = ((sg.c_first + (has ? own : 0)) * 2 + (!has || own == 0)) * DEC_G + h0;
#pragma unroll
                    for (int i = 0; i < DEC8_HPM; ++i) {
                        pm[i] = has ? __ldcg(p.part_m + at + i) : -INFINITY;
                        pl[i] = has ? __ldcg(p.part_l + at + i) : 0.f;
                    }
#pragma unroll
                    for (int c = 0; c < AHEAD; ++c)
#pragma unroll
                        for (int i = 0; i < DEC8_HPM; ++i) {
                            const bool on = c0 + c < sg.n_parts;
                            const int e = ((sg.c_first + (on ? c0 + c : 0)) * 2 + (!on || c0 + c == 0)) * DEC_G + h0 + i;
                            po[c][i] = on ? __ldcg(reinterpret_cast<const float2*>(p.part_o + e * DEC_D + 2 * lane)) : make_float2(0.f, 0.f);
                        }
#pragma unroll
                    for (int i = 0; i < DEC8_HPM; ++i) {
                        float top = pm[i];
#pragma unroll
                        for (int o = 1; o < AHEAD; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        top = fmaxf(m[i], __shfl_sync(0xffffffffu, top, 0));
                        const float base = top == -INFINITY ? 0.f : top, keep = ex2(m[i] - base), half = ex2(pm[i] - base), scl = half * half;
                        float sum = pl[i] * half * half;
#pragma unroll
                        for (int o = 1; o < AHEAD; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                        m[i] = top;
                        l[i] = l[i] * keep * keep + __shfl_sync(0xffffffffu, sum, 0);
                        a[i] *= keep * keep; b[i] *= keep * keep;
#pragma unroll
                        for (int c = 0; c < AHEAD; ++c) {
                            const float f = __shfl_sync(0xffffffffu, scl, c);
                            a[i] += po[c][i].x * f;
                            b[i] += po[c][i].y * f;
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < DEC8_HPM; ++i)
                if (h0 + i < p.n_rep) decode8_store(p, row + h0 + i, lane, m[i], l[i], a[i], b[i]);
        }
        if (lane == 0 && s_abort) atomicExch(&p.hdr->error, BN_ERR_TIMEOUT);
        return;
    }

    // --------------------------------------------------------------- consumers
    const int group = warp / DEC8_GWARPS, gwarp = warp % DEC8_GWARPS;
    const int hA = 2 * (lane % 4);       // the two heads whose softmax state this thread carries
    int before = 0;                      // stages of the range that lie before the segment
    bool ok = true;
    for (int n = 0; ok && iter.next(sc, sg, false); ++n) {
        const int buf = n % 2;
        if (!mbar_wait_warp(smem_u32(&q_full[buf]), n / 2 & 1, &s_abort)) break;
        // Q^T fragments: dims 16 c .. 16 c + 15 of head lane / 4, c = lane % 4
        uint32_t qb[8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 a = *reinterpret_cast<const uint4*>(&s_q[buf][lane / 4][8 * (lane % 4) + 4 * i]);
            qb[4 * i] = a.x; qb[4 * i + 1] = a.y; qb[4 * i + 2] = a.z; qb[4 * i + 3] = a.w;
        }
        const float fA = s_factor[buf][hA], fB = s_factor[buf][hA + 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&q_free[buf]));

        float m_run[2] = {-INFINITY, -INFINITY}, less[2] = {0.f, 0.f}, l_run[2] = {0.f, 0.f};
        float o[4][4];
        bool high = false;                             // a vs above 2^60 has been
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.f;

        for (int s = sg.s0 + ((before ^ group) & 1); s < sg.s1; s += DEC8_GROUPS) {
            const int nth = before + s - sg.s0, stage = nth % DEC8_NSTAGES;
            if (!mbar_wait_warp(smem_u32(&full_bar[stage]), (nth / DEC8_NSTAGES) & 1, &s_abort)) { ok = false; break; }
            // tokens of the warp's pages
            const int mine = min(DEC8_STAGE_TOKENS, sg.L - s * DEC8_STAGE_TOKENS) - gwarp * DEC8_PPW * BN_PAGE_TOKENS;
            if (mine > 0) {
                const uint32_t sbase = ring + stage * DEC8_STAGE_BYTES + gwarp * DEC8_PPW * BN_KV8_BLOCK;
                // thread owns heads hA, hA + 1 and tokens lane / 4 (+ 8) of each page
                float sv[DEC8_PPW][4], pr[DEC8_PPW][4], vs[DEC8_PPW][2];
                bool renew = high || m_run[0] == -INFINITY || m_run[1] == -INFINITY;
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
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        uint32_t a0, a1, a2, a3;
                        kv8_halves<VALUES>(a[kk], a0, a2);
                        kv8_halves<VALUES>(b[kk], a1, a3);
                        mma_f16_16816(sv[pi], a0, a1, a2, a3, qb[2 * kk], qb[2 * kk + 1]);
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
                    float most = 1.4210855e-14f;       // 2^-46: a vs above 2^60 renews
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        pr[pi][j] = ex2(fmaf(2.f, sv[pi][j], -2.f * less[j & 1]));
                        most = fmaxf(most, pr[pi][j]);
                    }
                    // (2^-86: the sum of weights does without vs, and has to stay a number where vs is very small)
                    renew |= most * fmaxf(fmaxf(vs[pi][0], vs[pi][1]), 1.2924697e-26f) > 16384.f;
                }
                if (__any_sync(0xffffffffu, renew)) {
                    float tmax[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int pi = 0; pi < DEC8_PPW; ++pi) {
                        high |= fmaxf(vs[pi][0], vs[pi][1]) > 1.1529215e18f;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            tmax[j & 1] = fmaxf(tmax[j & 1], fmaf(0.5f, lg2(fmaxf(vs[pi][j >> 1], 8.0779357e-28f)), sv[pi][j]));      // 2^-90
                    }
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        tmax[hh] = fmaxf(tmax[hh], __shfl_xor_sync(0xffffffffu, tmax[hh], 4));
                        tmax[hh] = fmaxf(tmax[hh], __shfl_xor_sync(0xffffffffu, tmax[hh], 8));
                        tmax[hh] = fmaxf(tmax[hh], __shfl_xor_sync(0xffffffffu, tmax[hh], 16));
                        const float m_new = fmaxf(m_run[hh], tmax[hh] - 4.f);
                        less[hh] = m_new == -INFINITY ? 0.f : m_new;
                        const float half = ex2(m_run[hh] - less[hh]), alpha = half * half;
                        m_run[hh] = m_new;
                        l_run[hh] = l_run[hh] * half * half;
#pragma unroll
                        for (int i = 0; i < 4; ++i) { o[i][hh] *= alpha; o[i][hh + 2] *= alpha; }
                    }
#pragma unroll
                    for (int pi = 0; pi < DEC8_PPW; ++pi)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float half = ex2(sv[pi][j] - less[j & 1]);
                            pr[pi][j] = half * half;
                        }
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
        }
        if (!ok) break;
        before += sg.s1 - sg.s0;

        // hand (m, l, O) to the mergers
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
            l_run[hh] += __shfl_xor_sync(0xffffffffu, l_run[hh], 4);
            l_run[hh] += __shfl_xor_sync(0xffffffffu, l_run[hh], 8);
            l_run[hh] += __shfl_xor_sync(0xffffffffu, l_run[hh], 16);
        }
        if (!mbar_wait_warp(smem_u32(&mrg_free[buf]), (n / 2 & 1) ^ 1u, &s_abort)) break;
        if (lane < 4) {
            mrg_m[buf][warp][hA] = m_run[0]; mrg_m[buf][warp][hA + 1] = m_run[1];
            mrg_l[buf][warp][hA] = l_run[0]; mrg_l[buf][warp][hA + 1] = l_run[1];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = i * 16 + 2 * (lane / 4);
            *reinterpret_cast<float2*>(&mrg_o[buf][warp][hA][d]) = make_float2(o[i][0], o[i][2]);
            *reinterpret_cast<float2*>(&mrg_o[buf][warp][hA + 1][d]) = make_float2(o[i][1], o[i][3]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&mrg_full[buf]));
    }
    if (s_abort && lane == 0) atomicExch(&p.hdr->error, BN_ERR_TIMEOUT);
}

}  // namespace bn

using namespace bn;

// Scratch: the error word, a ticket per merger and CTA, two partial results per CTA (a range cuts two segments at most)
constexpr size_t DEC8_PARTS = (size_t)2 * DEC8_MAX_CTAS * DEC_G;
constexpr size_t DEC8_TICKETS_AT = 256, DEC8_PARTS_AT = DEC8_TICKETS_AT + DEC8_MWARPS * DEC8_MAX_CTAS * sizeof(int);
constexpr size_t DEC8_SCRATCH_BYTES = DEC8_PARTS_AT + DEC8_PARTS * (DEC_D + 2) * sizeof(float);

extern "C" size_t bn_attn_decode_kv8_workspace_bytes(int B, int Hq, int Hkv, int D, int max_seq_len, int chunk_tokens) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || D != KV8_D || max_seq_len < 0 || chunk_tokens < 0 || chunk_tokens % 128) return 0;
    return DEC8_SCRATCH_BYTES;
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
        (long long)B * Hkv > 0x7fffffffLL / DEC8_MAX_CTAS || chunk_tokens > 0x7fffffff - DEC8_STAGE_TOKENS)
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
    if (!workspace || workspace_bytes < DEC8_SCRATCH_BYTES)
        return fail(BN_ERR_WORKSPACE, "%s: workspace of %zu bytes given, %zu needed", what, workspace_bytes, DEC8_SCRATCH_BYTES);
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
    p.tickets = reinterpret_cast<int*>(ws + DEC8_TICKETS_AT);
    p.part_m = reinterpret_cast<float*>(ws + DEC8_PARTS_AT);
    p.part_l = p.part_m + DEC8_PARTS;
    p.part_o = p.part_l + DEC8_PARTS;
    p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.n_rep = Hq / Hkv; p.max_pages = max_pages; p.max_seq_len = max_seq_len;
    p.min_stages = chunk_tokens > DEC8_STAGE_TOKENS ? (chunk_tokens + DEC8_STAGE_TOKENS - 1) / DEC8_STAGE_TOKENS : 1;
    p.rope_q = rope_q;
    p.half_scale_log2 = 0.5f * scale * LOG2E;
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
    const long long min_tokens = (long long)p.min_stages * DEC8_STAGE_TOKENS, ranges = (long long)B * Hkv * ((max_seq_len + min_tokens - 1) / min_tokens + 1);
    const int most = sm_count() < DEC8_MAX_CTAS ? sm_count() : DEC8_MAX_CTAS, grid = (int)(ranges < most ? ranges : most);
    p.most_heads = (int)(((int64_t)B * Hkv + grid - 1) / grid);
    launch_dependent(values == BN_KV8_E4M3 ? decode8_kernel<BN_KV8_E4M3> : decode8_kernel<BN_KV8_INT8>, (unsigned)grid, DEC8_THREADS, DEC8_SMEM_BYTES,
                     as_stream(stream), p);
    return launch_status(what);
}
