// What one-token decode kernels over paged caches share (attn_decode.cu, attn_decode8.cu): how the stages of a launch are cut into
// equal ranges, one per CTA, the partial results of a (sequence, KV head) that several CTAs hold, and their merge.
#pragma once

#include <math.h>

#include "common.cuh"
#include "ptx.cuh"

namespace bn {

using namespace ptx;

constexpr int DEC_D = 64;
constexpr int DEC_G = 8;                    // query heads per KV head served by one MMA (n = 8)
constexpr int DEC_MAX_SEQS = 1024;          // sequences per launch (prefix table in shared memory)
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct DecodeHeader {   // first 256 bytes of the scratch buffer
    int error;          // BN_ERR_TIMEOUT once a bounded wait ran out
};

struct DecodeLayout {
    size_t tickets, part_m, part_l, part_o, total;
    int max_parts;      // partial slots per (sequence, KV head)
};

// `ticket_slots` is the capacity of the ticket region, NOT B * Hkv: the tickets are the only words of the scratch
// that outlive a launch (a merging CTA re-arms the ones it used), so their place must not move with the batch
// size, or a later, larger batch would find its tickets where an earlier call wrote partials.
inline DecodeLayout decode_layout(int B, int Hkv, int max_seq_len, int min_tokens, size_t ticket_slots) {
    DecodeLayout L;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    // a (sequence, head) of n stages overlaps at most n / (min stages per CTA) + 2 CTA ranges
    L.max_parts = (max_seq_len + min_tokens - 1) / min_tokens + 2;
    size_t bg = (size_t)B * Hkv;
    L.tickets = 256;
    L.part_m = L.tickets + up(ticket_slots * sizeof(int));
    L.part_l = L.part_m + up(bg * L.max_parts * DEC_G * sizeof(float));
    L.part_o = L.part_l + up(bg * L.max_parts * DEC_G * sizeof(float));
    L.total = L.part_o + up(bg * L.max_parts * DEC_G * DEC_D * sizeof(float));
    return L;
}

// caller-owned scratch: room for the tickets of the largest batch a launch accepts, whatever B this call has
inline size_t regular_ticket_slots(int Hkv) { return (size_t)DEC_MAX_SEQS * Hkv; }

// The launch-wide schedule, derived from seq_lens by every thread of every CTA.
struct Schedule {
    const int* prefix;     // shared memory: prefix[b] = sum of stages of sequences < b (one KV head)
    const int* len;        // shared memory: clamped sequence lengths
    int Hkv, B;
    int T;                 // all stages of the launch (< 2^31)
    int G;                 // CTAs that take part
    bool whole;            // short sequences: a CTA takes whole (sequence, KV head) segments, nothing is split
    __device__ __forceinline__ int nst(int b) const { return prefix[b + 1] - prefix[b]; }
    // 32-bit division whenever the products fit (G <= 2^9 CTAs, T < 2^22 stages): the 64-bit form is an emulated
    // sequence several times longer, and these sit on the path to the first TMA load
    __device__ __forceinline__ bool small() const { return T < (1 << 22) && G <= (1 << 9); }
    __device__ __forceinline__ int range_begin(int cta) const {
        if (whole) {
            // segments [cta * n / G, (cta + 1) * n / G) of the n = B * Hkv segments, in (sequence, head) order
            const int n = B * Hkv, k = (int)((unsigned)cta * (unsigned)n / (unsigned)G);
            if (k >= n) return T;
            const int b = k / Hkv;
            return Hkv * prefix[b] + (k - b * Hkv) * nst(b);
        }
        return small() ? (int)((unsigned)cta * (unsigned)T / (unsigned)G) : (int)((long long)cta * T / G);
    }
    // the CTA whose range holds global stage x
    __device__ __forceinline__ int cta_of(int x) const {
        return small() ? (int)((((unsigned)x + 1u) * (unsigned)G - 1u) / (unsigned)T)
                       : (int)((((long long)x + 1) * G - 1) / T);
    }
    // first sequence b with Hkv * prefix[b + 1] > x
    __device__ __forceinline__ int seq_of(int x) const {
        int lo = 0, hi = B - 1;
        while (lo < hi) {
            int mid = (lo + hi) >> 1;
            if (Hkv * prefix[mid + 1] > x) hi = mid; else lo = mid + 1;
        }
        return lo;
    }
    // the same by a whole warp, which looks at 32 places at once (B <= 1024): two turns instead of up to ten
    __device__ __forceinline__ int seq_of_warp(int x) const {
        const int lane = threadIdx.x % 32, apart = (B + 31) / 32;
        const int block = __ffs(__ballot_sync(0xffffffffu, Hkv * prefix[min((lane + 1) * apart, B)] > x)) - 1, b = min(block * apart + lane, B - 1);
        return min(block * apart + __ffs(__ballot_sync(0xffffffffu, Hkv * prefix[b + 1] > x)) - 1, B - 1);
    }
};

// One segment of a CTA's range: stages [s0, s1) of (b, g).
struct Segment {
    int b, g, s0, s1, L;
    int c_first, n_parts;   // CTAs that hold a piece of this (b, g)
};

// Walks the segments of the range [pos, end).  Only the first step searches; later ones step to the next
// KV head / sequence.  Division-heavy lookups happen only for the (at most two) segments that a range
// boundary cuts.
struct SegmentIter {
    int pos, end, b, g;
    bool started;
    __device__ __forceinline__ void init(int lo, int hi) { pos = lo; end = hi; b = 0; g = 0; started = false; }
    // the range's first segment: known, or found by a whole warp, which has the same range in all lanes
    __device__ __forceinline__ void start_at(int first_b, int first_g) { b = first_b; g = first_g - 1; started = true; }
    __device__ __forceinline__ void search_warp(const Schedule& sc) {
        int first_b = 0, first_g = 0;
        if (pos < end) {
            first_b = sc.seq_of_warp(pos);
            const int n = sc.nst(first_b), at = pos - sc.Hkv * sc.prefix[first_b];
            first_g = sc.Hkv <= 32 ? __ffs(__ballot_sync(0xffffffffu, ((int)(threadIdx.x % 32) + 1) * n > at)) - 1 : at / n;
        }
        start_at(first_b, first_g);
    }
    // `want_parts` = false skips c_first / n_parts (two divisions), which the producer never reads
    __device__ __forceinline__ bool next(const Schedule& sc, Segment& sg, bool want_parts = true) {
        if (pos >= end) return false;
        int n;
        if (!started) {
            b = sc.seq_of(pos);
            n = sc.nst(b);
            g = (pos - sc.Hkv * sc.prefix[b]) / n;
            started = true;
        } else {
            if (++g == sc.Hkv) {
                g = 0;
                do { ++b; } while (sc.nst(b) == 0);
            }
            n = sc.nst(b);
        }
        const int sb = sc.Hkv * sc.prefix[b] + g * n;
        sg.b = b; sg.g = g;
        sg.s0 = pos - sb;
        sg.s1 = min(n, end - sb);
        sg.L = sc.len[b];
        if ((sg.s0 == 0 && sg.s1 == n) || !want_parts) {
            sg.c_first = blockIdx.x;
            sg.n_parts = 1;
        } else {
            sg.c_first = sc.cta_of(sb);
            sg.n_parts = sc.cta_of(sb + n - 1) - sg.c_first + 1;
        }
        pos = sb + sg.s1;
        return true;
    }
};

// Lengths and stages of all sequences into shared memory, by the whole block: an exclusive prefix sum, of 32 sequences a warp and then
// of the warps' sums.  (One warp alone, 32 after 32: 0.5 us more for 256 sequences, 2 us for 1000.)
template <int THREADS, int STAGE_TOKENS>
__device__ __forceinline__ void decode_prefix(const int32_t* seq_lens, int B, int max_seq_len, int* s_len, int* s_prefix, int* s_nmax) {
    __shared__ int s_sum[DEC_MAX_SEQS / 32], s_most[DEC_MAX_SEQS / 32];
    constexpr int TURNS = (DEC_MAX_SEQS + THREADS - 1) / THREADS;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, blocks = (B + 31) / 32;
    auto scan = [&](int v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += t;
        }
        return v;
    };
    int upto[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        const int k = warp + i * (THREADS / 32), b = k * 32 + lane;
        if (k >= blocks) break;
        const int L = b < B ? max(0, min(seq_lens[b], max_seq_len)) : 0, v = (L + STAGE_TOKENS - 1) / STAGE_TOKENS;
        if (b < B) s_len[b] = L;
        upto[i] = scan(v);
        const int most = __reduce_max_sync(0xffffffffu, v);
        if (lane == 31) { s_sum[k] = upto[i]; s_most[k] = most; }
    }
    __syncthreads();
    const int sums = scan(lane < blocks ? s_sum[lane] : 0);
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        const int k = warp + i * (THREADS / 32), b = k * 32 + lane;
        if (k >= blocks) break;
        const int before = __shfl_sync(0xffffffffu, sums, max(k - 1, 0));
        if (b < B) s_prefix[b + 1] = upto[i] + (k ? before : 0);
    }
    if (warp == 0) {
        const int most = __reduce_max_sync(0xffffffffu, lane < blocks ? s_most[lane] : 0);
        if (lane == 0) { s_prefix[0] = 0; *s_nmax = most; }
    }
    __syncthreads();
}

// A part of a (sequence, KV head) has been stored: takes a ticket for it and, in the CTA that holds the last one, merges all parts
template <typename Params> __device__ __forceinline__ void decode_combine(const Params& p, const Segment& sg, int lane) {
    __threadfence();     // the consumers' stores, observed through the barrier, before the ticket
    const int bgi = sg.b * p.Hkv + sg.g;
    int ticket = 0;
    if (lane == 0) ticket = atomicAdd(&p.tickets[bgi], 1);
    ticket = __shfl_sync(0xffffffffu, ticket, 0);
    if (ticket != sg.n_parts - 1) return;
    __threadfence();
    const size_t base = (size_t)bgi * p.max_parts;
    // lane -> head lane / 4, dims 16 * (lane % 4) .. + 15
    const int ch = lane / 4, cd = (lane % 4) * 16;
    // parts are merged four at a time: all their loads are issued before the first use, so a merge of up
    // to four parts costs one L2 round trip, not one per part
    float m2 = -INFINITY, l2 = 0.f, a2[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) a2[i] = 0.f;
    for (int c0 = 0; c0 < sg.n_parts; c0 += 4) {
        float pm[4], pl[4];
        float4 po[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool on = c0 + i < sg.n_parts;
            const size_t e = (base + (on ? c0 + i : 0)) * DEC_G + ch;
            pm[i] = on ? __ldcg(p.part_m + e) : -INFINITY;
            pl[i] = on ? __ldcg(p.part_l + e) : 0.f;
            const float4* src = reinterpret_cast<const float4*>(p.part_o + e * DEC_D + cd);
#pragma unroll
            for (int v = 0; v < 4; ++v) po[i][v] = on ? __ldcg(src + v) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float mnew = m2;
#pragma unroll
        for (int i = 0; i < 4; ++i) mnew = fmaxf(mnew, pm[i]);
        const float ms2 = mnew == -INFINITY ? 0.f : mnew;
        const float keep = ex2(m2 - ms2);          // 0 while nothing has been merged yet (m2 = -inf)
        l2 *= keep;
#pragma unroll
        for (int i = 0; i < 16; ++i) a2[i] *= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float scl = ex2(pm[i] - ms2);
            l2 += pl[i] * scl;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                a2[4 * v] += po[i][v].x * scl; a2[4 * v + 1] += po[i][v].y * scl;
                a2[4 * v + 2] += po[i][v].z * scl; a2[4 * v + 3] += po[i][v].w * scl;
            }
        }
        m2 = mnew;
    }
    if (lane == 0) p.tickets[bgi] = 0;   // leave the scratch clean for the next launch
    if (ch < p.n_rep) {
        const float inv = l2 > 0.f ? 1.f / l2 : 0.f;
        const size_t crow = (size_t)sg.b * p.Hq + (size_t)sg.g * p.n_rep + ch;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float r0 = a2[4 * i] * inv, r1 = a2[4 * i + 1] * inv, r2 = a2[4 * i + 2] * inv,
                        r3 = a2[4 * i + 3] * inv;
            if (p.out)
                *reinterpret_cast<uint2*>(p.out + crow * DEC_D + cd + 4 * i) =
                    make_uint2(pack_bf16(r0, r1), pack_bf16(r2, r3));
            if (p.out_f32)
                *reinterpret_cast<float4*>(p.out_f32 + crow * DEC_D + cd + 4 * i) = make_float4(r0, r1, r2, r3);
        }
        if (p.lse && lane % 4 == 0) p.lse[crow] = l2 > 0.f ? (m2 + log2f(l2)) * LN2 : -INFINITY;
    }
}

}  // namespace bn
