// Attention of few tokens over 4-bit pages (gfx950), split over the rows and
// joined.
//
// For the query tokens t and heads g that share a KV head,
//   o_tg = sum_r p_r v_r,  p_r = exp(c q_tg.k_r) / sum,  r <= sees(t).
// A workgroup takes one KV head, 16 NQ of its (token, head) columns and a share of
// the rows, with a running maximum and sum per column.
// Codes become f16 operands in registers, exactly: S^T = K Q^T takes 16 bytes of
// a key row per lane (32 channels of one group), O^T = V^T P^T 16 bytes of value
// codes (eight channels of four rows), whose column layouts agree, so neither
// the rows nor the weights pass through LDS.
// Bound by memory and then by the decoding's VALU work: two sequences of 128K rows
// 58-64 us (4.7-5.2 TB/s, the VALU busy for 71% of the cycles), 16 of 2K-32K 41 us with
// the join, five drafted tokens of eight sequences 41 us (35 columns, two groups that
// decode every row each; one group of 48 needs the registers of both wavefronts of a
// SIMD and took as long).
#pragma once

#include "int4_attn.h"

namespace {

constexpr int WT = 64;                       // rows per wavefront and step

// The codes and words of a wavefront's 64 rows, as four tiles of 16.
struct Rows {
    u32x4 k[4], v[4];
    u32x2 vw[4];
    uint32_t kw[4];
    uint32_t gone;                           // tiles of no page, which read page 0 (uniform)
};

template <int NQ, int NW>
struct DecodeSmem {
    float o[NW][16][D + 4];
    float m[NQ][NW][16], l[NQ][NW][16];
};

// Rows t0 .. of a sequence up to `stop`.  DIRECT: all of its rows, and what this
// gives are the outputs; else they are a partition's, at row `to` of the partials.
// ONE: a wavefront has one step at most.
template <bool F16, int NQ, int NW, bool ONE>
__device__ __forceinline__ void few_rows(const Int4Args &a, DecodeSmem<NQ, NW> &sm, int h, int col0, int seq, const Int4Seq s,
                                         int t0, int stop, bool direct, int64_t to)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    // The pages are looked up first (what max_tokens admits stands in the table, so a
    // first step need not wait for the lengths), then the queries are asked for, then
    // the first rows: neither waits for what it does not need.
    const Int4Pool &p = a.pool;
    const int32_t *table = p.tables + seq * p.bt_stride;
    constexpr int NEXT = WT * NW;
    int c0 = t0 + WT * wave;
    // lane l: the page of tile l % 4 of the rows that are asked for next, and of those after them
    int id_lane = 0, id_after = 0;
    auto look_up = [&](int c0) __attribute__((always_inline)) {
        const int row = c0 + 16 * (lane & 3);
        return table[(row < a.max_tokens ? row : a.max_tokens - 1) >> p.shift];
    };
    if (a.max_tokens > 0) {
        id_lane = look_up(c0);
        if constexpr (!ONE) id_after = look_up(c0 + NEXT);
    }
    const int cols = int4_asked<true>(a, s) * a.G;
    if (col0 >= cols) return;                // uniform
    const int colN = col0 + 16 * NQ < cols ? col0 + 16 * NQ : cols;
    const int sees0 = s.sees(col0 / a.G), sees1 = s.sees((colN - 1) / a.G);     // the first and last column's
    const int end = stop < sees1 + 1 ? stop : sees1 + 1;
    if (!direct && t0 >= end) return;        // uniform; the join does not read this partition
    // B operand: column c16, channels 32 g4 + 8 d .. + 7; its last row and factor
    u32x4 qb[NQ][4];
    int sees[NQ];
    float scale[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int col = col0 + 16 * n + c16 < colN ? col0 + 16 * n + c16 : colN - 1;
        const int t = col / a.G, g = col - t * a.G;
        sees[n] = s.sees(t);
        const uint16_t *qp = a.q + (int64_t)(s.t0 + t) * a.q_st + (int64_t)(h * a.G + g) * a.q_sh + 32 * g4;
#pragma unroll
        for (int d = 0; d < 4; ++d) qb[n][d] = ld16(qp + 8 * d);
    }
    const uint32_t kw0 = i4_key_words(p.B), v0 = i4_value_codes(p.B), vw0 = i4_value_words(p.B);
    const uint8_t *base = p.base + h * p.s_head;
    auto load = [&](Rows &r, int c0) __attribute__((always_inline)) {
        const uint32_t here = (uint32_t)__builtin_amdgcn_ballot_w64(c0 + 16 * (lane & 3) < end && (uint32_t)id_lane < (uint32_t)p.pages);
        r.gone = ~here & 15;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int id = here >> t & 1 ? __builtin_amdgcn_readlane(id_lane, t) : 0;
            const uint32_t row = (c0 + 16 * t) & (p.B - 1);              // a tile lies in one page, and its rows exist
            const uint8_t *head = base + (int64_t)id * p.s_page;
            r.k[t] = ldnt_at<u32x4>(head, 64 * row + 16 * (4 * c16 + g4));
            r.kw[t] = ldnt_at<uint16_t>(head, kw0 + 8 * row + 2 * (4 * c16 + g4));
            r.v[t] = ldnt_at<u32x4>(head, v0 + 64 * row + 16 * (16 * g4 + c16));
            r.vw[t] = ldnt_at<u32x2>(head, vw0 + 8 * row + 8 * (4 * g4 + (c16 >> 2)));
        }
    };
    Rows ra, rb;
    if (c0 < end) load(ra, c0);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        float x[4][8], most = 0.0f;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            query8<F16>(qb[n][d], x[d]);
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[d][i]));
        }
        const int shift = query_shift(xmax16(most));
        // the maximum is taken before the scale, which is made positive; logits that its size rounds to 0 are 0
        float f = __builtin_ldexpf(a.c_log2 < 0.0f ? -1.0f : 1.0f, shift);
        scale[n] = __builtin_ldexpf(fabsf(a.c_log2), -shift);
        if (scale[n] < 0x1p-110f) {
            f = 0.0f;
            scale[n] = 1.0f;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) qb[n][d][i] = pack2<true>(x[d][i] * f, x[d][i + 4] * f);
    }
    float m_run[NQ], l_run[NQ], poison[NQ];  // of column c16; l_run: this lane's rows; poison: NaN or 0
    f32x4 acc[NQ][8];                        // O^T rows 4 g4 + i of product j: channels 8 (4 g4 + i) + j, column c16
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m_run[n] = NEG_INF;
        l_run[n] = poison[n] = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[n][j] = f32x4{0, 0, 0, 0};
    }
    const I4Masks masks;
    auto take = [&](Rows &r, int c0) __attribute__((always_inline)) {
        f32x4 sc[NQ][4];                     // S^T rows 16 t + 4 g4 + i (cache rows), column c16
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const I4Scale w = i4_scale(r.kw[t]);
            u32x4 kf[4];
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) kf[d][i] = i4_value(masks.pair(r.k[t][d], i), lower(w.s), lower(w.c));
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                sc[n][t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int d = 0; d < 4; ++d) sc[n][t] = mma32<true>(kf[d], qb[n][d], sc[n][t]);
            }
        }
        if (r.gone || c0 + WT - 1 > sees0) {                 // uniform: rows that some column does not see
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int first = c0 + 16 * t + 4 * g4;
                const bool gone = r.gone >> t & 1;
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (gone || first + i > sees[n]) sc[n][t][i] = NEG_INF;
                // a weight of 0 does not hide a NaN: rows that no column sees become zeros, and so do
                // NaN words of the others, which poison the columns that see them
                uint32_t nan = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t half = 16 * (i & 1);
                    const bool out = gone || first + i > sees1;
                    const bool bad = !out && (r.vw[t][i >> 1] >> half & 0x7c00u) == 0x7c00u;
                    if (out || bad) r.vw[t][i >> 1] &= ~(0xffffu << half);
                    nan |= bad ? 1u << i : 0;
                }
                uint64_t lanes = __builtin_amdgcn_ballot_w64(nan != 0);
                for (; lanes; lanes &= lanes - 1) {
                    const int from = __builtin_ctzll(lanes);             // lane (channel block, row quad)
                    const uint32_t which = (uint32_t)__builtin_amdgcn_readlane((int)nan, from);
                    const int row = c0 + 16 * t + 4 * (from >> 4) + __builtin_ctz(which);
                    if (g4 == (from & 15) >> 2)                          // the lanes whose channels are of its group
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
                            if (row <= sees[n]) poison[n] = __builtin_nanf("");
                }
            }
        }
        u32x4 pb[NQ][2];                     // B operand: rows 16 (2 m) + 4 g4 + i, then 16 (2 m + 1) + 4 g4 + i
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float cmax = NEG_INF;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) cmax = fmaxf(cmax, sc[n][t][i]);
            const float m_new = fmaxf(m_run[n], xmax16(cmax) * scale[n]), m_use = m_new == NEG_INF ? 0.0f : m_new;
            float alpha = __builtin_amdgcn_exp2f(m_run[n] - m_use);
            const float less = I4_BIAS - m_use;
            float lsum = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(sc[n][t][i], scale[n], less));
#pragma unroll
                for (int i = 0; i < 2; ++i) pb[n][t >> 1][2 * (t & 1) + i] = pack2<true>(w[2 * i], w[2 * i + 1]);
                lsum += (w[0] + w[1]) + (w[2] + w[3]);
            }
            l_run[n] = fmaf(l_run[n], alpha, lsum);
            m_run[n] = m_new;
            if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
                asm volatile("" : "+v"(alpha));              // the products stay behind the branch
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[n][j] *= alpha;
            }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            I4Scale w[4];                    // of row pairs 0, 1 and 2, 3 of either tile
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = i4_scale(r.vw[2 * m + (i >> 1)][i & 1]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                u32x4 vf;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    vf[i] = i4_value(masks.pair(r.v[2 * m + (i >> 1)][2 * (i & 1) + (j >> 2)], j & 3), w[i].s, w[i].c);
#pragma unroll
                for (int n = 0; n < NQ; ++n) acc[n][j] = mma32<true>(vf, pb[n][m], acc[n][j]);
            }
        }
    };
    // The next rows travel while these are taken; their pages are looked up before
    // the rows ahead of them are asked for, whose arrival they need not wait for.
    if (ONE && c0 < end) take(ra, c0);
    if (!ONE && c0 < end) {
        for (;;) {
            id_lane = id_after;
            id_after = look_up(c0 + 2 * NEXT);
            load(rb, c0 + NEXT);
            take(ra, c0);
            c0 += NEXT;
            if (c0 >= end) break;
            id_lane = id_after;
            id_after = look_up(c0 + 2 * NEXT);
            load(ra, c0 + NEXT);
            take(rb, c0);
            c0 += NEXT;
            if (c0 >= end) break;
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        l_run[n] = xsum16(l_run[n]);
        __syncthreads();                     // what was there before has been read
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                f32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = acc[n][4 * half + e][i] + poison[n];
                *(f32x4 *)&sm.o[wave][c16][8 * (4 * g4 + i) + 4 * half] = x;
            }
        if (g4 == 0) {
            sm.m[n][wave][c16] = m_run[n];
            sm.l[n][wave][c16] = l_run[n];
        }
        __syncthreads();
        const int here = colN - (col0 + 16 * n) < 16 ? colN - (col0 + 16 * n) : 16;
        for (int i = tid; i < 32 * here; i += 64 * NW) {
            const int k = i >> 5, c = 4 * (i & 31), col = col0 + 16 * n + k;
            float M = NEG_INF;
#pragma unroll
            for (int w = 0; w < NW; ++w) M = fmaxf(M, sm.m[n][w][k]);
            const float use = M == NEG_INF ? 0.0f : M;
            float L = 0.0f;
            f32x4 o = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = __builtin_amdgcn_exp2f(sm.m[n][w][k] - use);
                L = fmaf(f, sm.l[n][w][k], L);
                const f32x4 x = *(const f32x4 *)&sm.o[w][k][c];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(f, x[e], o[e]);
            }
            const int t = col / a.G, hq = h * a.G + col - t * a.G;
            if (direct) {
                const int64_t at = (int64_t)(s.t0 + t) * a.o_st + hq * a.o_sh + c;
#pragma unroll
                for (int e = 0; e < 4; ++e) iq_store_as(a.out, at + e, L == 0.0f ? 0.0f : o[e] / L, a.odt);
            } else {
                const int64_t row = to + 16 * n + k;
                *(f32x4 *)(a.part.o + row * D + c) = o;
                if (c == 0) a.part.ml[row] = f32x2{M, L};
            }
        }
    }
}

// One sequence (blockIdx.z) each.
template <bool F16, int NQ, int NW>
__global__ __launch_bounds__(64 * NW, 2) void int4_whole(Int4Args a)
{
    __shared__ DecodeSmem<NQ, NW> sm;
    const int h = blockIdx.x % a.pool.H, group = blockIdx.x / a.pool.H;
    few_rows<F16, NQ, NW, true>(a, sm, h, group * 16 * NQ, blockIdx.z, int4_seq(a, blockIdx.z), 0, a.max_tokens, true, 0);
}

// An even share of the sequences' steps each.
template <bool F16, int NQ>
__global__ __launch_bounds__(256, 2) void int4_shared(Int4Args a)
{
    __shared__ DecodeSmem<NQ, 4> sm;
    // a group's workgroups one after the other: those of groups that no sequence has end
    // at once, and must not stand on the same XCDs (each eighth workgroup is on one's)
    const int per = a.pool.H * a.workers, group = blockIdx.x / per, rest = blockIdx.x - group * per;
    const int h = rest % a.pool.H, w = rest / a.pool.H, plane = h + a.pool.H * group;
    const Share r = int4_share(a, group);
    const int x0 = w * r.each, x1 = x0 + r.each < r.total ? x0 + r.each : r.total;
    for (int x = x0; x < x1;) {              // uniform
        const int seq = __builtin_popcountll(__builtin_amdgcn_ballot_w64(r.upto <= x));
        const int upto = __builtin_amdgcn_readlane(r.upto, seq), steps = __builtin_amdgcn_readlane(r.steps, seq);
        const int from = upto - steps, stop = upto < x1 ? upto : x1;
        few_rows<F16, NQ, 4, false>(a, sm, h, group * 16 * NQ, seq, r.of(seq), (x - from) * STEP, (stop - from) * STEP, stop - x == steps,
                             ((int64_t)plane * (a.workers + a.n_seq) + w + seq) * (16 * NQ));
        x = stop;
    }
}

}  // namespace
