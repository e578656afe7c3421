// One token's attention over exact pages (gfx950), split over the rows and
// joined, with the rows' accumulated weights on request.
//
// For sequence s, KV head h and the G query heads g that share it,
//   o_g = sum_r p_gr v_r,  p_gr = exp(c q_g.k_r - lse_g),
//   weights[r] += sum_g p_gr.
// Each workgroup takes one (KV head, partition of the rows, sequence) with a
// running maximum and sum per query head, and leaves the unnormalized output
// with (max, sum); a second launch joins the partitions.  The weights need the
// joined lse, so the first launch also leaves the logits (4 bytes per row and
// query head against 512 read per row and KV head).  For the matrix cores' second
// product the weights p round to the rows' type, by at most half a step each; the
// sums l and what is added to a row's weight stay in fp32 (300 rows in bf16, distance
// from 64 bits: 1.70e-3 of the output, and 1.65e-3 by its own rounding alone).
// Bound by HBM: 16 sequences of
// 2K-32K tokens, 28 heads over 4, 549 MB: 104 us (5.3 TB/s) and 5 for the join.
#include "dense_common.h"

namespace {

constexpr int D = 128;
constexpr int NT = 256;                      // threads of the join, and of a partition's workgroup
constexpr int WT = 64;                       // rows per wavefront and step
constexpr int PT = WT * NT / 64;             // rows per workgroup of a partition and step
constexpr int ONE_MOST = 512;                // rows that a workgroup takes in one step
constexpr float LOG2E = 1.44269504088896341f;

struct DecodeArgs {
    DensePool pool;
    const uint16_t *q;
    int64_t q_ss, q_sh;
    const int32_t *lengths;
    int32_t max_tokens, span, parts, G, Hq;  // span: rows per partition, a multiple of PT
    float c_log2;
    Partials part;                           // [n * Hq, parts] rows
    float *logits;                           // [n * Hq, l_stride] in log2 units, or null
    int64_t l_stride;
    void *out;
    int64_t o_ss, o_sh;
    int odt, accumulate;
};

// V rows of a step in LDS: 256 bytes each, the 16-byte chunk c of row r at
// slot c ^ 4 (r % 4) ^ 2 (r / 4 % 2), so that the transposed reads of 32 lanes
// (two groups of four rows, 32 bytes each) hit 64 distinct banks.
template <int NW>
struct __attribute__((aligned(16))) DecodeSmem {
    union {
        uint16_t v[NW][WT * D];
        float o[NW][16][D + 4];
    };
    float m[NW][16], l[NW][16];
    float lse[16];
};

// ds_read_b64_tr_b16: when lane s of 16 reads row K0 + s / 4, channels
// c0 + 4 (s % 4) .. + 3, lane i receives channel c0 + i of rows K0 .. K0 + 3.
typedef short gv16x4 __attribute__((__vector_size__(4 * sizeof(short))));
__device__ __forceinline__ u32x2 tr_read(const uint16_t *p)
{
    const gv16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) gv16x4 *)(__attribute__((address_space(3))) uint16_t *)p);
    return __builtin_bit_cast(u32x2, v);
}

__device__ __forceinline__ float row_max16(float v)
{
    v = fmaxf(v, dpp_f<0xb1>(v));            // as row_sum16
    v = fmaxf(v, dpp_f<0x4e>(v));
    v = fmaxf(v, dpp_f<0x141>(v));
    return fmaxf(v, dpp_f<0x140>(v));
}

// Adds the weights of cache rows r, r + NT, r + 2 NT and r + 3 NT (those below
// `end`) of a KV head, from their logits and the heads' lse; neighbouring lanes
// take neighbouring rows, which meet in one line.  load() asks for the logits of
// the first four heads.
struct FirstRows {
    float s[4][4];

    __device__ __forceinline__ static const float *logits(const DecodeArgs &a, int64_t q0, int g, int r)
    {
        return a.logits + (q0 + g) * a.l_stride + r;
    }
    __device__ __forceinline__ void load(const DecodeArgs &a, int64_t q0, int r, int end)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = r + i * NT < end ? r + i * NT : end - 1;
#pragma unroll
            for (int g = 0; g < 4; ++g) s[g][i] = *logits(a, q0, g < a.G ? g : a.G - 1, at);
        }
    }
    __device__ __forceinline__ void add(const DecodeArgs &a, const float *lse, int h, int seq, int64_t q0, int r, int end)
    {
        float w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (g < a.G) {
                const float x = lse[g];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] += __builtin_amdgcn_exp2f(s[g][i] - x);
            }
        for (int g = 4; g < a.G; ++g) {
            const float x = lse[g];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r + i * NT < end) w[i] += __builtin_amdgcn_exp2f(*logits(a, q0, g, r + i * NT) - x);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (r + i * NT >= end) break;
            const int64_t page = dense_page(a.pool, seq, r + i * NT);
            // added in memory, so that sequences that share a page lose no weight
            if (page >= 0)
                unsafeAtomicAdd(a.pool.weights + (page * a.pool.H + h) * a.pool.B + ((r + i * NT) & (a.pool.B - 1)), w[i]);
        }
    }
};

// PARTS: one of several partitions.  DIRECT: the only one; the outputs and
// weights are final.  ONE: the only one, and each wavefront's rows are one step,
// whose logits stay in registers until the lse is known.
enum Mode { PARTS, DIRECT_LOOP, ONE };

// lds_load16 past the caches, as the keys are read: rows are read once per call
// (16 sequences of 2K-32K tokens: 107 us, 110 with both through the caches, 114
// with one each way).
__device__ __forceinline__ void lds_load16_nt(const void *base, uint32_t voff, uint32_t lds_base)
{
    const uint64_t b = (uint64_t)(uintptr_t)base;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
    const uint64_t sb = (uint64_t)lo | ((uint64_t)hi << 32);
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(voff), "s"(sb),
                 "s"(__builtin_amdgcn_readfirstlane(lds_base))
                 : "memory");
}

template <bool F16, Mode MODE, int NW>
__global__ __launch_bounds__(64 * NW, 2) void dense_partials(DecodeArgs a)
{
    constexpr bool DIRECT = MODE != PARTS;
    constexpr int THREADS = 64 * NW;
    __shared__ DecodeSmem<NW> sm;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c16 = lane & 15, g4 = lane >> 4;
    const int h = blockIdx.x, part = blockIdx.y, seq = blockIdx.z;
    const int have = a.lengths[seq], len = have < a.max_tokens ? have : a.max_tokens;
    const int t0 = part * a.span;
    const DensePool &p = a.pool;
    const int32_t *table = p.tables + seq * p.bt_stride;
    // Ids of the pages of a step's four tiles, read beside the length and in the
    // loop a step ahead (300 rows 8.2 -> 7.8 us; 16 sequences of 2K-32K tokens 110
    // -> 107): what max_tokens admits stands in the table.
    int ids[4];
    auto look_up = [&](int c0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int row = c0 + 16 * t < a.max_tokens ? c0 + 16 * t : a.max_tokens - 1;
            ids[t] = table[row >> p.shift];
        }
    };
    if (a.max_tokens > 0) look_up(t0 + WT * wave);
    if (t0 >= len) {                         // uniform; the join does not read this partition
        if constexpr (DIRECT)                // no row: nothing to attend to
            for (int i = tid; i < D * a.G; i += THREADS)
                iq_store_as(a.out, seq * a.o_ss + (h * a.G + (i >> 7)) * a.o_sh + (i & 127), 0.0f, a.odt);
        return;
    }
    const int end = t0 + a.span < len ? t0 + a.span : len;
    u32x4 qb[4];                             // B operand: column c16 = query head, channels 32 d + 8 g4 .. + 7
    {
        const int g = c16 < a.G ? c16 : 0;
        const uint16_t *qp = a.q + seq * a.q_ss + (int64_t)(h * a.G + g) * a.q_sh + 8 * g4;
#pragma unroll
        for (int d = 0; d < 4; ++d) qb[d] = ld16(qp + 32 * d);
    }
    float m_run = NEG_INF, l_run = 0.0f;     // of column c16; l_run: this lane's rows
    f32x4 acc[8];                            // O^T rows 16 cb + 4 g4 + i (channels), column c16
#pragma unroll
    for (int cb = 0; cb < 8; ++cb) acc[cb] = f32x4{0, 0, 0, 0};
    const uint32_t lds_v = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t *)&sm.v[wave][0];
    f32x4 sc[4];                             // S^T rows 16 t + 4 g4 + i (cache rows), column c16
    int64_t at[4];                           // ONE: the tiles' first weights
    int last[4];                             // a tile's last live row; -1: none, or its page is not in the pool
    for (int c0 = t0 + WT * wave; c0 < end; c0 += WT * NW) {
        const uint16_t *kt[4], *vt[4];       // first row of each 16-row tile
        u32x4 kf[4][4];
        uint32_t outside = 0;                // tiles of ids outside the pool, which read page 0
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            // a tile past the end reads the first again (masked)
            const int want = c0 + 16 * t, tb = want < len ? want : c0;
            const int id = want < len ? ids[t] : ids[0];
            const bool ok = id >= 0 && id < p.pages;
            const int64_t page = ok ? id : 0;
            outside |= ok ? 0 : 1u << t;
            const int row = tb & (p.B - 1);
            kt[t] = p.key + page * p.k_sp + h * p.k_sh + row * p.k_st;
            vt[t] = p.value + page * p.v_sp + h * p.v_sh + row * p.v_st;
            at[t] = (page * p.H + h) * p.B + row;
            const int rest = len - 1 - tb;
            last[t] = rest < 15 ? rest : 15;
            const int r = c16 < last[t] ? c16 : last[t];
            const uint32_t off = (uint32_t)(r * (int)p.k_st + 8 * g4) * 2;
#pragma unroll
            for (int d = 0; d < 4; ++d) kf[t][d] = ldnt_at<u32x4>(kt[t], off + 64 * d);
            if (!ok || want >= len) last[t] = -1;
        }
        // the reads of the previous step's rows are done before theirs are overwritten
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int t = i >> 2, rl = 4 * (i & 3) + g4;
            const int lim = len - 1 - (c0 + 16 * t < len ? c0 + 16 * t : c0);
            const int r = rl < lim ? rl : lim;
            const int chunk = c16 ^ (4 * (rl & 3)) ^ (2 * ((rl >> 2) & 1));
            lds_load16_nt(vt[t], (uint32_t)(r * (int)p.v_st + 8 * chunk) * 2, lds_v + (uint32_t)(4 * i * D * 2));
        }
        // not before the wait above, which counts these reads too
        if constexpr (MODE != ONE) look_up(c0 + WT * NW);
#pragma unroll
        for (int t = 0; t < 4; ++t) sc[t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int t = 0; t < 4; ++t) sc[t] = mma32<F16>(kf[t][d], qb[d], sc[t]);
        float cmax = NEG_INF;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[t][i] = 4 * g4 + i <= last[t] ? sc[t][i] * a.c_log2 : NEG_INF;
                cmax = fmaxf(cmax, sc[t][i]);
            }
        if (MODE != ONE && a.logits && c16 < a.G) {
            float *lp = a.logits + (int64_t)(seq * a.Hq + h * a.G + c16) * a.l_stride + c0 + 4 * g4;
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (c0 + 16 * t < len) *(f32x4 *)(lp + 16 * t) = sc[t];
        }
        cmax = xmax16(cmax);
        const float m_new = fmaxf(m_run, cmax), m_use = m_new == NEG_INF ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
        float lsum = 0.0f;
        u32x4 pb[2];                         // B operand: rows 16 (2 m) + 4 g4 + i, then 16 (2 m + 1) + 4 g4 + i
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = __builtin_amdgcn_exp2f(sc[t][i] - m_use);
                lsum += w[i];
            }
            pb[t >> 1][2 * (t & 1)] = pack2<F16>(w[0], w[1]);
            pb[t >> 1][2 * (t & 1) + 1] = pack2<F16>(w[2], w[3]);
        }
        l_run = fmaf(l_run, alpha, lsum);
        m_run = m_new;
#pragma unroll
        for (int cb = 0; cb < 8; ++cb) acc[cb] *= alpha;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // this wavefront's V rows have landed
        const uint16_t *sv = sm.v[wave];
        // a weight of 0 does not hide what page 0 may hold (NaN, infinities)
        for (; outside; outside &= outside - 1) {
            uint16_t *rows = sm.v[wave] + 16 * __builtin_ctz(outside) * D;
#pragma unroll
            for (int i = 0; i < 4; ++i) *(u32x4 *)(rows + (4 * i + g4) * D + 8 * c16) = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int cb = 0; cb < 8; ++cb) {
                const int r = 32 * m + 4 * g4 + (c16 >> 2);
                const int slot = (2 * cb + ((c16 & 3) >> 1)) ^ (4 * (c16 >> 2)) ^ (2 * (g4 & 1));
                const u32x2 lo = tr_read(sv + r * D + 8 * slot + 4 * (c16 & 1));
                const u32x2 hi = tr_read(sv + (r + 16) * D + 8 * slot + 4 * (c16 & 1));
                acc[cb] = mma32<F16>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pb[m], acc[cb]);
            }
    }
    l_run = xsum16(l_run);
    // the wavefront's own V rows have been read: its outputs take their place
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int cb = 0; cb < 8; ++cb) *(f32x4 *)&sm.o[wave][c16][16 * cb + 4 * g4] = acc[cb];
    if (g4 == 0) {
        sm.m[wave][c16] = m_run;
        sm.l[wave][c16] = l_run;
    }
    __syncthreads();
    for (int i = tid; i < 32 * a.G; i += THREADS) {
        const int g = i >> 5, c = 4 * (i & 31);
        float M = NEG_INF;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm.m[w][g]);
        const float use = M == NEG_INF ? 0.0f : M;
        float L = 0.0f;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm.m[w][g] - use);
            L = fmaf(f, sm.l[w][g], L);
            const f32x4 x = *(const f32x4 *)&sm.o[w][g][c];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(f, x[e], o[e]);
        }
        if constexpr (DIRECT) {
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            const int64_t at = seq * a.o_ss + (h * a.G + g) * a.o_sh + c;
#pragma unroll
            for (int e = 0; e < 4; ++e) iq_store_as(a.out, at + e, L == 0.0f ? 0.0f : o[e] * inv, a.odt);
            if (c == 0) sm.lse[g] = L == 0.0f ? __builtin_inff() : use + __builtin_amdgcn_logf(L);
        } else {
            const int64_t row = ((int64_t)seq * a.Hq + h * a.G + g) * a.parts + part;
            *(f32x4 *)(a.part.o + row * D + c) = o;
            if (c == 0) a.part.ml[row] = f32x2{M, L};
        }
    }
    if constexpr (MODE == ONE) {
        if (!a.accumulate) return;
        __syncthreads();                     // the lse of every head
        if (t0 + WT * wave >= end) return;   // a wavefront without rows has no logits either
        const float lse = c16 < a.G ? sm.lse[c16] : __builtin_inff();
        // lane (4 t + i, g4) takes row 16 t + 4 g4 + i
        float mine = 0.0f;
        int64_t base = at[0];
        int most = last[0];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            if (c16 >> 2 == t) {
                base = at[t];
                most = last[t];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = row_sum16(__builtin_amdgcn_exp2f(sc[t][i] - lse));
                if (c16 == 4 * t + i) mine = w;
            }
        }
        const int r = 4 * g4 + (c16 & 3);
        if (r <= most) unsafeAtomicAdd(p.weights + base + r, mine);
    }
    if constexpr (MODE == DIRECT_LOOP) {
        if (!a.logits) return;
        const int64_t q0 = (int64_t)seq * a.Hq + h * a.G;
        __syncthreads();                     // the logits and lse of every wavefront
        for (int r = tid; r < len; r += 4 * NT) {
            FirstRows rows;
            rows.load(a, q0, r, len);
            rows.add(a, sm.lse, h, seq, q0, r, len);
        }
    }
}

// Joins the partitions.  The first n * Hq workgroups write an output row each;
// the others add the weights of JW rows of a (sequence, KV head).
constexpr int JW = 1024;

struct JoinSmem {
    float o[8][D];
    float m[8], l[8];
    float lse[16];
};

__global__ __launch_bounds__(NT) void dense_join(DecodeArgs a, int n)
{
    __shared__ JoinSmem sm;
    const int tid = threadIdx.x, rows = n * a.Hq;
    if ((int)blockIdx.x < rows) {
        const int seq = blockIdx.x / a.Hq, hq = blockIdx.x % a.Hq;
        const int have = a.lengths[seq], len = have < a.max_tokens ? have : a.max_tokens;
        const int live = len > 0 ? (len + a.span - 1) / a.span : 0;
        const int64_t base = (int64_t)blockIdx.x * a.parts;
        const int grp = tid >> 5, c = 4 * (tid & 31);
        float M = NEG_INF, L = 0.0f;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll 2
        for (int p = grp; p < live; p += 8) {
            const f32x2 ml = a.part.ml[base + p];
            const f32x4 x = *(const f32x4 *)(a.part.o + (base + p) * D + c);
            const float m = fmaxf(M, ml[0]), use = m == NEG_INF ? 0.0f : m;
            const float f0 = __builtin_amdgcn_exp2f(M - use), f1 = __builtin_amdgcn_exp2f(ml[0] - use);
            L = L * f0 + ml[1] * f1;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = o[e] * f0 + x[e] * f1;
            M = m;
        }
        *(f32x4 *)&sm.o[grp][c] = o;
        if (c == 0) {
            sm.m[grp] = M;
            sm.l[grp] = L;
        }
        __syncthreads();
        if (tid >= D) return;
        float mx = NEG_INF;
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, sm.m[i]);
        const float use = mx == NEG_INF ? 0.0f : mx;
        float sum = 0.0f, v = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = __builtin_amdgcn_exp2f(sm.m[i] - use);
            sum = fmaf(f, sm.l[i], sum);
            v = fmaf(f, sm.o[i][tid], v);
        }
        // a sequence without a live row attends to nothing: zeros
        iq_store_as(a.out, seq * a.o_ss + hq * a.o_sh + tid, sum == 0.0f ? 0.0f : v / sum, a.odt);
        return;
    }
    const int chunks = (a.max_tokens + JW - 1) / JW;
    const int item = (int)blockIdx.x - rows, H = a.pool.H;
    const int chunk = item % chunks, h = item / chunks % H, seq = item / chunks / H;
    const int have = a.lengths[seq], len = have < a.max_tokens ? have : a.max_tokens;
    const int r0 = chunk * JW, r1 = r0 + JW < len ? r0 + JW : len;
    if (r0 >= len) return;
    const int live = (len + a.span - 1) / a.span, lane = tid & 63;
    const int64_t q0 = (int64_t)seq * a.Hq + h * a.G;
    // the first rows' logits travel while the lse is made
    FirstRows first;
    first.load(a, q0, r0 + tid, r1);
    for (int g = tid >> 6; g < a.G; g += NT / 64) {
        float M = NEG_INF, L = 0.0f;
        for (int p = lane; p < live; p += 64) {
            const f32x2 ml = a.part.ml[(q0 + g) * a.parts + p];
            const float m = fmaxf(M, ml[0]), use = m == NEG_INF ? 0.0f : m;
            L = L * __builtin_amdgcn_exp2f(M - use) + ml[1] * __builtin_amdgcn_exp2f(ml[0] - use);
            M = m;
        }
        const float m = xmax16(row_max16(M)), use = m == NEG_INF ? 0.0f : m;
        L = xsum16(row_sum16(L * __builtin_amdgcn_exp2f(M - use)));
        if (lane == 0) sm.lse[g] = L == 0.0f ? __builtin_inff() : use + __builtin_amdgcn_logf(L);
    }
    __syncthreads();
    first.add(a, sm.lse, h, seq, q0, r0 + tid, r1);
}

struct Split {
    int64_t span, parts, logits, floats;     // floats: the whole workspace
};

Split split_of(int64_t Hq, int64_t H, int64_t n, int64_t max_tokens, bool accumulate)
{
    // Workgroups: a few rounds of the 512 that run at once.  Batches take more,
    // shorter ones, as their lengths differ (16 sequences of 2K-32K tokens, 28
    // heads over 4: 144 us with 1024 places, 121 with 2048, 114 with 4096, 120
    // with 8192; two of 128K, 32 over 8: 244, 251, 257, 269 with the join).
    // Up to ONE_MOST rows are left to one workgroup, which saves the join and the
    // logits' way through memory (one sequence of 300 rows, 28 heads over 4: 14.3
    // us in two launches, 10.9 in one of four wavefronts that loops).
    const int64_t steps = (max_tokens + PT - 1) / PT;
    const int64_t target = n < 4 ? 1024 : 4096, per = (n * H * steps + target - 1) / target;
    Split s;
    const bool one = max_tokens <= ONE_MOST;
    s.span = one ? ONE_MOST : PT * per;
    s.parts = max_tokens > 0 ? (max_tokens + s.span - 1) / s.span : 1;
    s.logits = accumulate && !one ? (max_tokens + 63) / 64 * 64 : 0;
    s.floats = n * Hq * ((s.parts > 1 ? s.parts * (D + 2) : 0) + s.logits);
    return s;
}

}  // namespace

extern "C" int64_t iq_dense_workspace_floats(int64_t Hq, int64_t H, int64_t n_seq, int64_t max_tokens, int accumulate)
{
    return split_of(Hq, H, n_seq, max_tokens, accumulate != 0).floats;
}

extern "C" int iq_dense_decode(const void *q, int dtype, int64_t q_ss, int64_t q_sh, int64_t Hq, int64_t n_seq,
                               const iq_dense_pages *pages, const int32_t *tables, int64_t bt_stride, int64_t bt_cols,
                               const int32_t *lengths, int64_t max_tokens, float scale, int accumulate,
                               float *workspace, int64_t workspace_floats, void *out, int64_t o_ss, int64_t o_sh,
                               int out_dtype, void *stream)
{
    DensePool pool;
    if (const int e = dense_pool("iq_dense_decode", pages, dtype, tables, bt_stride, bt_cols, n_seq, pool)) return e;
    IQ_CHECK_ARG(q && lengths && out, "iq_dense_decode: null pointer");
    IQ_CHECK_ARG((uintptr_t)q % 16 == 0 && (q_ss | q_sh) % 8 == 0, "iq_dense_decode: query rows must be 16-byte aligned");
    IQ_CHECK_ARG(Hq >= 1 && Hq % pool.H == 0 && Hq / pool.H <= 16, "iq_dense_decode: heads %lld / %d", (long long)Hq,
                 pool.H);
    IQ_CHECK_ARG(out_dtype >= IQ_F32 && out_dtype <= IQ_F16, "iq_dense_decode: bad output dtype");
    IQ_CHECK_ARG(max_tokens >= 0 && max_tokens <= bt_cols * pool.B && max_tokens <= 0x3fffffff,
                 "iq_dense_decode: max_tokens past the block tables");
    IQ_CHECK_ARG(!accumulate || pool.weights, "iq_dense_decode: pages without weights");
    if (n_seq == 0) return IQ_OK;
    const Split s = split_of(Hq, pool.H, n_seq, max_tokens, accumulate != 0);
    IQ_CHECK_ARG(s.floats == 0 || (workspace && workspace_floats >= s.floats), "iq_dense_decode: workspace too small");
    const int64_t chunks = accumulate ? (max_tokens + JW - 1) / JW : 0;
    const int64_t joins = n_seq * Hq + n_seq * pool.H * chunks;
    IQ_CHECK_ARG(s.parts <= 65535 && joins <= 0xffffff, "iq_dense_decode: too many rows");
    float *part = workspace + n_seq * Hq * s.logits;
    const DecodeArgs a{pool, (const uint16_t *)q, q_ss, q_sh, lengths, (int32_t)max_tokens, (int32_t)s.span,
                       (int32_t)s.parts, (int32_t)(Hq / pool.H), (int32_t)Hq, scale * LOG2E,
                       Partials{part, (f32x2 *)(part + n_seq * Hq * s.parts * D)},
                       s.logits ? workspace : nullptr, s.logits, out, o_ss, o_sh, out_dtype, accumulate};
    const bool f16 = dtype == IQ_F16, direct = s.parts == 1;
    const dim3 grid((unsigned)pool.H, (unsigned)s.parts, (unsigned)n_seq);
    if (max_tokens <= ONE_MOST && max_tokens > PT) {
        const auto kernel = f16 ? dense_partials<true, ONE, 8> : dense_partials<false, ONE, 8>;
        hipLaunchKernelGGL(kernel, grid, dim3(2 * NT), 0, (hipStream_t)stream, a);
    } else {
        const auto kernel = max_tokens <= PT ? f16 ? dense_partials<true, ONE, 4> : dense_partials<false, ONE, 4>
                            : direct ? f16 ? dense_partials<true, DIRECT_LOOP, 4> : dense_partials<false, DIRECT_LOOP, 4>
                                     : f16 ? dense_partials<true, PARTS, 4> : dense_partials<false, PARTS, 4>;
        hipLaunchKernelGGL(kernel, grid, dim3(NT), 0, (hipStream_t)stream, a);
    }
    if (!direct) hipLaunchKernelGGL(dense_join, dim3((unsigned)joins), dim3(NT), 0, (hipStream_t)stream, a, (int)n_seq);
    IQ_CHECK_LAUNCH("dense_decode");
    return IQ_OK;
}

extern "C" int iq_dense_decode_from(const iq_dense_decode_args *a)
{
    IQ_CHECK_ARG(a, "iq_dense_decode: null arguments");
    return iq_dense_decode((const void *)a->q, (int)a->dtype, a->q_ss, a->q_sh, a->Hq, a->n_seq,
                           (const iq_dense_pages *)a->pages, (const int32_t *)a->tables, a->bt_stride, a->bt_cols,
                           (const int32_t *)a->lengths, a->max_tokens, (float)a->scale, (int)a->accumulate,
                           (float *)a->workspace, a->workspace_floats, (void *)a->out, a->o_ss, a->o_sh,
                           (int)a->out_dtype, (void *)a->stream);
}
