// Attention of many tokens over 4-bit pages (gfx950): a chunk of a prompt.
//
// One workgroup takes 256 of the (token, head) columns that share a KV head,
// eight wavefronts of 32, and a partition of the rows in tiles of 64: S^T = K Q^T
// and O^T = V^T P^T on 32x32x16 products, the weights staying in the lanes that
// the second product reads them from.  The codes of a tile become f16 operands
// once per workgroup, exactly, on their way into LDS, beside the products: 16
// bytes of key codes are four chunks of eight channels, 16 bytes of value codes
// are eight channels of four rows, which stand in LDS as the product reads them,
// channel by channel, so nothing is transposed.
//
// Bound by the matrix cores and the arithmetic of the weights beside them, which
// the two wavefronts of a SIMD take in turn (below): 0.93-1.02 ms by the card for 2048
// tokens behind 32K rows, 28 heads over 4, 0.91-1.00 PFLOP/s.  Workgroups of 128 columns, each
// with its own coded rows, and every wavefront at its products at the same time:
// 1.65 ms.  64 columns a wavefront halve what is read from LDS, but their products'
// sums do not fit the registers that the weights' arithmetic can use.
#pragma once

#include <type_traits>

#include "int4_attn.h"

namespace {

constexpr int KT = 64;                       // rows per tile
constexpr int NW = 8;                        // wavefronts per workgroup, two per SIMD
constexpr int QT = 32 * NW;                  // columns per workgroup
constexpr int AHEAD = 6;                     // operands read before their products

typedef __attribute__((ext_vector_type(16))) float f32x16;

// K: rows of 256 bytes, whose 16-byte chunk c is at slot c ^ (row % 16).  V:
// [quad of rows][channel] 8 bytes of four rows; of the four 16-byte slots of
// eight channels, the one of channels 2 k and 2 k + 1 is at k ^ (channel / 32).
// A stage's address is told from the other's by one bit, hence the alignment.
struct __attribute__((aligned(32768))) ChunkSmem {
    uint16_t k[2][KT * D], v[2][KT * D];
    // NaN words of masked tiles [tile % 4][16 rows][row % 4]: bit 16 (row / 4 % 4) + 4 group
    uint64_t nan[4][4][4];
};

__device__ __forceinline__ f32x16 mma3232(u32x4 a, u32x4 b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) uint16_t lds_u16;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
__device__ __forceinline__ uint32_t lds_at(const uint16_t *p) { return (uint32_t)(uintptr_t)(lds_u16 *)p; }

__device__ __forceinline__ float pair_max(float v)
{
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}

__device__ __forceinline__ float pair_sum(float v)
{
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

template <bool F16, bool DIRECT>
__global__ __launch_bounds__(64 * NW, 2) void int4_chunk(Int4Args a, int tiles, int share)
{
    __shared__ ChunkSmem sm;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c32 = lane & 31, h32 = lane >> 5;
    // an XCD takes a contiguous range of (KV head, tile): its workgroups read the
    // rows of one or two heads out of its L2
    const int item = (int)(blockIdx.x & 7) * share + (int)(blockIdx.x >> 3);
    if (item >= tiles * a.pool.H) return;
    const int h = item / tiles, place = tiles - 1 - (item - h * tiles);
    const int part = blockIdx.y, seq = blockIdx.z;
    const Int4Seq s = int4_seq(a, seq);
    const int cols = int4_asked<false>(a, s) * a.G, col0 = place * QT;
    if (col0 >= cols) return;                // uniform
    const Int4Pool &p = a.pool;
    const int32_t *table = p.tables + seq * p.bt_stride;
    const int colN = col0 + QT < cols ? col0 + QT : cols;
    const int sees0 = s.sees(col0 / a.G), sees1 = s.sees((colN - 1) / a.G);
    const int t0 = part * a.span, end = t0 + a.span < sees1 + 1 ? t0 + a.span : sees1 + 1;
    if (!DIRECT && t0 >= end) return;        // uniform; the join does not read this partition
    const int w0 = col0 + 32 * wave;
    const int wave0 = s.sees((w0 < colN ? w0 : colN - 1) / a.G);     // this wavefront's first
    const int col = w0 + c32 < colN ? w0 + c32 : colN - 1, t = col / a.G, hq = h * a.G + col - t * a.G;
    const int sees = s.sees(t);
    u32x4 qb[8];                             // B operand: column c32, channels 16 d + 8 h32 .. + 7
    float c_log2;
    {
        const uint16_t *qp = a.q + (int64_t)(s.t0 + t) * a.q_st + (int64_t)hq * a.q_sh + 8 * h32;
        float x[8][8], most = 0.0f;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            query8<F16>(ld16(qp + 16 * d), x[d]);
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[d][i]));
        }
        const int shift = query_shift(pair_max(most));
        // the maximum is taken before the scale, which is made positive; logits that its size rounds to 0 are 0
        float f = __builtin_ldexpf(a.c_log2 < 0.0f ? -1.0f : 1.0f, shift);
        c_log2 = __builtin_ldexpf(fabsf(a.c_log2), -shift);
        if (c_log2 < 0x1p-110f) {
            f = 0.0f;
            c_log2 = 1.0f;
        }
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) qb[d][i] = pack2<true>(x[d][i] * f, x[d][i + 4] * f);
    }
    float m_run = NEG_INF, l_run = 0.0f;     // l_run: this lane's share of the column's sum
    uint32_t poison = 0;                     // groups whose NaN this column sees in a masked tile
    f32x16 acc[4];                           // O^T rows 32 db .. 32 db + 31 (output channels)
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[db][i] = 0.0f;
    // A tile's codes: four wavefronts take the keys' and four the values', a
    // wavefront sixteen rows: a lane 16 bytes of key codes (row lane / 4, group
    // lane % 4) or of value codes (quad lane / 16, channels 8 (lane % 16) ..).
    const bool keys = wave >= 4;             // uniform
    const int sixteen = wave & 3;
    const I4Masks masks;
    u32x4 codes, codes_next;                 // of the tile that is coded, of the one after it
    u32x2 words, words_next = {0, 0};
    int id_lane;                             // lane l: the page of a tile's sixteen l % 4
    auto look_up = [&](int k0) __attribute__((always_inline)) {
        const int row = k0 + 16 * (lane & 3);
        id_lane = table[(row < end ? row : end - 1) >> p.shift];
    };
    // asks for the codes of the tile that was looked up; which sixteens have no page
    auto fetch = [&](int k0) __attribute__((always_inline)) {
        const bool ok = k0 + 16 * (lane & 3) < end && (uint32_t)id_lane < (uint32_t)p.pages;
        const int gone = ~(int)__builtin_amdgcn_ballot_w64(ok) & 15;
        const int id = gone >> sixteen & 1 ? 0 : __builtin_amdgcn_readlane(id_lane, sixteen);
        const uint8_t *head = p.base + (int64_t)id * p.s_page + h * p.s_head;
        const uint32_t row = (uint32_t)(k0 + 16 * sixteen) & (p.B - 1);
        codes_next = ldg_at<u32x4>(head, (keys ? 0 : i4_value_codes(p.B)) + 64 * row + 16 * lane);
        if (keys) words_next[0] = ldg_at<uint16_t>(head, i4_key_words(p.B) + 8 * row + 2 * lane);
        else words_next = ldg_at<u32x2>(head, i4_value_words(p.B) + 8 * row + 8 * (lane >> 2));
        return gone;
    };
    // Coding in pieces, each beside a product: 2 d and 2 d + 1 are two pairs of dword
    // d each of the keys, of a lane's channels 2 d and 2 d + 1 of the values.
    I4Scale scale0, scale1;
    uint32_t to;                             // LDS addresses, whose 16-byte slots are told apart by exclusive or
    u32x4 coded;
    auto arrived = [&]() __attribute__((always_inline)) {
        codes = codes_next;
        words = words_next;
        asm volatile("" : "+v"(codes), "+v"(words));         // before the next are asked for
    };
    auto begin_keys = [&](int st) __attribute__((always_inline)) {
        const int r = 16 * sixteen + (lane >> 2);
        scale0 = i4_scale(words[0]);
        to = lds_at(sm.k[st] + r * D + 8 * ((4 * (lane & 3)) ^ (r & 15)));
    };
    auto begin_values = [&](int k0, int i, int gone) __attribute__((always_inline)) {
        const int quad = 4 * sixteen + (lane >> 4), c = lane & 15;
        if (gone || k0 + KT - 1 > sees0) {                   // uniform: rows that some column does not see
            // A weight of 0 does not hide a NaN: rows that no column sees become
            // zeros, and so do NaN words of the others, which are noted
            const int first = k0 + 4 * quad;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t half = 16 * (e & 1);
                const bool out = (gone >> sixteen & 1) || first + e >= end;
                const bool bad = !out && (words[e >> 1] >> half & 0x7c00u) == 0x7c00u;
                if (out || bad) words[e >> 1] &= ~(0xffffu << half);
                const uint64_t note = __builtin_amdgcn_ballot_w64(bad);
                if (lane == 0) sm.nan[i & 3][sixteen][e] = note;
            }
        }
        scale0 = i4_scale(words[0]);
        scale1 = i4_scale(words[1]);
        to = lds_at(sm.v[i & 1] + 4 * (quad * D + 8 * c) + 8 * (c >> 2));
    };
    auto piece = [&](auto keys_too, int n) __attribute__((always_inline)) {
        const int d = n >> 1, half = 2 * (n & 1);
        if constexpr (decltype(keys_too)::value) {
#pragma unroll
            for (int i = half; i < half + 2; ++i) coded[i] = i4_value(masks.pair(codes[d], i), lower(scale0.s), lower(scale0.c));
            if (n & 1) *(lds_u32x4 *)(to ^ 16 * d) = coded;
        } else {                                             // channel n: its two pairs of rows
            coded[half] = i4_value(masks.pair(codes[n >> 2], n & 3), scale0.s, scale0.c);
            coded[half + 1] = i4_value(masks.pair(codes[2 + (n >> 2)], n & 3), scale1.s, scale1.c);
            if (n & 1) *(lds_u32x4 *)(to ^ 16 * d) = coded;
        }
    };
    f32x16 sc[2];                            // rows k0 + 32 b + 8 (i / 4) + 4 h32 + i % 4 of column c32
    u32x4 pb[2][2];                          // B operand of the 16 rows (b, c): registers 8 c .. 8 c + 7
    // Operands are read AHEAD products early: a wavefront that has the matrix cores
    // for itself waits for nothing else.
    // Addresses of this lane's first operands of the keys' and the values' stage,
    // carried from period to period (what follows from them alone is made anew in
    // each: kept, it would not fit the registers).
    uint32_t from_k = lds_at(sm.k[0] + c32 * D + 8 * (h32 ^ (c32 & 15)));
    uint32_t from_v = lds_at(sm.v[0] + 4 * (h32 * D + c32));
    auto key_operand = [&](int i) __attribute__((always_inline)) {       // i: 16 channels, then which 32 rows
        return *(lds_u32x4 *)((from_k ^ 32 * (i >> 1)) + 64 * D * (i & 1));
    };
    // channel 32 db + c32 of rows 16 (i / 4) + 4 h32 + 0..3 and + 8..11, db = i % 4
    auto value_operand = [&](int i) __attribute__((always_inline)) {
        const uint32_t from = (from_v ^ 16 * (i & 3)) + 8 * D * (4 * (i >> 2)) + 8 * 32 * (i & 3);
        const u32x2 lo = *(lds_u32x2 *)from, hi = *(lds_u32x2 *)(from + 8 * D * 2);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    // Products from .. to - 1 of a period: 0 .. 15 of the values, 16 .. 31 of the keys, and the pieces of
    // what this group codes beside the last sixteen.
    u32x4 x[AHEAD];
    auto read = [&](int i) __attribute__((always_inline)) {
        x[i % AHEAD] = i < 16 ? value_operand(i) : key_operand(i - 16);
    };
    auto first_operands = [&](auto from) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) read(decltype(from)::value + i);
    };
    auto products = [&](auto from, auto to, auto group) __attribute__((always_inline)) {
        constexpr int FROM = decltype(from)::value, TO = decltype(to)::value;
        if constexpr (TO > 16)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[b][i] = 0.0f;
#pragma unroll
        for (int i = FROM; i < TO; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if (i < 16) acc[i & 3] = mma3232(x[i % AHEAD], pb[i >> 3][i >> 2 & 1], acc[i & 3]);
            else sc[i & 1] = mma3232(x[i % AHEAD], qb[(i - 16) >> 1], sc[i & 1]);
            if (i + AHEAD < TO) read(i + AHEAD);
            if (i >= TO - 16 && (i & 1)) piece(group, (i - (TO - 16)) >> 1);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr std::integral_constant<int, 0> VALUES{};
    constexpr std::integral_constant<int, 16> KEYS{};
    constexpr std::integral_constant<int, 32> ALL{};
    auto weights = [&](int k0, int gone) __attribute__((always_inline)) {
        if (gone || k0 + KT - 1 > wave0) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 32 * b + 8 * (i >> 2) + 4 * h32 + (i & 3);
                    if (k0 + r > sees || (gone >> (r >> 4) & 1)) sc[b][i] = NEG_INF;
                }
        }
        float cmax = NEG_INF;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) cmax = fmaxf(cmax, sc[b][i]);
        cmax = pair_max(cmax) * c_log2;
        // The reference is the maximum itself, at every tile: the largest weight is a power of two, whose
        // rounding to f16 vanishes.  (One that moved only past 2^8: f16 chunks of five prompts 2.7e-4 from 32-bit
        // weights' outputs, root of the mean square, instead of 1.4e-4, and 517 us instead of 529.)
        const float m_new = fmaxf(m_run, cmax), m_use = m_new == NEG_INF ? 0.0f : m_new;
        float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
        const float less = I4_BIAS - m_use;
        float lsum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[b][8 * c + 2 * w], c_log2, less));
                    const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[b][8 * c + 2 * w + 1], c_log2, less));
                    pb[b][c][w] = pack2<true>(p0, p1);
                    // by additions: a dot product of the packed pair runs on the matrix cores here, and waits
                    // for the other wavefront's products
                    lsum[w & 1] += p0;
                    lsum[w & 1] += p1;
                    // made here, beside the other wavefront's products, not where it is used
                    asm volatile("" : "+v"(pb[b][c][w]));
                }
        l_run = fmaf(l_run, alpha, lsum[0] + lsum[1]);
        m_run = m_new;
        if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
            asm volatile("" : "+v"(alpha));                  // the products stay behind the branch
#pragma unroll
            for (int db = 0; db < 4; ++db) acc[db] *= alpha;
        }
    };
    // LDS writes before a barrier are seen after it; loads in flight stay so
    auto meet = []() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    auto poisoned = [&](int k0, int i, int gone) __attribute__((always_inline)) {    // by the noted NaN of tile i
        if (!gone && k0 + KT - 1 <= sees0) return;           // uniform: no notes were made
#pragma nounroll
        for (int e = 0; e < 16; ++e) {
            const uint64_t note = sm.nan[i & 3][e >> 2][e & 3];
            if (!__builtin_amdgcn_ballot_w64(note != 0)) continue;
#pragma nounroll
            for (int j = 0; j < 16; ++j)     // quad j / 4 of the sixteen, group j % 4
                if (note >> (4 * j) & 1 && k0 + 16 * (e >> 2) + 4 * (j >> 2) + (e & 3) <= sees) poison |= 1u << (j & 3);
        }
    };
    // The two wavefronts of a SIMD complement each other: in period i the first
    // group multiplies (the values of tile i - 1, the keys of tile i) and then
    // makes the weights of tile i; the second makes those of tile i - 1 first and
    // multiplies then.  In the shadow of its products the first codes the values
    // of tile i, the second the keys of tile i + 1.  So a period reads the values
    // of tile i - 1 and the keys of tile i, and writes the other stages.
    auto run = [&](auto group) __attribute__((always_inline)) {
        constexpr bool K = decltype(group)::value;           // the second group, which codes the keys
        // gone[j]: the sixteens of tile i + j that have no page; what is asked for next is of tile i + 2 + LEAD
        constexpr int LEAD = K ? 1 : 0;
        int gone[3 + LEAD];
        look_up(t0);
        gone[0] = fetch(t0);
        look_up(t0 + KT);
        arrived();
        gone[1] = fetch(t0 + KT);
        look_up(t0 + 2 * KT);
        if constexpr (K) {
            begin_keys(0);
#pragma unroll
            for (int n = 0; n < 8; ++n) piece(group, n);
            arrived();
            gone[2] = fetch(t0 + 2 * KT);
            look_up(t0 + 3 * KT);
            begin_keys(1);
        } else {
            begin_values(t0, 0, gone[0]);
        }
        meet();
        int i = 0, k0 = t0;
        first_operands(KEYS);
        products(KEYS, ALL, group);
        constexpr uint32_t STAGE = 2 * KT * D;
        from_k ^= STAGE;
        for (;;) {
            if constexpr (K) meet();
            weights(k0, gone[0]);
            // past the last tile what is asked for and coded is not read
            arrived();
            gone[2 + LEAD] = fetch(k0 + (2 + LEAD) * KT);
            look_up(k0 + (3 + LEAD) * KT);   // taken a tile later: nothing waits for the table
            if constexpr (!K) {
                begin_values(k0 + KT, i + 1, gone[1]);
                meet();
            } else {
                begin_keys(i & 1);
            }
            poisoned(k0, i, gone[0]);
            first_operands(VALUES);
#pragma unroll
            for (int j = 0; j < 2 + LEAD; ++j) gone[j] = gone[j + 1];
            k0 += KT;
            ++i;
            products(VALUES, ALL, group);    // past the last tile too: of the keys' part nothing is taken
            if (k0 >= end) break;
            from_k ^= STAGE;
            from_v ^= STAGE;
        }
    };
    if (t0 < end) {
        if (keys) run(std::true_type{});
        else run(std::false_type{});
    }
    l_run = pair_sum(l_run);
    if (w0 + c32 >= colN) return;
#pragma unroll
    for (int db = 0; db < 4; ++db)
        if (poison >> db & 1)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[db][i] = __builtin_nanf("");
    if constexpr (DIRECT) {
        const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
        const int64_t o = (int64_t)(s.t0 + t) * a.o_st + hq * a.o_sh + 4 * h32;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                iq_store_as(a.out, o + 32 * db + 8 * (i >> 2) + (i & 3), l_run == 0.0f ? 0.0f : acc[db][i] * inv, a.odt);
    } else {
        const int64_t row = (int4_place(a, seq, s, t) * a.Hq + hq) * a.parts + part;
        float *o = a.part.o + row * D + 4 * h32;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *(f32x4 *)(o + 32 * db + 8 * g) =
                    f32x4{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
        if (h32 == 0) a.part.ml[row] = f32x2{m_run, l_run};
    }
}

}  // namespace
