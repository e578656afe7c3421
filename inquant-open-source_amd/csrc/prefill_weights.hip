// The weight each key of a prompt receives from the prompt's queries (gfx950):
//   weights[h][j] = sum over the queries i >= j and the query heads g of KV
//   head h of exp(scale q_gi . k_j - lse_gi),
// over all queries, whose lse the attention left, or over the last `window`
// of each sequence, whose lse is computed here first.
//
// Keys are the rows of S^T = K Q^T on v_mfma_f32_32x32x16 and stay in
// registers (64 per wavefront, 256 per workgroup) while tiles of 64 queries
// stream through LDS, so a key's sum over the queries is one fp32 add per
// logit in the lane that holds it, and is added over the 32 lanes (queries of
// a tile) once, at the end.  Bound by the matrix cores and the VALU together: a
// 32 x 64 half tile has 16 products of 32 cycles and, per lane, 32 exponentials
// of 8 and 64 fused multiply-adds and adds of 4, which overlap in part (311 ns a
// half and SIMD in a loop of nothing else, the products alone 227).  8192 causal
// queries, 28 heads over 4, with the heads' sums: 238-241 us, 1.0 PFLOP/s (32768:
// 3.38 ms, 1.14).
#include <type_traits>

#include "decode_common.h"

namespace {

constexpr int D = 128;
constexpr int NW = 4, NT = 64 * NW;
constexpr int KW = 64;                       // keys per wavefront
constexpr int KG = KW * NW;                  // keys per workgroup
constexpr int QT = 64;                       // queries per tile
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;

typedef __attribute__((ext_vector_type(16))) float f32x16;

struct WeightArgs {
    const uint16_t *q, *k;
    int64_t q_st, q_sh, k_st, k_sh;          // element strides (token, head)
    const int32_t *cu;
    int n_seq, max_len, H, Hq, G;              // a sequence's rows past max_len are left out
    int window;                              // WINDOW: queries of each sequence from its end
    int chunk, chunks;                       // a workgroup's queries at most, and their ranges
    float c_log2;
    const float *lse;                        // natural log, token i of head hq at hq * lse_sh + i; with lse_sh 0
    int64_t lse_sh;                          // window row r of (seq, h) at (seq * H + h) * G * window + r
    f32x2 *ml;                               // the lse pass: (max, sum) per [64-key tile, H, window row of the slice]
    int tiles64;                             // a sequence's first of those tiles: see tile_base
    int row0, ml_rows;                       // the slice: window rows row0 .. row0 + ml_rows - 1 of each KV head
    float *out;                              // [H, out_sh]; all queries: [ranges, Hq, out_sh]
    int64_t out_sh;
};

// The last queries of a sequence, and the window's rows of a KV head: row
// g n + i is query `lo` + i of its query head g.
struct Window {
    int lo, n, rows;
};

__device__ __forceinline__ Window window_of(const WeightArgs &a, int len)
{
    const int n = len < a.window ? len : a.window;
    return {len - n, n, n * a.G};
}

// Row r = g n + i of a window is query i of head g.  The quotient by a reciprocal
// is exact: rows are below 2^21, and the half keeps its error (2^-22 of it) from
// the next whole number.
__device__ __forceinline__ uint32_t head_of(int row, float rcp)
{
    return (uint32_t)(((float)row + 0.5f) * rcp);
}

// Three stages: a tile is computed while the next two are on their way.
constexpr int ST = 3;

struct __attribute__((aligned(16))) WeightSmem {
    uint16_t q[ST][QT * D];                  // chunk c of row r at slot c ^ (r % 16)
    float lse[ST][NW][QT];                   // a copy per wavefront
};
static_assert(2 * sizeof(WeightSmem) <= 160 * 1024, "two workgroups per compute unit");

// lds_load16 from an address of each lane's own
__device__ __forceinline__ void lds_gather16(const void *p, uint32_t lds_base)
{
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"((uint64_t)(uintptr_t)p),
                 "s"(__builtin_amdgcn_readfirstlane(lds_base))
                 : "memory");
}

__device__ __forceinline__ void lds_gather4(const void *p, uint32_t lds_base)
{
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dword %0, off" ::"v"((uint64_t)(uintptr_t)p),
                 "s"(__builtin_amdgcn_readfirstlane(lds_base))
                 : "memory");
}

// lds_load16 with four bytes per lane
__device__ __forceinline__ void lds_load4(const void *base, uint32_t voff, uint32_t lds_base)
{
    const uint64_t b = (uint64_t)(uintptr_t)base;
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32));
    const uint64_t sb = (uint64_t)lo | ((uint64_t)hi << 32);
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(sb),
                 "s"(__builtin_amdgcn_readfirstlane(lds_base))
                 : "memory");
}

template <bool F16>
__device__ __forceinline__ f32x16 mma3232(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
}

__device__ __forceinline__ int length_of(const WeightArgs &a, int seq)
{
    const int len = a.cu[seq + 1] - a.cu[seq];
    return len < a.max_len ? len : a.max_len;
}

// The lse pass keeps its (max, sum) per 64 keys: sequence i's from tile i * tiles64
// on, or with tiles64 0 from cu[i] / 64 + i on (no two overlap: of consecutive
// sequences the base grows by cu[i + 1] / 64 - cu[i] / 64 + 1, at least the tiles
// of sequence i), so that one long prompt of a batch does not size the others'.
__device__ __forceinline__ int64_t tile_base(const WeightArgs &a, int seq)
{
    return a.tiles64 ? (int64_t)seq * a.tiles64 : (int64_t)(a.cu[seq] / KW) + seq;
}

// over the lane pair l, l ^ 32 (one query's two halves)
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

// Of 2 N values of each lane, lanes with bit N set keep the upper half, the others
// the lower, with their partner's (CTRL; its bit N is the other) added.
template <int N, int CTRL>
__device__ __forceinline__ void halve(float *v, int lane)
{
    const bool upper = lane & N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float keep = upper ? v[i + N] : v[i], give = upper ? v[i] : v[i + N];
        v[i] = keep + dpp_f<CTRL>(give);
    }
}

enum Pass { ALL, WINDOW, WINDOW_LSE };

// ALL: the keys' sums over the queries of one query head and range; WINDOW:
// over the rows of the window (packed: the query heads of a KV head follow each
// other, so that small windows fill the tiles); WINDOW_LSE: (max, sum) of every
// window row over this workgroup's keys, per wavefront.
template <bool F16, Pass PASS>
__global__ __launch_bounds__(NT, 2) void prefill_weights(WeightArgs a)
{
    constexpr bool LSEPASS = PASS == WINDOW_LSE, ROWS = PASS != ALL;
    __shared__ WeightSmem sm;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c32 = lane & 31, h32 = lane >> 5;
    // An item is a (query range, key tile, sequence, head), the longest first:
    // ranges that see all of a key tile's queries (the last range, which may be
    // short, after the others), then the ranges on the diagonal, whose j-th key
    // tile sees all queries but 256 j.
    const int lists = ROWS ? a.H : a.Hq;
    int rest = blockIdx.x / lists;
    const int list = blockIdx.x - rest * lists, h = ROWS ? list : list / a.G;
    const int seq = rest % a.n_seq;
    rest /= a.n_seq;
    int tile = rest, range = 0;
    if constexpr (!ROWS) {
        const int m = a.chunk / KG, full = m * a.chunks * (a.chunks - 1) / 2;    // key tiles per range; whole items
        if (rest < full) {
            range = a.chunks > 2 ? a.chunks - 2 : 1;
            while (tile >= range * m) {
                tile -= range * m;
                range = range > 1 ? range - 1 : a.chunks - 1;
            }
        } else {
            rest -= full;
            range = a.chunks - 1 - rest % a.chunks;
            tile = range * m + rest / a.chunks;
        }
    }
    const int start = a.cu[seq], len = length_of(a, seq);
    const int g0 = tile * KG, from = range * a.chunk;
    // "queries" are query positions, or with ROWS rows of the window
    const Window win = window_of(a, len);
    const int slice = LSEPASS ? a.row0 + a.ml_rows : win.rows;
    const int end = ROWS ? win.rows < slice ? win.rows : slice : len - from < a.chunk ? len : from + a.chunk;
    const int q0 = LSEPASS ? a.row0 : ROWS ? 0 : g0 > from ? g0 : from;  // the first that sees one of these keys
    if (g0 >= (ROWS ? len : end) || from >= len || LSEPASS && q0 >= end) return;     // uniform
    const int k0 = g0 + KW * wave;           // this wavefront's first key
    f32x2 *const ml = LSEPASS ? a.ml + ((tile_base(a, seq) + k0 / KW) * a.H + h) * a.ml_rows - a.row0 : nullptr;
    u32x4 kf[2][8];                          // A operand: key k0 + 32 kb + c32, channels 16 d + 8 h32 .. + 7
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        const int key = k0 + 32 * kb + c32, kk = key < len ? key : len - 1;
        const uint16_t *kp = a.k + (int64_t)(start + kk) * a.k_st + (int64_t)h * a.k_sh + 8 * h32;
#pragma unroll
        for (int d = 0; d < 8; ++d) kf[kb][d] = ld16(kp + 16 * d);
    }
    f32x16 sum[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[kb][i] = 0.0f;
    const int total = (end - q0 - 1) / QT + 1;
    const int last_tile = q0 + (total - 1) * QT;            // the tiles go from the last back
    const uint32_t lds_q = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t *)&sm.q[0][0];
    const uint32_t lds_l = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) float *)&sm.lse[0][wave][0];
    // Direct loads of the next tile, and its place: sixteen of its rows per
    // wavefront, four (1 KB) per load, and its lse; rows past the end repeat
    // the last one.
    int next_qa = last_tile;
    const uint32_t row_bytes = (uint32_t)a.q_st * 2, head_bytes = (uint32_t)a.q_sh * 2;
    const float win_rcp = 1.0f / (float)win.n;
    uint32_t whole[4];                       // a load's offset where no row is past the end
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 16 * wave + 4 * i + (lane >> 4);
        whole[i] = r * row_bytes + 16 * ((lane & 15) ^ (r & 15));
    }
    const float *own_lse = a.lse + (int64_t)(seq * a.H + h) * a.G * a.window;
    auto load_tile = [&](int st) {
        const int last = end - 1 - next_qa;
        const uint32_t to_l = lds_l + (uint32_t)(st * NW * QT * 4);
        if constexpr (ROWS) {
            // query head (of this KV head) and query of the tile's row r
            auto place = [&](int r, uint32_t &g, uint32_t &i) {
                const int row = next_qa + (r < last ? r : last);
                g = head_of(row, win_rcp);
                i = (uint32_t)row - g * (uint32_t)win.n;
                return row;
            };
            uint32_t g, i;
            if constexpr (!LSEPASS) {
                const int row = place(lane, g, i);
                lds_gather4(a.lse_sh ? (const char *)(a.lse + (int64_t)h * a.G * a.lse_sh + start + win.lo) +
                                           (int64_t)g * a.lse_sh * 4 + 4 * i
                                     : (const char *)(own_lse + row), to_l);
            }
            const char *first = (const char *)(a.q + (int64_t)(start + win.lo) * a.q_st + (int64_t)h * a.G * a.q_sh);
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const int r = 16 * wave + 4 * l + (lane >> 4);
                place(r, g, i);
                lds_gather16(first + (uint64_t)i * row_bytes + (uint64_t)g * head_bytes + 16 * ((lane & 15) ^ (r & 15)),
                             lds_q + (uint32_t)((st * QT + 16 * wave + 4 * l) * D * 2));
            }
        } else {
            const uint16_t *qt = a.q + (int64_t)(start + next_qa) * a.q_st + (int64_t)list * a.q_sh;
            lds_load4(a.lse + (int64_t)list * a.lse_sh + start + next_qa, (uint32_t)(lane < last ? lane : last) * 4, to_l);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t off = whole[i];
                if (last < QT - 1) {
                    const int r = 16 * wave + 4 * i + (lane >> 4);
                    off -= (uint32_t)(r > last ? r - last : 0) * row_bytes;
                }
                lds_load16(qt, off, lds_q + (uint32_t)((st * QT + 16 * wave + 4 * i) * D * 2));
            }
        }
        next_qa -= QT;
    };
    load_tile(0);
    if (total > 1) load_tile(1);
    if (total > 2) load_tile(2);
    // the keys are waited for here, not in the loop
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int d = 0; d < 8; ++d) asm volatile("" : "+v"(kf[kb][d]));
    // Operands of 32 queries (column 32 b + c32, channels 16 d + 8 h32 .. + 7)
    // and their logits S^T (keys k0 + 32 kb + 8 (i / 4) + 4 h32 + i % 4).  Each
    // operand is replaced by the next half tile's as soon as it was used.
    u32x4 qv[8];
    auto operand = [&](int st, int b, int d) {
        return *(const u32x4 *)(sm.q[st] + (32 * b + c32) * D + 8 * ((2 * d + h32) ^ (c32 & 15)));
    };
    // Logits that are still to be worked off, of the half tile before: their
    // query's lse, or the row whose (max, sum) they give.
    f32x16 late[2];
    float late_lse2 = 0.0f;
    int late_row = -1;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) late[kb][i] = NEG_INF;
    float m = 0.0f, use = 0.0f, l = 0.0f;
    // Two of a lane's 32 logits, in half e of step d of 8.
    auto work_off = [&](int d, int part) {
        if constexpr (LSEPASS) {
            if (d == 0 && part == 0) {
                m = NEG_INF;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) m = fmaxf(m, late[kb][i]);
                m = pair_max(m * a.c_log2);
                use = m == NEG_INF ? 0.0f : m;
                l = 0.0f;
            }
#pragma unroll
            for (int e = 2 * part; e < 2 * part + 2; ++e)
                l += __builtin_amdgcn_exp2f(fmaf(late[d >> 2][4 * (d & 3) + e], a.c_log2, -use));
            if (d == 7 && part == 1) {
                l = pair_sum(l);
                if (h32 == 0 && late_row >= 0) ml[late_row] = f32x2{m, l};
            }
        } else {
#pragma unroll
            for (int e = 2 * part; e < 2 * part + 2; ++e) {
                const int kb = d >> 2, i = 4 * (d & 3) + e;
                sum[kb][i] += __builtin_amdgcn_exp2f(fmaf(late[kb][i], a.c_log2, -late_lse2));
            }
        }
    };
    // The products of a half tile beside what the half before leaves to do: the
    // matrix cores and the VALU have about the same work here (16 products of 32
    // cycles; 32 exponentials of 8 and 64 other instructions of 4), and the
    // barriers hold the compiler to it.
    auto products = [&](int st, int b, f32x16 *sc) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kb][i] = 0.0f;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            sc[0] = mma3232<F16>(kf[0][d], qv[d], sc[0]);
            work_off(d, 0);
            __builtin_amdgcn_sched_barrier(0);
            sc[1] = mma3232<F16>(kf[1][d], qv[d], sc[1]);
            qv[d] = operand(st, b, d);
            work_off(d, 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!LSEPASS) asm volatile("" : "+v"(sum[0]), "+v"(sum[1]));   // added here, not at the loop's end
    };
    constexpr int LOADS = LSEPASS ? 4 : 5;   // of a tile, per wavefront
    int qa = last_tile, it = 0;
    // Half b of the tile in stage st, leaving the operands of the next half.
    auto half = [&](auto st_, auto b_) {
        constexpr int st = decltype(st_)::value, b = decltype(b_)::value;
        const int query = qa + 32 * b + c32;
        // a query past the end weighs nothing
        float lse2 = 0.0f;
        if constexpr (!LSEPASS) lse2 = query < end ? sm.lse[st][wave][32 * b + c32] * LOG2E : __builtin_inff();
        if constexpr (b == 1) {
            // This half's operands are in registers, so the tile has been read;
            // the next tile's loads have landed; after the barrier both hold for
            // every wavefront.
            if (it + 2 < total)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (it + 3 < total) load_tile(st);
        }
        f32x16 sc[2];
        products(b ? (st + 1) % ST : st, 1 - b, sc);
        const bool masked = (ROWS ? win.lo : qa + 32 * b) < k0 + KW || k0 + KW > len;    // uniform
        // A lane's keys, in the order of bit 16 kb + i, that its query does not see.  Taken
        // apart as one mask: a compare and a selection per key wait for each other's
        // condition (18 cycles a key, and 8).
        uint32_t unseen = 0;
        if (masked) {
            const int row = query < end ? query : end - 1;
            const int at = ROWS ? win.lo + row - (int)head_of(row, win_rcp) * win.n : row;
            const int n = at - k0 - 4 * h32 + 1;             // keys up to the query's own, from k0 + 4 h32
            const int bits = n <= 0 ? 0 : 4 * (n >> 3) + ((n & 7) < 4 ? n & 7 : 4);
            unseen = bits < 32 ? ~0u << bits : 0;
        }
        auto instead = [&](int kb, int i, uint32_t other, float x) {    // `other` where the key is unseen
            uint32_t y;
            asm("v_bfi_b32 %0, %1, %2, %3"
                : "=v"(y)
                : "v"(__builtin_amdgcn_sbfe((int)unseen, 16 * kb + i, 1)), "s"(other), "v"(__float_as_uint(x)));
            return __uint_as_float(y);
        };
        late[0] = sc[0];
        late[1] = sc[1];
        late_lse2 = lse2;
        late_row = query < end && k0 < len ? query : -1;
        if (masked) {
            // an lse that is NaN or -inf would turn the unseen's -inf into NaN
            if (LSEPASS || !__builtin_amdgcn_ballot_w64(!(lse2 > NEG_INF))) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)             // the scale is positive
                        late[kb][i] = instead(kb, i, __float_as_uint(NEG_INF), sc[kb][i]);
            } else {
                // added at once, the unseen left out, so that nothing is pending
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float w = __builtin_amdgcn_exp2f(fmaf(sc[kb][i], a.c_log2, -lse2));
                        sum[kb][i] += instead(kb, i, 0, w);
                        late[kb][i] = NEG_INF;
                    }
                late_lse2 = 0.0f;
            }
        }
    };
    auto next = [&]() {
        qa -= QT;
        return ++it < total;
    };
    if (total > 2) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int d = 0; d < 8; ++d) qv[d] = operand(0, 0, d);
    const std::integral_constant<int, 0> zero{};
    const std::integral_constant<int, 1> one{};
    const std::integral_constant<int, 2> two{};
    while (true) {
        half(zero, zero);
        half(zero, one);
        if (!next()) break;
        half(one, zero);
        half(one, one);
        if (!next()) break;
        half(two, zero);
        half(two, one);
        if (!next()) break;
    }
#pragma unroll
    for (int d = 0; d < 16; ++d) work_off(d >> 1, d & 1);
    if constexpr (!LSEPASS) {
        float *out = a.out + ((int64_t)range * a.Hq + list) * a.out_sh + start;
        // Sums over the 32 queries: a swap of the odd 16-lane rows of one key's
        // lanes with the even ones of another's leaves both keys in one register
        // (the first block's in the even rows, the second's in the odd); then the
        // lanes of a row halve the 16 keys that they add for each other, until
        // lane i holds key i.
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum[0][i]), __float_as_uint(sum[1][i]),
                                                            false, false);
            v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
        halve<8, 0x140>(v, lane);                            // row_mirror
        halve<4, 0x141>(v, lane);                            // row_half_mirror
        halve<2, 0x4e>(v, lane);                             // quad_perm: xor 2
        halve<1, 0xb1>(v, lane);                             // xor 1
        const int i = lane & 15, key = k0 + 32 * ((lane >> 4) & 1) + 8 * (i >> 2) + 4 * h32 + (i & 3);
        if (key < len) out[key] = v[0];
    }
}

// lse of the window's rows from the (max, sum) of their key tiles: sixteen rows
// of a (sequence, KV head) per workgroup, the key tiles over 64 groups of lanes.
constexpr int LR = 16, LG = 64;

__global__ __launch_bounds__(LR * LG) void window_lse(WeightArgs a, float *lse)
{
    __shared__ f32x2 sm[LG][LR];
    const int seq = blockIdx.z, h = blockIdx.y, lane = threadIdx.x % LR, group = threadIdx.x / LR;
    const int len = length_of(a, seq), row = a.row0 + blockIdx.x * LR + lane;
    const Window win = window_of(a, len);
    const bool live = row < win.rows && row < a.row0 + a.ml_rows;
    f32x2 mine = {NEG_INF, 0.0f};
    auto join = [](f32x2 x, f32x2 y) {
        const float m = fmaxf(x[0], y[0]), use = m == NEG_INF ? 0.0f : m;
        return f32x2{m, x[1] * __builtin_amdgcn_exp2f(x[0] - use) + y[1] * __builtin_amdgcn_exp2f(y[0] - use)};
    };
    if (live) {
        // the tiles that hold a key at or before the last query (the others' keys are unseen: (-inf, 0))
        const f32x2 *ml = a.ml + (tile_base(a, seq) * a.H + h) * a.ml_rows + row - a.row0;
#pragma unroll 4
        for (int t = group; t <= (len - 1) / KW; t += LG) mine = join(mine, ml[(int64_t)t * a.H * a.ml_rows]);
    }
    sm[group][lane] = mine;
    __syncthreads();
    if (group >= 4) return;                  // the first wavefront
#pragma unroll
    for (int g = group + 4; g < LG; g += 4) mine = join(mine, sm[g][lane]);
#pragma unroll
    for (int d = 16; d < 64; d *= 2) mine = join(mine, f32x2{__shfl_xor(mine[0], d), __shfl_xor(mine[1], d)});
    if (group == 0 && live) {
        const int g = (int)head_of(row, 1.0f / (float)win.n);
        float *to = a.lse_sh ? lse + (int64_t)(h * a.G + g) * a.lse_sh + a.cu[seq] + win.lo + row - g * win.n
                             : lse + ((int64_t)seq * a.H + h) * a.G * a.window + row;
        // as the attention's: a maximum of -inf leaves -inf, or NaN if one logit was
        *to = (mine[0] + __builtin_amdgcn_logf(mine[1])) * LN2;
    }
}

// The sums of each KV head's query heads and of the query ranges that see a key.
__global__ __launch_bounds__(256) void add_heads(WeightArgs a, const float *part, int64_t tokens, float *out,
                                                 int64_t out_sh)
{
    const int h = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x, len = length_of(a, blockIdx.z);
    if (i >= len) return;
    const int64_t at = a.cu[blockIdx.z] + i;
    float v = 0.0f;
    for (int range = i / a.chunk; range <= (len - 1) / a.chunk; ++range)
        for (int g = 0; g < a.G; ++g) v += part[((int64_t)range * a.Hq + h * a.G + g) * tokens + at];
    out[h * out_sh + at] = v;
}

struct Scratch {
    int64_t lse, ml, part;                   // floats of each
    int64_t tiles;                           // 64-key tiles that ml holds of each head and row
    bool by_seq;                             // a sequence's tiles: as many for each; else by its tokens
    int64_t lse_sh;                          // the own lse: 0 by window rows, else [Hq, tokens]
};

// The lse pass goes over the window's rows in slices whose (max, sum) take 256 MiB
// at most, or 64 rows: a 4096-query window over 32K tokens, 28 heads over 4, has
// 470 MB of them, 64 queries over 32K 7 (one slice, as everything below the bound).
constexpr int64_t ML_MOST = 1 << 26;         // floats

// Queries of a workgroup at most, a power of two and of whole key tiles (so that a
// range sees a whole key tile or ends before it): the one for which the longest
// prompt ends first, by the 64-query tiles of all workgroups over the 512 places,
// those of the longest workgroup, and some of its tail; a workgroup's start counts
// as four tiles.  The starts weigh against short ranges, idle places against long
// ones (28 heads over 4, 8192 queries: 4096 a workgroup, 241 us, and 255 with all of
// them; 4096 queries: 1024, 84 us against 92 with the tiles in order and no
// estimate; 1000 queries: 512, 23 us, and 26 with 256; 32768 queries: 16384, 3.38 ms,
// 3.41 with 8192 and 3.43 with all of them.  From 64K on the sizes are within 2%).
int64_t chunk_of(int64_t Hq, int64_t n_seq, int64_t max_seqlen)
{
    int64_t best = 512;
    double least = 1e30;
    for (int64_t chunk = best; chunk <= 131072; chunk *= 2) {
        const int64_t ranges = (max_seqlen + chunk - 1) / chunk;
        double all = 0, longest = 0;
        for (int64_t r = 0; r < ranges; ++r) {
            const int64_t n = max_seqlen - r * chunk < chunk ? max_seqlen - r * chunk : chunk;   // its queries
            const double whole = (double)((n + QT - 1) / QT), diagonal = (double)((n + KG - 1) / KG);
            all += (double)(r * chunk / KG) * (whole + 4) + diagonal * (whole / 2 + 4);
            longest = whole + 4 > longest ? whole + 4 : longest;
        }
        all *= (double)(Hq * n_seq) / 512;
        const double cost = (all > longest ? all : longest) + longest / 8;
        if (cost < least) {
            least = cost;
            best = chunk;
        }
        if (ranges == 1) break;
    }
    return best;
}

Scratch scratch_of(int64_t Hq, int64_t n_seq, int64_t max_seqlen, int64_t tokens, int64_t window, bool lse)
{
    Scratch s{};
    if (window > 0 && !lse) {
        const int64_t even = n_seq * ((max_seqlen + KW - 1) / KW), sum = tokens / KW + n_seq;
        s.by_seq = even <= sum || 2 * even * Hq * window <= ML_MOST;
        s.tiles = s.by_seq ? even : sum;
        s.lse_sh = n_seq * window <= tokens ? 0 : tokens;
        s.lse = Hq * (s.lse_sh ? tokens : n_seq * window);
        const int64_t whole = 2 * s.tiles * Hq * window, least = 2 * s.tiles * Hq * QT;
        const int64_t most = ML_MOST > least ? ML_MOST : least;
        s.ml = whole < most ? whole : most;
    }
    if (window == 0) {
        const int64_t chunk = chunk_of(Hq, n_seq, max_seqlen);
        s.part = (max_seqlen + chunk - 1) / chunk * Hq * tokens;
    }
    return s;
}

}  // namespace

extern "C" int64_t iq_prefill_weights_floats(int64_t Hq, int64_t n_seq, int64_t max_seqlen, int64_t tokens,
                                             int64_t window, int have_lse)
{
    const Scratch s = scratch_of(Hq, n_seq, max_seqlen, tokens, window, have_lse != 0);
    return s.lse + s.ml + s.part;
}

extern "C" int iq_prefill_weights(const void *q, const void *k, int dtype, int64_t q_st, int64_t q_sh, int64_t k_st,
                                  int64_t k_sh, const int32_t *cu_seqlens, int64_t n_seq, int64_t max_seqlen,
                                  int64_t tokens, int64_t Hq, int64_t H, int64_t window, float scale, const float *lse,
                                  int64_t lse_sh, float *workspace, int64_t workspace_floats, float *out,
                                  int64_t out_sh, void *stream)
{
    IQ_CHECK_ARG(q && k && cu_seqlens && out, "iq_prefill_weights: null pointer");
    IQ_CHECK_ARG(dtype == IQ_BF16 || dtype == IQ_F16, "iq_prefill_weights: q/k must be bf16 or f16");
    IQ_CHECK_ARG(H >= 1 && Hq >= 1 && Hq % H == 0 && Hq <= 65535, "iq_prefill_weights: heads %lld / %lld",
                 (long long)Hq, (long long)H);
    IQ_CHECK_ARG(n_seq >= 1 && n_seq <= 65535 && max_seqlen >= 1 && max_seqlen <= 0x3fffffff && tokens >= 0 &&
                     tokens <= 0x7fffffffLL,
                 "iq_prefill_weights: bad sequence count or length");
    IQ_CHECK_ARG(((uintptr_t)q | (uintptr_t)k) % 16 == 0 && (q_st | q_sh | k_st | k_sh) % 8 == 0,
                 "iq_prefill_weights: q/k rows must be 16-byte aligned");
    // a query tile's rows are addressed by 32-bit byte offsets from its first row
    IQ_CHECK_ARG(q_st >= 0 && q_st < (1LL << 25) && q_sh >= 0 && q_sh < (1LL << 31),
                 "iq_prefill_weights: query strides too large");
    IQ_CHECK_ARG(Hq / H * window < (1LL << 21), "iq_prefill_weights: window too large");
    IQ_CHECK_ARG(scale > 0.0f, "iq_prefill_weights: the scale must be positive");
    IQ_CHECK_ARG(window >= 0 && window <= 65536 && (window > 0 || lse), "iq_prefill_weights: no window and no lse");
    IQ_CHECK_ARG(!lse || lse_sh > 0, "iq_prefill_weights: bad lse stride");
    // Few rows: all of them as one window, whose workgroups sum the query heads
    // themselves (called in a row, two prompts of 20 tokens, 28 heads over 4, 140
    // rows: 9.8 us, and 11.2 with a launch that adds the heads' sums; of 40
    // tokens, 280 rows: 13.9 and 11.1).
    if (window == 0 && Hq / H * max_seqlen <= 192) window = max_seqlen;
    const Scratch s = scratch_of(Hq, n_seq, max_seqlen, tokens, window, lse != nullptr);
    IQ_CHECK_ARG(s.lse + s.ml + s.part == 0 || (workspace && workspace_floats >= s.lse + s.ml + s.part),
                 "iq_prefill_weights: workspace too small");
    const int64_t tiles = (max_seqlen + KG - 1) / KG, G = Hq / H;
    const int64_t chunk = window ? 1 << 30 : chunk_of(Hq, n_seq, max_seqlen), chunks = (max_seqlen + chunk - 1) / chunk;
    WeightArgs a{(const uint16_t *)q, (const uint16_t *)k, q_st, q_sh, k_st, k_sh, cu_seqlens, (int)n_seq,
                 (int)max_seqlen, (int)H, (int)Hq, (int)G, (int)window, (int)chunk, (int)chunks,
                 scale * LOG2E, lse, lse_sh, (f32x2 *)workspace, s.by_seq ? (int)((max_seqlen + KW - 1) / KW) : 0, 0, 0,
                 out, out_sh};
    const hipStream_t st = (hipStream_t)stream;
    const bool f16 = dtype == IQ_F16;
    const int64_t m = chunk / KG, units = window ? tiles : m * chunks * (chunks - 1) / 2 + m * chunks;
    const int64_t items = units * (window ? H : Hq) * n_seq;
    IQ_CHECK_ARG(items <= 0xffffff, "iq_prefill_weights: too many key tiles");
    const dim3 grid((unsigned)items), block(NT);
    if (window > 0) {
        if (!lse) {
            float *own = workspace + s.ml;
            const int64_t fit = s.ml / (2 * s.tiles * H);    // whole tiles of rows, as without slices
            a.lse_sh = s.lse_sh;
            a.ml_rows = (int)(fit < G * window ? fit / QT * QT : G * window);
            for (int64_t row0 = 0; row0 < G * window; row0 += a.ml_rows) {
                const int64_t rows = G * window - row0 < a.ml_rows ? G * window - row0 : a.ml_rows;
                a.row0 = (int)row0;
                hipLaunchKernelGGL((f16 ? prefill_weights<true, WINDOW_LSE> : prefill_weights<false, WINDOW_LSE>), grid,
                                   block, 0, st, a);
                hipLaunchKernelGGL(window_lse, dim3((unsigned)((rows + LR - 1) / LR), (unsigned)H, (unsigned)n_seq),
                                   dim3(LR * LG), 0, st, a, own);
            }
            a.lse = own;
        }
        hipLaunchKernelGGL((f16 ? prefill_weights<true, WINDOW> : prefill_weights<false, WINDOW>), grid, block, 0, st,
                           a);
    } else {
        const bool whole = G == 1 && chunks == 1;            // each sum is one workgroup's
        if (!whole) {
            a.out = workspace;
            a.out_sh = tokens;
        }
        hipLaunchKernelGGL((f16 ? prefill_weights<true, ALL> : prefill_weights<false, ALL>), grid, block, 0, st, a);
        if (!whole)
            hipLaunchKernelGGL(add_heads, dim3((unsigned)((max_seqlen + 255) / 256), (unsigned)H, (unsigned)n_seq),
                               dim3(256), 0, st, a, workspace, tokens, out, out_sh);
    }
    IQ_CHECK_LAUNCH("prefill_weights");
    return IQ_OK;
}

extern "C" int iq_prefill_weights_from(const iq_prefill_weights_args *a)
{
    IQ_CHECK_ARG(a, "iq_prefill_weights: null arguments");
    return iq_prefill_weights((const void *)a->q, (const void *)a->k, (int)a->dtype, a->q_st, a->q_sh, a->k_st,
                              a->k_sh, (const int32_t *)a->cu_seqlens, a->n_seq, a->max_seqlen, a->tokens, a->Hq,
                              a->H, a->window, (float)a->scale, (const float *)a->lse, a->lse_sh,
                              (float *)a->workspace, a->workspace_floats, (float *)a->out, a->out_sh,
                              (void *)a->stream);
}
