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
// a tile) once, at the end.
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
    int heads;                               // query heads a workgroup sums: 1, or G
    int64_t window;                          // queries of each sequence from its end (all: its length)
    int chunk, chunks, tiles;                // a workgroup's queries at most, their ranges, and key tiles
    float c_log2;
    const float *lse;                        // natural log; token i of head hq at hq * lse_sh + i, or with
    int64_t lse_sh;                          // `windowed`, window row i at ((seq * Hq) + hq) * window + i
    int windowed;
    f32x2 *ml;                               // the lse pass: (max, sum) per [seq, 64-key tile, Hq, window]
    int tiles64;
    float *out;                              // [H or Hq, out_sh]
    int64_t out_sh;
};

// Three stages: a tile is computed while the next two are on their way.
constexpr int ST = 3;

struct __attribute__((aligned(16))) WeightSmem {
    uint16_t q[ST][QT * D];                  // chunk c of row r at slot c ^ (r % 16)
    float lse[ST][NW][QT];                   // a copy per wavefront
};
static_assert(2 * sizeof(WeightSmem) <= 160 * 1024, "two workgroups per compute unit");

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

__device__ __forceinline__ float pair_max(float v) { return fmaxf(v, __shfl_xor(v, 32)); }

__device__ __forceinline__ float pair_sum(float v) { return v + __shfl_xor(v, 32); }

// LSEPASS: (max, sum) of every window query over this workgroup's keys, per
// wavefront; else the keys' sums of exp(logit - lse).
template <bool F16, bool LSEPASS>
__global__ __launch_bounds__(NT, 2) void prefill_weights(WeightArgs a)
{
    __shared__ WeightSmem sm;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c32 = lane & 31, h32 = lane >> 5;
    // An item is a (query range, key tile, sequence, head); the ranges go from
    // the last back and the key tiles from the first on, so the workgroups that
    // start together read the same queries and the ranges' short last items
    // (on the diagonal) come after their long ones.
    const int lists = a.Hq / a.heads;
    int rest = blockIdx.x / lists;
    const int first_head = (blockIdx.x - rest * lists) * a.heads, h = first_head / a.G;
    const int seq = rest % a.n_seq;
    rest /= a.n_seq;
    const int tile = rest % a.tiles, range = a.chunks - 1 - rest / a.tiles;
    const int start = a.cu[seq], len = length_of(a, seq);
    const int g0 = tile * KG, from = range * a.chunk;
    const int end = len - from < a.chunk ? len : from + a.chunk;             // queries before it
    if (g0 >= end || from >= len) return;    // uniform
    int q0 = (int64_t)len > a.window ? len - (int)a.window : 0;              // the window's first query
    const int lo = q0;
    q0 = q0 > g0 ? q0 : g0;                  // the first that sees one of these keys
    q0 = q0 > from ? q0 : from;
    const int k0 = g0 + KW * wave;           // this wavefront's first key
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
    const int last_tile = q0 + (end - q0 - 1) / QT * QT;    // a head's tiles go from its last query back
    const int total = ((end - q0 - 1) / QT + 1) * a.heads;
    const uint32_t lds_q = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t *)&sm.q[0][0];
    const uint32_t lds_l = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) float *)&sm.lse[0][wave][0];
    // Direct loads of the next tile, and its place: sixteen of its rows per
    // wavefront, four (1 KB) per load, and its lse; rows past the end repeat
    // the last one.
    int next_head = first_head, next_qa = last_tile;
    const uint32_t row_bytes = (uint32_t)a.q_st * 2;
    uint32_t whole[4];                       // a load's offset where no row is past the end
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 16 * wave + 4 * i + (lane >> 4);
        whole[i] = r * row_bytes + 16 * ((lane & 15) ^ (r & 15));
    }
    auto load_tile = [&](int st) {
        const uint16_t *qt = a.q + (int64_t)(start + next_qa) * a.q_st + (int64_t)next_head * a.q_sh;
        const int last = end - 1 - next_qa;
        if constexpr (!LSEPASS) {
            const float *lt = a.lse + (a.windowed ? ((int64_t)seq * a.Hq + next_head) * a.window + (next_qa - lo)
                                                  : (int64_t)next_head * a.lse_sh + start + next_qa);
            lds_load4(lt, (uint32_t)(lane < last ? lane : last) * 4, lds_l + (uint32_t)(st * NW * QT * 4));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t off = whole[i];
            if (last < QT - 1) {
                const int r = 16 * wave + 4 * i + (lane >> 4);
                off -= (uint32_t)(r > last ? r - last : 0) * row_bytes;
            }
            lds_load16(qt, off, lds_q + (uint32_t)((st * QT + 16 * wave + 4 * i) * D * 2));
        }
        next_qa -= QT;
        if (next_qa < q0) {
            next_qa = last_tile;
            ++next_head;
        }
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
    // logits whose weights are still to be added, and their query's lse
    f32x16 late[2];
    float late_lse2 = 0.0f;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) late[kb][i] = NEG_INF;
    auto add_weight = [&](int kb, int i) {
        sum[kb][i] += __builtin_amdgcn_exp2f(fmaf(late[kb][i], a.c_log2, -late_lse2));
    };
    // The products of a half tile, in the lse pass alone, else beside the
    // weights of the half before: the matrix cores and the VALU have about the
    // same work here (16 products of 32 cycles; 32 exponentials of 8 and 64
    // other instructions of 4), and the barriers hold the compiler to it.
    auto products = [&](int st, int b, f32x16 *sc) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kb][i] = 0.0f;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) sc[kb] = mma3232<F16>(kf[kb][d], qv[d], sc[kb]);
            qv[d] = operand(st, b, d);
            if constexpr (!LSEPASS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) add_weight(d >> 2, 4 * (d & 3) + e);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (!LSEPASS) asm volatile("" : "+v"(sum[0]), "+v"(sum[1]));   // added here, not at the loop's end
    };
    constexpr int LOADS = LSEPASS ? 4 : 5;   // of a tile, per wavefront
    int head = first_head, qa = last_tile, it = 0;
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
        const bool masked = qa + 32 * b < k0 + KW || k0 + KW > len;          // uniform
        const int lim = (query < len ? query : len - 1) - k0 - 4 * h32;      // the last key that the query sees
        auto seen = [&](int kb, int i) { return 32 * kb + 8 * (i >> 2) + (i & 3) <= lim; };
        if constexpr (!LSEPASS) {
            late[0] = sc[0];
            late[1] = sc[1];
            late_lse2 = lse2;
            if (masked) {
                // added at once, the unseen left out (whatever their logit and lse), so that nothing is pending
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float w = __builtin_amdgcn_exp2f(fmaf(sc[kb][i], a.c_log2, -lse2));
                        sum[kb][i] += seen(kb, i) ? w : 0.0f;
                        late[kb][i] = NEG_INF;
                    }
                late_lse2 = 0.0f;
            }
        } else if (k0 < len && k0 <= qa + QT - 1) {          // some query of this tile sees a key of this wavefront
            if (masked) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sc[kb][i] = seen(kb, i) ? sc[kb][i] : NEG_INF;   // the scale is positive
            }
            float m = NEG_INF, l = 0.0f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) m = fmaxf(m, sc[kb][i]);
            m = pair_max(m * a.c_log2);
            const float use = m == NEG_INF ? 0.0f : m;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) l += __builtin_amdgcn_exp2f(fmaf(sc[kb][i], a.c_log2, -use));
            l = pair_sum(l);
            if (h32 == 0 && query < end)
                a.ml[(((int64_t)seq * a.tiles64 + k0 / KW) * a.Hq + head) * a.window + (query - lo)] = f32x2{m, l};
        }
    };
    auto next = [&]() {
        qa -= QT;
        if (qa < q0) {
            qa = last_tile;
            ++head;
        }
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
    if constexpr (!LSEPASS) {
#pragma unroll
        for (int i = 0; i < 32; ++i) add_weight(i >> 4, i & 15);
        float *out = a.out + ((int64_t)range * a.Hq + (a.heads == 1 ? first_head : h)) * a.out_sh + start;
        // Sums over the 32 queries: a swap of the odd 16-lane rows of one key's
        // lanes with the even ones of another's leaves both keys in one register
        // (the first block's in the even rows, the second's in the odd).
        const int kb = (lane >> 4) & 1;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum[0][i]), __float_as_uint(sum[1][i]),
                                                            false, false);
            const float v = row_sum16(__uint_as_float(r[0]) + __uint_as_float(r[1]));
            const int key = k0 + 32 * kb + 8 * (i >> 2) + 4 * h32 + (i & 3);
            if ((lane & 15) == 0 && key < len) out[key] = v;
        }
    }
}

// lse of the window's queries from the (max, sum) of their key tiles: 64 rows
// (query heads and window queries of a sequence) per workgroup, the key tiles
// over its wavefronts.
__global__ __launch_bounds__(1024) void window_lse(WeightArgs a, float *lse)
{
    __shared__ float sm_m[16][64], sm_l[16][64];
    const int seq = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int len = length_of(a, seq);
    const int lo = (int64_t)len > a.window ? len - (int)a.window : 0;
    const int64_t rows = (int64_t)a.Hq * a.window, row = (int64_t)blockIdx.x * 64 + lane;
    const int i = row < rows ? (int)(row % a.window) : 0, query = lo + i;
    float M = NEG_INF, L = 0.0f;
    if (row < rows && query < len) {
        // tiles with a key at or before the query; the workgroup of a tile wrote every query from its first key on
        for (int t = wave; t <= query / KW; t += 16) {
            const f32x2 ml = a.ml[((int64_t)seq * a.tiles64 + t) * rows + row];
            const float m = fmaxf(M, ml[0]), use = m == NEG_INF ? 0.0f : m;
            L = L * __builtin_amdgcn_exp2f(M - use) + ml[1] * __builtin_amdgcn_exp2f(ml[0] - use);
            M = m;
        }
    }
    sm_m[wave][lane] = M;
    sm_l[wave][lane] = L;
    __syncthreads();
    if (wave || row >= rows || query >= len) return;
    float m = NEG_INF, l = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) m = fmaxf(m, sm_m[w][lane]);
    const float use = m == NEG_INF ? 0.0f : m;
#pragma unroll
    for (int w = 0; w < 16; ++w) l = fmaf(__builtin_amdgcn_exp2f(sm_m[w][lane] - use), sm_l[w][lane], l);
    lse[(int64_t)seq * rows + row] = (use + __builtin_amdgcn_logf(l)) * LN2;
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
};

// Queries of a workgroup: 4096, or fewer while that leaves the 512 that run at
// once without a second one (a multiple of the key tile, so that a range either
// sees a whole key tile or ends before it).
int64_t chunk_of(int64_t Hq, int64_t n_seq, int64_t max_seqlen)
{
    int64_t chunk = 4096;
    const int64_t tiles = (max_seqlen + KG - 1) / KG;
    while (chunk > 512 && tiles * Hq * n_seq * ((max_seqlen + chunk - 1) / chunk) < 1024) chunk /= 2;
    return chunk;
}

Scratch scratch_of(int64_t Hq, int64_t n_seq, int64_t max_seqlen, int64_t tokens, int64_t window, bool lse)
{
    Scratch s{0, 0, 0};
    if (window > 0 && !lse) {
        s.lse = n_seq * Hq * window;
        s.ml = 2 * n_seq * ((max_seqlen + KW - 1) / KW) * Hq * window;
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
    IQ_CHECK_ARG(q_st >= 0 && q_st < (1LL << 25), "iq_prefill_weights: token stride too large");
    IQ_CHECK_ARG(scale > 0.0f, "iq_prefill_weights: the scale must be positive");
    IQ_CHECK_ARG(window >= 0 && window <= 65536 && (window > 0 || lse), "iq_prefill_weights: no window and no lse");
    const Scratch s = scratch_of(Hq, n_seq, max_seqlen, tokens, window, lse != nullptr);
    IQ_CHECK_ARG(s.lse + s.ml + s.part == 0 || (workspace && workspace_floats >= s.lse + s.ml + s.part),
                 "iq_prefill_weights: workspace too small");
    const int64_t tiles = (max_seqlen + KG - 1) / KG, G = Hq / H;
    const int64_t chunk = window ? 1 << 30 : chunk_of(Hq, n_seq, max_seqlen), chunks = (max_seqlen + chunk - 1) / chunk;
    WeightArgs a{(const uint16_t *)q, (const uint16_t *)k, q_st, q_sh, k_st, k_sh, cu_seqlens, (int)n_seq, (int)max_seqlen, (int)H,
                 (int)Hq, (int)G, (int)(window ? G : 1), window ? window : max_seqlen, (int)chunk, (int)chunks, (int)tiles, scale * LOG2E, lse, lse_sh, 0,
                 (f32x2 *)workspace, (int)((max_seqlen + KW - 1) / KW), out, out_sh};
    const hipStream_t st = (hipStream_t)stream;
    const bool f16 = dtype == IQ_F16;
    const int64_t items = chunks * tiles * (Hq / a.heads) * n_seq;
    IQ_CHECK_ARG(items <= 0xffffff, "iq_prefill_weights: too many key tiles");
    const dim3 grid((unsigned)items), block(NT);
    if (window > 0 && !lse) {
        float *own = workspace + s.ml;
        hipLaunchKernelGGL((f16 ? prefill_weights<true, true> : prefill_weights<false, true>), grid, block, 0, st, a);
        hipLaunchKernelGGL(window_lse, dim3((unsigned)((Hq * window + 63) / 64), (unsigned)n_seq), dim3(1024), 0, st, a,
                           own);
        a.lse = own;
        a.windowed = 1;
    }
    if (window == 0) {
        a.out = workspace;
        a.out_sh = tokens;
    }
    hipLaunchKernelGGL((f16 ? prefill_weights<true, false> : prefill_weights<false, false>), grid, block, 0, st, a);
    if (window == 0 && tokens > 0)
        hipLaunchKernelGGL(add_heads, dim3((unsigned)((max_seqlen + 255) / 256), (unsigned)H, (unsigned)n_seq),
                           dim3(256), 0, st, a, workspace, tokens, out, out_sh);
    IQ_CHECK_LAUNCH("prefill_weights");
    return IQ_OK;
}
