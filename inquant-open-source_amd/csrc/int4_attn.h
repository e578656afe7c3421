// What the attention kernels over 4-bit pages share: arguments, the queries as
// matrix operands, and the join of partitions.
#pragma once

#include "int4_common.h"

namespace {

constexpr int D = 128;
constexpr float I4_LOG2E = 1.44269504088896341f;
// Softmax weights are at most 1; as f16 operands (and in the sums they are
// divided by) they are 2^14 times that, so that a weight keeps its eleven bits down
// to 2^-28 of the largest instead of 2^-14.
constexpr float I4_BIAS = 14.0f;

struct Int4Args {
    Int4Pool pool;
    const uint16_t *q;
    int64_t q_st, q_sh;                      // element strides (token, head)
    const int32_t *cu, *lengths;             // cu null: token i is the one of sequence i
    int32_t tokens, max_seqlen, max_tokens, G, Hq;
    int32_t span, parts;                     // many columns: rows per partition, partitions
    int32_t n_seq, groups, workers, width;   // few: see Share
    int32_t few;                             // sequences of at most so many columns are its, the others the kernel's for many
    float c_log2;
    Partials part;                           // many: [places * Hq, parts] rows (int4_place); few: [planes, workers + n_seq, width]
    void *out;
    int64_t o_st, o_sh;
    int odt;
};

// A sequence: its rows, its query tokens and the first of them.
struct Int4Seq {
    int32_t len, m, t0;
    __device__ __forceinline__ int32_t sees(int t) const { return len - m + t; }   // the last cache row of token t
};

__device__ __forceinline__ Int4Seq int4_seq(const Int4Args &a, int seq)
{
    Int4Seq s;
    const int32_t have = a.lengths[seq];
    s.len = have < 0 ? 0 : have < a.max_tokens ? have : a.max_tokens;
    s.t0 = a.cu ? a.cu[seq] : seq;
    const int32_t m = a.cu ? a.cu[seq + 1] - s.t0 : 1;
    s.m = m > 0 ? m : 0;
    return s;
}

// Query tokens of a sequence that a call answers; 0 where the other kernel does.
template <bool FEW>
__device__ __forceinline__ int32_t int4_asked(const Int4Args &a, const Int4Seq &s)
{
    int32_t m = s.m < a.max_seqlen ? s.m : a.max_seqlen;
    if (s.t0 < 0) return 0;
    const int32_t rest = a.tokens - s.t0;    // no token behind the last of the tensor
    m = m < rest ? m : rest > 0 ? rest : 0;
    return (m * a.G <= a.few) == FEW ? m : 0;
}

// Where partials of token t of a sequence stand: by the tensor's tokens, or by the
// sequences' where those cannot be as many (a tensor may hold rows of no sequence).
__device__ __forceinline__ int64_t int4_place(const Int4Args &a, int seq, const Int4Seq &s, int t)
{
    const int64_t most = (int64_t)a.n_seq * a.max_seqlen;
    return most < a.tokens ? (int64_t)seq * a.max_seqlen + t : (int64_t)(s.t0 + t);
}

// Eight channels of a query in f32.
template <bool F16>
__device__ __forceinline__ void query8(u32x4 raw, float (&x)[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = to_f32<F16>(raw[i] & 0xffffu);
        x[2 * i + 1] = to_f32<F16>(raw[i] >> 16);
    }
}

// The power of two that brings a query's largest value to 2^14 .. 2^15, as an
// exponent: below 2^-38 of that value it rounds, of bf16's range nothing is lost
// (the largest power of f32 brings its least value, 2^-133, to 2^-6).
__device__ __forceinline__ int query_shift(float largest)
{
    const int e = 14 + 127 - (int)(__float_as_uint(largest) >> 23);
    return e < 127 ? e : 127;
}

// Few columns: the rows of a launch's sequences (at most 64), in steps of 256,
// one after the other, are shared out evenly over `workers` workgroups for each
// plane (a KV head and `width` of its columns): every one has the same number of
// steps, whatever the sequences' lengths (16 sequences of 2K-32K tokens, split
// alike instead: 46 us in the best of five splits, 57 in the worst).  Lane i holds
// sequence i.  A workgroup w leaves its part of sequence i at slot w + i of the
// plane, which no other part has.
constexpr int STEP = 256;

struct Share {
    Int4Seq own;                             // this lane's sequence
    int32_t steps, upto;                     // its steps; with those before it
    int32_t each, total;                     // of a workgroup; of all (uniform)
    __device__ __forceinline__ Int4Seq of(int seq) const
    {
        return {__builtin_amdgcn_readlane(own.len, seq), __builtin_amdgcn_readlane(own.m, seq),
                __builtin_amdgcn_readlane(own.t0, seq)};
    }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ int32_t dpp_i(int32_t v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }

// Of group `group`: sequences that ask for fewer columns have no steps there.
__device__ __forceinline__ Share int4_share(const Int4Args &a, int group)
{
    const int lane = threadIdx.x & 63;
    Share r;
    r.own = int4_seq(a, lane < a.n_seq ? lane : a.n_seq - 1);
    r.steps = lane < a.n_seq && int4_asked<true>(a, r.own) * a.G > group * a.width ? (r.own.len + STEP - 1) / STEP : 0;
    int32_t v = r.steps;
    v += dpp_i<0x111, 0xf>(v);               // row_shr:1
    v += dpp_i<0x112, 0xf>(v);
    v += dpp_i<0x114, 0xf>(v);
    v += dpp_i<0x118, 0xf>(v);
    v += dpp_i<0x142, 0xa>(v);               // row_bcast:15 into rows 1 and 3
    v += dpp_i<0x143, 0xc>(v);               // row_bcast:31 into rows 2 and 3
    r.upto = v;
    r.total = __builtin_amdgcn_readlane(v, 63);
    r.each = (r.total + a.workers - 1) / a.workers;
    return r;
}

// Joins the partitions of a token and query head.  FEW: those of the workgroups
// that shared its sequence, by one workgroup whose eight teams of 32 lanes split
// them, and which takes every gridDim.x / Hq th token; else those of `span` rows, by
// one team.
template <bool FEW>
__global__ __launch_bounds__(256) void int4_join(Int4Args a)
{
    __shared__ float so[FEW ? 8 : 1][FEW ? 128 : 1], sm[8], sl[8];
    const int tid = threadIdx.x, team = tid >> 5, c = 4 * (tid & 31), seq = blockIdx.y;
    const Int4Seq s = int4_seq(a, seq);
    const uint32_t item = FEW ? blockIdx.x : blockIdx.x * 8 + team;
    const int t0 = (int)(item / (uint32_t)a.Hq), hq = (int)(item - (uint32_t)t0 * (uint32_t)a.Hq);
    const int asked = int4_asked<FEW>(a, s);
    for (int t = t0; t < asked; t += FEW ? (int)(gridDim.x / (uint32_t)a.Hq) : asked) {  // with FEW the whole workgroup's
        const int last = s.sees(t);
        int first = 0, live;                 // partitions first .. live - 1
        int64_t base, next;                  // rows of the first of them, from one to the next
        if constexpr (FEW) {
            const int h = hq / a.G, col = t * a.G + hq - h * a.G, group = col / a.width;
            const Share r = int4_share(a, group);
            const int steps = __builtin_amdgcn_readlane(r.steps, seq), from = __builtin_amdgcn_readlane(r.upto, seq) - steps;
            if (steps == 0 || last < 0) live = 0;
            else {
                first = from / r.each;
                live = (from + last / STEP) / r.each + 1;
                if (first == (from + steps - 1) / r.each) continue;      // one workgroup had them all
            }
            next = a.width;
            base = ((int64_t)(h + a.pool.H * group) * (a.workers + a.n_seq) + first + seq) * next + col - group * a.width;
        } else {
            live = last < 0 ? 0 : last / a.span + 1;
            base = (int4_place(a, seq, s, t) * a.Hq + hq) * a.parts;
            next = 1;
        }
        live -= first;
        float M = NEG_INF, L = 0.0f;
        f32x4 o = {0, 0, 0, 0};
#pragma unroll 2
        for (int p = FEW ? team : 0; p < live; p += FEW ? 8 : 1) {
            const f32x2 ml = a.part.ml[base + p * next];
            const f32x4 x = *(const f32x4 *)(a.part.o + (base + p * next) * 128 + c);
            const float m = fmaxf(M, ml[0]), use = m == NEG_INF ? 0.0f : m;
            const float f0 = __builtin_amdgcn_exp2f(M - use), f1 = __builtin_amdgcn_exp2f(ml[0] - use);
            L = L * f0 + ml[1] * f1;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = o[e] * f0 + x[e] * f1;
            M = m;
        }
        if constexpr (FEW) {
            __syncthreads();                 // what was there before has been read
            *(f32x4 *)&so[team][c] = o;
            if (c == 0) {
                sm[team] = M;
                sl[team] = L;
            }
            __syncthreads();
            if (team) continue;
            M = NEG_INF;
#pragma unroll
            for (int i = 0; i < 8; ++i) M = fmaxf(M, sm[i]);
            const float use = M == NEG_INF ? 0.0f : M;
            L = 0.0f;
            o = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = __builtin_amdgcn_exp2f(sm[i] - use);
                L = fmaf(f, sl[i], L);
                const f32x4 x = *(const f32x4 *)&so[i][c];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(f, x[e], o[e]);
            }
        }
        const int64_t at = (int64_t)(s.t0 + t) * a.o_st + hq * a.o_sh + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) iq_store_as(a.out, at + e, L == 0.0f ? 0.0f : o[e] / L, a.odt);
    }
}

}  // namespace
