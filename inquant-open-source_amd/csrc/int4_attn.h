// What the attention kernels over 4-bit pages share: arguments, the queries as
// matrix operands, and the join of partitions.
#pragma once

#include "int4_common.h"

namespace {

constexpr int D = 128;
constexpr float I4_LOG2E = 1.44269504088896341f;
// Softmax weights are at most 1; as f16 operands (and in the sums they are
// divided by) they are 2^14 times that, so that a weight keeps its eleven bits
// down to 2^-28 of the largest instead of 2^-14.
constexpr float I4_BIAS = 14.0f;

struct Int4Args {
    Int4Pool pool;
    const uint16_t *q;
    int64_t q_st, q_sh;                      // element strides (token, head)
    const int32_t *cu, *lengths;             // cu null: token i is the one of sequence i
    int32_t tokens, max_seqlen, max_tokens, span, parts, G, Hq;
    float c_log2;
    Partials part;                           // [tokens * Hq, parts] rows
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

// Query tokens of a sequence that a call answers.
__device__ __forceinline__ int32_t int4_asked(const Int4Args &a, const Int4Seq &s)
{
    int32_t m = s.m < a.max_seqlen ? s.m : a.max_seqlen;
    if (s.t0 < 0) return 0;
    const int32_t rest = a.tokens - s.t0;    // no token behind the last of the tensor
    return m < rest ? m : rest > 0 ? rest : 0;
}

// Eight channels of a query in f32, times f, as an f16 operand in the order of
// i4_pair's pairs: channels 0, 4, 1, 5, 2, 6, 3, 7.
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
// exponent: below 2^-38 of that value it rounds, of bf16's range nothing is lost.
__device__ __forceinline__ int query_shift(float largest)
{
    const int e = 14 + 127 - (int)(__float_as_uint(largest) >> 23);
    return e < 100 ? e : 100;
}

// Joins the partitions of a token and query head.  TEAM: one workgroup a row,
// whose eight teams of 32 lanes split the partitions; else a team a row.
template <bool TEAM>
__global__ __launch_bounds__(256) void int4_join(Int4Args a)
{
    __shared__ float so[TEAM ? 8 : 1][TEAM ? 128 : 1], sm[8], sl[8];
    const int tid = threadIdx.x, team = tid >> 5, c = 4 * (tid & 31), seq = blockIdx.y;
    const Int4Seq s = int4_seq(a, seq);
    const uint32_t item = TEAM ? blockIdx.x : blockIdx.x * 8 + team;
    const int t = (int)(item / (uint32_t)a.Hq), hq = (int)(item - (uint32_t)t * (uint32_t)a.Hq);
    if (t >= int4_asked(a, s)) return;       // with TEAM the whole workgroup's
    const int last = s.sees(t), live = last < 0 ? 0 : last / a.span + 1;
    const int64_t base = ((int64_t)(s.t0 + t) * a.Hq + hq) * a.parts;
    float M = NEG_INF, L = 0.0f;
    f32x4 o = {0, 0, 0, 0};
#pragma unroll 2
    for (int p = TEAM ? team : 0; p < live; p += TEAM ? 8 : 1) {
        const f32x2 ml = a.part.ml[base + p];
        const f32x4 x = *(const f32x4 *)(a.part.o + (base + p) * 128 + c);
        const float m = fmaxf(M, ml[0]), use = m == NEG_INF ? 0.0f : m;
        const float f0 = __builtin_amdgcn_exp2f(M - use), f1 = __builtin_amdgcn_exp2f(ml[0] - use);
        L = L * f0 + ml[1] * f1;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = o[e] * f0 + x[e] * f1;
        M = m;
    }
    if constexpr (TEAM) {
        *(f32x4 *)&so[team][c] = o;
        if (c == 0) {
            sm[team] = M;
            sl[team] = L;
        }
        __syncthreads();
        if (team) return;
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

}  // namespace
