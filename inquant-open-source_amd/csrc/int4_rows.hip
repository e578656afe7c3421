// New rows into pages with the position rotation on the way, and rows of pages
// read back (gfx950).
//
// For a token at position p, pairs (a, b) of a query's or key's channels turn
// by the table's angles of that position,
//   a' = a cos - b sin,  b' = b cos + a sin,
// the two products and their sum rounded to f32 each; a per-channel factor then
// multiplies queries and divides keys.  Keys and values go to exact pages,
// rounded once, or to 4-bit pages: per group of 32 channels, with lo and hi the
// least and largest of them and 0,
//   s = (hi - lo) / 15 within 2^-14 .. 2048, rounded up to six bits,
//   z = rint(-lo / s),  n = rint(x / s) + z, both within 0 .. 15,
// decided as in exact arithmetic: rows of 16 bits often lie on the border
// between two codes, or span exactly 15 steps.  A group with an infinity or a
// NaN is stored as NaN.
#include <type_traits>

#include "dense_common.h"
#include "int4_common.h"

namespace {

constexpr int NT = 256, TEAMS = NT / 16;     // sixteen lanes a row, eight channels each
constexpr float S_LEAST = 0x1p-14f, S_MOST = 2048.0f;
constexpr uint32_t NAN_WORD = 0x7e00u;

struct AppendArgs {
    const uint16_t *q, *k, *v;               // q may be null
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh;   // element strides (token, head)
    uint16_t *out;                           // the rotated queries
    const int32_t *cu, *start, *positions;   // start and positions may be null
    const float *rotation;                   // [angles, rotary] cos | sin
    int64_t angles;
    const float *factors;                    // [H, 128] or null
    int32_t rotary, interleaved, Hq, H, G;
    uint32_t max_len;
    int32_t tokens;                          // of the tensors
    DensePool dense;                         // one of the two, by the kernel
    Int4Pool int4;
};

// The first token of a sequence and how many of it a call takes: none in front of
// the tensors or behind them, whatever the offsets say.
struct RowSpan {
    int64_t t0;
    uint32_t len;
};

__device__ __forceinline__ RowSpan row_span(const int32_t *cu, int seq, uint32_t max_len, int32_t tokens)
{
    const int32_t t0 = cu[seq], behind = cu[seq + 1], end = behind < tokens ? behind : tokens;
    const uint32_t n = t0 >= 0 && end > t0 ? end - t0 : 0;
    return {t0, n < max_len ? n : max_len};
}

template <bool F16>
__device__ __forceinline__ void unpack8(u32x4 raw, float (&x)[8])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = to_f32<F16>(raw[i] & 0xffffu);
        x[2 * i + 1] = to_f32<F16>(raw[i] >> 16);
    }
}

template <bool F16>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8])
{
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<F16>(x[2 * i], x[2 * i + 1]);
    return r;
}

// Rotates channels 8 c .. 8 c + 7 of a row (x, unpacked from raw); the pairs' other
// halves come from their lane (loaded again, past what the first cache holds:
// 274 us for 60K tokens into 4-bit pages).  A position that the table does not hold
// gives NaN.
template <bool F16>
__device__ __forceinline__ void rotate8(const AppendArgs &a, u32x4 raw, int64_t pos, int c, float (&x)[8])
{
    const int per = a.rotary >> 4;           // 16-byte chunks of a half
    if (c >= 2 * per) return;
    const bool known = pos >= 0 && pos < a.angles;
    const float *table = a.rotation + (known ? pos : 0) * a.rotary;
    if (a.interleaved) {
        const f32x4 cos = *(const f32x4 *)(table + 4 * c), sin = *(const f32x4 *)(table + 8 * per + 4 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float u = x[2 * i], w = x[2 * i + 1];
            x[2 * i] = u * cos[i] - w * sin[i];
            x[2 * i + 1] = w * cos[i] + u * sin[i];
        }
    } else {
        const bool first = c < per;
        const int j = first ? c : c - per;
        const int other = (int)(threadIdx.x & 48) + (first ? c + per : j);
        u32x4 there;
#pragma unroll
        for (int i = 0; i < 4; ++i) there[i] = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * other, (int)raw[i]);
        float y[8];
        unpack8<F16>(there, y);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x4 cos = *(const f32x4 *)(table + 8 * j + 4 * h);
            const f32x4 sin = *(const f32x4 *)(table + 8 * per + 8 * j + 4 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = x[4 * h + i] * cos[i], w = y[4 * h + i] * sin[i];
                x[4 * h + i] = first ? u - w : u + w;
            }
        }
    }
    if (!known)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
}

// Over the four lanes that hold a group of 32 channels.
__device__ __forceinline__ float quad_max(float v)
{
    v = fmaxf(v, dpp_f<0xb1>(v));
    return fmaxf(v, dpp_f<0x4e>(v));
}

// rint(x / s) as in exact arithmetic, ties to even, for a quotient within
// +-16 (beyond, something past that): the product with the reciprocal is at most one
// off, and what is left of x decides (exact: n s has at most eleven bits).
__device__ __forceinline__ float rint_steps(float x, float s, float per)
{
    float n = rintf(fminf(fmaxf(x * per, -20.0f), 20.0f));
    const float left = fmaf(-n, s, x), most = 0.5f * s, far = fabsf(left);
    if (far > most || (far == most && ((int)n & 1))) n += left < 0.0f ? -1.0f : 1.0f;
    return n;
}

// The codes of this lane's eight channels and the word of their group.
__device__ __forceinline__ uint32_t code8(const float (&x)[8], uint32_t &word)
{
    float hi = 0.0f, lo = 0.0f, size = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi = fmaxf(hi, x[i]);
        lo = fmaxf(lo, -x[i]);               // of the negated values
        size = size + (x[i] - x[i]);         // 0, or NaN once a value is infinite or NaN
    }
    hi = quad_max(hi);
    lo = quad_max(lo);
    size += dpp_f<0xb1>(size);
    size += dpp_f<0x4e>(size);
    const double range = (double)hi + (double)lo;
    const float wide = fminf(fmaxf((hi + lo) * (1.0f / 15.0f), S_LEAST), S_MOST);
    uint32_t bits = (__float_as_uint(wide) + 0x3ffffu) & ~0x3ffffu;
    // one step of the six bits up or down, should the product have crossed one
    const float below = __uint_as_float(bits - 0x40000u);
    if (below >= S_LEAST && (double)(15.0f * below) >= range) bits -= 0x40000u;
    else if (__uint_as_float(bits) < S_MOST && (double)(15.0f * __uint_as_float(bits)) < range) bits += 0x40000u;
    const float s = __uint_as_float(bits), per = 1.0f / s;
    const float z = fminf(rint_steps(lo, s, per), 15.0f);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        codes |= (uint32_t)fminf(fmaxf(rint_steps(x[i], s, per) + z, 0.0f), 15.0f) << (4 * i);
    const bool fine = size == 0.0f;
    word = fine ? (uint32_t)iq_f32_to_f16(s) | (uint32_t)z : NAN_WORD;
    return fine ? codes : 0;
}

// Bound by memory: seven prompts into exact pages 268-270 us (5.7 TB/s read and
// written), 60K tokens into 4-bit pages 232-255 us (a kernel trace's).  Sixteen lanes take a row, heads innermost, so that a
// workgroup reads one range of a token-major batch and its rows share the
// table's line.
// Rows of queries and keys (and values of exact pages) go first; the values
// of 4-bit pages follow, four cache rows of a head at a time, since their codes
// interleave in sixteen bytes.
// A team takes R rows, sixteen apart, and asks for all of them first: with one row
// each a workgroup of a long call is over before its latencies are paid for.
template <bool F16, bool INT4, int R>
__global__ __launch_bounds__(NT) void append_kernel(AppendArgs a)
{
    const int seq = blockIdx.y, c = threadIdx.x & 15;
    const auto [t0, len] = row_span(a.cu, seq, a.max_len, a.tokens);
    const int64_t start = a.start ? a.start[seq] : 0;
    const int64_t pos0 = a.positions ? (int64_t)a.positions[seq] : start;
    const uint32_t H = (uint32_t)a.H, per_token = (uint32_t)a.Hq + (INT4 ? H : 2 * H);
    const uint64_t rows = (uint64_t)len * per_token, first = (uint64_t)blockIdx.x * (TEAMS * R);
    if (first < rows) {                      // uniform
        u32x4 raw[R];
        uint32_t ts[R], hss[R];
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const uint64_t item = first + j * TEAMS + (threadIdx.x >> 4);
            const uint32_t i = (uint32_t)(item < rows ? item : rows - 1);
            const uint32_t t = ts[j] = i / per_token, hs = hss[j] = i - t * per_token;
            const bool query = hs < (uint32_t)a.Hq, value = !INT4 && hs >= (uint32_t)a.Hq + H;
            const uint16_t *row = query ? a.q + (t0 + t) * a.q_st + hs * a.q_sh
                                  : value ? a.v + (t0 + t) * a.v_st + (hs - a.Hq - H) * a.v_sh
                                          : a.k + (t0 + t) * a.k_st + (hs - a.Hq) * a.k_sh;
            raw[j] = ld16(row + 8 * c);
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            if (first + j * TEAMS + (threadIdx.x >> 4) >= rows) break;
            const uint32_t t = ts[j], hs = hss[j];
            const int64_t token = t0 + t;
            const bool query = hs < (uint32_t)a.Hq, value = !INT4 && hs >= (uint32_t)a.Hq + H;
            const uint32_t h = query ? hs / (uint32_t)a.G : value ? hs - a.Hq - H : hs - a.Hq;
            float x[8];
            if (!value) {
                unpack8<F16>(raw[j], x);
                if (a.rotary) rotate8<F16>(a, raw[j], pos0 + t, c, x);
                if (a.factors) {
                    const float *f = a.factors + h * 128 + 8 * c;
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = query ? x[i] * f[i] : x[i] / f[i];
                }
                if (!INT4 || query) raw[j] = pack8<F16>(x);
            }
            if (query) {
                u32x4 *to = (u32x4 *)(a.out + token * a.o_st + hs * a.o_sh + 8 * c);
                if constexpr (R > 1) __builtin_nontemporal_store(raw[j], to);
                else *to = raw[j];
                continue;
            }
            const int64_t at = start + t;
            if constexpr (INT4) {
                uint32_t word;
                const uint32_t codes = code8(x, word);
                const Int4Pool &p = a.int4;
                const int64_t page = i4_page(p, seq, at);
                if (page < 0) continue;
                uint8_t *head = p.base + page * p.s_page + h * p.s_head;
                const uint32_t r = (uint32_t)at & (p.B - 1);
                *(uint32_t *)(head + 64 * r + 4 * c) = codes;
                if ((c & 3) == 0) *(uint16_t *)(head + i4_key_words(p.B) + 8 * r + 2 * (c >> 2)) = (uint16_t)word;
            } else {
                const DensePool &p = a.dense;
                const int64_t page = dense_page(p, seq, at), r = at & (p.B - 1);
                if (page < 0) continue;
                uint16_t *to = value ? p.value + page * p.v_sp + h * p.v_sh + r * p.v_st
                                     : p.key + page * p.k_sp + h * p.k_sh + r * p.k_st;
                __builtin_nontemporal_store(raw[j], (u32x4 *)(to + 8 * c));
                if (!value && c == 0 && p.weights) {
                    const int64_t o = (page * p.H + h) * p.B + r;
                    p.weights[o] = 0.0f;
                    p.positions[o] = (int32_t)(pos0 + t);
                }
            }
        }
        return;
    }
    if constexpr (INT4) {
        // whole workgroups of either kind
        if (len == 0) return;
        const int64_t quad = start >> 2, quads = ((start + len + 3) >> 2) - quad;
        const uint64_t i = (blockIdx.x - (rows + TEAMS * R - 1) / (TEAMS * R)) * TEAMS + (threadIdx.x >> 4);
        if (i >= (uint64_t)quads * H) return;
        const uint32_t j = (uint32_t)(i / H), h = (uint32_t)(i - (uint64_t)j * H);
        const int64_t first = (quad + j) * 4;            // a cache row
        const Int4Pool &p = a.int4;
        const int64_t page = i4_page(p, seq, first);
        if (page < 0) return;
        uint32_t codes[4], words[4], live = 0;
        u32x4 raw[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t t = first + r - start;
            raw[r] = u32x4{0, 0, 0, 0};
            if (t >= 0 && t < (int64_t)len) {
                raw[r] = ld16(a.v + (t0 + t) * a.v_st + h * a.v_sh + 8 * c);
                live |= 1u << r;
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            codes[r] = words[r] = 0;
            if (live >> r & 1) {
                float x[8];
                unpack8<F16>(raw[r], x);
                codes[r] = code8(x, words[r]);
            }
        }
        uint8_t *head = p.base + page * p.s_page + h * p.s_head;
        const uint32_t r4 = ((uint32_t)first & (p.B - 1)) >> 2;
        uint8_t *to = head + i4_value_codes(p.B) + 256 * r4 + 16 * c;
        uint8_t *wto = head + i4_value_words(p.B) + 32 * r4 + 8 * (c >> 2);
        if (live == 15) {
            u32x4 all;
#pragma unroll
            for (int d = 0; d < 2; ++d) {                // rows 2 d and 2 d + 1, lower and upper four channels
                all[2 * d] = (codes[2 * d] & 0xffffu) | codes[2 * d + 1] << 16;
                all[2 * d + 1] = codes[2 * d] >> 16 | (codes[2 * d + 1] & 0xffff0000u);
            }
            *(u32x4 *)to = all;
            if ((c & 3) == 0) *(u32x2 *)wto = u32x2{words[0] | words[1] << 16, words[2] | words[3] << 16};
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (live >> r & 1) {
                    *(uint16_t *)(to + 8 * (r >> 1) + 2 * (r & 1)) = (uint16_t)codes[r];
                    *(uint16_t *)(to + 8 * (r >> 1) + 4 + 2 * (r & 1)) = (uint16_t)(codes[r] >> 16);
                    if ((c & 3) == 0) *(uint16_t *)(wto + 2 * r) = (uint16_t)words[r];
                }
        }
    }
}

struct ReadArgs {
    void *k, *v;
    int64_t k_st, k_sh, v_st, v_sh;          // element strides (token, head)
    const int32_t *cu, *start;               // start may be null
    int32_t H;
    uint32_t max_len;
    int32_t tokens;                          // of the tensors
    DensePool dense;
    Int4Pool int4;
};

// Eight values of f16 as rows of the output type.
template <int ODT>
__device__ __forceinline__ void store8(void *base, int64_t at, u32x4 v)
{
    if constexpr (ODT == IQ_F16) {
        __builtin_nontemporal_store(v, (u32x4 *)((uint16_t *)base + at));
    } else {
        float x[8];
        unpack8<true>(v, x);
        if constexpr (ODT == IQ_BF16) {
            __builtin_nontemporal_store(pack8<false>(x), (u32x4 *)((uint16_t *)base + at));
        } else {
            __builtin_nontemporal_store(f32x4{x[0], x[1], x[2], x[3]}, (f32x4 *)((float *)base + at));
            __builtin_nontemporal_store(f32x4{x[4], x[5], x[6], x[7]}, (f32x4 *)((float *)base + at + 4));
        }
    }
}

// Four cache rows of a head by sixteen lanes, eight channels each; a row of a
// page outside the pool or the table is not written.  Bound by memory: 124 us for
// 662 MB (5.4 TB/s), most of them written.
template <int ODT>
__global__ __launch_bounds__(NT) void read_int4_kernel(ReadArgs a)
{
    const int seq = blockIdx.y, c = threadIdx.x & 15;
    const auto [t0, len] = row_span(a.cu, seq, a.max_len, a.tokens);
    if (len == 0) return;
    const int64_t start = a.start ? a.start[seq] : 0;
    const uint32_t H = (uint32_t)a.H;
    const int64_t quad = start >> 2, quads = ((start + len + 3) >> 2) - quad;
    const uint64_t item = (uint64_t)blockIdx.x * TEAMS + (threadIdx.x >> 4);
    if (item >= (uint64_t)quads * H) return;
    // quads innermost: a workgroup reads one range of a head's pages
    const uint32_t h = (uint32_t)(item / (uint64_t)quads);
    const int64_t first = (quad + (int64_t)(item - (uint64_t)h * quads)) * 4;
    const Int4Pool &p = a.int4;
    const int64_t page = i4_page(p, seq, first);
    if (page < 0) return;
    const I4Masks masks;
    const uint8_t *head = p.base + page * p.s_page + h * p.s_head;
    const uint32_t r0 = (uint32_t)first & (p.B - 1);
    uint32_t kc[4];
    uint16_t kw[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        kc[r] = ldg<uint32_t>(head + 64 * (r0 + r) + 4 * c);
        kw[r] = ldg<uint16_t>(head + i4_key_words(p.B) + 8 * (r0 + r) + 2 * (c >> 2));
    }
    const u32x4 vc = ld16(head + i4_value_codes(p.B) + 64 * r0 + 16 * c);
    const u32x2 vw = ldg<u32x2>(head + i4_value_words(p.B) + 8 * r0 + 8 * (c >> 2));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t t = first + r - start;
        if (t < 0 || t >= (int64_t)len) continue;
        const I4Scale sk = i4_scale(kw[r]);
        uint32_t pair[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pair[i] = i4_value(masks.pair(kc[r], i), lower(sk.s), lower(sk.c));
        u32x4 out;                           // pair i holds channels i and i + 4
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            out[i] = (pair[2 * i] & 0xffffu) | pair[2 * i + 1] << 16;
            out[2 + i] = pair[2 * i] >> 16 | (pair[2 * i + 1] & 0xffff0000u);
        }
        store8<ODT>(a.k, (t0 + t) * a.k_st + h * a.k_sh + 8 * c, out);
    }
#pragma unroll
    for (int d = 0; d < 2; ++d) {            // rows 2 d and 2 d + 1 in the halves
        const I4Scale sv = i4_scale(vw[d]);
        uint32_t pair[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pair[i] = i4_value(masks.pair(vc[2 * d + (i >> 2)], i & 3), sv.s, sv.c);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int64_t t = first + 2 * d + r - start;
            if (t < 0 || t >= (int64_t)len) continue;
            u32x4 out;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                out[i] = r == 0 ? (pair[2 * i] & 0xffffu) | pair[2 * i + 1] << 16
                                : pair[2 * i] >> 16 | (pair[2 * i + 1] & 0xffff0000u);
            store8<ODT>(a.v, (t0 + t) * a.v_st + h * a.v_sh + 8 * c, out);
        }
    }
}

// Rows of exact pages: sixteen lanes a row of keys and of values.  Bound by memory:
// eight prefixes, 156K rows of 8 heads, 218 us for 1281 MB (5.9 TB/s).
__global__ __launch_bounds__(NT) void read_dense_kernel(ReadArgs a)
{
    const int seq = blockIdx.y, c = threadIdx.x & 15;
    const auto [t0, len] = row_span(a.cu, seq, a.max_len, a.tokens);
    const int64_t start = a.start ? a.start[seq] : 0;
    const uint64_t item = (uint64_t)blockIdx.x * TEAMS + (threadIdx.x >> 4);
    if (item >= (uint64_t)len * (uint32_t)a.H) return;
    const uint32_t t = (uint32_t)(item / (uint32_t)a.H), h = (uint32_t)(item - (uint64_t)t * (uint32_t)a.H);
    const DensePool &p = a.dense;
    const int64_t page = dense_page(p, seq, start + t), r = (start + t) & (p.B - 1);
    if (page < 0) return;
    const u32x4 k = ld16(p.key + page * p.k_sp + h * p.k_sh + r * p.k_st + 8 * c);
    const u32x4 v = ld16(p.value + page * p.v_sp + h * p.v_sh + r * p.v_st + 8 * c);
    __builtin_nontemporal_store(k, (u32x4 *)((uint16_t *)a.k + (t0 + t) * a.k_st + h * a.k_sh + 8 * c));
    __builtin_nontemporal_store(v, (u32x4 *)((uint16_t *)a.v + (t0 + t) * a.v_st + h * a.v_sh + 8 * c));
}

// Rows of a call (of queries, keys and exact pages' values) past which a team takes
// four.  Exact pages: 18K rows 4.5 us by ones and 5.5 by fours, 74K rows 9.6 and 8.3, 1.2M
// rows 126 and 112.  4-bit pages, whose groups cost more: 32 rows 3.4 and 4.3, 2K rows 6.5
// either way, 16K rows 7.9 and 7.4, 65K rows 13.9 and 11.0.
constexpr int64_t ONES_DENSE = 32768, ONES_INT4 = 8192;
constexpr int64_t GRID_MOST = 0xffffffffLL / NT;         // workgroups of a launch's first dimension

constexpr int64_t ANY_TOKENS = 0x7fffffff;   // more than offsets can tell

bool aligned(const void *p, int64_t strides) { return (uintptr_t)p % 16 == 0 && strides % 8 == 0; }

int append_rows(const void *q, const void *k, const void *v, int dtype, int64_t q_st, int64_t q_sh, int64_t k_st,
                int64_t k_sh, int64_t v_st, int64_t v_sh, int64_t Hq, const int32_t *cu_seqlens, int64_t n_seq,
                int64_t max_seqlen, int64_t tokens, const int32_t *start, const int32_t *positions, const float *rotation,
                int64_t angles, int64_t rotary, int interleaved, const float *factors, const iq_dense_pages *dense,
                const iq_int4_pages *int4, const int32_t *tables, int64_t bt_stride, int64_t bt_cols, void *out,
                int64_t o_st, int64_t o_sh, void *stream)
{
    IQ_CHECK_ARG((dense != nullptr) != (int4 != nullptr), "iq_append_rows: one kind of pages");
    AppendArgs a{};
    if (dense) {
        if (const int e = dense_pool("iq_append_rows", dense, dtype, tables, bt_stride, bt_cols, n_seq, a.dense)) return e;
        a.H = a.dense.H;
    } else {
        if (const int e = int4_pool("iq_append_rows", int4, tables, bt_stride, bt_cols, n_seq, a.int4)) return e;
        a.H = a.int4.H;
    }
    IQ_CHECK_ARG(k && v && cu_seqlens, "iq_append_rows: null pointer");
    IQ_CHECK_ARG(dtype == IQ_BF16 || dtype == IQ_F16, "iq_append_rows: rows must be bf16 or f16");
    IQ_CHECK_ARG(!q || (out && Hq >= 1 && Hq <= 65535 && Hq % a.H == 0), "iq_append_rows: heads %lld / %d", (long long)Hq,
                 a.H);
    IQ_CHECK_ARG(aligned(q, q_st | q_sh) && aligned(k, k_st | k_sh) && aligned(v, v_st | v_sh) &&
                     aligned(out, o_st | o_sh), "iq_append_rows: rows must be 16-byte aligned");
    IQ_CHECK_ARG(rotation ? rotary >= 16 && rotary <= 128 && rotary % 16 == 0 && angles >= 0 && angles < (1LL << 40) &&
                                (uintptr_t)rotation % 16 == 0
                          : rotary == 0, "iq_append_rows: bad rotation");
    IQ_CHECK_ARG(!rotation || angles > 0, "iq_append_rows: an empty rotation");
    IQ_CHECK_ARG((uintptr_t)factors % 16 == 0, "iq_append_rows: factors must be 16-byte aligned");
    IQ_CHECK_ARG(max_seqlen >= 0 && max_seqlen <= 0x7fffffffLL && tokens >= 0, "iq_append_rows: bad length");
    if (max_seqlen > tokens) max_seqlen = tokens;
    if (n_seq == 0 || max_seqlen == 0) return IQ_OK;
    a.q = (const uint16_t *)q, a.k = (const uint16_t *)k, a.v = (const uint16_t *)v, a.out = (uint16_t *)out;
    a.q_st = q_st, a.q_sh = q_sh, a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh, a.o_st = o_st, a.o_sh = o_sh;
    a.cu = cu_seqlens, a.start = start, a.positions = positions, a.rotation = rotation, a.angles = angles;
    a.factors = factors, a.rotary = (int32_t)rotary, a.interleaved = interleaved;
    a.Hq = q ? (int32_t)Hq : 0, a.G = q ? (int32_t)(Hq / a.H) : 1, a.max_len = (uint32_t)max_seqlen;
    a.tokens = (int32_t)(tokens < ANY_TOKENS ? tokens : ANY_TOKENS);
    // four rows may lie in two quads
    const int64_t rows = max_seqlen * (a.Hq + (dense ? 2 : 1) * (int64_t)a.H);
    const int64_t quads = dense ? 0 : (max_seqlen + 6) / 4 * a.H;
    const bool four = rows > (dense ? ONES_DENSE : ONES_INT4) / n_seq;
    const int64_t each = TEAMS * (four ? 4 : 1), groups = (rows + each - 1) / each + (quads + TEAMS - 1) / TEAMS;
    IQ_CHECK_ARG(rows <= 0xffffffffLL && groups <= GRID_MOST, "iq_append_rows: too many rows");
    const dim3 grid((unsigned)groups, (unsigned)n_seq);
    const bool f16 = dtype == IQ_F16;
    const auto kernel = four ? dense ? f16 ? append_kernel<true, false, 4> : append_kernel<false, false, 4>
                                     : f16 ? append_kernel<true, true, 4> : append_kernel<false, true, 4>
                        : dense ? f16 ? append_kernel<true, false, 1> : append_kernel<false, false, 1>
                                : f16 ? append_kernel<true, true, 1> : append_kernel<false, true, 1>;
    hipLaunchKernelGGL(kernel, grid, dim3(NT), 0, (hipStream_t)stream, a);
    IQ_CHECK_LAUNCH("append_rows");
    return IQ_OK;
}

int read_rows(const iq_dense_pages *dense, const iq_int4_pages *int4, int dtype, const int32_t *tables, int64_t bt_stride,
              int64_t bt_cols, const int32_t *cu_seqlens, int64_t n_seq, int64_t max_seqlen, int64_t tokens,
              const int32_t *start, void *k, int64_t k_st, int64_t k_sh, void *v, int64_t v_st, int64_t v_sh, void *stream)
{
    IQ_CHECK_ARG((dense != nullptr) != (int4 != nullptr), "iq_read_rows: one kind of pages");
    ReadArgs a{};
    if (dense) {
        if (const int e = dense_pool("iq_read_rows", dense, dtype, tables, bt_stride, bt_cols, n_seq, a.dense)) return e;
        a.H = a.dense.H;
    } else {
        if (const int e = int4_pool("iq_read_rows", int4, tables, bt_stride, bt_cols, n_seq, a.int4)) return e;
        a.H = a.int4.H;
        IQ_CHECK_ARG(dtype >= IQ_F32 && dtype <= IQ_F16, "iq_read_rows: bad output dtype");
    }
    IQ_CHECK_ARG(k && v && cu_seqlens, "iq_read_rows: null pointer");
    IQ_CHECK_ARG(aligned(k, k_st | k_sh) && aligned(v, v_st | v_sh), "iq_read_rows: rows must be 16-byte aligned");
    IQ_CHECK_ARG(max_seqlen >= 0 && max_seqlen <= 0x7fffffffLL && tokens >= 0, "iq_read_rows: bad length");
    if (max_seqlen > tokens) max_seqlen = tokens;
    if (n_seq == 0 || max_seqlen == 0) return IQ_OK;
    a.k = k, a.v = v, a.k_st = k_st, a.k_sh = k_sh, a.v_st = v_st, a.v_sh = v_sh;
    a.cu = cu_seqlens, a.start = start, a.max_len = (uint32_t)max_seqlen;
    a.tokens = (int32_t)(tokens < ANY_TOKENS ? tokens : ANY_TOKENS);
    const int64_t items = (dense ? max_seqlen : (max_seqlen + 6) / 4) * (int64_t)a.H;
    IQ_CHECK_ARG((items + TEAMS - 1) / TEAMS <= GRID_MOST, "iq_read_rows: too many rows");
    const dim3 grid((unsigned)((items + TEAMS - 1) / TEAMS), (unsigned)n_seq);
    const auto kernel = dense ? read_dense_kernel : dtype == IQ_F16 ? read_int4_kernel<IQ_F16>
                                                  : dtype == IQ_BF16 ? read_int4_kernel<IQ_BF16> : read_int4_kernel<IQ_F32>;
    hipLaunchKernelGGL(kernel, grid, dim3(NT), 0, (hipStream_t)stream, a);
    IQ_CHECK_LAUNCH("read_rows");
    return IQ_OK;
}

}  // namespace

extern "C" int iq_append_rows(const void *q, const void *k, const void *v, int dtype, int64_t q_st, int64_t q_sh,
                              int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, int64_t Hq,
                              const int32_t *cu_seqlens, int64_t n_seq, int64_t max_seqlen, const int32_t *start,
                              const int32_t *positions, const float *rotation, int64_t angles, int64_t rotary,
                              int interleaved, const float *factors, const iq_dense_pages *dense,
                              const iq_int4_pages *int4, const int32_t *tables, int64_t bt_stride, int64_t bt_cols,
                              void *out, int64_t o_st, int64_t o_sh, void *stream)
{
    return append_rows(q, k, v, dtype, q_st, q_sh, k_st, k_sh, v_st, v_sh, Hq, cu_seqlens, n_seq, max_seqlen, ANY_TOKENS,
                       start, positions, rotation, angles, rotary, interleaved, factors, dense, int4, tables, bt_stride,
                       bt_cols, out, o_st, o_sh, stream);
}

extern "C" int iq_append_rows_from(const iq_append_rows_args *a)
{
    IQ_CHECK_ARG(a, "iq_append_rows: null arguments");
    return append_rows((const void *)a->q, (const void *)a->k, (const void *)a->v, (int)a->dtype, a->q_st, a->q_sh, a->k_st,
                       a->k_sh, a->v_st, a->v_sh, a->Hq, (const int32_t *)a->cu_seqlens, a->n_seq, a->max_seqlen, a->tokens,
                       (const int32_t *)a->start, (const int32_t *)a->positions, (const float *)a->rotation, a->angles,
                       a->rotary, (int)a->interleaved, (const float *)a->factors, (const iq_dense_pages *)a->dense,
                       (const iq_int4_pages *)a->int4, (const int32_t *)a->tables, a->bt_stride, a->bt_cols, (void *)a->out,
                       a->o_st, a->o_sh, (void *)a->stream);
}

extern "C" int iq_read_rows(const iq_dense_pages *dense, const iq_int4_pages *int4, int dtype, const int32_t *tables,
                            int64_t bt_stride, int64_t bt_cols, const int32_t *cu_seqlens, int64_t n_seq,
                            int64_t max_seqlen, const int32_t *start, void *k, int64_t k_st, int64_t k_sh, void *v,
                            int64_t v_st, int64_t v_sh, void *stream)
{
    return read_rows(dense, int4, dtype, tables, bt_stride, bt_cols, cu_seqlens, n_seq, max_seqlen, ANY_TOKENS, start, k, k_st,
                     k_sh, v, v_st, v_sh, stream);
}

extern "C" int iq_read_rows_from(const iq_read_rows_args *a)
{
    IQ_CHECK_ARG(a, "iq_read_rows: null arguments");
    return read_rows((const iq_dense_pages *)a->dense, (const iq_int4_pages *)a->int4, (int)a->dtype,
                     (const int32_t *)a->tables, a->bt_stride, a->bt_cols, (const int32_t *)a->cu_seqlens, a->n_seq,
                     a->max_seqlen, a->tokens, (const int32_t *)a->start, (void *)a->k, a->k_st, a->k_sh, (void *)a->v,
                     a->v_st, a->v_sh, (void *)a->stream);
}
