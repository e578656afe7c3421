// 4-bit pages as the kernels see them: layout, codes, and host checks.
//
// A page holds, for each of its heads, B rows of 128 channels of keys and of
// values at 4 bits: B * 144 bytes,
//   key codes    [row][64 bytes]: channel c in the nibble c % 2 of byte c / 2;
//   value codes  [row / 4][channel / 8][row / 2 % 2][channel / 4 % 2][row % 2]
//                units of 16 bits: nibble c % 4 of the unit;
//   key words    [row][4 groups of 32 channels], value words [row / 4][group][row % 4].
// A word is the f16 pattern of the group's step s with the zero point z in its
// lowest four bits; code n stands for (n - z) s.  s has six significant bits
// within 2^-14 .. 2048, so (16 + n) s and (16 + z) s fit the eleven of an f16
// and their difference is (n - z) s exactly: the matrix cores take the rows as
// they are, without a rounding.
// The layouts follow the operands of the 16- and 32-row matrix products: 16
// bytes of a key row are 32 channels of one group, and 16 bytes of value codes
// are eight channels of four rows, neighbouring rows in the halves of a dword.
#pragma once

#include "decode_common.h"

namespace {

constexpr uint32_t I4_ROW = 144;             // bytes of a row's key and value

struct Int4Pool {
    uint8_t *base;
    int64_t s_page, s_head;                  // bytes
    int32_t pages, H, B, shift;              // B = 1 << shift
    const int32_t *tables;                   // [n, bt_stride], bt_cols entries used
    int64_t bt_stride, bt_cols;
};

// Eight nibbles of a dword as four pairs of f16 (16 + nibble): pair i holds
// nibbles i and i + 4, at bits 6 .. 9 of either half, whose unit is 1 there.
// The masks stand in registers, so that one instruction takes both (as literals
// they take two: no instruction of three operands holds one).
struct I4Masks {
    uint32_t field, unit;
    __device__ __forceinline__ I4Masks()
    {
        field = 0x03c003c0u;
        unit = 0x4c004c00u;
        asm("" : "+s"(field));
        asm("" : "+v"(unit));
    }
    __device__ __forceinline__ uint32_t pair(uint32_t x, int i) const
    {
        const uint32_t y = i == 0 ? x << 6 : i == 1 ? x << 2 : i == 2 ? x >> 2 : x >> 6;
        return (y & field) | unit;
    }
};

__device__ __forceinline__ f16x2 as_f16x2(uint32_t x) { return __builtin_bit_cast(f16x2, x); }
__device__ __forceinline__ uint32_t as_u32(f16x2 x) { return __builtin_bit_cast(uint32_t, x); }

// Steps and offsets (16 + z) s of two words.
struct I4Scale {
    f16x2 s, c;
};

__device__ __forceinline__ I4Scale i4_scale(uint32_t words)
{
    I4Scale r;
    r.s = as_f16x2(words & 0xffe0ffe0u);
    r.c = as_f16x2(((words << 6) & 0x03c003c0u) | 0x4c004c00u) * r.s;
    return r;
}

// (16 + n) s - (16 + z) s of a pair, in one rounding (of which there is none).
__device__ __forceinline__ uint32_t i4_value(uint32_t pair, f16x2 s, f16x2 c)
{
    return as_u32(__builtin_elementwise_fma(as_f16x2(pair), s, -c));
}

__device__ __forceinline__ f16x2 lower(f16x2 x) { return f16x2{x[0], x[0]}; }
__device__ __forceinline__ f16x2 upper(f16x2 x) { return f16x2{x[1], x[1]}; }

// Byte offsets of a head's fields within its part of a page.
__device__ __forceinline__ uint32_t i4_value_codes(uint32_t B) { return 64 * B; }
__device__ __forceinline__ uint32_t i4_key_words(uint32_t B) { return 128 * B; }
__device__ __forceinline__ uint32_t i4_value_words(uint32_t B) { return 136 * B; }

// The pool page of cache row `row` of a sequence, or -1: a row outside the
// block table, or an id outside the pool.
__device__ __forceinline__ int64_t i4_page(const Int4Pool &p, int64_t seq, int64_t row)
{
    const int64_t column = row >> p.shift;
    if (row < 0 || column >= p.bt_cols) return -1;
    const int32_t id = p.tables[seq * p.bt_stride + column];
    return id >= 0 && id < p.pages ? id : -1;
}

// Checks the pages and block tables of an entry point and fills `pool`.
inline int int4_pool(const char *who, const iq_int4_pages *pages, const int32_t *tables, int64_t bt_stride,
                     int64_t bt_cols, int64_t n_seq, Int4Pool &pool)
{
    IQ_CHECK_ARG(pages && pages->pool, "%s: null pages", who);
    IQ_CHECK_ARG(pages->heads >= 1 && pages->heads <= 65535, "%s: %lld KV heads", who, (long long)pages->heads);
    IQ_CHECK_ARG(pages->pages >= 1 && pages->pages <= 0x7fffffffLL, "%s: bad page count", who);
    const int64_t B = pages->block_tokens;
    IQ_CHECK_ARG(B == 16 || B == 32 || B == 64 || B == 128 || B == 256, "%s: %lld tokens per page", who, (long long)B);
    IQ_CHECK_ARG(pages->pool % 16 == 0 && (pages->s_page | pages->s_head) % 16 == 0 && pages->s_page >= 0 && pages->s_head >= 0,
                 "%s: pages must be 16-byte aligned", who);
    IQ_CHECK_ARG(n_seq >= 0 && n_seq <= 65535, "%s: bad sequence count", who);
    IQ_CHECK_ARG(bt_cols >= 0 && bt_cols * B <= 0x7fffffffLL && (tables || n_seq == 0 || bt_cols == 0),
                 "%s: bad block tables", who);
    int shift = 4;
    while ((1 << shift) < B) ++shift;
    pool = Int4Pool{(uint8_t *)pages->pool, pages->s_page, pages->s_head, (int32_t)pages->pages, (int32_t)pages->heads,
                    (int32_t)B, shift, tables, bt_stride, bt_cols};
    return IQ_OK;
}

}  // namespace
