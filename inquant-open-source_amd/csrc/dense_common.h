// The exact pages of a layer as the kernels see them, and their host checks.
#pragma once

#include "decode_common.h"

namespace {

struct DensePool {
    uint16_t *key, *value;                   // [pages, H, B, 128]
    float *weights;                          // [pages, H, B] or null
    int32_t *positions;                      // [pages, H, B] or null
    int64_t k_sp, k_sh, k_st, v_sp, v_sh, v_st;   // element strides (page, head, row)
    int32_t pages, H, B, shift;              // B = 1 << shift
    const int32_t *tables;                   // [n, bt_stride], bt_cols entries used
    int64_t bt_stride, bt_cols;
};

// The pool page of cache row `row` of a sequence, or -1: a row outside the
// block table, or an id outside the pool.
__device__ __forceinline__ int64_t dense_page(const DensePool &p, int64_t seq, int64_t row)
{
    const int64_t column = row >> p.shift;
    if (row < 0 || column >= p.bt_cols) return -1;
    const int32_t id = p.tables[seq * p.bt_stride + column];
    return id >= 0 && id < p.pages ? id : -1;
}

// Copies cache rows from[i] of a head to cache rows to[i] (16 lanes: a row each
// of key and value, and by the first lane its weight and position; rows below 0
// are none).  All loads go before all stores: no row is both read and written.
template <int N>
__device__ __forceinline__ void dense_move(const DensePool &p, int64_t seq, int64_t h, const int32_t *from,
                                           const int32_t *to, int lane)
{
    int64_t pf[N], pt[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        pf[i] = dense_page(p, seq, from[i]);
        pt[i] = dense_page(p, seq, to[i]);
    }
    u32x4 k[N], v[N];
    float w[N];
    int32_t pos[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (pf[i] >= 0 && pt[i] >= 0) {
            const int64_t r = from[i] & (p.B - 1), o = (pf[i] * p.H + h) * p.B + r;
            k[i] = ld16(p.key + pf[i] * p.k_sp + h * p.k_sh + r * p.k_st + 8 * lane);
            v[i] = ld16(p.value + pf[i] * p.v_sp + h * p.v_sh + r * p.v_st + 8 * lane);
            w[i] = p.weights[o];
            pos[i] = p.positions[o];
        }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (pf[i] >= 0 && pt[i] >= 0) {
            const int64_t r = to[i] & (p.B - 1), o = (pt[i] * p.H + h) * p.B + r;
            *(u32x4 *)(p.key + pt[i] * p.k_sp + h * p.k_sh + r * p.k_st + 8 * lane) = k[i];
            *(u32x4 *)(p.value + pt[i] * p.v_sp + h * p.v_sh + r * p.v_st + 8 * lane) = v[i];
            if (lane == 0) {
                p.weights[o] = w[i];
                p.positions[o] = pos[i];
            }
        }
}

// Checks the pages and block tables of an entry point and fills `pool`.
inline int dense_pool(const char *who, const iq_dense_pages *pages, int dtype, const int32_t *tables,
                      int64_t bt_stride, int64_t bt_cols, int64_t n_seq, DensePool &pool)
{
    IQ_CHECK_ARG(pages && pages->key && pages->value, "%s: null pages", who);
    IQ_CHECK_ARG(dtype == IQ_BF16 || dtype == IQ_F16, "%s: rows must be bf16 or f16", who);
    IQ_CHECK_ARG(pages->heads >= 1 && pages->heads <= 65535, "%s: %lld KV heads", who, (long long)pages->heads);
    IQ_CHECK_ARG(pages->pages >= 1 && pages->pages <= 0x7fffffffLL, "%s: bad page count", who);
    const int64_t B = pages->block_tokens;
    IQ_CHECK_ARG(B == 16 || B == 32 || B == 64 || B == 128 || B == 256, "%s: %lld tokens per page", who, (long long)B);
    IQ_CHECK_ARG((pages->key | pages->value) % 16 == 0 &&
                     (pages->k_sp | pages->k_sh | pages->k_st | pages->v_sp | pages->v_sh | pages->v_st) % 8 == 0,
                 "%s: page rows must be 16-byte aligned", who);
    // the rows of a 64-token tile are addressed by 32-bit byte offsets
    IQ_CHECK_ARG(pages->k_st >= 0 && pages->v_st >= 0 && pages->k_st < (1LL << 24) && pages->v_st < (1LL << 24),
                 "%s: row stride too large", who);
    IQ_CHECK_ARG((pages->weights == 0) == (pages->positions == 0) && (pages->weights | pages->positions) % 16 == 0,
                 "%s: weights and positions go together, 16-byte aligned", who);
    IQ_CHECK_ARG(n_seq >= 0 && n_seq <= 65535, "%s: bad sequence count", who);
    IQ_CHECK_ARG(bt_cols >= 0 && bt_cols * B <= 0x7fffffffLL && (tables || n_seq == 0 || bt_cols == 0),
                 "%s: bad block tables", who);
    int shift = 4;
    while ((1 << shift) < B) ++shift;
    pool = DensePool{(uint16_t *)pages->key, (uint16_t *)pages->value, (float *)pages->weights,
                     (int32_t *)pages->positions, pages->k_sp, pages->k_sh, pages->k_st, pages->v_sp, pages->v_sh,
                     pages->v_st, (int32_t)pages->pages, (int32_t)pages->heads, (int32_t)B, shift, tables, bt_stride,
                     bt_cols};
    return IQ_OK;
}

}  // namespace
