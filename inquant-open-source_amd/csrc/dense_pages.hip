// Exact pages (gfx950): rows into pages, the rows a budget keeps of a prompt,
// and eviction in place.
//
// A pool holds key and value [pages, H, B, 128] of 16-bit rows and, beside
// every row, its accumulated attention weight (f32) and its position in the
// sequence (i32), [pages, H, B] each.  Cache row r of a sequence is row r % B
// of the page that its block table names at r / B; the heads of a sequence
// hold the same number of rows but, once rows were evicted, not the same
// positions.
#include <type_traits>

#include "dense_common.h"

namespace {

// ---------------------------------------------------------------- rows into pages

// Rows of sequence `seq` that an entry point considers.
__device__ __forceinline__ uint32_t dense_length(const int32_t *cu, int seq, uint32_t max_len)
{
    const int32_t have = cu[seq + 1] - cu[seq];
    const uint32_t len = have > 0 ? (uint32_t)have : 0;
    return len < max_len ? len : max_len;
}

struct WriteArgs {
    const uint16_t *k, *v;
    int64_t k_st, k_sh, v_st, v_sh;          // element strides (token, head)
    const int32_t *cu, *start, *positions;   // start / positions may be null
    const float *weights;                    // [H, w_stride] or null
    int64_t w_stride;
    const int32_t *keep;                     // [n, H, kept] or null
    int64_t kept;
    uint32_t max_len;                        // a sequence's rows past it are left out
    DensePool pool;
};

// Bound by memory: 512 bytes of keys and values are read and written per row
// and head.  Sixteen lanes move a row (16 bytes of its key and of its value
// each), a workgroup sixteen (row, head) pairs, heads innermost: it reads one
// contiguous range of token-major rows (with `keep` rows are innermost: it
// writes one contiguous range of a head's pages).  The rows stream past the
// caches, and one row per lane keeps eight wavefronts on a SIMD: 61994 rows of
// seven prompts, 8 heads: 92 us (5.6 TB/s), 98 with ordinary stores, 106 with
// four rows a lane one after the other, 111 with four at once.
constexpr int WR_ITEMS = 16;

__global__ __launch_bounds__(256) void write_rows_kernel(WriteArgs a)
{
    const int seq = blockIdx.y, lane = threadIdx.x & 15;
    const uint32_t H = (uint32_t)a.pool.H, kept = (uint32_t)a.kept;
    const int64_t t0 = a.cu[seq];
    const uint32_t len = dense_length(a.cu, seq, a.max_len), item = blockIdx.x * WR_ITEMS + (threadIdx.x >> 4);
    if (item >= (uint64_t)(a.keep ? kept : len) * H) return;
    uint32_t h, j, source;
    if (a.keep) {
        h = item / kept;
        j = item - h * kept;
        source = (uint32_t)a.keep[((int64_t)seq * H + h) * kept + j];
    } else {
        j = source = item / H;
        h = item - j * H;
    }
    const int64_t start = a.start ? a.start[seq] : 0, row = start + j;
    const int64_t page = dense_page(a.pool, seq, row), at = row & (a.pool.B - 1), token = t0 + source;
    if (source >= len || page < 0) return;               // an entry below 0 is past any length
    const u32x4 kv = ld16(a.k + token * a.k_st + h * a.k_sh + 8 * lane);
    const u32x4 vv = ld16(a.v + token * a.v_st + h * a.v_sh + 8 * lane);
    __builtin_nontemporal_store(
        kv, (u32x4 *)(a.pool.key + page * a.pool.k_sp + h * a.pool.k_sh + at * a.pool.k_st + 8 * lane));
    __builtin_nontemporal_store(
        vv, (u32x4 *)(a.pool.value + page * a.pool.v_sp + h * a.pool.v_sh + at * a.pool.v_st + 8 * lane));
    if (lane == 0 && a.pool.weights) {
        const int64_t o = (page * H + h) * a.pool.B + at;
        a.pool.weights[o] = a.weights ? a.weights[h * a.w_stride + token] : 0.0f;
        a.pool.positions[o] = (a.positions ? a.positions[seq] : (int32_t)start) + (int32_t)source;
    }
}

// ---------------------------------------------------------------- selection

// The `budget` largest of a row of sort keys, ties to the lowest index, by one
// workgroup: the key of rank `budget` from three radix passes (11, 11 and 10
// bits, histograms in LDS), then ranks in index order from one sum over the
// threads.  A thread holds up to 32 consecutive keys of a chunk of 32768 in
// registers, and what it finds of them (kept, tied) as masks of 32 bits.  Its
// wavefront reads them side by side and passes them on through LDS (a lane's own
// keys are 128 bytes from the next lane's: 9500 cycles of 40000 for a row of
// 32000, read so).  Longer rows are read again in every pass.
constexpr int SEL_NT = 1024, SEL_WAVES = SEL_NT / 64, SEL_CHUNK = SEL_NT * 32;

// Greater is better: NaN, then -inf .. +inf (both zeros alike), then the rows
// that are always kept.  0 is no row.
__device__ __forceinline__ uint32_t sort_key(float w, bool always)
{
    const uint32_t u = __float_as_uint(w + 0.0f);   // -0 + 0 = +0
    const uint32_t key = w != w ? 1u : u & 0x80000000u ? ~u : u | 0x80000000u;
    return always ? 0xffffffffu : key;
}

struct __attribute__((aligned(16))) SelectSmem {
    union {
        uint32_t stage[SEL_NT * 36];          // a thread's keys, 16 bytes apart from the next thread's
        uint32_t hist[4][2048 + 8];           // neighbouring lanes count apart, on other banks
    };
    uint32_t wave_sum[SEL_WAVES], wave_ties[SEL_WAVES];
    uint32_t prefix, need, match;             // threshold bits so far, entries still to take of those that match them, these
};

// Inclusive sum over the wavefront: sums of 1, 2, 4, .. 16 lanes of a row by
// row shifts, then a row's last lane broadcast to the rows behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}

__device__ __forceinline__ uint32_t wave_inclusive(uint32_t v)
{
    v += dpp_u<0x111, 0xf>(v);               // row_shr:1
    v += dpp_u<0x112, 0xf>(v);
    v += dpp_u<0x114, 0xf>(v);
    v += dpp_u<0x118, 0xf>(v);
    v += dpp_u<0x142, 0xa>(v);               // row_bcast:15 into rows 1 and 3
    return v + dpp_u<0x143, 0xc>(v);         // row_bcast:31 into rows 2 and 3
}

// load(index, end, from, to, whole) -> the sort keys of four indices, of which only
// those below `end` count (all, if whole), for a wavefront that takes [from, to);
// emit(index, rows, kept, rank): of the 32 indices from `index` on, the mask of those that are rows and of those
// that are kept, and the number of kept ones before.  K keys per thread and
// chunk.
template <int K, bool ONE, class Load, class Emit>
__device__ __forceinline__ void select_largest(SelectSmem &sm, uint32_t len, uint32_t budget, Load load, Emit emit)
{
    constexpr uint32_t CHUNK = SEL_NT * K;     // ONE: at least the row
    constexpr bool STAGED = ONE && K > 4;
    // copies of the first pass's histogram, which counts every key (32000 rows: 33000
    // cycles with 4, 34000 with 2 or 8; an atomic of 64 keys takes 17)
    constexpr int COPIES = K > 16 ? 4 : 2;
    const uint32_t t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    uint32_t key[K];
    uint32_t rows = 0;                           // mask of those that are rows
    bool whole = false;                          // uniform: all of the wavefront's are
    auto read = [&](uint32_t base, uint32_t n, auto all) {
        const uint32_t from = base + wave * 64 * K;
#pragma unroll
        for (int j = 0; j < K; j += 4) {
            const uint32_t i = STAGED ? 64 * j + 4 * lane : lane * K + j;    // of the wavefront's keys
            u32x4 v = load(from + i, base + n, from, from + 64 * K, all);
            if (!all)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) v[e] = from + i + e < base + n ? v[e] : 0;
            if constexpr (STAGED) *(u32x4 *)(sm.stage + (64 * wave + i / K) * (K + 4) + i % K) = v;
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) key[j + e] = v[e];
        }
        if constexpr (STAGED) {                  // within the wavefront
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
            for (int j = 0; j < K; j += 4) {
                const u32x4 v = *(const u32x4 *)(sm.stage + t * (K + 4) + j);
#pragma unroll
                for (int e = 0; e < 4; ++e) key[j + e] = v[e];
            }
        }
    };
    auto fill = [&](uint32_t base) {
        const uint32_t n = len - base < CHUNK ? len - base : CHUNK, at = t * K;
        rows = at >= n ? 0 : n - at >= K ? (uint32_t)((1ull << K) - 1) : (1u << (n - at)) - 1;
        whole = (wave + 1) * 64 * K <= n;
        if (whole) read(base, n, std::true_type{});
        else read(base, n, std::false_type{});
    };
    // mask of this thread's keys for which f holds: a compare and an add with its carry each
    auto where = [&](auto f) {
        uint32_t m = 0;
#pragma unroll
        for (int j = K - 1; j >= 0; --j) m = m + m + (f(key[j]) ? 1u : 0u);
        return m;
    };
    if (ONE && len) fill(0);
    uint32_t prefix = 1, need = 0;               // len <= budget: every row's key is at least 1
    bool all = true;                             // uniform: whose key is the threshold is kept
    if (len > budget) {
        prefix = 0;
        need = budget;
        if (STAGED) __syncthreads();             // the histograms take the place of the staged keys
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const uint32_t mask = pass == 2 ? 1023 : 2047;
            const uint32_t above = pass == 0 ? 0 : pass == 1 ? 0xffe00000u : 0xfffffc00u;
            const int copies = pass == 0 ? COPIES : 2;
#pragma unroll
            for (int c = 0; c < COPIES; ++c)
                if (c < copies) sm.hist[c][t] = sm.hist[c][t + SEL_NT] = 0;
            __syncthreads();
            uint32_t *const hist = sm.hist[lane & (copies - 1)];
            for (uint32_t base = 0; base < len; base += CHUNK) {
                if (!ONE) fill(base);
                // what is no row counts as the lowest key, below every threshold
                if (pass == 0 && whole) {
#pragma unroll
                    for (int j = 0; j < K; ++j) atomicAdd(&hist[key[j] >> 21], 1u);
                } else if (pass == 0) {
#pragma unroll
                    for (int j = 0; j < K; ++j)
                        if (key[j]) atomicAdd(&hist[key[j] >> 21], 1u);
                } else {
#pragma unroll
                    for (int j = 0; j < K; ++j)
                        if ((key[j] & above) == prefix) atomicAdd(&hist[(key[j] >> shift) & mask], 1u);
                }
            }
            __syncthreads();
            // thread t takes the bins 2047 - 2 t and 2046 - 2 t: sums from the largest down
            uint32_t hi = 0, lo = 0;
#pragma unroll
            for (int c = 0; c < COPIES; ++c)
                if (c < copies) {
                    hi += sm.hist[c][2047 - 2 * t];
                    lo += sm.hist[c][2046 - 2 * t];
                }
            const uint32_t upto = wave_inclusive(hi + lo);
            if (lane == 63) sm.wave_sum[wave] = upto;
            __syncthreads();
            uint32_t before = upto - hi - lo;
#pragma unroll
            for (uint32_t w = 0; w < SEL_WAVES; ++w) before += w < wave ? sm.wave_sum[w] : 0;
            if (before < need && need <= before + hi + lo) {
                const bool top = need <= before + hi;
                sm.prefix = prefix | ((top ? 2047 - 2 * t : 2046 - 2 * t) << shift);
                sm.need = need - before - (top ? 0 : hi);
                sm.match = top ? hi : lo;
            }
            __syncthreads();
            prefix = sm.prefix;
            need = sm.need;
        }
        all = __builtin_amdgcn_readfirstlane(sm.match == need);
    }
    uint32_t sure0 = 0, ties0 = 0;               // kept for sure, and ties, in the chunks before
    for (uint32_t base = 0; base < len; base += CHUNK) {
        if (!ONE) fill(base);
        const uint32_t floor = all ? prefix - 1 : prefix;    // the threshold is a row's key, at least 1
        uint32_t kept = where([&](uint32_t k) { return k > floor; });
        const uint32_t ns = (uint32_t)__popc(kept), us = wave_inclusive(ns);
        uint32_t ties = 0, nt = 0, ut = 0;
        if (!all) {
            ties = where([&](uint32_t k) { return k == prefix; });
            nt = (uint32_t)__popc(ties);
            ut = wave_inclusive(nt);
        }
        if (lane == 63) {
            sm.wave_sum[wave] = us;
            sm.wave_ties[wave] = ut;
        }
        __syncthreads();
        uint32_t s = sure0 + us - ns, e = ties0 + ut - nt;
#pragma unroll
        for (uint32_t w = 0; w < SEL_WAVES; ++w) {
            const uint32_t ws = sm.wave_sum[w], wt = sm.wave_ties[w];
            sure0 += ws;
            ties0 += wt;
            s += w < wave ? ws : 0;
            e += w < wave ? wt : 0;
        }
        __syncthreads();
        // of the ties the first `need` of the row are kept
        uint32_t take = e < need ? need - e : 0;
        if (take < nt) {
            uint32_t rest = ties;
            for (; take; --take) rest &= rest - 1;
            ties &= ~rest;
        }
        emit(base + t * K, rows, kept | ties, s + (e < need ? e : need));
    }
}

// The same with as few keys per thread as the row needs.
template <class Load, class Emit>
__device__ __forceinline__ void select_rows_of(SelectSmem &sm, uint32_t len, uint32_t budget, Load load, Emit emit)
{
    if (len <= SEL_NT * 4) select_largest<4, true>(sm, len, budget, load, emit);
    else if (len <= SEL_NT * 8) select_largest<8, true>(sm, len, budget, load, emit);
    else if (len <= SEL_NT * 16) select_largest<16, true>(sm, len, budget, load, emit);
    else if (len <= SEL_CHUNK) select_largest<32, true>(sm, len, budget, load, emit);
    else select_largest<32, false>(sm, len, budget, load, emit);
}

struct SelectArgs {
    const float *weights;
    int64_t w_stride;
    const int32_t *cu;
    uint32_t max_len;                        // a sequence's rows past it are left out
    int64_t budget, sink, recent;
    int32_t *keep;
};

// Four floats from index i on, at a 4-byte alignment; those from `end` on are
// not read.
typedef float f32x4_unaligned __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ f32x4 load_four(const float *p, uint32_t i, uint32_t end)
{
    if (i + 4 <= end) return (f32x4)ldg_at<f32x4_unaligned>(p, 4 * i);
    f32x4 x = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
        if (i + e < end) x[e] = ldg_at<float>(p, 4 * (i + e));
    return x;
}

__global__ __launch_bounds__(SEL_NT) void select_rows_kernel(SelectArgs a)
{
    __shared__ SelectSmem sm;
    const int h = blockIdx.x, seq = blockIdx.y;
    const float *w = a.weights + h * a.w_stride + a.cu[seq];
    int32_t *keep = a.keep + ((int64_t)seq * gridDim.x + h) * a.budget;
    const uint32_t rows = dense_length(a.cu, seq, a.max_len), sink = (uint32_t)a.sink, recent = (uint32_t)a.recent;
    select_rows_of(
        sm, rows, (uint32_t)a.budget, [&](uint32_t i, uint32_t end, uint32_t from, uint32_t to, auto whole) {
            u32x4 keys;
            const f32x4 x = whole ? (f32x4)ldg_at<f32x4_unaligned>(w, 4 * i) : load_four(w, i, end);
            if (whole && from >= sink && to + recent <= rows) {          // uniform: none is kept always
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) keys[e] = sort_key(x[e], false);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) keys[e] = sort_key(x[e], i + e < sink || i + e + recent >= rows);
            }
            return keys;
        },
        [&](uint32_t i, uint32_t, uint32_t kept, uint32_t rank) {
            for (; kept; kept &= kept - 1) keep[rank++] = (int32_t)(i + __builtin_ctz(kept));
        });
    for (int64_t i = (int64_t)rows + threadIdx.x; i < a.budget; i += SEL_NT) keep[i] = -1;
}

// ---------------------------------------------------------------- eviction

struct EvictArgs {
    DensePool pool;
    const int32_t *lengths, *seen;
    int64_t max_tokens, budget, sink, recent, most;   // most: moves of a head at most
    int32_t *new_lengths;                             // null where another launch writes them
    int32_t *moves;                                   // [n * H, 1 + 2 most]: count, evicted places, rows from behind
};

__device__ __forceinline__ void evict_length(const EvictArgs &a, int seq)
{
    const int32_t have = a.lengths[seq];
    a.new_lengths[seq] = have < a.budget ? have : (int32_t)a.budget;
}

// Chooses the rows of one (head, sequence) and lists the moves: the evicted
// places below the budget in order, and the kept rows behind it from the last.
// MOVE: at most FEW of them, listed in LDS and made here (16 sequences of 2049
// rows, one to move: 8.7 us, and 12 with a launch of its own for the move).
constexpr int FEW = IQ_DENSE_FEW_MOVES;

template <bool MOVE>
__global__ __launch_bounds__(SEL_NT) void evict_select_kernel(EvictArgs a)
{
    __shared__ SelectSmem sm;
    __shared__ int32_t few[1 + 2 * FEW];
    const int h = blockIdx.x, seq = blockIdx.y, H = a.pool.H, B = a.pool.B;
    const int64_t have = a.lengths[seq];
    const int64_t len = have < a.max_tokens ? have : a.max_tokens;
    int32_t *list = MOVE ? few : a.moves + ((int64_t)seq * H + h) * (1 + 2 * a.most);
    if (MOVE && a.new_lengths && h == 0 && threadIdx.x == 0) evict_length(a, seq);
    if (len <= a.budget) {
        if (!MOVE && threadIdx.x == 0) list[0] = 0;
        return;
    }
    const int64_t newest = (int64_t)a.seen[seq] - a.recent;
    int32_t *holes = list + 1, *behind = holes + a.most;
    const int32_t *table = a.pool.tables + seq * a.pool.bt_stride;
    const uint32_t budget = (uint32_t)a.budget;
    select_rows_of(
        sm, (uint32_t)len, budget,
        [&](uint32_t i, uint32_t end, uint32_t, uint32_t, auto whole) {
            // four rows of one page; a row of an id outside the pool counts as NaN
            const int32_t id = table[whole || i < end ? i >> a.pool.shift : 0];
            const bool ok = id >= 0 && id < a.pool.pages;
            const int64_t o = ((int64_t)(ok ? id : 0) * H + h) * B + (i & (B - 1));
            const f32x4 w = ldg<f32x4>(a.pool.weights + o);
            const i32x4 p = ldg<i32x4>(a.pool.positions + o);
            u32x4 keys;
#pragma unroll
            for (int e = 0; e < 4; ++e) keys[e] = ok ? sort_key(w[e], p[e] < a.sink || p[e] >= newest) : 1u;
            return keys;
        },
        [&](uint32_t i, uint32_t rows, uint32_t kept, uint32_t rank) {
            const uint32_t below = i >= budget ? 0 : budget - i >= 32 ? ~0u : (1u << (budget - i)) - 1;
            // evicted places below the budget: as many before one as indices less kept ones
            uint32_t hole = i - rank;
            for (uint32_t m = rows & ~kept & below; m; m &= m - 1) holes[hole++] = (int32_t)(i + __builtin_ctz(m));
            rank += (uint32_t)__popc(kept & below);
            if (i < budget && budget - i <= 32 && (below & rows) >> (budget - 1 - i)) list[0] = (int32_t)(budget - rank);
            for (uint32_t m = kept & ~below; m; m &= m - 1)
                behind[budget - 1 - rank++] = (int32_t)(i + __builtin_ctz(m));
        });
    if constexpr (MOVE) {
        __syncthreads();
        const int n = list[0];
        int32_t from[FEW * 16 / SEL_NT], to[FEW * 16 / SEL_NT];
#pragma unroll
        for (int i = 0; i < FEW * 16 / SEL_NT; ++i) {
            const int m = i * (SEL_NT / 16) + (threadIdx.x >> 4);
            from[i] = m < n ? behind[n - 1 - m] : -1;
            to[i] = m < n ? holes[m] : -1;
        }
        dense_move<FEW * 16 / SEL_NT>(a.pool, seq, h, from, to, threadIdx.x & 15);
    }
}

// New lengths in the place of the old ones or of the tokens seen, which every
// head's workgroup reads: by the launch after them.
__global__ void evict_lengths_kernel(EvictArgs a, int n)
{
    const int seq = blockIdx.x * 256 + threadIdx.x;
    if (seq < n) evict_length(a, seq);
}

// Moves the kept rows into the evicted places; sixteen lanes a row.
constexpr int MV_ROWS = 16;

__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a)
{
    const int h = blockIdx.y % a.pool.H, seq = blockIdx.y / a.pool.H, lane = threadIdx.x & 15;
    const int32_t *list = a.moves + (int64_t)blockIdx.y * (1 + 2 * a.most);
    const int n = list[0];
    const int32_t *holes = list + 1, *behind = holes + a.most;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) evict_length(a, seq);
    if ((int)blockIdx.x * MV_ROWS >= n) return;
    int32_t from[MV_ROWS / 16], to[MV_ROWS / 16];
#pragma unroll
    for (int i = 0; i < MV_ROWS / 16; ++i) {
        const int m = blockIdx.x * MV_ROWS + 16 * i + (threadIdx.x >> 4);
        from[i] = m < n ? behind[n - 1 - m] : -1;
        to[i] = m < n ? holes[m] : -1;
    }
    dense_move<MV_ROWS / 16>(a.pool, seq, h, from, to, lane);
}

}  // namespace

extern "C" int iq_dense_write(const void *k, const void *v, int dtype, int64_t k_st, int64_t k_sh, int64_t v_st,
                              int64_t v_sh, const int32_t *cu_seqlens, int64_t n_seq, int64_t max_seqlen,
                              const int32_t *start, const int32_t *positions, const float *weights, int64_t w_stride,
                              const int32_t *keep, int64_t kept, const iq_dense_pages *pages, const int32_t *tables,
                              int64_t bt_stride, int64_t bt_cols, void *stream)
{
    DensePool pool;
    if (const int e = dense_pool("iq_dense_write", pages, dtype, tables, bt_stride, bt_cols, n_seq, pool)) return e;
    IQ_CHECK_ARG(k && v && cu_seqlens, "iq_dense_write: null pointer");
    IQ_CHECK_ARG(((uintptr_t)k | (uintptr_t)v) % 16 == 0 && (k_st | k_sh | v_st | v_sh) % 8 == 0,
                 "iq_dense_write: key/value rows must be 16-byte aligned");
    IQ_CHECK_ARG(max_seqlen >= 0 && max_seqlen <= 0x7fffffffLL && kept >= 0 && kept <= 0x7fffffffLL,
                 "iq_dense_write: bad row count");
    const int64_t rows = keep ? kept : max_seqlen;
    if (n_seq == 0 || rows == 0) return IQ_OK;
    const int64_t groups = (rows * pool.H + WR_ITEMS - 1) / WR_ITEMS;
    IQ_CHECK_ARG(groups <= 0xffffff, "iq_dense_write: too many rows");
    const WriteArgs a{(const uint16_t *)k, (const uint16_t *)v, k_st, k_sh, v_st, v_sh, cu_seqlens, start, positions,
                      weights, w_stride, keep, kept, (uint32_t)max_seqlen, pool};
    hipLaunchKernelGGL(write_rows_kernel, dim3((unsigned)groups, (unsigned)n_seq), dim3(256), 0, (hipStream_t)stream,
                       a);
    IQ_CHECK_LAUNCH("dense_write");
    return IQ_OK;
}

extern "C" int iq_select_rows(const float *weights, int64_t w_stride, int64_t H, const int32_t *cu_seqlens,
                              int64_t n_seq, int64_t max_seqlen, int64_t budget, int64_t sink, int64_t recent,
                              int32_t *keep, void *stream)
{
    IQ_CHECK_ARG(weights && cu_seqlens && keep, "iq_select_rows: null pointer");
    IQ_CHECK_ARG(H >= 1 && H <= 65535 && n_seq >= 0 && n_seq <= 65535 && max_seqlen >= 0 && max_seqlen <= 0x3fffffff,
                 "iq_select_rows: bad head or sequence count or length");
    IQ_CHECK_ARG(sink >= 0 && recent >= 0 && budget >= 1 && budget <= 0x7fffffffLL && sink + recent <= budget,
                 "iq_select_rows: sink and recent rows must fit the budget");
    if (n_seq == 0) return IQ_OK;
    const SelectArgs a{weights, w_stride, cu_seqlens, (uint32_t)max_seqlen, budget, sink, recent, keep};
    hipLaunchKernelGGL(select_rows_kernel, dim3((unsigned)H, (unsigned)n_seq), dim3(SEL_NT), 0, (hipStream_t)stream,
                       a);
    IQ_CHECK_LAUNCH("select_rows");
    return IQ_OK;
}

extern "C" int64_t iq_dense_evict_ints(int64_t H, int64_t n_seq, int64_t max_tokens, int64_t budget)
{
    const int64_t over = max_tokens > budget ? max_tokens - budget : 0, most = over < budget ? over : budget;
    return most <= FEW ? 0 : n_seq * H * (1 + 2 * most);
}

extern "C" int iq_dense_evict(const iq_dense_pages *pages, int dtype, const int32_t *tables, int64_t bt_stride,
                              int64_t bt_cols, const int32_t *lengths, const int32_t *seen, int64_t n_seq,
                              int64_t max_tokens, int64_t budget, int64_t sink, int64_t recent, int32_t *new_lengths,
                              int32_t *workspace, int64_t workspace_ints, void *stream)
{
    DensePool pool;
    if (const int e = dense_pool("iq_dense_evict", pages, dtype, tables, bt_stride, bt_cols, n_seq, pool)) return e;
    IQ_CHECK_ARG(pool.weights && pool.positions, "iq_dense_evict: pages without weights and positions");
    IQ_CHECK_ARG(lengths && seen && new_lengths, "iq_dense_evict: null pointer");
    IQ_CHECK_ARG(max_tokens >= 0 && max_tokens <= bt_cols * pool.B, "iq_dense_evict: max_tokens past the block tables");
    IQ_CHECK_ARG(sink >= 0 && recent >= 0 && budget >= 1 && budget <= 0x7fffffffLL && sink + recent <= budget,
                 "iq_dense_evict: sink and recent rows must fit the budget");
    const int64_t ints = iq_dense_evict_ints(pool.H, n_seq, max_tokens, budget);
    IQ_CHECK_ARG(ints == 0 || (workspace && workspace_ints >= ints), "iq_dense_evict: workspace too small");
    IQ_CHECK_ARG(n_seq * pool.H <= 65535, "iq_dense_evict: too many sequences");
    if (n_seq == 0) return IQ_OK;
    const auto away = [&](const int32_t *p) { return new_lengths + n_seq <= p || p + n_seq <= new_lengths; };
    // in the place of another sequence's length a new one would be read as its old one
    IQ_CHECK_ARG(new_lengths == lengths || away(lengths), "iq_dense_evict: new and old lengths overlap in part");
    const int64_t over = max_tokens > budget ? max_tokens - budget : 0, most = over < budget ? over : budget;
    EvictArgs a{pool, lengths, seen, max_tokens, budget, sink, recent, most, new_lengths, workspace};
    const dim3 rows((unsigned)pool.H, (unsigned)n_seq), block(SEL_NT);
    const hipStream_t st = (hipStream_t)stream;
    if (most <= FEW) {
        const bool apart = away(lengths) && away(seen);
        if (!apart) a.new_lengths = nullptr;
        hipLaunchKernelGGL(evict_select_kernel<true>, rows, block, 0, st, a);
        a.new_lengths = new_lengths;
        if (!apart)
            hipLaunchKernelGGL(evict_lengths_kernel, dim3((unsigned)((n_seq + 255) / 256)), dim3(256), 0, st, a,
                               (int)n_seq);
    } else {
        hipLaunchKernelGGL(evict_select_kernel<false>, rows, block, 0, st, a);
        hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)((most + MV_ROWS - 1) / MV_ROWS),
                                                   (unsigned)(n_seq * pool.H)), dim3(256), 0, st, a);
    }
    IQ_CHECK_LAUNCH("dense_evict");
    return IQ_OK;
}

extern "C" int iq_dense_write_from(const iq_dense_write_args *a)
{
    IQ_CHECK_ARG(a, "iq_dense_write: null arguments");
    return iq_dense_write((const void *)a->k, (const void *)a->v, (int)a->dtype, a->k_st, a->k_sh, a->v_st, a->v_sh,
                          (const int32_t *)a->cu_seqlens, a->n_seq, a->max_seqlen, (const int32_t *)a->start,
                          (const int32_t *)a->positions, (const float *)a->weights, a->w_stride,
                          (const int32_t *)a->keep, a->kept, (const iq_dense_pages *)a->pages,
                          (const int32_t *)a->tables, a->bt_stride, a->bt_cols, (void *)a->stream);
}

extern "C" int iq_select_rows_from(const iq_select_rows_args *a)
{
    IQ_CHECK_ARG(a, "iq_select_rows: null arguments");
    return iq_select_rows((const float *)a->weights, a->w_stride, a->H, (const int32_t *)a->cu_seqlens, a->n_seq,
                          a->max_seqlen, a->budget, a->sink, a->recent, (int32_t *)a->keep, (void *)a->stream);
}

extern "C" int iq_dense_evict_from(const iq_dense_evict_args *a)
{
    IQ_CHECK_ARG(a, "iq_dense_evict: null arguments");
    return iq_dense_evict((const iq_dense_pages *)a->pages, (int)a->dtype, (const int32_t *)a->tables, a->bt_stride,
                          a->bt_cols, (const int32_t *)a->lengths, (const int32_t *)a->seen, a->n_seq, a->max_tokens,
                          a->budget, a->sink, a->recent, (int32_t *)a->new_lengths, (int32_t *)a->workspace,
                          a->workspace_ints, (void *)a->stream);
}
