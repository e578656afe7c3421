// Attention over 4-bit pages (gfx950): how a call is split, and the entry points.
#include "int4_few_dev.h"
#include "int4_many_dev.h"

namespace {

// Columns (query tokens times query heads of a KV head) from which on the kernel
// for many takes a call: below, its workgroups of 256 columns are mostly empty
// (8 sequences of up to 16K rows, 252 columns 104 us by the kernel for few and 126,
// 315 columns 160 and 128; one of 32K rows 46 and 69, 67 and 53; one of 2000 rows, where
// either ends soon, 17 and 29, 21 and 29).
constexpr int64_t MANY = 256;
constexpr int64_t ONE_MOST = 512;            // rows that one workgroup takes in a step, with no join
constexpr int64_t BATCH = 64;                // sequences of a launch that shares their rows out

// A call for many that some sequences ask little of (a chunk of a prompt beside
// single and drafted tokens) leaves sequences of at most MIXED columns to the kernel
// for few, which shares their rows out: one workgroup would walk through each (2048
// tokens beside 31 single ones behind 2K-32K rows 433 us, 2456 without; beside 31 times
// five drafted ones 556 and 2630; 1024 beside 63 single ones behind 0.5K-4K 189 and 647; the
// launches cost 8-14 in batches that have none: 4 x 512 tokens 261 and 275).
constexpr int64_t MIXED = 64;

struct Split {
    bool many, mixed;                        // the kernel for many columns; beside the one for few
    int64_t span, parts;                     // many: rows per partition, partitions
    int64_t groups, workers, width;          // few: groups of columns, workgroups that share a plane's rows (0: none), columns
    int64_t floats;                          // the whole workspace
};

Split split_of(int64_t Hq, int64_t H, int64_t n, int64_t tokens, int64_t max_seqlen, int64_t max_tokens)
{
    Split s{};
    if (max_seqlen > tokens) max_seqlen = tokens;
    if (H < 1 || Hq < H || n < 1 || max_seqlen < 1) return s;
    const int64_t cols = Hq / H * max_seqlen;
    s.many = cols > MANY;
    if (s.many) {
        // as many workgroups as run at once (one per compute unit), of eight tiles of rows at least
        const int64_t each = (cols + QT - 1) / QT, all = (tokens * (Hq / H) + QT - 1) / QT;
        const int64_t tiles = H * (n * each < all ? n * each : all), steps = (max_tokens + KT - 1) / KT;
        const int64_t parts = tiles >= 192 ? 1 : 256 / tiles, most = (steps + 7) / 8;
        const int64_t want = parts < most ? parts : most < 1 ? 1 : most;
        s.span = KT * ((steps + want - 1) / want);
        if (s.span < KT) s.span = KT;
        s.parts = max_tokens > 0 ? (max_tokens + s.span - 1) / s.span : 1;
        // Whether some sequence asks little stands on the device only (the tensor may hold tokens of no sequence), so
        // a call of more than one sequence reckons with it; but where all workgroups run at once, of eight tiles at
        // most, a short one costs less than two launches do (64 tokens beside five behind 2000 rows 29 us, 50 with
        // them; two of 64 31 and 34; 2048 tokens beside 31 single ones in a tensor of 67K 380, 2200 without)
        s.mixed = n > 1 && (H * n * each * s.parts > 256 || s.span > 8 * KT);
        // a place for each token that a sequence can have (int4_place): at most 256 * QT columns, 34 MB
        const int64_t places = n * max_seqlen < tokens ? n * max_seqlen : tokens;
        s.floats = s.parts > 1 ? places * Hq * s.parts * (D + 2) : 0;
    }
    if (!s.many || s.mixed) {
        const int64_t most = s.mixed ? MIXED : cols;
        s.width = most <= 16 ? 16 : 32;
        s.groups = (most + s.width - 1) / s.width;
        const int64_t planes = H * s.groups, steps = (max_tokens + STEP - 1) / STEP, batch = n < BATCH ? n : BATCH;
        if (max_tokens > ONE_MOST) {
            // Two workgroups per compute unit where each has enough to do, else one (one
            // sequence of 32K rows, 28 heads over 4: 16.5 us with 512, 14.2 with 256; 16 of
            // 2K-32K: 40.6 and 42.5, with 768 42.7, with 1024 47).
            const int64_t busy = s.mixed ? H : planes;       // mixed: most have one group of columns, the others end at once
            const int64_t all = batch * busy * steps > 4096 ? 512 : 256;
            s.workers = (all + busy - 1) / busy;
            if (s.workers > batch * steps) s.workers = batch * steps;
            const int64_t floats = planes * (s.workers + batch) * s.width * (D + 2);
            if (floats > s.floats) s.floats = floats;        // the two take turns with it
        }
    }
    return s;
}

// `most`: tokens of a sequence that have workgroups of their own in the join
template <bool F16, int NQ>
void launch_few(Int4Args a, int64_t most, int64_t n, hipStream_t stream)
{
    const unsigned planes = (unsigned)(a.pool.H * a.groups);
    if (a.workers == 0) {
        if (a.max_tokens > STEP) hipLaunchKernelGGL((int4_whole<F16, NQ, 8>), dim3(planes, 1, (unsigned)n), dim3(512), 0, stream, a);
        else hipLaunchKernelGGL((int4_whole<F16, NQ, 4>), dim3(planes, 1, (unsigned)n), dim3(256), 0, stream, a);
        return;
    }
    const int32_t *const lengths = a.lengths, *const cu = a.cu, *const tables = a.pool.tables;
    const uint16_t *const q = a.q;
    char *const out = (char *)a.out;
    const int tokens = a.tokens;
    for (int64_t s0 = 0; s0 < n; s0 += BATCH) {
        a.n_seq = (int32_t)(n - s0 < BATCH ? n - s0 : BATCH);
        a.lengths = lengths + s0;
        a.pool.tables = tables + s0 * a.pool.bt_stride;
        if (cu) a.cu = cu + s0;
        else {                               // token i is sequence i's
            a.q = q + s0 * a.q_st;
            a.out = out + s0 * a.o_st * (a.odt == IQ_F32 ? 4 : 2);
            a.tokens = tokens - (int32_t)s0;
        }
        hipLaunchKernelGGL((int4_shared<F16, NQ>), dim3(planes * (unsigned)a.workers), dim3(256), 0, stream, a);
        hipLaunchKernelGGL(int4_join<true>, dim3((unsigned)(a.Hq * most), (unsigned)a.n_seq), dim3(256), 0, stream, a);
    }
}

template <bool F16>
void launch_chunk(const Int4Args &a, int64_t cols, int64_t n, hipStream_t stream)
{
    const int tiles = (int)((cols + QT - 1) / QT), share = (tiles * a.pool.H + 7) / 8;
    const dim3 grid((unsigned)(8 * share), (unsigned)a.parts, (unsigned)n);
    if (a.parts > 1) {
        hipLaunchKernelGGL((int4_chunk<F16, false>), grid, dim3(64 * NW), 0, stream, a, tiles, share);
        hipLaunchKernelGGL(int4_join<false>, dim3((unsigned)((a.Hq * (int64_t)a.max_seqlen + 7) / 8), (unsigned)n), dim3(256), 0,
                           stream, a);
    }
    else hipLaunchKernelGGL((int4_chunk<F16, true>), grid, dim3(64 * NW), 0, stream, a, tiles, share);
}

}  // namespace

extern "C" int64_t iq_int4_workspace_floats(int64_t Hq, int64_t H, int64_t n_seq, int64_t tokens, int64_t max_seqlen,
                                            int64_t max_tokens)
{
    return split_of(Hq, H, n_seq, tokens, max_seqlen, max_tokens).floats;
}

extern "C" int iq_int4_attention(const void *q, int dtype, int64_t q_st, int64_t q_sh, int64_t Hq,
                                 const int32_t *cu_seqlens, int64_t n_seq, int64_t tokens, int64_t max_seqlen,
                                 const iq_int4_pages *pages, const int32_t *tables, int64_t bt_stride, int64_t bt_cols,
                                 const int32_t *lengths, int64_t max_tokens, float scale, float *workspace,
                                 int64_t workspace_floats, void *out, int64_t o_st, int64_t o_sh, int out_dtype,
                                 void *stream)
{
    Int4Pool pool;
    if (const int e = int4_pool("iq_int4_attention", pages, tables, bt_stride, bt_cols, n_seq, pool)) return e;
    IQ_CHECK_ARG(q && lengths && out, "iq_int4_attention: null pointer");
    IQ_CHECK_ARG(dtype == IQ_BF16 || dtype == IQ_F16, "iq_int4_attention: queries must be bf16 or f16");
    IQ_CHECK_ARG((uintptr_t)q % 16 == 0 && (q_st | q_sh) % 8 == 0, "iq_int4_attention: query rows must be 16-byte aligned");
    IQ_CHECK_ARG(Hq >= 1 && Hq % pool.H == 0 && Hq / pool.H <= 16, "iq_int4_attention: heads %lld / %d", (long long)Hq,
                 pool.H);
    IQ_CHECK_ARG(out_dtype >= IQ_F32 && out_dtype <= IQ_F16, "iq_int4_attention: bad output dtype");
    IQ_CHECK_ARG(max_tokens >= 0 && max_tokens <= bt_cols * pool.B && max_tokens <= 0x3fffffff,
                 "iq_int4_attention: max_tokens past the block tables");
    IQ_CHECK_ARG(tokens >= 0 && tokens <= 0x3fffffff && max_seqlen >= 0 && max_seqlen <= 0x3fffffff &&
                     (cu_seqlens || (max_seqlen == 1 && tokens == n_seq)), "iq_int4_attention: bad query tokens");
    if (n_seq == 0 || tokens == 0 || max_seqlen == 0) return IQ_OK;
    if (max_seqlen > tokens) max_seqlen = tokens;
    const Split s = split_of(Hq, pool.H, n_seq, tokens, max_seqlen, max_tokens);
    IQ_CHECK_ARG(s.floats == 0 || (workspace && workspace_floats >= s.floats), "iq_int4_attention: workspace too small");
    IQ_CHECK_ARG(s.floats == 0 || (uintptr_t)workspace % 16 == 0, "iq_int4_attention: the workspace must be 16-byte aligned");
    const int64_t G = Hq / pool.H, cols = G * max_seqlen;
    IQ_CHECK_ARG(s.parts <= 65535 && cols <= 0x3fffffff && s.groups * pool.H * (s.workers + 1) <= 0xffffff &&
                     Hq * max_seqlen <= (s.many ? 0x3fffffff : 0xffffff), "iq_int4_attention: too many rows");
    const int64_t rows = s.floats / (D + 2);
    const Int4Args a{pool, (const uint16_t *)q, q_st, q_sh, cu_seqlens, lengths, (int32_t)tokens, (int32_t)max_seqlen,
                     (int32_t)max_tokens, (int32_t)G, (int32_t)Hq, (int32_t)s.span, (int32_t)s.parts, (int32_t)n_seq,
                     (int32_t)s.groups, (int32_t)s.workers, (int32_t)s.width,
                     (int32_t)(!s.many ? MANY : s.mixed ? MIXED : 0), scale * I4_LOG2E,
                     Partials{workspace, (f32x2 *)(workspace + rows * D)}, out, o_st, o_sh, out_dtype};
    const hipStream_t st = (hipStream_t)stream;
    const bool f16 = dtype == IQ_F16;
    if (s.many) f16 ? launch_chunk<true>(a, cols, n_seq, st) : launch_chunk<false>(a, cols, n_seq, st);
    if (!s.many || s.mixed) {
        const int64_t most = s.many ? 1 : max_seqlen;        // mixed: most sequences have one
        if (s.width == 16) f16 ? launch_few<true, 1>(a, most, n_seq, st) : launch_few<false, 1>(a, most, n_seq, st);
        else f16 ? launch_few<true, 2>(a, most, n_seq, st) : launch_few<false, 2>(a, most, n_seq, st);
    }
    IQ_CHECK_LAUNCH("int4_attention");
    return IQ_OK;
}

extern "C" int iq_int4_attention_from(const iq_int4_attention_args *a)
{
    IQ_CHECK_ARG(a, "iq_int4_attention: null arguments");
    return iq_int4_attention((const void *)a->q, (int)a->dtype, a->q_st, a->q_sh, a->Hq, (const int32_t *)a->cu_seqlens,
                             a->n_seq, a->tokens, a->max_seqlen, (const iq_int4_pages *)a->pages,
                             (const int32_t *)a->tables, a->bt_stride, a->bt_cols, (const int32_t *)a->lengths,
                             a->max_tokens, (float)a->scale, (float *)a->workspace, a->workspace_floats, (void *)a->out,
                             a->o_st, a->o_sh, (int)a->out_dtype, (void *)a->stream);
}
