"""Exact pages: a paged cache of rows as they are, cut back by accumulated attention weight.

The packed pages of ``layout`` code every row; these hold bf16 or f16 rows
[pages, kv_heads, block_size, 128] (the shape ``pack_pages_into`` seals), and
beside every row the attention weight it has accumulated and its position.

* ``write_rows``       a prompt's rows, or the ones a selection kept, or the
                       new rows of running sequences, into the pages;
* ``dense_decode``     one token's attention per sequence over the pages, which
                       on request adds each row's weight;
* ``prefill_weights``  the weight each key of a prompt receives from its
                       queries, or from the last few of them;
* ``select_rows``      the rows a budget keeps of each prompt and KV head;
* ``evict_rows``       the pages of running sequences cut back to the budget,
                       in place.

Everything is enqueued on the current stream of the tensors' GPU; nothing is
read back.  Lengths, positions, block tables and kept rows live on the device
and are trusted as the other entry points trust them: page ids outside the pool
and rows outside a block table are skipped, not reported.  The reference has no
counterpart.
"""
from __future__ import annotations

import ctypes
import math
import struct
from dataclasses import dataclass

import torch

from inquant import _native as nat
from .layout import BLOCK_SIZES

_ROWS = (torch.bfloat16, torch.float16)
_I32, _F32 = torch.int32, torch.float32
_current = getattr(torch._C, "_cuda_getDevice", None)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_FEW_MOVES = 128        # iq_dense_evict takes no workspace up to here (IQ_DENSE_FEW_MOVES)


def _strides(pages):
    """Strides of page, head and row; any will do for a dimension of one."""
    return [s if n > 1 else 8 for n, s in zip(pages.shape[:3], pages.stride())]


@dataclass(frozen=True, eq=False)
class DensePages:
    """The exact pages of one layer: ``key`` and ``value`` [pages, kv_heads,
    block_size, 128] of bf16 or f16 (any page, head and row strides that are
    multiples of 8 elements, 16-byte aligned; two views of one pool will do) and,
    where rows are to be evicted, ``weights`` f32 and ``positions`` int32
    [pages, kv_heads, block_size].  The tensors' addresses are taken here, once:
    they must keep their memory.  A deep copy or a pickle holds memory of its own."""
    key: torch.Tensor
    value: torch.Tensor
    weights: torch.Tensor | None = None
    positions: torch.Tensor | None = None

    def __post_init__(self):
        key, value = self.key, self.value
        if key.ndim != 4 or key.shape != value.shape or key.shape[-1] != 128 or key.shape[2] not in BLOCK_SIZES \
                or key.shape[0] < 1 or key.shape[1] < 1:
            raise ValueError("Expected key and value pages [pages, kv_heads, 16/32/64/128/256, 128]")
        if key.dtype not in _ROWS or value.dtype != key.dtype:
            raise ValueError("Exact pages hold BF16 or FP16 rows")
        for t in (key, value):
            if t.stride(3) != 1 or any(s % 8 or s <= 0 for s in _strides(t)) or t.data_ptr() % 16:
                raise ValueError("page rows must be contiguous, 16-byte aligned and not expanded")
        if (self.weights is None) != (self.positions is None):
            raise ValueError("Weights and positions go together")
        if self.weights is not None:
            for t, dtype in ((self.weights, torch.float32), (self.positions, torch.int32)):
                if t.shape != key.shape[:3] or t.dtype != dtype or not t.is_contiguous() or t.data_ptr() % 16:
                    raise ValueError("Expected contiguous, 16-byte aligned float32 weights and int32 positions "
                                     "[pages, kv_heads, block_size]")
        side = (self.weights, self.positions)
        if len({t.device for t in (key, value, *side) if t is not None}) != 1:
            raise ValueError("all tensors must share one GPU")
        p = nat.DensePagesDesc(key.data_ptr(), value.data_ptr(), *(0 if t is None else t.data_ptr() for t in side),
                               *_strides(key), *_strides(value), *key.shape[:3])
        # what every call asks for: the descriptor and its address, the dtype and its code, the GPU, and the sizes
        for name, value in (("_pages", p), ("_desc", ctypes.addressof(p)), ("_dtype", key.dtype), ("_gpu", key.get_device()),
                            ("_code", nat.dtype_code(key.dtype)), ("block_size", key.shape[2]),
                            ("heads", key.shape[1])):
            object.__setattr__(self, name, value)

    def __reduce__(self):       # copies and pickles describe the tensors that they hold
        return type(self), (self.key, self.value, self.weights, self.positions)

    @classmethod
    def allocate(cls, pages, block_size, heads, dtype=torch.bfloat16, device="cuda", *, evictable=True):
        """A pool of its own; the rows' weights and positions start at zero."""
        shape = (pages, heads, block_size)
        side = [torch.zeros(shape, dtype=t, device=device) if evictable else None
                for t in (torch.float32, torch.int32)]
        return cls(torch.empty((*shape, 128), dtype=dtype, device=device),
                   torch.empty((*shape, 128), dtype=dtype, device=device), *side)

    @property
    def nbytes(self):
        """Bytes of the rows and of what stands beside them."""
        return sum(t.numel() * t.element_size() for t in (self.key, self.value, self.weights, self.positions)
                   if t is not None)


def _on_gpu(gpu, what, *tensors):
    """All tensors on one GPU, whose index is ``gpu``.  The common case costs one
    integer per tensor, any other takes require_gpu's errors."""
    for t in tensors:
        if t is not None and t.get_device() != gpu:
            break
    else:
        if gpu >= 0:
            return
    nat.require_gpu(*tensors, what=what)
    raise ValueError("all tensors must share one GPU")


# The arguments of the entry points that take them as a struct, 8 bytes each: Q an
# address (0: none), q a number, d the scale.  ctypes takes 2 us to convert twenty
# arguments one by one, 0.4 for a packed struct.
_ARGUMENTS = {name: struct.Struct("=" + fields).pack for name, fields in {
    "iq_dense_write": "2Q5qQ2q3QqQq2Q2qQ", "iq_select_rows": "Q2qQ5q2Q", "iq_dense_evict": "QqQ2q2Q5q2QqQ",
    "iq_dense_decode": "Q5q2Q2qQqdqQqQ3qQ", "iq_prefill_weights": "2Q5qQ6qdQqQqQqQ",
    "iq_append_rows": "3Q8qQ3q3Q3q4Q2qQ2qQ", "iq_read_rows": "2QqQ2qQ3q2Q2qQ2qQ",
    "iq_int4_attention": "Q4qQ3q2Q2qQqdQqQ3qQ"}.items()}
_entries: dict = {}


def _entry(name):
    """A library function, looked up once; with ``_from`` beside what packs its arguments."""
    found = _entries.get(name)
    if found is None:
        found = getattr(nat.lib(), name)
        if name.endswith("_from"):
            found = found, _ARGUMENTS[name[:-5]]
        _entries[name] = found
    return found


def _status(gpu, name, *args):
    """Calls the entry point with its GPU current."""
    call, pack = _entries.get(name) or _entry(name)
    args = pack(*args)
    if gpu == _current():
        return call(args)
    with torch.cuda.device(gpu):
        return call(args)


def _call(gpu, name, *args):
    """The same on the GPU's current stream; a failure raises."""
    status = _status(gpu, name, *args, _stream(gpu))
    if status:
        nat.check(status)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _ints(t, shape, what):
    if t.shape != shape or t.dtype is not _I32:
        raise ValueError(f"Expected int32 {what}")
    return t if t.is_contiguous() else t.contiguous()


def _cu(cu_seqlens):
    """The offsets, contiguous, and the number of sequences."""
    shape = cu_seqlens.shape
    if cu_seqlens.dtype is not _I32 or len(shape) != 1 or shape[0] < 2:
        raise ValueError("cu_seqlens must be an int32 [sequences + 1] tensor")
    return cu_seqlens if cu_seqlens.is_contiguous() else cu_seqlens.contiguous(), shape[0] - 1


def _tables(block_tables, n):
    shape, stride = block_tables.shape, block_tables.stride()
    if len(shape) != 2 or shape[0] != n or block_tables.dtype is not _I32 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError("Expected int32 block tables [sequences, pages per sequence]")
    return block_tables.data_ptr(), stride[0], shape[1]


def _token_rows(t, what, heads=None):
    """Shape and (token, head) strides of token-major rows."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[2] != 128 or (heads is not None and shape[1] != heads):
        raise ValueError(f"Expected {what} [tokens, heads, 128]")
    # any stride will do for a dimension of one
    st, sh = stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0
    if stride[2] != 1 or st % 8 or sh % 8 or t.data_ptr() % 16:
        raise ValueError(f"{what} rows must be contiguous and 16-byte aligned")
    return shape, (st, sh)


def _apart(n, m, a, b):
    """Whether rows of 128 elements at i a + j b, i < n and j < m, overlap nowhere."""
    at = sorted(i * a + j * b for i in range(n) for j in range(m))
    return all(y - x >= 128 for x, y in zip(at, at[1:]))


def _meet(x, y):
    """Whether two float32 tensors of rows of unit stride may share memory."""
    x0, y0 = x.data_ptr(), y.data_ptr()
    return x0 < y0 + 4 * ((y.shape[0] - 1) * y.stride(0) + y.shape[1]) \
        and y0 < x0 + 4 * ((x.shape[0] - 1) * x.stride(0) + x.shape[1])


def _budget(budget, sink, recent):
    if budget < 1 or sink < 0 or recent < 0 or sink + recent > budget:
        raise ValueError("sink and recent rows must fit a budget of at least one row")


def write_rows(key, value, cu_seqlens, max_seqlen, pages, block_tables, start=None, *, positions=None, weights=None,
               keep=None):
    """Rows of token-major key/value [tokens, kv_heads, 128] into the pages.

    Row t of sequence i (cu_seqlens int32 [sequences + 1]; rows from max_seqlen
    on are left out) goes to cache row start[i] + t of every head (``start`` int32
    [sequences], None: 0); with ``keep`` int32 [sequences, kv_heads, kept]
    (``select_rows``) head h takes only the rows keep[i, h, j], to cache row
    start[i] + j, and entries outside the sequence are skipped.  Where the pages
    have weights, the row's is weights[h, cu_seqlens[i] + t] (``weights`` f32
    [kv_heads, tokens], None: 0) and its position positions[i] + t
    (``positions`` int32 [sequences], None: ``start``).  Rows that a block table
    [sequences, pages per sequence] does not reach are left out.  key and value
    must not lie in the rows that are written."""
    heads = pages.heads
    shape, ks = _token_rows(key, "key", heads)
    vshape, vs = _token_rows(value, "value", heads)
    if shape != vshape or key.dtype is not pages._dtype or value.dtype is not pages._dtype:
        raise ValueError("key and value must have one shape and the pages' dtype")
    (cu, n), tokens = _cu(cu_seqlens), shape[0]
    table = _tables(block_tables, n)
    if start is not None:
        start = _ints(start, (n,), "start rows [sequences]")
    if positions is not None:
        positions = _ints(positions, (n,), "positions [sequences]")
    ws = (0, 1) if weights is None else weights.stride()
    if weights is not None and (weights.shape != (heads, tokens) or weights.dtype is not _F32
                                or ws[1] != 1 and tokens > 1):
        raise ValueError("Expected float32 weights [kv_heads, tokens]")
    if keep is not None:
        if keep.ndim != 3 or keep.shape[:2] != (n, heads):
            raise ValueError("Expected int32 kept rows [sequences, kv_heads, kept]")
        keep = _ints(keep, keep.shape, "kept rows [sequences, kv_heads, kept]")
    gpu = pages._gpu
    _on_gpu(gpu, "write_rows", key, value, cu, block_tables, start, positions, weights, keep)
    # a selection of no row is an address of 0, which stands for every row
    if tokens == 0 or table[2] == 0 or keep is not None and keep.shape[2] == 0:
        return
    _call(gpu, "iq_dense_write_from", key.data_ptr(), value.data_ptr(), pages._code, ks[0], ks[1], vs[0], vs[1],
          cu.data_ptr(), n, int(max_seqlen), _ptr(start), _ptr(positions), _ptr(weights), ws[0], _ptr(keep),
          0 if keep is None else keep.shape[2], pages._desc, *table)


def select_rows(weights, cu_seqlens, max_seqlen, budget, *, sink=0, recent=0, output=None):
    """The rows that a budget keeps of each sequence and KV head: the first
    ``sink`` and the last ``recent`` rows, then by weight (``weights`` f32
    [kv_heads, tokens], as ``prefill_weights`` gives them), ties to the lowest
    row, NaN last.  Returns int32 [sequences, kv_heads, budget]: ascending rows
    within the sequence, -1 behind the last.  A sequence longer than max_seqlen
    counts as its first max_seqlen rows, as ``prefill_weights`` takes it."""
    budget, sink, recent = int(budget), int(sink), int(recent)
    _budget(budget, sink, recent)
    if weights.ndim != 2 or weights.dtype is not _F32 or weights.shape[0] < 1 \
            or weights.stride(1) != 1 and weights.shape[1] > 1:
        raise ValueError("Expected float32 weights [kv_heads, tokens]")
    (cu, n), (h, tokens) = _cu(cu_seqlens), weights.shape
    gpu = weights.get_device()
    _on_gpu(gpu, "select_rows", weights, cu, output)
    if output is None:
        output = torch.empty((n, h, budget), dtype=_I32, device=weights.device)
    elif output.shape != (n, h, budget) or output.dtype is not _I32 or not output.is_contiguous():
        raise ValueError("output must be a contiguous int32 [sequences, kv_heads, budget] tensor")
    if tokens == 0:
        return output.fill_(-1)
    _call(gpu, "iq_select_rows_from", weights.data_ptr(), weights.stride(0), h, cu.data_ptr(), n, int(max_seqlen), budget,
          sink, recent, output.data_ptr())
    return output


def evict_rows(pages, block_tables, lengths, seen, max_tokens, budget, *, sink=0, recent=0, output=None):
    """Cuts every sequence of more than ``budget`` rows back to ``budget``, each
    KV head by its own weights, in place.

    lengths int32 [sequences]: the rows that each holds (max_tokens >= all of
    them); seen int32 [sequences]: the tokens that it has seen.  Kept are the
    rows at positions below ``sink`` or from seen - recent on, then by weight,
    ties to the lowest cache row, NaN last.  The evicted cache rows below the
    budget take, in order, the kept rows from the budget on, so only those
    move; every other row stays as it is.  Returns the new lengths
    min(lengths, budget), int32 [sequences] (``output`` may be ``lengths`` or ``seen``, and overlap ``lengths`` no
    other way).
    No page may belong to two of the sequences."""
    budget, sink, recent, max_tokens = int(budget), int(sink), int(recent), int(max_tokens)
    _budget(budget, sink, recent)
    if pages.weights is None:
        raise ValueError("Eviction needs pages with weights and positions")
    if lengths.ndim != 1:
        raise ValueError("Expected int32 lengths [sequences]")
    n = lengths.shape[0]
    lengths, seen = _ints(lengths, (n,), "lengths [sequences]"), _ints(seen, (n,), "tokens seen [sequences]")
    table = _tables(block_tables, n)
    if not 0 <= max_tokens <= table[2] * pages.block_size:
        raise ValueError("max_tokens must fit the block tables")
    gpu = pages._gpu
    _on_gpu(gpu, "evict_rows", lengths, seen, block_tables, output)
    if output is None:
        output = torch.empty_like(lengths)
    elif output.shape != (n,) or output.dtype is not _I32 or not output.is_contiguous():
        raise ValueError("output must be a contiguous int32 [sequences] tensor")
    elif 0 < abs(output.data_ptr() - lengths.data_ptr()) < 4 * n:
        raise ValueError("output must be lengths itself or not overlap them")
    if n == 0:
        return output
    # few moves are listed on the chip
    need, scratch = 0, None
    if max_tokens - budget > _FEW_MOVES:
        need = _entry("iq_dense_evict_ints")(pages.heads, n, max_tokens, budget)
        scratch = torch.empty(need, dtype=_I32, device=lengths.device)
    _call(gpu, "iq_dense_evict_from", pages._desc, pages._code, *table, lengths.data_ptr(), seen.data_ptr(), n, max_tokens,
          budget, sink, recent, output.data_ptr(), _ptr(scratch), need)
    return output


def dense_decode(query, pages, block_tables, lengths, max_tokens, scale, workspace, output=None, *,
                 accumulate=False):
    """One token's attention per sequence over its exact pages.

    query [sequences, Hq, 128] of the pages' dtype, at most 16 query heads per
    KV head; block_tables int32 [sequences, pages per sequence]; lengths int32
    [sequences], the rows each sequence holds, the newest token's among them
    (max_tokens >= all of them; a sequence without rows gives zeros).  Returns
    (or fills) output [sequences, Hq, 128] of the query dtype or float32.
    ``accumulate=True`` adds to each row's weight the softmax weights that the
    query heads of its KV head gave it (for a page that two sequences share,
    in an order that is not fixed); past 512 rows that takes 4 bytes of the
    workspace per sequence, query head and token of max_tokens.  The workspace
    must live as long as a graph that captured the call."""
    shape, hkv, max_tokens = query.shape, pages.heads, int(max_tokens)
    if len(shape) != 3 or shape[2] != 128 or query.dtype is not pages._dtype:
        raise ValueError("Expected a query [sequences, heads, 128] of the pages' dtype")
    n, hq, _ = shape
    if hq < 1 or hq % hkv or hq // hkv > 16:
        raise ValueError("Expected 1..16 query heads per KV head")
    if accumulate and pages.weights is None:
        raise ValueError("Accumulation needs pages with weights and positions")
    lengths = _ints(lengths, (n,), "lengths [sequences]")
    table = _tables(block_tables, n)
    if not 0 <= max_tokens <= table[2] * pages.block_size:
        raise ValueError("max_tokens must fit the block tables")
    if not math.isfinite(scale):
        raise ValueError("the scale must be finite")
    gpu = pages._gpu
    _on_gpu(gpu, "dense_decode", query, block_tables, lengths, output)
    qs = query.stride()
    if qs[2] != 1 or qs[0] % 8 or qs[1] % 8 or query.data_ptr() % 16:
        query = query.clone(memory_format=torch.contiguous_format)
        qs = query.stride()
    if output is None:
        output = torch.empty(shape, dtype=query.dtype, device=query.device)
    dtype, os = output.dtype, output.stride()
    if output.shape != shape or os[2] != 1 or dtype is not pages._dtype and dtype is not _F32:
        raise ValueError("output must be [sequences, heads, 128] of the query dtype or float32")
    if (os[1] < 128 or os[0] < 128 + os[1] * (hq - 1)) and not _apart(n, hq, *os[:2]):
        raise ValueError("the output's rows must not overlap")
    if n == 0:
        return output
    # the scratch that is there serves most calls; the library says when it does not
    scratch, have, stream = workspace.floats(0, query.device)
    args = [query.data_ptr(), pages._code, qs[0], qs[1], hq, n, pages._desc, *table, lengths.data_ptr(), max_tokens,
            scale, bool(accumulate), scratch, have, output.data_ptr(), os[0], os[1],
            nat.IQ_F32 if dtype is _F32 else pages._code, stream]
    status = _status(gpu, "iq_dense_decode_from", *args)
    if status:
        need = _entry("iq_dense_workspace_floats")(hq, hkv, n, max_tokens, bool(accumulate))
        if need > have:
            args[14:16] = workspace.floats(need, query.device)[:2]
            status = _status(gpu, "iq_dense_decode_from", *args)
        nat.check(status)
    return output


def prefill_weights(query, key, cu_seqlens, max_seqlen, scale, *, lse=None, window=None, output=None):
    """The softmax weight that each key of a prompt receives, summed over the
    queries that see it and over the query heads of its KV head: float32
    [kv_heads, tokens].

    query [tokens, Hq, 128], key [tokens, kv_heads, 128] (bf16 or f16),
    sequences as ``prefill_attention`` takes them.  Over all queries, whose
    ``lse`` [Hq, tokens] ``prefill_attention(..., lse=...)`` wrote, or with
    ``window=w`` over the last w queries of each sequence (lse optional; w at
    most 4096, or all with the lse).
    Scratch of a call: without a window 4 bytes per token, query head and range of
    queries (1 to 16 of them, by the sizes); for a window's own lse up to 256 MiB
    (or 512 bytes per query head and 64 keys, if that is more) and 4 bytes per
    query head and window row.
    A sequence longer than max_seqlen counts as its first max_seqlen tokens.
    Tokens of no sequence, and those past max_seqlen, are not written."""
    (tokens, hq, _), qs = _token_rows(query, "query")
    (rows, h, _), ks = _token_rows(key, "key")
    if tokens != rows or query.dtype not in _ROWS or key.dtype is not query.dtype:
        raise ValueError("Expected BF16 or FP16 query and key of the same tokens")
    if h < 1 or hq < 1 or hq % h:
        raise ValueError("query heads must be a multiple of KV heads")
    (cu, n), max_seqlen = _cu(cu_seqlens), int(max_seqlen)
    if max_seqlen < 1 or not (scale > 0 and math.isfinite(scale)):
        raise ValueError("max_seqlen and the scale must be positive")
    if window is not None and int(window) < 1:
        raise ValueError("the window must hold at least one query")
    if window is None and lse is None:
        raise ValueError("Weights of all queries need the lse of prefill_attention")
    if lse is not None and (lse.shape != (hq, tokens) or lse.dtype is not _F32 or lse.stride(1) != 1 and tokens > 1):
        raise ValueError("Expected a float32 lse [query heads, tokens]")
    gpu = query.get_device()
    _on_gpu(gpu, "prefill_weights", query, key, cu, lse, output)
    if output is None:
        output = torch.empty((h, tokens), dtype=_F32, device=query.device)
    elif output.shape != (h, tokens) or output.dtype is not _F32 or output.stride(1) != 1 and tokens > 1:
        raise ValueError("output must be float32 [kv_heads, tokens]")
    elif h > 1 and output.stride(0) < tokens:
        raise ValueError("the output's heads must not overlap")
    if tokens == 0:
        return output
    if lse is not None and lse.stride(0) < 1:
        lse = lse.contiguous()               # one row for every head
    if lse is not None and _meet(lse, output):
        lse = lse.clone()                    # read while weights are written
    window = 0 if window is None else min(int(window), max_seqlen)
    if lse is not None and window == max_seqlen:
        window = 0                           # every query
    if window > 4096:
        raise ValueError("Windows of more than 4096 queries and less than all are not supported")
    need = _entry("iq_prefill_weights_floats")(hq, n, max_seqlen, tokens, window, lse is not None)
    scratch = torch.empty(need, dtype=_F32, device=query.device)
    _call(gpu, "iq_prefill_weights_from", query.data_ptr(), key.data_ptr(), nat.dtype_code(query.dtype), qs[0], qs[1], ks[0],
          ks[1], cu.data_ptr(), n, max_seqlen, tokens, hq, h, window, scale, _ptr(lse),
          0 if lse is None else max(1, lse.stride(0)), scratch.data_ptr(), need, output.data_ptr(), output.stride(0))
    return output
