"""4-bit pages: a paged cache whose rows are coded one by one, and appended in place.

The packed pages of ``layout`` code a page once it is full, with a dense tail
beside it, and answer one token per step.  These hold every row at 4 bits from
the start (144 bytes per token and KV head, 512 in exact pages), so a row goes to
its place at once and any number of new tokens reads them.

* ``append_rows``     the new tokens of running sequences: queries and keys
                      rotated by their positions, keys and values into exact
                      pages (``DensePages``) or 4-bit pages, in one launch;
* ``read_rows``       rows of either kind of pages as token-major rows;
* ``int4_decode``     one token's attention per sequence over 4-bit pages;
* ``int4_attention``  the attention of the last tokens of each sequence: drafted
                      tokens, or a chunk of a prompt.

Per group of 32 channels a row holds a step s and a zero point z; code n stands
for (n - z) s, off by at most s / 2 from a value within the group's range, which
takes in 0.  s is the range's 15th, rounded up to six significant bits, from
2^-14 to 2048: values beyond 15 * 2048 saturate.  A group with an infinity or a
NaN reads as NaN.

Everything is enqueued on the current stream of the tensors' GPU; nothing is
read back.  Lengths, positions and block tables live on the device and are
trusted as the other entry points trust them: page ids outside the pool and rows
outside a block table are skipped, not reported.  The reference has no
counterpart.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from inquant import _native as nat
from .dense import DensePages, _F32, _ROWS, _apart, _call, _cu, _entry, _ints, _on_gpu, _ptr, _status, _tables
from .layout import BLOCK_SIZES

ROW_BYTES = 144          # of a token and head: 2 x 64 of codes, 2 x 8 of steps and zero points


@dataclass(frozen=True, eq=False)
class Int4Pages:
    """The 4-bit pages of one layer: ``pool`` uint8 [pages, kv_heads, block_size *
    144] (page and head strides that are multiples of 16, 16-byte aligned).  The
    tensor's address is taken here, once: it must keep its memory.  A deep copy or
    a pickle holds memory of its own."""
    pool: torch.Tensor

    def __post_init__(self):
        pool = self.pool
        if pool.ndim != 3 or pool.dtype != torch.uint8 or pool.shape[0] < 1 or pool.shape[1] < 1 \
                or pool.shape[2] not in [ROW_BYTES * b for b in BLOCK_SIZES]:
            raise ValueError("Expected a uint8 pool [pages, kv_heads, 16/32/64/128/256 * 144]")
        # any stride will do for a dimension of one
        sp, sh = (s if n > 1 else 16 for n, s in zip(pool.shape[:2], pool.stride()))
        if pool.stride(2) != 1 or sp % 16 or sh % 16 or sp <= 0 or sh <= 0 or pool.data_ptr() % 16:
            raise ValueError("pages must be contiguous per head, 16-byte aligned and not expanded")
        block = pool.shape[2] // ROW_BYTES
        p = nat.Int4PagesDesc(pool.data_ptr(), sp, sh, pool.shape[0], pool.shape[1], block)
        for name, value in (("_pages", p), ("_desc", ctypes.addressof(p)), ("_gpu", pool.get_device()),
                            ("block_size", block), ("heads", pool.shape[1])):
            object.__setattr__(self, name, value)

    def __reduce__(self):       # copies and pickles describe the tensor that they hold
        return type(self), (self.pool,)

    @classmethod
    def allocate(cls, pages, block_size, heads, device="cuda"):
        """A pool of its own."""
        return cls(torch.empty((pages, heads, block_size * ROW_BYTES), dtype=torch.uint8, device=device))

    @property
    def nbytes(self):
        """Bytes of the rows."""
        return self.pool.numel()


def _kind(pages):
    """Addresses of the descriptors of exact and of 4-bit pages, one of them 0."""
    if isinstance(pages, DensePages):
        return pages._desc, 0
    if isinstance(pages, Int4Pages):
        return 0, pages._desc
    raise ValueError("Expected DensePages or Int4Pages")


def _rows(t, what, heads=None):
    """(tokens, heads, token stride, head stride, address) of token-major rows."""
    shape, stride, at = t.shape, t.stride(), t.data_ptr()
    if len(shape) != 3 or shape[2] != 128 or heads is not None and shape[1] != heads:
        raise ValueError(f"Expected {what} [tokens, heads, 128]")
    n, h, _ = shape
    # any stride will do for a dimension of one
    st, sh = stride[0] if n > 1 else 0, stride[1] if h > 1 else 0
    if stride[2] != 1 or (st | sh) % 8 or at % 16:
        raise ValueError(f"{what} rows must be contiguous and 16-byte aligned")
    return n, h, st, sh, at


def _overlap(x, y, size):
    """Whether rows x and y (as _rows gives them, of elements of ``size`` bytes) may
    share memory.  Heads of one tensor [tokens, heads, 128] side by side do not, nor
    rows side by side within a head [tokens, heads, 3 * 128]."""
    n, h, st, sh, x0 = x
    m, g, yt, yh, y0 = y
    wx, wy = size * ((h - 1) * sh + 128), size * ((g - 1) * yh + 128)    # of a token
    if x0 + size * (n - 1) * st + wx <= y0 or y0 + size * (m - 1) * yt + wy <= x0:
        return False
    if n == m and n > 1 and st == yt and st > 0:         # a token's rows within each stride
        at = (y0 - x0) % (size * st)
        if at >= wx and at + wy <= size * st and wx <= size * st:
            return False
    # any row of either lies whole strides from its first
    every = size * math.gcd(st, sh, yt, yh)
    return not every or not 128 * size <= (y0 - x0) % every <= every - 128 * size


def _rows_apart(n, h, st, sh):
    """Whether no two of n x h rows of 128 elements share memory."""
    if sh >= 128 and st >= sh * (h - 1) + 128:
        return True
    if n * h < 2:
        return True
    if n == 1 or h == 1:
        return (sh if n == 1 else st) >= 128
    return st >= 128 and sh >= st * (n - 1) + 128


def append_rows(query, key, value, cu_seqlens, max_seqlen, pages, block_tables, start=None, *, rotation=None,
                positions=None, interleaved=False, factors=None, output=None):
    """New tokens of running sequences into the pages (``DensePages`` or
    ``Int4Pages``), with the position rotation on the way; returns the rotated
    queries.

    query [tokens, Hq, 128] (None: none, and None is returned), key and value
    [tokens, kv_heads, 128] of bf16 or f16 (exact pages: of their dtype; views of
    one projection will do).  Row t of sequence i (cu_seqlens int32 [sequences +
    1]; rows from max_seqlen on are left out) goes to cache row start[i] + t
    (``start`` int32 [sequences], None: 0) and stands at position positions[i] + t
    (``positions`` int32 [sequences], None: ``start``).

    ``rotation`` f32 [positions, r], r a multiple of 16 up to 128: the cosines and
    then the sines of each position's r / 2 angles (None: no rotation).  Channels j
    and j + r / 2 are a pair, or 2 j and 2 j + 1 if ``interleaved``; channels from r
    on stay.  A position that the table does not hold gives NaN.  ``factors`` f32
    [kv_heads, 128] then multiply the queries of the KV head and divide its keys,
    which leaves their products (outlier channels brought to the others' size cost
    their group of 4-bit codes less).  Products and sums round to f32 each, what is
    stored or returned once more.

    Exact pages with weights get a weight of 0 and the position beside each row.
    ``output`` [tokens, Hq, 128] of the query dtype may be ``query`` itself.  Rows of
    no sequence, and those past max_seqlen, are not written; rows that a block
    table does not reach are left out.  Whatever cu_seqlens says, no row lies past
    the tensors, and a sequence whose offset is negative has none.  The inputs must
    not lie in the pages."""
    dense, int4 = _kind(pages)
    heads, gpu, dtype = pages.heads, pages._gpu, key.dtype
    k, v = _rows(key, "key", heads), _rows(value, "value", heads)
    tokens = k[0]
    if v[0] != tokens or dtype not in _ROWS or value.dtype is not dtype or dense and dtype is not pages._dtype:
        raise ValueError("key and value must have one shape and be BF16 or FP16, of the pages' dtype for exact pages")
    cu, n = _cu(cu_seqlens)
    table = _tables(block_tables, n)
    if start is not None:
        start = _ints(start, (n,), "start rows [sequences]")
    if positions is not None:
        positions = _ints(positions, (n,), "positions [sequences]")
    angles = rotary = 0
    if rotation is not None:
        if rotation.ndim != 2 or rotation.dtype is not _F32 or not rotation.is_contiguous() or rotation.data_ptr() % 16:
            raise ValueError("Expected a contiguous, 16-byte aligned float32 rotation [positions, channels]")
        angles, rotary = rotation.shape
        if angles < 1 or rotary % 16 or not 16 <= rotary <= 128:
            raise ValueError("A rotation has positions, and 16 to 128 channels in steps of 16")
    if factors is not None and (factors.shape != (heads, 128) or factors.dtype is not _F32
                                or not factors.is_contiguous() or factors.data_ptr() % 16):
        raise ValueError("Expected contiguous, 16-byte aligned float32 factors [kv_heads, 128]")
    max_seqlen = int(max_seqlen)
    if max_seqlen < 0:
        raise ValueError("max_seqlen must not be negative")
    _on_gpu(gpu, "append_rows", query, key, value, cu, block_tables, start, positions, rotation, factors, output)
    q = out = (0, 0, 0, 0, 0)
    if query is not None:
        q = _rows(query, "query")
        if q[0] != tokens or query.dtype is not dtype or q[1] < 1 or q[1] % heads:
            raise ValueError("Expected a query [tokens, heads, 128] of the key's dtype, its heads a multiple of KV heads")
        if output is None:
            output = torch.empty(query.shape, dtype=dtype, device=query.device)
        out = q if output is query else _rows(output, "output", q[1])
        if out[0] != tokens or output.dtype is not dtype or not _rows_apart(*out[:4]):
            raise ValueError("output must be [tokens, heads, 128] of the query's dtype, its rows apart")
        if tokens and (out != q and _overlap(out, q, 2) or _overlap(out, k, 2) or _overlap(out, v, 2)):
            raise ValueError("output must be the query itself or share no memory with the inputs")
    elif output is not None:
        raise ValueError("an output needs a query")
    max_seqlen = min(max_seqlen, tokens)
    if max_seqlen == 0:
        return output
    _call(gpu, "iq_append_rows_from", q[4], k[4], v[4], nat.dtype_code(dtype), q[2], q[3], k[2], k[3], v[2], v[3], q[1],
          cu.data_ptr(), n, max_seqlen, tokens, _ptr(start), _ptr(positions), _ptr(rotation), angles, rotary, bool(interleaved),
          _ptr(factors), dense, int4, *table, out[4], out[2], out[3])
    return output


def read_rows(pages, block_tables, cu_seqlens, max_seqlen, key, value, start=None):
    """Rows of the pages (``DensePages`` or ``Int4Pages``) into token-major key
    and value [tokens, kv_heads, 128], which are returned: of the pages' dtype, or
    of bf16, f16 or f32 for 4-bit pages, whose values bf16 alone rounds.

    Token t of sequence i (cu_seqlens int32 [sequences + 1]; tokens from max_seqlen
    on are left out) takes cache row start[i] + t (``start`` int32 [sequences], None:
    0).  Tokens of no sequence, and those whose row has no page, are not written, nor
    is anything past the tensors, whatever cu_seqlens says.  The rows must not lie
    in the pages."""
    dense, int4 = _kind(pages)
    heads, gpu, dtype = pages.heads, pages._gpu, key.dtype
    k, v = _rows(key, "key", heads), _rows(value, "value", heads)
    tokens = k[0]
    if v[0] != tokens or value.dtype is not dtype or (dtype is not pages._dtype if dense else dtype not in (*_ROWS, _F32)):
        raise ValueError("key and value must have one shape and the pages' dtype (BF16, FP16 or float32 for 4-bit pages)")
    size = 4 if dtype is _F32 else 2
    if not _rows_apart(*k[:4]) or not _rows_apart(*v[:4]) or tokens and _overlap(k, v, size):
        raise ValueError("the rows of key and value must not overlap")
    (cu, n), max_seqlen = _cu(cu_seqlens), int(max_seqlen)
    table = _tables(block_tables, n)
    if start is not None:
        start = _ints(start, (n,), "start rows [sequences]")
    if max_seqlen < 0:
        raise ValueError("max_seqlen must not be negative")
    _on_gpu(gpu, "read_rows", key, value, cu, block_tables, start)
    max_seqlen = min(max_seqlen, tokens)
    if max_seqlen:
        _call(gpu, "iq_read_rows_from", dense, int4, nat.dtype_code(dtype), *table, cu.data_ptr(), n, max_seqlen,
              tokens, _ptr(start), k[4], k[2], k[3], v[4], v[2], v[3])
    return key, value


def _attention(what, query, cu, n, max_seqlen, pages, block_tables, lengths, max_tokens, scale, workspace, output):
    if not isinstance(pages, Int4Pages):
        raise ValueError("Expected Int4Pages")
    shape, heads, max_tokens = query.shape, pages.heads, int(max_tokens)
    if len(shape) != 3 or shape[2] != 128 or query.dtype not in _ROWS:
        raise ValueError("Expected a BF16 or FP16 query [tokens, heads, 128]")
    tokens, hq, _ = shape
    if hq < 1 or hq % heads or hq // heads > 16:
        raise ValueError("Expected 1..16 query heads per KV head")
    lengths = _ints(lengths, (n,), "lengths [sequences]")
    table = _tables(block_tables, n)
    if not 0 <= max_tokens <= table[2] * pages.block_size:
        raise ValueError("max_tokens must fit the block tables")
    if not abs(scale) <= 2.0 ** 126:
        raise ValueError("the scale must be finite, as a float32 too")
    gpu = pages._gpu
    _on_gpu(gpu, what, query, cu, block_tables, lengths, output)
    qs = query.stride()
    if qs[2] != 1 or qs[0] % 8 or qs[1] % 8 or query.data_ptr() % 16:
        query = query.clone(memory_format=torch.contiguous_format)
        qs = query.stride()
    if output is None:
        output = torch.empty(shape, dtype=query.dtype, device=query.device)
    dtype, os = output.dtype, output.stride()
    if output.shape != shape or os[2] != 1 or dtype is not query.dtype and dtype is not _F32:
        raise ValueError("output must be [tokens, heads, 128] of the query dtype or float32")
    if not _rows_apart(tokens, hq, os[0], os[1]) and not _apart(tokens, hq, *os[:2]):
        raise ValueError("the output's rows must not overlap")
    if n == 0 or tokens == 0 or max_seqlen == 0:
        return output
    # a workgroup reads its queries before it writes their outputs, and no other's
    at, to = query.data_ptr(), output.data_ptr()
    if at < to + (4 if dtype is _F32 else 2) * ((tokens - 1) * os[0] + (hq - 1) * os[1] + 128) \
            and to < at + 2 * ((tokens - 1) * qs[0] + (hq - 1) * qs[1] + 128) and not (at == to and dtype is query.dtype and os == qs):
        raise ValueError("output must be the query itself or lie apart from it")
    # the scratch that is there serves most calls; the library says when it does not
    scratch, have, stream = workspace.floats(0, query.device)
    args = [at, nat.dtype_code(query.dtype), qs[0], qs[1], hq, _ptr(cu), n, tokens, max_seqlen,
            pages._desc, *table, lengths.data_ptr(), max_tokens, scale, scratch, have, to, os[0], os[1],
            nat.IQ_F32 if dtype is _F32 else nat.dtype_code(dtype), stream]
    status = _status(gpu, "iq_int4_attention_from", *args)
    if status:
        need = _entry("iq_int4_workspace_floats")(hq, heads, n, tokens, max_seqlen, max_tokens)
        if need > have:
            args[16:18] = workspace.floats(need, query.device)[:2]
            status = _status(gpu, "iq_int4_attention_from", *args)
        nat.check(status)
    return output


def int4_decode(query, pages, block_tables, lengths, max_tokens, scale, workspace, output=None):
    """One token's attention per sequence over its 4-bit pages.

    query [sequences, Hq, 128] of bf16 or f16, at most 16 query heads per KV head;
    block_tables int32 [sequences, pages per sequence]; lengths int32 [sequences],
    the rows each sequence holds, the newest token's among them (max_tokens >= all
    of them; a sequence without rows gives zeros).  Returns (or fills) output
    [sequences, Hq, 128] of the query dtype or float32.  The rows are taken as they
    are, logits and sums in 32 bits, softmax weights in f16 (11 bits down to 2^-28
    of the largest).  The workspace must live as long as a graph that captured the
    call."""
    return _attention("int4_decode", query, None, query.shape[0], 1, pages, block_tables, lengths, max_tokens, scale,
                      workspace, output)


def int4_attention(query, cu_seqlens, max_seqlen, pages, block_tables, lengths, max_tokens, scale, workspace,
                   output=None):
    """Causal attention of the last tokens of each sequence over its 4-bit pages.

    query [tokens, Hq, 128]: the tokens [cu_seqlens[i], cu_seqlens[i + 1]) of
    sequence i (cu_seqlens int32 [sequences + 1], max_seqlen >= every count; those
    past it are not written) are the last of the lengths[i] rows that it holds,
    which were appended before.  Each sees the rows up to its own; a token before
    the first row gives zeros.  Drafted tokens, or a chunk of a prompt behind the
    rows of the chunks before.  Otherwise as ``int4_decode``; tokens of no sequence
    are not written."""
    (cu, n), max_seqlen = _cu(cu_seqlens), int(max_seqlen)
    if max_seqlen < 0:
        raise ValueError("max_seqlen must not be negative")
    return _attention("int4_attention", query, cu, n, min(max_seqlen, query.shape[0]), pages, block_tables, lengths,
                      max_tokens, scale, workspace, output)
