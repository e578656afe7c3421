"""Exact pages on the GPU against plain 64-bit forms: decode and accumulated weights, writing, eviction and a
prompt's way through all of them."""
import math

import pytest
import torch

from densecase import (attend, cache_rows, generator, i32, keep_rows, offsets, output_bound, pool, rows, tables)

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _workspace():
    from inquant.triton_attention import SharedDecodeWorkspace
    return SharedDecodeWorkspace()


def _fields(pages):
    return [t for t in (pages.key, pages.value, pages.weights, pages.positions) if t is not None]


def _same(pages, want):
    """Every field bit for bit, a NaN like any other."""
    for name in ("key", "value", "weights", "positions"):
        got, exp = getattr(pages, name), getattr(want, name)
        if got is not None:
            bits = torch.int16 if got.element_size() == 2 else torch.int32
            differ = int((got.cpu().contiguous().view(bits) != exp.contiguous().view(bits)).sum())
            assert differ == 0, (name, differ)


# ---------------------------------------------------------------- decode

def _check_decode(q, pages, table, lengths, scale, out, before, accumulate):
    total = before.double().clone() if before is not None else None
    slacks = [0.0]
    for i, n in enumerate(lengths):
        if n == 0:
            assert (out[i] == 0).all()
            continue
        k, v = cache_rows(pages.key, table[i], n), cache_rows(pages.value, table[i], n)
        exp, _, w, slack = attend(q[i].unsqueeze(1), k, v, scale)
        bound = output_bound(v, pages.key.dtype, out.dtype, slack)
        err = float((out[i].double() - exp[:, 0]).abs().max())
        assert err <= bound, (i, n, err, bound)
        if accumulate:
            at = torch.arange(n, device="cuda")
            total[table[i, at // pages.block_size].long(), :, at % pages.block_size] += w.t()
            slacks.append(slack)
    if before is not None:
        got = pages.weights.double()
        # a weight: twice a logit's error and the roundings of exp, lse and the sums over heads and partitions
        bound = (got - before.double()).abs() * (4 * max(slacks) + 2.0 ** -18) + total.abs() * 2.0 ** -23
        assert ((got - total).abs() <= bound).all()


DECODE = [
    # hq, h, B, lengths
    (28, 4, 16, [1, 0, 15, 16, 17, 63]),
    (28, 4, 16, [300]),
    (16, 1, 16, [64, 65, 127, 128]),
    (8, 8, 32, [255, 256, 257, 2]),
    (14, 2, 64, [1000, 3, 511]),
    (32, 8, 128, [129, 700, 0]),
    (12, 1, 256, [5000, 256, 255]),
    (2, 2, 16, [0]),
    (28, 4, 16, [40000, 9, 33333]),
    (14, 2, 32, [512, 511, 449, 1, 0]),
    (28, 4, 64, [513, 600]),
    (8, 8, 16, [700] * 140),
]


@pytest.mark.parametrize("case", range(len(DECODE)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["plain", "halves", "token_major"])
def test_decode_matches_64_bits(case, dtype, layout):
    from inquant_vllm import DensePages, dense_decode
    hq, h, B, lengths = DECODE[case]
    print(f"dense decode {hq}/{h} B={B} {lengths} {dtype} {layout}", flush=True)
    gen = generator(case * 7 + 1)
    count = sum(-(-n // B) for n in lengths) + 3
    pages = pool(gen, count, h, B, dtype, layout)
    table = tables(gen, lengths, B, count, columns=-(-max(*lengths, 1) // B) + 2)
    # rows that no sequence holds are poisoned: nothing of them may be read into a result
    held = torch.zeros((count, B), dtype=torch.bool, device="cuda")
    for i, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        held[table[i, at // B].long(), at % B] = True
    bad = (~held)[:, None, :, None].expand(count, h, B, 128)
    pages.key.masked_fill_(bad, math.nan)
    pages.value.masked_fill_(bad, math.inf)
    q = rows(gen, len(lengths), hq, 128, dtype=dtype)
    longest, workspace = max(lengths), _workspace()
    n32 = i32(lengths)
    out = dense_decode(q, pages, table, n32, longest, SCALE, workspace)
    before = pages.weights.clone()
    out32 = torch.full(q.shape, math.nan, device="cuda")
    # a bound above the lengths changes nothing but the split
    dense_decode(q, pages, table, n32, table.shape[1] * B, SCALE, workspace, out32, accumulate=True)
    assert out.dtype == dtype
    _check_decode(q, pages, table, lengths, SCALE, out, None, False)
    _check_decode(q, pages, table, lengths, SCALE, out32, before, True)
    rest = ~held[:, None].expand_as(before)
    assert torch.equal(pages.weights[rest], before[rest])


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_decode_scales_and_strided_queries(scale):
    from inquant_vllm import dense_decode
    print(f"dense decode scale {scale}", flush=True)
    gen = generator(3)
    lengths, h, hq, B = [70, 333], 2, 6, 16
    pages = pool(gen, 40, h, B, torch.bfloat16)
    table = tables(gen, lengths, B, 40)
    fused = rows(gen, 2, hq + 5, 128, dtype=torch.bfloat16)
    out = torch.full((2, hq + 1, 128), 7.0, device="cuda")
    before = pages.weights.clone()
    dense_decode(fused[:, 3:3 + hq], pages, table, i32(lengths), 333, scale, _workspace(), out[:, :hq],
                 accumulate=True)
    _check_decode(fused[:, 3:3 + hq], pages, table, lengths, scale, out[:, :hq], before, True)
    assert (out[:, hq] == 7.0).all()


def test_decode_skips_ids_outside_the_pool_and_adds_shared_pages():
    from inquant_vllm import dense_decode
    gen = generator(4)
    h, hq, B = 2, 8, 16
    pages = pool(gen, 12, h, B, torch.float16)
    # sequence 0: page 3, an id below and one past the pool, page 5; sequences 1 and 2 share page 7
    table = i32([[3, -1, 12, 5], [7, 1, 0, 0], [7, 2, 0, 0], [-5, 99, 0, 0]])
    lengths = [60, 20, 32, 30]
    q = rows(gen, 4, hq, 128, dtype=torch.float16)
    before = pages.weights.clone()
    out = dense_decode(q, pages, table, i32(lengths), 60, SCALE, _workspace(), accumulate=True)
    total = before.double().clone()
    slacks = []
    live = [[(3, 16), (5, 12)], [(7, 16), (1, 4)], [(7, 16), (2, 16)], []]
    for i, parts in enumerate(live):
        if not parts:
            assert (out[i] == 0).all()
            continue
        k = torch.cat([pages.key[p, :, :m] for p, m in parts], 1)
        v = torch.cat([pages.value[p, :, :m] for p, m in parts], 1)
        exp, _, w, slack = attend(q[i].unsqueeze(1), k, v, SCALE)
        assert float((out[i].double() - exp[:, 0]).abs().max()) <= output_bound(v, torch.float16, out.dtype, slack)
        slacks.append(slack)
        at = 0
        for p, m in parts:
            total[p, :, :m] += w[:, at:at + m]
            at += m
    bound = (total - before.double()) * (4 * max(slacks) + 2.0 ** -18) + total * 2.0 ** -22
    assert ((pages.weights.double() - total).abs() <= bound).all()


def test_decode_one_query_of_odd_strides():
    from inquant_vllm import dense_decode
    gen = generator(6)
    pages = pool(gen, 10, 1, 16, torch.bfloat16)
    table, lengths = tables(gen, [77], 16, 10), i32([77])
    wide = rows(gen, 2 * 128 + 1, dtype=torch.bfloat16)
    want = dense_decode(wide[:128].clone().view(1, 1, 128), pages, table, lengths, 77, SCALE, _workspace())
    # rows of one sequence and head may have any stride
    out = torch.empty(300, dtype=torch.bfloat16, device="cuda").as_strided((1, 1, 128), (5, 3, 1))
    assert dense_decode(wide.as_strided((1, 1, 128), (3, 5, 1)), pages, table, lengths, 77, SCALE, _workspace(),
                        out).data_ptr() == out.data_ptr()
    assert torch.equal(out, want)
    with pytest.raises(ValueError, match="overlap"):
        dense_decode(wide[:128].view(1, 1, 128).expand(1, 4, 128), pages, table, lengths, 77, SCALE, _workspace(),
                     out.expand(1, 4, 128))
    # and a row that is not aligned is copied
    want = dense_decode(wide[1:129].clone().view(1, 1, 128), pages, table, lengths, 77, SCALE, _workspace())
    assert torch.equal(dense_decode(wide[1:129].view(1, 1, 128), pages, table, lengths, 77, SCALE, _workspace()), want)


@pytest.mark.parametrize("poison", [math.nan, math.inf])
@pytest.mark.parametrize("length,bound", [(60, 60), (200, 500), (1500, 1500), (700, 700)])
def test_ids_outside_the_pool_let_nothing_of_page_0_through(poison, length, bound):
    from inquant_vllm import dense_decode
    print(f"dense decode outside {poison} {length} {bound}", flush=True)
    gen = generator(length)
    h, hq, B, n = 4, 8, 16, 800 if length == 700 else 2     # 800 sequences: one workgroup takes all rows of each
    count = -(-length // B) + 1
    pages = pool(gen, count, h, B, torch.bfloat16)
    pages.key[0], pages.value[0] = poison, poison
    table = (1 + torch.arange(-(-bound // B), device="cuda") % (count - 1)).to(torch.int32).expand(n, -1).clone()
    outside = torch.arange(table.shape[1], device="cuda") % 3 == 1
    table[:, outside] = i32([-1, count])[torch.arange(int(outside.sum()), device="cuda") % 2]
    q = rows(gen, 1, hq, 128, dtype=torch.bfloat16).expand(n, -1, -1)
    before = pages.weights.clone()
    out = dense_decode(q, pages, table, i32([length] * n), bound, SCALE, _workspace(), accumulate=True)
    at = torch.arange(length, device="cuda")
    at = at[~outside[at // B]]
    page = table[0, at // B].long()
    k, v = (f[page, :, at % B].transpose(0, 1) for f in (pages.key, pages.value))
    exp, _, w, slack = attend(q[0].unsqueeze(1), k, v, SCALE)
    assert float((out.double() - exp[:, 0]).abs().max()) <= output_bound(v, torch.bfloat16, torch.bfloat16, slack)
    total = before.double()
    total[page, :, at % B] += n * w.t()
    # every sequence's weight is added in turn: n roundings of the sum
    bound = (total - before.double()).abs() * (4 * slack + 2.0 ** -18) + total.abs() * (n + 1) * 2.0 ** -24
    assert ((pages.weights.double() - total).abs() <= bound).all()


def test_pages_past_2_31_elements():
    """Rows past 2^32 bytes of the pool: decoded, written and evicted."""
    from inquant_vllm import DensePages, dense_decode, evict_rows, write_rows
    gen = generator(5)
    h, B, count, dtype = 8, 256, 9000, torch.bfloat16
    pages = DensePages.allocate(count, B, h, dtype)
    assert pages.key.numel() > 1 << 31
    table = i32([[8999, 0, 8500]])
    key, value = rows(gen, 700, h, 128, dtype=dtype), rows(gen, 700, h, 128, dtype=dtype)
    weights = torch.rand((h, 700), generator=gen, device="cuda")
    write_rows(key, value, offsets([700]), 700, pages, table, weights=weights)
    for field, want in ((pages.key, key), (pages.value, value)):
        assert torch.equal(cache_rows(field, table[0], 700), want.transpose(0, 1))
    assert torch.equal(cache_rows(pages.weights, table[0], 700), weights)
    q, before = rows(gen, 1, 16, 128, dtype=dtype), pages.weights.clone()
    out = dense_decode(q, pages, table, i32([700]), 700, SCALE, _workspace(), accumulate=True)
    _check_decode(q, pages, table, [700], SCALE, out, before, True)
    evict_rows(pages, table, i32([700]), i32([700]), 700, 300, sink=4, recent=100)
    kept = cache_rows(pages.positions, table[0], 300).long().sort(-1).values
    for head in range(h):
        assert set(range(4)) | set(range(600, 700)) <= set(kept[head].tolist())
        where = cache_rows(pages.positions, table[0], 300)[head].long()
        assert torch.equal(cache_rows(pages.key, table[0], 300)[head], key[where, head])
        assert torch.equal(cache_rows(pages.value, table[0], 300)[head], value[where, head])


def test_decode_in_a_graph_replays_with_new_lengths_on_another_stream():
    from inquant_vllm import dense_decode
    gen = generator(6)
    h, hq, B, dtype = 4, 28, 16, torch.bfloat16
    pages = pool(gen, 300, h, B, dtype)
    table = tables(gen, [1500, 900], B, 300)
    lengths, q = i32([1500, 3]), rows(gen, 2, hq, 128, dtype=dtype)
    out = torch.empty_like(q)
    start = pages.weights.clone()
    graph, stream, workspace = torch.cuda.CUDAGraph(), torch.cuda.Stream(), _workspace()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        dense_decode(q, pages, table, lengths, 1500, SCALE, workspace, out, accumulate=True)
    torch.cuda.current_stream().wait_stream(stream)
    with torch.cuda.graph(graph, stream=stream):
        dense_decode(q, pages, table, lengths, 1500, SCALE, workspace, out, accumulate=True)
    for now in ([1500, 3], [1, 900], [777, 0], [777, 512]):
        lengths.copy_(i32(now))
        q.copy_(rows(gen, 2, hq, 128, dtype=dtype))
        pages.weights.copy_(start)
        graph.replay()
        got, weights = out.clone(), pages.weights.clone()
        pages.weights.copy_(start)
        eager = dense_decode(q, pages, table, lengths, 1500, SCALE, _workspace(), accumulate=True)
        torch.cuda.synchronize()
        assert torch.equal(got, eager) and torch.equal(weights, pages.weights)
        _check_decode(q, pages, table, now, SCALE, got, start, True)


def test_decode_captured_before_its_workspace_grew():
    """A graph replays on the scratch it was captured with, whatever outgrew it since."""
    from inquant_vllm import dense_decode
    gen = generator(7)
    h, hq, B, dtype = 2, 16, 32, torch.float16
    pages = pool(gen, 700, h, B, dtype)
    table = tables(gen, [3000, 17000], B, 700)
    q, workspace = rows(gen, 2, hq, 128, dtype=dtype), _workspace()
    small, big = i32([3000]), i32([3000, 17000])
    out, start = torch.empty((1, hq, 128), dtype=dtype, device="cuda"), pages.weights.clone()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        dense_decode(q[:1], pages, table[:1], small, 3000, SCALE, workspace, out, accumulate=True)
    stream.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(stream):
            dense_decode(q, pages, table, big, 17000, SCALE, workspace, accumulate=True)
            others = [torch.full((1 << 18,), float(i), device="cuda") for i in range(8)]
            pages.weights.copy_(start)
            graph.replay()
        torch.cuda.synchronize()
        _check_decode(q[:1], pages, table, [3000], SCALE, out, start, True)
        assert all((x == float(i)).all() for i, x in enumerate(others))


# ---------------------------------------------------------------- writing

def _plain_write(pages, key, value, lengths, table, start, positions, weights, keep):
    B = pages.block_size
    first = 0
    for i, n in enumerate(lengths):
        for h in range(pages.heads):
            source = list(range(n)) if keep is None else keep[i, h].tolist()
            for j, r in enumerate(source):
                row = start[i] + j
                if not (0 <= r < n and 0 <= row < table.shape[1] * B):
                    continue
                p = int(table[i, row // B])
                if not 0 <= p < pages.key.shape[0]:
                    continue
                pages.key[p, h, row % B], pages.value[p, h, row % B] = key[first + r, h], value[first + r, h]
                if pages.weights is not None:
                    pages.weights[p, h, row % B] = 0.0 if weights is None else weights[h, first + r]
                    pages.positions[p, h, row % B] = positions[i] + r
        first += n


def _copy(pages):
    from inquant_vllm import DensePages
    return DensePages(*(t.cpu().clone(memory_format=torch.contiguous_format) for t in _fields(pages)))


WRITE = [
    # B, heads, lengths, start, kept, with weights, evictable, layout
    (16, 4, [1, 1, 1], [0, 15, 16], 0, True, True, "plain"),
    (16, 3, [37, 0, 50], None, 0, False, True, "halves"),
    (64, 2, [130, 5], [60, 0], 0, True, True, "token_major"),
    (256, 1, [300], [3], 0, False, False, "plain"),
    (32, 2, [90, 40, 7], None, 20, True, True, "halves"),
    (16, 8, [200, 33], [5, 250], 70, True, True, "plain"),
]


@pytest.mark.parametrize("case", range(len(WRITE)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write_rows_is_exact(case, dtype):
    from inquant_vllm import write_rows
    B, heads, lengths, start, kept, weighted, evictable, layout = WRITE[case]
    print(f"write rows {WRITE[case]} {dtype}", flush=True)
    gen = generator(20 + case)
    n, tokens = len(lengths), sum(lengths)
    pages = pool(gen, 60, heads, B, dtype, layout, evictable)
    table = torch.randperm(60, generator=gen, device="cuda")[:n * 17].view(n, 17).to(torch.int32)
    table[0, 1], table[-1, 2] = -1, 60                       # rows of ids outside the pool are left out
    fused = rows(gen, tokens, 2 * heads + 1, 128, dtype=dtype)
    key, value = fused[:, :heads], fused[:, heads + 1:]
    weights = torch.rand((heads, tokens + 3), generator=gen, device="cuda")[:, :tokens] if weighted else None
    keep = None
    if kept:
        keep = torch.full((n, heads, kept), -1, dtype=torch.int32, device="cuda")
        for i, x in enumerate(lengths):
            m = min(x, kept - 3)
            order = torch.rand((heads, x), generator=gen, device="cuda").argsort(-1)[:, :m].sort(-1).values
            keep[i, :, :m] = order.to(torch.int32)
            keep[i, :, kept - 1] = x                         # outside the sequence
    positions = None if start is None else [s + 1000 for s in start]
    exp = _copy(pages)
    _plain_write(exp, key.cpu(), value.cpu(), lengths, table.cpu(), start or [0] * n, positions or [0] * n,
                 None if weights is None else weights.cpu(), None if keep is None else keep.cpu())
    write_rows(key, value, offsets(lengths), max(lengths), pages, table, None if start is None else i32(start),
               positions=None if start is None else i32(positions), weights=weights, keep=keep)
    _same(pages, exp)


def test_write_one_token_of_odd_strides():
    from inquant_vllm import write_rows
    gen = generator(30)
    pages = pool(gen, 4, 1, 16, torch.float16)
    # dimensions of one, whose strides say nothing
    key = torch.as_strided(rows(gen, 4, 128, dtype=torch.float16), (1, 1, 128), (3, 5, 1))
    write_rows(key, key, offsets([1]), 1, pages, i32([[2]]), i32([7]))
    assert torch.equal(pages.key[2, 0, 7], key[0, 0]) and torch.equal(pages.value[2, 0, 7], key[0, 0])
    assert pages.weights[2, 0, 7] == 0 and pages.positions[2, 0, 7] == 7


# ---------------------------------------------------------------- selection

def _sel_weights(gen, h, tokens, kind):
    w = (2 * torch.randn((h, tokens), generator=gen, device="cuda")).exp()
    if kind == "ties":
        w = torch.randint(0, 3, (h, tokens), generator=gen, device="cuda").float() - 1
    elif kind == "odd":
        pick = torch.randint(0, 8, (h, tokens), generator=gen, device="cuda")
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45)):
            w[pick == i] = x
    elif kind == "equal":
        w = torch.full((h, tokens), 0.25, device="cuda")
    return w


SELECT = [
    # lengths, budget, sink, recent
    ([5, 0, 1, 9], 4, 1, 2),
    ([100, 64, 63, 65], 64, 4, 10),
    ([1000, 1024, 1025, 7], 300, 0, 0),
    ([3000], 3000, 4, 100),
    ([3000], 2999, 0, 2999),
    ([2048, 4097], 1, 1, 0),
    ([33000, 70001, 32768], 5000, 4, 128),
    ([66000], 40000, 0, 1),
]


@pytest.mark.parametrize("case", range(len(SELECT)))
@pytest.mark.parametrize("kind", ["spread", "ties", "odd", "equal"])
def test_select_rows_is_exact(case, kind):
    from inquant_vllm import select_rows
    lengths, budget, sink, recent = SELECT[case]
    print(f"select {SELECT[case]} {kind}", flush=True)
    gen = generator(40 + case)
    h = 3 if max(lengths) < 30000 else 2
    # the sequences start behind other tokens, in rows of a longer stride
    w = _sel_weights(gen, h, sum(lengths) + 11, kind)[:, 7:]
    cu = offsets(lengths)
    keep = select_rows(w, cu, max(lengths), budget, sink=sink, recent=recent)
    assert keep.shape == (len(lengths), h, budget) and keep.dtype == torch.int32
    host, got, first = w.cpu(), keep.cpu(), 0
    for i, n in enumerate(lengths):
        always = [j < sink or j >= n - recent for j in range(n)]
        for head in range(h):
            exp = keep_rows(host[head, first:first + n].tolist(), always, budget)
            assert got[i, head].tolist() == exp + [-1] * (budget - len(exp)), (i, head)
        first += n


# ---------------------------------------------------------------- eviction

def _plain_evict(pages, table, lengths, seen, budget, sink, recent):
    B = pages.block_size
    for i, n in enumerate(lengths):
        if n <= budget:
            continue
        at = torch.arange(n)
        page, row = table[i, at // B].long(), at % B
        for h in range(pages.heads):
            pos = pages.positions[page, h, row].tolist()
            kept = keep_rows(pages.weights[page, h, row].tolist(), [p < sink or p >= seen[i] - recent for p in pos],
                             budget)
            inside = set(kept)
            to = torch.tensor([j for j in range(budget) if j not in inside], dtype=torch.int64)
            origin = torch.tensor([j for j in kept if j >= budget], dtype=torch.int64)
            for field in _fields(pages):
                field[page[to], h, row[to]] = field[page[origin], h, row[origin]]


EVICT = [
    # B, heads, lengths, budget, sink, recent
    (16, 4, [33, 32, 5, 0, 40], 32, 4, 8),
    (16, 2, [65] * 7, 64, 4, 16),
    (64, 3, [500, 301, 299], 300, 0, 0),
    (256, 2, [900], 1, 0, 0),
    (32, 2, [1500, 1100], 1000, 4, 996),
    (128, 1, [2000, 37], 40, 1, 30),
    (256, 2, [34000, 33001], 33000, 4, 500),
    (16, 1, [70000], 1024, 4, 128),
    (64, 2, [9000, 4000], 4100, 4, 128),
]


@pytest.mark.parametrize("case", range(len(EVICT)))
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
def test_evict_rows_is_exact(case, kind):
    from inquant_vllm import evict_rows
    B, heads, lengths, budget, sink, recent = EVICT[case]
    print(f"evict {EVICT[case]} {kind}", flush=True)
    gen = generator(60 + case)
    count = sum(-(-n // B) for n in lengths) + 2
    pages = pool(gen, count, heads, B, torch.bfloat16, ["plain", "halves", "token_major"][case % 3])
    pages.weights.copy_(_sel_weights(gen, count, heads * B, kind).view(count, heads, B))
    table = tables(gen, lengths, B, count)
    seen = [3 * n + 5 for n in lengths]
    # positions: a random part of the tokens seen, each once a head, the newest among them
    for i, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        for h in range(heads):
            order = torch.randperm(3 * n + 5, generator=gen, device="cuda")[:n].to(torch.int32)
            pages.positions[table[i, at // B].long(), h, at % B] = order
    exp = _copy(pages)
    _plain_evict(exp, table.cpu(), lengths, seen, budget, sink, recent)
    first = [t.clone() for t in _fields(pages)]
    new = evict_rows(pages, table, i32(lengths), i32(seen), max(lengths), budget, sink=sink, recent=recent)
    assert new.tolist() == [min(n, budget) for n in lengths]
    _same(pages, exp)
    # the same with the new lengths in the place of the old ones
    for t, start in zip(_fields(pages), first):
        t.copy_(start)
    held = i32(lengths)
    assert evict_rows(pages, table, held, i32(seen), max(lengths), budget, sink=sink, recent=recent, output=held) is held
    assert held.tolist() == new.tolist()
    _same(pages, exp)


def test_evict_in_a_graph_and_lengths_as_output():
    from inquant_vllm import evict_rows
    gen = generator(80)
    B, h, budget, lengths = 16, 2, 100, [130, 101, 60]
    first = pool(gen, 30, h, B, torch.float16)
    pages = type(first)(*(t.clone() for t in _fields(first)))
    table, seen, held = tables(gen, lengths, B, 30), i32([900, 900, 900]), i32(lengths)
    evict_rows(pages, table, held.clone(), seen, 130, budget, sink=4, recent=20)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        evict_rows(pages, table, held, seen, 130, budget, sink=4, recent=20, output=held)
    for seed in range(3):
        for got, start in zip(_fields(pages), _fields(first)):
            got.copy_(start)
        pages.weights.copy_(_sel_weights(generator(seed), 30, h * B, "ties").view(30, h, B))
        held.copy_(i32(lengths))
        exp = _copy(pages)
        _plain_evict(exp, table.cpu(), lengths, [900] * 3, budget, 4, 20)
        graph.replay()
        torch.cuda.synchronize()
        assert held.tolist() == [100, 100, 60]
        _same(pages, exp)


@pytest.mark.parametrize("alias", ["lengths", "seen"])
def test_evict_into_its_own_arguments(alias):
    from inquant_vllm import evict_rows
    gen = generator(81)
    B, h, budget, lengths = 16, 8, 100, [130, 101, 60] * 20
    pages = pool(gen, 600, h, B, torch.bfloat16)
    table = tables(gen, lengths, B, 600)
    args = {"lengths": i32(lengths), "seen": i32([1000 + i for i in range(60)])}
    # positions that a wrong count of tokens seen would keep or not
    pages.positions.copy_(torch.randint(0, 1100, pages.positions.shape, generator=gen, device="cuda"))
    exp = _copy(pages)
    _plain_evict(exp, table.cpu(), lengths, args["seen"].tolist(), budget, 4, 60)
    got = evict_rows(pages, table, **args, max_tokens=130, budget=budget, sink=4, recent=60, output=args[alias])
    assert got is args[alias] and got.tolist() == [100, 100, 60] * 20
    _same(pages, exp)


@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
@pytest.mark.parametrize("lengths,budget", [([8192, 8193, 4097], 4096), ([12001, 16384], 12000), ([16385, 20003, 32767], 900)],
                         ids=str)
def test_select_rows_of_every_width(lengths, budget, kind):
    from inquant_vllm import select_rows
    gen, h = generator(60), 2
    print(f"select {lengths} {budget} {kind}", flush=True)
    w = _sel_weights(gen, h, sum(lengths), kind)
    got, cpu, first = select_rows(w, offsets(lengths), max(lengths), budget, sink=3, recent=70).cpu(), w.cpu(), 0
    for i, n in enumerate(lengths):
        for head in range(h):
            exp = keep_rows(cpu[head, first:first + n].tolist(), [j < 3 or j >= n - 70 for j in range(n)], budget)
            assert got[i, head].tolist() == exp, (i, head)
        first += n


@pytest.mark.parametrize("lengths,budget", [([130, 101], 100), ([9000], 600)], ids=str)
def test_evict_of_more_always_kept_rows_than_the_budget(lengths, budget):
    from inquant_vllm import evict_rows
    gen = generator(82)
    B, h = 16, 2
    pages = pool(gen, 600, h, B, torch.bfloat16)
    table = tables(gen, lengths, B, 600)
    pages.positions.copy_(torch.randint(0, 6, pages.positions.shape, generator=gen, device="cuda"))
    for sink, recent in ((5, 0), (0, 1), (6, 1)):            # of positions 0..5 seen
        exp = _copy(pages)
        _plain_evict(exp, table.cpu(), lengths, [6] * len(lengths), budget, sink, recent)
        evict_rows(pages, table, i32(lengths), i32([6] * len(lengths)), max(lengths), budget, sink=sink, recent=recent)
        _same(pages, exp)


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_prompt_kept_to_a_budget_then_decoded(dtype):
    """Two prompts: attention and weights, the kept rows into pages, then tokens appended, attended to and evicted;
    every step against the plain form of the state before it.  Full pages are then sealed as packed pages."""
    from inquant_vllm import (DensePages, PageLayout, dense_decode, evict_rows, pack_pages, prefill_attention,
                              prefill_weights, select_rows, write_rows)
    gen = generator(90)
    hq, h, B, budget, sink, recent = 14, 2, 16, 48, 4, 12
    lengths, n = [200, 30], 2
    tokens, cu = sum(lengths), offsets(lengths)
    q, k, v = (rows(gen, tokens, x, 128, dtype=dtype) for x in (hq, h, h))
    lse = torch.empty((hq, tokens), device="cuda")
    prefill_attention(q, k, v, cu, 200, SCALE, lse=lse)
    w = prefill_weights(q, k, cu, 200, SCALE, lse=lse)
    keep = select_rows(w, cu, 200, budget, sink=sink, recent=recent)
    pages = DensePages.allocate(12, B, h, dtype)
    table = torch.randperm(12, generator=gen, device="cuda")[:8].view(2, 4).to(torch.int32)
    for t in _fields(pages)[:2]:
        t.fill_(math.nan)
    write_rows(k, v, cu, 200, pages, table, weights=w, keep=keep)
    held, seen = [min(x, budget) for x in lengths], list(lengths)
    for i in range(n):
        pos = cache_rows(pages.positions, table[i], held[i])
        assert torch.equal(pos, keep[i, :, :held[i]])
    step, one, workspace = i32(held), offsets([1] * n), _workspace()
    ids = i32(seen)
    for _ in range(25):
        q1, k1, v1 = (rows(gen, n, x, 128, dtype=dtype) for x in (hq, h, h))
        write_rows(k1, v1, one, 1, pages, table, step, positions=ids)
        step += 1
        ids += 1
        held, seen = [x + 1 for x in held], [x + 1 for x in seen]
        before = pages.weights.clone()
        out = dense_decode(q1, pages, table, step, budget + 1, SCALE, workspace, accumulate=True)
        _check_decode(q1, pages, table, held, SCALE, out, before, True)
        exp = _copy(pages)
        _plain_evict(exp, table.cpu(), held, seen, budget, sink, recent)
        evict_rows(pages, table, step, ids, budget + 1, budget, sink=sink, recent=recent, output=step)
        held = [min(x, budget) for x in held]
        assert step.tolist() == held
        _same(pages, exp)
        for i in range(n):
            pos = cache_rows(pages.positions, table[i], held[i])
            for head in range(h):
                have = set(pos[head].tolist())
                assert len(have) == held[i] and set(range(seen[i] - recent, seen[i])) <= have
    full = table[0, :budget // B].long()
    packed = pack_pages(pages.key[full], pages.value[full], PageLayout(B, h))
    assert packed.shape == (budget // B, PageLayout(B, h).page_bytes)
