"""Edges of the 4-bit pages' operators on the GPU: how far weights and outputs are from 64 bits, token by token."""
import math

import pytest
import torch

import int4case as case
from densecase import EPS, i32
from inquant.triton_attention import SharedDecodeWorkspace
from inquant_vllm import DensePages, Int4Pages, append_rows, int4_attention, read_rows
from test_int4_gpu import check, gen_of, random_pool, tables_of

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def held_rows(key, value):
    """One sequence's rows [n, heads, 128] in pages of 16: the pages, their table, and the rows that they stand for."""
    n, h, _ = key.shape
    count = -(-n // 16)
    pages, table = Int4Pages.allocate(count, 16, h), torch.arange(count, dtype=torch.int32, device="cuda")[None]
    append_rows(None, key, value, i32([0, n]), n, pages, table)
    k, v = (torch.empty((n, h, 128), device="cuda") for _ in range(2))
    read_rows(pages, table, i32([0, n]), n, k, v)
    return pages, table, k.double(), v.double()


def line(weights, dtype):
    """Keys [n, 1, 128] whose logits with a query (1, 0, ...) are the numbers given, to three percent."""
    key = torch.zeros((len(weights), 1, 128), dtype=dtype, device="cuda")
    key[:, 0, 0] = weights.to(dtype)
    return key


@pytest.mark.parametrize("m, hq", [(80, 4), (300, 1), (3, 4), (40, 4)])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_a_row_with_most_of_the_weight_is_not_rounded(dtype, m, hq):
    """One row has all but a 40th of the weight, 2^5.4 times that of the row that was the largest before it.  Its own
    weight is the power of two that the others are measured by, so only they are rounded: by 2^-11 each.  The logits
    are one product each, of at most 7: with the scale 3 roundings of 2^-24, in the weights and in their sum."""
    n = 1000
    logits = torch.full((n,), -20.0, device="cuda")
    logits[0], logits[500] = 0.0, 5.3
    gen = torch.Generator().manual_seed(m)
    pages, table, k, v = held_rows(line(logits, dtype), torch.randn((n, 1, 128), generator=gen).to(dtype).cuda())
    q = torch.zeros((m, hq, 128), dtype=dtype, device="cuda")
    q[..., 0] = 1 + (torch.arange(m * hq, device="cuda").view(m, hq) % 16) / 64
    out = int4_attention(q, i32([0, m]), m, pages, table, i32([n]), n, math.log(2), SharedDecodeWorkspace(),
                         torch.empty(q.shape, dtype=F32, device="cuda"))
    p = (q[..., 0, None].double() * k[:, 0, 0] * math.log(2)).masked_fill(
        torch.arange(n, device="cuda") > n - m + torch.arange(m, device="cuda")[:, None, None], -math.inf).softmax(-1)
    rest = 1 - p[..., 500]
    assert rest.max() < 1 / 30
    bound = v.abs().max() * (rest * EPS[F16] + 2 * 7 * math.log(2) * 4 * 2.0 ** -24 + 2.0 ** -20)
    assert ((out.double() - p @ v[:, 0]).abs() <= bound[..., None]).all()


@pytest.mark.parametrize("m, hq", [(80, 4), (300, 1), (3, 4), (40, 4)])
@pytest.mark.parametrize("n", [500, 20000])             # one part, and several, most of which lack the largest weight
@pytest.mark.parametrize("least", [-22.4, -26.3])
def test_small_weights_keep_eleven_bits(m, hq, n, least):
    """Rows of 2^-22 .. 2^-28 of the largest weight, whose values alone count: each weight is rounded by 2^-11 of its
    own size.  The logits are one product each, of at most 28."""
    logits = torch.full((n,), least, device="cuda")
    logits[3] = 0.0
    value = torch.full((n, 1, 128), 0.9375, dtype=BF, device="cuda")
    value[3] = 0.0
    pages, table, k, v = held_rows(line(logits, BF), value)
    q = torch.zeros((m, hq, 128), dtype=BF, device="cuda")
    q[..., 0] = 1.0
    out = int4_attention(q, i32([0, m]), m, pages, table, i32([n]), n, math.log(2), SharedDecodeWorkspace(),
                         torch.empty(q.shape, dtype=F32, device="cuda"))
    sees = n - m + 1 + torch.arange(m, device="cuda")
    small = torch.exp2(k[0, 0, 0])
    assert 2.0 ** -28 < small < 2.0 ** -22
    want = (sees - 1) * small * 0.9375 / (1 + (sees - 1) * small)
    bound = want * (EPS[F16] + 2 * 28 * math.log(2) * 4 * 2.0 ** -24 + 2.0 ** -18)
    assert ((out.double() - want[:, None, None]).abs() <= bound[:, None, None]).all()


class Guarded:
    """A workspace of exactly what a call asks for, and a mark behind it."""
    def __init__(self):
        self.size, self.tensor = 0, None

    def floats(self, needed, device):
        if needed > self.size:
            self.size, self.tensor = needed, torch.full((needed + 65536,), 7.0, device=device)
        return 0 if self.tensor is None else self.tensor.data_ptr(), self.size, torch.cuda.current_stream().cuda_stream

    def kept(self):
        return self.tensor is None or bool((self.tensor[self.size:] == 7).all())


@pytest.mark.parametrize("hq, h, lengths, asked, before, behind", [
    (28, 4, [3000], [64], 0, 1000),
    (8, 2, [900, 700], [100, 70], 40, 400),
    (4, 1, [2000, 0, 5], [300, 0, 5], 0, 700),
    (28, 4, [3000, 2000, 5, 700, 900], [1, 300, 0, 4, 5], 3, 2000),          # a chunk beside single and drafted tokens
    (32, 8, [300] * 39 + [511], [1] * 20 + [80] + [16, 17] * 9 + [3], 5, 4000),          # the same, one workgroup's rows
    (8, 2, [900, 700], [100, 2], 0, 900),                                    # the same, all at once
    (28, 4, [700, 30, 5, 1300], [2, 1, 2, 0], 9, 50)])                       # few columns
@pytest.mark.parametrize("dtype", [BF, F16])
def test_padded_batches(dtype, hq, h, lengths, asked, before, behind):
    """Tokens of no sequence in front of the batch and behind it, more than the sequences could have."""
    gen, B = gen_of(hq + before), 16
    pages = sum(-(-n // B) for n in lengths) + 2
    held, key, value = random_pool(gen, pages, h, B)
    tables, tokens = tables_of(gen, lengths, B, pages), sum(asked)
    q = torch.randn((before + tokens + behind, hq, 128), generator=gen).to(dtype).cuda()
    out, workspace = torch.full(q.shape, 6.0, dtype=F32, device="cuda"), Guarded()
    cu = torch.tensor([0, *asked]).cumsum(0).add(before).int().cuda()
    int4_attention(q, cu, max(asked), held, tables.cuda(), i32(lengths), max(lengths), 0.09, workspace, out)
    own = slice(before, before + tokens)
    check(out[own], q[own], asked, lengths, key, value, tables, B, 0.09, F32)
    assert (out[:before] == 6).all() and (out[before + tokens:] == 6).all() and workspace.kept()


# offsets as they stand, and what of them lies within twenty tokens
OFFSETS = [([0, 5, 40], [0, 5, 20]), ([18, 25, 31], [18, 20, 20]), ([-3, 4, 20], [4, 4, 20]), ([0, 20, -7], [0, 20, 20]),
           ([2 ** 31 - 1, -2 ** 31, 12], [20, 20, 20]), ([30, 6, 19], [6, 6, 19])]


@pytest.mark.parametrize("cu, clamped", OFFSETS)
@pytest.mark.parametrize("kind", [Int4Pages, DensePages])
def test_offsets_past_the_tensors(kind, cu, clamped):
    """Offsets that run past the tensors, or start in front of them, touch nothing outside and no page: the tensors lie
    within larger ones."""
    gen, tokens = gen_of(3), 20
    wide = torch.randn((3, 60, 4, 128), generator=gen).to(BF).cuda()
    q, k, v = wide[0, 20:40], wide[1, 20:40, :2], wide[2, 20:40, :2]
    table, start, rotation = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4), i32([3, 6]), case.angles(80, 128).cuda()

    def pages():
        if kind is Int4Pages:
            return Int4Pages(torch.full((8, 2, 16 * 144), 0x55, dtype=torch.uint8, device="cuda"))
        return DensePages(*(torch.full((8, 2, 16, 128), 9.0, dtype=BF, device="cuda") for _ in range(2)))

    def run(offsets):
        held, out = pages(), torch.full((60, 4, 128), 5.0, dtype=BF, device="cuda")
        append_rows(q, k, v, i32(offsets), tokens, held, table, start, rotation=rotation, output=out[20:40])
        rows = torch.full((2, 60, 2, 128), 4.0, dtype=BF, device="cuda")
        read_rows(held, table, i32(offsets), tokens, rows[0, 20:40], rows[1, 20:40], start)
        return out, rows, *([held.pool] if kind is Int4Pages else [held.key, held.value])

    want = run(clamped)
    for t, plain in zip(run(cu), want):
        assert torch.equal(t, plain)
    out, rows = want[:2]
    assert (out[:20] == 5).all() and (out[40:] == 5).all() and (rows[:, :20] == 4).all() and (rows[:, 40:] == 4).all()


@pytest.mark.parametrize("tokens", [1, 37])
def test_rows_side_by_side_within_a_head(tokens):
    """One projection [tokens, heads, 3 x 128], queries rotated in place, and rows read back beside each other."""
    gen = gen_of(tokens)
    fused = torch.randn((tokens, 2, 3 * 128), generator=gen).to(BF).cuda()
    apart = [x.contiguous() for x in fused.split(128, 2)]
    table, cu, rotation = torch.arange(4, dtype=torch.int32, device="cuda")[None], i32([0, tokens]), case.angles(64, 128).cuda()
    held, plain = (Int4Pages(torch.zeros((4, 2, 16 * 144), dtype=torch.uint8, device="cuda")) for _ in range(2))
    want = append_rows(*apart, cu, tokens, plain, table, rotation=rotation)
    q, k, v = fused.split(128, 2)
    assert append_rows(q, k, v, cu, tokens, held, table, rotation=rotation, output=q) is q
    assert torch.equal(q, want) and torch.equal(held.pool, plain.pool)
    assert torch.equal(k, apart[1]) and torch.equal(v, apart[2])
    both, key, value = torch.zeros((tokens, 2, 2, 128), device="cuda"), *(torch.zeros((tokens, 2, 128), device="cuda") for _ in "kv")
    read_rows(plain, table, cu, tokens, key, value)
    read_rows(held, table, cu, tokens, both[:, :, 0], both[:, :, 1])
    assert torch.equal(both[:, :, 0], key) and torch.equal(both[:, :, 1], value)


def by_token(out, q, k, v, scale, sees):
    """Every token and head against 64 bits, each with its own bound.  q and out [m, hq, 128], k and v [n, h, 128]; token t
    sees the first sees[t] rows.  A logit is off by 134 roundings of 2^-24 of its products' sizes at most (128 products and
    sums, the scale), and a weight by that twice (its sum's too), 2^-11 for its rounding to f16, 2^-20 for exponentials and
    sums; below 2^-28 of the largest a weight is off by 2^-39 of that.  The output is rounded once."""
    n, h, hq = k.shape[0], k.shape[1], q.shape[1]
    hidden = torch.arange(n, device="cuda") >= sees[:, None]
    for head in range(hq):
        x, key, value = q[:, head].double(), k[:, head // (hq // h)].double(), v[:, head // (hq // h)].double()
        slack = (x.abs() @ key.abs().t() * abs(scale) * 134 * 2.0 ** -24).masked_fill(hidden, 0).amax(1, keepdim=True)
        p = (x @ key.t() * scale).masked_fill(hidden, -math.inf).softmax(-1)
        want = p @ value
        bound = p @ value.abs() * (torch.expm1(2 * slack) + EPS[F16] + 2.0 ** -20) + n * 2.0 ** -39 * value.abs().max()
        bound = bound * (1 + EPS[out.dtype]) + want.abs() * EPS[out.dtype]
        worst = float(((out[:, head].double() - want).abs() / bound).max())
        assert worst <= 1, (head, scale, worst)


@pytest.mark.parametrize("scale, low, high", [(-0.2, -60, 4), (0.0, -60, 4), (1e-42, -60, 4), (3.0, -60, 4), (3.0, -6, -2),
                                              (2.0 ** 100, -125, -104), (-2.0 ** 126, -132, -128)])
@pytest.mark.parametrize("m", [1, 20, 70])
def test_scales_token_by_token(m, scale, low, high):
    """Queries of very different sizes side by side: a large one does not hide what becomes of the small ones."""
    gen = gen_of(m)
    pages, table, k, v = held_rows(*(torch.randn((700, 2, 128), generator=gen).to(BF).cuda() for _ in range(2)))
    size = torch.exp2(torch.randint(low, high + 1, (m, 8, 1), generator=gen).double())
    q = (torch.randn((m, 8, 128), generator=gen).double() * size).to(BF).cuda()
    for out_dtype in (BF, F32):
        out = int4_attention(q, i32([0, m]), m, pages, table, i32([700]), 700, scale, SharedDecodeWorkspace(),
                             torch.empty(q.shape, dtype=out_dtype, device="cuda"))
        by_token(out, q, k, v, scale, 700 - m + 1 + torch.arange(m, device="cuda"))


@pytest.mark.parametrize("hq, h", [(28, 4), (8, 2)])
def test_a_captured_step_of_any_batch(hq, h):
    """One graph for every batch of up to four sequences and 200 tokens: rows appended, then attended to.  What the
    batches ask for stands on the device; replays and eager calls over one workspace in turn."""
    gen, B, n, tokens, rows = gen_of(hq), 16, 4, 200, 1600
    held = Int4Pages.allocate(n * rows // B, B, h)
    table = tables_of(gen, [rows] * n, B, n * rows // B).cuda()
    rotation, workspace, stream = case.angles(rows, 128).cuda(), SharedDecodeWorkspace(), torch.cuda.Stream()
    fused = torch.zeros((tokens, hq + 2 * h, 128), dtype=BF, device="cuda")
    cu, before, after = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (n + 1, n, n))
    out = torch.zeros((tokens, hq, 128), dtype=BF, device="cuda")
    kv = torch.randn((2, n * rows, h, 128), generator=gen).to(BF).cuda()

    def step():
        q = append_rows(fused[:, :hq], fused[:, hq:hq + h], fused[:, hq + h:], cu, tokens, held, table, before, rotation=rotation)
        torch.add(before, cu[1:] - cu[:-1], out=after)
        int4_attention(q, cu, tokens, held, table, after, rows, 0.09, workspace, out)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    batches = [([200, 0, 0, 0], [1400, 0, 3, 900]), ([1, 150, 5, 1], [1500, 20, 700, 0]), ([1] * 4, [900, 1, 64, 1599]),
               ([0] * 4, [5] * 4), ([3, 2, 1, 190], [0, 511, 512, 600]), ([70, 60, 50, 20], [256, 0, 15, 1000])]

    def play(run):
        append_rows(None, kv[0], kv[1], i32([0, rows, 2 * rows, 3 * rows, 4 * rows]), rows, held, table)
        torch.cuda.synchronize()
        got = []
        for seed, (asked, starts) in enumerate(batches):
            fused.copy_(torch.randn(fused.shape, generator=gen_of(seed)).to(BF))
            cu.copy_(torch.tensor([0, *asked]).cumsum(0).int()), before.copy_(torch.tensor(starts).int()), out.fill_(6.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                run()
            torch.cuda.synchronize()
            assert (out[sum(asked):] == 6).all()
            got.append(out.clone())
        return got

    want = play(step)
    for _ in range(2):
        for a, b in zip(want, play(graph.replay)):
            assert torch.equal(a, b)
    # the last batch against 64 bits
    asked, starts = batches[-1]
    key, value = (torch.empty((n * rows, h, 128), device="cuda") for _ in range(2))
    read_rows(held, table, i32([0, rows, 2 * rows, 3 * rows, 4 * rows]), rows, key, value)
    x = torch.randn(fused.shape, generator=gen_of(len(batches) - 1)).to(BF)
    at = torch.cat([torch.arange(a, a + m) for a, m in zip(starts, asked)])
    q = case.turned(x[:, :hq], case.angles(rows, 128)[at], False).to(BF).cuda()
    check(want[-1], q, asked, [a + m for a, m in zip(starts, asked)], key.view(-1, B, h, 128), value.view(-1, B, h, 128),
          torch.arange(n * rows // B).view(n, -1), B, 0.09, BF)
