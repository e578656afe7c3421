"""4-bit pages against plain forms in 64 bits: what is written, bit by bit; what is read back; attention of one token and
of many, at the lengths, masks, pages and batches where it can go wrong."""
import pytest
import torch

import int4case as case
from densecase import EPS, i32, offsets
from inquant.triton_attention import SharedDecodeWorkspace
from inquant_vllm import DensePages, Int4Pages, append_rows, int4_attention, int4_decode, read_rows

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen_of(seed):
    return torch.Generator().manual_seed(seed)


def tables_of(gen, rows, B, pages, columns=None):
    """Block tables (on the host) of sequences at random pages, -1 behind their last."""
    need = [-(-n // B) for n in rows]
    assert sum(need) <= pages
    order, out = torch.randperm(pages, generator=gen).int(), torch.full((len(rows), columns or max(1, *need)), -1, dtype=torch.int32)
    first = 0
    for i, n in enumerate(need):
        out[i, :n] = order[first:first + n]
        first += n
    return out


def same(a, b):
    """Equal values, NaN in the same places."""
    a, b = a.double().cpu(), b.double().cpu()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


# ---------------------------------------------------------------- rows into pages

def append_case(seed, *, lengths, starts, B, heads, hq, dtype, rotary, interleaved=False, factors=False, positions=None, edit=None):
    gen = gen_of(seed)
    tokens, pages = sum(lengths), 2 * sum(-(-(a + n) // B) for a, n in zip(starts, lengths)) + 1
    fused = torch.randn((tokens + 2, hq + 2 * heads, 128), generator=gen)                # two tokens of no sequence
    fused[:, hq:hq + heads, 17:19] *= 20
    if edit:
        edit(fused[:, hq:])
    fused = fused.to(dtype)
    pos = starts if positions is None else positions
    table = case.angles(max(p + n for p, n in zip(pos, lengths)) + 1, rotary) if rotary else None
    f = torch.rand((heads, 128), generator=gen) * 3 + 0.5 if factors else None
    tables = tables_of(gen, [a + n for a, n in zip(starts, lengths)], B, pages)
    where = [(i, t, int(tables[i, (starts[i] + t) // B]), (starts[i] + t) % B) for i, n in enumerate(lengths) for t in range(n)]
    at = torch.cat([torch.arange(p, p + n) for p, n in zip(pos, lengths)]) if tokens else torch.zeros(0, dtype=torch.int64)
    q, k, v = fused[:tokens, :hq], fused[:tokens, hq:hq + heads], fused[:tokens, hq + heads:]
    qr, kr = (case.turned(x, table[at], interleaved) if rotary else x.float() for x in (q, k))
    if factors:
        qr, kr = qr * f.repeat_interleave(hq // heads, 0), kr / f
    cuda = fused.cuda()
    call = dict(query=cuda[:, :hq], key=cuda[:, hq:hq + heads], value=cuda[:, hq + heads:], cu_seqlens=offsets(lengths),
                max_seqlen=max(lengths), block_tables=tables.cuda(), start=i32(starts), interleaved=interleaved,
                rotation=None if table is None else table.cuda(), factors=None if f is None else f.cuda(),
                positions=None if positions is None else i32(positions))
    return call, dict(q=qr.to(dtype), k=kr, v=v, where=where, pages=pages, at=at, gen=gen)


CASES = [
    dict(lengths=[1, 0, 3, 4, 5, 18], starts=[0, 7, 14, 3, 29, 30], B=16, heads=2, hq=8, dtype=BF, rotary=128),
    dict(lengths=[1] * 5, starts=[15, 16, 33, 0, 63], B=32, heads=4, hq=28, dtype=BF, rotary=128, factors=True),
    dict(lengths=[70, 9], starts=[0, 61], B=64, heads=1, hq=3, dtype=F16, rotary=64, interleaved=True),
    dict(lengths=[130, 2], starts=[1, 254], B=256, heads=3, hq=3, dtype=BF, rotary=96, factors=True),
    dict(lengths=[33, 31], starts=[0, 0], B=128, heads=2, hq=32, dtype=F16, rotary=16, positions=[5, 900]),
    dict(lengths=[6, 2], starts=[2, 3], B=16, heads=2, hq=2, dtype=BF, rotary=128, interleaved=True),
    dict(lengths=[25], starts=[4], B=16, heads=2, hq=4, dtype=F16, rotary=0),
    dict(lengths=[500, 37], starts=[3, 0], B=16, heads=1, hq=7, dtype=BF, rotary=128),
    dict(lengths=[900, 37, 901], starts=[3, 0, 6], B=16, heads=1, hq=15, dtype=BF, rotary=128),     # four rows a team
    dict(lengths=[1400], starts=[7], B=64, heads=1, hq=24, dtype=F16, rotary=64, interleaved=True, factors=True),
]


@pytest.mark.parametrize("n", range(len(CASES)))
def test_append_into_4_bit_pages(n):
    c = CASES[n]
    call, want = append_case(n, **c)
    pool = torch.randint(0, 256, (want["pages"], c["heads"], c["B"] * 144), generator=want["gen"], dtype=torch.uint8)
    expected, cuda = pool.clone(), pool.cuda()
    kc, vc = case.coded(want["k"]), case.coded(want["v"].float())
    for token, (i, t, page, row) in enumerate(want["where"]):
        for h in range(c["heads"]):
            case.put(expected[page, h], row, 0, kc[0][token, h], kc[1][token, h])
            case.put(expected[page, h], row, 1, vc[0][token, h], vc[1][token, h])
    out = torch.full(call["query"].shape, 3.0, dtype=c["dtype"], device="cuda")
    assert append_rows(**call, pages=Int4Pages(cuda), output=out) is out
    assert torch.equal(cuda.cpu(), expected)                                             # no other byte was touched
    tokens = len(want["where"])
    assert torch.equal(out[:tokens].cpu(), want["q"]) and (out[tokens:] == 3).all()


@pytest.mark.parametrize("n", range(len(CASES)))
def test_append_into_exact_pages(n):
    c = CASES[n]
    call, want = append_case(n, **c)
    pages = DensePages.allocate(want["pages"], c["B"], c["heads"], c["dtype"], evictable=n % 2 == 0)
    for t in (pages.key, pages.value):
        t.fill_(7.0)
    if pages.weights is not None:
        pages.weights.fill_(5.0), pages.positions.fill_(-9)
    key, value = pages.key.cpu(), pages.value.cpu()
    side = None if pages.weights is None else (pages.weights.cpu(), pages.positions.cpu())
    for token, (i, t, page, row) in enumerate(want["where"]):
        key[page, :, row], value[page, :, row] = want["k"][token].to(c["dtype"]), want["v"][token]
        if side:
            side[0][page, :, row], side[1][page, :, row] = 0.0, int(want["at"][token])
    q = call["query"]
    back = append_rows(**call, pages=pages, output=q)                                    # in place, beside the keys
    assert back is q and torch.equal(q[:len(want["where"])].cpu(), want["q"])
    assert torch.equal(pages.key.cpu(), key) and torch.equal(pages.value.cpu(), value)
    if side:
        assert torch.equal(pages.weights.cpu(), side[0]) and torch.equal(pages.positions.cpu(), side[1])


def edge_rows(kv):
    """Keys and values [tokens, 2 heads, 128]: ties, whole spans, constants, zeros, subnormals, large ones, NaN, infinities."""
    t = kv.shape[0]
    half = torch.arange(32) * 0.5
    rows = [half - 4.0, half, -half, torch.full((32,), 3.0), torch.zeros(32), torch.full((32,), 1e-6), half * 4000, half * 1e30,
            torch.cat((torch.tensor([float("nan")]), half[1:])), torch.cat((half[:-1], torch.tensor([float("inf")]))),
            torch.cat((torch.tensor([-float("inf")]), half[1:])), half * -60000, (half - 7.5) * 2 ** -14]
    for i in range(t):
        for h in range(kv.shape[1]):
            for g in range(4):
                kv[i, h, 32 * g:32 * g + 32] = rows[(i + 3 * h + 5 * g) % len(rows)]


@pytest.mark.parametrize("dtype", [BF, F16])
def test_codes_at_their_borders(dtype):
    call, want = append_case(77, lengths=[29], starts=[2], B=16, heads=2, hq=2, dtype=dtype, rotary=0, edit=edge_rows)
    pages = Int4Pages.allocate(want["pages"], 16, 2)
    append_rows(**call, pages=pages)
    got = case.rows_of(pages.pool.cpu())
    for name, rows in zip("kv", got):
        plain = case.stands_for(*case.coded(want[name].float()))
        for token, (i, t, page, row) in enumerate(want["where"]):
            assert same(rows[page, :, row], plain[token]), (name, token)
    key, value = (torch.empty((29, 2, 128), device="cuda") for _ in range(2))
    read_rows(pages, call["block_tables"], call["cu_seqlens"], 29, key, value, call["start"])
    assert same(key, case.stands_for(*case.coded(want["k"].float()))) and same(value, case.stands_for(*case.coded(want["v"].float())))


def test_positions_past_the_table_give_nan():
    call, want = append_case(5, lengths=[4, 3], starts=[0, 0], B=16, heads=2, hq=4, dtype=BF, rotary=64)
    call["rotation"], call["positions"] = call["rotation"][:2].contiguous(), i32([-1, 1])
    pages = Int4Pages.allocate(want["pages"], 16, 2)
    out = append_rows(**call, pages=pages)
    known = torch.tensor([False, True, True, False, True, False, False])
    assert (out[:7, :, :64].isnan().cpu() == ~known[:, None, None]).all() and not out[:7, :, 64:].isnan().any()
    key, value = (torch.empty((7, 2, 128), dtype=BF, device="cuda") for _ in range(2))
    read_rows(pages, call["block_tables"], call["cu_seqlens"], 4, key, value)
    assert (key[..., :64].isnan().cpu() == ~known[:, None, None]).all() and not key[..., 64:].isnan().any()
    assert not value.isnan().any()


def test_rows_that_have_no_page_are_left_out():
    """Ids outside the pool, rows past the block table, tokens past max_seqlen."""
    for kind in (Int4Pages, DensePages):
        call, want = append_case(6, lengths=[40, 20], starts=[0, 0], B=16, heads=2, hq=4, dtype=BF, rotary=128)
        tables = call["block_tables"].clone()
        tables[0, 1], tables[1, 1] = -5, want["pages"]
        call.update(block_tables=tables[:, :2], max_seqlen=30)
        pages = Int4Pages(torch.full((want["pages"], 2, 16 * 144), 0x77, dtype=torch.uint8, device="cuda")) if kind is Int4Pages \
            else DensePages(*(torch.full((want["pages"], 2, 16, 128), 9.0, dtype=BF, device="cuda") for _ in range(2)))
        before = pages.pool.clone() if kind is Int4Pages else pages.key.clone()
        out = append_rows(**call, pages=pages)
        after = pages.pool if kind is Int4Pages else pages.key
        changed = (before != after).flatten(1).any(1).nonzero().flatten().tolist()
        assert sorted(changed) == sorted([int(tables[0, 0]), int(tables[1, 0])])
        assert torch.equal(out[:30].cpu(), want["q"][:30]) and torch.equal(out[40:60].cpu(), want["q"][40:])
        key, value = (torch.full((60, 2, 128), 4.0, dtype=BF, device="cuda") for _ in range(2))
        read_rows(pages, tables[:, :2], call["cu_seqlens"], 30, key, value)
        for x in (key, value):                   # rows of no page, and past max_seqlen, keep what they held
            assert (x[16:40] == 4).all() and (x[56:] == 4).all() and not (x[:16] == 4).all() and not (x[40:56] == 4).all()


@pytest.mark.parametrize("B, heads, dtype", [(16, 4, BF), (64, 3, F16), (256, 1, F32), (32, 8, BF)])
def test_read_rows(B, heads, dtype):
    gen, lengths, starts = gen_of(B), [1, 0, 45, 70, 6], [0, 3, 17, 0, 2]
    rows = [a + n for a, n in zip(starts, lengths)]
    pages = sum(-(-n // B) for n in rows) + 3
    pool = case.fill(torch.empty((pages, heads, B * 144), dtype=torch.uint8), *(torch.randn((pages, heads, B, 128), generator=gen) * 3
                                                                                 for _ in range(2)))
    tables, held = tables_of(gen, rows, B, pages), case.rows_of(pool)
    both = torch.full((sum(lengths) + 1, 2 * heads, 128), 8.0, dtype=dtype, device="cuda")
    key, value = both[:, :heads], both[:, heads:]
    got = read_rows(Int4Pages(pool.cuda()), tables.cuda(), offsets(lengths), 70, key, value, i32(starts))
    assert got[0] is key and got[1] is value and (both[-1] == 8).all()
    token = 0
    for i, n in enumerate(lengths):
        at = torch.arange(starts[i], starts[i] + n)
        for x, plain in zip((key, value), held):
            assert same(x[token:token + n], plain[tables[i, at // B].long(), :, at % B].to(dtype))
        token += n
    if dtype is not F32:                         # exact pages: the rows themselves
        exact = [torch.randn((pages, heads, B, 128), generator=gen).to(dtype) for _ in range(2)]
        read_rows(DensePages(*(x.cuda() for x in exact)), tables.cuda(), offsets(lengths), 70, key, value, i32(starts))
        token = 0
        for i, n in enumerate(lengths):
            at = torch.arange(starts[i], starts[i] + n)
            for x, plain in zip((key, value), exact):
                assert torch.equal(x[token:token + n].cpu(), plain[tables[i, at // B].long(), :, at % B])
            token += n


# ---------------------------------------------------------------- attention

def random_pool(gen, pages, heads, B, gain=6.0):
    """Pages of random rows, coded on the GPU by the operator that the tests above pin: their pool and the rows in f32."""
    rows = torch.randn((2, pages * B, heads, 128), generator=gen)
    rows[0, :, :, 40:42] *= gain
    rows = rows.to(BF).cuda()
    held = Int4Pages(torch.zeros((pages, heads, B * 144), dtype=torch.uint8, device="cuda"))
    append_rows(None, rows[0], rows[1], i32([0, pages * B]), pages * B, held, torch.arange(pages, dtype=torch.int32, device="cuda")[None])
    key, value = (torch.empty((pages * B, heads, 128), device="cuda") for _ in range(2))
    read_rows(held, torch.arange(pages, dtype=torch.int32, device="cuda")[None], i32([0, pages * B]), pages * B, key, value)
    return held, key.view(pages, B, heads, 128), value.view(pages, B, heads, 128)


def check(out, q, asked, lengths, key, value, tables, B, scale, out_dtype, pool_ids=True):
    """Every token and head against 64 bits.  A weight carries twice a logit's error and one rounding to f16; the output
    one rounding of its own (and one of the sum they are divided by)."""
    first, hq, h = 0, q.shape[1], key.shape[2]
    for i, (n, m) in enumerate(zip(lengths, asked)):
        at = torch.arange(n, device="cuda")
        page = tables[i, :max(1, -(-n // B))].cuda().long()
        real = (page >= 0) & (page < key.shape[0])
        rows = real[at // B] if n else torch.zeros(0, dtype=torch.bool, device="cuda")
        k, v = (x[page[at // B][rows], at[rows] % B] for x in (key, value))              # [rows, h, 128]
        upto = torch.cat((torch.zeros(1, dtype=torch.int64, device="cuda"), rows.cumsum(0)))
        sees = upto[(n - m + 1 + torch.arange(m, device="cuda")).clamp(min=0)] if m else upto[:0]
        for head in range(hq):
            want, slack = case.attend(q[first:first + m, head], k[:, head // (hq // h)], v[:, head // (hq // h)], scale, sees)
            got = out[first:first + m, head].double()
            most = float(v.abs().max()) if v.numel() else 0.0
            bound = most * (2 * EPS[F16] + EPS[out_dtype] + 4 * slack + 2.0 ** -20)
            assert ((got - want).abs() <= bound).all(), (i, n, m, head, float((got - want).abs().max()), bound)
        first += m


LENGTHS = [0, 1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 511, 512]


@pytest.mark.parametrize("hq, h, B, dtype, lengths, out_dtype", [
    (7, 1, 16, BF, LENGTHS, BF), (16, 1, 32, F16, LENGTHS, F32), (4, 4, 64, BF, [512, 200, 3], F32),
    (28, 4, 16, BF, [513, 0, 1, 3000, 777], BF), (12, 2, 256, F16, [1025, 2047, 40], F16), (1, 1, 128, BF, [5000], F32),
    (14, 2, 16, F16, [300] * 7 + [1300] * 66, F16)])
def test_decode(hq, h, B, dtype, lengths, out_dtype):
    gen = gen_of(hq + B)
    pages = sum(-(-n // B) for n in lengths) + 2
    held, key, value = random_pool(gen, pages, h, B)
    tables = tables_of(gen, lengths, B, pages)
    q = torch.randn((len(lengths), hq, 128), generator=gen).to(dtype).cuda()
    out = torch.empty(q.shape, dtype=out_dtype, device="cuda")
    workspace = SharedDecodeWorkspace()
    got = int4_decode(q, held, tables.cuda(), i32(lengths), max(lengths), 0.09, workspace, out)
    assert got is out
    check(out, q, [1] * len(lengths), lengths, key, value, tables, B, 0.09, out_dtype)
    # a looser bound of the rows, a query and an output of other strides
    wide = torch.zeros((len(lengths), hq, 256), dtype=dtype, device="cuda")
    wide[..., :128] = q
    columns = torch.cat((tables, torch.full((len(lengths), 3), -1, dtype=torch.int32)), 1).cuda()
    other = torch.empty((hq, len(lengths), 128), dtype=out_dtype, device="cuda").transpose(0, 1)
    int4_decode(wide[..., :128], held, columns, i32(lengths), columns.shape[1] * B, 0.09, workspace, other)
    check(other, q, [1] * len(lengths), lengths, key, value, tables, B, 0.09, out_dtype)


@pytest.mark.parametrize("hq, h, B, dtype, lengths, asked", [
    (7, 1, 16, BF, [40, 3, 0, 17, 64], [2, 2, 1, 0, 1]),                     # sixteen columns, one workgroup's rows
    (28, 4, 16, BF, [700, 30, 5, 1300], [2, 1, 2, 0]),                       # sixteen columns, rows shared out
    (28, 4, 32, F16, [2000, 600, 4], [4, 1, 3]),                             # 32 columns
    (28, 4, 16, BF, [1000, 513, 64], [5, 5, 5]),                             # more than one group of them
    (16, 2, 64, F16, [900, 31, 300], [31, 31, 1]),                           # eight groups, every row asked for
    (32, 8, 16, BF, [700, 130], [130, 130]),                                 # many columns, split rows
    (14, 2, 256, F16, [300, 90, 1, 0, 33], [290, 90, 1, 0, 2]),              # many, fewer rows than tiles of columns
    (16, 1, 16, BF, [1100, 20], [40, 40]),                                   # more tokens than rows
    (8, 8, 16, BF, [600], [600]),                                            # a whole prompt, one head per KV head
    (4, 2, 16, F16, [400] + [40] * 70, [1] * 71),                            # more than a launch's sequences
    (28, 4, 16, BF, [3000, 2000, 5, 700, 900], [1, 300, 0, 4, 5]),           # a chunk beside single and drafted tokens
    (32, 4, 32, F16, [500, 310, 31, 1], [100, 1, 1, 1]),
    (16, 1, 16, BF, [600 + 20 * i for i in range(69)] + [64], [1, 2] * 34 + [40, 64])])
def test_attention(hq, h, B, dtype, lengths, asked):
    gen = gen_of(hq + 3 * B)
    pages = sum(-(-n // B) for n in lengths) + 2
    held, key, value = random_pool(gen, pages, h, B)
    tables = tables_of(gen, lengths, B, pages)
    tokens = sum(asked)
    q = torch.randn((tokens + 2, hq, 128), generator=gen).to(dtype).cuda()
    for out_dtype in (dtype, F32):
        out = torch.full(q.shape, 6.0, dtype=out_dtype, device="cuda")
        int4_attention(q, offsets(asked), max(asked), held, tables.cuda(), i32(lengths), max(lengths), 128 ** -0.5,
                       SharedDecodeWorkspace(), out)
        check(out, q, asked, lengths, key, value, tables, B, 128 ** -0.5, out_dtype)
        assert (out[tokens:] == 6).all()         # tokens of no sequence
    # a lower max_seqlen leaves the rest as it was
    if max(asked) > 1:
        again = torch.full_like(out, 6.0)
        int4_attention(q, offsets(asked), 1, held, tables.cuda(), i32(lengths), max(lengths), 128 ** -0.5, SharedDecodeWorkspace(), again)
        first = torch.tensor([sum(asked[:i]) for i in range(len(asked)) if asked[i]])
        assert (again[first] - out[first]).abs().max() <= 4 * EPS[F16] * value.abs().max()
        rest = torch.ones(q.shape[0], dtype=torch.bool)
        rest[first] = False
        assert (again[rest.cuda()] == 6).all()


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-42, 3.0])
@pytest.mark.parametrize("m", [1, 20, 70])
def test_scales(scale, m):
    gen = gen_of(9)
    held, key, value = random_pool(gen, 50, 2, 16)
    tables = tables_of(gen, [700], 16, 50)
    q = (torch.randn((m, 8, 128), generator=gen) * torch.exp2(torch.randint(-60, 5, (m, 8, 1), generator=gen).float())).to(BF).cuda()
    out = int4_attention(q, i32([0, m]), m, held, tables.cuda(), i32([700]), 700, scale, SharedDecodeWorkspace())
    check(out, q, [m], [700], key, value, tables, 16, scale, BF)


@pytest.mark.parametrize("m", [1, 3, 20, 80])
def test_pages_of_no_pool(m):
    """Ids outside the pool: their rows count as not there, whatever page 0 holds."""
    gen = gen_of(11)
    held, key, value = random_pool(gen, 60, 2, 16)
    tables = tables_of(gen, [700, 90], 16, 59) + 1                           # page 0 is nobody's
    tables[0, 3], tables[0, 20], tables[1, 0], tables[1, 5] = -1, 60, 1 << 30, -7
    held.pool[0] = 0xff                                                      # every word a NaN
    q = torch.randn((2 * m, 8, 128), generator=gen).to(BF).cuda()
    out = int4_attention(q, i32([0, m, 2 * m]), m, held, tables.cuda(), i32([700, 90]), 700, 0.1, SharedDecodeWorkspace())
    check(out, q, [m, m], [700, 90], key, value, tables, 16, 0.1, BF)


@pytest.mark.parametrize("m, n", [(1, 90), (1, 700), (4, 700), (20, 700), (90, 700), (90, 90)])
def test_rows_behind_the_length_hold_nan(m, n):
    gen = gen_of(12)
    held, key, value = random_pool(gen, 60, 2, 16)
    tables = tables_of(gen, [n], 16, 60)
    last = int(tables[0, n // 16])
    part = held.pool[last].view(2, -1)
    B, row = 16, n % 16
    part[:, 128 * B + 8 * row:136 * B] = 0xff
    words = part[:, 136 * B:].view(2, 4, 4, 4, 2)
    for r in range(row, 16):
        words[:, r // 4, :, r % 4] = 0xff
    q = torch.randn((m, 8, 128), generator=gen).to(BF).cuda()
    out = int4_attention(q, i32([0, m]), m, held, tables.cuda(), i32([n]), n, 0.1, SharedDecodeWorkspace())
    check(out, q, [m], [n], key, value, tables, 16, 0.1, BF)


@pytest.mark.parametrize("m, n, where", [(4, 300, 297), (4, 600, 599), (20, 700, 690), (90, 700, 650), (90, 700, 30), (64, 64, 5)])
def test_a_nan_reaches_those_that_see_it(m, n, where):
    """A NaN value row: its group of channels, for the tokens from its own on, and nothing else."""
    gen = gen_of(13)
    held, key, value = random_pool(gen, 60, 2, 16)
    tables = tables_of(gen, [n], 16, 60)
    page, r = int(tables[0, where // 16]), where % 16
    held.pool[page].view(2, -1)[1, 136 * 16:].view(4, 4, 4, 2)[r // 4, 2, r % 4] = torch.tensor([0, 0x7e], dtype=torch.uint8)
    q = torch.randn((m, 8, 128), generator=gen).to(F16).cuda()
    out = int4_attention(q, i32([0, m]), m, held, tables.cuda(), i32([n]), n, 0.1, SharedDecodeWorkspace())
    hit = torch.zeros(out.shape, dtype=torch.bool)
    hit[max(0, where - (n - m)):, 4:, 64:96] = True
    assert torch.equal(out.isnan().cpu(), hit)
    fine = out.masked_fill(hit.cuda(), 0)
    first = int4_attention(q, i32([0, m]), m, random_pool(gen_of(13), 60, 2, 16)[0], tables.cuda(), i32([n]), n, 0.1, SharedDecodeWorkspace())
    assert torch.equal(fine, first.masked_fill(hit.cuda(), 0))


def test_far_pages():
    """Pages past 2^32 bytes of a pool."""
    B, heads, pages = 256, 8, 14700                                          # 4.3 GB
    pool = torch.empty((pages, heads, B * 144), dtype=torch.uint8, device="cuda")
    assert pool.numel() > 1 << 32
    held, gen, n = Int4Pages(pool), gen_of(14), 600
    tables = torch.tensor([[pages - 1, 1, pages - 2]], dtype=torch.int32)
    kv = torch.randn((2, n, heads, 128), generator=gen).to(BF).cuda()
    append_rows(None, kv[0], kv[1], i32([0, n]), n, held, tables.cuda())
    key, value = (torch.empty((n, heads, 128), device="cuda") for _ in range(2))
    read_rows(held, tables.cuda(), i32([0, n]), n, key, value)
    for x, plain in zip((key, value), kv.cpu()):
        assert same(x, case.stands_for(*case.coded(plain.float())))
    view = torch.zeros((2, 3, B, heads, 128), device="cuda")
    view[0].view(-1, heads, 128)[:n], view[1].view(-1, heads, 128)[:n] = key, value
    for m in (1, 90):
        q = torch.randn((m, 16, 128), generator=gen).to(BF).cuda()
        out = int4_attention(q, i32([0, m]), m, held, tables.cuda(), i32([n]), n, 0.1, SharedDecodeWorkspace())
        check(out, q, [m], [n], view[0], view[1], torch.tensor([[0, 1, 2]]), B, 0.1, BF)


def test_strided_pool_and_other_streams():
    """Some heads of a wider pool, on a side stream with a workspace of its own."""
    gen, B = gen_of(15), 16
    wide = torch.full((40, 5, B * 144), 0x11, dtype=torch.uint8, device="cuda")
    held = Int4Pages(wide[:, 1:3])
    tables, stream = tables_of(gen, [530], B, 40), torch.cuda.Stream()
    kv = torch.randn((2, 530, 2, 128), generator=gen).to(F16).cuda()
    q = torch.randn((3, 8, 128), generator=gen).to(F16).cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        append_rows(None, kv[0], kv[1], i32([0, 530]), 530, held, tables.cuda())
        key, value = (torch.empty((530, 2, 128), device="cuda") for _ in range(2))
        read_rows(held, tables.cuda(), i32([0, 530]), 530, key, value)
        out = int4_attention(q, i32([0, 3]), 3, held, tables.cuda(), i32([530]), 530, 0.1, SharedDecodeWorkspace())
    stream.synchronize()
    assert (wide[:, [0, 3, 4]] == 0x11).all()
    assert same(key, case.stands_for(*case.coded(kv[0].float().cpu())))
    padded = torch.zeros((2, 34 * B, 2, 128), device="cuda")
    padded[0, :530], padded[1, :530] = key, value
    check(out, q, [3], [530], *padded.view(2, 34, B, 2, 128), torch.arange(34)[None], B, 0.1, F16)


@pytest.mark.parametrize("m", [1, 20, 90])
def test_no_rows_at_all(m):
    """max_tokens of 0 with empty block tables, and lengths that are all 0 or below."""
    held = Int4Pages(torch.full((3, 2, 16 * 144), 0xff, dtype=torch.uint8, device="cuda"))
    q = torch.ones((2 * m, 8, 128), dtype=BF, device="cuda")
    empty = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
    wide = torch.zeros((2, 70), dtype=torch.int32, device="cuda")
    for tables, lengths, most in ((empty, [0, 0], 0), (empty, [5, 9], 0), (wide, [0, -3], 1000), (wide, [0, 0], 300)):
        out = int4_attention(q, i32([0, m, 2 * m]), m, held, tables, i32(lengths), most, 0.1, SharedDecodeWorkspace())
        assert (out == 0).all()


def test_two_streams_at_once():
    """The operators on two streams at the same time, a workspace each, over the same pages."""
    gen = gen_of(20)
    held, _, _ = random_pool(gen, 700, 2, 16)
    tables, rows = tables_of(gen, [6000, 4000], 16, 700).cuda(), i32([6000, 4000])
    work = []
    for m in (1, 5, 80):
        q = torch.randn((2 * m, 8, 128), generator=gen).to(BF).cuda()
        args = (q, i32([0, m, 2 * m]), m, held, tables, rows, 6000, 0.1)
        work.append((args, int4_attention(*args, SharedDecodeWorkspace())))
    torch.cuda.synchronize()
    streams = [(torch.cuda.Stream(), SharedDecodeWorkspace(), []) for _ in range(2)]
    for _ in range(5):
        for args, _ in work:
            for stream, workspace, got in streams:
                with torch.cuda.stream(stream):
                    got.append(int4_attention(*args, workspace))
    torch.cuda.synchronize()
    for _, _, got in streams:
        for i, out in enumerate(got):
            assert torch.equal(out, work[i % 3][1])


def test_captured_steps_share_a_workspace():
    """A decode step and a draft step as two graphs over one workspace, replayed in turn with eager calls between."""
    gen, B, n = gen_of(16), 16, 5
    lengths, stream = [900, 64, 1, 333, 1500], torch.cuda.Stream()
    pages = sum(-(-(x + 60) // B) for x in lengths) + 2
    held, _, _ = random_pool(gen, pages, 2, B)
    tables = tables_of(gen, [x + 60 for x in lengths], B, pages).cuda()
    rotation = case.angles(2000, 128).cuda()
    workspace, one, many = SharedDecodeWorkspace(), offsets([1] * n), offsets([4] * n)
    bufs = {m: torch.zeros((n * m, 12, 128), dtype=BF, device="cuda") for m in (1, 4)}   # 8 query heads, 2 key, 2 value
    outs = {m: torch.zeros((n * m, 8, 128), dtype=BF, device="cuda") for m in (1, 4)}
    held_rows = i32(lengths)

    def step(m, cu):
        x = bufs[m]
        q = append_rows(x[:, :8], x[:, 8:10], x[:, 10:], cu, m, held, tables, held_rows, rotation=rotation)
        held_rows.add_(m)
        if m == 1:
            return int4_decode(q, held, tables, held_rows, tables.shape[1] * B, 0.09, workspace, outs[1])
        return int4_attention(q, cu, m, held, tables, held_rows, tables.shape[1] * B, 0.09, workspace, outs[4])

    start, pool = held_rows.clone(), held.pool.clone()
    with torch.cuda.stream(stream):
        for m, cu in ((1, one), (4, many)):
            step(m, cu)
    stream.synchronize()
    graphs = {}
    for m, cu in ((1, one), (4, many)):
        graphs[m] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[m], stream=stream):
            step(m, cu)
    torch.cuda.synchronize()
    feed = [(m, torch.randn(bufs[m].shape, generator=gen).to(BF).cuda()) for m in (1, 4, 1, 1, 4, 4, 1)]

    def play(run):
        held_rows.copy_(start), held.pool.copy_(pool)
        torch.cuda.synchronize()
        got = []
        for m, x in feed:
            with torch.cuda.stream(stream):
                bufs[m].copy_(x)
                run(m)
                got.append(outs[m].clone())
            torch.cuda.synchronize()
        return got

    want = play(lambda m: step(m, one if m == 1 else many))
    for _ in range(2):
        for a, b in zip(want, play(lambda m: graphs[m].replay())):
            assert torch.equal(a, b)


def test_a_prompt_in_chunks_then_tokens():
    """The operators as they are used: a prompt appended and attended to in chunks, then drafted and single tokens; every
    output against 64 bits over the rows that the pages stand for."""
    gen, B, hq, h, total = gen_of(17), 16, 14, 2, 777
    held = Int4Pages.allocate(60, B, h)
    tables = tables_of(gen, [total], B, 60)
    x = torch.randn((total, hq + 2 * h, 128), generator=gen).to(BF).cuda()
    rotation, workspace = case.angles(total, 128).cuda(), SharedDecodeWorkspace()
    outs, rotated, at = [], [], 0
    for m in (300, 200, 128, 64, 40, 20, 9, 5, 4, 3, 1, 1, 2):
        part = x[at:at + m]
        cu, start = i32([0, m]), i32([at])
        q = append_rows(part[:, :hq], part[:, hq:hq + h], part[:, hq + h:], cu, m, held, tables.cuda(), start, rotation=rotation)
        at += m
        rows = i32([at])
        outs.append(int4_attention(q, cu, m, held, tables.cuda(), rows, at, 0.09, workspace) if m > 1 else
                    int4_decode(q, held, tables.cuda(), rows, at, 0.09, workspace))
        rotated.append(q)
    assert at == total
    key, value = (torch.zeros((-(-total // B) * B, h, 128), device="cuda") for _ in range(2))
    read_rows(held, tables.cuda(), i32([0, total]), total, key, value)
    turned = case.turned(x[:, hq:hq + h].cpu(), case.angles(total, 128), False)
    assert same(key[:total], case.stands_for(*case.coded(turned)))
    check(torch.cat(outs), torch.cat(rotated), [total], [total], key.view(-1, B, h, 128), value.view(-1, B, h, 128),
          torch.arange(-(-total // B))[None], B, 0.09, BF)


def test_outputs_in_place_and_apart():
    gen = gen_of(19)
    held, _, _ = random_pool(gen, 120, 2, 16)
    tables, workspace = tables_of(gen, [900, 700], 16, 120).cuda(), SharedDecodeWorkspace()
    for m, lengths in ((1, [900, 700]), (1, [200, 500]), (5, [900, 30]), (60, [900, 700])):
        rows = i32(lengths)
        q = torch.randn((2 * m + 4, 8, 128), generator=gen).to(BF).cuda()
        args = (i32([0, m, 2 * m]), m, held, tables, rows, max(lengths), 0.1, workspace)
        want = int4_attention(q[:2 * m], *args)
        with pytest.raises(ValueError, match="apart from it"):
            int4_attention(q[:2 * m], *args, q[1:2 * m + 1])
        own = q[:2 * m]
        assert int4_attention(own, *args, own) is own and torch.equal(own, want)
    with pytest.raises(ValueError, match="finite"):
        int4_decode(q[:2], held, tables, rows, 900, 1e39, workspace)


def test_outputs_repeat():
    """The same call twice gives the same bits: nothing depends on an order that is not fixed."""
    gen = gen_of(18)
    held, _, _ = random_pool(gen, 300, 2, 16)
    tables, lengths = tables_of(gen, [3000, 900], 16, 300).cuda(), i32([3000, 900])
    for m in (1, 6, 80):
        q = torch.randn((2 * m, 8, 128), generator=gen).to(BF).cuda()
        one, two = (int4_attention(q, i32([0, m, 2 * m]), m, held, tables, lengths, 3000, 0.1, SharedDecodeWorkspace()) for _ in range(2))
        assert torch.equal(one, two)
