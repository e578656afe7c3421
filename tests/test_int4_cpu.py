"""4-bit pages on the host: what the operators refuse, and the plain codes that the GPU tests compare with."""
import ctypes

import pytest
import torch

import int4case as case
from inquant import _native as nat
from inquant_vllm import DensePages, Int4Pages, append_rows, int4_attention, int4_decode, read_rows

I32 = torch.int32


def _pages(block=16, heads=2):
    return Int4Pages.allocate(4, block, heads, device="cpu")


def _rows(tokens=3, heads=2, dtype=torch.bfloat16):
    return torch.zeros((tokens, heads, 128), dtype=dtype)


def test_pages_are_checked():
    pool = torch.zeros((4, 2, 16 * 144), dtype=torch.uint8)
    pages = Int4Pages(pool)
    assert (pages.block_size, pages.heads, pages.nbytes) == (16, 2, pool.numel())
    Int4Pages(torch.zeros((4, 3, 32 * 144), dtype=torch.uint8)[:, :2])                   # some heads of a pool
    for bad in (pool[0], pool.char(), pool[..., :-144], pool[:0], pool[:, :0], pool[:1].expand(4, -1, -1),
                torch.zeros((4, 2, 16 * 144 + 8), dtype=torch.uint8)[..., 8:],           # heads off 16 bytes
                torch.zeros(4 * 2 * 16 * 144 + 1, dtype=torch.uint8)[1:].view(4, 2, -1),
                torch.zeros((4, 16 * 144, 2), dtype=torch.uint8).transpose(1, 2)):
        with pytest.raises(ValueError):
            Int4Pages(bad)
    with pytest.raises(Exception):
        pages.pool = pool                                                                # fixed once made


def test_copies_describe_their_own_memory():
    import copy
    import pickle
    pages = _pages()
    for other in (copy.deepcopy(pages), pickle.loads(pickle.dumps(pages))):
        assert other._pages.pool == other.pool.data_ptr() != pages.pool.data_ptr()


def _good():
    k, cu, table = _rows(), torch.tensor([0, 3], dtype=I32), torch.zeros((1, 2), dtype=I32)
    return dict(query=_rows(3, 4), key=k, value=k.clone(), cu_seqlens=cu, max_seqlen=3, pages=_pages(), block_tables=table)


def test_cpu_tensors_are_refused():
    good = _good()
    k, cu, table = good["key"], good["cu_seqlens"], good["block_tables"]
    for pages in (good["pages"], DensePages.allocate(4, 16, 2, device="cpu")):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            append_rows(**{**good, "pages": pages})
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            read_rows(pages, table, cu, 3, k, k.clone())
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        int4_decode(_rows(1, 4), good["pages"], table, cu[1:], 3, 0.1, None)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        int4_attention(_rows(3, 4), cu, 3, good["pages"], table, cu[1:], 3, 0.1, None)


def _refused(fn, good, changes):
    for change in changes:
        with pytest.raises(ValueError):
            fn(**{**good, **change})


def test_append_rows_refusals(monkeypatch):
    import inquant_vllm.int4 as int4
    monkeypatch.setattr(int4, "_on_gpu", lambda *a: None)                                # what is checked behind it too
    monkeypatch.setattr(int4, "_call", lambda *a: None)
    good = _good()
    append_rows(**good)
    fused = torch.zeros((3, 8, 128), dtype=torch.bfloat16)
    q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
    assert append_rows(**{**good, "query": q, "key": k, "value": v, "output": q}) is q   # in place, beside the keys
    assert append_rows(**{**good, "query": None}) is None
    one = torch.zeros((1, 8, 128), dtype=torch.bfloat16)
    assert append_rows(**{**good, "query": one[:, :4], "key": one[:, 4:6], "value": one[:, 6:], "output": one[:, :4]}) is not None
    cu, rot = good["cu_seqlens"], torch.zeros((8, 64))
    _refused(append_rows, good, [
        dict(key=_rows(3, 3)), dict(key=good["key"][..., :64]), dict(value=_rows(4)), dict(key=good["key"].half()),
        dict(value=good["key"].half()), dict(key=good["key"].float(), value=good["key"].float()),
        dict(key=torch.zeros((3, 2, 129), dtype=torch.bfloat16)[..., 1:]), dict(query=_rows(4, 4)), dict(query=_rows(3, 3)),
        dict(query=_rows(3, 4).half()), dict(query=_rows(3, 0)), dict(pages=good["key"]), dict(max_seqlen=-1),
        dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[:1]), dict(block_tables=good["block_tables"].long()),
        dict(block_tables=torch.zeros((2, 2), dtype=I32)), dict(start=cu), dict(start=cu[:1].long()), dict(positions=cu),
        dict(rotation=rot.double()), dict(rotation=rot[:, ::2]), dict(rotation=rot[0]), dict(rotation=rot[:0]),
        dict(rotation=torch.zeros((8, 24))), dict(rotation=torch.zeros((8, 144))), dict(rotation=torch.zeros((8, 0))),
        dict(factors=torch.ones((4, 128))), dict(factors=torch.ones((2, 128)).double()),
        dict(output=_rows(3, 3)), dict(output=_rows(3, 4).half()), dict(output=_rows(3, 1).expand(3, 4, 128)),
        dict(output=_rows(1, 4).expand(3, 4, 128)), dict(query=None, output=_rows(3, 4)),
        dict(query=q, key=k, value=v, output=fused[:, 1:5]), dict(query=q, key=k, value=v, output=fused[:, 2:6]),
        dict(query=q, key=k, value=q[:, :2], output=q)])
    dense = DensePages.allocate(4, 16, 2, device="cpu")
    _refused(append_rows, {**good, "pages": dense}, [dict(key=good["key"].half(), value=good["key"].half(), query=None)])


def test_read_rows_refusals(monkeypatch):
    import inquant_vllm.int4 as int4
    monkeypatch.setattr(int4, "_on_gpu", lambda *a: None)
    monkeypatch.setattr(int4, "_call", lambda *a: None)
    k, cu, table = _rows(), torch.tensor([0, 3], dtype=I32), torch.zeros((1, 2), dtype=I32)
    good = dict(pages=_pages(), block_tables=table, cu_seqlens=cu, max_seqlen=3, key=k, value=k.clone())
    read_rows(**good)
    both = torch.zeros((3, 4, 128))
    read_rows(**{**good, "key": both[:, :2], "value": both[:, 2:]})                      # float32, side by side
    _refused(read_rows, good, [
        dict(value=k), dict(key=_rows(3, 3)), dict(value=_rows(4)), dict(key=k.double(), value=k.double()), dict(value=k.half()),
        dict(key=_rows(3, 1).expand(3, 2, 128)), dict(key=both[:, :2], value=both[:, 1:3]), dict(max_seqlen=-1),
        dict(start=cu), dict(cu_seqlens=cu.long()), dict(block_tables=table.long()), dict(pages=k)])
    dense = DensePages.allocate(4, 16, 2, device="cpu")
    _refused(read_rows, {**good, "pages": dense}, [dict(key=k.half(), value=k.half()), dict(key=both[:, :2], value=both[:, 2:])])


def test_attention_refusals():
    cu, table = torch.tensor([0, 3], dtype=I32), torch.zeros((1, 2), dtype=I32)
    good = dict(query=_rows(3, 4), cu_seqlens=cu, max_seqlen=3, pages=_pages(), block_tables=table, lengths=cu[1:], max_tokens=3,
                scale=0.1, workspace=None)
    _refused(int4_attention, good, [
        dict(query=_rows(3, 3)), dict(query=_rows(3, 34)), dict(query=_rows(3, 4).float()), dict(query=_rows(3, 4)[..., :64]),
        dict(query=_rows(3, 4)[0]), dict(pages=DensePages.allocate(4, 16, 2, device="cpu")), dict(max_tokens=33),
        dict(max_tokens=-1), dict(max_seqlen=-1), dict(lengths=cu), dict(lengths=cu[1:].long()), dict(cu_seqlens=cu.long()),
        dict(block_tables=table.long()), dict(scale=float("inf")), dict(scale=float("nan"))])
    decode = {k: v for k, v in good.items() if k not in ("cu_seqlens", "max_seqlen")} | dict(query=_rows(1, 4))
    _refused(int4_decode, decode, [dict(query=_rows(2, 4)), dict(query=_rows(1, 3)), dict(max_tokens=33), dict(scale=float("nan"))])


def test_entry_points_refuse_on_the_host():
    lib, fake = nat.lib(), 1 << 20
    pages = lambda **more: ctypes.addressof(keep.setdefault(tuple(more.items()), nat.Int4PagesDesc(
        **{**dict(pool=fake, s_page=2 * 2304, s_head=2304, pages=4, heads=2, block_tokens=16), **more})))
    keep = {}

    def attention(q=fake, dtype=nat.IQ_BF16, hq=4, cu=fake, n=1, tokens=3, most=3, p=None, cols=2, lengths=fake, rows=3,
                  ws=0, out=fake, odt=nat.IQ_BF16):
        return lib.iq_int4_attention(q, dtype, 512, 128, hq, cu, n, tokens, most, p or pages(), fake, cols, cols, lengths, rows,
                                     0.1, ws or None, 0, out, 512, 128, odt, None)

    bad = [dict(q=None), dict(q=fake + 8), dict(dtype=nat.IQ_F32), dict(hq=3), dict(hq=34), dict(hq=0), dict(lengths=None),
           dict(out=None), dict(odt=7), dict(rows=33), dict(rows=-1), dict(tokens=-1), dict(most=-1), dict(cu=None),
           dict(n=-1), dict(n=65536), dict(p=pages(pool=fake + 8)), dict(p=pages(s_head=2300)), dict(p=pages(block_tokens=48)),
           dict(p=pages(heads=0)), dict(p=pages(pages=0)), dict(rows=1000, cols=64)]     # the last: no workspace
    for change in bad:
        assert attention(**change) == -1 and b"iq_int4_attention" in lib.iq_last_error(), change
    # nothing to do: no launch either
    assert attention(n=0) == 0 and attention(tokens=0) == 0 and attention(most=0) == 0

    def append(k=fake, q=fake, hq=4, dense=None, p=-1, dtype=nat.IQ_BF16, st=256, rotation=None, angles=0, rotary=0, factors=None,
               most=3, out=fake, n=1):
        return lib.iq_append_rows(q, k, fake, dtype, 512, 128, st, 128, 256, 128, hq, fake, n, most, None, None, rotation, angles,
                                  rotary, 0, factors, dense, pages() if p == -1 else p, fake, 2, 2, out, 512, 128, None)

    for change in [dict(k=None), dict(k=fake + 8), dict(st=252), dict(hq=3), dict(out=None), dict(p=None), dict(dtype=nat.IQ_F32),
                   dict(dense=pages()), dict(rotary=64), dict(rotation=fake), dict(rotation=fake, angles=8, rotary=24),
                   dict(rotation=fake, angles=8, rotary=144), dict(rotation=fake + 4, angles=8, rotary=64),
                   dict(rotation=fake, angles=0, rotary=64), dict(factors=fake + 4), dict(most=-1), dict(most=1 << 31)]:
        assert append(**change) == -1 and b"iq_append_rows" in lib.iq_last_error(), change
    assert append(n=0) == 0 and append(most=0) == 0

    def read(k=fake, p=-1, dtype=nat.IQ_BF16, st=256, most=3):
        return lib.iq_read_rows(None, pages() if p == -1 else p, dtype, fake, 2, 2, fake, 1, most, None, k, st, 128, fake, 256, 128, None)

    for change in [dict(k=None), dict(k=fake + 8), dict(p=None), dict(dtype=nat.IQ_F64), dict(st=252), dict(most=-1)]:
        assert read(**change) == -1 and b"iq_read_rows" in lib.iq_last_error(), change
    assert read(most=0) == 0
    for name in ("iq_append_rows_from", "iq_read_rows_from", "iq_int4_attention_from"):
        assert getattr(lib, name)(None) == -1 and b"null arguments" in lib.iq_last_error()


def test_workspace_is_bounded():
    """Scratch for few columns goes with the workgroups, not with the rows; for many with the tokens and a few partitions."""
    floats = nat.lib().iq_int4_workspace_floats
    assert floats(28, 4, 16, 16, 1, 512) == 0                                            # one workgroup's rows: no join
    decode = [floats(28, 4, 16, 16, 1, n) for n in (513, 4096, 32768, 1 << 20)]
    assert 0 < max(decode) <= 4 * (128 + 16) * 16 * 130 * 2 and decode == sorted(decode)
    assert floats(28, 4, 0, 0, 1, 4096) == floats(28, 4, 3, 3, 0, 4096) == floats(28, 4, 3, 0, 5, 4096) == 0
    # a chunk beside 63 single tokens: 4 heads' two groups of 32 columns (64 are the most that a sequence beside a
    # chunk may have), 512 / 4 workgroups and 64 sequences each
    assert floats(32, 4, 64, 2048 + 63, 2048, 1 << 17) <= 4 * 2 * (128 + 64) * 32 * 130
    assert floats(28, 4, 1, 2048, 2048, 32768) == 0                                      # enough workgroups without
    assert 0 < floats(28, 4, 1, 64, 64, 32768) <= 64 * 28 * 64 * 130


def test_codes_are_within_half_a_step():
    """The plain codes' own properties: off by half a step at most within 15 * 2048, 0 kept, f16 exact."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn((400, 128), generator=gen) * torch.exp2(torch.randint(-16, 14, (400, 1), generator=gen).float())
    x[0], x[1] = 0.0, 5.0
    x[2, :32], x[3, 32:64] = -3.0, 1e-9
    code, word = case.coded(x)
    value = case.stands_for(code, word)
    step = (word & 0xffe0).short().view(torch.float16).double().repeat_interleave(32, -1)
    inside = x.unflatten(-1, (4, 32)).abs().amax(-1).repeat_interleave(32, -1) <= 15 * case.MOST / 2
    assert ((value - x.double()).abs() <= step / 2)[inside].all()
    assert (value[0] == 0).all() and torch.equal(value, value.half().double())
    # the step is the least of six bits that 15 of them span the range with
    group = x.double().unflatten(-1, (4, 32))
    span = group.amax(-1).clamp(min=0) - group.amin(-1).clamp(max=0)
    s = (word & 0xffe0).short().view(torch.float16).double()
    below = torch.nextafter(s.float(), torch.zeros_like(s.float()))                      # one f32 step down, then to six bits
    below = (below.view(torch.int32) & ~0x3ffff).view(torch.float32).double()
    assert ((15 * s >= span) | (s == case.MOST)).all() and ((15 * below < span) | (s == case.LEAST)).all()


def test_bytes_go_where_they_are_read():
    gen = torch.Generator().manual_seed(2)
    for B in (16, 32):
        rows = [torch.randn((2, 1, B, 128), generator=gen) for _ in range(2)]
        pool = case.fill(torch.full((2, 1, B * 144), 0x5a, dtype=torch.uint8), *rows)
        one = torch.full((B * 144,), 0x33, dtype=torch.uint8)
        for which in range(2):
            for r in range(B):
                code, word = case.coded(rows[which][1, 0, r])
                case.put(one, r, which, code, word)
        assert torch.equal(one, pool[1, 0])
        for got, want in zip(case.rows_of(pool), rows):
            assert torch.equal(got, case.stands_for(*case.coded(want)))
