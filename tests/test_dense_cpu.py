"""What the exact-page operators refuse, checked on the host."""
import pytest
import torch

from inquant_vllm import (DensePages, dense_decode, evict_rows, prefill_attention, prefill_weights, select_rows,
                          write_rows)

I32 = torch.int32


def _pages(**more):
    return DensePages.allocate(4, 16, 2, device="cpu", **more)


def _rows(tokens=3, heads=2, dtype=torch.bfloat16):
    return torch.zeros((tokens, heads, 128), dtype=dtype)


def test_pages_are_checked():
    key = torch.zeros((4, 2, 16, 128), dtype=torch.bfloat16)
    w, p = torch.zeros((4, 2, 16)), torch.zeros((4, 2, 16), dtype=I32)
    assert DensePages(key, key.clone(), w, p).nbytes == 2 * key.numel() * 2 + 2 * w.numel() * 4
    bad = [
        (key[..., :64], key[..., :64]), (key, key[:3]), (key[:, :, :12], key[:, :, :12]), (key[0], key[0]),
        (key.float(), key.float()), (key, key.half()),
        (key, key[:1].expand(4, -1, -1, -1)),                                  # pages that are one page
        (torch.zeros((4, 2, 16, 129), dtype=torch.bfloat16)[..., 1:], key),     # rows off 16 bytes
        (key, key, w, None), (key, key, None, p), (key, key, w.double(), p), (key, key, w, p.long()),
        (key, key, torch.zeros(4 * 2 * 16 + 1)[1:].view(4, 2, 16), p),         # weights off 16 bytes
        (key, key, w[:3], p), (key, key, w.transpose(0, 1).contiguous().transpose(0, 1), p),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            DensePages(*args)
    with pytest.raises(Exception):
        DensePages(key, key).key = w                                           # fixed once made


def test_cpu_tensors_are_refused():
    pages, k, cu = _pages(), _rows(), torch.tensor([0, 3], dtype=I32)
    table, n = torch.zeros((1, 2), dtype=I32), torch.tensor([3], dtype=I32)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        write_rows(k, k, cu, 3, pages, table)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        select_rows(torch.zeros((2, 3)), cu, 3, 2)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        evict_rows(pages, table, n, n, 3, 2)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        dense_decode(_rows(1, 4), pages, table, n, 3, 0.1, None)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        prefill_weights(_rows(3, 4), k, cu, 3, 0.1, window=2)


def _refused(fn, good, changes):
    for change in changes:
        with pytest.raises(ValueError):
            fn(**{**good, **change})


def test_write_rows_refusals():
    k, cu, table = _rows(), torch.tensor([0, 3], dtype=I32), torch.zeros((1, 2), dtype=I32)
    good = dict(key=k, value=k, cu_seqlens=cu, max_seqlen=3, pages=_pages(), block_tables=table)
    _refused(write_rows, good, [
        dict(key=_rows(3, 3)), dict(key=k[..., :64]), dict(value=_rows(4)), dict(key=k.half()), dict(value=k.half()),
        dict(key=torch.zeros((3, 2, 129), dtype=torch.bfloat16)[..., 1:]), dict(cu_seqlens=cu.long()),
        dict(cu_seqlens=cu[:1]), dict(block_tables=table.long()), dict(block_tables=table[0]),
        dict(block_tables=torch.zeros((2, 2), dtype=I32)), dict(start=cu), dict(start=cu[:1].long()),
        dict(positions=cu), dict(weights=torch.zeros((2, 4))), dict(weights=torch.zeros((2, 3)).double()),
        dict(keep=torch.zeros((1, 3, 5), dtype=I32)), dict(keep=torch.zeros((1, 2, 5))),
        dict(keep=torch.zeros((1, 2), dtype=I32))])


def test_select_rows_refusals():
    w, cu = torch.zeros((2, 3)), torch.tensor([0, 3], dtype=I32)
    _refused(select_rows, dict(weights=w, cu_seqlens=cu, max_seqlen=3, budget=2), [
        dict(budget=0), dict(sink=-1), dict(recent=-1), dict(sink=2, recent=1), dict(weights=w.double()),
        dict(weights=w[0]), dict(weights=torch.zeros((3, 2)).t()), dict(cu_seqlens=cu.long())])


def test_evict_rows_refusals():
    table, n = torch.zeros((1, 2), dtype=I32), torch.tensor([20], dtype=I32)
    _refused(evict_rows, dict(pages=_pages(), block_tables=table, lengths=n, seen=n, max_tokens=20, budget=8), [
        dict(pages=_pages(evictable=False)), dict(budget=0), dict(sink=4, recent=5), dict(max_tokens=33),
        dict(max_tokens=-1), dict(lengths=n.long()), dict(seen=n.long()), dict(seen=torch.zeros(2, dtype=I32)),
        dict(lengths=n[0]), dict(block_tables=torch.zeros((2, 2), dtype=I32))])


def test_dense_decode_refusals():
    table, n = torch.zeros((1, 2), dtype=I32), torch.tensor([20], dtype=I32)
    good = dict(query=_rows(1, 4), pages=_pages(), block_tables=table, lengths=n, max_tokens=20, scale=0.1,
                workspace=None)
    _refused(dense_decode, good, [
        dict(query=_rows(1, 3)), dict(query=_rows(1, 34)), dict(query=_rows(1, 4).half()), dict(query=_rows(2, 4)),
        dict(query=_rows(1, 4)[..., :64]), dict(query=_rows(1, 4)[0]), dict(max_tokens=33), dict(max_tokens=-1),
        dict(lengths=n.long()), dict(scale=float("nan")), dict(scale=float("inf")), dict(query=_rows(1, 0)),
        dict(pages=_pages(evictable=False), accumulate=True), dict(block_tables=table.long())])


def test_prefill_weights_refusals():
    q, k, cu = _rows(3, 4), _rows(), torch.tensor([0, 3], dtype=I32)
    good = dict(query=q, key=k, cu_seqlens=cu, max_seqlen=3, scale=0.1, window=2)
    _refused(prefill_weights, good, [
        dict(window=None), dict(window=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
        dict(max_seqlen=0), dict(query=_rows(3, 3)), dict(query=_rows(2, 4)), dict(query=q.half()),
        dict(query=q.float(), key=k.float()), dict(key=k[..., :64]), dict(lse=torch.zeros((4, 2))),
        dict(lse=torch.zeros((3, 4)).t()), dict(lse=torch.zeros((4, 3)).double()), dict(cu_seqlens=cu.long())])


def test_refusals_of_the_library():
    """The C entry points' own checks; the pointers are never dereferenced."""
    from inquant import _native as nat
    import ctypes
    lib, fake = nat.lib(), 1 << 20

    def pages(**more):
        f = dict(key=fake, value=fake, weights=fake, positions=fake, k_sp=4096, k_sh=2048, k_st=128, v_sp=4096,
                 v_sh=2048, v_st=128, pages=4, heads=2, block_tokens=16)
        return ctypes.byref(nat.DensePagesDesc(**{**f, **more}))

    def decode(p, hq=4, most=640, floats=1 << 30, dtype=nat.IQ_BF16, accumulate=0):
        return lib.iq_dense_decode(fake, dtype, 512, 128, hq, 1, p, fake, 40, 40, fake, most, 0.1, accumulate, fake, floats,
                                   fake, 512, 128, nat.IQ_BF16, None)
    bad = [dict(key=0), dict(heads=0), dict(pages=0), dict(block_tokens=48), dict(key=fake + 8), dict(k_st=100),
           dict(k_st=1 << 24), dict(weights=0)]
    for change in bad:
        assert decode(pages(**change)) == -1, change
    assert decode(pages(), hq=5) == -1 and decode(pages(), hq=34) == -1 and decode(pages(), most=641) == -1
    assert decode(pages(), floats=10, accumulate=1) == -1 and b"workspace" in lib.iq_last_error()
    assert decode(pages(), dtype=nat.IQ_F32) == -1
    assert decode(pages(weights=0, positions=0), accumulate=1) == -1
    evict = lambda p, budget=8, sink=0, ints=1 << 20: lib.iq_dense_evict(
        p, nat.IQ_BF16, fake, 40, 40, fake, fake, 1, 640, budget, sink, 0, fake, fake, ints, None)
    assert evict(pages(weights=0, positions=0)) == -1 and evict(pages(), budget=0) == -1
    assert evict(pages(), sink=9) == -1 and evict(pages(), budget=300, ints=3) == -1
    assert lib.iq_dense_evict_ints(2, 1, 640, 300) == 2 * 601 and lib.iq_dense_evict_ints(2, 1, 640, 600) == 0
    assert lib.iq_select_rows(fake, 8, 2, fake, 1, 8, 4, 3, 2, fake, None) == -1
    assert lib.iq_dense_write(fake, fake + 2, nat.IQ_BF16, 256, 128, 256, 128, fake, 1, 3, None, None, None, 0, None, 0,
                              pages(), fake, 2, 2, None) == -1
    weights = lambda scale=0.1, window=2, lse=None, q_st=512: lib.iq_prefill_weights(
        fake, fake, nat.IQ_BF16, q_st, 128, 256, 128, fake, 1, 8, 8, 4, 2, window, scale, lse, 8, fake, 1 << 20, fake, 8,
        None)
    assert weights(scale=0.0) == -1 and weights(window=0) == -1 and weights(q_st=1 << 25) == -1
    # the same with the arguments in a struct
    from inquant_vllm import dense
    pool = pages()
    assert lib.iq_dense_decode_from(dense._ARGUMENTS["iq_dense_decode"](
        fake, nat.IQ_BF16, 512, 128, 4, 1, ctypes.addressof(pool._obj), fake, 40, 40, fake, 641, 0.1, 0, fake, 1 << 30,
        fake, 512, 128, nat.IQ_BF16, 0)) == -1
    assert b"max_tokens" in lib.iq_last_error()
    for name in dense._ARGUMENTS:
        assert getattr(lib, name + "_from")(None) == -1 and b"null arguments" in lib.iq_last_error()


def test_prefill_attention_refuses_a_wrong_lse():
    q, k, cu = _rows(3, 4), _rows(), torch.tensor([0, 3], dtype=I32)
    for lse in (torch.zeros((4, 2)), torch.zeros((4, 3)).double(), torch.zeros((3, 4)).t(),
                torch.zeros(3).expand(4, 3)):
        with pytest.raises((ValueError, RuntimeError)):
            prefill_attention(q, k, k, cu, 3, 0.1, lse=lse)
