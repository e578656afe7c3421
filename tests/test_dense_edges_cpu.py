"""Calls of the exact-page operators that touch no row, their copies and what they ask for, checked on the host."""
import pytest
import torch

from inquant_vllm import DensePages, dense, write_rows

I32 = torch.int32


@pytest.fixture
def calls(monkeypatch):
    """What would go to the library, with CPU tensors taken for the GPU's."""
    made = []
    monkeypatch.setattr(dense, "_on_gpu", lambda *a: None)
    monkeypatch.setattr(dense, "_call", lambda gpu, name, *args: made.append((name, args)))
    return made


def test_an_empty_selection_writes_nothing(calls):
    pages = DensePages.allocate(4, 16, 2, device="cpu")
    k, cu, table = torch.zeros((3, 2, 128), dtype=torch.bfloat16), torch.tensor([0, 3], dtype=I32), torch.zeros((1, 2), dtype=I32)
    # a tensor without elements has no address, which the library reads as "every row"
    write_rows(k, k, cu, 3, pages, table, keep=torch.zeros((1, 2, 5), dtype=I32)[:, :, :0])
    assert calls == []
    write_rows(k, k, cu, 3, pages, table, keep=torch.zeros((1, 2, 5), dtype=I32)[:, :, :1])
    write_rows(k, k, cu, 3, pages, table)
    assert [name for name, _ in calls] == ["iq_dense_write_from"] * 2
    with pytest.raises(ValueError):
        write_rows(k, k, cu, 3, pages, table, keep=torch.zeros((1, 3, 0), dtype=I32))


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "copy"])
@pytest.mark.parametrize("evictable", [True, False])
@pytest.mark.parametrize("halves", [True, False])
def test_copies_of_pages_describe_their_own_memory(how, evictable, halves):
    import copy
    import ctypes
    import pickle
    from inquant import _native as nat
    if halves:
        both = torch.randn((4, 2, 3, 16, 128)).bfloat16()
        key, value = both[:, 0], both[:, 1]
    else:
        key, value = torch.randn((4, 16, 3, 128)).half().transpose(1, 2), torch.randn((4, 3, 16, 136)).half()[..., :128]
    side = (torch.randn((4, 3, 16)), torch.arange(192, dtype=I32).view(4, 3, 16)) if evictable else ()
    first = DensePages(key, value, *side)
    made = {"deepcopy": copy.deepcopy, "pickle": lambda x: pickle.loads(pickle.dumps(x)), "copy": copy.copy}[how](first)
    desc = ctypes.cast(made._desc, ctypes.POINTER(nat.DensePagesDesc)).contents
    own = ctypes.addressof(made._pages)
    assert made._desc == own and (how == "copy" or own != ctypes.addressof(first._pages))
    for name in ("key", "value", "weights", "positions"):
        mine, theirs = getattr(made, name), getattr(first, name)
        assert getattr(desc, name) == (0 if mine is None else mine.data_ptr())
        if mine is not None:
            assert torch.equal(mine, theirs) and (mine.data_ptr() == theirs.data_ptr()) == (how == "copy")
    assert (desc.k_sp, desc.k_sh, desc.k_st) == made.key.stride()[:3]
    assert (desc.v_sp, desc.v_sh, desc.v_st) == made.value.stride()[:3]
    assert (desc.pages, desc.heads, desc.block_tokens) == (4, 3, 16)
    assert (made.block_size, made.heads, made._dtype, made._code) == (16, 3, first._dtype, first._code)


def test_a_lent_workspace_keeps_a_bounded_past():
    """What a captured graph may still use is kept, counted, and never more than what is in use."""
    from inquant.triton_attention import SharedDecodeWorkspace

    class Pin:
        def check(self, device):
            return 0

    def fresh():
        ws = SharedDecodeWorkspace()
        ws._pin = Pin()
        return ws
    ws = fresh()
    ws.acquire((10, 10), "cpu")
    ws.acquire((11, 10), "cpu")
    assert ws.tensor.numel() == 110 and ws.nbytes == 440              # before a loan: what is asked for, nothing kept
    address, have, _ = ws.floats(64, "cpu")
    assert (address, have) == (ws.tensor.data_ptr(), 110)
    lent = [ws.tensor]
    for size in range(120, 4000, 37):                                 # a decode whose partitions grow with its context
        assert ws.acquire((size,), "cpu").shape == (size,)
        if ws.tensor is not lent[-1]:
            lent.append(ws.tensor)
        if size % 5 == 0:
            address, have, _ = ws.floats(size + 3, "cpu")
            assert have >= size + 3 and address == ws.tensor.data_ptr()
            if ws.tensor is not lent[-1]:
                lent.append(ws.tensor)
    assert [t.data_ptr() for t in ws._lent] == [t.data_ptr() for t in lent[:-1]]
    past = sum(t.numel() for t in ws._lent)
    assert len(lent) > 3 and past <= ws.tensor.numel()
    assert ws.nbytes == 4 * (past + ws.tensor.numel())
    ws = fresh()
    assert ws.floats(0, "cpu")[1] == 0 and ws.acquire((5,), "cpu").numel() == 5
    assert fresh().nbytes == 0 and ws.nbytes == 20
    ws = fresh()
    ws._lent = []                                                     # lent, but nothing allocated yet
    ws.acquire((3,), "cpu")
    assert ws.nbytes == 12


def _window_floats(hq, n, longest, tokens, window):
    from inquant import _native as nat
    return nat.lib().iq_prefill_weights_floats(hq, n, longest, tokens, window, 0)


@pytest.mark.parametrize("hq,n,longest,tokens,window", [
    (32, 16, 32768, 16 * 32768, 4096), (28, 8, 32768, 8 * 32768, 4096), (32, 1, 131072, 131072, 4096),
    (32, 64, 131072, 131072 + 63 * 100, 256), (16, 1000, 4096, 4096 + 999 * 10, 4096), (64, 1, 1 << 20, 1 << 20, 4096),
    (32, 60000, 32768, 92767, 64)])
def test_scratch_of_a_window_is_bounded(hq, n, longest, tokens, window):
    # (max, sum) of 256 MiB or of 64 rows, and the rows' lse, never more than one per token
    tiles = min(n * -(-longest // 64), tokens // 64 + n)
    most = max(1 << 26, 2 * tiles * hq * 64) + hq * min(n * window, tokens)
    assert _window_floats(hq, n, longest, tokens, window) <= most


def test_scratch_of_a_small_window_holds_every_tile_and_row():
    for hq, n, longest, window in ((28, 1, 32768, 64), (32, 3, 9000, 100), (16, 1, 1, 1)):
        assert _window_floats(hq, n, longest, n * longest, window) == \
            2 * n * -(-longest // 64) * hq * window + n * hq * window


def test_tiles_placed_by_their_tokens_do_not_overlap():
    import random
    rng = random.Random(1)
    for _ in range(300):
        at = start = rng.choice([0, 0, 63, 1000])
        ends, n = [0], rng.randint(1, 30)                    # an end of the sequence before: none below its base
        for i in range(n):
            base, length = at // 64 + i, rng.choice([0, 1, 63, 64, 65, rng.randint(0, 3000)])
            assert base >= ends[-1]
            ends.append(base + -(-length // 64))
            at += length
        assert ends[-1] <= at // 64 + n, start


def test_decode_refuses_outputs_whose_rows_overlap(calls, monkeypatch):
    from inquant_vllm import dense_decode
    from inquant.triton_attention import SharedDecodeWorkspace
    ran = []
    monkeypatch.setattr(dense, "_status", lambda *a: ran.append(a) or 0)
    monkeypatch.setattr(SharedDecodeWorkspace, "floats", lambda *a: (0, 0, 0))
    n, hq = 3, 4
    pages = DensePages.allocate(4, 16, 2, device="cpu")
    q, table, lengths = torch.zeros((n, hq, 128), dtype=torch.bfloat16), torch.zeros((n, 1), dtype=I32), torch.ones(n, dtype=I32)

    def call(*strides, n=n, hq=hq):
        out = torch.zeros(10000).as_strided((n, hq, 128), strides)
        return dense_decode(q[:n, :hq], pages, table[:n], lengths[:n], 16, 0.1, SharedDecodeWorkspace(), out)
    for strides in ((128, 128, 1), (256, 128, 1), (511, 128, 1), (128, 383, 1), (256, 256, 1), (0, 128, 1), (512, 64, 1),
                    (128, 256, 1)):
        with pytest.raises(ValueError, match="overlap"):
            call(*strides)
    assert ran == []
    for strides in ((512, 128, 1), (513, 128, 1), (128, 384, 1), (700, 130, 1), (128, 391, 1)):
        call(*strides)
    call(640, 256, 1)                                        # a sequence's rows between those of the next
    call(5, 128, 1, n=1)
    assert len(ran) == 7


def test_eviction_refuses_lengths_that_overlap_the_new_ones(calls):
    """In the place of the old ones or apart: a sequence's new length must not be another's old one."""
    import ctypes
    from inquant import _native as nat
    from inquant_vllm import evict_rows
    pages, table = DensePages.allocate(4, 16, 2, device="cpu"), torch.zeros((4, 2), dtype=I32)
    held, seen = torch.full((9,), 20, dtype=I32), torch.full((9,), 30, dtype=I32)
    for shift in (1, 3):
        for a, b in ((held[:4], held[shift:shift + 4]), (held[shift:shift + 4], held[:4])):
            with pytest.raises(ValueError, match="overlap"):
                evict_rows(pages, table, a, seen[:4], 32, 8, output=b)
    assert calls == []
    for out in (held[:4], held[4:8], seen[:4], seen[1:5], None):
        evict_rows(pages, table, held[:4], seen[:4], 32, 8, output=out)
    strided = held[:8:2]                                     # copied before the call
    evict_rows(pages, table, strided, seen[:4], 32, 8, output=held[1:5])
    assert len(calls) == 6
    # and the library
    fake = 1 << 20
    desc = nat.DensePagesDesc(fake, fake, fake, fake, 4096, 2048, 128, 4096, 2048, 128, 4, 2, 16)
    for new in (fake + 4, fake - 12):
        for most in (32, 640):
            assert nat.lib().iq_dense_evict(ctypes.byref(desc), nat.IQ_BF16, fake, 40, 40, fake, fake, 4, most, 300, 0,
                                            0, new, fake, 1 << 20, None) == -1
            assert b"overlap" in nat.lib().iq_last_error()


def test_weights_in_the_place_of_the_lse_read_a_copy(calls):
    """Workgroups write a key's weight while others still read the lse of its memory."""
    from inquant_vllm import prefill_weights
    q, k, cu = torch.zeros((20, 4, 128)).half(), torch.zeros((20, 4, 128)).half(), torch.tensor([0, 20], dtype=I32)
    memory = torch.zeros(400)

    def lse_address(lse, **more):
        prefill_weights(q, k, cu, 20, 0.1, lse=lse, **more)
        return calls[-1][1][15]
    lse = memory[:80].view(4, 20)
    for out in (lse, memory[40:120].view(4, 20), memory[60:260].view(4, 50)[:, :20], memory[79:159].view(4, 20)):
        assert not memory.data_ptr() <= lse_address(lse, output=out) < memory.data_ptr() + 1600
    apart = memory[80:160].view(4, 20)
    assert lse_address(lse, output=apart) == lse.data_ptr() == lse_address(lse)
    assert lse_address(apart, output=lse, window=3) == apart.data_ptr()


@pytest.mark.parametrize("tokens,ranges", [(1000, 2), (4096, 4), (8192, 2), (16384, 2), (32768, 2), (131072, 2)])
def test_ranges_of_a_prompts_queries(tokens, ranges):
    """The split that the kernel's comment gives times for (28 heads): one sum per range, head and token."""
    from inquant import _native as nat
    assert nat.lib().iq_prefill_weights_floats(28, 1, tokens, tokens, 0, 1) == ranges * 28 * tokens
