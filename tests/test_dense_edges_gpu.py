"""Edges of the exact-page operators on the GPU: calls that touch no row, sequences past their bound, overlaps."""
import pytest
import torch

from densecase import generator, i32, offsets, pool, rows

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _fields(pages):
    return [t for t in (pages.key, pages.value, pages.weights, pages.positions) if t is not None]


def _equal(pages, want):
    return all(torch.equal(a, b) for a, b in zip(_fields(pages), want))


def test_an_empty_selection_writes_nothing():
    from inquant_vllm import write_rows
    gen = generator(1)
    pages = pool(gen, 6, 2, 16, torch.bfloat16)
    start = [t.clone() for t in _fields(pages)]
    key = rows(gen, 40, 2, 128, dtype=torch.bfloat16)
    keep = torch.arange(10, device="cuda", dtype=torch.int32).expand(1, 2, 10)
    write_rows(key, key, offsets([40]), 40, pages, i32([[1, 4, 2]]), keep=keep[:, :, :0])
    assert _equal(pages, start)


def test_a_copy_of_pages_works_on_its_own_memory():
    import copy
    from inquant.triton_attention import SharedDecodeWorkspace
    from inquant_vllm import dense_decode, evict_rows, write_rows
    gen = generator(2)
    pages = pool(gen, 8, 2, 16, torch.bfloat16, "halves")
    start, fork, table = [t.clone() for t in _fields(pages)], copy.deepcopy(pages), i32([[5, 1, 7]])
    key, q = rows(gen, 40, 2, 128, dtype=torch.bfloat16), rows(gen, 1, 8, 128, dtype=torch.bfloat16)

    def use(p):
        write_rows(key, key, offsets([40]), 40, p, table)
        out = dense_decode(q, p, table, i32([40]), 40, SCALE, SharedDecodeWorkspace(), accumulate=True)
        evict_rows(p, table, i32([40]), i32([40]), 40, 30, sink=1, recent=4)
        return out
    got = use(fork)
    assert _equal(pages, start) and not _equal(fork, start)
    changed = [t.clone() for t in _fields(fork)]
    assert torch.equal(use(pages), got) and _equal(pages, changed) and _equal(fork, changed)


@pytest.mark.parametrize("h", [1, 3, 16])
def test_rows_past_max_seqlen_are_left_out(h):
    """Of sequences longer than the bound every operator takes the same first rows."""
    from densecase import cache_rows, keep_rows
    from inquant_vllm import prefill_weights, select_rows, write_rows
    bound, lengths = 37, [10, 50, 38, 0, 37]
    print(f"past max_seqlen {h}", flush=True)
    gen, tokens, n = generator(10 + h), sum(lengths), len(lengths)
    taken = [min(x, bound) for x in lengths]
    key, value = (rows(gen, tokens, h, 128, dtype=torch.bfloat16) for _ in range(2))
    cu, w = offsets(lengths), torch.rand((h, tokens), generator=gen, device="cuda")
    table = torch.arange(4 * n, device="cuda").view(n, 4).to(torch.int32)
    pages = pool(gen, 4 * n, h, 16, torch.bfloat16)
    start = [t.clone() for t in _fields(pages)]
    write_rows(key, value, cu, bound, pages, table, weights=w)
    first = 0
    for i, m in enumerate(taken):
        for field, want in zip(_fields(pages)[:3], (key.transpose(0, 1), value.transpose(0, 1), w)):
            assert torch.equal(cache_rows(field, table[i], m), want[:, first:first + m])
        for field, was in zip(_fields(pages), start):
            assert torch.equal(cache_rows(field, table[i], 64)[:, m:], cache_rows(was, table[i], 64)[:, m:])
        first += lengths[i]
    got, host, first = select_rows(w, cu, bound, 20, sink=2, recent=5).tolist(), w.cpu(), 0
    for i, m in enumerate(taken):
        always = [j < 2 or j >= m - 5 for j in range(m)]
        for head in range(h):
            exp = keep_rows(host[head, first:first + m].tolist(), always, 20)
            assert got[i][head] == exp + [-1] * (20 - len(exp)), (i, head)
        first += lengths[i]
    # kept rows past the bound are skipped as those outside the sequence are
    for t, was in zip(_fields(pages), start):
        t.copy_(was)
    keep = i32([[[36, 37, 9, 40]] * h] * n)
    write_rows(key, value, cu, bound, pages, table, weights=w, keep=keep)
    first = 0
    for i, m in enumerate(taken):
        for j, r in enumerate((36, 37, 9, 40)):
            want = key[first + r] if r < m else cache_rows(start[0], table[i], 64)[:, j]
            assert torch.equal(cache_rows(pages.key, table[i], 64)[:, j], want), (i, j)
        first += lengths[i]
    # the weights of a prompt are of the same rows: those of the sequences cut to the bound
    part = torch.cat([torch.arange(f, f + m, device="cuda") for f, m in zip(cu.tolist(), taken)])
    q = rows(gen, tokens, 2 * h, 128, dtype=torch.bfloat16)
    out = torch.full((h, tokens), -5.0, device="cuda")
    prefill_weights(q, key, cu, bound, SCALE, window=8, output=out)
    cut = prefill_weights(q[part], key[part], offsets(taken), bound, SCALE, window=8)
    assert torch.equal(out[:, part], cut) and int((out == -5.0).sum()) == h * (tokens - len(part))


@pytest.mark.parametrize("lengths,heads,window,dtype", [
    # several slices of rows, the tiles placed by their tokens
    ([5, 16500, 0, 64], (32, 2), 4096, torch.bfloat16),
    # several slices, a sequence's tiles as many for each
    ([17000], (32, 4), 4096, torch.float16),
    # one long prompt of many: tiles placed by their tokens, the lse by tokens
    ([0, 63, 64, 65, 129, 1, 5000] + [70, 3, 128] * 11, (16, 2), 1000, torch.float16),
    ([1] * 30 + [4096] + [2] * 9, (16, 16), 2048, torch.bfloat16),
], ids=["slices-tokens", "slices", "ragged", "ones"])
def test_a_window_in_slices_of_bounded_scratch(lengths, heads, window, dtype):
    from test_prefill_weights_gpu import _case, _close, _expected
    from inquant_vllm import prefill_attention, prefill_weights
    hq, h = heads
    print(f"window {window} of {lengths} {heads} {dtype}", flush=True)
    q, k, v, cu = _case(len(lengths) + hq, lengths, hq, h, dtype)
    total, _, slack = _expected(q, k, lengths, SCALE, window)
    longest, tokens = max(lengths), sum(lengths)
    got = prefill_weights(q, k, cu, longest, SCALE, window=window)
    _close(got, total, slack, window * hq // h)
    lse = torch.full((hq, tokens), float("nan"), device="cuda")
    prefill_attention(q, k, v, cu, longest, SCALE, lse=lse)
    _close(prefill_weights(q, k, cu, longest, SCALE, window=window, lse=lse), total, slack, window * hq // h)
    assert torch.equal(prefill_weights(q, k, cu, longest, SCALE, window=window), got)


@pytest.mark.parametrize("nan_key", [None, 0, 40, 299])
@pytest.mark.parametrize("window", [1, 20])
def test_a_window_over_logits_of_minus_infinity(nan_key, window):
    """A query whose logits are all -inf or NaN has no softmax: its own lse says so, as the attention's does."""
    from inquant_vllm import prefill_attention, prefill_weights
    n, scale = 300, 0.5
    print(f"window of -inf {nan_key} {window}", flush=True)
    gen = generator(20)
    q, k = (rows(gen, n, 2, 128, dtype=torch.bfloat16) for _ in range(2))
    q[:, 0] = 0
    q[:, 0, 5] = 1.0                                         # head 0 reads channel 5 only
    k[:, 0, 5] = float("-inf")
    if nan_key is not None:
        k[nan_key, 0, 5] = float("nan")
    cu, lse = offsets([n]), torch.empty((2, n), device="cuda")
    got = prefill_weights(q, k, cu, n, scale, window=window)
    at = torch.arange(n, device="cuda")
    logits = torch.where(at <= at[n - window:, None], k[:, 0, 5].double() * scale, float("-inf"))
    p = (logits - logits.logsumexp(-1, keepdim=True)).exp()
    p = torch.where(at <= at[n - window:, None], p, 0.0)     # an unseen key weighs nothing
    assert torch.equal(got[0].isnan(), p.sum(0).isnan()) and got[0].isnan().all()
    assert not got[1].isnan().any()
    prefill_attention(q, k, k, cu, n, scale, lse=lse)
    with_lse = prefill_weights(q, k, cu, n, scale, window=window, lse=lse)
    assert torch.equal(with_lse.isnan(), got.isnan())


@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2)], ids=str)
def test_weights_in_the_place_of_the_lse(heads, window):
    from inquant_vllm import prefill_attention, prefill_weights
    hq, h = heads
    gen, n = generator(30), 700
    q, k = rows(gen, n, hq, 128, dtype=torch.bfloat16), rows(gen, n, h, 128, dtype=torch.bfloat16)
    lse, cu = torch.empty((hq, n), device="cuda"), offsets([n])
    prefill_attention(q, k, k, cu, n, SCALE, lse=lse)
    want = prefill_weights(q, k, cu, n, SCALE, lse=lse, window=window)
    rest = lse[h:].clone()
    got = prefill_weights(q, k, cu, n, SCALE, lse=lse, window=window, output=lse[:h])
    assert got.data_ptr() == lse.data_ptr() and torch.equal(got, want) and torch.equal(lse[h:], rest)
