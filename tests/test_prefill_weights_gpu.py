"""The weight each key of a prompt receives, against 64 bits, and the lse of the prefill attention."""
import math

import pytest
import torch

from densecase import attend, generator, offsets, rows

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _case(seed, lengths, hq, h, dtype):
    gen = generator(seed)
    tokens = sum(lengths)
    fused = rows(gen, tokens, hq + 2 * h, 128, dtype=dtype)
    fused[:, hq:hq + h, 17:19] *= 8
    return fused[:, :hq], fused[:, hq:hq + h], fused[:, hq + h:], offsets(lengths)


def _expected(q, k, lengths, scale, window):
    """Weights [h, tokens], lse [hq, tokens] (of the window's queries; others NaN) and the logits' slack."""
    h, hq = k.shape[1], q.shape[1]
    total = torch.zeros((h, q.shape[0]), dtype=torch.float64, device="cuda")
    lses = torch.full((hq, q.shape[0]), math.nan, dtype=torch.float64, device="cuda")
    first, slack = 0, 0.0
    for n in lengths:
        if n:
            lo = max(0, n - window) if window else 0
            at = torch.arange(n, device="cuda")
            ks = k[first:first + n].transpose(0, 1)
            _, lse, w, e = attend(q[first + lo:first + n].transpose(0, 1), ks, ks, scale, at <= at[lo:, None])
            total[:, first:first + n], slack = w, max(slack, e)
            lses[:, first + lo:first + n] = lse
        first += n
    return total, lses, slack


def _close(got, total, slack, adds):
    # each weight: the errors of its logit and its lse (a weighted mean of logits' errors), exp and the lse's
    # rounding (|lse| < 2^7); then `adds` additions of positive numbers
    bound = total * (4 * slack + 2.0 ** -17 + adds * 2.0 ** -24) + 1e-30
    assert ((got.double() - total).abs() <= bound).all(), float(((got.double() - total).abs() / bound).max())


LENGTHS = [[1], [2], [63, 64, 65], [255, 256, 257], [1, 500, 0, 31], [1030]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("heads", [(28, 4), (4, 4), (16, 1)], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_of_all_queries(lengths, heads, dtype):
    from inquant_vllm import prefill_attention, prefill_weights
    hq, h = heads
    print(f"weights {lengths} {heads} {dtype}", flush=True)
    q, k, v, cu = _case(len(lengths) + hq, lengths, hq, h, dtype)
    longest, tokens = max(lengths), sum(lengths)
    lse = torch.full((hq, tokens + 2), math.nan, device="cuda")
    plain = prefill_attention(q, k, v, cu, longest, SCALE)
    out = prefill_attention(q, k, v, cu, longest, SCALE, lse=lse[:, 2:])
    assert torch.equal(out, plain)
    total, lses, slack = _expected(q, k, lengths, SCALE, 0)
    assert ((lse[:, 2:].double() - lses).abs() <= 2 * slack + lses.abs() * 2.0 ** -21 + 2.0 ** -20).all()
    got = torch.full((h, tokens + 1), math.nan, device="cuda")
    res = prefill_weights(q, k, cu, longest, SCALE, lse=lse[:, 2:], output=got[:, :tokens])
    assert res.data_ptr() == got.data_ptr() and got[:, tokens].isnan().all()
    _close(got[:, :tokens], total, slack, longest * hq // h)
    # every query's weights add up to one
    assert abs(float(got[:, :tokens].double().sum()) - hq * tokens) <= hq * tokens * (4 * slack + 2.0 ** -14)


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("window", [1, 16, 64, 100, 5000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_of_a_window(lengths, window, dtype):
    from inquant_vllm import prefill_attention, prefill_weights
    hq, h = 14, 2
    print(f"window {window} of {lengths} {dtype}", flush=True)
    q, k, v, cu = _case(window + len(lengths), lengths, hq, h, dtype)
    total, _, slack = _expected(q, k, lengths, SCALE, window)
    got = prefill_weights(q, k, cu, max(lengths), SCALE, window=window)
    assert got.shape == total.shape and got.dtype == torch.float32
    _close(got, total, slack, window * hq // h)
    lse = torch.full((hq, sum(lengths)), math.nan, device="cuda")
    prefill_attention(q, k, v, cu, max(lengths), SCALE, lse=lse)
    _close(prefill_weights(q, k, cu, max(lengths), SCALE, window=window, lse=lse), total, slack, window * hq // h)


def test_poisoned_neighbours_and_untouched_tokens():
    """A sequence of NaN rows and tokens of no sequence leave their neighbours' weights alone."""
    from inquant_vllm import prefill_attention, prefill_weights
    gen = generator(5)
    hq, h, tokens = 8, 2, 700
    q, k, v = (rows(gen, tokens, x, 128, dtype=torch.bfloat16) for x in (hq, h, h))
    q[100:300], k[100:300] = math.nan, math.inf
    cu = torch.tensor([40, 100, 300, 650], dtype=torch.int32, device="cuda")
    parts = [(40, 100), (300, 650)]
    for window in (None, 33):
        lse = torch.full((hq, tokens), 3.0, device="cuda")
        prefill_attention(q, k, v, cu, 350, SCALE, lse=lse)
        assert (lse[:, :40] == 3.0).all() and (lse[:, 650:] == 3.0).all()
        out = torch.full((h, tokens), -5.0, device="cuda")
        prefill_weights(q, k, cu, 350, SCALE, lse=None if window else lse, window=window, output=out)
        assert (out[:, :40] == -5.0).all() and (out[:, 650:] == -5.0).all()
        for a, b in parts:
            total, _, slack = _expected(q[a:b], k[a:b], [b - a], SCALE, window or 0)
            _close(out[:, a:b], total, slack, 350 * hq // h)


@pytest.mark.parametrize("window", [None, 200])
def test_a_nan_query_weighs_only_what_it_sees(window):
    from inquant_vllm import prefill_attention, prefill_weights
    hq, h, n, bad = 4, 2, 600, 500
    q, k, v, cu = _case(9, [n], hq, h, torch.bfloat16)
    q[bad, 1] = math.nan                                     # of KV head 0
    lse = torch.empty((hq, n), device="cuda")
    prefill_attention(q, k, v, cu, n, SCALE, lse=lse)
    got = prefill_weights(q, k, cu, n, SCALE, lse=None if window else lse, window=window)
    assert got[0, :bad + 1].isnan().all()
    q[bad, 1] = 0
    total, _, slack = _expected(q, k, [n], SCALE, window or 0)
    _close(got[0, bad + 1:], total[0, bad + 1:], slack, 2 * n)
    _close(got[1], total[1], slack, 2 * n)


@pytest.mark.parametrize("window", [None, 16])
@pytest.mark.parametrize("heads", [(4, 2), (1, 1)], ids=str)
def test_one_lse_for_every_head(window, heads):
    from inquant_vllm import prefill_weights
    hq, h = heads
    q, k, _, cu = _case(11, [150], hq, h, torch.bfloat16)
    lse = torch.full((150,), 3.0, device="cuda").expand(hq, 150)
    got = prefill_weights(q, k, cu, 150, SCALE, lse=lse, window=window)
    assert torch.equal(got, prefill_weights(q, k, cu, 150, SCALE, lse=lse.clone(), window=window))
    if h > 1:
        with pytest.raises(ValueError, match="overlap"):
            prefill_weights(q, k, cu, 150, SCALE, lse=lse, window=window, output=got[:1].expand(h, 150))


def test_weights_of_a_long_prompt():
    # more queries than one workgroup takes, keys past the first range, over one KV head
    from inquant_vllm import prefill_attention, prefill_weights
    lengths, hq, h = [9001, 4096, 70], 2, 1
    q, k, v, cu = _case(10, lengths, hq, h, torch.float16)
    lse = torch.empty((hq, sum(lengths)), device="cuda")
    prefill_attention(q, k, v, cu, 9001, SCALE, lse=lse)
    total, _, slack = _expected(q, k, lengths, SCALE, 0)
    _close(prefill_weights(q, k, cu, 9001, SCALE, lse=lse), total, slack, 9001 * 2)


def test_weights_in_a_graph():
    from inquant_vllm import prefill_attention, prefill_weights
    q, k, v, cu = _case(8, [300, 70], 28, 4, torch.bfloat16)
    q, k, v = q.clone(), k.clone(), v.clone()
    lse, full, part = (torch.empty(s, device="cuda") for s in ((28, 370), (4, 370), (4, 370)))

    def step():
        prefill_attention(q, k, v, cu, 300, SCALE, lse=lse)
        prefill_weights(q, k, cu, 300, SCALE, lse=lse, output=full)
        prefill_weights(q, k, cu, 300, SCALE, window=20, output=part)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        q.copy_(rows(generator(seed), 370, 28, 128, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = full.clone(), part.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], full) and torch.equal(got[1], part)
