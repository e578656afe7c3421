"""Exact pages, prompts and their plain 64-bit forms, for the tests of the exact-page operators."""
import math

import torch

EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative


def rows(gen, *shape, dtype, gain=None, device="cuda"):
    x = torch.randn(shape, generator=gen, device=device)
    if gain is not None:
        x[..., 17:19] *= gain
    return x.to(dtype)


def generator(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def pool(gen, pages, heads, B, dtype, layout="plain", evictable=True):
    """DensePages of random rows: its own tensors, one [pages, 2, H, B, D] pool's
    halves, or a token-major [pages, B, H, D] pool."""
    from inquant_vllm import DensePages
    if layout == "halves":
        both = rows(gen, pages, 2, heads, B, 128, dtype=dtype, gain=8)
        key, value = both[:, 0], both[:, 1]
    elif layout == "token_major":
        key = rows(gen, pages, B, heads, 128, dtype=dtype, gain=8).transpose(1, 2)
        value = rows(gen, pages, B, heads, 136, dtype=dtype)[..., :128].transpose(1, 2)
    else:
        key = rows(gen, pages, heads, B, 128, dtype=dtype, gain=8)
        value = rows(gen, pages, heads, B, 128, dtype=dtype)
    if not evictable:
        return DensePages(key, value)
    weights = (2 * torch.randn((pages, heads, B), generator=gen, device="cuda")).exp()
    positions = torch.randint(0, 1 << 30, (pages, heads, B), generator=gen, device="cuda").to(torch.int32)
    return DensePages(key, value, weights, positions)


def tables(gen, lengths, B, pages, columns=None):
    """Block tables int32 of sequences at random pages, -1 behind their last."""
    need = [-(-n // B) for n in lengths]
    assert sum(need) <= pages
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    out = torch.full((len(lengths), columns or max(1, *need)), -1, dtype=torch.int32, device="cuda")
    first = 0
    for i, n in enumerate(need):
        out[i, :n] = order[first:first + n]
        first += n
    return out


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return i32(out)


def cache_rows(field, table, n):
    """[H, n, ...] cache rows 0 .. n - 1 of a sequence, of a pool field [pages, H, B, ...]."""
    B = field.shape[2]
    at = torch.arange(n, device=field.device)
    return field[table[at // B].long(), :, at % B].transpose(0, 1)


def attend(q, k, v, scale, seen=None):
    """q [hq, m, D], k/v [h, n, D]: outputs, logits' lse and each key's summed weights in 64 bits, and a bound on
    the error of a 32-bit logit (any order of 128 products) in units of a logit."""
    h, n = k.shape[:2]
    g = q.shape[0] // h
    k, v = k.double(), v.double()
    outs, lses, slack = [], [], 0.0
    total = torch.zeros((h, n), dtype=torch.float64, device=k.device)
    for i in range(q.shape[0]):
        qi, ki, vi = q[i].double(), k[i // g], v[i // g]
        logits = (qi @ ki.t().contiguous()) * scale
        slack = max(slack, float((qi.abs() @ ki.abs().t().contiguous()).max()) * abs(scale) * 130 * 2.0 ** -24)
        if seen is not None:
            logits = logits.masked_fill(~seen, -math.inf)
        lse = logits.logsumexp(-1)
        p = (logits - lse[:, None]).exp()
        outs.append(p @ vi)
        lses.append(lse)
        total[i // g] += p.sum(0)
    return torch.stack(outs), torch.stack(lses), total, slack


def output_bound(v, dtype, out_dtype, slack):
    """A weight carries twice a logit's error and one rounding to the rows' type; the output one rounding of its own."""
    return float(v.double().abs().max()) * (EPS[dtype] + EPS[out_dtype] + 4 * slack + 2.0 ** -20)


def keep_rows(weights, always, budget):
    """Kept indices, ascending, of one head's weights (a list): always-kept first (the lowest of them, should they
    exceed the budget), then by weight, NaN last, ties low."""
    def worth(i):
        w = weights[i]
        return (False, False, 0.0, i) if always[i] else (True, w != w, -w if w == w else 0.0, i)
    return sorted(sorted(range(len(weights)), key=worth)[:budget])
