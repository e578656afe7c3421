"""Timed cases of the exact (unpacked) pages: what is kept of a prompt, the attention that reads it, and eviction.

Six kinds of work:

* ``decode``   one token's attention for a batch of sequences over exact pages, which adds each row's attention
               weight to the page's accumulated weights;
* ``prompt``   causal attention of a batch of prompts, and the weight each key received from all queries;
* ``window``   the weight each key of a prompt receives from the prompt's last few queries;
* ``select``   the rows of a prompt that a budget keeps, by accumulated weight;
* ``write``    a prompt's rows, all or the kept ones, into pages;
* ``evict``    new rows of running sequences written into their pages, and the pages cut back to the budget.

Keys and values are N(0, 1) with about 4% of the channels of each head, in runs of two and one, times 20 (keys of
pages and prompts); accumulated weights are exp(2 N(0, 1)), one in eight of them zero.  Pages sit at random places of
a pool that is an eighth larger than what they need.
"""
import math
import os
import random
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inquant-open-source_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
SCALE = 128 ** -0.5


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one layer of one short chat: the smallest call, where launches and the host count
        {"name": "decode_300", "kind": "decode", "hq": 28, "h": 4, "page": 16, "seqs": 1, "low": 300, "high": 300,
         "accumulate": True, "dtype": "bf16"},
        # a serving step of 16 requests between 2K and 32K tokens
        {"name": "decode_16seq", "kind": "decode", "hq": 28, "h": 4, "page": 16, "seqs": 16, "low": 2048,
         "high": 32768, "accumulate": False, "dtype": "bf16"},
        # two long documents, eight KV heads, with the weights that a later eviction goes by
        {"name": "decode_2x128k", "kind": "decode", "hq": 32, "h": 8, "page": 256, "seqs": 2, "low": 129000,
         "high": 131072, "accumulate": True, "dtype": "f16"},
        # an 8K prompt's attention and the weights of its keys
        {"name": "prompt_8k", "kind": "prompt", "hq": 28, "h": 4, "seqs": 1, "low": 8192, "high": 8192,
         "dtype": "bf16"},
        # a ragged batch of prompts in fp16
        {"name": "prompt_ragged", "kind": "prompt", "hq": 32, "h": 8, "seqs": 7, "low": 37, "high": 4100,
         "dtype": "f16"},
        # a 32K prompt judged by its last 64 queries
        {"name": "window_32k", "kind": "window", "hq": 28, "h": 4, "seqs": 1, "low": 32768, "high": 32768,
         "window": 64, "dtype": "bf16"},
        # 1024 rows of a 4K prompt, the sink and the newest among them
        {"name": "select_4k", "kind": "select", "h": 4, "seqs": 1, "low": 4096, "high": 4096, "budget": 1024,
         "sink": 4, "recent": 128},
        # a batch of prompts up to 32K, eight heads
        {"name": "select_ragged", "kind": "select", "h": 8, "seqs": 12, "low": 1500, "high": 32768, "budget": 4096,
         "sink": 4, "recent": 500},
        # the kept rows of four long prompts into 16-token pages
        {"name": "write_kept", "kind": "write", "h": 4, "page": 16, "seqs": 4, "low": 8000, "high": 32768,
         "budget": 4096, "dtype": "bf16"},
        # every row of a ragged batch of prompts
        {"name": "write_ragged", "kind": "write", "h": 8, "page": 64, "seqs": 7, "low": 37, "high": 16384,
         "budget": 0, "dtype": "f16"},
        # a decode step of 16 sequences at their budget: one new row each, one row evicted
        {"name": "evict_step", "kind": "evict", "h": 4, "page": 16, "seqs": 16, "budget": 2048, "low": 1, "high": 1,
         "sink": 4, "recent": 256, "dtype": "bf16"},
        # chunks of up to 2048 new rows into caches of 8192
        {"name": "evict_chunk", "kind": "evict", "h": 8, "page": 256, "seqs": 4, "budget": 8192, "low": 300,
         "high": 2048, "sink": 4, "recent": 2048, "dtype": "f16"},
    ]


HEADS = [(28, 4), (32, 8), (16, 2), (8, 8), (14, 2), (12, 1), (16, 1)]
PAGES = [16, 16, 32, 64, 128, 256]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prompt", "window", "select", "write", "evict"])
    hq, h = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        high = _log(rng, 1, min(131072, 2000000 // (seqs * h)))
        return {"kind": kind, "hq": hq, "h": h, "page": rng.choice(PAGES), "seqs": seqs,
                "low": max(1, high // rng.choice([1, 3, 20])), "high": high, "accumulate": rng.random() < 0.6,
                "dtype": dtype}
    if kind == "prompt":
        seqs = rng.choice([1, 1, 2, 4, 9])
        high = _log(rng, 1, int(math.sqrt(1.8e9 / (seqs * hq))))
        return {"kind": kind, "hq": hq, "h": h, "seqs": seqs, "low": max(1, high // rng.choice([1, 2, 10])),
                "high": high, "dtype": dtype}
    if kind == "window":
        seqs = rng.choice([1, 1, 3])
        high = _log(rng, 1, 32768 // seqs)
        return {"kind": kind, "hq": hq, "h": h, "seqs": seqs, "low": max(1, high // rng.choice([1, 2, 10])),
                "high": high, "window": _log(rng, 1, 100), "dtype": dtype}
    if kind == "select":
        seqs = _log(rng, 1, 12)
        high = _log(rng, 16, 32768)
        low = max(8, high // rng.choice([1, 2, 10]))
        budget = _log(rng, 4, low - 2)
        sink = rng.choice([0, 1, 2])
        return {"kind": kind, "h": h, "seqs": seqs, "low": low, "high": high, "budget": budget, "sink": sink,
                "recent": rng.randint(0, budget - sink - 2)}
    if kind == "write":
        seqs = _log(rng, 1, 16)
        high = _log(rng, 1, min(32768, 400000 // (seqs * h)))
        return {"kind": kind, "h": h, "page": rng.choice(PAGES), "seqs": seqs,
                "low": max(1, high // rng.choice([1, 2, 10])), "high": high,
                "budget": rng.choice([0, _log(rng, 1, high)]), "dtype": dtype}
    seqs, budget = _log(rng, 1, 16), _log(rng, 8, 8192)
    recent = _log(rng, 1, budget // 2)
    high = rng.choice([1, rng.randint(1, recent)])
    return {"kind": kind, "h": h, "page": rng.choice(PAGES), "seqs": seqs, "budget": budget, "low": 1, "high": high,
            "sink": min(4, budget - recent), "recent": recent, "dtype": dtype}


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """The sequences' lengths (``evict``: their new rows), part of the case: the same for every seed."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["low"], case["high"]))
    return [rng.randint(case["low"], case["high"]) for _ in range(case["seqs"])]


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def _gain(rng, h):
    """[h, 1, 128] factors: runs of two, two and one outlier channels, times 20."""
    gain = torch.ones((h, 1, 128))
    for head in range(h):
        for width in (2, 2, 1):
            start = rng.randrange(128 - width + 1)
            gain[head, 0, start:start + width] = 20.0
    return gain.to(DEV)


def _scores(gen, *shape):
    """Accumulated weights: over some orders of magnitude, one in eight rows never attended to."""
    w = (2 * _randn(gen, *shape)).exp_()
    return w * (torch.rand(shape, generator=gen, device=DEV) >= 0.125)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).to(DEV)


def _offsets(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return _i32(total)


def _pool(gen, rng, case, rows, dtype):
    """A pool of exact pages and the block tables of sequences that hold up to `rows` rows each."""
    h, B = case["h"], case["page"]
    width = [-(-n // B) for n in rows]
    used = sum(width)
    pages = used + used // 8 + 1
    key = (_randn(gen, pages, h, B, 128) * _gain(rng, h)).to(dtype)
    value = _randn(gen, pages, h, B, 128).to(dtype)
    at = torch.randperm(pages, generator=gen, device=DEV)[:used].to(torch.int32)
    tables = torch.full((len(rows), max(width)), -1, dtype=torch.int32, device=DEV)
    first = 0
    for i, n in enumerate(width):
        tables[i, :n] = at[first:first + n]
        first += n
    return {"key": key, "value": value, "weights": _scores(gen, pages, h, B),
            "positions": torch.zeros((pages, h, B), dtype=torch.int32, device=DEV), "tables": tables}


def prepare(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    kind, h, lengths = case["kind"], case["h"], _lengths(case)
    n, longest = len(lengths), max(lengths)
    state = {"case": case}
    if kind == "select":
        state.update(weights=_scores(gen, h, sum(lengths)), cu=_offsets(lengths), longest=longest)
        return state
    dtype = DTYPES[case["dtype"]]
    if kind == "decode":
        state.update(_pool(gen, rng, case, lengths, dtype))
        state.update(q=_randn(gen, n, case["hq"], 128).to(dtype), lengths=_i32(lengths), longest=longest)
        state["out"] = torch.empty_like(state["q"])
        if own:
            from inquant.triton_attention import SharedDecodeWorkspace
            state["workspace"] = SharedDecodeWorkspace()
    elif kind in ("prompt", "window"):
        tokens = sum(lengths)
        state.update(q=_randn(gen, tokens, case["hq"], 128).to(dtype),
                     k=(_randn(gen, tokens, h, 128) * _gain(rng, h)[:, 0]).to(dtype),
                     v=_randn(gen, tokens, h, 128).to(dtype), cu=_offsets(lengths), longest=longest)
        state["out"] = torch.empty_like(state["q"])
        state["lse"] = torch.empty((case["hq"], tokens), dtype=torch.float32, device=DEV)
        state["weights"] = torch.empty((h, tokens), dtype=torch.float32, device=DEV)
    elif kind == "write":
        tokens, budget = sum(lengths), case["budget"]
        state.update(_pool(gen, rng, case, [min(x, budget) if budget else x for x in lengths], dtype))
        state.update(k=_randn(gen, tokens, h, 128).to(dtype), v=_randn(gen, tokens, h, 128).to(dtype),
                     w=_scores(gen, h, tokens), cu=_offsets(lengths), longest=longest, keep=None)
        if budget:
            # the rows a selection kept, ascending, -1 behind the last
            keep = torch.full((n, h, budget), -1, dtype=torch.int32, device=DEV)
            for i, x in enumerate(lengths):
                m = min(x, budget)
                picked = torch.rand((h, x), generator=gen, device=DEV).topk(m, -1).indices
                keep[i, :, :m] = picked.sort(-1).values.to(torch.int32)
            state["keep"] = keep
    else:
        budget, recent, tokens = case["budget"], case["recent"], sum(lengths)
        state.update(_pool(gen, rng, case, [budget + x for x in lengths], dtype))
        # what the caches hold: the newest rows and a spread of older ones, in the order that evictions left
        seen = budget * 4 + 7
        old = torch.arange(budget - recent, device=DEV) * (seen - recent) // max(1, budget - recent)
        held = torch.cat((old, torch.arange(seen - recent, seen, device=DEV))).to(torch.int32)
        order = torch.rand((n, h, budget), generator=gen, device=DEV).argsort(-1)
        page, row = _places(state["tables"], budget, case["page"])
        state["positions"][page.unsqueeze(1), torch.arange(h, device=DEV)[:, None], row] = held[order]
        state.update(k=_randn(gen, tokens, h, 128).to(dtype), v=_randn(gen, tokens, h, 128).to(dtype),
                     w=_scores(gen, h, tokens), cu=_offsets(lengths), longest=longest, new=_i32(lengths),
                     held=_i32([budget] * n), full=_i32([budget + x for x in lengths]), seen=_i32([seen] * n))
    if own and "tables" in state:
        from inquant_vllm import DensePages
        state["pages"] = DensePages(state["key"], state["value"], state["weights"], state["positions"])
    return state


# ------------------------------------------------------------------ plain forms

def _places(tables, rows, B):
    """Page [n, rows] and row in the page [rows] of cache rows 0 .. rows - 1."""
    row = torch.arange(rows, device=DEV)
    return tables[:, row // B].long().clamp_(min=0), row % B


def _padded(x, cu, longest):
    """[n, longest, ...] rows of the sequences of x, whose rows past the end repeat its last one, and which are real."""
    at = cu[:-1, None].long() + torch.arange(longest, device=DEV)
    real = at < cu[1:, None]
    return x[torch.minimum(at, cu[1:, None].long() - 1)], real


def _softmax(logits, seen):
    """softmax over the last axis of the entries `seen`, in place."""
    logits.masked_fill_(~seen, -math.inf)
    logits.sub_(logits.amax(-1, keepdim=True)).exp_()
    return logits.div_(logits.sum(-1, keepdim=True))


def _decode(s):
    case, longest = s["case"], s["longest"]
    n, h, g = case["seqs"], case["h"], case["hq"] // case["h"]
    page, row = _places(s["tables"], longest, case["page"])
    heads = torch.arange(h, device=DEV)[:, None]
    k = s["key"][page.unsqueeze(1), heads, row].float()                     # [n, h, longest, 128]
    v = s["value"][page.unsqueeze(1), heads, row].float()
    q = s["q"].float().view(n, h, g, 128)
    live = torch.arange(longest, device=DEV) < s["lengths"][:, None]
    p = _softmax((q @ k.transpose(-1, -2)).mul_(SCALE), live[:, None, None])
    s["out"].copy_((p @ v).view(n, h * g, 128))
    if not case["accumulate"]:
        return s["out"]
    where = (page.unsqueeze(1), heads, row)
    fresh = s["weights"][where] + p.sum(2)
    # places past a sequence's end belong to nobody or to another sequence: nothing is added there
    some = live[:, None].expand_as(fresh)
    s["weights"].index_put_(tuple(x.expand_as(fresh)[some] for x in where), fresh[some])
    return s["out"], s["weights"]


def _queries_and_keys(s):
    case = s["case"]
    h, g, longest = case["h"], case["hq"] // case["h"], s["longest"]
    k, real = _padded(s["k"], s["cu"], longest)
    return h, g, longest, k.float().transpose(1, 2), real                   # [n, h, longest, 128]


def _scatter_rows(x, real, out):
    """out [h, tokens] from x [n, h, longest]."""
    out.copy_(x.transpose(0, 1)[:, real])
    return out


def _prompt(s):
    h, g, longest, k, real = _queries_and_keys(s)
    v = _padded(s["v"], s["cu"], longest)[0].float().transpose(1, 2)
    q = _padded(s["q"], s["cu"], longest)[0].float().transpose(1, 2)        # [n, hq, longest, 128]
    n = q.shape[0]
    at = torch.arange(longest, device=DEV)
    logits = (q.reshape(n, h, g * longest, 128) @ k.transpose(-1, -2)).mul_(SCALE).view(n, h, g, longest, longest)
    p = _softmax(logits, at <= at[:, None])
    out = (p.view(n, h, g * longest, longest) @ v).view(n, h * g, longest, 128).transpose(1, 2)
    s["out"].copy_(out[real])
    p.mul_(real[:, None, None, :, None])
    return s["out"], _scatter_rows(p.sum((2, 3)), real, s["weights"])


def _window(s):
    h, g, longest, k, real = _queries_and_keys(s)
    W, cu = s["case"]["window"], s["cu"].long()
    n, size = k.shape[0], (cu[1:] - cu[:-1])[:, None]
    at = size - W + torch.arange(W, device=DEV)                             # the window's queries, from the end
    there = at >= 0
    at = at.clamp_(min=0)
    q = s["q"][cu[:-1, None] + at].float().transpose(1, 2)                  # [n, hq, W, 128]
    logits = (q.reshape(n, h, g * W, 128) @ k.transpose(-1, -2)).mul_(SCALE).view(n, h, g, W, longest)
    p = _softmax(logits, (torch.arange(longest, device=DEV) <= at[..., None])[:, None, None])
    p.mul_(there[:, None, None, :, None])
    return _scatter_rows(p.sum((2, 3)), real, s["weights"])


def _kept(weights, first, live, budget):
    """Which rows [..., rows] a budget keeps: those of `first`, then by weight, ties to the lowest index."""
    worth = weights.masked_fill(first, math.inf).masked_fill_(~live, -math.inf)
    order = worth.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    return torch.zeros_like(live).scatter_(-1, order, True) & live


def _select(s):
    case, longest = s["case"], s["longest"]
    w, live = _padded(s["weights"].t(), s["cu"], longest)
    w, live = w.transpose(1, 2), live[:, None]                              # [n, h, longest]
    at = torch.arange(longest, device=DEV)
    size = (s["cu"][1:] - s["cu"][:-1])[:, None, None]
    first = (at < case["sink"]) | (at >= size - case["recent"])
    kept = _kept(w, first.expand_as(w), live.expand_as(w), case["budget"])
    rank = kept.cumsum(-1).sub_(1).masked_fill_(~kept, case["budget"])
    keep = torch.full((*w.shape[:2], case["budget"] + 1), -1, dtype=torch.int32, device=DEV)
    keep.scatter_(-1, rank, at.to(torch.int32).expand_as(rank).contiguous())
    return keep[..., :-1].contiguous()


def _write(s, start=None, positions=None):
    """Rows of every sequence (or the kept ones of each head) into the pages from cache row `start`."""
    B, cu, keep, h = s["case"]["page"], s["cu"].long(), s.get("keep"), s["case"]["h"]
    size = (cu[1:] - cu[:-1])[:, None, None]
    if keep is None:
        source = torch.arange(s["longest"], device=DEV).expand(size.shape[0], h, s["longest"])
        real = source < size
    else:
        source, real = keep.long(), keep >= 0
    zero = torch.zeros(size.shape[0], dtype=torch.int64, device=DEV)
    start = zero if start is None else start.long()
    positions = start if positions is None else positions.long()
    target = start[:, None, None] + torch.arange(source.shape[-1], device=DEV).expand_as(source)
    seq, head, column = real.nonzero(as_tuple=True)
    source, target = source[real], target[real]
    place = (s["tables"][seq, target // B].long(), head, target % B)
    row = cu[seq] + source
    s["key"][place] = s["k"][row, head]
    s["value"][place] = s["v"][row, head]
    s["weights"][place] = s["w"][head, row]
    s["positions"][place] = (positions[seq] + source).to(torch.int32)
    return s["key"], s["value"], s["weights"], s["positions"]


def _evict(s):
    case = s["case"]
    _write(s, s["held"], s["seen"])
    s["seen"].add_(s["new"])
    budget, rows, h = case["budget"], case["budget"] + s["longest"], case["h"]
    page, row = _places(s["tables"], rows, case["page"])
    where = (page.unsqueeze(1), torch.arange(h, device=DEV)[:, None], row)
    w, pos = s["weights"][where], s["positions"][where]
    at = torch.arange(rows, device=DEV)
    live = (at < s["full"][:, None])[:, None].expand_as(w)
    first = (pos < case["sink"]) | (pos >= (s["seen"] - case["recent"])[:, None, None])
    kept = _kept(w, first, live, budget)
    # kept rows behind the budget move, in order, to the evicted places before it
    holes, movers = ~kept & (at < budget), kept & (at >= budget)
    source = at.expand_as(w).clone()
    source[holes] = at.expand_as(w)[movers]
    source = source[..., :budget]
    place = tuple(x.expand_as(w)[..., :budget] for x in where)
    origin = (s["tables"].long().unsqueeze(1).expand(-1, h, -1).gather(-1, source // case["page"]), place[1],
              source % case["page"])
    for name in ("key", "value", "weights", "positions"):
        s[name][place] = s[name][origin]
    return s["key"], s["value"], s["weights"], s["positions"], s["full"].clamp(max=budget)


# ------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"decode": _decode, "prompt": _prompt, "window": _window, "select": _select, "write": _write,
                "evict": _evict}[kind](s)
    import inquant_vllm as iv
    if kind == "decode":
        out = iv.dense_decode(s["q"], s["pages"], s["tables"], s["lengths"], s["longest"], SCALE, s["workspace"],
                              s["out"], accumulate=case["accumulate"])
        return (out, s["weights"]) if case["accumulate"] else out
    if kind == "prompt":
        out = iv.prefill_attention(s["q"], s["k"], s["v"], s["cu"], s["longest"], SCALE, s["out"], lse=s["lse"])
        return out, iv.prefill_weights(s["q"], s["k"], s["cu"], s["longest"], SCALE, lse=s["lse"],
                                       output=s["weights"])
    if kind == "window":
        return iv.prefill_weights(s["q"], s["k"], s["cu"], s["longest"], SCALE, window=case["window"],
                                  output=s["weights"])
    if kind == "select":
        return iv.select_rows(s["weights"], s["cu"], s["longest"], case["budget"], sink=case["sink"],
                              recent=case["recent"])
    if kind == "write":
        iv.write_rows(s["k"], s["v"], s["cu"], s["longest"], s["pages"], s["tables"], weights=s["w"], keep=s["keep"])
        return s["key"], s["value"], s["weights"], s["positions"]
    iv.write_rows(s["k"], s["v"], s["cu"], s["longest"], s["pages"], s["tables"], s["held"], positions=s["seen"],
                  weights=s["w"])
    s["seen"].add_(s["new"])
    lengths = iv.evict_rows(s["pages"], s["tables"], s["full"], s["seen"], case["budget"] + s["longest"],
                            case["budget"], sink=case["sink"], recent=case["recent"])
    return s["key"], s["value"], s["weights"], s["positions"], lengths


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind, h, lengths = case["kind"], case["h"], _lengths(case)
    n, tokens = len(lengths), sum(lengths)
    if kind == "decode":
        rows = tokens * h * (512 + (8 if case["accumulate"] else 0))
        return {"bytes": rows + n * case["hq"] * 512 + 4 * sum(-(-x // case["page"]) for x in lengths),
                "flops": 4 * case["hq"] * 128 * tokens}
    if kind == "prompt":
        # queries, keys, values and output once, weights once; the products of keys and of values once
        return {"bytes": tokens * (case["hq"] * 512 + h * 516),
                "flops": sum(2 * case["hq"] * 128 * x * (x + 1) for x in lengths)}
    if kind == "window":
        W = case["window"]
        pairs = sum(min(W, x) * x - min(W, x) * (min(W, x) - 1) // 2 for x in lengths)
        return {"bytes": tokens * h * 260 + sum(min(W, x) for x in lengths) * case["hq"] * 256,
                "flops": 2 * case["hq"] * 128 * pairs}
    if kind == "select":
        return {"bytes": 4 * h * (tokens + n * case["budget"]), "flops": h * tokens}
    if kind == "write":
        budget = case["budget"]
        rows = sum(min(x, budget) if budget else x for x in lengths) * h
        return {"bytes": rows * (1024 + 12 + (4 if budget else 0)), "flops": rows}
    # the new rows written, their kept copies moved (the newest are kept), weights and positions of all rows read
    rows = tokens * h
    return {"bytes": rows * (1024 + 12) + rows * (1024 + 16) + 8 * h * (n * case["budget"] + tokens),
            "flops": h * (n * case["budget"] + tokens)}


# ------------------------------------------------------------------ 64-bit values

def _weights_of(q, k, v, first):
    """Causal attention of queries [hq, m, 128], the first at key `first`, over keys and values [h, x, 128], in 64 bits:
    output [hq, m, 128] and the keys' summed weights [h, x]."""
    h, x = k.shape[:2]
    g, m = q.shape[0] // h, q.shape[1]
    out, total = torch.empty(q.shape, dtype=torch.float64, device=DEV), torch.zeros((h, x), dtype=torch.float64,
                                                                                    device=DEV)
    for head in range(h):
        kh, vh = k[head].double(), v[head].double()
        for low in range(0, m, 2048):
            high = min(m, low + 2048)
            ahead = torch.arange(x, device=DEV) > first + torch.arange(low, high, device=DEV).unsqueeze(1)
            for one in range(head * g, (head + 1) * g):
                logits = (q[one, low:high].double() @ kh.t().contiguous() * SCALE).masked_fill_(ahead, -math.inf)
                p = torch.softmax(logits, -1)
                out[one, low:high] = p @ vh
                total[head] += p.sum(0)
    return out, total


def _exact_select(weights, first, budget):
    """Kept rows, ascending, of one head, on the host."""
    order = sorted(range(len(weights)), key=lambda i: (not first[i], -weights[i], i))
    return sorted(order[:budget])


def _exact_pages(s, case, sequences):
    """The pools in 64 bits after `sequences` yields (sequence, head, cache row, source row, position) of each write."""
    pools = {name: s[name].double().cpu() for name in ("key", "value", "weights")}
    pools["positions"] = s["positions"].cpu().clone()
    tables, B, cu = s["tables"].cpu().long(), case["page"], s["cu"].cpu().long()
    k, v, w = s["k"].double().cpu(), s["v"].double().cpu(), s["w"].double().cpu()
    for i, head, rows, sources, positions in sequences:
        page, row = tables[i, rows // B], rows % B
        pools["key"][page, head, row] = k[cu[i] + sources, head]
        pools["value"][page, head, row] = v[cu[i] + sources, head]
        pools["weights"][page, head, row] = w[head, cu[i] + sources]
        pools["positions"][page, head, row] = positions.to(torch.int32)
    return pools


def exact(case, seed):
    s = prepare(case, seed)
    kind, h, lengths = case["kind"], case["h"], _lengths(case)
    if kind == "decode":
        out, total = [], s["weights"].double()
        for i, x in enumerate(lengths):
            page, row = _places(s["tables"][i:i + 1], x, case["page"])
            k, v = (s[name][page[0], :, row].transpose(0, 1) for name in ("key", "value"))
            o, w = _weights_of(s["q"][i].unsqueeze(1), k, v, x)
            out.append(o[:, 0])
            total[page[0], :, row] += w.t()
        return (torch.stack(out), total) if case["accumulate"] else torch.stack(out)
    if kind in ("prompt", "window"):
        outs, totals, first = [], [], 0
        for x in lengths:
            m = x if kind == "prompt" else min(x, case["window"])
            q, k, v = (s[name][first:first + x].transpose(0, 1) for name in "qkv")
            o, w = _weights_of(q[:, x - m:], k, v, x - m)
            outs.append(o.transpose(0, 1))
            totals.append(w)
            first += x
        return (torch.cat(outs), torch.cat(totals, 1)) if kind == "prompt" else torch.cat(totals, 1)
    if kind == "select":
        keep, weights, first = torch.full((len(lengths), h, case["budget"]), -1, dtype=torch.int32), s["weights"].cpu(), 0
        for i, x in enumerate(lengths):
            protect = [j < case["sink"] or j >= x - case["recent"] for j in range(x)]
            for head in range(h):
                rows = _exact_select(weights[head, first:first + x].tolist(), protect, case["budget"])
                keep[i, head, :len(rows)] = torch.tensor(rows, dtype=torch.int32)
            first += x
        return keep
    if kind == "write":
        def written():
            for i, x in enumerate(lengths):
                for head in range(h):
                    if case["budget"]:
                        source = s["keep"][i, head].cpu().long()
                        source = source[source >= 0]
                    else:
                        source = torch.arange(x)
                    yield i, head, torch.arange(len(source)), source, source
        pools = _exact_pages(s, case, written())
        return pools["key"], pools["value"], pools["weights"], pools["positions"]
    budget, seen = case["budget"], s["seen"].cpu().long()

    def appended():
        for i, x in enumerate(lengths):
            for head in range(h):
                yield i, head, budget + torch.arange(x), torch.arange(x), seen[i] + torch.arange(x)
    pools = _exact_pages(s, case, appended())
    tables, B = s["tables"].cpu().long(), case["page"]
    for i, x in enumerate(lengths):
        at = torch.arange(budget + x)
        page, row = tables[i, at // B], at % B
        for head in range(h):
            pos = pools["positions"][page, head, row]
            protect = ((pos < case["sink"]) | (pos >= seen[i] + x - case["recent"])).tolist()
            kept = _exact_select(pools["weights"][page, head, row].tolist(), protect, budget)
            stays = set(kept)
            holes = [j for j in range(budget) if j not in stays]
            movers = [j for j in kept if j >= budget]
            to, origin = torch.tensor(holes, dtype=torch.int64), torch.tensor(movers, dtype=torch.int64)
            for pool in pools.values():
                pool[page[to], head, row[to]] = pool[page[origin], head, row[origin]]
    return (pools["key"], pools["value"], pools["weights"], pools["positions"],
            torch.tensor([min(budget, budget + x) for x in lengths], dtype=torch.int32))
