"""Timed cases of 4-bit pages and of appending with the position rotation.

Five kinds of work:

* ``append``  a step's or a prompt's queries and keys rotated by their positions, keys and values written into exact
              (16-bit) pages;
* ``store``   the same into 4-bit pages, and the rows just written read back as 16-bit rows (what is held in 4 bits
              shows as the values it stands for);
* ``read``    rows of 4-bit pages as token-major 16-bit rows;
* ``decode``  one token's attention for a batch of sequences over 4-bit pages;
* ``chunk``   the attention of the last few to many tokens of each sequence over 4-bit pages.

Keys and values are N(0, 1) with about 4% of the channels of each head's keys, in runs of two and one, times 20.  Pages
sit at random places of a pool that is an eighth larger than what they need.

A 4-bit page holds, for each of its heads, the codes of ``page`` rows of keys (64 bytes each, two channels a byte, the
lower one first), those of the values, and a word per row and group of 32 channels for either.  The values' codes
interleave four rows: 16-bit units of four channels, [row / 4][channel / 8][row / 2 % 2][channel / 4 % 2][row % 2].  The
keys' words are [row][group], the values' [row / 4][group][row % 4].  A word is the f16 pattern of the step s, whose five
low bits are zero but for the zero point z in the lowest four: code n stands for (n - z) s.  Over a group's values and 0,
s is a 15th of their range within 2^-14 .. 2048, rounded up to six significant bits, z = rint(-lowest / s), and
n = rint(x / s) + z, both within 0 .. 15.  A group with an infinity or a NaN stands for NaN.
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
GROUP = 32
LEAST, MOST = 2.0 ** -14, 2048.0
BASE = 1000000.0


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # a decode step of 16 requests: one new token each, some thousand rows in their exact pages
        {"name": "append_step", "kind": "append", "hq": 28, "h": 4, "page": 16, "seqs": 16, "low": 1, "high": 1,
         "before": 3000, "rotary": 128, "interleaved": False, "dtype": "bf16"},
        # every row of a ragged batch of prompts, a rotation of half the channels in neighbouring pairs
        {"name": "append_ragged", "kind": "append", "hq": 32, "h": 8, "page": 64, "seqs": 7, "low": 37, "high": 16384,
         "before": 0, "rotary": 64, "interleaved": True, "dtype": "f16"},
        # the decode step into 4-bit pages
        {"name": "store_step", "kind": "store", "hq": 28, "h": 4, "page": 16, "seqs": 16, "low": 1, "high": 1,
         "before": 3000, "rotary": 128, "interleaved": False, "factors": True, "dtype": "bf16"},
        # a batch of prompts into 4-bit pages
        {"name": "store_ragged", "kind": "store", "hq": 28, "h": 4, "page": 16, "seqs": 7, "low": 37, "high": 16384,
         "before": 0, "rotary": 128, "interleaved": False, "factors": False, "dtype": "bf16"},
        # a short shared prefix read back
        {"name": "read_600", "kind": "read", "h": 4, "page": 16, "seqs": 2, "low": 300, "high": 300, "dtype": "bf16"},
        # eight long prefixes
        {"name": "read_ragged", "kind": "read", "h": 8, "page": 256, "seqs": 8, "low": 5000, "high": 32768,
         "dtype": "f16"},
        # one layer of one short chat: the smallest call, where launches and the host count
        {"name": "decode_300", "kind": "decode", "hq": 28, "h": 4, "page": 16, "seqs": 1, "low": 300, "high": 300,
         "dtype": "bf16"},
        # a serving step of 16 requests between 2K and 32K tokens
        {"name": "decode_16seq", "kind": "decode", "hq": 28, "h": 4, "page": 16, "seqs": 16, "low": 2048,
         "high": 32768, "dtype": "bf16"},
        # two long documents, eight KV heads
        {"name": "decode_2x128k", "kind": "decode", "hq": 32, "h": 8, "page": 256, "seqs": 2, "low": 129000,
         "high": 131072, "dtype": "f16"},
        # five drafted tokens of eight requests
        {"name": "draft_8seq", "kind": "chunk", "hq": 28, "h": 4, "page": 16, "seqs": 8, "low": 1000, "high": 16384,
         "least": 5, "tokens": 5, "dtype": "bf16"},
        # the last 2048 tokens of a 32K prompt
        {"name": "chunk_32k", "kind": "chunk", "hq": 28, "h": 4, "page": 16, "seqs": 1, "low": 32768, "high": 32768,
         "least": 2048, "tokens": 2048, "dtype": "bf16"},
        # chunks of several prompts, some of one token
        {"name": "chunk_ragged", "kind": "chunk", "hq": 32, "h": 8, "page": 64, "seqs": 5, "low": 2100, "high": 9000,
         "least": 1, "tokens": 2048, "dtype": "f16"},
    ]


HEADS = [(28, 4), (32, 8), (16, 2), (8, 8), (14, 2), (12, 1), (16, 1)]
PAGES = [16, 16, 32, 64, 128, 256]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "store", "read", "decode", "decode", "chunk", "chunk"])
    hq, h = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    case = {"kind": kind, "h": h, "page": rng.choice(PAGES), "dtype": dtype}
    if kind == "read":
        seqs = _log(rng, 1, 16)
        high = _log(rng, 1, min(32768, 1200000 // (seqs * h)))
        return {**case, "seqs": seqs, "low": max(1, high // rng.choice([1, 3, 20])), "high": high}
    case["hq"] = hq
    if kind in ("append", "store"):
        seqs = _log(rng, 1, 16)
        high = rng.choice([1, _log(rng, 1, min(16384, 1500000 // (seqs * hq)))])
        case.update(seqs=seqs, low=max(1, high // rng.choice([1, 2, 10])), high=high,
                    before=rng.choice([0, _log(rng, 1, 4000)]), rotary=rng.choice([128, 128, 64, 96, 32]),
                    interleaved=rng.random() < 0.3)
        if kind == "store":
            case["factors"] = rng.random() < 0.5
        return case
    if kind == "decode":
        seqs = _log(rng, 1, 64)
        high = _log(rng, 1, min(131072, 2000000 // (seqs * h)))
        return {**case, "seqs": seqs, "low": max(1, high // rng.choice([1, 3, 20])), "high": high}
    seqs = rng.choice([1, 1, 2, 4, 9])
    tokens = _log(rng, 2, 2048)
    # logits of one pass in their plain form: up to 1.8e9
    high = _log(rng, max(8, tokens // 2), max(tokens, min(40000, int(1.8e9 / (seqs * hq * tokens)))))
    return {**case, "seqs": seqs, "low": max(1, high // rng.choice([1, 2, 10])), "high": high,
            "least": max(1, tokens // rng.choice([1, 4, 2048])), "tokens": tokens}


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """The sequences' rows (``append`` and ``store``: their new ones), part of the case: the same for every seed."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["low"], case["high"]))
    return [rng.randint(case["low"], case["high"]) for _ in range(case["seqs"])]


def _starts(case):
    rng = random.Random("%d %d" % (case["seqs"], case["before"]))
    return [rng.randint(case["before"] // 3, case["before"]) for _ in range(case["seqs"])]


def _asked(case, lengths):
    """The query tokens of each sequence: the last ones of its rows."""
    rng = random.Random("%d %d" % (case["least"], case["tokens"]))
    return [min(x, rng.randint(case["least"], case["tokens"])) for x in lengths]


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


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).to(DEV)


def _offsets(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return _i32(total)


def _tables(gen, case, rows):
    """Block tables of sequences of `rows` rows, and the pages of the pool."""
    width = [-(-n // case["page"]) for n in rows]
    used = sum(width)
    pages = used + used // 8 + 1
    at = torch.randperm(pages, generator=gen, device=DEV)[:used].to(torch.int32)
    tables = torch.full((len(rows), max(width)), -1, dtype=torch.int32, device=DEV)
    first = 0
    for i, n in enumerate(width):
        tables[i, :n] = at[first:first + n]
        first += n
    return tables, pages


def _coded_pool(gen, gain, case, pages):
    """A pool of 4-bit pages that hold random rows, some pages at a time."""
    h, B = case["h"], case["page"]
    pool = torch.empty((pages, h, B * 144), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 18) // (h * B))
    for low in range(0, pages, step):
        n = min(step, pages - low)
        key, value = _randn(gen, n, h, B, 128) * gain, _randn(gen, n, h, B, 128)
        part = [_key_bytes(*_codes(key)), _value_bytes(*_codes(value))]
        pool[low:low + n] = torch.cat((part[0][0], part[1][0], part[0][1], part[1][1]), -1)
    return pool


def _angles(positions, rotary):
    """cos | sin of the positions' angles, made in 64 bits, float32 [positions, rotary]."""
    step = BASE ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEV) / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * step
    return torch.cat((angle.cos(), angle.sin()), -1).float()


def prepare(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    kind, h, lengths, dtype = case["kind"], case["h"], _lengths(case), DTYPES[case["dtype"]]
    n, B = len(lengths), case["page"]
    gain = _gain(rng, h)
    state = {"case": case}
    if kind in ("append", "store"):
        starts, tokens = _starts(case), sum(lengths)
        tables, pages = _tables(gen, case, [a + x for a, x in zip(starts, lengths)])
        # the projections of one product side by side, as a model has them
        both = _randn(gen, tokens, case["hq"] + 2 * h, 128)
        both[:, case["hq"]:case["hq"] + h] *= gain[:, 0]
        both = both.to(dtype)
        state.update(q=both[:, :case["hq"]], k=both[:, case["hq"]:case["hq"] + h], v=both[:, case["hq"] + h:],
                     cu=_offsets(lengths), longest=max(lengths), start=_i32(starts), tables=tables,
                     angles=_angles(max(a + x for a, x in zip(starts, lengths)), case["rotary"]), factors=None)
        state["out"] = torch.empty((tokens, case["hq"], 128), dtype=dtype, device=DEV)
        if kind == "append":
            state.update(key=torch.zeros((pages, h, B, 128), dtype=dtype, device=DEV),
                         value=torch.zeros((pages, h, B, 128), dtype=dtype, device=DEV))
        else:
            state["pool"] = torch.zeros((pages, h, B * 144), dtype=torch.uint8, device=DEV)
            state["rows"] = [torch.empty((tokens, h, 128), dtype=dtype, device=DEV) for _ in range(2)]
            if case["factors"]:
                # what a calibration leaves: the keys' channels brought to about one size
                state["factors"] = gain[:, 0] * (0.9 + 0.2 * torch.rand((h, 128), generator=gen, device=DEV))
    else:
        tables, pages = _tables(gen, case, lengths)
        state.update(pool=_coded_pool(gen, gain, case, pages), tables=tables, lengths=_i32(lengths),
                     longest=max(lengths))
        if kind == "read":
            state.update(cu=_offsets(lengths))
            state["rows"] = [torch.empty((sum(lengths), h, 128), dtype=dtype, device=DEV) for _ in range(2)]
        else:
            asked = [1] * n if kind == "decode" else _asked(case, lengths)
            state["q"] = _randn(gen, sum(asked), case["hq"], 128).to(dtype)
            state["out"] = torch.empty_like(state["q"])
            state.update(cu=_offsets(asked), most=max(asked))
    if own:
        from inquant.triton_attention import SharedDecodeWorkspace
        from inquant_vllm import DensePages, Int4Pages
        state["pages"] = Int4Pages(state["pool"]) if "pool" in state else DensePages(state["key"], state["value"])
        state["workspace"] = SharedDecodeWorkspace()
    return state


# ------------------------------------------------------------------ plain forms

def _codes(x):
    """Codes [..., 128] and words [..., 4] (int16) of rows of float32; 64 bits decide what lies next to a border."""
    group = x.unflatten(-1, (4, GROUP))
    fine = group.isfinite().all(-1, keepdim=True)
    group = group.double().masked_fill_(~fine, 0)
    low, high = group.amin(-1, keepdim=True).clamp_(max=0), group.amax(-1, keepdim=True).clamp_(min=0)
    step = (high - low).div_(torch.full_like(high, 15)).clamp_(LEAST, MOST)
    # up to six significant bits: 47 of a double's 52 go
    step = ((step.view(torch.int64) + ((1 << 47) - 1)) & -(1 << 47)).view(torch.float64)
    zero = (-low / step).round_().clamp_(0, 15)
    code = (group / step).round_().add_(zero).clamp_(0, 15).to(torch.uint8).flatten(-2)
    word = step.half().view(torch.int16) | zero.to(torch.int16)
    return code, word.masked_fill_(~fine, 0x7e00).squeeze(-1)


def _key_bytes(code, word):
    """Bytes of the keys of pages [..., B, 128]: codes [..., 64 B] and words [..., 8 B]."""
    pair = code.unflatten(-1, (64, 2))
    return (pair[..., 0] | pair[..., 1] << 4).flatten(-2), word.view(torch.uint8).flatten(-2)


def _value_bytes(code, word):
    pair = code.unflatten(-1, (64, 2))
    byte = (pair[..., 0] | pair[..., 1] << 4).unflatten(-1, (16, 2, 2)).unflatten(-4, (-1, 2, 2))
    # [..., quad, pair, row, eight channels, half, byte] -> [..., quad, eight channels, pair, half, row, byte]
    byte = byte.movedim((-5, -4, -3, -2), (-4, -2, -5, -3)).contiguous()
    return byte.flatten(-6), word.unflatten(-2, (-1, 4)).transpose(-1, -2).contiguous().view(torch.uint8).flatten(-3)


def _steps(word):
    """Steps and zero points of words."""
    return (word & -32).view(torch.float16).float(), (word & 15).float()


def _nibbles(byte):
    return torch.stack((byte & 15, byte >> 4), -1).flatten(-2)


def _unpacked(pool, B):
    """Float32 keys and values [..., B, 128] that heads of pages [..., 144 B] stand for."""
    code = [_nibbles(pool[..., 64 * B * i:64 * B * (i + 1)]) for i in range(2)]
    word = [pool[..., (128 + 8 * i) * B:(136 + 8 * i) * B].contiguous().view(torch.int16) for i in range(2)]
    key = code[0].unflatten(-1, (B, 4, GROUP))
    # [..., quad, eight channels, pair, half, row, four channels] -> [..., quad, pair, row, eight channels, half, ...]
    value = code[1].unflatten(-1, (B // 4, 16, 2, 2, 2, 4)).movedim((-5, -4, -3, -2), (-3, -5, -2, -4))
    value = value.flatten(-3).unflatten(-1, (4, GROUP)).flatten(-5, -3)
    out = []
    for n, w in ((key, word[0].unflatten(-1, (B, 4))),
                 (value, word[1].unflatten(-1, (B // 4, 4, 4)).transpose(-1, -2).flatten(-3, -2))):
        step, zero = _steps(w.unsqueeze(-1))
        out.append((n.float() - zero).mul_(step).flatten(-2))
    return out


def _rotated(x, angles, interleaved):
    """Rows [tokens, heads, 128] in float32, rotated by their tokens' angles [tokens, rotary]."""
    r = angles.shape[-1]
    x = x.float()
    cos, sin = (t.unsqueeze(1) for t in angles.split(r // 2, -1))
    a, b = (x[..., :r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, x[..., r:]), -1)


def _tokens(s):
    """Sequence and place of every new token, and its page and row in the page."""
    cu = s["cu"].long()
    token = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(cu, token, right=True) - 1
    row = s["start"].long()[seq] + token - cu[seq]
    B = s["case"]["page"]
    return row, s["tables"][seq, row // B].long(), row % B


def _append(s):
    case = s["case"]
    row, page, at = _tokens(s)
    angles, heads = s["angles"][row], torch.arange(case["h"], device=DEV)
    q, k = (_rotated(s[x], angles, case["interleaved"]) for x in "qk")
    if s["factors"] is not None:
        q = q.unflatten(1, (case["h"], -1)).mul_(s["factors"].unsqueeze(1)).flatten(1, 2)
        k = k / s["factors"]
    s["out"].copy_(q)
    if case["kind"] == "append":
        where = (page[:, None], heads, at[:, None])
        s["key"][where] = k.to(s["key"].dtype)
        s["value"][where] = s["v"]
        return s["out"], s["key"], s["value"]
    B = case["page"]
    pool = s["pool"]
    parts = [pool[..., :64 * B].unflatten(-1, (B, 64)), pool[..., 64 * B:128 * B].unflatten(-1, (B // 4, 16, 2, 2, 2, 2)),
             pool[..., 128 * B:136 * B].unflatten(-1, (B, 4, 2)), pool[..., 136 * B:].unflatten(-1, (B // 4, 4, 4, 2))]
    code, word = _codes(k)
    pair = code.unflatten(-1, (64, 2))
    p, r, hh = page[:, None], at[:, None], heads
    parts[0][p, hh, r] = pair[..., 0] | pair[..., 1] << 4
    parts[2][p, hh, r] = word.unsqueeze(-1).view(torch.uint8)
    code, word = _codes(s["v"].float())
    pair = code.unflatten(-1, (64, 2))
    eight, half = torch.arange(16, device=DEV)[:, None], torch.arange(2, device=DEV)
    p, r, hh = page[:, None, None, None], at[:, None, None, None], heads[:, None, None]
    parts[1][p, hh, r // 4, eight, r // 2 % 2, half, r % 2] = (pair[..., 0] | pair[..., 1] << 4).unflatten(-1, (16, 2, 2))
    p, r, hh = page[:, None, None], at[:, None, None], heads[:, None]
    parts[3][p, hh, r // 4, torch.arange(4, device=DEV), r % 4] = word.unsqueeze(-1).view(torch.uint8)
    rows = _rows_of(s, page, at)
    for out, x in zip(s["rows"], rows):
        out.copy_(x)
    return s["out"], s["rows"][0], s["rows"][1]


def _rows_of(s, page, at):
    """Keys and values [tokens, heads, 128] of one row of one page for each token, in float32."""
    B, pool = s["case"]["page"], s["pool"]
    h, p, r = torch.arange(s["case"]["h"], device=DEV), page[:, None], at[:, None]
    key = _nibbles(pool[..., :64 * B].unflatten(-1, (B, 64))[p, h, r])
    value = pool[..., 64 * B:128 * B].unflatten(-1, (B // 4, 16, 2, 2, 2, 2))
    eight, half = torch.arange(16, device=DEV)[:, None], torch.arange(2, device=DEV)
    p4, r4, h4 = page[:, None, None, None], at[:, None, None, None], h[:, None, None]
    value = _nibbles(value[p4, h4, r4 // 4, eight, r4 // 2 % 2, half, r4 % 2].flatten(-3))
    words = [pool[..., 128 * B:136 * B].unflatten(-1, (B, 4, 2))[p, h, r],
             pool[..., 136 * B:].unflatten(-1, (B // 4, 4, 4, 2))[
                 p[..., None], h[:, None], r[..., None] // 4, torch.arange(4, device=DEV), r[..., None] % 4]]
    out = []
    for code, w in ((key, words[0]), (value, words[1])):
        step, zero = _steps(w.contiguous().view(torch.int16))
        out.append((code.unflatten(-1, (4, GROUP)).float() - zero).mul_(step).flatten(-2))
    return out


def _read(s):
    cu, B = s["cu"].long(), s["case"]["page"]
    token = torch.arange(s["rows"][0].shape[0], device=DEV)
    seq = torch.searchsorted(cu, token, right=True) - 1
    row = token - cu[seq]
    for out, x in zip(s["rows"], _rows_of(s, s["tables"][seq, row // B].long(), row % B)):
        out.copy_(x)
    return s["rows"][0], s["rows"][1]


def _attention(s):
    case, longest, m = s["case"], s["longest"], s["most"]
    n, h, g, B = case["seqs"], case["h"], case["hq"] // case["h"], case["page"]
    cols = -(-longest // B)
    k, v = _unpacked(s["pool"][s["tables"][:, :cols].long().clamp_(min=0)], B)     # [n, cols, h, B, 128]
    k, v = (x.transpose(1, 2).reshape(n, h, cols * B, 128)[:, :, :longest] for x in (k, v))
    # the query tokens, m for each sequence: those past its own repeat its last one
    cu = s["cu"].long()
    at = torch.minimum(cu[:-1, None] + torch.arange(m, device=DEV), cu[1:, None] - 1)
    q = s["q"][at].float().transpose(1, 2).reshape(n, h, g * m, 128)
    sees = s["lengths"][:, None] - cu[1:, None] + at                               # [n, m]: the last row of each
    p = (q @ k.transpose(-1, -2)).mul_(SCALE).view(n, h, g, m, longest)
    p.masked_fill_((torch.arange(longest, device=DEV) > sees[..., None])[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    o = (p.view(n, h, g * m, longest) @ v).view(n, h * g, m, 128).transpose(1, 2)
    real = torch.arange(m, device=DEV) < (cu[1:] - cu[:-1])[:, None]
    s["out"].copy_(o[real])
    return s["out"]


# ------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"append": _append, "store": _append, "read": _read, "decode": _attention, "chunk": _attention}[kind](s)
    import inquant_vllm as iv
    if kind in ("append", "store"):
        out = iv.append_rows(s["q"], s["k"], s["v"], s["cu"], s["longest"], s["pages"], s["tables"], s["start"],
                             rotation=s["angles"], interleaved=case["interleaved"], factors=s["factors"], output=s["out"])
        if kind == "append":
            return out, s["key"], s["value"]
        iv.read_rows(s["pages"], s["tables"], s["cu"], s["longest"], *s["rows"], s["start"])
        return out, s["rows"][0], s["rows"][1]
    if kind == "read":
        return iv.read_rows(s["pages"], s["tables"], s["cu"], s["longest"], *s["rows"])
    if kind == "decode":
        return iv.int4_decode(s["q"], s["pages"], s["tables"], s["lengths"], s["longest"], SCALE, s["workspace"],
                              s["out"])
    return iv.int4_attention(s["q"], s["cu"], s["most"], s["pages"], s["tables"], s["lengths"], s["longest"], SCALE,
                             s["workspace"], s["out"])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind, h, lengths = case["kind"], case["h"], _lengths(case)
    tokens = sum(lengths)
    if kind in ("append", "store"):
        # queries read and written, keys and values read; rows of 512 or 144 bytes written; 144 and 512 to read back
        rows = h * tokens * (512 + 512 if kind == "append" else 512 + 144 + 144 + 512)
        return {"bytes": tokens * case["hq"] * 512 + rows, "flops": 3 * tokens * (case["hq"] + h) * case["rotary"]}
    if kind == "read":
        return {"bytes": tokens * h * (144 + 512), "flops": 2 * tokens * h * 256}
    asked = [1] * len(lengths) if kind == "decode" else _asked(case, lengths)
    pairs = sum(m * x - m * (m - 1) // 2 for x, m in zip(lengths, asked))
    return {"bytes": tokens * h * 144 + sum(asked) * case["hq"] * 512 + 4 * sum(-(-x // case["page"]) for x in lengths),
            "flops": 4 * case["hq"] * 128 * pairs}


# ------------------------------------------------------------------ 64-bit values

def _held(x):
    """What 4 bits hold of rows [..., 128], in 64 bits."""
    x = x.double()
    out = torch.empty_like(x)
    for g in range(4):
        part = x[..., 32 * g:32 * g + 32]
        low = torch.minimum(part.min(-1, keepdim=True).values, torch.zeros((), dtype=x.dtype, device=DEV))
        high = torch.maximum(part.max(-1, keepdim=True).values, torch.zeros((), dtype=x.dtype, device=DEV))
        wide = ((high - low) / 15).clamp(LEAST, MOST)
        mantissa, exponent = torch.frexp(wide)                                # mantissa in [1/2, 1)
        step = torch.ldexp(torch.ceil(mantissa * 64) / 64, exponent)
        zero = torch.round(-low / step).clamp(0, 15)
        out[..., 32 * g:32 * g + 32] = ((torch.round(part / step) + zero).clamp(0, 15) - zero) * step
    return out


def _turned(x, angles, interleaved):
    """Rows [tokens, heads, 128] rotated in 64 bits, as a product with each pair's complex number."""
    r = angles.shape[-1]
    x, angles = x.double().clone(), angles.double()
    turn = torch.complex(angles[:, :r // 2], angles[:, r // 2:]).unsqueeze(1)
    first = torch.arange(0, r, 2, device=DEV) if interleaved else torch.arange(r // 2, device=DEV)
    second = first + (1 if interleaved else r // 2)
    z = torch.complex(x[..., first], x[..., second]) * turn
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _stands_for(s, i, rows):
    """Keys and values [h, rows, 128] of sequence i in 64 bits, nibble by nibble."""
    B, pool = s["case"]["page"], s["pool"]
    r, c = torch.arange(rows, device=DEV)[:, None], torch.arange(128, device=DEV)
    page = s["tables"][i, (r // B).flatten()].long()[:, None]
    r = r % B
    places = (r * 64 + c // 2, c % 2,
              64 * B + 2 * ((((r // 4 * 16 + c // 8) * 2 + r % 4 // 2) * 2 + c % 8 // 4) * 2 + r % 2) + c % 4 // 2, c % 2)
    words = (128 * B + 2 * (r * 4 + c // 32), 136 * B + 2 * (r // 4 * 16 + c // 32 * 4 + r % 4))
    out = []
    for part in range(2):
        heads = []
        for head in range(pool.shape[1]):
            code = pool[page, head, places[2 * part]].long() >> 4 * places[2 * part + 1] & 15
            word = pool[page, head, words[part]].long() | pool[page, head, words[part] + 1].long() << 8
            step = torch.ldexp(1 + (word >> 5 & 31).double() / 32, (word >> 10) - 15)
            heads.append((code - (word & 15)).double() * step)
        out.append(torch.stack(heads))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind, lengths = case["kind"], _lengths(case)
    if kind in ("append", "store"):
        starts, first, q, k = _starts(case), 0, [], []
        for a, x in zip(starts, lengths):
            for name, rows in (("q", q), ("k", k)):
                rows.append(_turned(s[name][first:first + x], s["angles"][a:a + x], case["interleaved"]))
            first += x
        q, k, v = torch.cat(q), torch.cat(k), s["v"].double()
        if s["factors"] is not None:
            f = s["factors"].double()
            q, k = q * f.repeat_interleave(case["hq"] // case["h"], 0), k / f
        if kind == "store":
            return q, _held(k), _held(v)
        pools, first = [s[name].double() for name in ("key", "value")], 0
        for i, (a, x) in enumerate(zip(starts, lengths)):
            row = torch.arange(a, a + x, device=DEV)
            page = s["tables"][i, row // case["page"]].long()
            for pool, rows in zip(pools, (k, v)):
                pool[page, :, row % case["page"]] = rows[first:first + x]
            first += x
        return q, pools[0], pools[1]
    if kind == "read":
        keys, values = zip(*(_stands_for(s, i, x) for i, x in enumerate(lengths)))
        return tuple(torch.cat(rows, 1).transpose(0, 1).contiguous() for rows in (keys, values))
    g, outs, first = case["hq"] // case["h"], [], 0
    for i, (x, m) in enumerate(zip(lengths, [1] * len(lengths) if kind == "decode" else _asked(case, lengths))):
        k, v = _stands_for(s, i, x)
        out = torch.empty((m, case["hq"], 128), dtype=torch.float64, device=DEV)
        ahead = torch.arange(x, device=DEV) > x - m + torch.arange(m, device=DEV)[:, None]
        for head in range(case["hq"]):
            q = s["q"][first:first + m, head].double()
            logits = (q @ k[head // g].t().contiguous() * SCALE).masked_fill_(ahead, -math.inf)
            out[:, head] = torch.softmax(logits, -1) @ v[head // g]
        outs.append(out)
        first += m
    return torch.cat(outs)
