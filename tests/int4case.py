"""4-bit pages in plain form, for the tests of the 4-bit operators: the codes of rows in 64 bits, the pages' bytes one by
one, and the rows that they stand for.  Everything here is on the host."""
import math

import torch

LEAST, MOST = 2.0 ** -14, 2048.0


def coded(x):
    """Codes [..., 128] and words [..., 4] of rows of any floating type, decided in 64 bits."""
    x = x.double().unflatten(-1, (4, 32))
    fine = x.isfinite().all(-1, keepdim=True)
    x = torch.where(fine, x, torch.zeros_like(x))
    low, high = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    mantissa, exponent = torch.frexp(((high - low) / 15).clamp(LEAST, MOST))          # mantissa in [1/2, 1)
    step = torch.ldexp(torch.ceil(mantissa * 64) / 64, exponent)
    zero = torch.round(-low / step).clamp(0, 15)
    code = (torch.round(x / step) + zero).clamp(0, 15)
    word = step.half().view(torch.int16).int() & 0xffff | zero.int()
    word = torch.where(fine, word, torch.full_like(word, 0x7e00)).squeeze(-1)
    return torch.where(fine, code, torch.zeros_like(code)).int().flatten(-2), word


def stands_for(code, word):
    """The rows, in 64 bits."""
    step = (word & 0xffe0).short().view(torch.float16).double()
    return ((code.unflatten(-1, (4, 32)).double() - (word & 15).double().unsqueeze(-1)) * step.unsqueeze(-1)).flatten(-2)


def _places(B):
    """Byte and nibble of the key and the value code [B, 128], and the first byte of their words [B, 4]."""
    r, c, g = torch.arange(B)[:, None], torch.arange(128), torch.arange(4)
    unit = ((r // 4 * 16 + c // 8) * 2 + r // 2 % 2) * 4 + c // 4 % 2 * 2 + r % 2
    nibble = (c % 2).expand(B, 128)
    return [(64 * r + c // 2, nibble, 128 * B + 8 * r + 2 * g),
            (64 * B + 2 * unit + c % 4 // 2, nibble, 136 * B + 2 * (r // 4 * 16 + 4 * g + r % 4))]


def put(page, row, which, code, word):
    """Writes one row's codes and words into a head's part of a page (a uint8 tensor)."""
    byte, nibble, at = (t[row] for t in _places(page.numel() // 144)[which])
    for c in range(128):
        b, shift = int(byte[c]), 4 * int(nibble[c])
        page[b] = int(page[b]) & (0xf0 >> shift) | int(code[c]) << shift
    for g in range(4):
        page[int(at[g])], page[int(at[g]) + 1] = int(word[g]) & 0xff, int(word[g]) >> 8


def fill(pool, keys, values):
    """Pages' bytes [pages, H, B * 144] of rows [pages, H, B, 128], all at once."""
    B = keys.shape[2]
    for which, rows in enumerate((keys, values)):
        code, word = coded(rows)
        byte, nibble, at = _places(B)[which]
        for half in range(2):
            mine = nibble == half
            low = code[..., mine] << 4 * half
            where = byte[mine]
            if half == 0:
                pool[..., where] = low.to(torch.uint8)
            else:
                pool[..., where] |= low.to(torch.uint8)
        pool[..., at], pool[..., at + 1] = (word & 0xff).to(torch.uint8), (word >> 8).to(torch.uint8)
    return pool


def rows_of(pool):
    """Keys and values [pages, H, B, 128] in 64 bits that pages' bytes stand for."""
    B = pool.shape[2] // 144
    out = []
    for byte, nibble, at in _places(B):
        code = pool[..., byte].int() >> 4 * nibble & 15
        out.append(stands_for(code, pool[..., at].int() | pool[..., at + 1].int() << 8))
    return out


def turned(x, angles, interleaved):
    """Rows [tokens, heads, 128] in float32 rotated by [tokens, r] cosines and sines: each product and sum rounded."""
    r = angles.shape[1]
    x = x.float()
    cos, sin = angles[:, None, :r // 2], angles[:, None, r // 2:]
    a, b = (x[..., :r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    a, b = a * cos - b * sin, b * cos + a * sin
    first = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((first, x[..., r:]), -1)


def angles(positions, rotary, base=10000.0):
    step = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * step
    return torch.cat((angle.cos(), angle.sin()), -1).float()


def attend(q, k, v, scale, sees):
    """q [m, 128], k and v [n, 128], query t sees the first sees[t] rows: outputs in 64 bits (zeros where it sees none),
    and a bound on a 32-bit logit's error (any order of 128 products)."""
    q, k, v = q.double(), k.double(), v.double()
    logits = q @ k.t() * scale
    slack = float((q.abs() @ k.abs().t()).max()) * abs(scale) * 130 * 2.0 ** -24 if logits.numel() else 0.0
    hidden = torch.arange(k.shape[0], device=q.device) >= sees[:, None]
    p = logits.masked_fill(hidden, -math.inf).softmax(-1)
    return torch.where((sees > 0)[:, None], torch.where(hidden, torch.zeros_like(p), p) @ v, torch.zeros_like(q)), slack
