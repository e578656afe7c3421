"""Edges of the 4-bit pages' operators on the host: scratch of padded batches."""
import ctypes
import itertools

import pytest
import torch

from inquant import _native as nat
from inquant_vllm import Int4Pages, append_rows, read_rows


def test_rows_of_no_sequence_take_no_scratch():
    """What a call can ask for goes with the sequences' tokens: a padded tensor of queries adds none.  Many columns: 256
    workgroups' columns at most, 256 each.  Few: parts of 32 columns by workgroup and by sequence (64 a launch) of every
    plane, a KV head and 32 of its columns: eight planes a head, whose workgroups are 512 and one more a plane at most, or
    two beside many columns, where a head has as many workgroups and so each of its planes."""
    floats = nat.lib().iq_int4_workspace_floats
    for (hq, h), n, most, tokens, rows in itertools.product([(28, 4), (32, 8), (16, 1), (8, 8)], [1, 2, 16], [64, 300, 512, 2048],
                                                            [2048, 8192, 65536], [600, 4096, 32768, 1 << 20]):
        few = max(512 + 65 * 8 * h, 2 * 512 + 65 * 2 * h) * 32 * 130
        assert floats(hq, h, n, tokens, most, rows) <= max(256 * 256 * 130, few), (hq, h, n, most, tokens, rows)
    alone = floats(28, 4, 1, 512, 512, 32768)
    assert 0 < alone == floats(28, 4, 1, 8192, 512, 32768) == floats(28, 4, 1, 1 << 20, 512, 32768)


def test_rows_of_no_sequence_do_not_change_how_short_sequences_are_answered():
    """A chunk beside single tokens: their rows are shared out, which takes scratch, whatever stands behind the batch."""
    floats = nat.lib().iq_int4_workspace_floats
    alone = floats(28, 4, 32, 80000, 2048, 32768)                                        # many columns are not split there
    for most, tokens in ((2048, 2048 + 31), (512, 512 + 31), (2048, 31 * 2048 + 9), (512, 80000)):
        assert floats(28, 4, 32, tokens, most, 32768) >= alone > 0


def test_a_workspace_off_its_alignment_is_refused():
    """Partials are read and written sixteen bytes at a time."""
    lib, fake = nat.lib(), 1 << 20
    pages = nat.Int4PagesDesc(pool=fake, s_page=2 * 2304, s_head=2304, pages=4, heads=2, block_tokens=16)
    need = lib.iq_int4_workspace_floats(4, 2, 1, 3, 3, 1000)
    assert need > 0
    for off in (4, 8):
        assert lib.iq_int4_attention(fake, nat.IQ_BF16, 512, 128, 4, fake, 1, 3, 3, ctypes.addressof(pages), fake, 64, 64, fake, 1000, 0.1,
                                     fake + off, need, fake, 512, 128, nat.IQ_BF16, None) == -1
        assert b"aligned" in lib.iq_last_error()


def test_rows_side_by_side_within_a_head(monkeypatch):
    """One projection [tokens, heads, 3 x 128], or [tokens, heads, 2, 128] for what is read back: rows between each other's
    rows, none of which share memory.  What does share it is still refused."""
    import inquant_vllm.int4 as int4
    monkeypatch.setattr(int4, "_on_gpu", lambda *a: None)
    monkeypatch.setattr(int4, "_call", lambda *a: None)
    cu, table = torch.tensor([0, 3], dtype=torch.int32), torch.zeros((1, 2), dtype=torch.int32)
    pages = Int4Pages.allocate(4, 16, 2, device="cpu")
    for tokens in (1, 3):
        q, k, v = torch.zeros((tokens, 2, 3 * 128), dtype=torch.bfloat16).split(128, 2)
        assert append_rows(q, k, v, cu, 3, pages, table, output=q) is q
        for wide in (2, 5):                                                  # and gaps behind a token's heads
            both = torch.zeros((tokens, wide, 2, 128))[:, :2]
            read_rows(pages, table, cu, 3, both[:, :, 0], both[:, :, 1])
        turned = torch.zeros((2, tokens, 3, 128), dtype=torch.bfloat16).transpose(0, 1)  # heads outside
        assert append_rows(turned[:, :, 0], turned[:, :, 1], turned[:, :, 2], cu, 3, pages, table, output=turned[:, :, 0]) is not None
        flat = torch.zeros((tokens, 2, 4 * 128), dtype=torch.bfloat16)
        for at in (0, 64, 120, 192, 312, 320):                               # outputs that reach into keys or values
            with pytest.raises(ValueError, match="share no memory"):
                append_rows(flat[..., 384:], flat[..., :128], flat[..., 192:320], cu, 3, pages, table,
                            output=flat[..., at:at + 128])
        both = torch.zeros((tokens, 2, 256))
        for at in (0, 8, 64, 120):
            with pytest.raises(ValueError, match="overlap"):
                read_rows(pages, table, cu, 3, both[..., :128], both[..., at:at + 128])


def test_overlaps_as_they_are():
    """Rows that are taken to be apart are apart: every byte compared."""
    import random
    import inquant_vllm.int4 as int4
    rng, apart = random.Random(5), 0
    for _ in range(20000):
        n, size = rng.randint(1, 3), rng.choice([2, 4])
        x, y = ((n, rng.randint(1, 3), *(rng.choice([8, 64, 128, 136, 256, 384, 512, 768, 1152]) for _ in range(2)),
                 16 * rng.randint(0, 400)) for _ in range(2))
        if rng.random() < 0.6:
            y = (*y[:2], *x[2:4], y[4])
        rows = [{at + size * (t * st + h * sh) for t in range(n) for h in range(heads)} for n, heads, st, sh, at in (x, y)]
        meet = any(abs(a - b) < 128 * size for a in rows[0] for b in rows[1])
        if not int4._overlap(x, y, size):
            assert not meet, (x, y, size)
            apart += 1
    assert apart > 2000
