"""Edges of the 4-bit pages' operators on the host: scratch of padded batches."""
import ctypes
import itertools

from inquant import _native as nat


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
