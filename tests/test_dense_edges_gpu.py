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
