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
