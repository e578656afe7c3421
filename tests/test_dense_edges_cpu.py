"""Calls of the exact-page operators that touch no row, their copies and what they ask for, checked on the host."""
import pytest
import torch

from inquant_vllm import DensePages, dense, write_rows

I32 = torch.int32


@pytest.fixture
def calls(monkeypatch):
    """What would go to the library, with CPU tensors taken for the GPU's."""
    made = []
    monkeypatch.setattr(dense, "_on_gpu", lambda *a: None)
    monkeypatch.setattr(dense, "_call", lambda gpu, name, *args: made.append((name, args)))
    return made


def test_an_empty_selection_writes_nothing(calls):
    pages = DensePages.allocate(4, 16, 2, device="cpu")
    k, cu, table = torch.zeros((3, 2, 128), dtype=torch.bfloat16), torch.tensor([0, 3], dtype=I32), torch.zeros((1, 2), dtype=I32)
    # a tensor without elements has no address, which the library reads as "every row"
    write_rows(k, k, cu, 3, pages, table, keep=torch.zeros((1, 2, 5), dtype=I32)[:, :, :0])
    assert calls == []
    write_rows(k, k, cu, 3, pages, table, keep=torch.zeros((1, 2, 5), dtype=I32)[:, :, :1])
    write_rows(k, k, cu, 3, pages, table)
    assert [name for name, _ in calls] == ["iq_dense_write_from"] * 2
    with pytest.raises(ValueError):
        write_rows(k, k, cu, 3, pages, table, keep=torch.zeros((1, 3, 0), dtype=I32))
