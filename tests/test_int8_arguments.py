"""What products in 8 bits hand their kernels of the tokens' layout."""
import types

import pytest
import torch

from leone_b200.ops.int8 import Int8Matrix, Int8Products, PerThread


def _step(x, monkeypatch):
    """Elements between the rows of ``x`` as its kernel gets them."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    got = []
    products = Int8Products.__new__(Int8Products)
    products.ops = types.SimpleNamespace(_stream=lambda: 0, status=None, device=torch.device("cpu"))
    products.calls = types.SimpleNamespace(leone_linear_i8=lambda *args: got.append(args) or 0)
    products.sm_count, products.plans, products.buffers = 148, {}, PerThread()
    w = Int8Matrix(torch.zeros((32, x.shape[1]), dtype=torch.int8), torch.zeros(32))
    assert products.run(x, w, torch.zeros((x.shape[0], 32)), 1, None, None) == 2
    return got[0][2]


def test_elements_between_rows(monkeypatch):
    x = torch.zeros((3, 64))
    assert _step(x, monkeypatch) == 64 and _step(x[:, :48], monkeypatch) == 64
    assert _step(x[:1].expand(5, 64), monkeypatch) == 0
    # of one row there is nothing between
    assert _step(x.flatten().as_strided((1, 48), (7, 1)), monkeypatch) == 48
    far = torch.empty(1, device="meta").as_strided((2, 64), (1 << 32, 1))
    with pytest.raises(OverflowError, match="apart"):
        _step(far, monkeypatch)
    assert _step(far[:1], monkeypatch) == 64
