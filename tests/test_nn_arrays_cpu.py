"""What xgboost.nn's Python layer makes of the arrays that it is given: their
devices, streams and flags. Without a GPU: tensors are stand-ins with torch's
methods, and what would be handed to the library is recorded instead."""
import sys

import pytest
import torch

import xgboost as xgb
from xgboost import nn


class Tensor:
    """A contiguous CUDA tensor by its methods; nothing reads its memory."""

    is_cuda = True

    def __init__(self, *shape, dtype=torch.float32, device=0, ptr=4096):
        self.shape, self.dtype, self.ordinal, self.ptr = torch.Size(shape), dtype, device, ptr

    def data_ptr(self):
        return self.ptr

    def stride(self):
        return torch.empty(self.shape, device="meta").stride()

    def get_device(self):
        return self.ordinal

    def is_contiguous(self):
        return True

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def element_size(self):
        return self.dtype.itemsize

    def new_empty(self, *shape, dtype=None):
        return Tensor(*shape, dtype=dtype or self.dtype, device=self.ordinal, ptr=1 << 20)


def test_a_workspace_on_another_device_is_refused():
    n = 1 << 14
    g, k = Tensor(n, 2), Tensor(n, dtype=torch.int32)
    space = Tensor(nn.embedding_backward_workspace(n, 1, 4, 2), dtype=torch.uint8, device=1)
    with pytest.raises(xgb.XGBoostError, match="different devices"):
        nn.embedding_backward(g, k, 4, out=Tensor(4, 2, ptr=8192), workspace=space)
    x, stats, w = Tensor(3, 400), Tensor(3), Tensor(400)
    space = Tensor(nn.layer_norm_backward_workspace(3, 400), dtype=torch.uint8, device=1)
    with pytest.raises(xgb.XGBoostError, match="different devices"):
        nn.layer_norm_backward(x, x, stats, stats, w, out=Tensor(3, 400, ptr=8192), dweight=Tensor(400),
                               dbias=Tensor(400), workspace=space)


def test_torch_counts_as_known_only_when_all_of_it_is(monkeypatch):
    """_codes is what other threads look at: nothing may still be missing when it is filled."""
    codes, dtypes = {}, {}
    for name, value in (("_codes", codes), ("_dtypes", dtypes), ("_raw_stream", None), ("_empty_like", None)):
        monkeypatch.setattr(nn, name, value)
    seen = []

    class Torch:
        def __getattr__(self, name):  # where another thread may come in between
            seen.append(name)
            assert not codes or (dtypes and nn._raw_stream and nn._empty_like), name
            return getattr(torch, name)

    monkeypatch.setitem(sys.modules, "torch", Torch())
    nn._know_torch()
    assert "_C" in seen and len(codes) == len(dtypes) == 5 and nn._raw_stream and nn._empty_like
