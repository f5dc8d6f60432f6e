"""What xgboost.nn's Python layer makes of the arrays that it is given: their
devices, streams and flags. Without a GPU: tensors are stand-ins with torch's
methods, and what would be handed to the library is recorded instead."""
import os
import re
import struct
import subprocess
import sys

import numpy as np
import pytest
import torch

import xgboost as xgb
from xgboost import nn


class Tensor:
    """A contiguous CUDA tensor by its methods; nothing reads its memory."""

    is_cuda, requires_grad = True, False

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


class Array:
    """A device array by its interface alone; nothing reads its memory."""

    def __init__(self, *shape, typestr="<f4", ptr=1 << 16, read_only=False, **more):
        self.__cuda_array_interface__ = {"data": (ptr, read_only), "shape": shape, "typestr": typestr, "version": 3,
                                         **more}


@pytest.fixture
def enqueued(monkeypatch):
    """The library's calls in their order, (name, arguments), none of which is made. Torch's current stream is 77."""
    calls = []
    nn._codes or nn._know_torch()
    monkeypatch.setattr(nn, "_call", lambda function, args: calls.append((function.__name__, args)))
    monkeypatch.setattr(nn, "_raw_stream", lambda device: 77)
    return calls


FORMS = {"XGBBEmbedding": ("PPQQqqqqifPPPQQqqiii4x", 12), "XGBBEmbeddingBackward": ("PPQQqqqqifPPPPNQQqqiiii", 13),
         "XGBBEmbeddingScaleBackward": ("PPQQqqqqifPPPPQQqqiii4x", 13), "XGBBLayerNorm": ("PPPPPPPQQqqiiif", 6),
         "XGBBLayerNormBackward": ("PPPPPPPPPPNQQqqqiii4x", 9)}


def _stream(call):
    form, at = FORMS[call[0]]
    return struct.unpack("@" + form, call[1])[at]


def _calls(kind, at, own={}, **more):
    """Every operator with arrays of which all are plain but number `at`: a tensor of the given kind, or an array whose
    interface has `own`."""
    def make(i, *shape, typestr="<f4", dtype=torch.float32):
        if i == at and kind is not Array:
            return kind(*shape, dtype=dtype)
        return Array(*shape, typestr=typestr, ptr=(i + 1) << 16, **(own if i == at else {}))

    def tokens(i):
        return make(i, 3, 5, typestr="<i4", dtype=torch.int32)

    yield lambda: nn.embedding(tokens(0), make(1, 4, 2), bag=True, token_scale=make(2, 3, 5), out=make(3, 3, 2), **more)
    yield lambda: nn.embedding_backward(make(0, 3, 2), tokens(1), 4, bag=True, token_scale=make(2, 3, 5),
                                        out=make(3, 4, 2), **more)
    yield lambda: nn.embedding_scale_backward(make(0, 3, 2), tokens(1), make(2, 4, 2), bag=True, out=make(3, 3, 5),
                                              **more)
    yield lambda: nn.layer_norm(make(0, 3, 4), make(1, 4), make(2, 4), out=make(3, 3, 4), mean=make(4, 3),
                                rstd=make(5, 3), **more)
    yield lambda: nn.layer_norm_backward(make(0, 3, 4), make(1, 3, 4), make(2, 3), make(3, 3), make(4, 4),
                                         out=make(5, 3, 4), dweight=make(6, 4), dbias=make(7, 4), **more)


@pytest.mark.parametrize("at", range(8))
def test_any_tensor_brings_torchs_current_stream(enqueued, at):
    for call, count in zip(_calls(Tensor, at), (4, 4, 4, 6, 8)):
        call()
        assert _stream(enqueued[-1]) == (77 if at < count else 0)
    for call in _calls(Tensor, None, stream=55):
        call()
        assert _stream(enqueued[-1]) == 55


@pytest.mark.parametrize("at", range(8))
def test_any_tensor_is_told_of_the_stream_that_is_given(enqueued, monkeypatch, at):
    told = []

    class Told(Tensor):
        device = torch.device("cuda", 0)

        def record_stream(self, stream):
            told.append(stream)

    class Stream:
        device = torch.device("cuda", 0)
        cuda_stream = 99

        def __init__(self, handle, device):
            assert handle == 99 and device == self.device

    class Current:
        def __init__(self, stream):
            self.handle = stream.cuda_stream

        def __enter__(self):
            monkeypatch.setattr(nn, "_raw_stream", lambda device: self.handle)

        def __exit__(self, *_):
            monkeypatch.setattr(nn, "_raw_stream", lambda device: 77)

    monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", Current)
    for call, count in zip(_calls(Told, at, stream=99), (4, 4, 4, 6, 8)):
        told.clear()
        call()
        assert _stream(enqueued[-1]) == 99
        assert bool(told) == (at < count)


def test_a_stream_of_another_device_is_refused(enqueued, monkeypatch):
    class Stream:
        device = torch.device("cuda", 1)

    class There(Tensor):
        device = torch.device("cuda", 0)

        def record_stream(self, stream):
            raise AssertionError("told of a stream that is not used")

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: pytest.fail("made current"))
    for call in _calls(There, 1, stream=Stream()):
        with pytest.raises(xgb.XGBoostError, match="another device"):
            call()
    assert not enqueued


@pytest.mark.parametrize("at", range(8))
def test_the_stream_of_an_array_is_waited_for(enqueued, monkeypatch, at):
    monkeypatch.setattr(nn._LIB, "XGBBStreamWait", lambda *args: enqueued.append(("wait", args)) or 0)
    for call, count in zip(_calls(Array, at, dict(stream=99), stream=55), (4, 4, 4, 6, 8)):
        enqueued.clear()
        call()
        assert [c[0] == "wait" for c in enqueued] == [True] * (at < count) + [False]
        assert at >= count or enqueued[0][1] == (-1, 55, 99)
    for same in (None, 55):
        for call in _calls(Array, at, dict(stream=same), stream=55):
            enqueued.clear()
            call()
            assert len(enqueued) == 1


def test_results_are_not_written_to_read_only_arrays(enqueued):
    firsts = (3, 3, 3, 3, 5)  # of the results, the last arrays of a call
    for at in range(8):
        for call, first, count in zip(_calls(Array, at, dict(read_only=True)), firsts, (4, 4, 4, 6, 8)):
            enqueued.clear()
            if first <= at < count:
                with pytest.raises(xgb.XGBoostError, match="read-only"):
                    call()
                assert not enqueued
            else:
                call()
                assert enqueued
    n = 1 << 14
    space = Array(nn.embedding_backward_workspace(n, 1, 4, 2), typestr="|u1", ptr=1 << 20, read_only=True)
    with pytest.raises(xgb.XGBoostError, match="workspace is read-only"):
        nn.embedding_backward(Array(n, 2), Array(n, typestr="<i4"), 4, out=Array(4, 2, ptr=8192), workspace=space)


def test_what_takes_no_part_in_automatic_differentiation(enqueued):
    class Leaf(Tensor):
        requires_grad = True

    refused = [call for i, call in enumerate(_calls(Leaf, 1)) if i in (0, 3)]  # the table, the norm's weight
    for call in refused:
        with pytest.raises(xgb.XGBoostError, match="automatic differentiation"):
            call()
    with pytest.raises(xgb.XGBoostError, match="differentiation needs tensors"):
        nn.embedding(Array(3, typestr="<i4"), Leaf(4, 2))
    with pytest.raises(xgb.XGBoostError, match="differentiation needs tensors"):
        nn.layer_norm(Leaf(3, 4), Array(4))
    assert not enqueued
    with torch.no_grad():
        for call in refused:
            call()
    assert len(enqueued) == 2


def test_out_dtype_is_looked_at_where_out_is_given(enqueued, monkeypatch):
    def calls(**more):
        yield lambda: nn.embedding(Array(3, typestr="<i4"), Array(4, 2), out=Array(3, 2, ptr=8192), **more)
        yield lambda: nn.embedding_backward(Array(3, 2), Array(3, typestr="<i4"), 4, out=Array(4, 2, ptr=8192), **more)

    monkeypatch.setattr(nn, "_codes", {})  # as before the first tensor
    for dtype in (torch.float64, torch.int32, np.float64, "int8", object()):
        for call in calls(out_dtype=dtype):
            with pytest.raises(xgb.XGBoostError, match="out_dtype must be"):
                call()
    for call in calls(out_dtype=torch.float16):
        with pytest.raises(xgb.XGBoostError, match="another type"):
            call()
    assert not enqueued
    for dtype in (torch.float32, np.float32, "float32"):
        for call in calls(out_dtype=dtype):
            call()
    assert len(enqueued) == 6


STRUCTS = {"XGBBEmbeddingArgs": nn._pack_embedding, "XGBBEmbeddingBackwardArgs": nn._pack_embedding_backward,
           "XGBBEmbeddingScaleBackwardArgs": nn._pack_embedding_scale_backward, "XGBBLayerNormArgs": nn._pack_layer_norm,
           "XGBBLayerNormBackwardArgs": nn._pack_layer_norm_backward}


def _fields(header, name):
    body = re.search(r"typedef struct \{([^}]*)\} %s;" % name, header).group(1)
    for names in re.findall(r"[\s*](\w+(?:, \w+)*);", body):
        yield from names.split(", ")


def test_every_argument_lies_where_the_header_has_it(tmp_path):
    """Each field of each structure packed with a value of its own, and read back by a C program by its name."""
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    with open(os.path.join(include, "xgb_b200.h")) as f:
        header = f.read()
    inner, lines, want = ["tokens." + f for f in _fields(header, "XGBBTokens")], [], []
    for at, (name, pack) in enumerate(STRUCTS.items()):
        fields = [f for field in _fields(header, name) for f in (inner if field == "tokens" else [field])]
        values = [100 + i for i in range(len(fields))]
        data = tmp_path / name
        data.write_bytes(pack(*values))
        want += values
        lines.append('{ %s a; FILE* f = fopen("%s", "rb"); if (fread(&a, 1, sizeof a + 1, f) != sizeof a) return %d;' %
                     (name, data, at + 1))
        lines += ['printf("%%.0f ", (double)%sa.%s);' % ("" if f in ("tokens.scale", "eps") else "(uint64_t)", f)
                  for f in fields]
        lines.append("fclose(f); }")
    source = tmp_path / "read.c"
    source.write_text("#include <stdio.h>\n#include <string.h>\n#include \"xgb_b200.h\"\nint main(void) {\n%s\nreturn 0; }" %
                      "\n".join(lines))
    program = str(tmp_path / "read")
    subprocess.run(["gcc", "-I", include, str(source), "-o", program], check=True)
    got = subprocess.run([program], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in got] == want
