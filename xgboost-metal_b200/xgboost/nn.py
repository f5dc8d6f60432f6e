"""Device operators for a model on top of a booster's leaf indices.

Every leaf of every tree is a token, a row's leaves are its bag of tokens, and
each token has a learned vector:

    tokens, vocab = xgboost.nn.leaf_tokens(booster, dmatrix)   # int32 [rows, trees]
    h = xgboost.nn.embedding(tokens, table, bag=True)          # [rows, dim]
    y, mean, rstd = xgboost.nn.layer_norm(h, weight, bias)

with the gradients `embedding_backward`, `embedding_scale_backward` and
`layer_norm_backward`. Arrays are device memory: tensors with torch's methods
(`data_ptr`, `stride`, `new_empty`), or any object with a
`__cuda_array_interface__`, whose outputs and workspaces the caller passes in.
Values are float32, float16 or bfloat16, tokens int32 or int64. Rows may have
any stride; the values of a row are contiguous.

Work is enqueued and not waited for: on `stream` where one is given (a handle,
or an object that has one as `cuda_stream` or `ptr`), else on torch's current
stream of the arrays' device, or the default stream for other arrays. Equal
inputs give equal bits. These functions have no counterpart in the reference.
"""
import contextlib
import ctypes
import json
import sys

import numpy as np

from .core import _LIB, XGBoostError, _check_call

__all__ = ["embedding", "embedding_backward", "embedding_backward_workspace", "embedding_scale_backward",
           "layer_norm", "layer_norm_backward", "layer_norm_backward_workspace", "leaf_tokens"]

_F32, _F16, _BF16, _I32, _I64 = 1, 3, 4, 7, 8
_P, _I, _U, _S, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_uint64, ctypes.c_int64, ctypes.c_float
_TOKENS = [_P, _I, _U, _U, _S, _S]

_LIB.XGBBEmbedding.argtypes = [_I] + _TOKENS + [_P, _I, _U, _U, _S, _F, _P, _S, _S, _P, _I, _S, _P]
_LIB.XGBBEmbeddingBackwardWorkspace.argtypes = [_U, _U, _U, _U, _P]
_LIB.XGBBEmbeddingBackward.argtypes = ([_I, _P, _I, _S] + _TOKENS +
                                       [_U, _U, _F, _P, _S, _S, _P, _I, _S, _I, _P, ctypes.c_size_t, _P])
_LIB.XGBBEmbeddingScaleBackward.argtypes = [_I, _P, _I, _S] + _TOKENS + [_P, _I, _U, _U, _S, _F, _P, _P]
_LIB.XGBBLayerNorm.argtypes = [_I, _P, _I, _U, _U, _S, _P, _P, _I, _F, _P, _S, _P, _P, _P]
_LIB.XGBBLayerNormBackwardWorkspace.argtypes = [_U, _U, _P]
_LIB.XGBBLayerNormBackward.argtypes = [_I, _P, _S, _P, _I, _U, _U, _S, _P, _P, _P, _I, _P, _S, _P, _P, _P,
                                       ctypes.c_size_t, _P]

_TYPESTR = {"<f4": _F32, "<f2": _F16, "<i4": _I32, "<i8": _I64}
_torch_codes = {}


def _torch():
    return sys.modules["torch"]


def _torch_code(dtype):
    if not _torch_codes:
        t = _torch()
        _torch_codes.update({t.float32: _F32, t.float16: _F16, t.bfloat16: _BF16, t.int32: _I32, t.int64: _I64})
    return _torch_codes.get(dtype, 0)


class _View:
    """What a call needs of an array: pointer, shape, strides (in elements),
    dtype code, device ordinal (-1: the current one) and the tensor, if it is
    one."""
    __slots__ = ("ptr", "shape", "strides", "code", "device", "tensor")

    def __init__(self, a, what):
        if hasattr(a, "data_ptr"):
            if not a.is_cuda:
                raise XGBoostError("%s must be in device memory" % what)
            self.ptr, self.shape, self.strides = a.data_ptr(), a.shape, a.stride()
            self.code, self.device, self.tensor = _torch_code(a.dtype), a.get_device(), a
            return
        inf = getattr(a, "__cuda_array_interface__", None)
        if inf is None:
            raise XGBoostError("%s must be a device array: a CUDA tensor, or an object with a "
                               "__cuda_array_interface__" % what)
        self.ptr, self.shape, self.code = int(inf["data"][0] or 0), tuple(inf["shape"]), _TYPESTR.get(inf["typestr"], 0)
        self.device, self.tensor = -1, None
        if inf.get("mask") is not None:
            raise XGBoostError("%s must not be masked" % what)
        size = int(inf["typestr"][2:])
        if inf.get("strides") is None:
            strides, step = [], 1
            for n in reversed(self.shape):
                strides.append(step)
                step *= n
            self.strides = tuple(reversed(strides))
        else:
            if any(s % size for s in inf["strides"]):
                raise XGBoostError("%s has strides that are no multiples of its item size" % what)
            self.strides = tuple(s // size for s in inf["strides"])


def _flat(shape, strides, what):
    """(count, stride) of dimensions that one stride walks in order."""
    count, stride = 1, 0
    for n, s in zip(reversed(shape), reversed(strides)):
        if n == 1:
            continue
        if count == 1:
            stride = s
        elif n and count and s != stride * count:
            raise XGBoostError("%s has leading dimensions that one stride cannot walk; make it contiguous" % what)
        count *= n
    return count, stride


def _matrix(v, what):
    """(rows, columns, row stride) of an array of rows with contiguous values."""
    if not v.shape:
        raise XGBoostError("%s must have at least one dimension" % what)
    if v.code not in (_F32, _F16, _BF16):
        raise XGBoostError("%s must be float32, float16 or bfloat16" % what)
    n = v.shape[-1]
    if n > 1 and v.strides[-1] != 1:
        raise XGBoostError("%s must have contiguous values in its last dimension" % what)
    if len(v.shape) == 2:
        return v.shape[0], n, v.strides[0]
    rows, stride = _flat(v.shape[:-1], v.strides[:-1], what)
    return rows, n, stride


def _token_grid(v, bag):
    """(rows, per_row, row stride, column stride, leading shape) of tokens."""
    if v.code not in (_I32, _I64):
        raise XGBoostError("tokens must be int32 or int64")
    shape, strides = v.shape, v.strides
    if not bag:
        if len(shape) == 1:
            return shape[0], 1, strides[0], 0, shape
        rows, stride = _flat(shape, strides, "tokens")
        return rows, 1, stride, 0, shape
    if not shape:
        raise XGBoostError("a bag of tokens must have at least one dimension")
    if len(shape) == 2:
        return shape[0], shape[1], strides[0], strides[1], shape[:-1]
    rows, stride = _flat(shape[:-1], strides[:-1], "tokens")
    return rows, shape[-1], stride, strides[-1], shape[:-1]


def _token_scale(scale, tokens, bag):
    """The view and strides of token_scale, broadcast to the tokens' shape."""
    if scale is None:
        return None, 0, 0
    if hasattr(scale, "expand"):
        try:
            scale = scale.expand(tokens.shape)
        except RuntimeError as e:
            raise XGBoostError("token_scale does not broadcast to the tokens' shape: %s" % e) from None
    v = _View(scale, "token_scale")
    if tuple(v.shape) != tuple(tokens.shape):
        raise XGBoostError("token_scale must have the tokens' shape")
    if v.code != _F32:
        raise XGBoostError("token_scale must be float32")
    if not bag:
        return v, _flat(v.shape, v.strides, "token_scale")[1], 0
    return v, _flat(v.shape[:-1], v.strides[:-1], "token_scale")[1], v.strides[-1]


def _device(*views):
    device = -1
    for v in views:
        if v is not None and v.device >= 0:
            if device >= 0 and v.device != device:
                raise XGBoostError("the arrays are on different devices")
            device = v.device
    return device


def _handle(stream, device, tensor):
    """The stream's handle."""
    if stream is None:
        return _torch().cuda.current_stream(device).cuda_stream if tensor is not None else 0
    for name in ("cuda_stream", "ptr"):
        if hasattr(stream, name):
            return int(getattr(stream, name))
    return int(stream)


@contextlib.contextmanager
def _on(stream, tensors):
    """Makes a given stream torch's current one, so that results and workspaces
    come from its own memory, and tells torch that the inputs are used on it."""
    tensors = [t for t in tensors if hasattr(t, "record_stream")]
    if not tensors:
        yield
        return
    torch, device = _torch(), tensors[0].device
    handle = _handle(stream, device, None)
    s = stream if isinstance(stream, torch.cuda.Stream) else \
        torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
    with torch.cuda.stream(s):
        for t in tensors:
            t.record_stream(s)
        yield


def _dtype_code(dtype):
    if isinstance(dtype, (str, np.dtype, type)):
        return _TYPESTR.get(np.dtype(dtype).str, 0)
    return _torch_code(dtype)


def _result(out, shape, code, like, what):
    """The array that a result goes to, and its view: `out`, checked, or a new
    one of like's kind."""
    if out is None:
        if like.tensor is None:
            raise XGBoostError("%s must be given where the inputs are no tensors" % what)
        dtype = like.tensor.dtype if code == like.code else \
            next((d for d, c in _torch_codes.items() if c == code), None)
        if dtype is None:
            raise XGBoostError("%s must be float32, float16 or bfloat16" % what)
        out = like.tensor.new_empty(shape, dtype=dtype)
        return out, _View(out, what)
    v = _View(out, what)
    if tuple(v.shape) != tuple(shape):
        raise XGBoostError("%s must have the shape %s" % (what, tuple(shape)))
    if code and v.code != code:
        raise XGBoostError("%s has another type than it must have" % what)
    return out, v


def _vector(v, n, codes, what):
    if v is None:
        return
    if tuple(v.shape) != (n,) or (n > 1 and v.strides[0] != 1):
        raise XGBoostError("%s must be %d contiguous values" % (what, n))
    if v.code not in codes:
        raise XGBoostError("%s must be float32 or have x's type" % what)


def _stats(v, lead, rows, what):
    if tuple(v.shape) != tuple(lead) or (rows > 1 and _flat(v.shape, v.strides, what)[1] != 1):
        raise XGBoostError("%s must be contiguous, one value a row" % what)
    if v.code != _F32:
        raise XGBoostError("%s must be float32" % what)


def _workspace(workspace, size, like):
    if not size:
        return None
    if workspace is None:
        if like.tensor is None:
            raise XGBoostError("workspace must be given where the inputs are no tensors")
        workspace = like.tensor.new_empty(size, dtype=_torch().uint8)
        return workspace
    v = _View(workspace, "workspace")
    items = int(np.prod(v.shape, dtype=np.int64))
    width = v.tensor.element_size() if v.tensor is not None else \
        int(workspace.__cuda_array_interface__["typestr"][2:])
    if items * width < size or (items > 1 and _flat(v.shape, v.strides, "workspace")[1] != 1):
        raise XGBoostError("workspace must be %d contiguous bytes" % size)
    return workspace


def _pointer(array):
    return None if array is None else _View(array, "workspace").ptr


def embedding(tokens, table, *, scale=1.0, token_scale=None, bag=False, out=None, out_dtype=None, stream=None):
    """scale * token_scale * table[tokens]: shape tokens.shape + (dim,), or
    with `bag` the sum over the tokens' last dimension, tokens.shape[:-1] +
    (dim,).

    A token below 0 is missing and adds nothing (a row of missing tokens is
    zeros); one past the table makes its row NaN. token_scale (float32)
    broadcasts to the tokens' shape. Sums are float32. The result has the
    table's type, or `out_dtype`; of the two types one is float32 or both are
    the same."""
    if stream is not None and hasattr(table, "data_ptr"):
        with _on(stream, (tokens, table, token_scale, out)):
            return embedding(tokens, table, scale=scale, token_scale=token_scale, bag=bag, out=out,
                             out_dtype=out_dtype)
    k, w = _View(tokens, "tokens"), _View(table, "table")
    if len(w.shape) != 2:
        raise XGBoostError("table must have two dimensions")
    rows, per_row, stride_row, stride_col, lead = _token_grid(k, bag)
    vocab, dim, table_stride = _matrix(w, "table")
    s, s_row, s_col = _token_scale(token_scale, k, bag)
    code = w.code if out_dtype is None else _dtype_code(out_dtype)
    out, y = _result(out, (*lead, dim), 0 if out is not None and out_dtype is None else code, w, "out")
    y_rows, _, y_stride = _matrix(y, "out")
    device = _device(k, w, s, y)
    _check_call(_LIB.XGBBEmbedding(device, k.ptr, k.code, rows, per_row, stride_row, stride_col, w.ptr, w.code, vocab,
                                   dim, table_stride, scale, s and s.ptr, s_row, s_col, y.ptr, y.code, y_stride,
                                   _handle(stream, device, w.tensor)))
    return out


def embedding_backward_workspace(rows, per_row, vocab, dim):
    """Bytes of workspace that embedding_backward needs for `rows` bags of
    `per_row` tokens (1 without `bag`)."""
    size = ctypes.c_size_t()
    _check_call(_LIB.XGBBEmbeddingBackwardWorkspace(rows, per_row, vocab, dim, ctypes.byref(size)))
    return size.value


def embedding_backward(grad, tokens, vocab, *, scale=1.0, token_scale=None, bag=False, out=None, out_dtype=None,
                       accumulate=False, workspace=None, stream=None):
    """The gradient [vocab, dim] of embedding's table from its result's
    gradient `grad`. Missing tokens and those past the table add nothing.
    With `accumulate` it is added to what `out` holds. It has grad's type, or
    `out_dtype`; of the two types one is float32 or both are the same."""
    if stream is not None and hasattr(grad, "data_ptr"):
        with _on(stream, (grad, tokens, token_scale, out, workspace)):
            return embedding_backward(grad, tokens, vocab, scale=scale, token_scale=token_scale, bag=bag, out=out,
                                      out_dtype=out_dtype, accumulate=accumulate, workspace=workspace)
    g, k = _View(grad, "grad"), _View(tokens, "tokens")
    rows, per_row, stride_row, stride_col, lead = _token_grid(k, bag)
    g_rows, dim, g_stride = _matrix(g, "grad")
    if tuple(g.shape[:-1]) != tuple(lead):
        raise XGBoostError("grad must have the shape of the lookup's result")
    if accumulate and out is None:
        raise XGBoostError("accumulate needs out")
    s, s_row, s_col = _token_scale(token_scale, k, bag)
    code = g.code if out_dtype is None else _dtype_code(out_dtype)
    out, y = _result(out, (vocab, dim), 0 if out is not None and out_dtype is None else code, g, "out")
    _, _, y_stride = _matrix(y, "out")
    device = _device(g, k, s, y)
    size = embedding_backward_workspace(rows, per_row, vocab, dim)
    workspace = _workspace(workspace, size, g)
    _check_call(_LIB.XGBBEmbeddingBackward(device, g.ptr, g.code, g_stride, k.ptr, k.code, rows, per_row, stride_row,
                                           stride_col, vocab, dim, scale, s and s.ptr, s_row, s_col, y.ptr, y.code,
                                           y_stride, bool(accumulate), _pointer(workspace), size,
                                           _handle(stream, device, g.tensor)))
    return out


def embedding_scale_backward(grad, tokens, table, *, scale=1.0, bag=False, out=None, stream=None):
    """The gradient of embedding's token_scale, float32 in the tokens' shape: 0
    for a missing token, NaN for one past the table. (Where token_scale was
    broadcast, its own gradient is this one's sum over the broadcast
    dimensions.)"""
    if stream is not None and hasattr(grad, "data_ptr"):
        with _on(stream, (grad, tokens, table, out)):
            return embedding_scale_backward(grad, tokens, table, scale=scale, bag=bag, out=out)
    g, k, w = _View(grad, "grad"), _View(tokens, "tokens"), _View(table, "table")
    if len(w.shape) != 2:
        raise XGBoostError("table must have two dimensions")
    rows, per_row, stride_row, stride_col, lead = _token_grid(k, bag)
    vocab, dim, table_stride = _matrix(w, "table")
    g_rows, g_dim, g_stride = _matrix(g, "grad")
    if tuple(g.shape[:-1]) != tuple(lead) or g_dim != dim:
        raise XGBoostError("grad must have the shape of the lookup's result")
    out, y = _result(out, tuple(k.shape), _F32, g, "out")
    if rows * per_row > 1 and _flat(y.shape, y.strides, "out")[1] != 1:
        raise XGBoostError("out must be contiguous")
    device = _device(g, k, w, y)
    _check_call(_LIB.XGBBEmbeddingScaleBackward(device, g.ptr, g.code, g_stride, k.ptr, k.code, rows, per_row,
                                                stride_row, stride_col, w.ptr, w.code, vocab, dim, table_stride,
                                                scale, y.ptr, _handle(stream, device, g.tensor)))
    return out


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, out=None, mean=None, rstd=None, stream=None):
    """(y, mean, rstd) of a layer norm over x's last dimension: y = (x - mean)
    * rstd * weight + bias in x's type, mean and rstd = 1 / sqrt(variance +
    eps) in float32, one a row. weight and bias have x's type or are float32,
    both the same."""
    if stream is not None and hasattr(x, "data_ptr"):
        with _on(stream, (x, weight, bias, out, mean, rstd)):
            return layer_norm(x, weight, bias, eps=eps, out=out, mean=mean, rstd=rstd)
    v = _View(x, "x")
    rows, dim, stride = _matrix(v, "x")
    w = None if weight is None else _View(weight, "weight")
    b = None if bias is None else _View(bias, "bias")
    _vector(w, dim, (v.code, _F32), "weight")
    _vector(b, dim, (v.code, _F32), "bias")
    if w is not None and b is not None and w.code != b.code:
        raise XGBoostError("weight and bias must have the same type")
    param = w.code if w is not None else b.code if b is not None else _F32
    lead = v.shape[:-1]
    out, y = _result(out, v.shape, v.code, v, "out")
    mean, m = _result(mean, lead, _F32, v, "mean")
    rstd, q = _result(rstd, lead, _F32, v, "rstd")
    _stats(m, lead, rows, "mean")
    _stats(q, lead, rows, "rstd")
    _, _, y_stride = _matrix(y, "out")
    device = _device(v, w, b, y, m, q)
    _check_call(_LIB.XGBBLayerNorm(device, v.ptr, v.code, rows, dim, stride, w and w.ptr, b and b.ptr, param, eps,
                                   y.ptr, y_stride, m.ptr, q.ptr, _handle(stream, device, v.tensor)))
    return out, mean, rstd


def layer_norm_backward_workspace(rows, dim):
    """Bytes of workspace that layer_norm_backward needs for the gradients of
    weight and bias."""
    size = ctypes.c_size_t()
    _check_call(_LIB.XGBBLayerNormBackwardWorkspace(rows, dim, ctypes.byref(size)))
    return size.value


def layer_norm_backward(grad, x, mean, rstd, weight=None, *, bias_grad=True, out=None, dweight=None, dbias=None,
                        workspace=None, stream=None):
    """(dx, dweight, dbias) from the gradient `grad` of layer_norm's y and the
    mean and rstd that it returned. Without a weight (then y is the normalised
    x) dweight and dbias are None; without `bias_grad` dbias is None."""
    if stream is not None and hasattr(grad, "data_ptr"):
        with _on(stream, (grad, x, mean, rstd, weight, out, dweight, dbias, workspace)):
            return layer_norm_backward(grad, x, mean, rstd, weight, bias_grad=bias_grad, out=out, dweight=dweight,
                                       dbias=dbias, workspace=workspace)
    g, v = _View(grad, "grad"), _View(x, "x")
    rows, dim, stride = _matrix(v, "x")
    _, _, g_stride = _matrix(g, "grad")
    if tuple(g.shape) != tuple(v.shape) or g.code != v.code:
        raise XGBoostError("grad must have x's shape and type")
    m, q = _View(mean, "mean"), _View(rstd, "rstd")
    lead = v.shape[:-1]
    _stats(m, lead, rows, "mean")
    _stats(q, lead, rows, "rstd")
    w = None if weight is None else _View(weight, "weight")
    _vector(w, dim, (v.code, _F32), "weight")
    out, dx = _result(out, v.shape, v.code, v, "out")
    _, _, dx_stride = _matrix(dx, "out")
    dw = db = None
    size = 0
    if w is not None:
        dweight, dw = _result(dweight, (dim,), w.code, w, "dweight")
        _vector(dw, dim, (w.code,), "dweight")
        if bias_grad:
            dbias, db = _result(dbias, (dim,), w.code, w, "dbias")
            _vector(db, dim, (w.code,), "dbias")
        size = layer_norm_backward_workspace(rows, dim)
        workspace = _workspace(workspace, size, v)
    elif dweight is not None or dbias is not None:
        raise XGBoostError("dweight and dbias need weight")
    device = _device(g, v, m, q, w, dx, dw, db)
    _check_call(_LIB.XGBBLayerNormBackward(device, g.ptr, g_stride, v.ptr, v.code, rows, dim, stride, m.ptr, q.ptr,
                                           w and w.ptr, w.code if w is not None else _F32, dx.ptr, dx_stride,
                                           dw and dw.ptr, db and db.ptr, _pointer(workspace) if size else None, size,
                                           _handle(stream, device, v.tensor)))
    return out, dweight, dbias


def leaf_tokens(booster, data, iteration_range=(0, 0)):
    """The leaves that a booster's trees send `data` to, as tokens: (int32
    [rows, trees], number of tokens). Each leaf of each tree has a number of
    its own, tree after tree."""
    leaves = booster.predict(data, pred_leaf=True, strict_shape=True, iteration_range=iteration_range)
    rounds, groups = leaves.shape[1], int(np.prod(leaves.shape[2:], dtype=np.int64))
    trees = json.loads(bytes(booster.save_raw("json")).decode())["learner"]["gradient_booster"]["model"]["trees"]
    first = int(iteration_range[0]) * groups
    nodes = leaves.reshape(leaves.shape[0], rounds * groups).astype(np.int32)
    tokens, vocab = np.empty_like(nodes), 0
    for t in range(nodes.shape[1]):
        is_leaf = np.asarray(trees[first + t]["left_children"]) < 0
        number = vocab + np.cumsum(is_leaf) - 1
        tokens[:, t] = number[nodes[:, t]]
        vocab += int(is_leaf.sum())
    return tokens, vocab
