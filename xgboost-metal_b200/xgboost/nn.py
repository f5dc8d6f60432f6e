"""Device operators for a model on top of a booster's leaf indices.

Every leaf of every tree is a token, a row's leaves are its bag of tokens, and
each token has a learned vector:

    tokens, vocab = xgboost.nn.leaf_tokens(booster, dmatrix)   # int32 [rows, trees], on the host
    tokens = torch.from_numpy(tokens).cuda()
    h = xgboost.nn.embedding(tokens, table, bag=True)          # [rows, dim] of a table [vocab, dim]
    y, mean, rstd = xgboost.nn.layer_norm(h, weight, bias)

with the gradients `embedding_backward`, `embedding_scale_backward` and
`layer_norm_backward`, which torch's autograd calls too (once: their results are
not differentiated). Arrays are device memory: tensors with torch's methods
(`data_ptr`, `stride`, `new_empty`), or any object with a
`__cuda_array_interface__`, whose outputs and workspaces the caller passes in.
Values are float32, float16 or bfloat16, tokens int32 or int64. Rows may have
any stride; the values of a row are contiguous.

Work is enqueued and not waited for: on `stream` where one is given (a handle,
or an object that has one as `cuda_stream` or `ptr`), else on torch's current
stream of the arrays' device where one of them is a tensor, else on the default
stream. It runs after what is enqueued on the streams that the arrays'
interfaces name. Equal inputs give equal bits. These functions have no
counterpart in the reference.
"""
import contextlib
import ctypes
import functools
import json
import struct
import sys

import numpy as np

from .core import _LIB, XGBoostError, _check_call

__all__ = ["embedding", "embedding_backward", "embedding_backward_workspace", "embedding_scale_backward",
           "layer_norm", "layer_norm_backward", "layer_norm_backward_workspace", "leaf_tokens"]

_F32, _F16, _BF16, _I32, _I64 = 1, 3, 4, 7, 8
_FLOATS, _INTS = (_F32, _F16, _BF16), (_I32, _I64)

# The argument structures of include/xgb_b200.h.
_TOKENS = "PPQQqqqqif"
_pack_embedding = struct.Struct("@" + _TOKENS + "PPPQQqqiii4x").pack
_pack_embedding_backward = struct.Struct("@" + _TOKENS + "PPPPNQQqqiiii").pack
_pack_embedding_scale_backward = struct.Struct("@" + _TOKENS + "PPPPQQqqiii4x").pack
_pack_layer_norm = struct.Struct("@PPPPPPPQQqqiiif").pack
_pack_layer_norm_backward = struct.Struct("@PPPPPPPPPPNQQqqqiii4x").pack

for _name in ("XGBBEmbedding", "XGBBEmbeddingBackward", "XGBBEmbeddingScaleBackward", "XGBBLayerNorm",
              "XGBBLayerNormBackward"):
    getattr(_LIB, _name).argtypes = [ctypes.c_char_p]
_SIZES = [ctypes.c_uint64] * 4
_LIB.XGBBEmbeddingBackwardWorkspace.argtypes = _SIZES + [ctypes.c_void_p]
_LIB.XGBBLayerNormBackwardWorkspace.argtypes = _SIZES[:2] + [ctypes.c_void_p]
_LIB.XGBBStreamWait.argtypes = [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p]

_TYPESTR = {"<f4": _F32, "<f2": _F16, "<i4": _I32, "<i8": _I64}
_codes, _dtypes = {}, {}  # torch's dtypes by code and back, filled when the first tensor comes
_raw_stream = _empty_like = None


def _know_torch():
    global _raw_stream, _empty_like
    t = sys.modules["torch"]
    _empty_like = t.empty_like
    _raw_stream = getattr(t._C, "_cuda_getCurrentRawStream", None) or \
        (lambda device: t.cuda.current_stream(device).cuda_stream)
    codes = {t.float32: _F32, t.float16: _F16, t.bfloat16: _BF16, t.int32: _I32, t.int64: _I64}
    _dtypes.update({c: d for d, c in codes.items()})
    _codes.update(codes)  # last: other threads take it that all is known


def _call(function, args):
    if function(args) != 0:
        _check_call(-1)


def _view(a, what, written=False):
    """What a call needs of an array: (pointer, shape, strides in elements,
    dtype code, device ordinal or -1 for the current one, the tensor or None)."""
    try:
        ptr = a.data_ptr()
    except AttributeError:
        return _interface_view(a, what, written)
    if not a.is_cuda:
        raise XGBoostError("%s must be in device memory" % what)
    if not _codes:
        _know_torch()
    return ptr, a.shape, a.stride(), _codes.get(a.dtype, 0), a.get_device(), a


def _interface_view(a, what, written):
    inf = getattr(a, "__cuda_array_interface__", None)
    if inf is None:
        raise XGBoostError("%s must be a device array: a CUDA tensor, or an object with a "
                           "__cuda_array_interface__" % what)
    if inf.get("mask") is not None:
        raise XGBoostError("%s must not be masked" % what)
    if written and inf["data"][1]:
        raise XGBoostError("%s is read-only" % what)
    shape, size = tuple(inf["shape"]), int(inf["typestr"][2:])
    if inf.get("strides") is None:
        strides, step = [], 1
        for n in reversed(shape):
            strides.append(step)
            step *= n
        strides = tuple(reversed(strides))
    else:
        if any(s % size for s in inf["strides"]):
            raise XGBoostError("%s has strides that are no multiples of its item size" % what)
        strides = tuple(s // size for s in inf["strides"])
    return int(inf["data"][0] or 0), shape, strides, _TYPESTR.get(inf["typestr"], 0), -1, None


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
    shape, strides = v[1], v[2]
    if v[3] not in _FLOATS:
        raise XGBoostError("%s must be float32, float16 or bfloat16" % what)
    if not shape:
        raise XGBoostError("%s must have at least one dimension" % what)
    n = shape[-1]
    if n > 1 and strides[-1] != 1:
        raise XGBoostError("%s must have contiguous values in its last dimension" % what)
    if len(shape) == 2:
        return shape[0], n, strides[0]
    rows, stride = _flat(shape[:-1], strides[:-1], what)
    return rows, n, stride


def _token_grid(v, bag):
    """(rows, per_row, row stride, column stride, leading shape) of tokens."""
    shape, strides = v[1], v[2]
    if v[3] not in _INTS:
        raise XGBoostError("tokens must be int32 or int64")
    if not bag:
        if len(shape) == 1:
            return shape[0], 1, strides[0], 0, shape
        rows, stride = _flat(shape, strides, "tokens")
        return rows, 1, stride, 0, shape
    if not shape:
        raise XGBoostError("a bag of tokens must have at least one dimension")
    if len(shape) == 2:
        return shape[0], shape[1], strides[0], strides[1], shape[:1]
    rows, stride = _flat(shape[:-1], strides[:-1], "tokens")
    return rows, shape[-1], stride, strides[-1], shape[:-1]


def _expand(scale, shape, bag):
    """token_scale broadcast to the tokens' shape, where it can tell how; as a copy
    where one stride cannot walk it. The caller holds it until the call is made."""
    if hasattr(scale, "expand"):
        try:
            if scale.shape != shape:
                scale = scale.expand(shape)
            lead = len(shape) - bool(bag)
            _flat(scale.shape[:lead], scale.stride()[:lead], "token_scale")
        except RuntimeError as e:
            raise XGBoostError("token_scale does not broadcast to the tokens' shape: %s" % e) from None
        except XGBoostError:
            scale = scale.contiguous()
    return scale


def _scale_grid(scale, tokens, bag):
    """(pointer, row stride, column stride, device) of token_scale in the tokens'
    shape."""
    if scale is None:
        return 0, 0, 0, -1
    ptr, shape, strides, code, device, _ = _view(scale, "token_scale")
    if tuple(shape) != tuple(tokens[1]):
        raise XGBoostError("token_scale must have the tokens' shape")
    if code != _F32:
        raise XGBoostError("token_scale must be float32")
    if not bag:
        return ptr, _flat(shape, strides, "token_scale")[1], 0, device
    return ptr, _flat(shape[:-1], strides[:-1], "token_scale")[1], strides[-1], device


def _one_device(*devices):
    device = devices[0]
    for d in devices:
        if d != device and d >= 0:
            if device >= 0:
                raise XGBoostError("the arrays are on different devices")
            device = d
    return device


def _stream_handle(stream):
    for name in ("cuda_stream", "ptr"):
        if hasattr(stream, name):
            return int(getattr(stream, name))
    return int(stream)


def _handle(stream, device, *arrays):
    """The handle of the stream to use: torch's current one where any array is a
    tensor, as the device tells then. It waits for the streams that the arrays'
    interfaces name, where their producers may still be at work."""
    if device >= 0:
        handle = _raw_stream(device)
    else:
        handle = 0 if stream is None else _stream_handle(stream)
    waited = {None, handle}
    for a in arrays:
        if a is not None and not hasattr(a, "data_ptr"):
            after = a.__cuda_array_interface__.get("stream")
            if after not in waited:
                waited.add(after)
                _check_call(_LIB.XGBBStreamWait(device, handle, after))
    return handle


def _tensors(*arrays):
    return any(hasattr(a, "data_ptr") for a in arrays)


@contextlib.contextmanager
def _on(stream, tensors):
    """Makes a given stream torch's current one, so that results and workspaces
    come from its own memory, and tells torch that the inputs are used on it."""
    torch = sys.modules["torch"]
    tensors = [t for t in tensors if hasattr(t, "record_stream") and t.is_cuda]
    if not tensors:  # refused by the call
        yield
        return
    device = tensors[0].device
    if isinstance(stream, torch.cuda.Stream):
        s = stream
    else:
        handle = _stream_handle(stream)
        s = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
    if s.device != device:
        raise XGBoostError("stream is one of another device than the arrays'")
    with torch.cuda.stream(s):
        for t in tensors:
            t.record_stream(s)
        yield


def _dtype_code(dtype):
    """The code of a given out_dtype, one of a float type."""
    if not _codes and "torch" in sys.modules:
        _know_torch()
    try:
        code = _codes[dtype] if dtype in _codes else _TYPESTR.get(np.dtype(dtype).str, 0)
    except TypeError:
        code = 0
    if code not in _FLOATS:
        raise XGBoostError("out_dtype must be float32, float16 or bfloat16")
    return code


def _new(shape, code, like, what):
    """(tensor, pointer) of a new result of like's kind."""
    tensor = like[5]
    if tensor is None:
        raise XGBoostError("%s must be given where the inputs are no tensors" % what)
    if code not in _FLOATS:
        raise XGBoostError("%s must be float32, float16 or bfloat16" % what)
    # Sizes one by one are read faster than a tuple of them.
    if not shape:
        out = tensor.new_empty((), dtype=_dtypes[code])
    elif code == like[3]:
        out = tensor.new_empty(*shape)
    else:
        out = tensor.new_empty(*shape, dtype=_dtypes[code])
    return out, out.data_ptr()


def _result(out, shape, code, like, what):
    """(array, pointer, dtype code, row stride, device) of a result: `out`,
    checked, or a new one of like's kind. Any float type does where code is 0."""
    if out is None:
        out, ptr = _new(shape, code, like, what)
        return out, ptr, code, shape[-1] if shape else 1, like[4]
    v = _view(out, what, True)
    if tuple(v[1]) != tuple(shape):
        raise XGBoostError("%s must have the shape %s" % (what, tuple(shape)))
    if code and v[3] != code:
        raise XGBoostError("%s has another type than it must have" % what)
    return out, v[0], v[3], _matrix(v, what)[2] if shape else 1, v[4]


def _flat_result(out, shape, code, like, what):
    """(array, pointer, device) of a result of contiguous values."""
    if out is None:
        out, ptr = _new(shape, code, like, what)
        return out, ptr, like[4]
    v = _view(out, what, True)
    if tuple(v[1]) != tuple(shape):
        raise XGBoostError("%s must have the shape %s" % (what, tuple(shape)))
    if v[3] != code:
        raise XGBoostError("%s has another type than it must have" % what)
    n, stride = _flat(v[1], v[2], what)
    if n > 1 and stride != 1:
        raise XGBoostError("%s must be contiguous" % what)
    return out, v[0], v[4]


def _vector(a, dim, code, what):
    """The view of weight or bias."""
    v = _view(a, what)
    if len(v[1]) != 1 or v[1][0] != dim or (dim > 1 and v[2][0] != 1):
        raise XGBoostError("%s must be %d contiguous values" % (what, dim))
    if v[3] != code and v[3] != _F32:
        raise XGBoostError("%s must be float32 or have x's type" % what)
    return v


def _row_values(a, lead, what):
    """(pointer, device) of mean or rstd."""
    ptr, shape, strides, code, device, _ = _view(a, what)
    if code != _F32:
        raise XGBoostError("%s must be float32" % what)
    if shape == lead:
        if len(shape) == 1 and (strides[0] == 1 or shape[0] == 1):
            return ptr, device
        n, stride = _flat(shape, strides, what)
        if n <= 1 or stride == 1:
            return ptr, device
    raise XGBoostError("%s must be contiguous, one value a row" % what)


def _space(workspace, size, like):
    """(workspace, pointer, device) of `size` bytes."""
    if workspace is None:
        if like[5] is None:
            raise XGBoostError("workspace must be given where the inputs are no tensors")
        workspace = like[5].new_empty(size, dtype=sys.modules["torch"].uint8)
        return workspace, workspace.data_ptr(), like[4]
    v = _view(workspace, "workspace", True)
    n, stride = _flat(v[1], v[2], "workspace")
    width = v[5].element_size() if v[5] is not None else int(workspace.__cuda_array_interface__["typestr"][2:])
    if n * width < size or (n > 1 and stride != 1):
        raise XGBoostError("workspace must be %d contiguous bytes" % size)
    return workspace, v[0], v[4]


# Automatic differentiation. The library's gradients, not torch's, run backward:
# what they give is not differentiated again.


def _tracked(*arrays):
    """Whether torch records what is done with one of them."""
    for a in arrays:
        if getattr(a, "requires_grad", False):
            return sys.modules["torch"].is_grad_enabled()
    return False


def _recorded(function, arrays, results, *rest):
    """A call that torch records, of arrays that are all tensors, if any; `results`
    that the caller brings would not be part of the record."""
    if any(r is not None for r in results):
        raise XGBoostError("results that are given take no part in automatic differentiation: "
                           "call with torch.no_grad() or with detached inputs")
    if not all(a is None or hasattr(a, "requires_grad") for a in arrays):
        raise XGBoostError("automatic differentiation needs tensors: "
                           "call with torch.no_grad() or with detached inputs")
    return _functions()[function].apply(*arrays, *rest)


@functools.lru_cache(maxsize=None)
def _functions():
    from torch.autograd import Function
    from torch.autograd.function import once_differentiable

    class Embedding(Function):
        @staticmethod
        def forward(ctx, tokens, table, token_scale, scale, bag, out_dtype):
            ctx.save_for_backward(tokens, table if ctx.needs_input_grad[2] else None, token_scale)
            ctx.rest = scale, bag, table.shape[0], table.dtype
            return embedding(tokens, table, scale=scale, token_scale=token_scale, bag=bag, out_dtype=out_dtype)

        @staticmethod
        @once_differentiable
        def backward(ctx, grad):
            tokens, table, token_scale = ctx.saved_tensors
            scale, bag, vocab, dtype = ctx.rest
            grad, d_table, d_scale = grad.contiguous(), None, None
            if ctx.needs_input_grad[1]:
                d_table = embedding_backward(grad, tokens, vocab, scale=scale, token_scale=token_scale, bag=bag,
                                             out_dtype=dtype)
            if ctx.needs_input_grad[2]:
                d_scale = embedding_scale_backward(grad, tokens, table, scale=scale, bag=bag)
            return None, d_table, d_scale, None, None, None

    class LayerNorm(Function):
        @staticmethod
        def forward(ctx, x, weight, bias, eps):
            y, mean, rstd = layer_norm(x, weight, bias, eps=eps)
            ctx.save_for_backward(x, weight, mean, rstd)
            ctx.bias_type = None if bias is None else bias.dtype
            ctx.mark_non_differentiable(mean, rstd)
            ctx.set_materialize_grads(False)
            return y, mean, rstd

        @staticmethod
        @once_differentiable
        def backward(ctx, grad, _mean, _rstd):
            if grad is None:
                return None, None, None, None
            x, weight, mean, rstd = ctx.saved_tensors
            of_bias = ctx.needs_input_grad[2]
            dbias = x.new_empty(x.shape[-1], dtype=ctx.bias_type) if of_bias and weight is None else None
            dx, dweight, dbias = layer_norm_backward(grad.contiguous(), x, mean, rstd, weight, bias_grad=of_bias,
                                                     dbias=dbias)
            return dx, dweight, dbias, None

    return {"embedding": Embedding, "layer_norm": LayerNorm}


# The calls below take contiguous tensors of one device a short way, which asks
# only what such tensors can be wrong in: a small call's time is mostly Python's.
# Where that way finds anything else it gives None (or _Long), and the long way
# takes the call or says what is wrong.


class _Long(Exception):
    pass


def _plain(a, device, dim=None):
    """(pointer, dtype code) of a contiguous tensor on `device`, of `dim` values in
    one dimension if given."""
    if a.get_device() != device or not a.is_contiguous() or \
            (dim is not None and (a.numel() != dim or a.dim() != 1)):
        raise _Long
    return a.data_ptr(), _codes[a.dtype]


def _short_way(f):
    @functools.wraps(f)
    def call(*args):
        try:
            return f(*args)
        except (_Long, AttributeError, KeyError, IndexError, ZeroDivisionError):
            return None
    return call


@_short_way
def _embedding_short(tokens, table, scale, token_scale, bag, out_dtype):
    device = table.get_device()
    if device < 0 or table.dim() != 2:
        return None
    if (table.requires_grad or (token_scale is not None and token_scale.requires_grad)) and \
            _tracked(table, token_scale):
        return None
    w, code = _plain(table, device)
    k, k_code = _plain(tokens, device)
    shape, (vocab, dim) = tokens.shape, table.shape
    if code not in _FLOATS or k_code not in _INTS:
        return None
    s = 0
    if token_scale is not None:
        s, s_code = _plain(token_scale, device)
        if s_code != _F32 or token_scale.shape != shape:
            return None
    per_row = shape[-1] if bag else 1
    rows = tokens.numel() // per_row
    lead = shape[:-1] if bag else shape
    y_code = code if out_dtype is None else _codes[out_dtype]
    if y_code not in _FLOATS:
        return None
    out = table.new_empty(*lead, dim) if y_code == code else table.new_empty(*lead, dim, dtype=out_dtype)
    _call(_LIB.XGBBEmbedding, _pack_embedding(
        k, s, rows, per_row, per_row, 1, per_row, 1, k_code, scale, w, out.data_ptr(), _raw_stream(device), vocab, dim,
        dim, dim, code, y_code, device))
    return out


@_short_way
def _embedding_backward_short(grad, tokens, vocab, scale, token_scale, bag, out_dtype):
    device = grad.get_device()
    if device < 0:
        return None
    g, code = _plain(grad, device)
    k, k_code = _plain(tokens, device)
    shape = tokens.shape
    g_shape = grad.shape
    if code not in _FLOATS or k_code not in _INTS or g_shape[:-1] != (shape[:-1] if bag else shape):
        return None
    s = 0
    if token_scale is not None:
        s, s_code = _plain(token_scale, device)
        if s_code != _F32 or token_scale.shape != shape:
            return None
    per_row, dim = shape[-1] if bag else 1, g_shape[-1]
    rows = tokens.numel() // per_row
    y_code = code if out_dtype is None else _codes[out_dtype]
    if y_code not in _FLOATS:
        return None
    size = embedding_backward_workspace(rows, per_row, vocab, dim)
    out = grad.new_empty(vocab, dim) if y_code == code else grad.new_empty(vocab, dim, dtype=out_dtype)
    space = grad.new_empty(size, dtype=sys.modules["torch"].uint8) if size else None
    _call(_LIB.XGBBEmbeddingBackward, _pack_embedding_backward(
        k, s, rows, per_row, per_row, 1, per_row, 1, k_code, scale, g, out.data_ptr(), space.data_ptr() if size else 0,
        _raw_stream(device), size, vocab, dim, dim, dim, code, y_code, 0, device))
    return out


@_short_way
def _embedding_scale_backward_short(grad, tokens, table, scale, bag):
    device = grad.get_device()
    if device < 0 or table.dim() != 2:
        return None
    g, code = _plain(grad, device)
    k, k_code = _plain(tokens, device)
    w, w_code = _plain(table, device)
    shape, g_shape, (vocab, dim) = tokens.shape, grad.shape, table.shape
    if code not in _FLOATS or w_code not in _FLOATS or k_code not in _INTS or g_shape[-1] != dim or \
            g_shape[:-1] != (shape[:-1] if bag else shape):
        return None
    per_row = shape[-1] if bag else 1
    out = grad.new_empty(*shape, dtype=_dtypes[_F32])
    _call(_LIB.XGBBEmbeddingScaleBackward, _pack_embedding_scale_backward(
        k, 0, tokens.numel() // per_row, per_row, per_row, 1, 0, 0, k_code, scale, g, w, out.data_ptr(),
        _raw_stream(device), vocab, dim, dim, dim, code, w_code, device))
    return out


@_short_way
def _layer_norm_short(x, weight, bias, eps):
    device = x.get_device()
    if device < 0:
        return None
    if x.requires_grad and _tracked(x):
        return None
    v, code = _plain(x, device)
    shape = x.shape
    dim = shape[-1]
    w = b = 0
    param = _F32
    if weight is not None:
        if weight.requires_grad and _tracked(weight):
            return None
        w, param = _plain(weight, device, dim)
    if bias is not None:
        if bias.requires_grad and _tracked(bias):
            return None
        b, b_code = _plain(bias, device, dim)
        if weight is not None and b_code != param:
            return None
        param = b_code
    if code not in _FLOATS or (param != code and param != _F32):
        return None
    out = _empty_like(x)
    if len(shape) == 2:
        rows = shape[0]
        mean = x.new_empty(rows, dtype=_dtypes[_F32])
    else:
        rows = x.numel() // dim
        mean = x.new_empty(shape[:-1], dtype=_dtypes[_F32])
    rstd = _empty_like(mean)
    _call(_LIB.XGBBLayerNorm, _pack_layer_norm(
        v, w, b, out.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _raw_stream(device), rows, dim, dim, dim, code,
        param, device, eps))
    return out, mean, rstd


@_short_way
def _layer_norm_backward_short(grad, x, mean, rstd, weight, bias_grad):
    device = x.get_device()
    if device < 0:
        return None
    v, code = _plain(x, device)
    g, g_code = _plain(grad, device)
    m, m_code = _plain(mean, device)
    q, q_code = _plain(rstd, device)
    shape = x.shape
    dim = shape[-1]
    lead = shape[:-1]
    w, param = _plain(weight, device, dim)
    if code not in _FLOATS or g_code != code or grad.shape != shape or m_code != _F32 or q_code != _F32 or \
            mean.shape != lead or rstd.shape != lead or (param != code and param != _F32):
        return None
    rows = shape[0] if len(shape) == 2 else x.numel() // dim
    out, dweight = _empty_like(x), _empty_like(weight)
    dbias = _empty_like(weight) if bias_grad else None
    size = layer_norm_backward_workspace(rows, dim)
    space = x.new_empty(size, dtype=sys.modules["torch"].uint8) if size else None
    _call(_LIB.XGBBLayerNormBackward, _pack_layer_norm_backward(
        g, v, m, q, w, out.data_ptr(), dweight.data_ptr(), dbias.data_ptr() if bias_grad else 0,
        space.data_ptr() if size else 0, _raw_stream(device), size, rows, dim, dim, dim, dim, code, param, device))
    return out, dweight, dbias


def embedding(tokens, table, *, scale=1.0, token_scale=None, bag=False, out=None, out_dtype=None, stream=None):
    """scale * token_scale * table[tokens]: shape tokens.shape + (dim,), or
    with `bag` the sum over the tokens' last dimension, tokens.shape[:-1] +
    (dim,).

    A token below 0 is missing and adds nothing (a row of missing tokens is
    zeros); one past the table makes its row NaN. token_scale (float32)
    broadcasts to the tokens' shape. Sums are float32. The result has the
    table's type, or `out_dtype`; of the two types one is float32 or both are
    the same. Torch's autograd gets the gradients of table and token_scale."""
    if stream is not None and _tensors(tokens, table, token_scale, out):
        with _on(stream, (tokens, table, token_scale, out)):
            return embedding(tokens, table, scale=scale, token_scale=token_scale, bag=bag, out=out,
                             out_dtype=out_dtype)
    if out is None:
        got = _embedding_short(tokens, table, scale, token_scale, bag, out_dtype)
        if got is not None:
            return got
    if _tracked(table, token_scale):
        return _recorded("embedding", (tokens, table, _expand(token_scale, _view(tokens, "tokens")[1], bag)), (out,),
                         scale, bag, out_dtype)
    k, w = _view(tokens, "tokens"), _view(table, "table")
    rows, per_row, stride_row, stride_col, lead = _token_grid(k, bag)
    vocab, dim, table_stride = _matrix(w, "table")
    if len(w[1]) != 2:
        raise XGBoostError("table must have two dimensions")
    token_scale = _expand(token_scale, k[1], bag)
    s, s_row, s_col, s_device = _scale_grid(token_scale, k, bag)
    code = w[3] if out_dtype is None else _dtype_code(out_dtype)
    out, y, code, y_stride, y_device = _result(out, (*lead, dim), 0 if out is not None and out_dtype is None else code,
                                               w, "out")
    device = _one_device(w[4], k[4], s_device, y_device)
    handle = _handle(stream, device, tokens, table, token_scale, out)
    _call(_LIB.XGBBEmbedding, _pack_embedding(
        k[0], s, rows, per_row, stride_row, stride_col, s_row, s_col, k[3], scale, w[0], y,
        handle, vocab, dim, table_stride, y_stride, w[3], code, device))
    return out


@functools.lru_cache(maxsize=1024)
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
    if stream is not None and _tensors(grad, tokens, token_scale, out, workspace):
        with _on(stream, (grad, tokens, token_scale, out, workspace)):
            return embedding_backward(grad, tokens, vocab, scale=scale, token_scale=token_scale, bag=bag, out=out,
                                      out_dtype=out_dtype, accumulate=accumulate, workspace=workspace)
    if out is None and workspace is None and not accumulate:
        got = _embedding_backward_short(grad, tokens, vocab, scale, token_scale, bag, out_dtype)
        if got is not None:
            return got
    g, k = _view(grad, "grad"), _view(tokens, "tokens")
    rows, per_row, stride_row, stride_col, lead = _token_grid(k, bag)
    _, dim, g_stride = _matrix(g, "grad")
    if g[1][:-1] != lead:
        raise XGBoostError("grad must have the shape of the lookup's result")
    if accumulate and out is None:
        raise XGBoostError("accumulate needs out")
    token_scale = _expand(token_scale, k[1], bag)
    s, s_row, s_col, s_device = _scale_grid(token_scale, k, bag)
    size = embedding_backward_workspace(rows, per_row, vocab, dim)
    code = g[3] if out_dtype is None else _dtype_code(out_dtype)
    out, y, code, y_stride, y_device = _result(out, (vocab, dim), 0 if out is not None and out_dtype is None else code,
                                               g, "out")
    space, space_device = 0, -1
    if size:
        workspace, space, space_device = _space(workspace, size, g)
    device = _one_device(g[4], k[4], s_device, y_device, space_device)
    handle = _handle(stream, device, grad, tokens, token_scale, out, workspace)
    _call(_LIB.XGBBEmbeddingBackward, _pack_embedding_backward(
        k[0], s, rows, per_row, stride_row, stride_col, s_row, s_col, k[3], scale, g[0], y, space,
        handle, size, vocab, dim, g_stride, y_stride, g[3], code, bool(accumulate), device))
    return out


def embedding_scale_backward(grad, tokens, table, *, scale=1.0, bag=False, out=None, stream=None):
    """The gradient of embedding's token_scale, float32 in the tokens' shape: 0
    for a missing token, NaN for one past the table. (Where token_scale was
    broadcast, its own gradient is this one's sum over the broadcast
    dimensions.)"""
    if stream is not None and _tensors(grad, tokens, table, out):
        with _on(stream, (grad, tokens, table, out)):
            return embedding_scale_backward(grad, tokens, table, scale=scale, bag=bag, out=out)
    if out is None:
        got = _embedding_scale_backward_short(grad, tokens, table, scale, bag)
        if got is not None:
            return got
    g, k, w = _view(grad, "grad"), _view(tokens, "tokens"), _view(table, "table")
    rows, per_row, stride_row, stride_col, lead = _token_grid(k, bag)
    vocab, dim, table_stride = _matrix(w, "table")
    if len(w[1]) != 2:
        raise XGBoostError("table must have two dimensions")
    _, g_dim, g_stride = _matrix(g, "grad")
    if g[1][:-1] != lead or g_dim != dim:
        raise XGBoostError("grad must have the shape of the lookup's result")
    out, y, y_device = _flat_result(out, k[1], _F32, g, "out")
    device = _one_device(g[4], k[4], w[4], y_device)
    handle = _handle(stream, device, grad, tokens, table, out)
    _call(_LIB.XGBBEmbeddingScaleBackward, _pack_embedding_scale_backward(
        k[0], 0, rows, per_row, stride_row, stride_col, 0, 0, k[3], scale, g[0], w[0], y,
        handle, vocab, dim, g_stride, table_stride, g[3], w[3], device))
    return out


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, out=None, mean=None, rstd=None, stream=None):
    """(y, mean, rstd) of a layer norm over x's last dimension: y = (x - mean)
    * rstd * weight + bias in x's type, mean and rstd = 1 / sqrt(variance +
    eps) in float32, one a row. weight and bias have x's type or are float32,
    both the same. Torch's autograd gets y's gradients with respect to x, weight
    and bias; mean and rstd have none."""
    if stream is not None and _tensors(x, weight, bias, out, mean, rstd):
        with _on(stream, (x, weight, bias, out, mean, rstd)):
            return layer_norm(x, weight, bias, eps=eps, out=out, mean=mean, rstd=rstd)
    if out is None and mean is None and rstd is None:
        got = _layer_norm_short(x, weight, bias, eps)
        if got is not None:
            return got
    if _tracked(x, weight, bias):
        return _recorded("layer_norm", (x, weight, bias), (out, mean, rstd), eps)
    v = _view(x, "x")
    rows, dim, stride = _matrix(v, "x")
    w = b = None
    param, w_device, b_device = _F32, -1, -1
    if weight is not None:
        w, _, _, param, w_device, _ = _vector(weight, dim, v[3], "weight")
    if bias is not None:
        b, _, _, b_code, b_device, _ = _vector(bias, dim, v[3], "bias")
        if weight is not None and param != b_code:
            raise XGBoostError("weight and bias must have the same type")
        param = b_code
    lead = v[1][:-1]
    if out is None and v[5] is not None and x.is_contiguous():
        out = _empty_like(x)
        y, y_stride, y_device = out.data_ptr(), dim, v[4]
    else:
        out, y, _, y_stride, y_device = _result(out, v[1], v[3], v, "out")
    mean, m, m_device = _flat_result(mean, lead, _F32, v, "mean")
    rstd, q, q_device = _flat_result(rstd, lead, _F32, v, "rstd")
    device = _one_device(v[4], w_device, b_device, y_device, m_device, q_device)
    handle = _handle(stream, device, x, weight, bias, out, mean, rstd)
    _call(_LIB.XGBBLayerNorm, _pack_layer_norm(
        v[0], w or 0, b or 0, y, m, q, handle, rows, dim, stride, y_stride, v[3], param, device, eps))
    return out, mean, rstd


@functools.lru_cache(maxsize=1024)
def layer_norm_backward_workspace(rows, dim):
    """Bytes of workspace that layer_norm_backward needs for the gradients of
    weight and bias."""
    size = ctypes.c_size_t()
    _check_call(_LIB.XGBBLayerNormBackwardWorkspace(rows, dim, ctypes.byref(size)))
    return size.value


def layer_norm_backward(grad, x, mean, rstd, weight=None, *, bias_grad=True, out=None, dweight=None, dbias=None,
                        workspace=None, stream=None):
    """(dx, dweight, dbias) from the gradient `grad` of layer_norm's y and the
    mean and rstd that it returned. Without a weight dweight is None, and dbias
    too where no array for it is given (float32 or of x's type); without
    `bias_grad` dbias is None."""
    if stream is not None and _tensors(grad, x, mean, rstd, weight, out, dweight, dbias, workspace):
        with _on(stream, (grad, x, mean, rstd, weight, out, dweight, dbias, workspace)):
            return layer_norm_backward(grad, x, mean, rstd, weight, bias_grad=bias_grad, out=out, dweight=dweight,
                                       dbias=dbias, workspace=workspace)
    if weight is not None and out is None and dweight is None and dbias is None and workspace is None:
        got = _layer_norm_backward_short(grad, x, mean, rstd, weight, bias_grad)
        if got is not None:
            return got
    g, v = _view(grad, "grad"), _view(x, "x")
    rows, dim, stride = _matrix(v, "x")
    _, _, g_stride = _matrix(g, "grad")
    if g[1] != v[1] or g[3] != v[3]:
        raise XGBoostError("grad must have x's shape and type")
    lead = v[1][:-1]
    m, m_device = _row_values(mean, lead, "mean")
    q, q_device = _row_values(rstd, lead, "rstd")
    if out is None and v[5] is not None and x.is_contiguous():
        out = _empty_like(x)
        dx, dx_stride, dx_device = out.data_ptr(), dim, v[4]
    else:
        out, dx, _, dx_stride, dx_device = _result(out, v[1], v[3], v, "out")
    w = dw = db = space = size = 0
    w_code, w_device, dw_device, db_device, space_device = _F32, -1, -1, -1, -1
    if weight is not None:
        wv = _vector(weight, dim, v[3], "weight")
        w, _, _, w_code, w_device, _ = wv
        dweight, dw, dw_device = _flat_result(dweight, (dim,), w_code, wv, "dweight")
        if bias_grad:
            dbias, db, db_device = _flat_result(dbias, (dim,), w_code, wv, "dbias")
    elif dweight is not None:
        raise XGBoostError("dweight would need weight")
    elif dbias is not None and bias_grad:
        w_code = _F32 if _view(dbias, "dbias")[3] == _F32 else v[3]
        dbias, db, db_device = _flat_result(dbias, (dim,), w_code, v, "dbias")
    if dw or db:
        size = layer_norm_backward_workspace(rows, dim)
        if size:
            workspace, space, space_device = _space(workspace, size, v)
    device = _one_device(v[4], g[4], m_device, q_device, w_device, dx_device, dw_device, db_device, space_device)
    handle = _handle(stream, device, grad, x, mean, rstd, weight, out, dweight, dbias, workspace)
    _call(_LIB.XGBBLayerNormBackward, _pack_layer_norm_backward(
        g[0], v[0], m, q, w, dx, dw, db, space, handle, size, rows, dim, g_stride, stride,
        dx_stride, v[3], w_code, device))
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
