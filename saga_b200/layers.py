"""The language-model operators of the b200opt C ABI on torch tensors.

Embedding lookup, layer norm and the vocabulary loss (softmax cross entropy with
the classifier's product), forward and gradient.  These are plain calls, without
autograd: a training step calls the forward functions, then the backward ones
with what the forward ones returned, and lets the parameters' gradients land in
the gradient buffers of an ``AdamGroup`` (``grad_weight=`` and the like take
tensors made from ``AdamGroup.buffers``), which ``AdamGroup.exec`` reads.

Tensors must be CUDA tensors of one device with a contiguous last dimension;
leading dimensions are flattened where that needs no copy.  fp16 and fp32, the
optimizer's two groups.  A call runs on torch's current stream of that device,
or on the raw CUDA stream given as ``stream``; it allocates what the caller does
not pass (outputs, workspace) from torch's allocator, which is refused for a raw
stream, because that allocator would not know of it.
"""
import ctypes as C
import functools
import math

import torch

from . import capi
from .capi import check, lib

_DTYPES = {torch.float16: capi.HALF, torch.float32: capi.FLOAT}
_raw_stream = torch._C._cuda_getCurrentRawStream     # what current_stream().cuda_stream is, without the object


def _dtype(t, what):
    kind = _DTYPES.get(t.dtype)
    if kind is None:
        raise TypeError(f"{what} is {t.dtype}: float16 or float32 expected")
    return kind


def _device(t, what):
    """Index of the CUDA device that the tensor is on."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    return t.get_device()


def _on(index, what, t):
    if _device(t, what) != index:
        raise ValueError(f"{what} must be on cuda:{index}")


def _rows(t, what, cols=None, dtype=None):
    """(rows, row length, row stride) of a tensor seen as a matrix of its last dimension."""
    shape = t.shape
    if not shape:
        raise ValueError(f"{what} needs at least one dimension")
    d = shape[-1]
    if cols is not None and d != cols:
        raise ValueError(f"{what} has rows of {d} elements, {cols} expected")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what} is {t.dtype}, {dtype} expected")
    n = math.prod(shape[:-1])
    if n == 0 or d == 0 or t.is_contiguous():
        return n, d, max(d, 1)
    strides = t.stride()
    if d > 1 and strides[-1] != 1:
        raise ValueError(f"{what} must be contiguous in its last dimension")
    stride, expect = d, None
    for size, step in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if expect is None:
            stride = step
        elif step != expect:
            raise ValueError(f"{what} cannot be seen as a matrix without a copy")
        expect = step * size
    if n > 1 and stride < d:
        raise ValueError(f"{what} has rows that overlap")
    return n, d, max(stride, d)


def _matrix(t, what, rows, cols, dtype, index):
    """Row stride of an output or gradient that must have the given shape."""
    _on(index, what, t)
    n, _, stride = _rows(t, what, cols, dtype)
    if n != rows:
        raise ValueError(f"{what} has {n} rows, {rows} expected")
    return stride


def _vector(t, what, n, dtype, index):
    if t is None:
        return None
    _on(index, what, t)
    if t.dtype != dtype:
        raise TypeError(f"{what} is {t.dtype}, {dtype} expected")
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous with {n} elements")
    return t.data_ptr()


def _vector_out(t, what, shape, n, dtype, like, index, stream):
    """(tensor, address) of a vector that a call fills: the caller's, or a new one (made after
    `like` where that is such a vector already, which is cheaper)."""
    if t is None:
        t = (_new_like(like, what, stream) if like.dtype == dtype and like.shape == shape
             else _new(like, shape, dtype, what, stream))
        return t, t.data_ptr()
    return t, _vector(t, what, n, dtype, index)


def _index(t, what, index):
    _on(index, what, t)
    if t.dtype != torch.int64 and t.dtype != torch.int32:
        raise TypeError(f"{what} is {t.dtype}: int32 or int64 expected")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return t.data_ptr(), t.element_size()


def _new(like, shape, dtype, what, stream):
    if stream is not None:
        raise ValueError(f"pass {what} when a raw stream is given")
    return like.new_empty(shape, dtype=dtype)


def _new_like(t, what, stream):
    """A contiguous tensor of t's shape and type."""
    if stream is not None:
        raise ValueError(f"pass {what} when a raw stream is given")
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


@functools.lru_cache(maxsize=1024)
def _bytes(query, *sizes):
    """What a _workspace function says: it depends on the sizes alone."""
    need = C.c_size_t()
    check(getattr(lib(), query)(*sizes, C.byref(need)))
    return need.value


def _workspace(given, need, like, index, stream):
    """(tensor, address, bytes) of the caller's workspace or of a new one."""
    if given is None:
        if not need:
            return None, None, 0
        given = _new(like, (need,), torch.uint8, "workspace", stream)
    else:
        _on(index, "workspace", given)
        if not given.is_contiguous():
            raise ValueError("workspace must be contiguous")
    return given, given.data_ptr(), given.numel() * given.element_size()


def _call(function, index, stream, *args):
    """Runs a C entry with the tensors' device current, on the given or torch's current stream."""
    if torch._C._cuda_getDevice() == index:
        check(function(*args, _raw_stream(index) if stream is None else stream))
    else:
        with torch.cuda.device(index):
            check(function(*args, _raw_stream(index) if stream is None else stream))


def embedding_forward(ids, weight, scale=1.0, out=None, stream=None):
    """out[...] = scale * weight[ids[...]]; an id outside the table gives a row of zeros."""
    dev = _device(weight, "weight")
    vocab, dim, ws = _rows(weight, "weight")
    dtype = _dtype(weight, "weight")
    ids_ptr, wide = _index(ids, "ids", dev)
    tokens = ids.numel()
    if out is None:
        out, os = _new(weight, (*ids.shape, dim), weight.dtype, "out", stream), max(dim, 1)
    else:
        os = _matrix(out, "out", tokens, dim, weight.dtype, dev)
    _call(lib().b200opt_embedding_fwd, dev, stream, dtype, tokens, vocab, dim, ids_ptr, wide,
          weight.data_ptr(), ws, scale, out.data_ptr(), os)
    return out


def embedding_workspace(tokens, vocab, dim):
    """Bytes of workspace that embedding_backward needs."""
    return _bytes("b200opt_embedding_bwd_workspace", tokens, vocab, dim)


def embedding_backward(ids, grad_out, vocab, scale=1.0, grad_weight=None, accumulate=False,
                       workspace=None, stream=None):
    """The dense gradient [vocab, dim] of the table; rows that no id names become zero, or keep
    their values with ``accumulate`` (which needs ``grad_weight``)."""
    dev = _device(grad_out, "grad_out")
    tokens, dim, ys = _rows(grad_out, "grad_out")
    dtype = _dtype(grad_out, "grad_out")
    ids_ptr, wide = _index(ids, "ids", dev)
    if ids.numel() != tokens:
        raise ValueError(f"{ids.numel()} ids, but {tokens} rows in grad_out")
    if grad_weight is not None:
        gs = _matrix(grad_weight, "grad_weight", vocab, dim, grad_out.dtype, dev)
    elif accumulate:
        raise ValueError("accumulate needs grad_weight")
    else:
        grad_weight = _new(grad_out, (vocab, dim), grad_out.dtype, "grad_weight", stream)
        gs = max(dim, 1)
    keep, wp, wb = _workspace(workspace, embedding_workspace(tokens, vocab, dim), grad_out, dev, stream)
    _call(lib().b200opt_embedding_bwd, dev, stream, dtype, tokens, vocab, dim, ids_ptr, wide,
          grad_out.data_ptr(), ys, scale, grad_weight.data_ptr(), gs, int(accumulate), wp, wb)
    return grad_weight


def layernorm_forward(x, gamma=None, beta=None, eps=1e-5, out=None, mean=None, rstd=None,
                      stream=None):
    """(y, mean, rstd) over the last dimension; mean and rstd are fp32, one per row."""
    dev = _device(x, "x")
    rows, dim, xs = _rows(x, "x")
    dtype = _dtype(x, "x")
    given = gamma if gamma is not None else beta
    params = given.dtype if given is not None else torch.float32
    if out is None:
        out, ys = _new_like(x, "out", stream), max(dim, 1)
    else:
        ys = _matrix(out, "out", rows, dim, x.dtype, dev)
    mean, mp = _vector_out(mean, "mean", x.shape[:-1], rows, torch.float32, x, dev, stream)
    rstd, rp = _vector_out(rstd, "rstd", x.shape[:-1], rows, torch.float32, mean, dev, stream)
    _call(lib().b200opt_layernorm_fwd, dev, stream, dtype, _DTYPES.get(params, -1), rows, dim,
          x.data_ptr(), xs, _vector(gamma, "gamma", dim, params, dev),
          _vector(beta, "beta", dim, params, dev), eps, out.data_ptr(), ys, mp, rp)
    return out, mean, rstd


def layernorm_workspace(rows, dim):
    """Bytes of workspace that layernorm_backward needs."""
    return _bytes("b200opt_layernorm_bwd_workspace", rows, dim)


def layernorm_backward(grad_y, x, gamma, mean, rstd, grad_x=None, grad_gamma=None, grad_beta=None,
                       accumulate=False, workspace=None, stream=None):
    """(grad_x, grad_gamma, grad_beta); the last two in gamma's dtype (fp32 without gamma)."""
    dev = _device(x, "x")
    rows, dim, xs = _rows(x, "x")
    dtype = _dtype(x, "x")
    params = gamma.dtype if gamma is not None else torch.float32
    ys = _matrix(grad_y, "grad_y", rows, dim, x.dtype, dev)
    if accumulate and (grad_gamma is None or grad_beta is None):
        raise ValueError("accumulate needs grad_gamma and grad_beta")
    if grad_x is None:
        grad_x, dxs = _new_like(x, "grad_x", stream), max(dim, 1)
    else:
        dxs = _matrix(grad_x, "grad_x", rows, dim, x.dtype, dev)
    grad_gamma, gp = _vector_out(grad_gamma, "grad_gamma", (dim,), dim, params, x, dev, stream)
    grad_beta, bp = _vector_out(grad_beta, "grad_beta", (dim,), dim, params, grad_gamma, dev, stream)
    keep, wp, wb = _workspace(workspace, layernorm_workspace(rows, dim), x, dev, stream)
    _call(lib().b200opt_layernorm_bwd, dev, stream, dtype, _DTYPES.get(params, -1), rows, dim,
          grad_y.data_ptr(), ys, x.data_ptr(), xs, _vector(gamma, "gamma", dim, params, dev),
          _vector(mean, "mean", rows, torch.float32, dev),
          _vector(rstd, "rstd", rows, torch.float32, dev), grad_x.data_ptr(), dxs, gp, bp,
          int(accumulate), wp, wb)
    return grad_x, grad_gamma, grad_beta


def _head(hidden, weight, targets):
    dev = _device(hidden, "hidden")
    _on(dev, "weight", weight)
    tokens, dim, xs = _rows(hidden, "hidden", dtype=torch.float16)
    vocab, _, ws = _rows(weight, "weight", dim, torch.float16)
    y, wide = _index(targets, "targets", dev)
    if targets.numel() != tokens:
        raise ValueError(f"{targets.numel()} targets, but {tokens} rows in hidden")
    return dev, (tokens, vocab, dim), (hidden.data_ptr(), xs, weight.data_ptr(), ws, y, wide)


def vocab_loss_workspace(tokens, vocab, dim):
    """Bytes of workspace that (vocab_loss_forward, vocab_loss_backward) need."""
    return (_bytes("b200opt_vocab_loss_fwd_workspace", tokens, vocab, dim),
            _bytes("b200opt_vocab_loss_bwd_workspace", tokens, vocab, dim))


def vocab_loss_forward(hidden, weight, targets, loss=None, lse=None, stats=None, workspace=None,
                       stream=None):
    """(loss, lse, stats) of softmax cross entropy with logits hidden @ weight.T, which are never
    stored.  loss and lse: fp32 per token; stats: fp32 {sum of losses, tokens counted}.  Targets
    outside the vocabulary are ignored."""
    dev, sizes, args = _head(hidden, weight, targets)
    n, shape, f32 = sizes[0], targets.shape, torch.float32
    loss, lp = _vector_out(loss, "loss", shape, n, f32, hidden, dev, stream)
    lse, ep = _vector_out(lse, "lse", shape, n, f32, loss, dev, stream)
    stats, sp = _vector_out(stats, "stats", (2,), 2, f32, hidden, dev, stream)
    keep, wp, wb = _workspace(workspace, _bytes("b200opt_vocab_loss_fwd_workspace", *sizes), hidden,
                              dev, stream)
    _call(lib().b200opt_vocab_loss_fwd, dev, stream, *sizes, *args, lp, ep, sp, wp, wb)
    return loss, lse, stats


def _scale_address(t, index):
    """Device address of the loss scale; None where there is none."""
    if t is None:
        return None
    if isinstance(t, capi.DeviceAddress):
        if not t:
            raise ValueError("loss_scale is the null address: None stands for no loss scale")
        return t
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"loss_scale is a {type(t).__name__}: a one-element CUDA tensor or a "
                        "capi.DeviceAddress expected (give a number as grad_scale)")
    return _vector(t, "loss_scale", 1, torch.float32, index)


def vocab_loss_backward(hidden, weight, targets, lse, stats=None, grad_scale=1.0, loss_scale=None,
                        grad_hidden=None, grad_weight=None, accumulate=False, workspace=None,
                        stream=None):
    """(grad_hidden, grad_weight) of the losses' mean (``stats`` of the forward pass given) or sum,
    times grad_scale and times the loss scale: a one-element fp32 tensor, or a
    ``capi.DeviceAddress`` such as ``AdamGroup.device_scale_ptr()`` returns.  A scale that the host
    knows, a plain number, is part of grad_scale."""
    dev, sizes, args = _head(hidden, weight, targets)
    scale_ptr = _scale_address(loss_scale, dev)
    tokens, vocab, dim = sizes
    if accumulate and grad_weight is None:
        raise ValueError("accumulate needs grad_weight")
    if grad_hidden is None:
        grad_hidden = _new_like(hidden, "grad_hidden", stream)
        xs = dim
    else:
        xs = _matrix(grad_hidden, "grad_hidden", tokens, dim, torch.float16, dev)
    if grad_weight is None:
        grad_weight = _new_like(weight, "grad_weight", stream)
        ws = dim
    else:
        ws = _matrix(grad_weight, "grad_weight", vocab, dim, torch.float16, dev)
    keep, wp, wb = _workspace(workspace, _bytes("b200opt_vocab_loss_bwd_workspace", *sizes), hidden,
                              dev, stream)
    _call(lib().b200opt_vocab_loss_bwd, dev, stream, *sizes, *args,
          _vector(lse, "lse", tokens, torch.float32, dev),
          _vector(stats, "stats", 2, torch.float32, dev), grad_scale, scale_ptr,
          grad_hidden.data_ptr(), xs, grad_weight.data_ptr(), ws, int(accumulate), wp, wb)
    return grad_hidden, grad_weight
