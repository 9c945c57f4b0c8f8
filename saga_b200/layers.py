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
import math

import torch

from . import capi
from .capi import check, lib

_DTYPES = {torch.float16: capi.HALF, torch.float32: capi.FLOAT}


def _dtype(t, what):
    if t.dtype not in _DTYPES:
        raise TypeError(f"{what} is {t.dtype}: float16 or float32 expected")
    return _DTYPES[t.dtype]


def _on(device, what, t):
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda" or t.device != device:
        raise ValueError(f"{what} must be a CUDA tensor on {device}")
    return t


def _cuda(t, what):
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise ValueError(f"{what} must be a CUDA tensor")
    return t.device


def _rows(t, what, cols=None, dtype=None):
    """(rows, row length, row stride) of a tensor seen as a matrix of its last dimension."""
    if t.dim() < 1:
        raise ValueError(f"{what} needs at least one dimension")
    if cols is not None and t.shape[-1] != cols:
        raise ValueError(f"{what} has rows of {t.shape[-1]} elements, {cols} expected")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what} is {t.dtype}, {dtype} expected")
    n, d = math.prod(t.shape[:-1]), t.shape[-1]
    if t.numel() == 0:
        return n, d, max(d, 1)
    if d > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what} must be contiguous in its last dimension")
    stride, expect = d, None
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
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


def _matrix(t, what, rows, cols, dtype, device):
    """Row stride of an output or gradient that must have the given shape."""
    _on(device, what, t)
    n, _, stride = _rows(t, what, cols, dtype)
    if n != rows:
        raise ValueError(f"{what} has {n} rows, {rows} expected")
    return stride


def _vector(t, what, n, dtype, device):
    if t is None:
        return None
    _on(device, what, t)
    if t.dtype != dtype:
        raise TypeError(f"{what} is {t.dtype}, {dtype} expected")
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous with {n} elements")
    return t.data_ptr()


def _index(t, what, device):
    _on(device, what, t)
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what} is {t.dtype}: int32 or int64 expected")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return t.data_ptr(), t.element_size()


class _Call:
    """Current device and stream of one call, and what it allocates."""

    def __init__(self, device, stream):
        self.device, self.raw = device, stream
        self.guard = torch.cuda.device(device)

    def __enter__(self):
        self.guard.__enter__()
        self.stream = (torch.cuda.current_stream(self.device).cuda_stream if self.raw is None
                       else self.raw)
        return self

    def __exit__(self, *exc):
        return self.guard.__exit__(*exc)

    def new(self, what, shape, dtype):
        if self.raw is not None:
            raise ValueError(f"pass {what} when a raw stream is given")
        return torch.empty(shape, dtype=dtype, device=self.device)

    def workspace(self, given, query, *sizes):
        """(tensor, address, bytes) of the caller's workspace or of a new one."""
        need = C.c_size_t()
        check(getattr(lib(), query)(*sizes, C.byref(need)))
        if given is None:
            given = self.new("workspace", (need.value,), torch.uint8) if need.value else None
        if given is None:
            return None, None, 0
        _on(self.device, "workspace", given)
        if not given.is_contiguous():
            raise ValueError("workspace must be contiguous")
        return given, given.data_ptr(), given.numel() * given.element_size()


def embedding_forward(ids, weight, scale=1.0, out=None, stream=None):
    """out[...] = scale * weight[ids[...]]; an id outside the table gives a row of zeros."""
    device = _cuda(weight, "weight")
    vocab, dim, ws = _rows(weight, "weight")
    dtype = _dtype(weight, "weight")
    ids_ptr, wide = _index(ids, "ids", device)
    with _Call(device, stream) as call:
        if out is None:
            out = call.new("out", (*ids.shape, dim), weight.dtype)
        os = _matrix(out, "out", ids.numel(), dim, weight.dtype, device)
        check(lib().b200opt_embedding_fwd(dtype, ids.numel(), vocab, dim, ids_ptr, wide,
                                          weight.data_ptr(), ws, scale, out.data_ptr(), os,
                                          call.stream))
    return out


def embedding_workspace(tokens, vocab, dim):
    """Bytes of workspace that embedding_backward needs."""
    need = C.c_size_t()
    check(lib().b200opt_embedding_bwd_workspace(tokens, vocab, dim, C.byref(need)))
    return need.value


def embedding_backward(ids, grad_out, vocab, scale=1.0, grad_weight=None, accumulate=False,
                       workspace=None, stream=None):
    """The dense gradient [vocab, dim] of the table; rows that no id names become zero, or keep
    their values with ``accumulate`` (which needs ``grad_weight``)."""
    device = _cuda(grad_out, "grad_out")
    tokens, dim, ys = _rows(grad_out, "grad_out")
    dtype = _dtype(grad_out, "grad_out")
    ids_ptr, wide = _index(ids, "ids", device)
    if ids.numel() != tokens and dim:
        raise ValueError(f"{ids.numel()} ids, but {tokens} rows in grad_out")
    if accumulate and grad_weight is None:
        raise ValueError("accumulate needs grad_weight")
    with _Call(device, stream) as call:
        if grad_weight is None:
            grad_weight = call.new("grad_weight", (vocab, dim), grad_out.dtype)
        gs = _matrix(grad_weight, "grad_weight", vocab, dim, grad_out.dtype, device)
        keep, wp, wb = call.workspace(workspace, "b200opt_embedding_bwd_workspace", tokens, vocab,
                                      dim)
        check(lib().b200opt_embedding_bwd(dtype, tokens, vocab, dim, ids_ptr, wide,
                                          grad_out.data_ptr(), ys, scale, grad_weight.data_ptr(),
                                          gs, int(accumulate), wp, wb, call.stream))
    return grad_weight


def layernorm_forward(x, gamma=None, beta=None, eps=1e-5, out=None, mean=None, rstd=None,
                      stream=None):
    """(y, mean, rstd) over the last dimension; mean and rstd are fp32, one per row."""
    device = _cuda(x, "x")
    rows, dim, xs = _rows(x, "x")
    dtype = _dtype(x, "x")
    given = gamma if gamma is not None else beta
    params = given.dtype if given is not None else torch.float32
    g = _vector(gamma, "gamma", dim, params, device)
    b = _vector(beta, "beta", dim, params, device)
    with _Call(device, stream) as call:
        out = call.new("out", x.shape, x.dtype) if out is None else out
        mean = call.new("mean", x.shape[:-1], torch.float32) if mean is None else mean
        rstd = call.new("rstd", x.shape[:-1], torch.float32) if rstd is None else rstd
        ys = _matrix(out, "out", rows, dim, x.dtype, device)
        check(lib().b200opt_layernorm_fwd(
            dtype, _dtype(given, "gamma") if given is not None else capi.FLOAT, rows, dim,
            x.data_ptr(), xs, g, b, eps, out.data_ptr(), ys,
            _vector(mean, "mean", rows, torch.float32, device),
            _vector(rstd, "rstd", rows, torch.float32, device), call.stream))
    return out, mean, rstd


def layernorm_workspace(rows, dim):
    """Bytes of workspace that layernorm_backward needs."""
    need = C.c_size_t()
    check(lib().b200opt_layernorm_bwd_workspace(rows, dim, C.byref(need)))
    return need.value


def layernorm_backward(grad_y, x, gamma, mean, rstd, grad_x=None, grad_gamma=None, grad_beta=None,
                       accumulate=False, workspace=None, stream=None):
    """(grad_x, grad_gamma, grad_beta); the last two in gamma's dtype (fp32 without gamma)."""
    device = _cuda(x, "x")
    rows, dim, xs = _rows(x, "x")
    dtype = _dtype(x, "x")
    params = gamma.dtype if gamma is not None else torch.float32
    g = _vector(gamma, "gamma", dim, params, device)
    ys = _matrix(grad_y, "grad_y", rows, dim, x.dtype, device)
    mu = _vector(mean, "mean", rows, torch.float32, device)
    rs = _vector(rstd, "rstd", rows, torch.float32, device)
    if accumulate and (grad_gamma is None or grad_beta is None):
        raise ValueError("accumulate needs grad_gamma and grad_beta")
    with _Call(device, stream) as call:
        grad_x = call.new("grad_x", x.shape, x.dtype) if grad_x is None else grad_x
        grad_gamma = call.new("grad_gamma", (dim,), params) if grad_gamma is None else grad_gamma
        grad_beta = call.new("grad_beta", (dim,), params) if grad_beta is None else grad_beta
        dxs = _matrix(grad_x, "grad_x", rows, dim, x.dtype, device)
        keep, wp, wb = call.workspace(workspace, "b200opt_layernorm_bwd_workspace", rows, dim)
        check(lib().b200opt_layernorm_bwd(
            dtype, _DTYPES.get(params, -1), rows, dim, grad_y.data_ptr(), ys, x.data_ptr(), xs, g,
            mu, rs, grad_x.data_ptr(), dxs, _vector(grad_gamma, "grad_gamma", dim, params, device),
            _vector(grad_beta, "grad_beta", dim, params, device), int(accumulate), wp, wb,
            call.stream))
    return grad_x, grad_gamma, grad_beta


def _head(hidden, weight, targets):
    device = _cuda(hidden, "hidden")
    _on(device, "weight", weight)
    tokens, dim, xs = _rows(hidden, "hidden", dtype=torch.float16)
    vocab, _, ws = _rows(weight, "weight", dim, torch.float16)
    y, wide = _index(targets, "targets", device)
    if targets.numel() != tokens:
        raise ValueError(f"{targets.numel()} targets, but {tokens} rows in hidden")
    return device, (tokens, vocab, dim), (hidden.data_ptr(), xs, weight.data_ptr(), ws, y, wide)


def vocab_loss_workspace(tokens, vocab, dim):
    """Bytes of workspace that (vocab_loss_forward, vocab_loss_backward) need."""
    a, b = C.c_size_t(), C.c_size_t()
    check(lib().b200opt_vocab_loss_fwd_workspace(tokens, vocab, dim, C.byref(a)))
    check(lib().b200opt_vocab_loss_bwd_workspace(tokens, vocab, dim, C.byref(b)))
    return a.value, b.value


def vocab_loss_forward(hidden, weight, targets, loss=None, lse=None, stats=None, workspace=None,
                       stream=None):
    """(loss, lse, stats) of softmax cross entropy with logits hidden @ weight.T, which are never
    stored.  loss and lse: fp32 per token; stats: fp32 {sum of losses, tokens counted}.  Targets
    outside the vocabulary are ignored."""
    device, sizes, args = _head(hidden, weight, targets)
    with _Call(device, stream) as call:
        loss = call.new("loss", targets.shape, torch.float32) if loss is None else loss
        lse = call.new("lse", targets.shape, torch.float32) if lse is None else lse
        stats = call.new("stats", (2,), torch.float32) if stats is None else stats
        keep, wp, wb = call.workspace(workspace, "b200opt_vocab_loss_fwd_workspace", *sizes)
        check(lib().b200opt_vocab_loss_fwd(
            *sizes, *args, _vector(loss, "loss", sizes[0], torch.float32, device),
            _vector(lse, "lse", sizes[0], torch.float32, device),
            _vector(stats, "stats", 2, torch.float32, device), wp, wb, call.stream))
    return loss, lse, stats


def vocab_loss_backward(hidden, weight, targets, lse, stats=None, grad_scale=1.0, loss_scale=None,
                        grad_hidden=None, grad_weight=None, accumulate=False, workspace=None,
                        stream=None):
    """(grad_hidden, grad_weight) of the losses' mean (``stats`` of the forward pass given) or sum,
    times grad_scale and times the loss scale: a one-element fp32 tensor, or a device address such
    as ``AdamGroup.device_scale_ptr()`` returns."""
    device, sizes, args = _head(hidden, weight, targets)
    tokens, vocab, dim = sizes
    lse_ptr = _vector(lse, "lse", tokens, torch.float32, device)
    stats_ptr = _vector(stats, "stats", 2, torch.float32, device)
    scale_ptr = (loss_scale if loss_scale is None or isinstance(loss_scale, int)
                 else _vector(loss_scale, "loss_scale", 1, torch.float32, device))
    if accumulate and grad_weight is None:
        raise ValueError("accumulate needs grad_weight")
    with _Call(device, stream) as call:
        if grad_hidden is None:
            grad_hidden = call.new("grad_hidden", hidden.shape, torch.float16)
        if grad_weight is None:
            grad_weight = call.new("grad_weight", weight.shape, torch.float16)
        xs = _matrix(grad_hidden, "grad_hidden", tokens, dim, torch.float16, device)
        ws = _matrix(grad_weight, "grad_weight", vocab, dim, torch.float16, device)
        keep, wp, wb = call.workspace(workspace, "b200opt_vocab_loss_bwd_workspace", *sizes)
        check(lib().b200opt_vocab_loss_bwd(
            *sizes, *args, lse_ptr, stats_ptr, grad_scale, scale_ptr, grad_hidden.data_ptr(), xs,
            grad_weight.data_ptr(), ws, int(accumulate), wp, wb, call.stream))
    return grad_hidden, grad_weight
