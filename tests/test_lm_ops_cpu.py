"""Refusals of the language-model operators: decided on the host, before any CUDA call."""
import ctypes as C
import os

import pytest
import torch

from saga_b200 import capi, layers

A = 1 << 20          # stands for an aligned device address; a refused call never reads it
BIG = capi.LM_MAX + 1


def _call(name, defaults, **changed):
    assert not set(changed) - set(defaults)
    return getattr(capi.lib(), name)(*{**defaults, **changed}.values())


def _need(name, *sizes):
    n = C.c_size_t(7)
    assert getattr(capi.lib(), name)(*sizes, C.byref(n)) == capi.OK
    assert n.value % 4 == 0
    return n.value


EMB_FWD = dict(dtype=capi.HALF, tokens=5, vocab=10, dim=16, ids=A, ib=8, w=A, ws=16, scale=1.0,
               out=A, os=16, stream=None)
EMB_BWD = dict(dtype=capi.HALF, tokens=500, vocab=10, dim=16, ids=A, ib=8, dy=A, ys=16, scale=1.0,
               dw=A, ws=16, acc=0, wk=A, wb=1 << 40, stream=None)
LN_FWD = dict(dtype=capi.HALF, pdtype=capi.HALF, rows=5, dim=16, x=A, xs=16, g=A, b=A, eps=1e-5,
              y=A, ys=16, mean=A, rstd=A, stream=None)
LN_BWD = dict(dtype=capi.HALF, pdtype=capi.HALF, rows=5, dim=16, dy=A, ys=16, x=A, xs=16, g=A,
              mean=A, rstd=A, dx=A, dxs=16, dg=A, db=A, acc=0, wk=A, wb=1 << 40, stream=None)
VL_FWD = dict(tokens=5, vocab=10, dim=16, x=A, xs=16, w=A, ws=16, y=A, ib=8, loss=A, lse=A,
              stats=A, wk=A, wb=1 << 40, stream=None)
VL_BWD = dict(tokens=5, vocab=10, dim=16, x=A, xs=16, w=A, ws=16, y=A, ib=8, lse=A, stats=A,
              gs=1.0, ls=A, dx=A, dxs=16, dw=A, dws=16, acc=0, wk=A, wb=1 << 40, stream=None)

REFUSED = [
    ("b200opt_embedding_fwd", EMB_FWD, [
        dict(dtype=2), dict(dtype=-1), dict(ib=2), dict(ids=None), dict(ids=A + 4), dict(w=None),
        dict(w=A + 1), dict(ws=15), dict(out=None), dict(out=A + 1), dict(os=15), dict(os=1 << 62)]),
    ("b200opt_embedding_bwd", EMB_BWD, [
        dict(dtype=2), dict(ib=0), dict(ids=None), dict(dy=None), dict(dy=A + 1), dict(ys=15),
        dict(dw=None), dict(dw=A + 1), dict(ws=15), dict(ws=1 << 62)]),
    ("b200opt_layernorm_fwd", LN_FWD, [
        dict(dtype=2), dict(pdtype=2), dict(dtype=capi.FLOAT), dict(x=None), dict(x=A + 1),
        dict(xs=15), dict(y=None), dict(y=A + 1), dict(ys=15), dict(g=A + 1), dict(b=A + 1),
        dict(eps=-1.0), dict(eps=float("nan")), dict(mean=A + 2), dict(rstd=A + 2)]),
    ("b200opt_layernorm_bwd", LN_BWD, [
        dict(dtype=2), dict(pdtype=2), dict(dtype=capi.FLOAT), dict(x=None), dict(xs=15),
        dict(dy=None), dict(dy=A + 1), dict(ys=15), dict(mean=None), dict(rstd=None),
        dict(mean=A + 2), dict(dx=A + 1), dict(dxs=15), dict(g=A + 1), dict(dg=A + 1),
        dict(db=A + 1)]),
    ("b200opt_vocab_loss_fwd", VL_FWD, [
        dict(vocab=0), dict(dim=0), dict(dim=12), dict(x=None), dict(x=A + 8), dict(xs=20),
        dict(xs=8), dict(w=None), dict(w=A + 8), dict(ws=20), dict(ws=8), dict(y=None),
        dict(y=A + 4), dict(ib=2), dict(loss=None), dict(lse=None), dict(loss=A + 2),
        dict(stats=A + 2)]),
    ("b200opt_vocab_loss_bwd", VL_BWD, [
        dict(vocab=0), dict(dim=0), dict(dim=12), dict(x=None), dict(x=A + 8), dict(xs=20),
        dict(w=None), dict(ws=8), dict(y=None), dict(ib=2), dict(lse=None), dict(lse=A + 2),
        dict(ls=A + 2), dict(dx=A + 8), dict(dxs=20), dict(dxs=8), dict(dw=A + 8), dict(dws=20),
        dict(dws=8)]),
]


@pytest.mark.parametrize("name,defaults,changes", REFUSED, ids=[r[0] for r in REFUSED])
def test_bad_arguments_are_refused(built_library, name, defaults, changes):
    for change in changes:
        assert _call(name, defaults, **change) == capi.EINVAL, change
    for key in ("tokens", "rows", "vocab", "dim"):
        if key in defaults:
            assert _call(name, defaults, **{key: BIG}) == capi.ETOOBIG, key


@pytest.mark.parametrize("name,defaults,sizes", [
    ("b200opt_embedding_bwd", EMB_BWD, ("tokens", "vocab", "dim")),
    ("b200opt_layernorm_bwd", LN_BWD, ("rows", "dim")),
    ("b200opt_vocab_loss_fwd", VL_FWD, ("tokens", "vocab", "dim")),
    ("b200opt_vocab_loss_bwd", VL_BWD, ("tokens", "vocab", "dim"))])
def test_workspace_is_checked(built_library, name, defaults, sizes):
    shape = [defaults[k] for k in sizes]
    query = name + "_workspace"
    need = _need(query, *shape)
    if need:
        assert _call(name, defaults, wb=need - 1) == capi.EINVAL
        assert _call(name, defaults, wk=None) == capi.EINVAL
        assert _call(name, defaults, wk=A + 128) == capi.EINVAL
    fn = getattr(capi.lib(), query)
    assert fn(*shape, None) == capi.EINVAL
    n = C.c_size_t()
    assert fn(*([BIG] + shape[1:]), C.byref(n)) == capi.ETOOBIG
    # no tokens is a size too
    assert _need(query, *([0] + shape[1:])) <= need
    # larger sizes never need less
    assert _need(query, *[8 * s for s in shape]) >= need


def test_empty_calls_do_nothing(built_library):
    """Nothing to do: OK without a GPU, whatever the pointers."""
    none = dict(ids=None, w=None, out=None)
    assert _call("b200opt_embedding_fwd", EMB_FWD, tokens=0, **none) == capi.OK
    assert _call("b200opt_embedding_fwd", EMB_FWD, dim=0, **none) == capi.OK
    assert _call("b200opt_embedding_bwd", EMB_BWD, vocab=0, dw=None) == capi.OK
    assert _call("b200opt_vocab_loss_fwd", VL_FWD, tokens=0, stats=None, x=None, y=None) == capi.OK
    assert _call("b200opt_vocab_loss_bwd", VL_BWD, tokens=0, dw=None, x=None, y=None) == capi.OK
    assert _call("b200opt_layernorm_fwd", LN_FWD, rows=0, x=None, y=None) == capi.OK
    assert _call("b200opt_layernorm_bwd", LN_BWD, dim=0, x=None, dy=None) == capi.OK


def test_tensor_checks():
    """The Python layer refuses what it cannot hand on, before it loads anything."""
    cpu = torch.zeros(4, 8)
    with pytest.raises(ValueError):
        layers.embedding_forward(torch.zeros(3, dtype=torch.int64), cpu)
    with pytest.raises(ValueError):
        layers.layernorm_forward(cpu)
    with pytest.raises(ValueError):
        layers.vocab_loss_forward(cpu.half(), cpu.half(), torch.zeros(4, dtype=torch.int64))
    # what a matrix is: rows of one stride, contiguous elements
    t = torch.zeros(6, 10, 16)
    assert layers._rows(t, "t") == (60, 16, 16)
    assert layers._rows(t[..., :8], "t") == (60, 8, 16)
    assert layers._rows(t[:, :1, :8], "t") == (6, 8, 160)
    assert layers._rows(t[:, ::2], "t") == (30, 16, 32)
    assert layers._rows(t[2, 3], "t") == (1, 16, 16)
    assert layers._rows(torch.zeros(3, 0), "t") == (3, 0, 1)
    for bad in (t[..., ::2], t[:, 1:9:3], t.transpose(0, 1), torch.zeros(1, 8).expand(4, 8),
                torch.zeros(())):
        with pytest.raises(ValueError):
            layers._rows(bad, "t")


def test_loss_scale_that_is_a_number_is_refused():
    """A number is not an address: only a tensor, or a value that says it is one, is read from."""
    for number in (1024, 0, True, 1024.0, C.c_float(1.0)):
        with pytest.raises(TypeError, match="grad_scale"):
            layers._scale_address(number, 0)
    with pytest.raises(ValueError):
        layers._scale_address(torch.ones(1), 0)          # not on a GPU
    with pytest.raises(ValueError, match="null"):
        layers._scale_address(capi.DeviceAddress(0), 0)
    assert layers._scale_address(None, 0) is None
    assert layers._scale_address(capi.DeviceAddress(A), 0) == A


def test_no_kernel_takes_its_lanes_from_what_happens_to_run():
    """__activemask is whatever lanes arrived together, which CUDA does not promise to be all that took
    a branch: ranks and counts made from it could split a warp's tokens."""
    csrc = os.path.join(os.path.dirname(capi.LIB_PATH), "csrc")
    for name in sorted(os.listdir(csrc)):
        with open(os.path.join(csrc, name)) as f:
            assert "__activemask" not in f.read(), name
