"""The language-model operators on a GPU against their definitions in 64 bits.

Tolerances are error bounds, element by element.  u = 2^-24 is half a step of
fp32.  A sum of n terms that no addend passes more than h additions of is off by
at most h u times the sum of the magnitudes; h <= n always, and the bounds below
use h = n where n is small and the length of the longest chain otherwise.
Results in fp16 are off by half a step, 2^-11 of their size (2^-25 below the
normal range).  SLACK covers the products of such terms and the few steps of exp,
log, division and square root that a bound does not name one by one.
"""
import ctypes as C
import os
import subprocess
import sys
import threading

import pytest
import torch

from saga_b200 import AdamGroup, FlatLayout, capi, layers

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SLACK = 1.05
DEV = "cuda:0"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def normal(g, *shape, std=1.0, mean=0.0, dtype=torch.float16):
    return torch.empty(*shape, device=DEV).normal_(mean, std, generator=g).to(dtype)


def integers(g, n, low, high, dtype=torch.int64):
    return torch.randint(low, high, (n,), generator=g, device=DEV).to(dtype)


def half_step(exact, dtype):
    """What the last rounding may be off by."""
    if dtype == torch.float16:
        return exact.abs() * 2.0 ** -11 + 2.0 ** -25
    return exact.abs() * U + 2.0 ** -149


def close(got, exact, tol):
    assert got.shape == exact.shape
    off = (got.double() - exact).abs()
    bad = ~(off <= tol * SLACK)
    assert not bad.any(), (int(bad.sum()), float(off[bad].max()), float((off / (tol + 1e-300)).max()))


def strided(t, stride, shift=0):
    """A copy of the matrix with another row stride, `shift` elements off its allocation's start,
    between guard values; and a check that nothing around its rows was written."""
    rows, cols = t.shape
    buf = torch.full((shift + rows * stride + 16,), 77.0, device=DEV, dtype=t.dtype)
    view = torch.as_strided(buf, (rows, cols), (stride, 1), shift)
    view.copy_(t)

    def untouched():
        keep = view.clone()
        view.fill_(77.0)
        ok = bool((buf == 77.0).all())
        view.copy_(keep)
        return ok
    return view, untouched


# ----------------------------------------------------------------- embedding

EMB_SIZES = [  # tokens, vocab, dim
    (1, 1, 1), (1, 1000, 64), (7, 3, 5), (64, 1000, 333), (1000, 17, 40), (1025, 5003, 96),
    (300, 300, 1032), (2049, 1, 24), (33, 70001, 8), (20011, 211, 16), (50, 700, 2304), (40, 20, 70000),
    (128, 1000, 333), (129, 1000, 333), (100, 50021, 520), (120, 5, 2304), (300, 700, 2304),
    (2048, 3000, 1032), (1500, 40, 4104), (129, 64000, 600), (40961, 90001, 16), (70000, 3, 8), (33000, 300000, 8)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,vocab,dim", EMB_SIZES)
def test_embedding_forward(tokens, vocab, dim, dtype):
    g = gen(tokens + vocab)
    w = normal(g, vocab, dim, dtype=dtype)
    ids = integers(g, tokens, -1, vocab + 1, torch.int32 if tokens % 2 else torch.int64)
    out, clean = strided(torch.zeros(tokens, dim, device=DEV, dtype=dtype), dim + 3, 1)
    layers.embedding_forward(ids, w, scale=1.7, out=out)
    ok = (ids >= 0) & (ids < vocab)
    scale = float(torch.tensor(1.7, dtype=torch.float32))
    exact = w[torch.where(ok, ids, 0).long()].double() * scale * ok[:, None]
    close(out, exact, exact.abs() * U + half_step(exact, dtype))
    assert (out[~ok] == 0).all() and clean()
    same = layers.embedding_forward(ids, w, scale=1.7)
    assert torch.equal(same, out)


def embedding_exact(ids, dy, vocab, scale):
    ok = (ids >= 0) & (ids < vocab)
    at = torch.where(ok, ids, 0).long()
    scale = float(torch.tensor(scale, dtype=torch.float32))
    d = dy.double() * ok[:, None]
    zero = torch.zeros(vocab, dy.shape[1], device=DEV, dtype=torch.float64)
    n = torch.zeros(vocab, device=DEV, dtype=torch.float64).index_add_(0, at, ok.double())
    exact = zero.index_add(0, at, d) * scale
    size = zero.index_add(0, at, d.abs()) * abs(scale)
    return exact, size * ((n + 1) * U)[:, None], n      # at most n additions, one product


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,vocab,dim", EMB_SIZES)
def test_embedding_backward(tokens, vocab, dim, dtype):
    g = gen(2 * tokens + vocab)
    dy, _ = strided(normal(g, tokens, dim, dtype=dtype), dim + 1, 1)
    ids = integers(g, tokens, -1, vocab + 1, torch.int64 if tokens % 2 else torch.int32)
    ids[tokens // 2:] = ids[tokens // 2].clone()              # one token has at least half of all places
    exact, tol, n = embedding_exact(ids, dy, vocab, 0.75)
    dw, clean = strided(torch.full((vocab, dim), float("nan"), device=DEV, dtype=dtype), dim + 2, 3)
    layers.embedding_backward(ids, dy, vocab, scale=0.75, grad_weight=dw)
    close(dw, exact, tol + half_step(exact, dtype))
    assert (dw[n == 0] == 0).all() and clean()
    again = layers.embedding_backward(ids, dy, vocab, scale=0.75)
    assert torch.equal(again, dw)                     # the same bits, whatever ran when
    # accumulating: rows without a token are not touched, not even a NaN
    base = normal(g, vocab, dim, dtype=dtype)
    base[n == 0] = float("nan")
    got = layers.embedding_backward(ids, dy, vocab, scale=0.75, grad_weight=base.clone(), accumulate=True)
    assert torch.equal(got[n == 0].isnan(), base[n == 0].isnan())
    total = exact + base.double()
    close(got[n > 0], total[n > 0], (tol + total.abs() * U + half_step(total, dtype))[n > 0])


@pytest.mark.parametrize("pattern", ["none", "all the same", "sorted", "reversed", "two", "one block"])
@pytest.mark.parametrize("tokens", [31, 32, 33, 127, 128, 129, 4096, 16384, 16385, 32769, 40000])
def test_embedding_backward_orders(tokens, pattern):
    """Orders of ids that leave a sort or a split of a long run nothing to hide behind."""
    g, vocab, dim = gen(tokens), 30011, 24
    dy = normal(g, tokens, dim)
    ids = {"none": lambda: torch.full((tokens,), -100, device=DEV),
           "all the same": lambda: torch.full((tokens,), vocab - 1, device=DEV),
           "sorted": lambda: integers(g, tokens, 0, vocab).sort().values,
           "reversed": lambda: integers(g, tokens, 0, vocab).sort(descending=True).values,
           "two": lambda: torch.where(integers(g, tokens, 0, 2) > 0, 29999, 3),
           "one block": lambda: torch.arange(tokens, device=DEV) % 50 * (593 if tokens <= 128 else 148)}[pattern]()
    exact, tol, n = embedding_exact(ids, dy, vocab, 1.0)
    close(layers.embedding_backward(ids, dy, vocab), exact, tol + half_step(exact, dy.dtype))


def test_embedding_non_finite_values_stay_in_their_rows():
    ids = torch.tensor([5, 6, 5, 9], device=DEV)
    dy = torch.ones(4, 40, device=DEV)
    dy[1], dy[3, 7] = float("nan"), float("inf")
    dw = layers.embedding_backward(ids, dy, 12)
    assert dw[6].isnan().all() and dw[9, 7] == float("inf")
    assert (dw[5] == 2).all() and (dw[9, :7] == 1).all() and dw[[0, 1, 2, 3, 4, 7, 8, 10, 11]].abs().sum() == 0


@pytest.mark.parametrize("tokens", [100, 1000, 20000])
def test_embedding_padding_may_hold_anything(tokens):
    """NaN in the rows of padding ids, first, last and in between, reaches nothing."""
    g, vocab, dim = gen(tokens), 500, 40
    ids = integers(g, tokens, 0, vocab)
    pad = torch.rand(tokens, generator=g, device=DEV) < 0.4
    pad[0] = pad[-1] = True
    ids[pad] = torch.where(integers(g, int(pad.sum()), 0, 2) > 0, -1, 2 ** 40)
    dy = normal(g, tokens, dim)
    clean = dy.clone()
    dy[pad] = float("nan")
    clean[pad] = 0
    got = layers.embedding_backward(ids, dy, vocab)
    assert torch.equal(got, layers.embedding_backward(ids, clean, vocab))
    exact, tol, _ = embedding_exact(ids, clean, vocab, 1.0)
    close(got, exact, tol + half_step(exact, dy.dtype))


# ---------------------------------------------------------------- layer norm

LN_SIZES = [  # rows, dim
    (1, 1), (1, 2), (3, 7), (64, 512), (5, 1001), (33, 1024), (9, 4096), (2, 8193), (300, 40),
    (1030, 264), (4, 16384), (3, 40001), (2000, 8),
    # several rows a pass, and each width of a group in the gradient
    (4740, 256), (9500, 72), (2370, 1024), (1200, 2048), (1190, 4096), (300, 4100), (40, 12288), (600, 600),
    (5, 65544)]
KINDS = [(torch.float16, torch.float16), (torch.float16, torch.float32), (torch.float32, torch.float32)]


def chain(n):
    """Longest chain of additions over n terms of a row: 32 lanes or more, then a tree."""
    return min(n, n / 32 + 16)


def layernorm_exact(x, gamma, beta, eps):
    d = x.shape[1]
    xd = x.double()
    mean = xd.mean(1, keepdim=True)
    c = xd - mean
    var = c.square().mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    h = chain(d) + 2
    e_mean = h * U * xd.abs().mean(1, keepdim=True)
    # each centred value is off by e_mean and one rounding of the difference
    e_c = e_mean + U * c.abs()
    e_var = (2 * c.abs() * e_c + e_c.square()).mean(1, keepdim=True) + (h + 2) * U * var
    e_rstd = rstd * (0.5 * e_var / (var + eps) + 4 * U)
    g = gamma.double() if gamma is not None else torch.ones(d, device=DEV, dtype=torch.float64)
    b = beta.double() if beta is not None else torch.zeros(d, device=DEV, dtype=torch.float64)
    y = c * rstd * g + b
    e_y = g.abs() * (e_c * rstd + c.abs() * e_rstd) + 3 * U * (c * rstd * g).abs() + U * y.abs()
    return y, mean[:, 0], rstd[:, 0], e_y, e_mean[:, 0], e_rstd[:, 0]


@pytest.mark.parametrize("dtype,params", KINDS)
@pytest.mark.parametrize("rows,dim", LN_SIZES)
def test_layernorm_forward(rows, dim, dtype, params):
    g = gen(rows + dim)
    x = normal(g, rows, dim, mean=3.0, std=0.5, dtype=dtype)
    x[0] = 1.25                                                  # a row without variance
    gamma, beta = normal(g, dim, dtype=params), normal(g, dim, dtype=params)
    for shift, ga, be in ((0, gamma, beta), (1, gamma, None), (8, None, beta), (0, None, None)):
        xs, _ = strided(x, dim + shift, shift)
        out, clean = strided(torch.zeros_like(x), dim + 2 * shift, shift)
        eps = float(torch.tensor(1e-5))
        y, mean, rstd, e_y, e_m, e_r = layernorm_exact(x, ga, be, eps)
        got, gm, gr = layers.layernorm_forward(xs, ga, be, eps=1e-5, out=out)
        close(got, y, e_y + half_step(y, dtype))
        close(gm, mean, e_m + half_step(mean, torch.float32))
        close(gr, rstd, e_r + half_step(rstd, torch.float32))
        assert clean()


@pytest.mark.parametrize("dtype,params", KINDS)
@pytest.mark.parametrize("rows,dim", LN_SIZES)
def test_layernorm_backward(rows, dim, dtype, params):
    g = gen(3 * rows + dim)
    x = normal(g, rows, dim, mean=0.5, dtype=dtype)
    gamma = normal(g, dim, mean=1.0, std=0.2, dtype=params)
    dy = normal(g, rows, dim, std=0.3, dtype=dtype)
    xd = x.double()
    mean = xd.mean(1).float()
    rstd = (1.0 / torch.sqrt((xd - xd.mean(1, keepdim=True)).square().mean(1) + 1e-5)).float()
    for shift, ga in ((0, gamma), (1, gamma), (8, None)):
        kind = params if ga is not None else torch.float32
        gd = ga.double() if ga is not None else torch.ones(dim, device=DEV, dtype=torch.float64)
        rs = rstd.double()[:, None]
        xh = (xd - mean.double()[:, None]) * rs
        e_xh = 2 * U * xh.abs() + U * rs * xd.abs()
        d = dy.double() * gd
        a, b = d.mean(1, keepdim=True), (d * xh).mean(1, keepdim=True)
        h = chain(dim) + 4
        e_a = h * U * d.abs().mean(1, keepdim=True)
        e_b = h * U * (d * xh).abs().mean(1, keepdim=True) + (d.abs() * e_xh).mean(1, keepdim=True)
        dx = rs * (d - a - xh * b)
        e_dx = rs * (4 * U * (d.abs() + a.abs() + (xh * b).abs()) + e_a + xh.abs() * e_b + e_xh * b.abs())
        dg, db = (dy.double() * xh).sum(0), dy.double().sum(0)
        # all rows in one chain would be the longest order; a block's share and a tree is shorter
        e_dg = (rows + 3) * U * (dy.double() * xh).abs().sum(0) + (dy.double().abs() * e_xh).sum(0)
        e_db = (rows + 1) * U * dy.double().abs().sum(0)
        xs, _ = strided(x, dim + shift, shift)
        ys, _ = strided(dy, dim + 2 * shift, shift)
        out, clean = strided(torch.zeros_like(x), dim + shift, shift)
        gx, gg, gb = layers.layernorm_backward(ys, xs, ga, mean, rstd, grad_x=out)
        close(gx, dx, e_dx + half_step(dx, dtype))
        close(gg, dg, e_dg + half_step(dg, kind))
        close(gb, db, e_db + half_step(db, kind))
        assert clean()
        same = layers.layernorm_backward(ys, xs, ga, mean, rstd)
        assert all(torch.equal(p, q) for p, q in zip(same, (gx, gg, gb)))
        bg, bb = normal(g, dim, dtype=kind), normal(g, dim, dtype=kind)
        _, ag, ab = layers.layernorm_backward(ys, xs, ga, mean, rstd, grad_gamma=bg.clone(),
                                              grad_beta=bb.clone(), accumulate=True)
        close(ag, dg + bg.double(), e_dg + U * (dg.abs() + bg.double().abs()) + half_step(dg + bg.double(), kind))
        close(ab, db + bb.double(), e_db + U * (db.abs() + bb.double().abs()) + half_step(db + bb.double(), kind))


def test_layernorm_outputs_that_are_not_wanted():
    """Each output alone, through the C entry, equals the one of the full call."""
    g = gen(6)
    rows, dim = 70, 264
    x, dy, gamma = normal(g, rows, dim), normal(g, rows, dim), normal(g, dim, dtype=torch.float32)
    y, mean, rstd = layers.layernorm_forward(x, gamma)
    vp = lambda t: C.c_void_p(t.data_ptr() if t is not None else None)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    alone = torch.empty_like(y)
    assert capi.lib().b200opt_layernorm_fwd(capi.HALF, capi.FLOAT, rows, dim, vp(x), dim, vp(gamma), None,
                                            1e-5, vp(alone), dim, None, None, stream) == capi.OK
    assert torch.equal(alone, y)
    want = layers.layernorm_backward(dy, x, gamma, mean, rstd)
    ws = torch.empty(layers.layernorm_workspace(rows, dim), dtype=torch.uint8, device=DEV)
    for keep in ((0,), (1,), (2,), (0, 2), (1, 2), ()):
        out = [torch.zeros_like(t) if k in keep else None for k, t in enumerate(want)]
        assert capi.lib().b200opt_layernorm_bwd(
            capi.HALF, capi.FLOAT, rows, dim, vp(dy), dim, vp(x), dim, vp(gamma), vp(mean), vp(rstd),
            vp(out[0]), dim, vp(out[1]), vp(out[2]), 0, vp(ws), ws.numel(), stream) == capi.OK
        for k in keep:
            assert torch.equal(out[k], want[k]), (keep, k)


def test_layernorm_large_mean_and_non_finite_rows():
    g = gen(5)
    x = normal(g, 6, 777, mean=4096.0, std=1.0, dtype=torch.float32)
    y, mean, rstd, e_y, e_m, e_r = layernorm_exact(x, None, None, float(torch.tensor(1e-5)))
    x[2, 5], x[4, 0] = float("inf"), float("nan")
    got, gm, gr = layers.layernorm_forward(x)
    keep = [0, 1, 3, 5]
    close(got[keep], y[keep], (e_y + half_step(y, torch.float32))[keep])
    assert got[2].isnan().any() and got[4].isnan().all()


@pytest.mark.parametrize("dtype,params", KINDS)
def test_layernorm_rows_without_elements(dtype, params):
    """A mean over nothing is NaN, as the formula has it, and not what the memory held."""
    x, none = torch.zeros(700, 0, device=DEV, dtype=dtype), torch.zeros(0, device=DEV, dtype=params)
    mean, rstd = torch.full((700,), 3.0, device=DEV), torch.full((700,), 4.0, device=DEV)
    y, m, r = layers.layernorm_forward(x, none, none, mean=mean, rstd=rstd)
    assert y.shape == (700, 0) and m.isnan().all() and r.isnan().all()
    gx, gg, gb = layers.layernorm_backward(x, x, none, m, r)
    assert gx.shape == (700, 0) and gg.shape == gb.shape == (0,)


def test_layernorm_no_rows_gives_zero_parameter_gradients():
    x = torch.zeros(0, 96, device=DEV)
    s = torch.zeros(0, device=DEV)
    gamma = torch.ones(96, device=DEV)
    full = lambda: torch.full((96,), 3.0, device=DEV)
    _, dg, db = layers.layernorm_backward(x, x, gamma, s, s, grad_gamma=full(), grad_beta=full())
    assert (dg == 0).all() and (db == 0).all()
    _, dg, db = layers.layernorm_backward(x, x, gamma, s, s, grad_gamma=full(), grad_beta=full(), accumulate=True)
    assert (dg == 3).all() and (db == 3).all()


def test_layernorm_gradient_against_differences():
    """<dL/dx, w> against (L(x + e w) - L(x - e w)) / 2e with L = sum(c * y), fp32 forward pass.
    L is off by the rounding of y, at most sum|c| |y| 8 u; the difference by e^2/6 |L'''|, taken
    as e^2 times the sum of magnitudes."""
    g = gen(8)
    x = normal(g, 16, 200, dtype=torch.float32)
    gamma, c = normal(g, 200, dtype=torch.float32), normal(g, 16, 200, dtype=torch.float32)
    w = torch.sign(normal(g, 16, 200, dtype=torch.float32))
    _, mean, rstd = layers.layernorm_forward(x, gamma)
    dx, _, _ = layers.layernorm_backward(c, x, gamma, mean, rstd)
    e = 2.0 ** -7
    ys = [layers.layernorm_forward(x + s * e * w, gamma)[0].double() for s in (1, -1)]
    diff = ((ys[0] - ys[1]) * c.double()).sum() / (2 * e)
    size = (c.double() * ys[0]).abs().sum()
    assert abs(float((dx.double() * w.double()).sum() - diff)) <= float(size * (8 * U / e + e * e))


# ----------------------------------------------------------- vocabulary loss

VL_SIZES = [  # tokens, vocab, dim
    (1, 1, 8), (1, 1000, 64), (3, 7, 64), (64, 1000, 256), (127, 255, 72), (128, 256, 128),
    (129, 257, 136), (300, 5003, 264), (1000, 333, 1032), (2, 20011, 2048), (513, 1025, 520)]


def head_exact(x, w, y, factor, mean=True):
    """Loss, gradients and what each may be off by."""
    xd, wd = x.double(), w.double()
    vocab, dim = w.shape
    ok = (y >= 0) & (y < vocab)
    at = torch.where(ok, y, 0).long()
    z = xd @ wd.t()
    # products of fp16 are exact in fp32; a tensor core may cut instead of round: 2u an addition
    e_z = 2 * dim * U * (xd.abs() @ wd.abs().t())
    lse = torch.logsumexp(z, 1)
    e_lse = e_z.amax(1) + (chain(vocab) + 16) * U + 2 * U * lse.abs() + 4 * U * z.abs().amax(1)
    zt = z.gather(1, at[:, None])[:, 0]
    loss = torch.where(ok, lse - zt, 0.0)
    e_loss = torch.where(ok, e_lse + e_z.amax(1) + U * loss.abs(), 0.0)
    n = ok.double().sum()
    stats = torch.stack([loss.sum(), n])
    e_stats = torch.stack([e_loss.sum() + chain(len(y)) * U * loss.sum() + len(y) * U * loss.mean(), 0 * n])
    f = factor / n.clamp(min=1.0) if mean else torch.tensor(factor, device=DEV, dtype=torch.float64)
    p = torch.exp(z - lse[:, None]) * ok[:, None]
    one = torch.zeros_like(p).scatter_(1, at[:, None], ok.double()[:, None])
    dz = p - one
    e_exp = (e_z + e_lse[:, None] + 4 * U * (1 + (z - lse[:, None]).abs()))
    # fp16 of 2^15 dz: half a step, 2^-25 / 2^15 below the normal range
    e_dz = (p * e_exp + (2.0 ** -11 + U) * dz.abs() + 2.0 ** -40) * ok[:, None]
    dx, dw = f * dz @ wd, f * dz.t() @ xd
    tokens = len(y)
    e_dx = f * (e_dz @ wd.abs() + 2 * vocab * U * (dz.abs() @ wd.abs())) + 4 * U * dx.abs()
    e_dw = f * (e_dz.t() @ xd.abs() + 2 * tokens * U * (dz.abs().t() @ xd.abs())) + 4 * U * dw.abs()
    return dict(loss=loss, lse=lse, stats=stats, dx=dx, dw=dw, e_loss=e_loss, e_lse=e_lse,
                e_stats=e_stats, e_dx=e_dx, e_dw=e_dw, ok=ok)


def head_inputs(tokens, vocab, dim, seed=0, ignored=0.25):
    g = gen(tokens + vocab + dim + seed)
    x = normal(g, tokens, dim)
    w = normal(g, vocab, dim, std=dim ** -0.5 * 1.5)
    y = integers(g, tokens, 0, vocab)
    if ignored:
        y[torch.rand(tokens, generator=g, device=DEV) < ignored] = -100
        y[tokens // 3] = vocab
    return x, w, y


def check_head(x, w, y, got_f, got_b, factor, mean=True, base=None):
    r = head_exact(x, w, y, factor, mean)
    loss, lse, stats = got_f
    close(lse, r["lse"], r["e_lse"] + half_step(r["lse"], torch.float32))
    close(loss, r["loss"], r["e_loss"] + half_step(r["loss"], torch.float32))
    close(stats, r["stats"], r["e_stats"] + half_step(r["stats"], torch.float32))
    assert (loss[~r["ok"]] == 0).all()
    if got_b is None:
        return
    dx, dw = got_b
    close(dx, r["dx"], r["e_dx"] + half_step(r["dx"], torch.float16))
    if base is None:
        close(dw, r["dw"], r["e_dw"] + half_step(r["dw"], torch.float16))
    else:
        total = r["dw"] + base.double()
        close(dw, total, r["e_dw"] + U * total.abs() + half_step(total, torch.float16))
    assert (dx[~r["ok"]] == 0).all()


@pytest.mark.parametrize("tokens,vocab,dim", VL_SIZES)
def test_vocab_loss(tokens, vocab, dim):
    x, w, y = head_inputs(tokens, vocab, dim)
    scale = torch.full((1,), 64.0, device=DEV)
    f = layers.vocab_loss_forward(x, w, y)
    b = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=0.5, loss_scale=scale)
    check_head(x, w, y, f, b, 32.0)
    f2 = layers.vocab_loss_forward(x, w, y)
    b2 = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=0.5, loss_scale=scale)
    assert all(torch.equal(p, q) for p, q in zip(f + b, f2 + b2))


@pytest.mark.parametrize("tokens,vocab,dim", [(65, 300, 72), (260, 130, 200), (5, 1001, 64), (4100, 300, 72)])
def test_vocab_loss_strides_sum_accumulate_int32(tokens, vocab, dim):
    x, w, y = head_inputs(tokens, vocab, dim, seed=3)
    xs, _ = strided(x, dim + 8, 8)
    ws, _ = strided(w, dim + 24, 16)
    base = normal(gen(1), vocab, dim)
    dw, clean_w = strided(base, dim + 8, 8)
    dx, clean_x = strided(torch.full_like(x, float("nan")), dim + 16, 8)
    f = layers.vocab_loss_forward(xs, ws, y.int())
    b = layers.vocab_loss_backward(xs, ws, y.int(), f[1], grad_scale=0.25, grad_hidden=dx,
                                   grad_weight=dw, accumulate=True)
    check_head(x, w, y, f, b, 0.25, mean=False, base=base)
    assert clean_x() and clean_w()


@pytest.mark.parametrize("tokens,vocab,dim,accumulate", [
    (300, 9400, 520, False), (300, 9400, 520, True), (40, 9300, 1024, False), (700, 9400, 1000, True)])
def test_vocab_loss_wide_tiles(tokens, vocab, dim, accumulate):
    """Enough of the table's gradient for tiles of 512 columns, the last of them ragged or whole,
    with fewer and with more stages of tokens than the ring holds."""
    x, w, y = head_inputs(tokens, vocab, dim, seed=9)
    base = normal(gen(2), vocab, dim) if accumulate else None
    f = layers.vocab_loss_forward(x, w, y)
    b = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=512.0, accumulate=accumulate,
                                   grad_weight=base.clone() if accumulate else None)
    check_head(x, w, y, f, b, 512.0, base=base)


@pytest.mark.parametrize("tokens,vocab,dim,ignored,accumulate", [
    (1600, 9400, 520, 0.2, False), (1600, 9400, 520, 0.2, True), (1600, 9300, 1024, 0.98, False),
    (1537, 9400, 1000, 0.9, True), (1700, 9400, 520, 0.999, False), (4100, 9400, 512, 0.5, True)])
def test_vocab_loss_wide_tiles_of_many_tokens(tokens, vocab, dim, ignored, accumulate):
    """Tokens enough for tiles of 512 columns; those that are left of them fill many stages of the
    ring, a few or one."""
    x, w, y = head_inputs(tokens, vocab, dim, seed=10, ignored=ignored)
    y[7] = 5
    base = normal(gen(2), vocab, dim) if accumulate else None
    f = layers.vocab_loss_forward(x, w, y)
    b = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=512.0, accumulate=accumulate,
                                   grad_weight=base.clone() if accumulate else None)
    check_head(x, w, y, f, b, 512.0, base=base)


@pytest.mark.parametrize("tokens,vocab", [(8200, 20000), (9600, 14000)])
def test_vocab_loss_several_pieces_of_the_vocabulary(tokens, vocab):
    """With the sums of grad_hidden in parts, and whole."""
    x, w, y = head_inputs(tokens, vocab, 64)
    f = layers.vocab_loss_forward(x, w, y)
    b = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=4096.0)
    check_head(x, w, y, f, b, 4096.0)


@pytest.mark.parametrize("tokens,vocab,dim,ignored", [
    (1000, 6000, 264, 0.5), (1000, 6000, 264, 0.97), (700, 9000, 64, 0.999), (2000, 300, 520, 0.9),
    (4500, 40000, 64, 0.6)])
def test_vocab_loss_mostly_ignored(tokens, vocab, dim, ignored):
    """Few tokens left of many: the gradient's products are cut for those that are left."""
    x, w, y = head_inputs(tokens, vocab, dim, seed=5, ignored=ignored)
    f = layers.vocab_loss_forward(x, w, y)
    b = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=256.0)
    check_head(x, w, y, f, b, 256.0)


@pytest.mark.parametrize("vocab,masked", [
    (1000, [(0, 32)]), (1000, [(64, 96), (200, 300)]), (1000, [(0, 256)]), (1000, [(0, 1), (2, 1000)]),
    (1000, [(0, 999)]), (1001, [(960, 1001)]), (1030, [(256, 1024)]), (40000, [(5, 39000)])])
def test_vocab_loss_masked_vocabulary(vocab, masked):
    """Whole stretches of logits of -inf, from a column of the table that holds -inf in masked rows
    and 0 in the others: they count for nothing, in the losses and in both gradients."""
    tokens, dim = 70, 72
    x, w, y = head_inputs(tokens, vocab, dim, seed=6)
    keep = torch.ones(vocab, dtype=torch.bool, device=DEV)
    for a, b in masked:
        keep[a:b] = False
    left = keep.nonzero()[:, 0]
    x[:, -1], w[:, -1] = 1.0, 0.0
    ok = (y >= 0) & (y < vocab)
    y = torch.where(ok, left[y.clamp(0, vocab - 1) % len(left)], y)      # targets that are not masked
    small = torch.where(ok, torch.searchsorted(left, y), -1)
    w[~keep, -1] = -float("inf")
    f = layers.vocab_loss_forward(x, w, y)
    dx, dw = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=32.0)
    assert (dw[~keep] == 0).all()
    assert dx[ok, -1].isnan().all() and (dx[~ok, -1] == 0).all()        # 0 * -inf, as the formula has it
    dx[:, -1] = layers.vocab_loss_backward(x, w[keep], small, f[1], stats=f[2], grad_scale=32.0)[0][:, -1]
    check_head(x, w[keep], small, f, (dx, dw[keep]), 32.0)


def test_vocab_loss_infinite_logits():
    """A token whose logits are all -inf, then one of them +inf, beside ordinary tokens."""
    x, w, y = head_inputs(40, 700, 64, ignored=0)
    x[:, 0], w[:, 0], x[7] = 0.0, -1.0, 0.0
    x[7, 0] = float("inf")
    y[y == 300] = 299
    others = [t for t in range(40) if t != 7]
    for at_300, lse, loss in ((-1.0, -float("inf"), None), (1.0, float("inf"), float("inf"))):
        w[300, 0] = at_300
        got = layers.vocab_loss_forward(x, w, y)
        assert got[1][7] == lse and (got[0][7].isnan() if loss is None else got[0][7] == loss)
        check_head(x[others], w, y[others], (got[0][others], got[1][others],
                                             layers.vocab_loss_forward(x[others], w, y[others])[2]), None, 1.0)


@pytest.mark.parametrize("std", [0.0, 30.0])
def test_vocab_loss_flat_and_peaked_distributions(std):
    g = gen(17)
    x, w = normal(g, 70, 64), normal(g, 900, 64, std=std)
    y = integers(g, 70, 0, 900)
    f = layers.vocab_loss_forward(x, w, y)
    b = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=8.0)
    check_head(x, w, y, f, b, 8.0)


def test_vocab_loss_next_to_certainty():
    """Targets with probabilities up to 1 - 1e-5, and a vocabulary of one: p - 1 keeps what the
    rounding of lse leaves of it.  Values on a grid make the logits exact; then p is off by the
    rounding of lse (a step of it or two) and of one exponential."""
    tokens, vocab, dim = 64, 40, 8
    x = torch.zeros(tokens, dim, dtype=torch.float16, device=DEV)
    x[:, 0] = torch.linspace(0, 1, tokens, device=DEV).mul(64).round().div(64).half()
    w = torch.zeros(vocab, dim, dtype=torch.float16, device=DEV)
    w[3, 0] = 16.0
    y = torch.full((tokens,), 3, device=DEV)
    _, lse, _ = layers.vocab_loss_forward(x, w, y)
    dx, dw = layers.vocab_loss_backward(x, w, y, lse, grad_scale=2.0 ** 14)
    z = x.double() @ w.double().t()
    exact = torch.logsumexp(z, 1)
    close(lse, exact, exact.abs() * 2 * U + 8 * U)
    dz = torch.exp(z[:, 3] - exact) - 1
    want = 2.0 ** 14 * 16.0 * dz
    e_p = 2 * U * exact.abs() + 16 * U
    tol = 2.0 ** 14 * 16.0 * (e_p + dz.abs() * 2.0 ** -11) + half_step(want, torch.float16)
    fits = want.abs() + tol < 65504          # beyond fp16's range the result is infinite
    close(dx[fits, 0].double(), want[fits], tol[fits])
    assert (dx[want.abs() - tol > 65520, 0] == -float("inf")).all()
    one = layers.vocab_loss_forward(x, w[3:4], y * 0)
    assert (one[0] == 0).all()
    dx, dw = layers.vocab_loss_backward(x, w[3:4], y * 0, one[1])
    assert (dx == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("vocab,top,gap", [(2, 24.0, 13.75), (2, 1000.0, 14.0), (40, 1000.0, 14.0),
                                           (2, -500.0, 12.0), (300, 30000.0, 16.0), (1, 24.0, 0.0)])
def test_vocab_loss_small_losses_under_large_logits(vocab, top, gap):
    """Logits that are exact: `top` for the target, `top - gap` for the others.  The loss is
    log(1 + (vocab - 1) exp(-gap)): vocab - 1 additions to a sum near 1, a half step each, and a few
    steps of exp and log; nothing of the size of the logits."""
    x = torch.zeros(40, 8, dtype=torch.float16, device=DEV)
    x[:, 0] = 1.0
    w = torch.zeros(vocab, 8, dtype=torch.float16, device=DEV)
    w[:, 0] = top - gap
    w[vocab // 2, 0] = top
    assert float(w[0, 0]) == (top - gap if vocab > 1 else top) and float(w[vocab // 2, 0]) == top
    y = torch.full((40,), vocab // 2, device=DEV)
    loss, lse, stats = layers.vocab_loss_forward(x, w, y)
    exact = torch.log1p((vocab - 1) * torch.exp(torch.full((40,), -gap, device=DEV, dtype=torch.float64)))
    tol = exact * 32 * U + (vocab - 1) * U
    close(loss, exact, tol)
    close(stats[0], exact.sum(), tol.sum() + 40 * U * exact.sum())
    close(lse, exact + top, tol + abs(top) * U)


def test_vocab_loss_all_ignored():
    x, w, y = head_inputs(40, 100, 64)
    y[:] = -1
    f = layers.vocab_loss_forward(x, w, y)
    b = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=1024.0)
    assert (f[0] == 0).all() and f[2].tolist() == [0.0, 0.0]
    assert (b[0] == 0).all() and (b[1] == 0).all()


def test_vocab_loss_no_tokens():
    x, w, y = torch.zeros(0, 64, device=DEV).half(), normal(gen(2), 100, 64), torch.zeros(0, device=DEV).long()
    f = layers.vocab_loss_forward(x, w, y)
    assert f[2].tolist() == [0.0, 0.0]
    dx, dw = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2])
    assert dx.shape == (0, 64) and (dw == 0).all()
    base = normal(gen(3), 100, 64)
    _, dw = layers.vocab_loss_backward(x, w, y, f[1], grad_weight=base.clone(), accumulate=True)
    assert torch.equal(dw, base)


def test_vocab_loss_non_finite_tokens_stay_in_their_rows():
    """A NaN token spoils its own loss and the table's gradient, which the optimizer's flags then
    report, but no other token's loss or gradient; an ignored NaN token spoils nothing."""
    x, w, y = head_inputs(300, 500, 64, ignored=0)
    y3, x3 = y.clone(), x.clone()
    y3[[7, 200, 299]] = -1
    x3[7], x3[200, 3], x3[299] = float("nan"), float("inf"), float("-inf")
    good3 = layers.vocab_loss_forward(x, w, y3)
    f3 = layers.vocab_loss_forward(x3, w, y3)
    assert torch.equal(f3[0], good3[0]) and torch.equal(f3[2], good3[2])
    want3 = layers.vocab_loss_backward(x, w, y3, good3[1], stats=good3[2])
    got3 = layers.vocab_loss_backward(x3, w, y3, f3[1], stats=f3[2])
    assert all(torch.equal(p, q) for p, q in zip(got3, want3))
    clean = layers.vocab_loss_forward(x, w, y)
    x2 = x.clone()
    x2[7], x2[200, 3] = float("nan"), float("inf")
    f = layers.vocab_loss_forward(x2, w, y)
    keep = torch.ones(300, dtype=torch.bool, device=DEV)
    keep[[7, 200]] = False
    assert torch.equal(f[0][keep], clean[0][keep]) and not f[0][7].isfinite() and not f[0][200].isfinite()
    dx, dw = layers.vocab_loss_backward(x2, w, y, f[1], grad_scale=1.0)
    good, _ = layers.vocab_loss_backward(x, w, y, clean[1], grad_scale=1.0)
    assert torch.equal(dx[keep], good[keep]) and not dx[7].isfinite().any()
    assert not dw.isfinite().all()


def test_vocab_loss_partial_gradients():
    """Either gradient alone, through the C entry, equals the one of the full call."""
    x, w, y = head_inputs(100, 700, 72)
    f = layers.vocab_loss_forward(x, w, y)
    dx, dw = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2])
    ws = torch.empty(layers.vocab_loss_workspace(100, 700, 72)[1], dtype=torch.uint8, device=DEV)
    vp = lambda t: C.c_void_p(t.data_ptr() if t is not None else None)
    for keep in (0, 1):
        out = [torch.zeros_like(dx), None] if keep == 0 else [None, torch.zeros_like(dw)]
        rc = capi.lib().b200opt_vocab_loss_bwd(
            100, 700, 72, vp(x), 72, vp(w), 72, vp(y), 8, vp(f[1]), vp(f[2]), 1.0, None, vp(out[0]),
            72, vp(out[1]), 72, 0, vp(ws), ws.numel(),
            C.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == capi.OK
        assert torch.equal(out[keep], (dx, dw)[keep])


def test_vocab_loss_gradient_against_differences():
    """<dL/dx, s> against (L(x + e s) - L(x - e s)) / 2e, s = +-1, e = 2^-5, x on a grid that
    keeps x +- e exact in fp16.  The losses are off by their bound; the difference by e^2/6 of a
    third derivative, at most (2 max|w s|_1)^3 per token, which the grid of weights keeps small."""
    g = gen(31)
    tokens, vocab, dim = 24, 500, 64
    x = torch.round(normal(g, tokens, dim, dtype=torch.float32) * 32).div(32).half()
    w = normal(g, vocab, dim, std=0.02)
    y = integers(g, tokens, 0, vocab)
    s = torch.sign(normal(g, tokens, dim, dtype=torch.float32)).half()
    e = 2.0 ** -5
    loss = [layers.vocab_loss_forward(x + k * e * s, w, y)[0].double() for k in (1, -1)]
    bound = sum(float(head_exact(x + k * e * s, w, y, 1.0)["e_loss"].sum()) for k in (1, -1))
    _, lse, _ = layers.vocab_loss_forward(x, w, y)
    dx, _ = layers.vocab_loss_backward(x, w, y, lse, grad_scale=1024.0)
    r = head_exact(x, w, y, 1024.0, mean=False)
    span = (s.double() @ w.double().t()).abs().amax(1) * 2
    tol = bound / (2 * e) + float((span ** 3).sum()) * e * e / 6
    tol += float((r["e_dx"] + half_step(r["dx"], torch.float16)).sum()) / 1024
    diff = float((loss[0] - loss[1]).sum() / (2 * e))
    assert abs(float((dx.double() * s.double()).sum()) / 1024 - diff) <= tol * SLACK


# ------------------------------------------------------ offsets over 32 bits

def test_far_offsets():
    """Tables and activations of more than 2^31 elements: what lies at their ends."""
    rows, dim = 1_060_000, 2048
    g = gen(12)
    big = torch.empty(rows, dim, dtype=torch.float16, device=DEV).normal_(generator=g)
    ids = torch.tensor([rows - 1, 0, rows - 7, rows, rows - 1, 1_048_576], device=DEV)
    out = layers.embedding_forward(ids, big)
    assert torch.equal(out[[0, 1, 2, 5]], big[ids[[0, 1, 2, 5]]]) and (out[3] == 0).all()
    y, mean, rstd = layers.layernorm_forward(big)
    tail = slice(rows - 50, rows)
    ty, tm, tr = layers.layernorm_forward(big[tail].clone())
    assert torch.equal(y[tail], ty) and torch.equal(mean[tail], tm) and torch.equal(rstd[tail], tr)
    dx, _, db = layers.layernorm_backward(y, big, None, mean, rstd)
    tdx, _, _ = layers.layernorm_backward(ty, big[tail].clone(), None, tm, tr)
    assert torch.equal(dx[tail], tdx)
    del dx
    y.fill_(float("nan"))
    dw = layers.embedding_backward(ids, out, rows, grad_weight=y)
    assert torch.equal(dw[rows - 7], out[2]) and torch.equal(dw[1_048_576], out[5])
    two = (out[0].float() * 2).half()
    assert torch.equal(dw[rows - 1], two)
    dw[ids[[0, 1, 2, 5]]] = 0
    assert int(dw.view(torch.int16).count_nonzero()) == 0


def test_embedding_gradient_of_the_largest_table():
    """As many rows as are allowed, and ids outside the table behind the others."""
    vocab, tokens = capi.LM_MAX, 300
    ids = torch.tensor([vocab - 1, 0, vocab - 1, vocab // 2], device=DEV).repeat(tokens // 4)
    ids[100:150] = -1
    ids[200] = vocab
    dy = normal(gen(14), tokens, 1)
    dw = layers.embedding_backward(ids, dy, vocab)
    for row in (vocab - 1, 0, vocab // 2):
        mine = dy[ids == row].double()
        exact = mine.sum()
        tol = mine.abs().sum() * U * len(mine) + half_step(exact, dy.dtype)
        assert abs(float(dw[row, 0]) - float(exact)) <= float(tol) * SLACK
        dw[row] = 0
    assert all(int(part.count_nonzero()) == 0 for part in dw.view(-1).view(torch.int16).split(1 << 28))


def test_vocab_loss_far_offsets():
    tokens, vocab, dim = 70, 530_000, 4096
    g = gen(13)
    w = torch.empty(vocab, dim, dtype=torch.float16, device=DEV).normal_(std=0.02, generator=g)
    x = normal(g, tokens, dim)
    y = integers(g, tokens, vocab - 300, vocab)
    loss, lse, stats = layers.vocab_loss_forward(x, w, y)
    top = torch.full((tokens,), -float("inf"), device=DEV, dtype=torch.float64)
    for at in range(0, vocab, 53_000):
        top = torch.logaddexp(top, torch.logsumexp(x.double() @ w[at:at + 53_000].double().t(), 1))
    e_z = 2 * dim * U * float((x.double().abs().sum(1).max() * 0.12))
    close(lse, top, e_z + (chain(vocab) + 64) * U + 0 * top)
    dx, dw = layers.vocab_loss_backward(x, w, y, lse, stats=stats, grad_scale=4096.0)
    tail = slice(vocab - 400, vocab)
    p = torch.exp(x.double() @ w[tail].double().t() - top[:, None])
    p[torch.arange(tokens, device=DEV), y - (vocab - 400)] -= 1
    f = 4096.0 / tokens
    want = f * p.t() @ x.double()
    size = f * p.abs().t() @ x.double().abs()
    close(dw[tail], want, size * (2.0 ** -11 + 2 * e_z + 2 * tokens * U) + half_step(want, torch.float16))


def grid(g, *shape, steps, unit):
    """Whole multiples of `unit`, up to `steps` of them either way: products and sums of such values
    are exact in fp32 as long as they stay under 2^24 units, in any order."""
    return torch.randint(-steps, steps + 1, shape, generator=g, device=DEV, dtype=torch.int8).half().mul_(unit)


def exact_logits_dz(z, lse, e_lse, y):
    """p - onehot from exact logits, and what the fp16 value that the products read may be off by."""
    p = torch.exp(z - lse[:, None])
    dz = p.clone()
    dz[torch.arange(len(y), device=DEV), y] -= 1
    return dz, p * (e_lse[:, None] + 4 * U * (1 + (z - lse[:, None]).abs())) + (2.0 ** -11 + U) * dz.abs() + 2.0 ** -40


@pytest.mark.parametrize("tokens,vocab,dim", [(300, 5003, 512), (129, 20011, 1032), (1000, 999, 64)])
def test_vocab_loss_with_exact_logits(tokens, vocab, dim):
    """Logits without any error leave nothing but the exponentials, the sums and the logarithm to the
    losses: bounds hundreds of times closer than those of rounded products."""
    g = gen(tokens)
    x, w = grid(g, tokens, dim, steps=4, unit=0.25), grid(g, vocab, dim, steps=8, unit=2.0 ** -6)
    y = integers(g, tokens, 0, vocab)
    assert dim * 4 * 8 < 2 ** 24
    loss, lse, stats = layers.vocab_loss_forward(x, w, y)
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1)
    e_lse = (chain(vocab) + 16) * U + 2 * U * want.abs() + 4 * U * (z.amax(1) - z.amin(1))
    close(lse, want, e_lse + half_step(want, torch.float32))
    exact = want - z.gather(1, y[:, None])[:, 0]
    e_loss = e_lse + 2 * U * exact
    close(loss, exact, e_loss)
    close(stats[0], exact.sum(), e_loss.sum() + chain(tokens) * U * exact.sum())
    dx, dw = layers.vocab_loss_backward(x, w, y, lse, stats=stats, grad_scale=1024.0)
    f = 1024.0 / tokens
    dz, e_dz = exact_logits_dz(z, want, e_lse + half_step(want, torch.float32), y)
    for got, ref, size, e, n in ((dx, dz @ w.double(), dz.abs() @ w.double().abs(), e_dz @ w.double().abs(), vocab),
                                 (dw, dz.t() @ x.double(), dz.t().abs() @ x.double().abs(),
                                  e_dz.t() @ x.double().abs(), tokens)):
        ref = f * ref
        close(got, ref, f * (e + 2 * n * U * size) + 4 * U * ref.abs() + half_step(ref, torch.float16))


def test_vocab_loss_far_rows_decide():
    """The rows of the table beyond 2^31 elements hold the targets and nearly all of the probability:
    losses and both gradients are theirs.  Exact logits, as above.  Left out, they would move lse by
    more than 10; what the other rows add to a gradient is rounded relative to their own small sums."""
    tokens, vocab, dim = 70, 530_000, 4096
    far = 2 ** 31 // dim
    g = gen(15)
    w = torch.empty(vocab, dim, dtype=torch.float16, device=DEV)
    for at in range(0, vocab, 53_000):
        w[at:at + 53_000] = grid(g, 53_000, dim, steps=2, unit=2.0 ** -6)
    w[far:] *= 16
    x = grid(g, tokens, dim, steps=4, unit=0.25)
    y = integers(g, tokens, far + 500, vocab)
    assert dim * 4 * 2 * 16 < 2 ** 24
    loss, lse, stats = layers.vocab_loss_forward(x, w, y)
    dx, dw = layers.vocab_loss_backward(x, w, y, lse, stats=stats, grad_scale=4096.0)
    xd, parts = x.double(), [(a, min(a + 53_000, far)) for a in range(0, far, 53_000)] + [(far, vocab)]
    logits = lambda a, b: xd @ w[a:b].double().t()
    near = torch.full((tokens,), -float("inf"), device=DEV, dtype=torch.float64)
    low = -near
    for a, b in parts[:-1]:
        z = logits(a, b)
        near, low = torch.logaddexp(near, torch.logsumexp(z, 1)), torch.minimum(low, z.amin(1))
    z = logits(far, vocab)
    want = torch.logaddexp(near, torch.logsumexp(z, 1))
    assert (want - near > 10).all()
    e_lse = (chain(vocab) + 16) * U + 2 * U * want + 4 * U * (z.amax(1) - torch.minimum(low, z.amin(1)))
    close(lse, want, e_lse + half_step(want, torch.float32))
    exact = want - z.gather(1, (y - far)[:, None])[:, 0]
    close(loss, exact, e_lse + 2 * U * exact)
    f = 4096.0 / tokens
    e_lse += half_step(want, torch.float32)
    dz, e_dz = exact_logits_dz(z, want, e_lse, y - far)
    ref, size = f * dz.t() @ xd, f * dz.t().abs() @ xd.abs()
    close(dw[far:], ref, f * e_dz.t() @ xd.abs() + 2 * tokens * U * size + 4 * U * ref.abs() + half_step(ref, torch.float16))
    ref = dz @ w[far:].double()
    tol = e_dz @ w[far:].double().abs() + 2 * (vocab - far + 128) * U * (dz.abs() @ w[far:].double().abs())
    for a, b in parts[:-1]:
        z, wd = logits(a, b), w[a:b].double()
        p = torch.exp(z - want[:, None])
        ref += p @ wd
        tol += (p * (e_lse[:, None] + 4 * U * (1 + (z - want[:, None]).abs()) + 2.0 ** -11 + 2 * vocab * U) + 2.0 ** -40) @ wd.abs()
    ref, tol = f * ref, f * tol
    close(dx, ref, tol + 4 * U * ref.abs() + half_step(ref, torch.float16))


# -------------------------------------------- streams, graphs, several at once

def _calls():
    """A call of each kind: (inputs that change, a function that runs it, its outputs)."""
    g = gen(4)
    vocab, dim, tokens = 700, 72, 300
    ids = integers(g, tokens, 0, vocab)
    table, x = normal(g, vocab, dim, std=0.2), normal(g, tokens, dim)
    gamma = normal(g, dim, dtype=torch.float32)

    def run(out=None):
        e = layers.embedding_forward(ids, table)
        y, mean, rstd = layers.layernorm_forward(x, gamma)
        loss, lse, stats = layers.vocab_loss_forward(y, table, ids)
        dh, dw = layers.vocab_loss_backward(y, table, ids, lse, stats=stats, grad_scale=256.0)
        dx, dg, db = layers.layernorm_backward(dh, x, gamma, mean, rstd)
        layers.embedding_backward(ids, dx, vocab, grad_weight=dw, accumulate=True)
        return [e, y, mean, rstd, loss, lse, stats, dh, dx, dg, db, dw]
    return (ids, x), run


def test_captured_and_replayed():
    inputs, run = _calls()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                     # two graphs of the same calls, each with its own memory
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run()
        graphs.append((graph, out))
    for seed in (1, 2):
        g = gen(100 + seed)
        inputs[0].copy_(integers(g, len(inputs[0]), -3, 705))
        inputs[1].copy_(normal(g, *inputs[1].shape))
        want = run()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, _), s in zip(graphs, streams):    # at the same time
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))

@pytest.mark.parametrize("tokens,vocab,dim", [(1, 3, 8), (129, 700, 72), (513, 1009, 264),
                                              (1001, 2100, 520), (33001, 500, 24)])
def test_workspaces_may_hold_anything(tokens, vocab, dim):
    gen = torch.Generator(device=DEV).manual_seed(tokens)
    x = torch.randn(tokens, dim, generator=gen, device=DEV).half()
    dy = torch.randn(tokens, dim, generator=gen, device=DEV).half()
    w = (torch.randn(vocab, dim, generator=gen, device=DEV) * 0.1).half()
    ids = torch.randint(-1, vocab, (tokens,), generator=gen, device=DEV)
    gamma = torch.randn(dim, generator=gen, device=DEV).half()
    _, mean, rstd = layers.layernorm_forward(x, gamma)

    def run(byte):
        def ws(n):
            return torch.full((n,), byte, dtype=torch.uint8, device=DEV)
        fwd, bwd = layers.vocab_loss_workspace(tokens, vocab, dim)
        out = [layers.embedding_backward(ids, dy, vocab,
                                         workspace=ws(layers.embedding_workspace(tokens, vocab, dim)))]
        out += layers.layernorm_backward(dy, x, gamma, mean, rstd,
                                         workspace=ws(layers.layernorm_workspace(tokens, dim)))
        head = layers.vocab_loss_forward(x, w, ids, workspace=ws(fwd))
        out += head
        out += layers.vocab_loss_backward(x, w, ids, head[1], head[2], workspace=ws(bwd))
        return out

    for a, b in zip(run(0), run(255)):      # 255: NaN in either type, -1 as a whole number
        assert torch.equal(a, b) and a.isfinite().all()



def test_first_call_of_a_process_inside_a_capture():
    """Nothing has to be called before a capture is open: kernels load and their shared-memory limits
    are set under it."""
    code = """
import torch
from saga_b200 import layers
d = 'cuda:0'
torch.manual_seed(3)
x, w = torch.randn(300, 72, device=d).half(), torch.randn(700, 72, device=d).half()
y = torch.randint(0, 700, (300,), device=d)
def run():
    a, mean, rstd = layers.layernorm_forward(layers.embedding_forward(y, w))
    loss, lse, stats = layers.vocab_loss_forward(a, w, y)
    dh, dw = layers.vocab_loss_backward(a, w, y, lse, stats=stats)
    dx, dg, db = layers.layernorm_backward(dh, x, None, mean, rstd)
    layers.embedding_backward(y, dx, 700, grad_weight=dw, accumulate=True)
    return [loss, dh, dw, dx, dg, db, layers.embedding_backward(y[:20], dx[:20], 700)]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = run()
g.replay()
want = run()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(out, want))
print('same')
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "same" in res.stdout, res.stderr[-2000:]


def test_two_host_threads():
    """Calls from two threads, each on a stream of its own, at the same time."""
    inputs, run = _calls()
    want = run()
    torch.cuda.synchronize()
    got, errors = [], []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got.append(run())
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # reported by the test, not lost with the thread
            errors.append(e)
    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert len(got) == 20 and all(torch.equal(a, b) for out in got for a, b in zip(out, want))


def test_two_streams_at_once_and_a_raw_stream():
    inputs, run = _calls()
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append(run())
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    ids, x = inputs
    out = torch.empty(300, 72, dtype=torch.float16, device=DEV)
    raw = streams[0].cuda_stream
    layers.layernorm_forward(x, out=out, mean=torch.empty(300, device=DEV), rstd=torch.empty(300, device=DEV), stream=raw)
    torch.cuda.synchronize()
    assert torch.equal(out, layers.layernorm_forward(x)[0])
    with pytest.raises(ValueError):
        layers.layernorm_forward(x, stream=raw)


def test_tensor_refusals():
    x = torch.zeros(4, 16, device=DEV)
    ids = torch.zeros(4, dtype=torch.int64, device=DEV)
    for call in (lambda: layers.embedding_forward(ids.float(), x),
                 lambda: layers.embedding_forward(ids, x.double()),
                 lambda: layers.embedding_forward(ids.cpu(), x),
                 lambda: layers.embedding_forward(ids, x, out=torch.zeros(3, 16, device=DEV)),
                 lambda: layers.embedding_backward(ids[:3], x, 10),
                 lambda: layers.embedding_backward(ids, x, 10, accumulate=True),
                 lambda: layers.layernorm_forward(x, gamma=torch.zeros(15, device=DEV)),
                 lambda: layers.layernorm_forward(x, out=x.half()),
                 lambda: layers.layernorm_forward(x, beta=torch.zeros(16, device=DEV).half()),
                 lambda: layers.vocab_loss_forward(x, x, ids),
                 lambda: layers.vocab_loss_forward(x.half(), x.half(), ids[:2]),
                 lambda: layers.vocab_loss_forward(x.half()[:, :12], x.half()[:, :12], ids),
                 lambda: layers.vocab_loss_forward(x.half(), x.half()[:, :8], ids)):
        with pytest.raises((ValueError, TypeError, capi.B200OptError)):
            call()


def test_loss_scale_is_a_tensor_or_a_device_address():
    x, w, y = head_inputs(20, 100, 64)
    f = layers.vocab_loss_forward(x, w, y)
    scale = torch.full((1,), 1024.0, device=DEV)
    want = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], grad_scale=1024.0)
    for given in (scale, capi.DeviceAddress(scale.data_ptr())):
        got = layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], loss_scale=given)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for number in (1024, 1024.0, True):
        with pytest.raises(TypeError):
            layers.vocab_loss_backward(x, w, y, f[1], stats=f[2], loss_scale=number)


# -------------------------------------------------- together with the optimizer

def test_training_step_of_a_tied_model_through_the_optimizer():
    """Embedding -> layer norm -> vocabulary loss with one table for both ends, gradients written
    into the optimizer's flat buffers (fp16 and fp32 group), loss scale kept on the device: the
    gradients against torch's in 64 bits, then the fused step, for three steps; then a scale so
    large that the step must see an overflow and halve it."""
    vocab, dim, tokens = 1000, 64, 200
    half, flt = FlatLayout([vocab * dim]), FlatLayout([dim, dim])
    group = AdamGroup.create(0, 1, 0, half.total, flt.total)
    try:
        (wh, gh), (wf, gf) = group.buffers(capi.HALF), group.buffers(capi.FLOAT)
        pick = lambda buf, lay, k, *shape: buf[lay.slices()[k]].view(*shape)
        table, d_table = pick(wh, half, 0, vocab, dim), pick(gh, half, 0, vocab, dim)
        gamma, d_gamma = pick(wf, flt, 0, dim), pick(gf, flt, 0, dim)
        beta, d_beta = pick(wf, flt, 1, dim), pick(gf, flt, 1, dim)
        g = gen(77)
        table.copy_(normal(g, vocab, dim, std=0.1))
        gamma.fill_(1.0), beta.fill_(0.0)
        stream = torch.cuda.current_stream().cuda_stream
        group.init_master(stream)
        group.device_scale_enable(1024.0)
        scale_ptr = group.device_scale_ptr()
        scale = 1024.0
        for step in range(4):
            if step == 3:
                group.device_scale_enable(2.0 ** 40)
                scale = 2.0 ** 40
            ids, y = integers(g, tokens, 0, vocab), integers(g, tokens, 0, vocab)
            y[::5] = -100
            h = layers.embedding_forward(ids, table, scale=8.0)
            n, mean, rstd = layers.layernorm_forward(h, gamma, beta)
            loss, lse, stats = layers.vocab_loss_forward(n, table, y)
            dn, _ = layers.vocab_loss_backward(n, table, y, lse, stats=stats, loss_scale=scale_ptr,
                                               grad_weight=d_table)
            dh, _, _ = layers.layernorm_backward(dn, h, gamma, mean, rstd, grad_gamma=d_gamma,
                                                 grad_beta=d_beta)
            layers.embedding_backward(ids, dh, vocab, scale=8.0, grad_weight=d_table, accumulate=True)
            if step < 3:
                leaf = [t.double().requires_grad_() for t in (table, gamma, beta)]
                e = leaf[0][ids] * 8.0
                nn = torch.nn.functional.layer_norm(e, (dim,), leaf[1], leaf[2], 1e-5)
                want = torch.nn.functional.cross_entropy(nn @ leaf[0].t(), y, ignore_index=-100)
                want.backward()
                # activations and gradients pass five fp16 roundings on the way: 2^-11 each
                for got, ref in zip((d_table, d_gamma, d_beta), leaf):
                    ref = ref.grad * scale
                    rel = float((got.double() - ref).norm() / ref.norm())
                    assert rel <= 5 * 2.0 ** -11, rel
                assert abs(float(stats[0] / stats[1]) - want.item()) <= 5 * 2.0 ** -11 * want.item()
                before = table.clone()
            group.exec_device_scale(1e-2, 0.0, stream)
            new, log = group.device_scale_read(stream)
            if step < 3:
                assert log[-1][:3] == (0, 0, 0)
                scale = float(new)
                moved = (table != before).any(1)
                assert moved[ids].all()           # every row that was looked up has been updated
            else:
                assert log[-1][1] + log[-1][2] > 0 and float(new) == 2.0 ** 39
    finally:
        group.destroy()
