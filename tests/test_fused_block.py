"""Layer norm, linear and token log probabilities against their formulas in
64 bits, on the CPU path and (gpu-marked) on the kernels.

Tolerances are bounds, derived per element from the inputs: U = 2^-24 is half
a step of a 32-bit float, HALF[t] half a step of the stored type relative to
the value.  A sum of n terms added one after the other is off by at most
n U sum|terms|; the kernels' chains are shorter than the counts used here.
"""
import itertools
import math

import pytest
import torch

from cpd_amd.models import (FusedLayerNorm, FusedLinear, fused_layer_norm,
                            fused_linear)
from cpd_amd.utils import accuracy, token_logprobs

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF = {t: torch.finfo(t).eps / 2 for t in TYPES}
# half of the smallest step there is: what a value near zero may be off by
TINY = {t: torch.finfo(t).tiny * torch.finfo(t).eps for t in TYPES}
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
on_devices = pytest.mark.parametrize("device", DEVICES)
on_types = pytest.mark.parametrize(
    "dtype", TYPES, ids=lambda t: str(t).split(".")[-1])


def normal(gen, *shape, dtype, device, scale=1.0, shift=0.0):
    x = torch.randn(*shape, generator=gen, dtype=torch.float64)
    return (x * scale + shift).to(dtype).to(device)


def rng(*seed):
    return torch.Generator().manual_seed(hash(seed) & 0x7FFFFFFF)


def within(got, want, tol, what=""):
    """|got - want| <= tol everywhere; infinities and NaN in the same
    places."""
    got, want, tol = got.detach().cpu().double(), want.cpu(), tol.cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    odd = ~torch.isfinite(want)
    assert torch.equal(got[odd].nan_to_num(7, 8, 9),
                       want[odd].nan_to_num(7, 8, 9)), what
    off = (got - want).abs()[~odd]
    allowed = tol.expand_as(want)[~odd]
    bad = ~(off <= allowed)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {off.numel()} outside, worst "
        f"{(off / allowed).max():.3g} times the bound")


def stored(want, dtype):
    """The rounding of a result to its type."""
    return want.abs() * HALF[dtype] + TINY[dtype]


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------

def norm_oracle(x, w, b, eps, res, dy, ds):
    """(results, bounds) in 64 bits; x, res, dy, ds are [rows, cols]."""
    t = x.dtype
    s = x if res is None else (x.double() + res.double()).to(t)
    s64 = s.double()
    c = s.shape[-1]
    one, zero = torch.ones(c, dtype=torch.float64), torch.zeros(
        c, dtype=torch.float64)
    w64 = one if w is None else w.cpu().double()
    b64 = zero if b is None else b.cpu().double()
    mean = s64.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((s64 - mean) ** 2).mean(-1, keepdim=True) + eps)
    hat = (s64 - mean) * rstd
    y = hat * w64 + b64
    # a row's sums: at most 32 values a thread, 6 steps in a wave, 16 waves,
    # and the same again where a long row loops: under 100 additions
    big = s64.abs().amax(-1, keepdim=True) * rstd
    n = 100 + c / 1024
    err_hat = n * U * (hat.abs() + big)
    got, tol = {"y": y, "s": s64}, {"s": torch.zeros(())}
    tol["y"] = err_hat * w64.abs() + 4 * U * (
        (hat * w64).abs() + b64.abs()) + stored(y, t)
    if dy is not None:
        dy64 = dy.double()
        g = dy64 * w64
        mg, mgh = g.mean(-1, keepdim=True), (g * hat).mean(-1, keepdim=True)
        dx = rstd * (g - mg - hat * mgh)
        # every part of dx with hat off by err_hat, and its own sums
        wide = hat.abs() + big
        tol["dx"] = 4 * n * U * rstd * (
            g.abs() + g.abs().mean(-1, keepdim=True)
            + wide * (g.abs() * wide).mean(-1, keepdim=True))
        if ds is not None:
            dx = dx + ds.double()
            tol["dx"] = tol["dx"] + 2 * U * dx.abs()
        got["dx"], tol["dx"] = dx, tol["dx"] + stored(dx, t)
        wt = t if w is None else w.dtype
        # a column's sum: its rows in turn
        m = n + x.shape[0]
        got["dw"], got["db"] = (dy64 * hat).sum(0), dy64.sum(0)
        tol["dw"] = 2 * m * U * (dy64.abs() * wide).sum(0) + stored(
            got["dw"], wt)
        tol["db"] = m * U * dy64.abs().sum(0) + stored(got["db"], wt)
    return got, tol


def run_norm(device, dtype, rows, cols, residual, wtype=None, affine="wb",
             eps=1e-5, shift=0.25):
    g = rng(rows, cols, residual)
    t = lambda *s, **k: normal(g, *s, dtype=dtype, device=device, **k)  # noqa: E731
    x = t(rows, cols, shift=shift)
    res = t(rows, cols, scale=0.5) if residual else None
    wtype = wtype or dtype
    w = normal(g, cols, dtype=wtype, device=device, scale=0.2, shift=1.0) \
        if "w" in affine else None
    b = normal(g, cols, dtype=wtype, device=device, scale=0.2) \
        if "b" in affine else None
    dy, ds = t(rows, cols), (t(rows, cols) if residual else None)
    leaves = [v for v in (x, res, w, b) if v is not None]
    for v in leaves:
        v.requires_grad_(True)
    out = fused_layer_norm(x, w, b, eps, res)
    y, s = out if residual else (out, None)
    grads = dict(zip([n for n, v in zip(("x", "res", "w", "b"),
                                        (x, res, w, b)) if v is not None],
                     torch.autograd.grad(
                         [y] + ([s] if residual else []), leaves,
                         [dy] + ([ds] if residual else []))))
    cpu = lambda v: None if v is None else v.detach().cpu()  # noqa: E731
    want, tol = norm_oracle(cpu(x), cpu(w), cpu(b), eps, cpu(res), cpu(dy),
                            cpu(ds))
    assert y.dtype == dtype
    within(y, want["y"], tol["y"], "y")
    within(grads["x"], want["dx"], tol["dx"], "dx")
    if residual:
        within(s, want["s"], tol["s"], "s")
        within(grads["res"], want["dx"], tol["dx"], "dres")
    if w is not None:
        assert grads["w"].dtype == wtype
        within(grads["w"], want["dw"], tol["dw"], "dw")
    if b is not None:
        within(grads["b"], want["db"], tol["db"], "db")
    # without gradients the same numbers come
    with torch.no_grad():
        again = fused_layer_norm(x, w, b, eps, res)
    assert torch.equal(again[0] if residual else again, y)


# one element; less than a vector; a vector and one; each way of sharing a
# row, its last size and the first of the next; the looping rows
NORM_SHAPES = [(1, 1), (3, 5), (7, 8), (2, 17), (300, 64), (33, 257),
               (5, 511), (130, 512), (17, 513), (3, 2048), (9, 2049),
               (2, 8192), (3, 8193), (600, 1024), (1, 16384), (2, 33000)]


@on_devices
@on_types
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_norm(device, dtype, rows, cols, residual):
    run_norm(device, dtype, rows, cols, residual)


@on_devices
@pytest.mark.parametrize("affine", ["", "w", "b", "wb"])
@pytest.mark.parametrize("cols", [40, 1000])
def test_norm_learned_in_float(device, affine, cols):
    run_norm(device, torch.bfloat16, 19, cols, True, torch.float32, affine)


@on_devices
def test_norm_far_from_zero(device):
    # a mean a hundred times the spread: the variance is taken around it
    run_norm(device, torch.float32, 9, 1000, False, shift=100.0)


@on_devices
@on_types
def test_norm_constant_rows(device, dtype):
    # no spread: y is the bias, and eps keeps the gradient finite
    x = torch.full((3, 96), 2.0, dtype=dtype, device=device,
                   requires_grad=True)
    b = torch.arange(96, device=device).to(dtype)
    y = fused_layer_norm(x, None, b, eps=1e-5)
    assert torch.equal(y, b.expand(3, 96))
    y.sum().backward()
    assert torch.equal(x.grad, torch.zeros_like(x))


@on_devices
def test_norm_rows_of_nothing(device):
    x = torch.zeros(0, 4, 64, device=device, requires_grad=True)
    w = torch.ones(64, device=device, requires_grad=True)
    y, s = fused_layer_norm(x, w, None, residual=torch.zeros_like(x))
    assert y.shape == s.shape == (0, 4, 64)
    (y.sum() + s.sum()).backward()
    assert torch.equal(w.grad, torch.zeros(64, device=device))
    assert x.grad.shape == x.shape


@on_devices
@on_types
def test_norm_strides(device, dtype):
    """Rows of a wider tensor, transposed and broadcast inputs, a misaligned
    start: the same numbers as from contiguous copies."""
    g = rng(5)
    wide = normal(g, 6, 5, 300, dtype=dtype, device=device)
    flat = normal(g, 6 * 5 * 129 + 3, dtype=dtype, device=device)
    xs = [wide[..., 7:136], wide[:, 1:3, :129], wide.transpose(0, 1)[..., :129],
          wide[:, :1, :129].expand(6, 4, 129), flat[3:].view(6, 5, 129),
          wide[0].t()[:129], wide[::2, ::2, 1:130]]
    w = normal(g, 129, dtype=dtype, device=device)
    for x in xs:
        w_ = w[:x.shape[-1]] if x.shape[-1] < 129 else w
        for res in (None, x.flip(0) if x.dim() > 2 else x):
            a = x.detach().requires_grad_(True)
            c = x.detach().clone(
                memory_format=torch.contiguous_format).requires_grad_(True)
            r = None if res is None else res.clone(
                memory_format=torch.contiguous_format)
            got, want = (fused_layer_norm(v, w_, w_, residual=q)
                         for v, q in ((a, res), (c, r)))
            got, want = (v if res is not None else (v,) for v in (got, want))
            assert all(torch.equal(p, q) for p, q in zip(got, want))
            sum(p.float().square().sum() for p in got).backward()
            sum(p.float().square().sum() for p in want).backward()
            assert torch.equal(a.grad, c.grad)


@on_devices
def test_norm_one_gradient_missing(device):
    g = rng(8)
    x = normal(g, 4, 70, dtype=torch.float32, device=device)
    x.requires_grad_(True)
    w = normal(g, 70, dtype=torch.float32, device=device)
    w.requires_grad_(True)
    y, s = fused_layer_norm(x, w, None, residual=torch.ones_like(x))
    gx, gw = torch.autograd.grad(s.sum(), [x, w], retain_graph=True,
                                 allow_unused=True)
    assert torch.equal(gx, torch.ones_like(x))
    assert gw is None or torch.equal(gw, torch.zeros_like(w))
    gx, = torch.autograd.grad(y.sum(), [x])
    assert torch.isfinite(gx).all()


def test_norm_gradient_against_differences():
    """The formula the kernels are held to, against central differences."""
    g = rng(9)
    x = normal(g, 3, 12, dtype=torch.float64, device="cpu")
    w, b = torch.rand(12, generator=g), torch.rand(12, generator=g)
    dy = normal(g, 3, 12, dtype=torch.float64, device="cpu")
    f = lambda v: (torch.nn.functional.layer_norm(  # noqa: E731
        v, (12,), w.double(), b.double(), 1e-5) * dy).sum()
    x32 = x.float()
    want = norm_oracle(x32, w, b, 1e-5, None, dy.float(), None)[0]["dx"]
    h = 1e-6
    for i, j in itertools.product(range(3), range(12)):
        up, down = x32.double().clone(), x32.double().clone()
        up[i, j] += h
        down[i, j] -= h
        # dy was rounded to 32 bits for the formula
        assert abs((f(up) - f(down)) / (2 * h) - want[i, j]) < 1e-5


@on_devices
def test_norm_refuses(device):
    x = torch.randn(4, 16, device=device)
    w = torch.randn(16, device=device)
    for bad in (dict(x=x.double()), dict(x=x.long()), dict(w=w.double()),
                dict(x=x.bfloat16(), w=w.half()), dict(res=x.half()),
                dict(b=w.double())):
        with pytest.raises(TypeError):
            fused_layer_norm(bad.get("x", x), bad.get("w", w), bad.get("b"),
                             residual=bad.get("res"))
    with pytest.raises(TypeError):
        fused_layer_norm(x.half(), w, w.half())
    for bad in (dict(w=w[:15]), dict(w=w[None]), dict(b=torch.cat([w, w])),
                dict(res=x[:3]), dict(x=x[:, :0], w=w[:0]),
                dict(res=x[0])):
        with pytest.raises(ValueError):
            fused_layer_norm(bad.get("x", x), bad.get("w", w), bad.get("b"),
                             residual=bad.get("res"))
    with pytest.raises(ValueError):
        FusedLayerNorm(8)(torch.zeros(2, 16))


# ---------------------------------------------------------------------------
# linear
# ---------------------------------------------------------------------------

ACTS = [None, "relu", "gelu", "silu"]


def act_oracle(z, act):
    """Value, slope, and the most the slope changes with its argument."""
    if act == "relu":
        return z.clamp_min(0), (z > 0).double(), 0.0
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        pdf = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf, 0.8
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), 0.5
    return z, torch.ones_like(z), 0.0


def run_linear(device, dtype, m, k, n, act=None, residual=False, bias=True,
               btype=None, whole=False, lead=None):
    g = rng(m, k, n)
    if act == "relu" or whole:
        # whole numbers and a bias of halves: z is exact in every order of
        # the sum, and never zero, where relu's slope jumps
        draw = lambda *s: torch.randint(  # noqa: E731
            -2, 3, s, generator=g).to(dtype).to(device)
        x, w = draw(m, k), draw(n, k)
        b = (draw(n).float() + 0.5).to(dtype) if bias else None
        if act == "relu" and not bias:
            raise AssertionError("relu's cases have a bias")
    else:
        x = normal(g, m, k, dtype=dtype, device=device)
        w = normal(g, n, k, dtype=dtype, device=device, scale=k ** -0.5)
        b = normal(g, n, dtype=dtype, device=device, scale=0.3) \
            if bias else None
    if b is not None and btype is not None:
        b = b.to(btype)
    res = normal(g, m, n, dtype=dtype, device=device) if residual else None
    dy = normal(g, m, n, dtype=dtype, device=device)
    if lead:  # leading axes
        x = x.view(*lead, k)
        dy = dy.view(*lead, n)
        res = res.view(*lead, n) if residual else None
    leaves = [v for v in (x, w, b, res) if v is not None]
    for v in leaves:
        v.requires_grad_(True)
    y = fused_linear(x, w, b, act, res)
    grads = iter(torch.autograd.grad(y, leaves, dy))
    assert y.dtype == dtype and y.shape == dy.shape

    x64, w64, dy64 = (v.detach().cpu().double().view(-1, v.shape[-1])
                      for v in (x, w, dy))
    b64 = torch.zeros(n, dtype=torch.float64) if b is None else \
        b.detach().cpu().double()
    z = x64 @ w64.t() + b64
    a, slope, bend = act_oracle(z, act)
    # a product's sum: k terms, and the bias
    err_z = (k + 64) * U * (x64.abs() @ w64.abs().t() + b64.abs())
    value = a if res is None else a + res.detach().cpu().double().view(-1, n)
    # no activation here has a slope over 1.13; exp and erf are good to 16 U
    err_y = 1.13 * err_z + 16 * U * (z.abs() + a.abs() + value.abs())
    within(y.reshape(-1, n), value, err_y + stored(value, dtype), "y")
    # backward: z is kept in the type, dz is rounded to it
    dz = dy64 * slope
    err_dz = dy64.abs() * (bend * (err_z + stored(z, dtype)) + 32 * U * (
        1 + z.abs()))
    if act in (None, "relu"):
        err_dz = torch.zeros_like(dz)
    sum_dz = err_dz.clone()
    if act in ("gelu", "silu"):
        err_dz = err_dz + stored(dz, dtype)
    dx = dz @ w64
    within(next(grads).reshape(-1, k), dx,
           err_dz @ w64.abs() + (n + 64) * U * (dz.abs() @ w64.abs())
           + stored(dx, dtype), "dx")
    dw = dz.t() @ x64
    within(next(grads), dw,
           err_dz.t() @ x64.abs() + (m + 64) * U * (dz.abs().t() @ x64.abs())
           + stored(dw, dtype), "dw")
    if b is not None:
        db = dz.sum(0)
        got = next(grads)
        assert got.dtype == b.dtype
        within(got, db, sum_dz.sum(0) + (m + 64) * U * dz.abs().sum(0)
               + stored(db, b.dtype), "db")
    if res is not None:
        assert torch.equal(next(grads), dy)
    with torch.no_grad():
        assert torch.equal(fused_linear(x, w, b, act, res), y)


# (m, k, n): single elements and tokens, sizes on both sides of every tile's
# edge, sizes that no vector divides
LINEAR_SHAPES = [(1, 1, 1), (1, 64, 100), (2, 7, 3), (5, 129, 65),
                 (16, 256, 64), (17, 72, 40), (64, 64, 64), (65, 96, 130),
                 (128, 128, 128), (100, 333, 71), (129, 200, 257),
                 (256, 64, 256), (300, 520, 264), (64, 66, 31), (33, 130, 47),
                 (1, 9001, 20), (40, 20000, 17), (70, 2600, 150),
                 (257, 1300, 40)]


@on_devices
@on_types
@pytest.mark.parametrize("m,k,n", LINEAR_SHAPES)
def test_linear(device, dtype, m, k, n):
    run_linear(device, dtype, m, k, n)


# sizes that the largest tiles are taken for, forward, in dx and in dW; k of
# less than a tile, one, two and three tiles, and some more
@pytest.mark.gpu
@on_types
@pytest.mark.parametrize("m,k,n", [
    (4100, 40, 4100), (4100, 64, 4100), (4100, 128, 4100), (4100, 192, 4100),
    (4100, 330, 4099), (4096, 4100, 330), (330, 4100, 4096),
    (2050, 1000, 700)])
def test_linear_large(dtype, m, k, n):
    """Whole numbers, so that every sum is exact: equal to the formula in 64
    bits, rounded once."""
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    draw = lambda *s: torch.randint(  # noqa: E731
        -2, 3, s, generator=g, device="cuda").to(dtype)
    x, w, b, res, dy = draw(m, k), draw(n, k), draw(n) + 0.5, draw(m, n), \
        draw(m, n)
    for v in (x, w, b, res):
        v.requires_grad_(True)
    y = fused_linear(x, w, b, "relu", res)
    got = torch.autograd.grad(y, [x, w, b], dy)
    x64, w64, dy64 = (v.detach().double() for v in (x, w, dy))
    z = x64 @ w64.t() + b.detach().double()
    assert torch.equal(y, (z.clamp_min(0) + res.detach().double()).to(dtype))
    dz = torch.where(z > 0, dy64, 0.0)
    for a, c in zip(got, (dz @ w64, dz.t() @ x64, dz.sum(0))):
        assert torch.equal(a, c.to(dtype))


@pytest.mark.gpu
def test_linear_rows_far_apart():
    """Rows 2^23 elements apart, more than a tile's offsets reach."""
    wide = torch.zeros(140, 1 << 23, dtype=torch.bfloat16, device="cuda")
    x = wide[:, :128]
    x.copy_(torch.randint(-2, 3, (140, 128), device="cuda"))
    w = torch.randint(-2, 3, (200, 128), device="cuda").bfloat16()
    y = fused_linear(x, w)
    assert torch.equal(y, (x.double() @ w.double().t()).bfloat16())
    dx, dw = (v.detach().requires_grad_(True) for v in (x, w))
    fused_linear(dx, dw).backward(torch.ones_like(y))
    assert torch.equal(dw.grad, x.double().sum(0).bfloat16().expand(200, 128))


@pytest.mark.parametrize("m,k,n", [(4, 1 << 22, 2), (4, 2, 1 << 22)])
@pytest.mark.gpu
def test_linear_refuses_sizes(m, k, n):
    x = torch.zeros(m, k, dtype=torch.float16, device="cuda")
    w = torch.zeros(n, k, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        fused_linear(x, w)


@on_devices
@on_types
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("residual", [False, True])
def test_linear_epilogue(device, dtype, act, residual):
    run_linear(device, dtype, 77, 40, 90, act, residual)
    run_linear(device, dtype, 3, 48, 130, act, residual)


@on_devices
def test_linear_bias(device):
    run_linear(device, torch.bfloat16, 33, 65, 66, "gelu", bias=False)
    run_linear(device, torch.bfloat16, 33, 65, 66, "gelu",
               btype=torch.float32)
    run_linear(device, torch.float16, 6, 24, 40, "silu", True, bias=False,
               lead=(2, 3))


@on_devices
@on_types
def test_linear_nothing(device, dtype):
    for m, n in ((0, 5), (4, 0)):
        x = torch.ones(m, 6, dtype=dtype, device=device, requires_grad=True)
        w = torch.ones(n, 6, dtype=dtype, device=device, requires_grad=True)
        b = torch.ones(n, dtype=dtype, device=device, requires_grad=True)
        y = fused_linear(x, w, b, "gelu", torch.ones(m, n, dtype=dtype,
                                                     device=device))
        assert y.shape == (m, n)
        y.sum().backward()
        for v in (x, w, b):
            assert torch.equal(v.grad, torch.zeros_like(v))


@on_devices
@on_types
def test_linear_strides(device, dtype):
    """Slices, transposes, broadcasts and misaligned starts: the numbers of
    contiguous copies."""
    g = rng(12)
    # whole numbers: every order of the sums gives the same
    draw = lambda *s: torch.randint(-2, 3, s, generator=g).to(dtype).to(  # noqa: E731
        device)
    wide, wide_w, wide_r = draw(6, 5, 200), draw(90, 200), draw(6, 5, 91)
    xs = [wide[..., :73], wide[..., 1:74], wide.transpose(0, 1)[..., :73],
          wide[:, :1, :73].expand(6, 5, 73), wide[0].t()[:73].t()]
    ws = [wide_w[:, :73], wide_w[:, 3:76], wide_w[::2, :73],
          draw(73, 60).t(), wide_w[:1, :73].expand(70, 73)]
    for x, w in itertools.product(xs, ws):
        res = wide_r[..., :w.shape[0]].expand(
            *x.shape[:-1], w.shape[0]) if x.shape[:-1] == (6, 5) and \
            w.shape[0] <= 91 else None
        a, b = (v.detach().requires_grad_(True) for v in (x, w))
        c, d = (v.detach().contiguous().clone().requires_grad_(True)
                for v in (x, w))
        got = fused_linear(a, b, None, "relu", res)
        want = fused_linear(c, d, None, "relu",
                            None if res is None else res.contiguous())
        assert torch.equal(got, want)
        got.sum().backward()          # a broadcast gradient
        want.backward(torch.ones_like(want))
        assert torch.equal(a.grad, c.grad) and torch.equal(b.grad, d.grad)


@on_devices
def test_linear_some_gradients(device):
    g = rng(14)
    x, w, b = (normal(g, *s, dtype=torch.float32, device=device)
               for s in ((9, 20), (30, 20), (30,)))
    dy = normal(g, 9, 30, dtype=torch.float32, device=device)
    ref = {}
    for need in itertools.product([True, False], repeat=3):
        if not any(need):
            continue
        leaves = [v.clone().requires_grad_(r) for v, r in
                  zip((x, w, b), need)]
        fused_linear(*leaves, "silu").backward(dy)
        for i, (v, r) in enumerate(zip(leaves, need)):
            assert (v.grad is not None) == r
            if r:
                assert torch.equal(ref.setdefault(i, v.grad), v.grad)


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_linear_slope_against_differences(act):
    z = torch.linspace(-6, 6, 241, dtype=torch.float64)
    h = 1e-5
    diff = (act_oracle(z + h, act)[0] - act_oracle(z - h, act)[0]) / (2 * h)
    value, slope, bend = act_oracle(z, act)
    assert (diff - slope).abs().max() < 1e-9
    bent = (act_oracle(z + h, act)[1] - act_oracle(z - h, act)[1]) / (2 * h)
    assert bent.abs().max() <= bend
    assert slope.abs().max() <= 1.13
    ref = {"gelu": torch.nn.functional.gelu,
           "silu": torch.nn.functional.silu}[act](z)
    assert (ref - value).abs().max() < 1e-14


@on_devices
@on_types
def test_linear_spreads_what_is_not_finite(device, dtype):
    """An infinity or NaN reaches its own row and column and no other."""
    x = torch.ones(70, 40, dtype=dtype, device=device)
    w = torch.ones(90, 40, dtype=dtype, device=device)
    x[3, 39] = math.inf
    x[69, 0] = math.nan
    w[7, 5] = -math.inf
    y = fused_linear(x, w).float().cpu()
    want = torch.full((70, 90), 40.0)
    want[3] = math.inf
    want[:, 7] = -math.inf
    want[3, 7] = math.nan
    want[69] = math.nan
    assert torch.equal(y.nan_to_num(1, 2, 3), want.nan_to_num(1, 2, 3))


@on_devices
def test_linear_refuses(device):
    x = torch.randn(4, 16, device=device)
    w = torch.randn(8, 16, device=device)
    b = torch.randn(8, device=device)
    r = torch.randn(4, 8, device=device)
    with pytest.raises(ValueError):
        fused_linear(x, w, b, "tanh")
    with pytest.raises(ValueError):
        FusedLinear(3, 4, activation="tanh")
    for args in ((x.double(), w.double()), (x.half(), w), (x, w, b.half()),
                 (x, w, b, None, r.half()), (x.int(), w.int()),
                 (x.half(), w.half(), b.bfloat16())):
        with pytest.raises(TypeError):
            fused_linear(*args)
    for args in ((x, w[:, :15]), (x, w[0]), (x, w, b[:7]), (x, w, b[None]),
                 (x, w, b, None, r[:3]), (x, w, b, None, r[:, :7]),
                 (x[:, :0], w[:, :0]), (x, w, None, None, r[None])):
        with pytest.raises(ValueError):
            fused_linear(*args)


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------

IGNORE = -100


def logprob_oracle(x, t, top_k, glp, gent):
    """(results, bounds) in 64 bits for rows without NaN and +inf."""
    dtype, v = x.dtype, x.shape[-1]
    x = x.double()
    kept = t != IGNORE
    none = (x == -math.inf).all(-1)
    m = torch.where(none, 0.0, x.amax(-1))[:, None]
    d = x - m
    e = d.exp()
    total = torch.where(none, 1.0, e.sum(-1))
    logs = total.log()[:, None]
    p = e / total[:, None]
    logp = d - logs
    safe = torch.where(p > 0, logp, 0.0)
    far = torch.where(p > 0, d.abs(), 0.0)
    ent = -(p * safe).sum(-1)
    chosen = logp.gather(-1, torch.where(kept, t, 0)[:, None])[:, 0]
    got = {"lp": torch.where(kept, torch.where(none, -math.inf, chosen), 0.0),
           "ent": torch.where(kept & ~none, ent, 0.0)}
    # each e^d is off by (2 |d| + 4) U of itself (the argument's two
    # roundings, exp's own), the sums by their chains: a wave's longest part
    # of a row, the joins
    chain = v / 64 + 128
    spread = (p * far).sum(-1)
    err_s = ((2 * (p * far).sum(-1) + 4) + chain) * U
    err_lp = err_s + 4 * U * (1 + logs[:, 0])
    tol = {"lp": torch.where(kept & ~none,
                             err_lp + 4 * U * chosen.nan_to_num(
                                 0, 0, 0).abs(), 0.0)}
    second = (p * far * far).sum(-1)
    tol["ent"] = err_lp + 2 * U * (2 * second + (4 + chain) * spread) \
        + err_s * spread + 4 * U * (ent.abs() + logs[:, 0])
    # the eager composition adds the terms p |log p|, whose sum is the entropy
    # itself, each off by its rounding and by log p's
    tol["ent"] = tol["ent"] + (chain + 8) * U * ent.abs()
    if top_k:
        key = x.clone()
        ids = torch.sort(key, dim=-1, descending=True, stable=True)[1][
            :, :top_k]
        got["ids"] = torch.where(kept[:, None], ids, -1)
        tops = torch.where(none[:, None], -math.inf, logp.gather(-1, ids))
        got["tops"] = torch.where(kept[:, None], tops, -math.inf)
        tol["tops"] = err_lp[:, None] + 4 * U * tops.nan_to_num(
            0, 0, 0).abs()
    if glp is not None or gent is not None:
        zero = torch.zeros(x.shape[0], dtype=torch.float64)
        live = (kept & ~none)[:, None]
        a = (zero if glp is None else glp.double())[:, None]
        b = (zero if gent is None else gent.double())[:, None]
        hit = torch.zeros_like(x).scatter_(-1, torch.where(kept, t, 0)[:, None],
                                           1.0)
        dx = a * (hit - p) - b * p * (safe + ent[:, None])
        got["dx"] = torch.where(live, dx, 0.0)
        err_p = p * (err_lp[:, None] + (4 * safe.abs() + 4 * far + 8) * U)
        size = a.abs() + b.abs() * (safe.abs() + ent[:, None].abs())
        tol["dx"] = err_p * size + p * (
            b.abs() * (tol["ent"][:, None] + err_lp[:, None]
                       + 8 * U * safe.abs()) + 8 * U * size) \
            + 4 * U * a.abs() * hit + stored(got["dx"], dtype) + 1e-36
        # what is below the smallest normal float may be taken as zero
    return got, tol


def make_logits(g, dtype, device, rows, vocab, scale=2.0):
    x = normal(g, rows, vocab, dtype=torch.float64, device="cpu", scale=scale)
    x = x.to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g)
    if rows > 2:
        t[rows // 2] = IGNORE
    return x, t


def run_logprobs(device, x, t, top_k, both=True, rounded=True):
    """x and t on the CPU."""
    g = rng(3)
    rows = x.shape[0]
    glp = torch.randn(rows, generator=g)
    gent = torch.randn(rows, generator=g)
    want, tol = logprob_oracle(x, t, top_k, glp, gent if both else None)
    leaf = x.to(device).requires_grad_(True)
    out = token_logprobs(leaf, t.to(device), top_k)
    assert out.logprobs.dtype == out.entropy.dtype == torch.float32
    within(out.logprobs, want["lp"], tol["lp"], "logprobs")
    within(out.entropy, want["ent"], tol["ent"], "entropy")
    if top_k:
        assert torch.equal(out.top_ids.cpu(), want["ids"])
        within(out.top_logprobs, want["tops"], tol["tops"], "top_logprobs")
        assert not out.top_ids.requires_grad
        assert not out.top_logprobs.requires_grad
    else:
        assert out.top_ids is None and out.top_logprobs is None
    loss = (out.logprobs * glp.to(device))
    kept = torch.isfinite(out.logprobs)
    outs, gs = [out.logprobs], [glp.to(device)]
    if both:
        outs.append(out.entropy)
        gs.append(gent.to(device))
    del loss, kept
    dx, = torch.autograd.grad(outs, [leaf], gs)
    assert dx.dtype == x.dtype
    within(dx, want["dx"], tol["dx"], "dx")
    with torch.no_grad():
        again = token_logprobs(leaf, t.to(device), top_k)
    for a, b in zip(again, out):
        assert (a is None and b is None) or torch.equal(a, b)


# a single entry; a wave a row up to its last size; a block a row; a row cut
# into parts; parts that end inside a step
LOGPROB_SHAPES = [(1, 1), (3, 2), (512, 10), (5, 100), (130, 1000),
                  (4, 1024), (4, 1025), (3, 2048), (2, 2049), (6, 5003),
                  (1, 40000), (70, 9000), (600, 2500), (1, 131072)]


@on_devices
@on_types
@pytest.mark.parametrize("rows,vocab", LOGPROB_SHAPES)
def test_logprobs(device, dtype, rows, vocab):
    x, t = make_logits(rng(rows, vocab), dtype, device, rows, vocab)
    run_logprobs(device, x, t, min(5, vocab))
    run_logprobs(device, x, t, 0, both=False)


@on_devices
@pytest.mark.parametrize("top_k", [1, 2, 31, 63, 64])
@pytest.mark.parametrize("rows,vocab", [(7, 64), (3, 700), (2, 30011),
                                        (520, 4099)])
def test_logprobs_top(device, top_k, rows, vocab):
    x, t = make_logits(rng(rows, vocab), torch.float32, device, rows, vocab)
    run_logprobs(device, x, t, top_k)


@on_devices
@on_types
def test_logprobs_equal_values(device, dtype):
    """Ties go to the lowest index, in every order the values may come in;
    the two zeros are one value."""
    vocab = 5000
    rows = [torch.zeros(vocab), torch.arange(vocab) // 1000 * 1.0,
            torch.arange(vocab).flip(0) // 1000 * 1.0,
            torch.arange(vocab) % 7 * 1.0, torch.arange(vocab) / 64.0,
            torch.arange(vocab).flip(0) / 64.0,
            torch.where(torch.arange(vocab) % 2 == 0, -0.0, 0.0)]
    x = torch.stack(rows).to(dtype)
    t = torch.arange(len(rows)) * 600
    run_logprobs(device, x, t, 40)


@on_devices
@on_types
@pytest.mark.parametrize("vocab", [9, 300, 20000])
def test_logprobs_masked(device, dtype, vocab):
    """-inf and the type's lowest value in places, in whole rows, and in all
    but one entry."""
    g = rng(vocab)
    x, _ = make_logits(g, dtype, device, 9, vocab)
    t = torch.randint(0, vocab, (9,), generator=g)
    low = torch.finfo(dtype).min
    x[0] = -math.inf
    x[1, torch.randperm(vocab, generator=g)[: vocab - 1]] = -math.inf
    x[2, vocab // 2:] = -math.inf
    t[2] = vocab - 1                # the target is masked
    x[3] = low
    x[4, vocab // 2:] = low
    t[4] = 0
    x[5, : vocab // 2] = -math.inf
    t[5] = vocab - 1
    t[6] = IGNORE
    x[6] = math.nan                 # passed over, whatever it holds
    x[7, 0] = torch.finfo(dtype).max
    t[7] = 0
    t[8] = IGNORE
    x[8] = -math.inf
    clean = x.clone()
    clean[6] = 0
    g1, g2 = torch.randn(9, generator=g), torch.randn(9, generator=g)
    top = min(5, vocab)
    want, tol = logprob_oracle(clean, t, top, g1, g2)
    leaf = x.to(device).requires_grad_(True)
    out = token_logprobs(leaf, t.to(device), top)
    within(out.logprobs, want["lp"], tol["lp"], "logprobs")
    within(out.entropy, want["ent"], tol["ent"], "entropy")
    assert torch.equal(out.top_ids.cpu(), want["ids"])
    within(out.top_logprobs, want["tops"], tol["tops"], "top")
    dx, = torch.autograd.grad([out.logprobs, out.entropy], leaf,
                              [g1.to(device), g2.to(device)])
    within(dx, want["dx"], tol["dx"], "dx")
    assert torch.equal(dx[0].cpu(), torch.zeros(vocab, dtype=dtype))


@on_devices
@pytest.mark.parametrize("vocab", [50, 3000, 30000])
def test_logprobs_not_finite(device, vocab):
    """NaN and +inf make a row NaN, and only that row; NaN is the largest of
    the alternatives; targets outside give NaN."""
    x, t = make_logits(rng(vocab), torch.float32, device, 6, vocab)
    t[3] = 1
    x[0, vocab - 1] = math.nan
    x[1, 3] = math.inf
    x[4] = -math.inf
    x[4, 7] = math.nan
    t[4] = 2
    t[2], t[5] = vocab, -1
    good, _ = logprob_oracle(x[3:4], t[3:4], 3, None, None)
    leaf = x.to(device).requires_grad_(True)
    out = token_logprobs(leaf, t.to(device), 3)
    assert torch.isnan(out.logprobs.cpu()[[0, 1, 2, 4, 5]]).all()
    assert torch.isnan(out.entropy.cpu()[[0, 1, 4]]).all()
    assert torch.isfinite(out.entropy.cpu()[[2, 3, 5]]).all()
    assert abs(out.logprobs[3].item() - good["lp"].item()) < 1e-4
    assert out.top_ids[0, 0].item() == vocab - 1
    assert out.top_ids[1, 0].item() == 3
    assert out.top_ids[4].tolist() == [7, 0, 1]
    dx, = torch.autograd.grad(out.logprobs.sum(), leaf)
    assert torch.isnan(dx.cpu()[[0, 1, 2, 4, 5]]).all()
    assert torch.isfinite(dx[3]).all()


@on_devices
def test_logprobs_shapes_and_strides(device):
    g = rng(21)
    for vocab in (70, 4500):
        wide = normal(g, 3, 4, vocab + 30, dtype=torch.bfloat16,
                      device=device)
        t = torch.randint(0, vocab, (4, 3), generator=g).to(device).t()
        for x in (wide[..., :vocab], wide[..., 5:vocab + 5],
                  wide.transpose(0, 1).contiguous().transpose(0, 1)[
                      ..., :vocab],
                  wide[:, :1, :vocab].expand(3, 4, vocab),
                  wide.flatten(0, 1).t().contiguous().t().view(
                      3, 4, -1)[..., :vocab]):
            a = x.detach().requires_grad_(True)
            c = x.detach().contiguous().clone().requires_grad_(True)
            p = token_logprobs(a, t, 3)
            q = token_logprobs(c, t.contiguous(), 3)
            assert p.top_ids.shape == (3, 4, 3)
            assert all(torch.equal(u, v) for u, v in zip(p, q))
            (p.logprobs.sum() + p.entropy.sum()).backward()
            (q.logprobs.sum() + q.entropy.sum()).backward()
            assert torch.equal(a.grad, c.grad)
    one = token_logprobs(wide[0, 0], torch.tensor(3, device=device), 2)
    assert one.logprobs.shape == () and one.top_ids.shape == (2,)
    none = token_logprobs(wide[:0], t[:0], 2)
    assert none.logprobs.shape == (0, 4) and none.top_ids.shape == (0, 4, 2)
    x = wide[:0].detach().requires_grad_(True)
    token_logprobs(x, t[:0]).logprobs.sum().backward()
    assert x.grad.shape == x.shape


def test_logprobs_gradient_against_differences():
    g = rng(31)
    x = normal(g, 2, 9, dtype=torch.float64, device="cpu").float()
    t = torch.tensor([4, 0])
    glp, gent = torch.tensor([0.7, -1.0]), torch.tensor([0.3, 2.0])

    def f(v):
        lp = torch.log_softmax(v, -1)
        return (lp.gather(-1, t[:, None])[:, 0] * glp.double()
                - (lp.exp() * lp).sum(-1) * gent.double()).sum()

    want = logprob_oracle(x, t, 0, glp, gent)[0]["dx"]
    h = 1e-6
    for i, j in itertools.product(range(2), range(9)):
        up, down = x.double().clone(), x.double().clone()
        up[i, j] += h
        down[i, j] -= h
        assert abs((f(up) - f(down)) / (2 * h) - want[i, j]) < 1e-8


@on_devices
def test_logprobs_refuses(device):
    x = torch.randn(4, 16, device=device)
    t = torch.zeros(4, dtype=torch.int64, device=device)
    for args in ((x.double(), t), (x.long(), t), (x, t.int()),
                 (x, t.float())):
        with pytest.raises(TypeError):
            token_logprobs(*args)
    for args in ((x, t[:3]), (x, t[:, None]), (x, t, -1), (x, t, 17),
                 (x.repeat(1, 9), t, 65), (x[:, :0], t),
                 (x[0, 0], t[0])):
        with pytest.raises((ValueError, IndexError)):
            token_logprobs(*args)


@on_devices
def test_logprobs_are_loss_and_accuracy(device):
    """What the trainers compute from the same logits."""
    g = rng(41)
    out = normal(g, 64, 10, dtype=torch.float32, device=device, scale=3.0)
    y = torch.randint(0, 10, (64,), generator=g).to(device)
    got = token_logprobs(out, y, 5)
    want = torch.nn.functional.cross_entropy(out, y)
    assert abs(-got.logprobs.mean() - want) < 1e-5
    hits = got.top_ids == y[:, None]
    for k, acc in zip((1, 5), accuracy(out, y, topk=(1, 5))):
        assert abs(hits[:, :k].sum() * 100.0 / 64 - acc) < 1e-3


@on_devices
def test_trainer_validates_from_one_read(device, capsys):
    """train_resnet18 --val_stats: the same line as without, and the
    entropy."""
    from cpd_amd.trainers.train_resnet18 import parse_args, validate
    assert parse_args(["--val_stats"]).val_stats
    assert not parse_args([]).val_stats
    torch.manual_seed(6)
    model = torch.nn.Linear(12, 10).to(device)
    data = [(torch.randn(32, 12), torch.randint(0, 10, (32,)))
            for _ in range(3)]
    said = []
    for stats in (False, True):
        prec = validate(data, model, torch.nn.CrossEntropyLoss(),
                        torch.device(device), 1, 0, stats)
        said.append((prec, capsys.readouterr().out.split()))
    (p, a), (q, b) = said
    assert abs(p - q) < 1e-4
    assert a[:3] == b[:3] == ["*", "All", "Loss"] and len(a) == 8
    for i in (3, 5, 7):
        assert abs(float(a[i]) - float(b[i])) < 2e-3
    with torch.no_grad():
        lp = torch.stack([torch.log_softmax(model(x.to(device)), -1)
                          for x, _ in data])
    assert b[8] == "Entropy"
    assert abs(float(b[9]) + (lp.exp() * lp).sum(-1).mean().item()) < 1e-3


# ---------------------------------------------------------------------------
# modules, and the run of them together
# ---------------------------------------------------------------------------

@on_devices
def test_modules_load_from_torch(device):
    torch.manual_seed(0)
    ln, ref = FusedLayerNorm(24).to(device), torch.nn.LayerNorm(24).to(device)
    fc, fref = FusedLinear(24, 12).to(device), torch.nn.Linear(24, 12).to(
        device)
    ln.load_state_dict(ref.state_dict())
    fc.load_state_dict(fref.state_dict())
    x = torch.randn(5, 24, device=device)
    torch.testing.assert_close(fc(ln(x)), fref(ref(x)))
    assert set(FusedLayerNorm(4, bias=False).state_dict()) == {"weight"}
    assert not FusedLayerNorm(4, affine=False).state_dict()
    assert set(FusedLinear(4, 4, bias=False).state_dict()) == {"weight"}


class Block(torch.nn.Module):
    """Two residual blocks and a head over a vocabulary."""

    def __init__(self, width, inner, vocab):
        super().__init__()
        self.norms = torch.nn.ModuleList(
            FusedLayerNorm(width) for _ in range(3))
        self.up = torch.nn.ModuleList(
            FusedLinear(width, inner, activation=a) for a in ("gelu", "silu"))
        self.down = torch.nn.ModuleList(
            FusedLinear(inner, width) for _ in range(2))
        self.head = FusedLinear(width, vocab, bias=False)

    def forward(self, x, targets, top_k=0):
        y = self.norms[0](x)
        x = self.down[0](self.up[0](y), residual=x)
        delta = self.down[1](self.up[1](self.norms[1](x)))
        y, x = self.norms[2](delta, residual=x)
        return token_logprobs(self.head(y), targets, top_k)


def plain_block(m, x, targets, dtype=torch.float64):
    p = {k: v.detach().cpu().to(dtype).requires_grad_(True)
         for k, v in m.named_parameters()}
    ln = lambda i, v: torch.nn.functional.layer_norm(  # noqa: E731
        v, v.shape[-1:], p[f"norms.{i}.weight"], p[f"norms.{i}.bias"], 1e-5)
    fc = lambda n, v: torch.nn.functional.linear(  # noqa: E731
        v, p[f"{n}.weight"], p.get(f"{n}.bias"))
    x = x.detach().cpu().to(dtype).requires_grad_(True)
    h = x + fc("down.0", torch.nn.functional.gelu(fc("up.0", ln(0, x))))
    h = h + fc("down.1", torch.nn.functional.silu(fc("up.1", ln(1, h))))
    lp = torch.log_softmax(fc("head", ln(2, h)), -1)
    return lp.gather(-1, targets.cpu()[..., None])[..., 0], p, x


@on_devices
def test_run_together(device):
    """Block and loss, forward and backward, against 64 bits.  In 32 bits the
    whole run is good to about 1e-6 of each gradient's size; a hundred times
    that is allowed."""
    torch.manual_seed(1)
    m = Block(48, 130, 301).to(device)
    x = torch.randn(3, 7, 48, device=device, requires_grad=True)
    t = torch.randint(0, 301, (3, 7), device=device)
    out = m(x, t, 4)
    loss = -out.logprobs.mean()
    loss.backward()
    lp, p, x64 = plain_block(m, x, t)
    (-lp.mean()).backward()
    assert (out.logprobs.detach().cpu() - lp.detach()).abs().max() < 1e-4
    for name, v in m.named_parameters():
        far = (v.grad.cpu() - p[name].grad).norm() / p[name].grad.norm()
        assert far < 1e-4, (name, far)
    assert (x.grad.cpu() - x64.grad).norm() / x64.grad.norm() < 1e-4


def test_run_together_in_the_trainer_step():
    """The modules' gradients land in the bucket and are reduced with the
    rest: one (8, 23) step is one plain SGD step."""
    from cpd_amd.parallel import DistModule
    from cpd_amd.trainers.core import LPTrainStep
    torch.manual_seed(2)
    m = Block(16, 20, 11)
    before = {k: v.detach().clone() for k, v in m.named_parameters()}
    x, t = torch.randn(6, 16), torch.randint(0, 11, (6,))
    _, p, _ = lp = plain_block(m, x, t, torch.float32)
    (-lp[0].mean()).backward()
    step = LPTrainStep(DistModule(m), torch.optim.SGD(m.parameters(), lr=0.5),
                       grad_exp=8, grad_man=23, use_APS=False)
    assert step.substep(-m(x, t).logprobs.mean())
    for k, v in m.named_parameters():
        # the gradients of two orders of the same 32-bit sums
        torch.testing.assert_close(v, before[k] - 0.5 * p[k].grad, rtol=1e-4,
                                   atol=1e-6)


# ---------------------------------------------------------------------------
# streams, graphs and whole results again (GPU)
# ---------------------------------------------------------------------------

def step_of(m, x, t):
    """One pass with gradients, all of its results, detached: a captured
    backward must not meet leaves that an eager graph still holds (torch ties
    them to that graph's stream, and the capture ends the process)."""
    out = m(x, t, 4)
    leaves = [x] + list(m.parameters())
    grads = torch.autograd.grad([out.logprobs.sum(), out.entropy.sum()],
                                leaves)
    return [v.detach() for v in [*out, *grads]]


@pytest.mark.gpu
def test_gpu_not_twice_differentiable():
    """Asked for a graph of the gradient, the kernels say no instead of
    leaving a part of it out."""
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    w = torch.randn(8, 16, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for y in (fused_layer_norm(x), fused_linear(x, w, activation="silu"),
              token_logprobs(x, t).logprobs):
        with pytest.raises(RuntimeError, match="twice"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


@pytest.mark.gpu
@on_types
def test_gpu_twice_the_same(dtype):
    torch.manual_seed(3)
    m = Block(256, 520, 2000).cuda().to(dtype)
    x = torch.randn(300, 256, device="cuda").to(dtype).requires_grad_(True)
    t = torch.randint(0, 2000, (300,), device="cuda")
    a, b = step_of(m, x, t), step_of(m, x, t)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_gpu_on_another_stream():
    """Two streams at once, neither the default one: each gets the numbers of
    a pass alone."""
    torch.manual_seed(4)
    m = Block(128, 384, 9000).cuda().bfloat16()
    xs = [torch.randn(r, 128, device="cuda").bfloat16().requires_grad_(True)
          for r in (1, 40)]
    ts = [torch.randint(0, 9000, (r,), device="cuda") for r in (1, 40)]
    want = [step_of(m, x, t) for x, t in zip(xs, ts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got[i] = step_of(m, xs[i], ts[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, w))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 65])
def test_gpu_captured(rows):
    """Forward and backward in two graphs that are replayed in turn, with
    eager work between the replays."""
    torch.manual_seed(5)
    m = Block(128, 384, 9000).cuda().bfloat16()
    inputs = [[torch.randn(rows, 128, device="cuda").bfloat16(),
               torch.randint(0, 9000, (rows,), device="cuda")]
              for _ in range(3)]
    want = []
    for x, t in inputs:
        leaf = x.clone().requires_grad_(True)
        want.append([v.clone() for v in step_of(m, leaf, t)])
    graphs = []
    for _ in range(2):
        x = inputs[0][0].clone().requires_grad_(True)
        t = inputs[0][1].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step_of(m, x, t)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step_of(m, x, t)
        graphs.append((graph, x, t, out))
    for i in range(6):
        graph, x, t, out = graphs[i % 2]
        with torch.no_grad():
            x.copy_(inputs[i % 3][0])
            t.copy_(inputs[i % 3][1])
        graph.replay()
        step_of(m, inputs[0][0].clone().requires_grad_(True), inputs[0][1])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[i % 3]))


@pytest.mark.gpu
def test_gpu_far_offsets():
    """Logits whose offsets pass 2^31 elements: the last rows are right."""
    rows, vocab = 16400, 131072
    x = torch.zeros(rows, vocab, dtype=torch.float16, device="cuda")
    x[-2:] = torch.randn(2, vocab, device="cuda").half()
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    t[-1] = vocab - 1
    x.requires_grad_(True)
    out = token_logprobs(x, t, 2)
    want, tol = logprob_oracle(x[-2:].detach().cpu(), t[-2:].cpu(), 2,
                               torch.ones(2), None)
    within(out.logprobs[-2:], want["lp"], tol["lp"])
    assert torch.equal(out.top_ids[-2:].cpu(), want["ids"])
    dx, = torch.autograd.grad(out.logprobs.sum(), x)
    within(dx[-2:], want["dx"], tol["dx"])
    del x, dx, out
    y = fused_layer_norm(torch.ones(1 << 17, 1 << 15, dtype=torch.float16,
                                    device="cuda"))
    assert not y[-1].any() and not y[0].any()


@pytest.mark.gpu
def test_gpu_forward_mode_refused():
    """A tangent is refused, with and without a recorded graph, and not
    dropped."""
    from torch.autograd import forward_ad
    x = torch.randn(4, 16, device="cuda")
    w = torch.randn(8, 16, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    for f in (fused_layer_norm, lambda v: fused_linear(v, w),
              lambda v: fused_linear(x, w, None, None, v @ w.t()),
              lambda v: token_logprobs(v, t).logprobs):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match="jvp"):
                f(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
                f(dual)


@on_devices
def test_gradients_have_their_own_memory(device):
    """Inputs that share one gradient get two tensors, and an input given
    twice gets the sum."""
    x, res = (torch.randn(6, 32, device=device, requires_grad=True)
              for _ in range(2))
    w = torch.randn(32, 32, device=device)
    dy = torch.randn(6, 32, device=device)
    for f in (lambda a, b: sum(fused_layer_norm(a, residual=b)),
              lambda a, b: fused_linear(a, w, residual=b)):
        x.grad = res.grad = None
        f(x, res).backward(dy)
        assert x.grad.data_ptr() != res.grad.data_ptr()
        assert dy.data_ptr() not in (x.grad.data_ptr(), res.grad.data_ptr())
        a, b = x.grad.clone(), res.grad.clone()
        x.grad.zero_()
        assert torch.equal(res.grad, b)
        x.grad = None
        f(x, x).backward(dy)
        f2 = x.grad
        x.grad = res.grad = None
        same = x.detach().clone().requires_grad_(True)
        f(x, same).backward(dy)
        assert torch.equal(f2, x.grad + same.grad)
        assert a.shape == b.shape


# rows that four waves share unevenly; the last size that a wave has alone,
# and the next
@on_devices
@on_types
@pytest.mark.parametrize("rows", [1, 3, 9])
@pytest.mark.parametrize("vocab", [3, 255, 1024, 1028, 2048, 2056])
def test_logprobs_gradient_sizes(device, dtype, rows, vocab):
    x, t = make_logits(rng(rows, vocab, 5), dtype, device, rows, vocab)
    run_logprobs(device, x, t, 0)


@pytest.mark.gpu
def test_gpu_two_threads():
    """Two threads, each on a stream of its own, get the numbers of a pass
    alone."""
    import threading
    torch.manual_seed(6)
    m = Block(128, 384, 9000).cuda().bfloat16()
    xs = [torch.randn(r, 128, device="cuda").bfloat16() for r in (3, 200)]
    ts = [torch.randint(0, 9000, (r,), device="cuda") for r in (3, 200)]
    want = [step_of(m, x.clone().requires_grad_(True), t)
            for x, t in zip(xs, ts)]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = step_of(m, xs[i].clone().requires_grad_(True),
                                     ts[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    assert not errors and not any(th.is_alive() for th in threads)
    for g, w in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, w))


# dbias over few and many rows: one slice, two, and more than are in flight
@on_devices
@on_types
@pytest.mark.parametrize("m", [1, 64, 65, 130, 3001, 9000])
def test_linear_bias_gradient_rows(device, dtype, m):
    g = rng(m, 7)
    x = normal(g, m, 3, dtype=dtype, device=device)
    w = normal(g, 37, 3, dtype=dtype, device=device)
    b = torch.zeros(37, device=device, requires_grad=True)
    dy = normal(g, m, 37, dtype=dtype, device=device)
    db, = torch.autograd.grad(fused_linear(x, w, b), b, dy)
    dy = dy.cpu().double()
    within(db, dy.sum(0), (m + 64) * U * dy.abs().sum(0))


# What a row's waves tell each other: rows that rise, fall, lie flat, or have
# all of their largest values in one wave's share, with equal values on both
# sides of every share's edge.
@on_devices
@on_types
@pytest.mark.parametrize("top_k", [1, 4, 5, 16, 64])
@pytest.mark.parametrize("vocab", [2100, 20000])
def test_logprobs_top_orders(device, dtype, top_k, vocab):
    i = torch.arange(vocab, dtype=torch.float64)
    g = rng(vocab, top_k)
    rows = torch.stack([
        i / vocab, -i / vocab, torch.zeros(vocab), (i % 7) / 8,
        (i // 512 % 4 == 2).double(), (i // 512 % 4 == 0) * (i % 512),
        (i // 64 % 3 == 1).double() - (i % 2), -(i // 100),
        torch.where(i < vocab - 3, -math.inf, 1.0),
        torch.where(i % 700 == 5, 3.0, -math.inf),
        torch.randint(0, 3, (vocab,), generator=g).double()])
    x = rows.to(dtype)
    t = torch.full((len(x),), 3)
    out = token_logprobs(x.to(device), t.to(device), top_k)
    ids = torch.sort(x.double(), dim=-1, descending=True, stable=True)[1][
        :, :top_k]
    assert torch.equal(out.top_ids.cpu(), ids)


@pytest.mark.gpu
def test_gpu_logprobs_top_many_rows():
    """More rows than blocks: what a block kept of one row must not reach the
    next one that it takes, whose values are smaller."""
    rows, vocab, last = (1 << 20) + 40, 2056, 40
    x = torch.full((rows, vocab), 50.0, dtype=torch.float16, device="cuda")
    x[:last] += torch.arange(vocab, device="cuda") / 128
    x[-last:] = torch.randn(last, vocab, device="cuda").half()
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    out = token_logprobs(x, t, 20)
    for at in (slice(0, last), slice(rows - last, rows)):
        want = torch.sort(x[at].double(), dim=-1, descending=True,
                          stable=True)[1][:, :20]
        assert torch.equal(out.top_ids[at], want)


@on_devices
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_linear_argument_out_of_range(device, act):
    """An argument that fp16 does not hold: far below zero value and slope are
    zero, not NaN."""
    x = torch.full((3, 8), 100.0, dtype=torch.float16, device=device)
    w = torch.full((5, 8), -100.0, dtype=torch.float16, device=device)
    w[1] = 0.25
    x.requires_grad_(True)
    w.requires_grad_(True)
    b = torch.zeros(5, dtype=torch.float16, device=device, requires_grad=True)
    y = fused_linear(x, w, b, act)
    assert torch.equal(y[:, [0, 2, 3, 4]], torch.zeros_like(y[:, :4]))
    y.backward(torch.ones_like(y))
    assert torch.equal(b.grad, torch.tensor([0, 3, 0, 0, 0.]).to(b))
    assert torch.equal(x.grad, torch.full_like(x, 0.25))
    assert torch.equal(w.grad[0], torch.zeros_like(w[0]))
    assert torch.equal(w.grad[1], torch.full_like(w[1], 300.0))


# the last length of each way of sharing a row, forward and backward, in 16 and
# in 32 bits, and the next one
@on_devices
@on_types
@pytest.mark.parametrize("cols", [
    64, 65, 128, 129, 256, 257, 1024, 1025, 1028, 4096, 4100, 4104, 8192, 8200,
    16392, 32768, 32776])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_lengths(device, dtype, cols, residual):
    run_norm(device, dtype, 5, cols, residual)


@pytest.mark.gpu
def test_gpu_linear_far_offsets():
    """Outputs and gradients whose offsets pass 2^31 elements."""
    m, k, n = (1 << 19) + 5, 64, 4200
    x = torch.randint(-2, 3, (m, k), device="cuda").bfloat16()
    w = torch.randint(-2, 3, (n, k), device="cuda").bfloat16()
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = fused_linear(x, w, None, "relu")
    dy = torch.zeros_like(y)
    dy[-3:] = 1
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    z = x.detach()[-3:].double() @ w.detach().double().t()
    assert torch.equal(y[-3:], z.clamp_min(0).bfloat16())
    dz = (z > 0).double()
    assert torch.equal(dx[-3:], (dz @ w.detach().double()).bfloat16())
    assert not dx[:-3].any()
    assert torch.equal(dw, (dz.t() @ x.detach()[-3:].double()).bfloat16())


@on_devices
@pytest.mark.parametrize("m", [8, 200])
@pytest.mark.parametrize("scale", [1e-30, 1e-34, 1e-37, 1e30])
def test_linear_small_and_large_floats(device, m, scale):
    """Beside the sum's rounding an input may lose two parts of less than
    2^-126 each."""
    g = rng(m, 31)
    x = normal(g, m, 64, dtype=torch.float64, device="cpu",
               scale=scale).float()
    w = normal(g, 40, 64, dtype=torch.float32, device="cpu")
    y = fused_linear(x.to(device), w.to(device))
    x, w = x.double(), w.double()
    want = x @ w.t()
    size = x.abs() @ w.abs().t()
    within(y, want, (64 + 64) * U * size + 2.0 ** -125 * w.abs().sum(-1)
           + stored(want, torch.float32))


# Behind gelu and silu small products keep the gradient in floats: what dx and
# dW are off by is their own rounding and what z's makes of the slope.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [(1, 24, 4480), (12, 896, 54), (70, 130, 61),
                                   (300, 520, 264), (2, 5, 3), (515, 33, 700)])
def test_gpu_linear_gradients_rounded_once(dtype, act, m, k, n):
    g = rng(m, k, n, 9)
    x, dy = (normal(g, m, c, dtype=dtype, device="cuda") for c in (k, n))
    w = normal(g, n, k, dtype=dtype, device="cuda", scale=k ** -0.5)
    x.requires_grad_(True)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(fused_linear(x, w, None, act), [x, w], dy)
    x64, w64, dy64 = (v.detach().cpu().double() for v in (x, w, dy))
    z = x64 @ w64.t()
    _, slope, bend = act_oracle(z, act)
    dz = dy64 * slope
    # a float cut to two parts keeps 16 bits: 2^-15 of it are lost at most, and
    # the product of two second parts, 2^-16, is left out
    cut = 2.0 ** -14
    err_z = (k + 64) * U * (x64.abs() @ w64.abs().t())
    err = dy64.abs() * (bend * (err_z + stored(z, dtype)) + 32 * U * (
        1 + z.abs())) + cut * dz.abs()
    for got, want, tol in (
            (dx, dz @ w64, err @ w64.abs() + (n + 64) * U * (
                dz.abs() @ w64.abs())),
            (dw, dz.t() @ x64, err.t() @ x64.abs() + (m + 64) * U * (
                dz.abs().t() @ x64.abs()))):
        within(got, want, tol + stored(want, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [40, 4100])
def test_gpu_linear_gradients_not_finite(dtype, m):
    """Infinities and a NaN reach their own rows and columns and no others,
    on both sides of the size from which the gradient is rounded."""
    k, n = 72, 1024
    x = torch.ones(m, k, dtype=dtype, device="cuda")
    w = torch.full((n, k), 2.0 ** -7, dtype=dtype, device="cuda")
    dy = torch.ones(m, n, dtype=dtype, device="cuda")
    x[2, 4] = w[5, 7] = math.inf   # z infinite there: a slope of one
    dy[3, 9] = math.nan
    x.requires_grad_(True)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(fused_linear(x, w, None, "silu"), [x, w], dy)
    for got, row, col in ((dx, 3, 7), (dw, 9, 4)):
        kinds = torch.zeros(got.shape, device="cuda")
        kinds[:, col] = 1
        kinds[row] = 2
        assert torch.equal(got == math.inf, kinds == 1)
        assert torch.equal(got.isnan(), kinds == 2)
        assert torch.equal(got.isfinite(), kinds == 0)


# a row cut into the most parts, whose lists are joined 64 keys at a time or one
# by one
@on_devices
@pytest.mark.parametrize("top_k", [1, 8, 15, 16, 64])
def test_logprobs_top_of_many_parts(device, top_k):
    x, t = make_logits(rng(top_k), torch.bfloat16, device, 3, 140001)
    run_logprobs(device, x, t, top_k)


# Few rows and large weights, whose rows lie a power of two apart or not: blocks
# then begin at different places of k, and wrap round
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [
    (33, 64, 131100), (48, 130, 66000), (64, 384, 22000), (40, 448, 19000),
    (64, 2104, 4100), (48, 8200, 1100), (34, 40000, 257), (48, 16384, 520),
    (128, 4096, 300), (100, 2048, 4200), (65, 10240, 1000), (1, 16384, 40),
    (7, 4096, 1000), (20, 8192, 260), (32, 2048, 2050)])
def test_gpu_linear_large_weights(dtype, m, k, n):
    """Whole numbers: equal to the formula in 64 bits, rounded once."""
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    draw = lambda *s: torch.randint(  # noqa: E731
        -2, 3, s, generator=g, device="cuda").to(dtype)
    x, w, b, res = draw(m, k), draw(n, k), draw(n) + 0.5, draw(m, n)
    want = (x.double() @ w.double().t() + b.double()).clamp_min(0)
    assert torch.equal(fused_linear(x, w, b, "relu", res),
                       (want + res.double()).to(dtype))
    # a misaligned start, and a k that ends inside a tile of wider rows
    wide = torch.cat([x, x], 1)[:, 3:k + 3]
    want = wide.double() @ w.double().t()
    assert torch.equal(fused_linear(wide, w), want.to(dtype))
    x, w = x[:, :k - 21], w[:, :k - 21]
    assert torch.equal(fused_linear(x, w),
                       (x.double() @ w.double().t()).to(dtype))


# both sides of the sizes up to which few rows go straight from memory
@pytest.mark.gpu
@on_types
@pytest.mark.parametrize("m", [16, 17, 32, 33, 64, 65])
@pytest.mark.parametrize("k,n", [(2048, 4090), (2048, 4102), (4096, 6100),
                                 (4096, 6200)])
def test_gpu_linear_few_rows(dtype, m, k, n):
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    draw = lambda *s: torch.randint(  # noqa: E731
        -2, 3, s, generator=g, device="cuda").to(dtype)
    x, w, b = draw(m, k), draw(n, k), draw(n)
    assert torch.equal(fused_linear(x, w, b), (
        x.double() @ w.double().t() + b.double()).to(dtype))


@on_devices
@on_types
@pytest.mark.parametrize("residual", [False, True])
def test_linear_relu_of_nan(device, dtype, residual):
    """relu leaves NaN as it is, and its gradient too: only what is zero or
    below takes it away."""
    x = torch.tensor([[math.nan, 1], [2, 1], [-3, 1], [-1, 1], [-math.inf, 1]],
                     dtype=dtype, device=device, requires_grad=True)
    w = torch.ones(3, 2, dtype=dtype, device=device, requires_grad=True)
    b = torch.zeros(3, dtype=dtype, device=device, requires_grad=True)
    res = torch.ones(5, 3, dtype=dtype, device=device) if residual else None
    y = fused_linear(x, w, b, "relu", res)
    more = 1.0 if residual else 0.0
    assert y[0].isnan().all()
    assert torch.equal(y[1:, 0].cpu(),
                       torch.tensor([3.0, 0, 0, 0], dtype=dtype) + more)
    y.backward(torch.ones_like(y))
    live = torch.tensor([1.0, 1, 0, 0, 0], dtype=dtype)
    assert torch.equal(x.grad.cpu(), 3 * live[:, None].expand(5, 2))
    assert torch.equal(b.grad.cpu(), torch.full((3,), 2.0, dtype=dtype))
    assert w.grad[:, 0].isnan().all()
    assert torch.equal(w.grad[:, 1].cpu(), torch.full((3,), 2.0, dtype=dtype))


@on_devices
@on_types
@pytest.mark.parametrize("eps", [1e-5, 0.0])
@pytest.mark.parametrize("cols", [24, 40000])
def test_norm_only_the_sum_used(device, dtype, eps, cols):
    """Where only s = x + residual goes on, its gradient is both inputs', also
    in rows that have no norm: an infinity, a NaN, no spread and no eps."""
    g = rng(cols, 77)
    x = normal(g, 4, cols, dtype=dtype, device=device)
    x[0, 1], x[1, 2] = math.inf, math.nan
    x[2] = 3.0
    res = torch.zeros_like(x).requires_grad_(True)
    x.requires_grad_(True)
    w, b = (torch.ones(cols, dtype=dtype, device=device, requires_grad=True)
            for _ in range(2))
    ds = normal(g, 4, cols, dtype=dtype, device=device)
    _, s = fused_layer_norm(x, w, b, eps, res)
    dx, dres, dw, db = torch.autograd.grad(s, [x, res, w, b], ds,
                                           allow_unused=True)
    assert torch.equal(dx, ds) and torch.equal(dres, ds)
    for v in (dw, db):
        assert v is None or torch.equal(v, torch.zeros_like(w))


@on_devices
@pytest.mark.parametrize("m", [8, 70, 200])
def test_linear_infinity_times_a_tiny_float(device, m):
    """An infinity times any float but zero is an infinity, however small that
    is, forward and in both gradients."""
    tiny = [2.0 ** -149, 2.0 ** -140, -2.0 ** -134, 2.0 ** -133, 2.0 ** -126,
            -1e-37, 1e-30, 1.0, 0.0]
    n = len(tiny)
    small = torch.tensor(tiny, device=device)
    # (the row that holds the infinity, in each operand)
    x = torch.zeros(m, 8, device=device)
    w = torch.zeros(n, 8, device=device)
    x[1, 3] = math.inf
    w[:, 3] = small
    want = torch.where(small == 0, math.nan, small * math.inf)
    same = lambda a, b: torch.equal(  # noqa: E731
        a.nan_to_num(5, 6, 7), b.nan_to_num(5, 6, 7))
    assert same(fused_linear(x, w)[1], want)
    x[1, 3], w[:, 3] = 0, 0
    x[:n, 3] = small[:m]
    w[2, 3] = -math.inf
    got = fused_linear(x, w)[:, 2]
    assert same(got[:n], -want[:m]) and got[n:].isnan().all()
    # dx = dy W, dW = dy^T x
    for big, little in (("dy", "w"), ("w", "dy"), ("dy", "x"), ("x", "dy")):
        v = {"x": torch.zeros(m, 8, device=device),
             "w": torch.zeros(n, 8, device=device),
             "dy": torch.zeros(m, n, device=device)}
        into = "x" if "w" in (big, little) else "w"
        if into == "x":   # summed over n
            (v["dy"][1, :1] if big == "dy" else v["w"][:1, 2]).fill_(math.inf)
            (v["dy"][1, :1] if little == "dy" else v["w"][:1, 2]).fill_(
                tiny[0])
        else:             # summed over m
            (v["dy"][:1, 1] if big == "dy" else v["x"][:1, 2]).fill_(math.inf)
            (v["dy"][:1, 1] if little == "dy" else v["x"][:1, 2]).fill_(
                tiny[0])
        leaf = v[into].requires_grad_(True)
        a, = torch.autograd.grad(fused_linear(v["x"], v["w"]), leaf, v["dy"])
        assert a[1, 2] == math.inf


@on_devices
@pytest.mark.parametrize("m", [1, 8, 70, 200])
@pytest.mark.parametrize("scale", [1e-30, 1e-34, 1e-36, 1e-37, 1e-40, 1e30])
def test_linear_small_and_large_gradients(device, m, scale):
    """Forward and both gradients with one operand of this size: beside the
    sum's rounding each operand may be off by 2^-133, where bf16 ends."""
    g = rng(m, 33)
    k, n = 64, 40
    tiny = 2.0 ** -133
    draw = lambda *s, scale=1.0: normal(  # noqa: E731
        g, *s, dtype=torch.float64, device="cpu", scale=scale).float()

    def bound(a, b, want):  # of a @ b.t()
        terms = a.shape[1]
        return (terms + 64) * U * (a.abs() @ b.abs().t()) + tiny * (
            a.abs().sum(-1)[:, None] + b.abs().sum(-1)) \
            + terms * TINY[torch.float32] + stored(want, torch.float32)

    def check(got, a, b, what):
        a, b = a.double(), b.double()
        want = a @ b.t()
        within(got, want, bound(a, b, want), what)

    x, w = draw(m, k, scale=scale), draw(n, k)
    check(fused_linear(x.to(device), w.to(device)), x, w, "y")
    x, dy = draw(m, k), draw(m, n, scale=scale)
    leaves = [v.to(device).requires_grad_(True) for v in (x, w)]
    dx, dw = torch.autograd.grad(fused_linear(*leaves), leaves, dy.to(device))
    check(dx, dy, w.t(), "dx")
    check(dw, dy.t(), x.t(), "dw")


# The largest tiles in the gradients: both in launches of their own and in one,
# and sums of one, two and three whole tiles of 64 (over n for dx, over m for dW)
# with and without a rest.  The plan is asserted, so that a size which no longer
# reaches its kernel is seen: (tile of dx, of dW, one launch).
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,plan", [
    (4096, 4096, 4096, (256, 256, False)), (4000, 3999, 3900, (256, 256, False)),
    (1030, 5000, 1100, (256, 256, True)), (2048, 4096, 2048, (256, 256, True)),
    (3900, 4090, 64, (256, 128, True)), (4096, 4096, 72, (256, 128, True)),
    (3900, 4090, 128, (256, 128, True)), (4096, 4096, 133, (256, 128, True)),
    (3900, 4090, 192, (256, 128, True)), (4096, 4090, 200, (256, 128, True)),
    (64, 3900, 4090, (128, 256, True)), (72, 4096, 4096, (128, 256, True)),
    (128, 3900, 4090, (128, 256, True)), (133, 4096, 4096, (128, 256, True)),
    (192, 3900, 4090, (128, 256, True)), (200, 4096, 4090, (128, 256, True))])
def test_gpu_linear_largest_tiles_in_gradients(dtype, m, k, n, plan):
    """Whole numbers, so that every sum is exact: equal to the formula in 64
    bits, rounded once; for both gradients, each alone, and again."""
    from cpd_amd import ops
    plan_of = ops.hip_ext().linear_plan
    p = plan_of(m, n, k, dtype, True, True)
    assert (p[2], p[4], bool(p[6])) == plan
    # alone, a gradient with the largest tiles has them too (but where those
    # paid for filling the CUs with the other one's)
    alone = (plan_of(m, n, k, dtype, True, False)[2],
             plan_of(m, n, k, dtype, False, True)[4])
    if plan != (256, 256, True):
        assert all(a == 256 for a, b in zip(alone, plan) if b == 256)
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    draw = lambda *s: torch.randint(  # noqa: E731
        -2, 3, s, generator=g, device="cuda").to(dtype)
    x, w, dy = draw(m, k), draw(n, k), draw(m, n)
    want = ((dy.double() @ w.double()).to(dtype),
            (dy.double().t().contiguous() @ x.double()).to(dtype))
    for need in ((True, True), (True, False), (False, True), (True, True)):
        a, b = (v.detach().requires_grad_(r) for v, r in zip((x, w), need))
        fused_linear(a, b).backward(dy)
        for v, r, c in zip((a, b), need, want):
            assert torch.equal(v.grad, c) if r else v.grad is None


def slope_case(dtype, m, k, n):
    """Inputs of whole numbers and a power of two, so that the activation's
    argument is exact before it is stored: z is about 1.5 in size."""
    g = rng(m, k, n, 13)
    draw = lambda *s: torch.randint(-7, 8, s, generator=g).double()  # noqa: E731
    x = draw(m, k)
    w = draw(n, k) * 2.0 ** -round(math.log2(18.7 * k ** 0.5 / 1.5))
    dy = normal(g, m, n, dtype=dtype, device="cpu")
    assert torch.equal(x.to(dtype).double(), x)
    assert torch.equal(w.to(dtype).double(), w)
    return x, w, dy.double()


def times_one_rounding(got, want, dtype):
    """The error's root mean square, in that of a single rounding."""
    rms = lambda v: v.square().mean().sqrt()  # noqa: E731
    return (rms(got.double() - want) / rms(want.to(dtype).double() - want)).item()


# dx and dW of 500 numbers or more each, up to 2^28 multiplications: sums over
# few and many rows and features
ROUNDED_ONCE = [(1, 1000, 700), (12, 896, 54), (70, 130, 61), (300, 520, 264),
                (515, 33, 700), (9, 64, 4480), (2000, 24, 40)]
on_rounded_once = pytest.mark.parametrize("m,k,n", ROUNDED_ONCE)
on_curved = pytest.mark.parametrize("act", ["gelu", "silu"])
on_16_bits = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])


# What dz in two bf16 parts adds (2^-15 of each term, of which n add up by their
# squares: at most an eighth of fp16's rounding of a sum) is under 1 % of the
# root mean square; dz rounded to the type makes it 1.41.  Halfway is 1.2.
@on_16_bits
@on_curved
@on_rounded_once
def test_rounding_twice_is_told_from_once(dtype, act, m, k, n):
    """The measure of the next test on the formula in 64 bits: what it says of
    a gradient whose dz was rounded, and of one whose dz was not."""
    x, w, dy = slope_case(dtype, m, k, n)
    dz = dy * act_oracle((x @ w.t()).to(dtype).double(), act)[1]
    for a, b in ((dz, w.t()), (dz.t(), x.t())):
        want = a @ b.t()
        twice = (a.to(dtype).double() @ b.t()).to(dtype)
        assert times_one_rounding(want.to(dtype), want, dtype) == 1
        assert times_one_rounding(twice, want, dtype) > 1.3


@pytest.mark.gpu
@on_16_bits
@on_curved
@on_rounded_once
def test_gpu_linear_gradients_off_by_one_rounding(dtype, act, m, k, n):
    """Behind gelu and silu, the slope taken at the argument as it is stored:
    dx and dW are each as near 64 bits as one rounding allows."""
    x, w, dy = slope_case(dtype, m, k, n)
    dz = dy * act_oracle((x @ w.t()).to(dtype).double(), act)[1]
    a, b = (v.to(dtype).cuda().requires_grad_(True) for v in (x, w))
    dx, dw = torch.autograd.grad(fused_linear(a, b, None, act), [a, b],
                                 dy.to(dtype).cuda())
    assert times_one_rounding(dx.cpu(), dz @ w, dtype) < 1.2
    assert times_one_rounding(dw.cpu(), dz.t() @ x, dtype) < 1.2


class WithoutMemory(torch.Tensor):
    """A tensor of a wrapper class: on the GPU by its own account, at address
    0."""

    @staticmethod
    def __new__(cls, like):
        return torch.Tensor._make_wrapper_subclass(
            cls, like.shape, dtype=like.dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError(f"{func} needs memory")


def test_refuses_inputs_without_memory():
    """Before anything is asked of a GPU."""
    from cpd_amd import ops
    try:
        ext = ops.hip_ext()
    except RuntimeError:
        pytest.skip("the HIP extension is not built")
    x = WithoutMemory(torch.zeros(4, 16))
    t = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ext.layer_norm(x, None, None, 1e-5, None),
                 lambda: ext.linear(x, x, None, 0, None),
                 lambda: ext.token_logprobs(x, t, 0, -100)):
        with pytest.raises(TypeError, match="memory"):
            call()


@pytest.mark.gpu
def test_gpu_refuses_tensors_without_memory():
    """Every operand, gradients among them, and results: tensors of a wrapper
    class, zeros known without being stored, a mode that follows shapes
    alone."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    x = torch.randn(4, 16, device="cuda")
    w = torch.randn(8, 16, device="cuda")
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    no = WithoutMemory
    zeros = torch._efficientzerotensor((4, 16), device="cuda")
    for call in (lambda: fused_layer_norm(zeros),
                 lambda: fused_layer_norm(x, no(x[0])),
                 lambda: fused_layer_norm(x, None, no(x[0])),
                 lambda: fused_layer_norm(x, residual=zeros),
                 lambda: fused_linear(x, no(w)),
                 lambda: fused_linear(x, w, no(w[:, 0])),
                 lambda: fused_linear(x, w, None, "relu", no(x[:, :8])),
                 lambda: token_logprobs(zeros, t),
                 lambda: token_logprobs(x, no(t))):
        with pytest.raises(TypeError, match="memory"):
            call()
    for f in (fused_layer_norm, lambda v: fused_linear(v, w, None, "gelu"),
              lambda v: token_logprobs(v, t).logprobs,
              lambda v: token_logprobs(v, t).entropy):
        y = f(x.detach().requires_grad_(True))
        dy = torch._efficientzerotensor(y.shape, device="cuda")
        with pytest.raises(TypeError, match="memory"):
            y.backward(dy)
    odd = torch.randn(70, 33, device="cuda").bfloat16()
    with FakeTensorMode(allow_non_fake_inputs=True):
        for call in (lambda: fused_layer_norm(x), lambda: fused_linear(x, w),
                     lambda: fused_linear(odd, odd),
                     lambda: token_logprobs(x, t, 2)):
            with pytest.raises(TypeError, match="memory"):
                call()
    torch.cuda.synchronize()
    assert torch.isfinite(fused_layer_norm(x)).all()


@on_devices
def test_negative_views(device):
    """A view that stands for the negative of its memory, as .imag of a
    conjugate does, is read as what it stands for: every operand and every
    incoming gradient."""
    neg = lambda v: torch._neg_view((-v).contiguous())  # noqa: E731
    g = rng(91)
    draw = lambda *s: normal(  # noqa: E731
        g, *s, dtype=torch.float32, device=device)
    x, res, w, b = draw(6, 16), draw(6, 16), draw(16, 16), draw(16)
    dy, dz, t = draw(6, 16), draw(6), torch.arange(6, device=device)
    c = torch.randn(6, 1, generator=g, dtype=torch.complex64).to(
        device).conj().imag
    assert c.is_neg() and neg(x).is_neg() and torch.equal(neg(x), x)
    one = torch.ones(1, 1, device=device)
    assert torch.equal(fused_linear(c, one), c.clone())

    def norm(x, res, w, b, dy, dz):
        y, s = fused_layer_norm(x, w[0], b, residual=res)
        return y, s, *torch.autograd.grad([y, s], [x, res, w, b], [dy, dy])

    def linear(x, res, w, b, dy, dz):
        y = fused_linear(x, w, b, "gelu", res)
        return y, *torch.autograd.grad(y, [x, w, b, res], dy)

    def logprobs(x, res, w, b, dy, dz):
        out = token_logprobs(x, t, 3)
        return *out, *torch.autograd.grad([out.logprobs, out.entropy], x,
                                          [dz, dz])

    for f in (norm, linear, logprobs):
        plain, negated = ([v.detach().requires_grad_(True) for v in ops] +
                          list(grads) for ops, grads in (
            ((x, res, w, b), (dy, dz)),
            (map(neg, (x, res, w, b)), (neg(dy), neg(dz)))))
        assert all(v.is_neg() for v in negated)
        assert all(torch.equal(p, q)
                   for p, q in zip(f(*negated), f(*plain)))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(64, 131072), (600, 50021), (40, 4096),
                                        (900, 1000)])
def test_gpu_logprobs_probabilities_as_exact_as_floats_are(rows, vocab):
    """The gradient of a log probability is minus the others' probabilities,
    e^(x - max) over its sum.  Each is off by the rounding of x - max (|x - max|
    between 8 and 16: up to 8 U, 4.6 U root mean square; the more so the less
    often), of e^, of its product and of the sum (1, 1 and at most 3 U).  Taken
    from the rounded log probability it would be 10 to 20 U, so 9 U are
    allowed."""
    g = rng(rows, vocab, 19)
    x = torch.randn(rows, vocab, generator=g) * 3
    t = torch.zeros(rows, dtype=torch.int64)
    leaf = x.cuda().requires_grad_(True)
    out = token_logprobs(leaf, t.cuda())
    dx, = torch.autograd.grad(out.logprobs.sum(), leaf)
    p = torch.softmax(leaf.detach().double(), -1)[:, 1:]
    off = (-dx[:, 1:].double() - p) / p
    assert off.square().mean().sqrt() < 9 * U


@pytest.mark.gpu
@on_types
@pytest.mark.parametrize("rows", [3, 520])
@pytest.mark.parametrize("rest", [-11.5, -11.9375, -12.0, -12.6875])
def test_gpu_logprobs_many_small_terms(dtype, rows, rest):
    """One entry far above 131071 equal ones, each of which is some tenths of a
    step of the sum that it is added to: what one addition loses all lose, so it
    has to be kept.  Off by: a step's 32 additions, 10 joins, e^'s own |rest| + 4;
    the logarithm and its differences 4: 64 U cover S, for the entropy |rest|
    times that beside it."""
    vocab = 131072
    x = torch.full((rows, vocab), rest, dtype=dtype, device="cuda")
    t = torch.arange(rows, device="cuda") * 97 % vocab
    x[torch.arange(rows, device="cuda"), t] = 0.0
    out = token_logprobs(x, t, 2)
    small = (vocab - 1) * math.exp(rest)
    logs = math.log1p(small)
    ent = logs - small * rest / (1 + small)
    assert (out.logprobs.double() + logs).abs().max() < 64 * U
    assert (out.entropy.double() - ent).abs().max() < 64 * U * (1 - rest)
    assert torch.equal(out.top_ids[:, 0], t)


TILES, ROWS, NARROW_B, NARROW_A, BRIEF = range(5)


# Floats with few features in or out and few rows: up to 16, up to 32 and one
# more; long sums in one slice and in several; the long operand read 32 or 128
# rows at a time; rows of it a multiple of 4 KB apart or not; sizes that end inside
# a vector, a tile and a strip of 64.  (way of y, of dx, of dW)
FEW_SHAPES = [
    (70, 300, 9, (NARROW_B, BRIEF, NARROW_A)),
    (200, 9, 301, (BRIEF, NARROW_B, NARROW_B)),
    (131, 32, 400, (BRIEF, NARROW_B, NARROW_B)),
    (131, 33, 400, (TILES, TILES, TILES)),
    (300, 1025, 31, (NARROW_B, BRIEF, NARROW_A)),
    (300, 1030, 33, (TILES, TILES, TILES)),
    (70, 9001, 20, (NARROW_B, BRIEF, NARROW_A)),
    (70, 4096, 16, (NARROW_B, BRIEF, NARROW_A)),
    (5003, 200, 7, (NARROW_B, BRIEF, NARROW_A)),
    (5003, 18, 201, (BRIEF, NARROW_B, NARROW_B)),
    (700, 4700, 9, (NARROW_B, BRIEF, NARROW_A)),
    (700, 25, 4703, (BRIEF, NARROW_B, NARROW_B)),
    (3000, 4610, 17, (NARROW_B, BRIEF, NARROW_A)),
    (20, 300, 5000, (ROWS, NARROW_A, BRIEF)),
    (3, 4900, 1003, (NARROW_A, NARROW_A, BRIEF)),
    (17, 4096, 1100, (NARROW_A, NARROW_A, BRIEF)),
    (32, 5000, 900, (NARROW_A, NARROW_A, BRIEF)),
    (1, 150, 1, (ROWS, BRIEF, BRIEF)),
    (129, 1, 1, (BRIEF, BRIEF, NARROW_B)),
    (9, 20, 30, (ROWS, TILES, TILES)),
    (128, 128, 20, (NARROW_B, TILES, TILES)),
    (129, 20, 30, (BRIEF, BRIEF, NARROW_B))]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,ways", FEW_SHAPES)
@pytest.mark.parametrize("act,residual", [(None, True), ("silu", False)])
def test_gpu_linear_few(m, k, n, ways, act, residual):
    from cpd_amd import ops
    plan = ops.hip_ext().linear_plan(m, n, k, torch.float32, True, True)
    assert tuple(plan[7:]) == ways
    run_linear("cuda", torch.float32, m, k, n, act, residual)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n,ways", FEW_SHAPES)
def test_gpu_linear_few_whole_numbers(m, k, n, ways):
    """Every sum exact: equal to the formula in 64 bits, from strided and
    misaligned operands too, and the gradients alone as together."""
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    draw = lambda *s: torch.randint(  # noqa: E731
        -2, 3, s, generator=g, device="cuda").float()
    b, res = draw(n) + 0.5, draw(m, n)
    for pad, off in ((0, 0), (5, 3)):
        x, w, dy = (draw(r, c + pad)[:, off:c + off]
                    for r, c in ((m, k), (n, k), (m, n)))
        x64, w64, dy64 = x.double(), w.double(), dy.double()
        z = x64 @ w64.t() + b.double()
        assert torch.equal(fused_linear(x, w, b, "relu", res),
                           (z.clamp_min(0) + res.double()).float())
        want = ((dy64 @ w64).float(), (dy64.t() @ x64).float(),
                dy64.sum(0).float())
        for need in ((True, True), (True, False), (False, True)):
            leaves = [v.detach().requires_grad_(r)
                      for v, r in zip((x, w, b), need + (need[0],))]
            fused_linear(*leaves).backward(dy)
            for v, c in zip(leaves, want):
                assert v.grad is None or torch.equal(v.grad, c)


@pytest.mark.gpu
def test_gpu_linear_few_far_offsets():
    """Operands and results whose offsets pass 2^31 elements, and 2^25 rows."""
    for m, k, n in (((1 << 19) + 5, 4200, 8), ((1 << 19) + 5, 8, 4200),
                    ((1 << 25) + 5, 4, 3)):
        x, dy = (torch.zeros(m, c, device="cuda") for c in (k, n))
        x[-3:] = torch.randint(-2, 3, (3, k), device="cuda").float()
        dy[-3:] = torch.randint(-2, 3, (3, n), device="cuda").float()
        w = torch.randint(-2, 3, (n, k), device="cuda").float()
        x.requires_grad_(True)
        w.requires_grad_(True)
        y = fused_linear(x, w)
        last, w64 = x.detach()[-3:].double(), w.detach().double()
        assert torch.equal(y[-3:], (last @ w64.t()).float())
        assert not y[:-3].any()
        dx, dw = torch.autograd.grad(y, [x, w], dy)
        assert torch.equal(dx[-3:], (dy[-3:].double() @ w64).float())
        assert not dx[:-3].any()
        assert torch.equal(dw, (dy[-3:].double().t().contiguous()
                                @ last).float())
        del x, dy, y, dx
    # more rows than a launch of few features could take
    x = torch.zeros((1 << 27) + 37, 33, device="cuda")
    x[-3:] = 1
    y = fused_linear(x, torch.ones(1, 33, device="cuda"))
    assert (y[-3:] == 33).all() and not y[:-3].any()


@pytest.mark.gpu
def test_gpu_linear_few_not_finite():
    """Infinities and NaN reach their own rows and columns and no others, and
    what lies behind an operand's end reaches none."""
    for m, k, n in ((200, 300, 9), (300, 20, 200), (5, 5000, 900)):
        x = torch.ones(m, k, device="cuda")
        w = torch.ones(n, k + 4, device="cuda")
        w[:, k:] = math.nan
        w = w[:, :k]
        x[1, k - 1], x[m - 1, 0], w[2, 5] = math.inf, math.nan, -math.inf
        y = fused_linear(x, w)
        want = torch.full((m, n), float(k), device="cuda")
        want[1] = math.inf
        want[:, 2] = -math.inf
        want[1, 2] = math.nan
        want[m - 1] = math.nan
        assert torch.equal(y.nan_to_num(1, 2, 3), want.nan_to_num(1, 2, 3))
        a, b = (torch.ones(*s, device="cuda", requires_grad=True)
                for s in ((m, k), (n, k)))
        dy = torch.ones(m, n, device="cuda")
        dy[3, n - 1] = math.inf
        dx, dw = torch.autograd.grad(fused_linear(a, b), [a, b], dy)
        assert dx.isinf().any(1).nonzero().flatten().tolist() == [3]
        assert dw.isinf().any(1).nonzero().flatten().tolist() == [n - 1]
        assert dx[3].isinf().all() and dw[n - 1].isinf().all()
        assert not dx.isnan().any() and not dw.isnan().any()


def test_cpu_second_derivatives_and_tangents():
    """What the docstrings say of the CPU path: second derivatives work, and
    tangents but beside a norm's residual."""
    from torch.autograd import forward_ad
    g = rng(51)
    x, w = (torch.randn(4, 16, generator=g) for _ in range(2))
    t = torch.arange(4)
    calls = [lambda v: fused_layer_norm(v, w[0]),
             lambda v: fused_linear(v, w, None, "gelu"),
             lambda v: token_logprobs(v, t).logprobs,
             lambda v: token_logprobs(v, t).entropy]
    for f in calls + [lambda v: fused_layer_norm(v, w[0], residual=w)[0]]:
        leaf = x.clone().requires_grad_(True)
        first, = torch.autograd.grad(f(leaf).square().sum(), leaf,
                                     create_graph=True)
        second, = torch.autograd.grad(first.square().sum(), leaf)
        assert second.isfinite().all() and second.abs().sum() > 0
    v = torch.randn(4, 16, generator=g)
    for f in calls:
        leaf = x.clone().requires_grad_(True)
        want = (torch.autograd.grad(f(leaf).sum(), leaf)[0] * v).sum()
        with forward_ad.dual_level():
            got = forward_ad.unpack_dual(f(forward_ad.make_dual(x, v)))
            torch.testing.assert_close(got.tangent.sum(), want, rtol=1e-3,
                                       atol=1e-5)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, v)
        with pytest.raises(RuntimeError):
            fused_layer_norm(dual, w[0], residual=w)


@on_devices
@pytest.mark.parametrize("vocab", [11, 5000])
def test_logprobs_target_outside(device, vocab):
    """A target outside the row: NaN where the log probability is used, and
    the entropy and its own gradient as with any target."""
    x, _ = make_logits(rng(vocab, 61), torch.float32, device, 3, vocab)
    bad = torch.tensor([vocab, -1, 2 ** 40]).to(device)
    good = torch.zeros(3, dtype=torch.int64, device=device)
    got = []
    for t in (bad, good):
        leaf = x.to(device).requires_grad_(True)
        out = token_logprobs(leaf, t)
        ent, = torch.autograd.grad(out.entropy.sum(), leaf, retain_graph=True)
        lp, = torch.autograd.grad(out.logprobs.sum(), leaf, retain_graph=True)
        both, = torch.autograd.grad((out.entropy + 0 * out.logprobs).sum(),
                                    leaf)
        got.append((out, ent, lp, both))
    (a, ent_a, lp_a, both_a), (b, ent_b, lp_b, _) = got
    assert a.logprobs.isnan().all() and b.logprobs.isfinite().all()
    assert torch.equal(a.entropy, b.entropy) and torch.equal(ent_a, ent_b)
    assert lp_a.isnan().all() and both_a.isnan().all()
    assert lp_b.isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(5003, 200, 7), (70, 9001, 20),
                                   (3, 4900, 1003), (700, 25, 4703)])
def test_gpu_linear_few_captured(m, k, n):
    """Forward and backward of few features, slices and their joining among
    them, in two graphs that are replayed in turn, with eager work between the
    replays."""
    g = torch.Generator(device="cuda").manual_seed(m)
    draw = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    inputs = [[draw(m, k), draw(n, k), draw(n), draw(m, n)] for _ in range(3)]

    def step(x, w, b, dy):
        leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
        y = fused_linear(*leaves, "gelu")
        return [v.detach() for v in (y, *torch.autograd.grad(y, leaves, dy))]

    want = [step(*v) for v in inputs]
    graphs = []
    for _ in range(2):
        static = [v.clone() for v in inputs[0]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((graph, static, out))
    for i in range(6):
        graph, static, out = graphs[i % 2]
        for a, b in zip(static, inputs[i % 3]):
            a.copy_(b)
        graph.replay()
        step(*inputs[(i + 1) % 3])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[i % 3]))
