"""The rendering network's operators (group normalisation with an activation, the gate of a gated convolution, both together)
against plain implementations in 64 bits, through the libTorch operators and through the C ABI.

Tolerances, element by element from the 64-bit reference's own intermediate values, derived before the first run. With t the image
type, every output is computed in 32 bits and rounded once: h |v|, h = finfo(t).eps / 2, and half the spacing of the numbers below
the smallest normal one. The 32-bit arithmetic in front of the rounding:
  e_u     relative error of a gated u: two exponentials (2 ulp + 1.2 |v| ulp each, |v| < 10: below 2^-20), two quotients of 2 ulp and
          products: 2^-18. For a plain u = x: 0.
  e_uhat  absolute error of uhat = (u - mean) rstd: R (e_u |u|) from u, R e_u rms(u) (1 + |uhat|) as the mean and the variance take it
          up, 2^-22 R |mean| from the rounded mean, 2^-20 (1 + |uhat|) from the sums (chains of some tens of additions) and rstd.
  e_z     |w| e_uhat + 2^-22 (|b| + |z|); y: times the activation's slope (at most 1.1), and 2^-18 |y| for the activation.
  e_dz    |dy| (e_z + 2^-18) (the activations' second derivatives are at most 1), without an activation behind the norm 0.
  dx      R (|w| e_dz + its group mean + |uhat| mean(|w| (e_dz |uhat| + |dz| e_uhat)) + e_uhat mean |w dz uhat|), and
          2^-19 + R e_u rms(u) of R (|w dz| + |c1| + |uhat c2|); the gate's factors are exact to 2^-18 of du times their bound.
  db, dw  the sums of e_dz and of e_dz |uhat| + |dz| e_uhat, and 2^-21 of the sums of the terms' magnitudes for the additions."""
import ctypes as C
import itertools

import pytest
import torch

from adop_b200 import build, capi
from tests.test_raster_gpu import eight_sm_stream  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
ACTS = ["none", "relu", "elu", "silu"]
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def op(cuda_lib):
    torch.ops.load_library(build.TORCH_OP_LIB)
    return torch.ops.adop


def half_step(t):
    return torch.finfo(t).eps / 2


# ---- the operators in 64 bits ---------------------------------------------------------------------------------------------
def act64(v, kind):
    if kind == "relu":
        return v.clamp(min=0)
    if kind == "elu":
        return torch.where(v > 0, v, torch.expm1(v.clamp(max=0)))
    return v / (1 + torch.exp(-v)) if kind == "silu" else v


def slope64(v, kind):
    if kind == "relu":
        return (v > 0).double()
    if kind == "elu":
        return torch.where(v > 0, torch.ones_like(v), torch.exp(v.clamp(max=0)))
    if kind == "silu":
        s = 1 / (1 + torch.exp(-v))
        return s + v * s * (1 - s)
    return torch.ones_like(v)


class Reference:
    """op: norm, gate or gated_norm. Results and, beside each, its bound."""

    def __init__(self, kind, x, groups, weight, bias, eps, act, dy=None):
        t = x.dtype
        h = half_step(t)
        x = x.detach().double()
        B, C2, H, W = x.shape
        Cc = C2 if kind == "norm" else C2 // 2
        view = lambda p: p.detach().double().view(1, -1, 1, 1)
        f, g = (x, None) if kind == "norm" else (x[:, :Cc], x[:, Cc:])
        if g is None:
            u = f
        else:
            fa, s = act64(f, act), 1 / (1 + torch.exp(-g))
            u = fa * s
        # half the spacing of the numbers below the type's smallest normal one
        tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
        if kind == "gate":
            self.y, self.y_tol = u, (h + 2.0 ** -18) * u.abs() + tiny
        else:
            one = torch.ones(1, Cc, 1, 1, dtype=torch.float64, device=x.device)
            w = view(weight) if weight is not None else one
            b = view(bias) if bias is not None else 0 * one
            ug = u.reshape(B, groups, -1)
            mean, var = ug.mean(2), ug.var(2, unbiased=False)
            rstd = 1 / torch.sqrt(var + eps)
            self.mean, self.rstd = mean, rstd
            wide = lambda v: v.repeat_interleave(Cc // groups, 1).view(B, Cc, 1, 1)
            mean_of = lambda v: wide(v.reshape(B, groups, -1).mean(2))
            M, R = wide(mean), wide(rstd)
            uhat = (u - M) * R
            z = uhat * w + b
            e_u = 0.0 if g is None else 2.0 ** -18
            common = R * e_u * mean_of(u * u).sqrt()  # relative error of mean (of the spread) and rstd
            e_uhat = R * e_u * u.abs() + common * (1 + uhat.abs()) + 2.0 ** -22 * R * M.abs() + 2.0 ** -20 * (1 + uhat.abs())
            e_z = w.abs() * e_uhat + 2.0 ** -22 * (b.abs() + z.abs())
            self.y = act64(z, act) if kind == "norm" else z
            self.y_tol = (h + 2.0 ** -18) * self.y.abs() + 1.1 * e_z + tiny
        if dy is None:
            return
        dy = dy.detach().double()
        du, du_tol = dy, 0 * dy
        if kind != "gate":
            dz = dy * slope64(z, act) if kind == "norm" else dy
            e_dz = dy.abs() * (e_z + 2.0 ** -18) if kind == "norm" and act != "none" else 0 * dy
            c1, c2 = mean_of(w * dz), mean_of(w * dz * uhat)
            du = R * (w * dz - c1 - uhat * c2)
            e_dw = e_dz * uhat.abs() + dz.abs() * e_uhat
            terms = w.abs() * e_dz + mean_of(w.abs() * e_dz) + uhat.abs() * mean_of(w.abs() * e_dw) + e_uhat * mean_of((w * dz * uhat).abs())
            du_tol = R * (terms + (2.0 ** -19 + common) * ((w * dz).abs() + c1.abs() + (uhat * c2).abs() + 2.0 ** -2 * (mean_of((w * dz).abs()) + uhat.abs() * mean_of((w * dz * uhat).abs()))))
            total = lambda v: v.sum((0, 2, 3))
            pt = max([half_step(p.dtype) for p in (weight, bias) if p is not None], default=0.0)
            self.db, self.dw = total(dz), total(dz * uhat)
            small = max([torch.finfo(p.dtype).smallest_normal * half_step(p.dtype) for p in (weight, bias) if p is not None], default=0.0)
            self.db_tol = pt * self.db.abs() + total(e_dz) + 2.0 ** -21 * total(dz.abs()) + small
            self.dw_tol = pt * self.dw.abs() + total(e_dw) + 2.0 ** -21 * total((dz * uhat).abs()) + small
        if g is None:
            self.dx, self.dx_tol = du, h * du.abs() + du_tol + tiny
        else:
            fs = slope64(f, act)
            to_f, to_g = fs * s, fa * s * (1 - s)
            self.dx = torch.cat([du * to_f, du * to_g], 1)
            error = lambda to, bound: h * (du * to).abs() + 2.0 ** -18 * du.abs() * bound + 1.01 * du_tol * to.abs() + tiny
            self.dx_tol = torch.cat([error(to_f, 1.1 * s), error(to_g, fa.abs() * s)], 1)


def check(got, want, tol, what):
    got = got.detach().double()
    assert got.shape == want.shape, what
    off = (got - want).abs()
    worst = (off / tol).max().item() if off.numel() else 0.0
    assert bool((off <= tol).all()), f"{what}: {worst:.3g} times its bound"


def image(shape, dtype, gen, order="channels_last", mean=0.5, spread=1.0):
    B, Cc, H, W = shape
    wide = {"channels_last": Cc, "planar": Cc, "slice": Cc + 8, "odd_slice": Cc + 3}[order]
    v = torch.randn((B, H, W, wide), device=DEV, generator=gen)
    v = v * (0.5 + torch.rand(wide, device=DEV, generator=gen)) * spread + mean * torch.randn(wide, device=DEV, generator=gen)
    v = v.to(dtype).permute(0, 3, 1, 2)
    if order == "planar":
        return v.contiguous()
    return v[:, {"slice": 8, "odd_slice": 3}.get(order, 0):][:, :Cc]


def call(op, kind, x, groups, w, b, eps, act):
    if kind == "norm":
        return op.group_norm(x, groups, w, b, eps, act)
    if kind == "gate":
        return op.gated_activation(x, act)
    return op.gated_group_norm(x, groups, w, b, eps, act)


def run_case(op, kind, shape, groups, dtype, act, wdtype=torch.float32, affine=True, order="channels_last", eps=1e-5, seed=0, mean=0.5):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    B, Cc, H, W = shape
    x = image((B, Cc if kind == "norm" else 2 * Cc, H, W), dtype, gen, order, mean).detach().requires_grad_(True)
    w = b = None
    if affine and kind != "gate":
        w = (1 + 0.3 * torch.randn(Cc, device=DEV, generator=gen)).to(wdtype).requires_grad_(True)
        b = (0.3 * torch.randn(Cc, device=DEV, generator=gen)).to(wdtype).requires_grad_(True)
    dy = image(shape, dtype, gen, "planar" if order == "planar" else "channels_last", 0.1)
    y = call(op, kind, x, groups, w, b, eps, act)
    assert y.dtype == dtype and y.shape == torch.Size(shape) and y.is_contiguous(memory_format=torch.channels_last)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    ref = Reference(kind, x, groups, w, b, eps, act, dy)
    check(y, ref.y, ref.y_tol, "y")
    if act == "relu" and kind == "norm":
        # the derivative's corner: where the 64-bit z is within its bound of zero either side is right
        near = (Reference(kind, x, groups, w, b, eps, "none").y.abs() <= 2.0 ** -16)
        ref.dx_tol = ref.dx_tol + near * (ref.rstd.max() * (w.abs().max().double() if w is not None else 1) * dy.abs().max().double())
    check(grads[0], ref.dx, ref.dx_tol, "dx")
    if w is not None:
        check(grads[1], ref.dw, ref.dw_tol, "dw")
        check(grads[2], ref.db, ref.db_tol, "db")
    # without gradients the same bits
    with torch.no_grad():
        assert torch.equal(call(op, kind, x, groups, w, b, eps, act), y)


SHAPES = [((1, 4, 1, 1), 2), ((2, 8, 3, 5), 1), ((3, 20, 7, 11), 5), ((1, 64, 8, 15), 8), ((2, 16, 33, 40), 4), ((5, 6, 9, 9), 3), ((2, 3, 12, 12), 1),
          ((2, 96, 17, 10), 32), ((1, 12, 64, 64), 12), ((2, 512, 6, 7), 32), ((1, 1, 31, 17), 1), ((3, 24, 31, 33), 4)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
@pytest.mark.parametrize("shape,groups", SHAPES, ids=str)
def test_shapes(op, shape, groups, kind, dtype):
    for k, act in enumerate(ACTS):
        run_case(op, kind, shape, groups, dtype, act, wdtype=[torch.float32, dtype][k % 2], affine=k != 3, seed=k)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
@pytest.mark.parametrize("order", ["planar", "slice", "odd_slice"])
def test_orders(op, order, kind, dtype):
    for shape, groups in (((2, 16, 19, 23), 4), ((3, 5, 6, 7), 5)):
        run_case(op, kind, shape, groups, dtype, "elu", order=order, seed=3)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["norm", "gated_norm"])
@pytest.mark.parametrize("shape,groups", [((4, 32, 128, 96), 8), ((1, 16, 270, 480), 4), ((2, 4, 300, 301), 2), ((40, 64, 16, 16), 8), ((1, 256, 64, 64), 32),
                                          ((700, 8, 5, 5), 2)], ids=str)
def test_larger_images(op, shape, groups, kind, dtype):
    run_case(op, kind, shape, groups, dtype, "silu", seed=5)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["norm", "gated_norm"])
@pytest.mark.parametrize("channels,groups", [(4096, 1), (4096, 4096), (2560, 32), (1030, 5), (1029, 3), (1100, 100)], ids=str)
def test_many_channels(op, channels, groups, kind, dtype):
    run_case(op, kind, (2, channels, 3, 3), groups, dtype, "elu", seed=7)


# ---- values at the edges --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape,groups", [((2, 16, 12, 20), 4), ((1, 16, 300, 400), 4)], ids=str)
def test_a_constant_image_is_its_bias(op, shape, groups, dtype):
    """Variance 0: uhat is 0 up to the rounding of mean rstd (2^-22 rstd |mean| as above, rstd = 1 / sqrt(eps))."""
    x = torch.full(shape, 1.5, device=DEV, dtype=dtype).contiguous(memory_format=torch.channels_last)
    b = torch.linspace(-1, 1, shape[1], device=DEV)
    y = op.group_norm(x, groups, None, b, 1e-5, "none").double()
    want = b.double().view(1, -1, 1, 1).expand(shape)
    assert bool(((y - want).abs() <= half_step(dtype) * want.abs() + 2.0 ** -22 * 1.5 * 1e-5 ** -0.5).all())


def test_groups_of_one_value(op):
    x = torch.randn((3, 8, 1, 1), device=DEV).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    y = op.group_norm(x, 8)
    gx, = torch.autograd.grad(y, [x], torch.randn_like(y))
    bound = 2.0 ** -22 * x.detach().abs().double() * 1e-5 ** -0.5
    assert bool((y.double().abs() <= bound).all())
    assert bool((gx.abs() <= 1e-2).all())  # rstd (dy - dy - uhat^2 dy): uhat is off by 2^-22 |mean| rstd


@pytest.mark.parametrize("offset", [100.0, -3000.0])
def test_far_from_zero(op, offset):
    """Means far beyond the spread, and one first pixel that is far from the others: the sums are about values of the data."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1)
    for shape in ((2, 8, 16, 24), (1, 8, 256, 260)):
        x = (offset + torch.randn(shape, device=DEV, generator=gen)).contiguous(memory_format=torch.channels_last)
        for first in (None, 0.0):
            if first is not None:
                x[:, :, 0, 0] = first
            ref = Reference("norm", x, 2, None, None, 1e-5, "none")
            check(op.group_norm(x, 2), ref.y, ref.y_tol, f"first {first}")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["norm", "gated_norm"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), "lowest"], ids=str)
@pytest.mark.parametrize("shape", [(2, 16, 9, 13), (2, 16, 256, 200)], ids=str)
def test_a_bad_value_stays_in_its_group(op, shape, value, kind, dtype):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(2)
    x = image((2, 16 if kind == "norm" else 32, *shape[2:]), dtype, gen)
    good = call(op, kind, x, 4, None, None, 1e-5, "elu")
    x[1, 6, 4, 5] = torch.finfo(dtype).max if value == "lowest" else value  # channel 6: group 1
    bad = call(op, kind, x, 4, None, None, 1e-5, "elu")
    assert torch.equal(good[0], bad[0])
    assert torch.equal(good[1, :4], bad[1, :4]) and torch.equal(good[1, 8:], bad[1, 8:])
    if value != "lowest":
        assert bool(torch.isnan(bad[1, 4:8]).any())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gates_at_the_ends(op, dtype):
    big = 60000.0
    f = torch.tensor([1.0, -2.0, big, -big, 0.0, -1e-4, 3.0, -0.5], device=DEV)
    g = torch.tensor([float("inf"), float("-inf"), big, -big, 90.0, -90.0, 0.0, float("nan")], device=DEV)
    ff, gg = torch.meshgrid(f, g, indexing="ij")
    x = torch.stack([ff, gg])[None].to(dtype).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    for act in ACTS:
        y = op.gated_activation(x, act)
        xd = x.detach().double().requires_grad_(True)
        fs, gs = xd[:, :1], xd[:, 1:]
        u = {"none": fs, "relu": fs.clamp(min=0), "elu": torch.nn.functional.elu(fs), "silu": fs / (1 + torch.exp(-fs))}[act]
        s = torch.sigmoid(gs)
        want = u * s
        assert torch.equal(torch.isnan(y), torch.isnan(want)), act
        ok = torch.isnan(want) | torch.isinf(y) | ((y.double() - want).abs() <= (half_step(dtype) + 2.0 ** -17) * want.abs() + 1e-32 + torch.finfo(dtype).smallest_normal)  # sigmoids below 2^-126 are 0
        assert bool(ok.all()), act
        gx, = torch.autograd.grad(y, [x], torch.ones_like(y))
        wx, = torch.autograd.grad(want, [xd], torch.ones_like(want))
        plain = torch.isfinite(wx) & torch.isfinite(xd) & (xd.abs() < 100)
        plain[:, :1] &= torch.isfinite(gs) & (gs.abs() < 100)
        plain[:, 1:] &= (fs.abs() < 100) & torch.isfinite(gs)
        plain[:, :1] &= fs.abs() > 0  # relu's corner
        near = (gx.double() - wx).abs() <= (half_step(dtype) + 2.0 ** -16) * wx.abs() + 2.0 ** -16 * torch.cat([s, u.abs() * s], 1).detach() + torch.finfo(dtype).smallest_normal
        assert bool((near | ~plain).all()), act


# ---- gradients against differences ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
@pytest.mark.parametrize("act", ["none", "elu", "silu"])
def test_gradients_against_differences(op, kind, act):
    """Along random directions, the kernel's gradients in 32 bits and central differences of the definition in 64 bits: their own error is
    (1e-4)^2 / 6 of third derivatives, 1e-8, and 1e-16 / 1e-4 of the values; the gradients' is 2^-18 of sums of some hundred terms."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    x = image((2, 8 if kind == "norm" else 16, 6, 7), torch.float32, gen).requires_grad_(True)
    w = (1 + 0.3 * torch.randn(8, device=DEV, generator=gen)).requires_grad_(True)
    b = (0.3 * torch.randn(8, device=DEV, generator=gen)).requires_grad_(True)
    dy = torch.randn((2, 8, 6, 7), device=DEV, generator=gen)
    leaves = [x] if kind == "gate" else [x, w, b]
    grads = torch.autograd.grad(call(op, kind, x, 2, w, b, 1e-5, act), leaves, dy)

    def loss(values):
        v = dict(zip("xwb", values))
        y = Reference64(kind, v["x"], 2, v.get("w"), v.get("b"), 1e-5, act)
        return float((y * dy.double()).sum())

    for which in range(len(leaves)):
        direction = torch.randn(leaves[which].shape, device=DEV, generator=gen, dtype=torch.float64)
        at = lambda e: [t.detach().double() + (e * direction if i == which else 0) for i, t in enumerate(leaves)]
        want = (loss(at(1e-4)) - loss(at(-1e-4))) / 2e-4
        got = float((grads[which].double() * direction).sum())
        scale = float((grads[which].double() * direction).abs().sum())
        assert abs(got - want) <= 2.0 ** -18 * scale + 1e-5 * (1 + scale ** 0.5), (which, got, want)


def Reference64(kind, x, groups, w, b, eps, act):
    C = x.shape[1] if kind == "norm" else x.shape[1] // 2
    u = x if kind == "norm" else act64(x[:, :C], act) / (1 + torch.exp(-x[:, C:]))
    if kind == "gate":
        return u
    ug = u.reshape(u.shape[0], groups, -1)
    uhat = ((ug - ug.mean(2, keepdim=True)) / torch.sqrt(ug.var(2, unbiased=False, keepdim=True) + eps)).reshape(u.shape)
    z = uhat * w.view(1, -1, 1, 1) + b.view(1, -1, 1, 1)
    return act64(z, act) if kind == "norm" else z


# ---- layouts, leaves, dtypes, refusals ----------------------------------------------------------------------------------------
def test_strides_that_are_taken_or_copied(op):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(4)
    base = image((6, 24, 10, 12), torch.float32, gen)
    one = image((1, 8, 10, 12), torch.float32, gen)
    views = {"every other image": base[::2, :8], "some rows": base[:, :8, 2:7], "every other column": base[:, :8, :, ::2], "one image, many times": one.expand(4, -1, -1, -1),
             "one pixel, many times": one[:, :, :1, :1].expand(2, 8, 5, 6), "one row": base[:, :8, :1], "one column": base[:, :8, :, :1], "flipped": base[:, :8].flip(0),
             "planar": base[:, :8].contiguous(), "channels strided": base[:, ::3], "off by one element": torch.randn(8 * 120 + 1, device=DEV)[1:].view(1, 10, 12, 8).permute(0, 3, 1, 2)}
    for name, x in views.items():
        dense = x.clone(memory_format=torch.contiguous_format).contiguous(memory_format=torch.channels_last)
        C = x.shape[1]
        w, b = torch.randn(C, device=DEV, generator=gen), torch.randn(C, device=DEV, generator=gen)
        ref = Reference("norm", dense, 4, w, b, 1e-5, "silu")
        check(op.group_norm(x, 4, w, b, 1e-5, "silu"), ref.y, ref.y_tol, name)
        ref = Reference("gated_norm", dense, 2, w[:C // 2], b[:C // 2], 1e-5, "elu")
        check(op.gated_group_norm(x, 2, w[:C // 2].contiguous(), b[:C // 2].contiguous()), ref.y, ref.y_tol, name)
        ref = Reference("gate", dense, 0, None, None, 0, "elu")
        check(op.gated_activation(x), ref.y, ref.y_tol, name)


def test_upstream_gradients_in_any_order(op):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    x = image((2, 16, 12, 14), torch.float32, gen).requires_grad_(True)
    y = op.group_norm(x, 4, None, None, 1e-5, "silu")
    ones = torch.ones_like(y)
    want, = torch.autograd.grad(y, [x], ones, retain_graph=True)
    for dy in (torch.ones((), device=DEV).expand(y.shape), torch.ones(y.shape, device=DEV), ones.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)):
        assert torch.equal(torch.autograd.grad(y, [x], dy, retain_graph=True)[0], want)
    (s,) = torch.autograd.grad(y.sum(), [x], retain_graph=True)
    assert torch.equal(s, want)
    for dy in (ones.double(), ones.bfloat16()):  # of another type: as if converted
        assert torch.equal(torch.autograd.grad(y, [x], dy, retain_graph=True)[0], want)
    # a leaf that is used twice gets both gradients
    two, = torch.autograd.grad(op.group_norm(x, 4, None, None, 1e-5, "silu") + op.group_norm(x, 4, None, None, 1e-5, "silu"), [x], ones)
    assert torch.allclose(two, 2 * want, rtol=1e-6, atol=0)


def test_gradients_of_some_leaves(op):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(6)
    x, dy = image((2, 16, 40, 30), torch.bfloat16, gen), image((2, 16, 40, 30), torch.bfloat16, gen)
    w, b = torch.randn(16, device=DEV), torch.randn(16, device=DEV)
    leaf = lambda t, on: t.detach().clone(memory_format=torch.preserve_format).requires_grad_(on)
    full = [leaf(t, True) for t in (x, w, b)]
    want = torch.autograd.grad(op.group_norm(full[0], 4, full[1], full[2], 1e-5, "elu"), full, dy)
    for on in itertools.product([False, True], repeat=3):
        if not any(on):
            continue
        leaves = [leaf(t, o) for t, o in zip((x, w, b), on)]
        got = torch.autograd.grad(op.group_norm(leaves[0], 4, leaves[1], leaves[2], 1e-5, "elu"), [t for t, o in zip(leaves, on) if o], dy)
        for g, k in zip(got, [k for k in range(3) if on[k]]):
            assert torch.equal(g, want[k])
    # weight or bias alone
    for args in ((w, None), (None, b)):
        p = [t.clone().requires_grad_(True) if t is not None else None for t in args]
        xs = leaf(x, True)
        y = op.group_norm(xs, 4, p[0], p[1], 1e-5, "elu")
        grads = torch.autograd.grad(y, [t for t in (xs, *p) if t is not None], dy)
        ref = Reference("norm", xs, 4, p[0], p[1], 1e-5, "elu", dy)
        check(y, ref.y, ref.y_tol, "y")
        check(grads[0], ref.dx, ref.dx_tol, "dx")
        check(grads[1], ref.dw if p[0] is not None else ref.db, ref.dw_tol if p[0] is not None else ref.db_tol, "parameter")


def test_empty(op):
    for shape in ((0, 8, 4, 4), (2, 8, 0, 4), (2, 8, 4, 0)):
        x = torch.randn(shape, device=DEV).requires_grad_(True)
        w, b = torch.ones(8, device=DEV, requires_grad=True), torch.zeros(8, device=DEV, requires_grad=True)
        y = op.group_norm(x, 2, w, b)
        assert y.shape == x.shape
        gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.ones_like(y))
        assert gx.shape == x.shape and not bool(gw.any()) and not bool(gb.any())
        assert op.gated_activation(x).shape == (shape[0], 4, *shape[2:])
        assert op.gated_group_norm(x, 2).shape == (shape[0], 4, *shape[2:])


def test_refusals(op):
    x = torch.randn((2, 12, 5, 6), device=DEV)
    w = torch.ones(12, device=DEV)
    bad = [lambda: op.group_norm(x.cpu(), 3), lambda: op.group_norm(x[0], 3), lambda: op.group_norm(x, 5), lambda: op.group_norm(x, 0), lambda: op.group_norm(x, -3),
           lambda: op.group_norm(x.double(), 3), lambda: op.group_norm(x.int(), 3), lambda: op.group_norm(x, 3, w[:6]), lambda: op.group_norm(x, 3, w.half()),
           lambda: op.group_norm(x, 3, w.cpu()), lambda: op.group_norm(x, 3, w, w.half()), lambda: op.group_norm(x, 3, torch.ones(24, device=DEV)[::2]),
           lambda: op.group_norm(x, 3, None, None, -1.0), lambda: op.group_norm(x, 3, None, None, float("nan")), lambda: op.group_norm(x, 3, None, None, 1e-5, "gelu"),
           lambda: op.gated_activation(x[:, :11]), lambda: op.gated_activation(x, "tanh"), lambda: op.gated_group_norm(x, 4), lambda: op.gated_group_norm(x, 3, w),
           lambda: op.group_norm(torch.zeros((1, 4097, 1, 1), device=DEV), 1), lambda: op.group_norm(x.half(), 3, w.bfloat16())]
    for k, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {k} was not refused")
    # a second derivative is refused, not silently wrong
    xg = x.clone().requires_grad_(True)
    for y in (op.group_norm(xg, 3), op.gated_activation(xg)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y.square().sum(), [xg], create_graph=True)


# ---- streams, graphs, devices ---------------------------------------------------------------------------------------------------
def step(op, kind, x, w, b, dy):
    y = call(op, kind, x, 4, w, b, 1e-5, "elu")
    leaves = [t for t in (x, w, b) if t is not None and t.requires_grad]
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def case(kind, size, seed, dtype=torch.bfloat16):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    B, H, W = size
    x = image((B, 16 if kind == "norm" else 32, H, W), dtype, gen).requires_grad_(True)
    w = b = None
    if kind != "gate":
        w, b = (torch.randn(16, device=DEV, generator=gen).requires_grad_(True) for _ in range(2))
    return x, w, b, image((B, 16, H, W), dtype, gen)


@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
@pytest.mark.parametrize("size", [(2, 20, 24), (4, 512, 384), (9, 768, 512)], ids=str)
def test_same_bits_every_time_and_on_two_streams_at_once(op, kind, size):
    cases = [case(kind, size, k) for k in range(2)]
    want = [step(op, kind, *c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(step(op, kind, *c))
        torch.cuda.synchronize()
        for g, v in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(g, v))


@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
@pytest.mark.parametrize("size", [(2, 12, 10), (4, 256, 300), (5, 768, 512)], ids=str)
def test_replay_from_cuda_graphs(op, kind, size):
    """Forward and backward captured, two graphs in one memory pool, beside copies, fills and a join of two streams; replayed with other values."""
    x, w, b, dy = case(kind, size, 7)
    static = x.detach().clone(memory_format=torch.preserve_format)
    out = torch.empty_like(dy)

    def body(leaf):
        leaf.data.copy_(static)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            leaf.data.mul_(1.5)
        torch.cuda.current_stream().wait_stream(side)
        out.zero_()
        r = step(op, kind, leaf, w, b, dy)
        out.copy_(r[0])
        return r

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        body(x)
        stream.synchronize()
        graphs, results, pool = [], [], None
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream, pool=pool):
                results.append(body(x))
            pool = g.pool()
            graphs.append(g)
        for seed in range(3):
            static.copy_(image(tuple(static.shape), static.dtype, torch.Generator(device=DEV).manual_seed(seed)))
            want = [t.clone() for t in body(x)]
            for g, r in zip(graphs, results):
                g.replay()
                stream.synchronize()
                assert all(torch.equal(p, q) for p, q in zip(r, want)), seed
                assert torch.equal(out, want[0])


def test_the_other_device(op):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    x = torch.randn((2, 16, 64, 64), device="cuda:1").requires_grad_(True)
    with torch.cuda.device(0):
        y = op.group_norm(x, 4)
        g, = torch.autograd.grad(y, [x], torch.ones_like(y))
    assert y.device == x.device == g.device


def test_a_stream_with_a_part_of_the_gpu(op, eight_sm_stream):
    """A green context with eight SMs: the same bits, since nobody waits for blocks that may not be resident."""
    cases = [(k, case(k, s, 3)) for k in ("norm", "gate", "gated_norm") for s in ((2, 20, 24), (4, 256, 300), (5, 768, 512))]
    want = [step(op, k, *c) for k, c in cases]
    torch.cuda.synchronize()
    with torch.cuda.stream(eight_sm_stream):
        got = [step(op, k, *c) for k, c in cases]
    torch.cuda.synchronize()
    for g, v in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, v))


# ---- the C ABI -------------------------------------------------------------------------------------------------------------------
def c_image(t, c0=0):
    return capi.AdopNormImage(t.data_ptr() + c0 * t.element_size(), t.stride(0), t.stride(3))


@pytest.mark.parametrize("size", [(2, 6, 7), (3, 300, 257)], ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_c_abi_writes_its_own_only(cuda_lib, size, dtype):
    """Outputs inside wider images, a workspace of exactly the bytes asked for: what lies around them stays as it was."""
    lib, (B, H, W) = cuda_lib, size
    gen = torch.Generator(device=DEV)
    gen.manual_seed(8)
    types = {torch.float32: capi.TYPE_F32, torch.float16: capi.TYPE_F16, torch.bfloat16: capi.TYPE_BF16}
    C_, G = 16, 4
    wide = lambda c: torch.full((B + 1, H + 1, W, c), 7.0, device=DEV, dtype=dtype).permute(0, 3, 1, 2)
    x, dy = wide(40), wide(24)
    x.copy_(torch.randn(x.shape, device=DEV, generator=gen))
    dy.copy_(torch.randn(dy.shape, device=DEV, generator=gen))
    y, dx, dg = wide(24), wide(24), wide(24)
    w, b = torch.randn(C_, device=DEV, generator=gen), torch.randn(C_, device=DEV, generator=gen)
    stats = torch.full((2 * B * G + 8,), 7.0, device=DEV)
    dw, db = torch.full((C_ + 8,), 7.0, device=DEV), torch.full((C_ + 8,), 7.0, device=DEV)
    p = capi.AdopNormParams(B, C_, H * W, G, types[dtype], capi.TYPE_F32, capi.ACTIVATION_ELU, 1e-5, w.data_ptr(), b.data_ptr())
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    for gated in (False, True):
        for t in (y, dx, dg, stats, dw, db):
            t.fill_(7.0)
        need = max(lib.adop_group_norm_workspace_bytes(C.byref(p), gated, k) for k in (0, 1))
        ws = torch.full((need + 64,), 77, device=DEV, dtype=torch.uint8)
        io = capi.AdopNormIO(x=c_image(x, 8), y=c_image(y, 8), grad_y=c_image(dy, 8), grad_x=c_image(dx, 8), mean=stats.data_ptr(), rstd=stats.data_ptr() + 4 * B * G,
                             grad_weight=dw.data_ptr(), grad_bias=db.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=need)
        if gated:
            io.gate, io.grad_gate = c_image(x, 24), c_image(dg, 8)
        capi.check(lib.adop_group_norm_forward(C.byref(p), C.byref(io), stream), "forward")
        capi.check(lib.adop_group_norm_backward(C.byref(p), C.byref(io), stream), "backward")
        torch.cuda.synchronize()
        part = lambda t, c0=8, c=16: t[:B, c0:c0 + c, :H]
        xin = torch.cat([part(x), part(x, 24)], 1) if gated else part(x)
        ref = Reference("gated_norm" if gated else "norm", xin, G, w, b, 1e-5, "elu", part(dy))
        check(part(y), ref.y, ref.y_tol, "y")
        check(torch.cat([part(dx), part(dg)], 1) if gated else part(dx), ref.dx, ref.dx_tol, "dx")
        check(dw[:C_], ref.dw, ref.dw_tol, "dw")
        check(db[:C_], ref.db, ref.db_tol, "db")
        check(stats[:B * G].view(B, G), ref.mean, 2.0 ** -18 * (1 + ref.mean.abs()), "mean")
        check(stats[B * G:2 * B * G].view(B, G), ref.rstd, 2.0 ** -16 * ref.rstd, "rstd")
        for t in (y, dx) + ((dg,) if gated else ()):
            kept = torch.ones(t.shape, dtype=torch.bool, device=DEV)
            kept[:B, 8:24, :H] = False
            assert bool((t[kept] == 7).all())
        assert bool((stats[2 * B * G:] == 7).all() and (dw[C_:] == 7).all() and (db[C_:] == 7).all() and (ws[need:] == 77).all())
    # the gate alone
    y.fill_(7.0); dx.fill_(7.0); dg.fill_(7.0)
    io = capi.AdopNormIO(x=c_image(x, 8), gate=c_image(x, 24), y=c_image(y, 8), grad_y=c_image(dy, 8), grad_x=c_image(dx, 8), grad_gate=c_image(dg, 8))
    capi.check(lib.adop_gated_activation_forward(C.byref(p), C.byref(io), stream), "forward")
    capi.check(lib.adop_gated_activation_backward(C.byref(p), C.byref(io), stream), "backward")
    torch.cuda.synchronize()
    ref = Reference("gate", torch.cat([part(x), part(x, 24)], 1), 0, None, None, 0, "elu", part(dy))
    check(part(y), ref.y, ref.y_tol, "y")
    check(torch.cat([part(dx), part(dg)], 1), ref.dx, ref.dx_tol, "dx")
    for t in (y, dx, dg):
        kept = torch.ones(t.shape, dtype=torch.bool, device=DEV)
        kept[:B, 8:24, :H] = False
        assert bool((t[kept] == 7).all())


def test_offsets_beyond_32_bits(op):
    """Two images whose elements lie more than 2^32 apart, and rows far apart: 9 GB of bfloat16."""
    far = (1 << 32) + 1 << 0
    big = torch.zeros(far + 4096 * 64, device=DEV, dtype=torch.bfloat16)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(9)
    stride = (far // 8) * 8
    x = big.as_strided((2, 32, 16, 16), (stride, 1, 16 * 32, 32))
    x.copy_(torch.randn((2, 32, 16, 16), device=DEV, generator=gen))
    rows = big.as_strided((1, 32, 1, 40), (0, 1, 0, stride // 64 // 8 * 8))
    for t in (x, rows):
        t.copy_(torch.randn(t.shape, device=DEV, generator=gen))
        dense = t.clone(memory_format=torch.contiguous_format)
        for kind in ("norm", "gate", "gated_norm"):
            ref = Reference(kind, dense, 4, None, None, 1e-5, "elu")
            check(call(op, kind, t, 4, None, None, 1e-5, "elu"), ref.y, ref.y_tol, kind)


# ---- as a renderer uses them --------------------------------------------------------------------------------------------------------
def test_from_descriptors_to_the_tonemapped_image(op):
    """Rasterized pyramid -> a gated block with normalisation, a basic block, a gated block without -> tonemapped image, gradients back to the
    descriptors; against the same network with the operators' definitions in torch, in 32 bits both. The convolutions and the rasterizer
    (float atomics) are the same on both sides; relative to the gradients' norms the sides differ by some 1e-6 each."""
    from adop_b200 import synth
    from tests.test_torch_op_gpu import _info
    torch.backends.cudnn.allow_tf32, before = False, torch.backends.cudnn.allow_tf32
    try:
        cfg = synth.make_config("c2", n_points=60_000, n_views=2, size=(160, 96))
        a, dev = cfg["arrays"], torch.device(DEV)
        texture = torch.from_numpy(a["texture"]).to(dev).requires_grad_(True)
        rest = [torch.from_numpy(a["background"]).to(dev), torch.from_numpy(a["position"]).to(dev),
                torch.zeros((a["poses"].shape[0], 6), dtype=torch.float64, device=dev), torch.from_numpy(a["intrinsics"]).to(dev)]
        gen = torch.Generator(device=DEV)
        gen.manual_seed(10)
        rnd = lambda *s: (torch.randn(s, device=DEV, generator=gen) / (s[1] * 9) ** 0.5).contiguous(memory_format=torch.channels_last).requires_grad_(True)
        conv = [rnd(32, 4, 3, 3), rnd(24, 16, 3, 3), rnd(6, 24, 3, 3)]
        norm = [torch.ones(16, device=DEV, requires_grad=True), torch.zeros(16, device=DEV, requires_grad=True),
                torch.ones(24, device=DEV, requires_grad=True), torch.zeros(24, device=DEV, requires_grad=True)]
        leaves = [texture, *conv, *norm]
        dy = torch.randn((2, 3, 96, 160), device=DEV, generator=gen)
        info = _info(cfg, dev)

        def network(x, blocks):
            c = lambda t, k: torch.nn.functional.conv2d(t, conv[k], padding=1)
            x = blocks[0](c(x.contiguous(memory_format=torch.channels_last), 0), 4, norm[0], norm[1])
            x = blocks[1](c(x, 1), 6, norm[2], norm[3])
            x = blocks[2](c(x, 2))
            return op.tonemap(x.contiguous(), None, None, None, None, None, None, None, 160, 96, 0.01)

        def plain_norm(u, groups, w, b):
            ug = u.reshape(u.shape[0], groups, -1)
            uhat = ((ug - ug.mean(2, keepdim=True)) * torch.rsqrt(ug.var(2, unbiased=False, keepdim=True) + 1e-5)).reshape(u.shape)
            return uhat * w.view(1, -1, 1, 1) + b.view(1, -1, 1, 1)

        def plain_gate(t):
            f, g = t.chunk(2, 1)
            return torch.nn.functional.elu(f) * torch.sigmoid(g)

        own = [lambda t, g, w, b: op.gated_group_norm(t, g, w, b), lambda t, g, w, b: op.group_norm(t, g, w, b, 1e-5, "silu"), lambda t: op.gated_activation(t)]
        plain = [lambda t, g, w, b: plain_norm(plain_gate(t), g, w, b), lambda t, g, w, b: torch.nn.functional.silu(plain_norm(t, g, w, b)), plain_gate]
        got, want = [], []
        for blocks, to in ((own, got), (plain, want)):
            pyramid = op.blend_point_cloud(texture, *rest, info)
            x = sum(torch.nn.functional.interpolate(t, size=(96, 160)) for t in pyramid[:cfg["num_layers"]])
            image_ = network(x, blocks)
            to.extend([image_.detach(), *torch.autograd.grad(image_, leaves, dy)])
        for k, (g, v) in enumerate(zip(got, want)):
            assert float((g - v).norm()) <= 1e-4 * float(v.norm()), k
        assert float(want[1].norm()) > 0
    finally:
        torch.backends.cudnn.allow_tf32 = before


def test_kernel_times_have_names(op, cuda_lib):
    x = torch.randn((4, 16, 300, 400), device=DEV)
    capi.profile_enable(True)
    op.group_norm(x, 4)
    op.gated_activation(x)
    torch.cuda.synchronize()
    times = capi.profile_collect()
    capi.profile_enable(False)
    assert {"k_norm_stats", "k_norm_apply", "k_gate"} <= set(times)
