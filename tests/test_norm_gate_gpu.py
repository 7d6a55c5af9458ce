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
            self.db_tol = pt * self.db.abs() + total(e_dz) + 2.0 ** -21 * total(dz.abs()) + 1e-30
            self.dw_tol = pt * self.dw.abs() + total(e_dw) + 2.0 ** -21 * total((dz * uhat).abs()) + 1e-30
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
