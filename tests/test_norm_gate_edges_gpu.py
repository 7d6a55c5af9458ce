"""The rendering network's operators where the other tests of theirs look less closely: gates and features in the tails in both directions,
gradients far from zero and beyond 32-bit offsets, rows wider than a block that go on for long.

Bounds of the sigmoid, derived before the first run: exp(-v) is 2^m with m = v log2(e) rounded once (2^-24 of m) from a constant that is off by
2^-26.1 of itself: 0.62 |v| 2^-23 of the exponential, and two units of the last place of its own. Then s = 1 / (1 + exp(-v)) has one rounding and one
unit more, (0.62 |v| + 4) 2^-23 of s; 1 - s = exp(-v) s another exponential's two units and a rounding, (0.62 |v| + 7) 2^-23: the error of the
exponential's argument enters both, at most once in all. Sigmoids below 2^-126 are 0. Where a feature's activation and its slope come with
exponentials of their own, 2^-18 as in the other tests."""
import ctypes as C
import gc

import pytest
import torch

from adop_b200 import capi
from tests.test_norm_gate_gpu import ACTS, DEV, TYPES, Reference, act64, call, check, half_step, image, op, run_case, slope64  # noqa: F401 (op is a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def gigabytes_given_back():
    """What later tests keep is not to lie in a cached block of these ones' sizes."""
    yield
    gc.collect()
    torch.cuda.empty_cache()

ULP = 2.0 ** -23


# ---- the tails of the gate --------------------------------------------------------------------------------------------------------
def test_the_sigmoid_up_to_its_smallest_values(op):
    """Feature 1 behind no activation: y = s and dg = s (1 - s), and behind SiLU df = s + f s (1 - s) at an open gate; float32."""
    v = torch.cat([torch.linspace(0, 87, 40001, device=DEV), torch.linspace(-87, 0, 40001, device=DEV)])
    v = v[: v.numel() // 8 * 8].view(1, 1, -1, 8)
    x = torch.cat([torch.ones_like(v), v], 1).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    y = op.gated_activation(x, "none")
    gx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    vd = v.double()
    s, ns = torch.sigmoid(vd), torch.sigmoid(-vd)
    size = 0.62 * vd.abs()
    check(y, s, (size + 4) * ULP * s, "s")
    # a float32 product below the smallest normal number is as fine as the numbers there
    check(gx[:, 1:], s * ns, (size + 4 + 7) * ULP * s * ns + 2.0 ** -126, "s (1 - s)")
    x = torch.cat([v, torch.full_like(v, 200.0)], 1).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    y = op.gated_activation(x, "silu")
    gx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    check(y, vd * s, (size + 5) * ULP * (vd * s).abs() + 2.0 ** -126, "silu")
    # 1 + v (1 - s) is a sum of terms of both signs
    check(gx[:, :1], s * (1 + vd * ns), (size + 4 + 1) * ULP * s * (1 + (vd * ns).abs()) + (size + 7) * ULP * s * (vd * ns).abs() + 2.0 ** -126 * (1 + vd.abs()), "silu'")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
def test_gates_and_features_in_the_tails(op, act, dtype):
    """Every finite feature with every gate up to the infinities, forward and backward: no overflow on the way, and nothing at all through a
    closed gate."""
    inf = float("inf")
    f = torch.tensor([0.0, 1.0, -2.0, 60000.0, -60000.0, 300.0, -300.0, 100.0, -100.0, 88.5, -88.5, 20.0, -20.0, 3.0, -0.5, 1e-4, -1e-4], device=DEV)
    g = torch.tensor([inf, -inf, 60000.0, -60000.0, 128.0, -128.0, 100.0, -100.0, 90.0, -90.0, 88.5, -88.5, 87.0, -87.0, 60.0, -60.0, 17.0, -17.0, 1.0, 0.0], device=DEV)
    ff, gg = torch.meshgrid(f, g, indexing="ij")
    x = torch.stack([ff, gg])[None].to(dtype).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    y = op.gated_activation(x, act)
    gx, = torch.autograd.grad(y, [x], torch.ones_like(y))
    xd = x.detach().double()
    fd, gd = xd[:, :1], xd[:, 1:]
    s, ns = torch.sigmoid(gd), torch.sigmoid(-gd)
    fs_, fns = torch.sigmoid(fd), torch.sigmoid(-fd)
    fa = fd * fs_ if act == "silu" else act64(fd, act)
    slope = fs_ * (1 + fd * fns) if act == "silu" else slope64(fd, act)
    h, tiny = half_step(dtype), torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    rel = 2.0 ** -18 + 0.62 * ULP * (gd.abs().clamp(max=88) + fd.abs().clamp(max=88))
    flush = 2.0 ** -125  # of a sigmoid, or of an exponential's product with one
    check(y, fa * s, (h + rel) * (fa * s).abs() + tiny + flush * (1 + fd.abs()), "y")
    check(gx[:, :1], slope * s, (h + rel) * (slope * s).abs() + tiny + flush * (1 + fd.abs()), "df")
    check(gx[:, 1:], fa * s * ns, (h + rel) * (fa * s * ns).abs() + tiny + flush * (1 + fd.abs()), "dg")
    closed = (gd <= -89).expand_as(fd)
    for t in (y, gx[:, :1], gx[:, 1:]):
        assert bool(torch.isfinite(t).all()) and not bool(t[closed].any())


# ---- gradients where offsets are large ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("offset", [100.0, -3000.0])
def test_gradients_far_from_zero(op, offset, act):
    """Means far beyond the spread, and one first pixel that is far from the others."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    for shape in ((2, 8, 16, 24), (1, 8, 256, 260)):
        x = (offset + torch.randn(shape, device=DEV, generator=gen)).contiguous(memory_format=torch.channels_last)
        w, b = (1 + 0.3 * torch.randn(8, device=DEV, generator=gen)).requires_grad_(True), (0.3 * torch.randn(8, device=DEV, generator=gen)).requires_grad_(True)
        dy = image(shape, torch.float32, gen)
        for first in (None, 0.0):
            if first is not None:
                x[:, :, 0, 0] = first
            leaf = x.clone(memory_format=torch.preserve_format).requires_grad_(True)
            y = op.group_norm(leaf, 2, w, b, 1e-5, act)
            ref = Reference("norm", x, 2, w, b, 1e-5, act, dy)
            check(y, ref.y, ref.y_tol, f"y, first {first}")
            for got, name in zip(torch.autograd.grad(y, [leaf, w, b], dy), ("dx", "dw", "db")):
                check(got, getattr(ref, name), getattr(ref, name + "_tol"), f"{name}, first {first}")


FAR = ((1 << 32) + 4096) // 8 * 8


@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
def test_gradients_beyond_32_bit_offsets(op, kind):
    """Inputs and upstream gradients whose images, or whose pixels, lie more than 2^32 elements apart: 9 GB of bfloat16."""
    big = torch.zeros(FAR + 4096 * 64, device=DEV, dtype=torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(9)
    step = FAR // 39 // 8 * 8
    out = 32 if kind == "norm" else 16
    views = [(lambda c, at: big.as_strided((2, c, 16, 16), (FAR, 1, 16 * c, c), at)), (lambda c, at: big.as_strided((1, c, 1, 40), (0, 1, 0, step), at))]
    assert 39 * step + 32 + 65536 < big.numel() and 39 * step > (1 << 32) - 65536
    for view in views:
        x, dy = view(32, 0).requires_grad_(True), view(out, 65536)
        x.data.copy_(torch.randn(x.shape, device=DEV, generator=gen))
        dy.copy_(torch.randn(dy.shape, device=DEV, generator=gen))
        y = call(op, kind, x, 4, None, None, 1e-5, "elu")
        gx, = torch.autograd.grad(y, [x], dy)
        ref = Reference(kind, x.detach().clone(memory_format=torch.contiguous_format), 4, None, None, 1e-5, "elu", dy.clone(memory_format=torch.contiguous_format))
        check(y, ref.y, ref.y_tol, "y")
        check(gx, ref.dx, ref.dx_tol, "dx")


@pytest.mark.parametrize("gated,norm", [(False, True), (True, True), (True, False)])
def test_results_beyond_32_bit_offsets(cuda_lib, gated, norm):
    """The same for what the calls write, through the C ABI; nothing is written anywhere else."""
    lib = cuda_lib
    big = torch.zeros(FAR + 4096 * 64, device=DEV, dtype=torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(10)
    c, B = 16, 2
    rnd = lambda: torch.randn((B, 16, 16, c), device=DEV, generator=gen).bfloat16().permute(0, 3, 1, 2)
    x, gate, dy = rnd(), rnd(), rnd()
    at = lambda k: big.as_strided((B, c, 16, 16), (FAR, 1, 32 * 16, 32), k * 16384)
    y, dx, dg = (at(k) for k in range(3))
    im = lambda t: capi.AdopNormImage(t.data_ptr(), t.stride(0), t.stride(3))
    p = capi.AdopNormParams(B, c, 256, 4, capi.TYPE_BF16, capi.TYPE_F32, capi.ACTIVATION_ELU, 1e-5, None, None)
    stats = torch.empty((2, B, 4), device=DEV)
    need = max(lib.adop_group_norm_workspace_bytes(C.byref(p), gated, k) for k in (0, 1))
    ws = torch.empty(need, device=DEV, dtype=torch.uint8)
    io = capi.AdopNormIO(x=im(x), y=im(y), grad_y=im(dy), grad_x=im(dx), mean=stats.data_ptr(), rstd=stats.data_ptr() + 4 * B * 4, workspace=ws.data_ptr(), workspace_bytes=need)
    if gated:
        io.gate, io.grad_gate = im(gate), im(dg)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    name = "adop_group_norm" if norm else "adop_gated_activation"
    capi.check(getattr(lib, name + "_forward")(C.byref(p), C.byref(io), stream), "forward")
    capi.check(getattr(lib, name + "_backward")(C.byref(p), C.byref(io), stream), "backward")
    ref = Reference(("gated_norm" if gated else "norm") if norm else "gate", torch.cat([x, gate], 1) if gated else x, 4, None, None, 1e-5, "elu", dy)
    check(y, ref.y, ref.y_tol, "y")
    check(torch.cat([dx, dg], 1) if gated else dx, ref.dx, ref.dx_tol, "dx")
    for t in (y, dx, dg):
        t.zero_()
    assert not bool(big.any())


# ---- rows wider than a block, many of them --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
@pytest.mark.parametrize("channels,groups", [(4096, 1), (4096, 4096), (2308, 4)], ids=str)
def test_wide_rows_that_go_on(op, kind, channels, groups, dtype):
    """A hundred and fifty images and more, one block each: several passes over the rows, each of more vectors than are under way at once."""
    run_case(op, kind, (150, channels, 7, 9), groups, dtype, "silu", seed=11)
