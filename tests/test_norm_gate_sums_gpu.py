"""Group norm over images that are much larger than the threads that add them up: two values in turn, the worst case of a chain of
additions in 32 bits, since every addition of the same number rounds the same way.

Bounds, derived before the first run: a thread adds up 256 values at most in 32 bits. Terms of one sign: each addition is off by 2^-24 of the
sum so far at most, half the last on average, so e = 2^-17 of the sum. With d = u - first value, 0 or D in turn: the sum of d^2 is twice the
squares about the mean, sum(d)^2 / n as much as these, so the squares about the mean are off by 2 e + 2 e of themselves, the variance by 4 e and
rstd by 2 e; the mean by e D / 2, which is e of the spread. uhat = +-1 is off by 3 e, and by 2^-22 |mean| rstd as everywhere. db and dw are
sums of one sign: e, and what uhat is off by."""
import gc

import pytest
import torch

from adop_b200 import capi
from tests.test_norm_gate_gpu import DEV, Reference, call, check, eight_sm_stream, image, op  # noqa: F401 (two are fixtures)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def gigabytes_given_back():
    """What later tests keep is not to lie in a cached block of these ones' sizes."""
    yield
    gc.collect()
    torch.cuda.empty_cache()

E = 2.0 ** -17


@pytest.mark.parametrize("dtype,channels,pixels,offset", [
    (torch.float32, 301, 148 * 14000, 1),   # single elements, 14000 rows to a block of 148
    (torch.float32, 500, 148 * 4 * 2000, 0),  # 16-byte vectors, four rows at a time
    (torch.bfloat16, 6, 148 * 512 * 600, 2),  # vectors of four bytes
], ids=str)
def test_two_values_in_turn(op, dtype, channels, pixels, offset):
    low, high = -0.25, 1.1241134 if dtype == torch.float32 else 1.125
    c1 = 0.7198558 if dtype == torch.float32 else 0.71875
    wide = channels + 2 * offset
    odd = (torch.arange(pixels, device=DEV) % 2).to(dtype)[:, None]
    two = lambda a, b: torch.tensor([a, b], device=DEV, dtype=dtype)[odd.long()]  # [pixels, 1], exactly the two
    x = two(low, high).expand(pixels, wide).contiguous().view(1, 1, pixels, wide).permute(0, 3, 1, 2)[:, offset:offset + channels].requires_grad_(True)
    dy = two(0.0, c1).expand(pixels, channels).contiguous().view(1, 1, pixels, channels).permute(0, 3, 1, 2)
    a, b, c1 = (float(v) for v in (torch.tensor([low, high, c1], dtype=dtype)))
    w, bias = torch.ones(channels, device=DEV, requires_grad=True), torch.zeros(channels, device=DEV, requires_grad=True)
    y = op.group_norm(x, channels, w, bias, 1e-5, "none")
    dx, dw, db = torch.autograd.grad(y, [x, w, bias], dy)
    mean, rstd = (a + b) / 2, 1 / (((b - a) / 2) ** 2 + 1e-5) ** 0.5
    uhat = (b - a) / 2 * rstd
    e_uhat = 3 * E + 2.0 ** -22 * abs(mean) * rstd + 2.0 ** -22
    h = torch.finfo(dtype).eps / 2
    ymin, ymax = (y[:, :, 0, k::2].float() for k in (0, 1))
    worst = max((ymin.double() + uhat).abs().max().item(), (ymax.double() - uhat).abs().max().item())
    print(f"y off by {worst:.3g}, bound {e_uhat + h:.3g}")
    assert worst <= e_uhat + h * uhat
    n = pixels // 2
    off = [((t.double() - v).abs().max() / v).item() for t, v in ((db, n * c1), (dw, n * c1 * uhat))]
    print(f"db, dw off by {off[0]:.3g}, {off[1]:.3g}, bounds {E + 2.0 ** -24:.3g}, {E + e_uhat + 2.0 ** -23:.3g}")
    assert off[0] <= E + 2.0 ** -24
    assert off[1] <= E + e_uhat + 2.0 ** -23
    # dz is c1 on one half: c1_mean = c1 / 2, c2 = c1 uhat / 2; dx = rstd (dz - c1 / 2 - uhat c2)
    for k, (dz, u) in enumerate(((0.0, -uhat), (c1, uhat))):
        want = rstd * (dz - c1 / 2 - u * uhat * c1 / 2)
        bound = rstd * c1 * (2 * E + 2 * (E + e_uhat) + 2.0 ** -20) + h * abs(want)
        assert (dx[:, :, 0, k::2].double() - want).abs().max().item() <= bound


def long_case(kind, size, seed):
    """Channels 4 to 19 (35) of wider images: vectors of 8 bytes, 438 of them for a thread of a 4K image, 512 for one of each of 75 blocks (which, behind a gate,
    do not overlap), a third more backward."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, H, W = size
    C = 16 if kind == "norm" else 32
    x = image((B, C + 4, H, W), torch.bfloat16, gen)[:, 4:].detach().requires_grad_(True)
    w, b = (torch.randn(16, device=DEV, generator=gen).requires_grad_(True) for _ in range(2))
    return x, w, b, image((B, 16, H, W), torch.bfloat16, gen)


def step(op, kind, x, w, b, dy):
    y = call(op, kind, x, 4, w, b, 1e-5, "silu")
    return [y.detach(), *torch.autograd.grad(y, [x, w, b], dy)]


def test_several_launches_are_what_these_are(op, cuda_lib):
    for kind, size in (("norm", (1, 2160, 3840)), ("gated_norm", (75, 256, 256))):
        x, w, b, _ = long_case(kind, size, 0)
        capi.profile_enable(True)
        call(op, kind, x, 4, w, b, 1e-5, "silu")
        torch.cuda.synchronize()
        times = capi.profile_collect()
        capi.profile_enable(False)
        assert times["k_norm_stats"][0] > times["k_norm_apply"][0]


@pytest.mark.parametrize("size", [(1, 2160, 3840), (75, 256, 256)], ids=str)
@pytest.mark.parametrize("kind", ["norm", "gated_norm"])
def test_several_launches_of_sums(op, kind, size, eight_sm_stream):
    """The values; and the same bits again, on two streams at once, on a stream with a part of the GPU and from a graph."""
    cases = [long_case(kind, size, k) for k in range(2)]
    want = [step(op, kind, *c) for c in cases]
    x, w, b, dy = cases[0]
    ref = Reference(kind, x, 4, w, b, 1e-5, "silu", dy)
    for got, name in zip(want[0], ("y", "dx", "dw", "db")):
        check(got, getattr(ref, name), getattr(ref, name + "_tol"), name)
    torch.cuda.synchronize()
    for streams in ([torch.cuda.Stream() for _ in cases], [eight_sm_stream] * 2):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(step(op, kind, *c))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for g, v in zip(got, want) for p, q in zip(g, v))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step(op, kind, *cases[0])
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step(op, kind, *cases[0])
        for _ in range(2):
            for t in got:
                t.zero_()
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want[0]))
