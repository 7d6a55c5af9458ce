"""The rendering network's operators and autograd: what they do not differentiate they refuse, and what autograd hands them (tensors whose
values are not as stored, arguments that are wrong) is taken for what it is."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from tests.test_norm_gate_gpu import DEV, call, image, op  # noqa: F401 (op is a fixture)

pytestmark = pytest.mark.gpu


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ---- forward-mode derivatives: refused, not dropped ---------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_a_tangent_of_an_input_is_refused(op, kind, grad_mode):
    x = image((2, 8 if kind == "norm" else 16, 6, 7), torch.float32, generator(1))
    w, b = torch.ones(8, device=DEV), torch.zeros(8, device=DEV)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        for which in range(1 if kind == "gate" else 3):
            for leaf in (False, True):  # a tensor that wants a gradient, too, carries a tangent
                args = [t.clone(memory_format=torch.preserve_format).requires_grad_(leaf) for t in (x, w, b)]
                args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(op, kind, args[0], 2, args[1], args[2], 1e-5, "elu")
        # a dual level without tangents is a call like any other
        y = call(op, kind, x, 2, w, b, 1e-5, "elu")
        assert forward_ad.unpack_dual(y).tangent is None
    assert torch.equal(y, call(op, kind, x, 2, w, b, 1e-5, "elu"))


@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
def test_a_tangent_of_the_upstream_gradient_is_refused(op, kind):
    x = image((2, 8 if kind == "norm" else 16, 6, 7), torch.float32, generator(2)).requires_grad_(True)
    with forward_ad.dual_level():
        y = call(op, kind, x, 2, None, None, 1e-5, "elu")
        scale = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad((y * scale).sum(), [x])


def test_functional_jvp_is_refused(op):
    x = image((2, 16, 6, 7), torch.float32, generator(3))
    for kind in ("norm", "gate", "gated_norm"):
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda v: call(op, kind, v, 2, None, None, 1e-5, "elu"), (x,), (torch.ones_like(x),))


# ---- tensors whose values are not as stored ---------------------------------------------------------------------------------------
def negated(t):
    """t's values as a view of their negatives."""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


@pytest.mark.parametrize("kind", ["norm", "gate", "gated_norm"])
def test_negated_views_are_taken_for_their_values(op, kind):
    gen = generator(4)
    C = 8 if kind == "norm" else 16
    x, dy = image((2, C, 6, 7), torch.float32, gen), image((2, 8, 6, 7), torch.float32, gen)
    w, b = torch.randn(8, device=DEV, generator=gen), torch.randn(8, device=DEV, generator=gen)
    want = call(op, kind, x, 2, w, b, 1e-5, "elu")
    assert torch.equal(call(op, kind, negated(x), 2, negated(w), negated(b), 1e-5, "elu"), want)
    leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_(True) for t in ((x,) if kind == "gate" else (x, w, b))]
    through = lambda f: call(op, kind, f(leaves[0]), 2, *(f(t) for t in leaves[1:]), 1e-5, "elu") if kind != "gate" else call(op, kind, f(leaves[0]), 0, None, None, 0, "elu")
    plain = torch.autograd.grad(through(lambda t: t), leaves, dy)
    y = through(lambda t: torch._neg_view(t.neg()))
    assert torch.equal(y, want)
    for got, grad in zip(torch.autograd.grad(y, leaves, negated(dy)), plain):
        assert torch.equal(got, grad)


def test_the_gradient_of_an_imaginary_part(op):
    """The upstream gradient is a view of a conjugate there: one channel, pixels two elements apart, negated."""
    gen = generator(5)
    x = image((2, 2, 6, 7), torch.float32, gen).requires_grad_(True)
    re, scale = (torch.randn((2, 1, 6, 7), device=DEV, generator=gen) for _ in range(2))
    seen = []
    y = op.gated_activation(x)
    y.register_hook(lambda g: seen.append(g.is_neg()))
    # |re + i y|^2 / 2 by way of a conjugate: dy = y scale
    loss = (torch.complex(re, y).conj().resolve_conj().abs().square() * scale).sum() / 2
    got, = torch.autograd.grad(loss, [x])
    assert seen == [True]
    want, = torch.autograd.grad(op.gated_activation(x), [x], y.detach() * scale)
    # dy by way of abs(): some rounding steps of 2^-24 of |re|^2 + y^2 over |z|; gx is dy times factors of at most 1.1
    bound = 2.0 ** -20 * (re.abs() + y.detach().abs()) * scale.abs() * 1.1 * (1 + x.detach().abs().sum(1, keepdim=True))
    assert bool(((got - want).abs() <= bound).all())
    assert bool((want.abs() > 4 * bound).any())


# ---- refusals of a recorded call ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("groups", [0, -4, 5, 17, 1 << 20, (1 << 31) - 1, 1 << 40, (1 << 63) - 1])
def test_groups_are_checked_before_anything_is_allocated_for_them(op, groups):
    x = image((2, 16, 6, 7), torch.float32, generator(6)).requires_grad_(True)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for kind in ("norm", "gated_norm"):
        with pytest.raises(RuntimeError, match="num_groups"):
            call(op, kind, x, groups, None, None, 1e-5, "elu")
    assert torch.cuda.max_memory_allocated() <= before + (1 << 20)
