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
