"""The rendering network's operators: what the C ABI refuses (nothing is launched), without a GPU."""
import ctypes as C

import pytest

from adop_b200 import capi

INVALID, UNSUPPORTED, CUDA, WORKSPACE, SIZE = 1, 2, 3, 4, 5
P = 1 << 20  # an address that is only ever looked at
ENTRIES = ["adop_group_norm_forward", "adop_group_norm_backward", "adop_gated_activation_forward", "adop_gated_activation_backward"]


@pytest.fixture(scope="module")
def lib():
    from adop_b200 import build
    build.build_library()
    return capi.load_library()


def params(**kw):
    p = capi.AdopNormParams()
    v = dict(batch=2, channels=16, pixels=60, num_groups=4, type=capi.TYPE_F16, param_type=capi.TYPE_F32, activation=capi.ACTIVATION_ELU, eps=1e-5)
    v.update(kw)
    for k, x in v.items():
        setattr(p, k, x)
    return p


def io(workspace_bytes=1 << 40, **kw):
    t = capi.AdopNormIO()
    image = lambda k: capi.AdopNormImage(P * (k + 1), 60 * 16, 16)
    for k, name in enumerate(("x", "gate", "y", "grad_y", "grad_x", "grad_gate")):
        setattr(t, name, image(k))
    t.mean, t.rstd, t.workspace, t.workspace_bytes = 64 * P, 65 * P, 66 * P, workspace_bytes
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def call(lib, entry, p, t):
    return getattr(lib, entry)(C.byref(p) if p else None, C.byref(t) if t else None, None)


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("bad,status", [(dict(batch=-1), INVALID), (dict(channels=0), INVALID), (dict(pixels=-1), INVALID), (dict(type=3), INVALID),
                                        (dict(activation=4), INVALID), (dict(activation=-1), INVALID), (dict(channels=4097), SIZE),
                                        (dict(batch=65536), SIZE), (dict(pixels=0x7F000001), SIZE)])
def test_sizes_and_types(lib, entry, bad, status):
    assert call(lib, entry, params(**bad), io()) == status
    assert lib.adop_last_error().decode()


@pytest.mark.parametrize("entry", ENTRIES[:2])
@pytest.mark.parametrize("bad", [dict(num_groups=0), dict(num_groups=3), dict(num_groups=-4), dict(eps=-1e-5), dict(eps=float("nan")), dict(eps=float("inf")),
                                 dict(param_type=capi.TYPE_BF16), dict(param_type=7)])
def test_normalisation(lib, entry, bad):
    p = params(**bad)
    assert call(lib, entry, p, io()) == INVALID
    assert lib.adop_group_norm_workspace_bytes(C.byref(p), 1, 1) == 0


@pytest.mark.parametrize("entry", ENTRIES)
def test_missing_structs(lib, entry):
    assert call(lib, entry, None, io()) == INVALID
    assert call(lib, entry, params(), None) == INVALID


def images_of(entry):
    return ["x", "gate", "y"] if entry.endswith("forward") else ["x", "gate", "grad_y", "grad_x", "grad_gate"]


@pytest.mark.parametrize("entry", ENTRIES)
def test_images(lib, entry):
    for name in images_of(entry):
        image = lambda *a: io(**{name: capi.AdopNormImage(*a)})
        if name != "gate" or "gated" in entry:  # a group norm without a gate is a call of its own
            assert call(lib, entry, params(), image(None, 960, 16)) == INVALID, name
        assert call(lib, entry, params(), image(P + 1, 960, 16)) == INVALID, name      # not aligned to its type
        assert call(lib, entry, params(), image(P, -960, 16)) == INVALID, name
        assert call(lib, entry, params(), image(P, 960, -16)) == INVALID, name
        assert call(lib, entry, params(), image(P, 1 << 56, 16)) == INVALID, name
        assert call(lib, entry, params(), image(P, 960, 1 << 51)) == INVALID, name
        if name in ("y", "grad_x", "grad_gate"):  # the pixels of an output do not overlap
            assert call(lib, entry, params(), image(P, 960, 15)) == INVALID, name
            assert call(lib, entry, params(), image(P, 959, 16)) == INVALID, name
            assert call(lib, entry, params(), image(P, 0, 16)) == INVALID, name


@pytest.mark.parametrize("backward", [0, 1])
def test_workspace_and_statistics(lib, backward):
    """Images that no cluster's shared memory holds; smaller ones may need no workspace."""
    entry, big = ENTRIES[backward], params(pixels=1 << 20)
    stride = (1 << 20) * 16
    images = {name: capi.AdopNormImage(P * (k + 1), stride, 16) for k, name in enumerate(("x", "gate", "y", "grad_y", "grad_x", "grad_gate"))}
    need = lib.adop_group_norm_workspace_bytes(C.byref(big), 1, backward)
    assert need > 0
    assert call(lib, entry, big, io(workspace_bytes=need - 1, **images)) == WORKSPACE
    assert call(lib, entry, big, io(workspace=None, **images)) == WORKSPACE
    assert call(lib, entry, big, io(workspace=66 * P + 8, **images)) == INVALID
    assert call(lib, entry, params(), io(mean=None)) == INVALID
    assert call(lib, entry, params(), io(rstd=None)) == INVALID
    assert call(lib, entry, params(), io(mean=64 * P + 2)) == INVALID
    assert call(lib, entry, params(weight=P + 2), io()) == INVALID
    assert call(lib, entry, params(bias=P + 1, param_type=capi.TYPE_F16), io()) == INVALID
    if backward:
        assert call(lib, entry, params(), io(grad_weight=P + 2)) == INVALID
        assert call(lib, entry, params(), io(grad_bias=P + 3)) == INVALID


@pytest.mark.parametrize("entry", ENTRIES)
def test_nothing_to_do(lib, entry):
    """An empty batch or image needs no tensors; the parameters' gradients would be zeroed, so none are given here."""
    for empty in (dict(batch=0), dict(pixels=0)):
        assert call(lib, entry, params(**empty), capi.AdopNormIO()) == 0
        assert lib.adop_group_norm_workspace_bytes(C.byref(params(**empty)), 0, 1) == 0


def test_workspace_grows_with_the_batch_only_as_needed(lib):
    sizes = [lib.adop_group_norm_workspace_bytes(C.byref(params(batch=b, pixels=512 * 512)), 0, 1) for b in (1, 4, 16)]
    assert 0 < sizes[0] and sizes[-1] <= 64 << 20
