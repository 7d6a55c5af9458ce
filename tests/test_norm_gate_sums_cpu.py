"""Group norm: a thread's chain of 32-bit additions does not grow with the image, as the workspace shows; no GPU."""
import ctypes as C
import math

import pytest

from adop_b200 import capi

CHAIN = 256     # vectors that a thread adds up at most
THREADS = 512   # of a block, at most


@pytest.fixture(scope="module")
def lib():
    from adop_b200 import build
    build.build_library()
    return capi.load_library()


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("kind,size", [(capi.TYPE_F32, 4), (capi.TYPE_F16, 2), (capi.TYPE_BF16, 2)])
@pytest.mark.parametrize("batch,pixels,channels,groups", [(1, 0x7F000000, 4, 2), (1, 0x7F000000, 1, 1), (3, 1 << 24, 37, 37), (200, 512 * 512, 48, 6), (1, 1 << 20, 4096, 1)])
def test_large_images_have_partial_sums_enough(lib, batch, pixels, channels, groups, kind, size, gated, backward):
    """Vectors of four elements, which some tensor of these sizes allows, are the longest: a block adds up CHAIN of them a thread at most then.
    (Those of one or two go on in a second chain of as many.)"""
    p = capi.AdopNormParams(batch, channels, pixels, groups, kind, capi.TYPE_F32, capi.ACTIVATION_ELU, 1e-5, None, None)
    parts = math.ceil(pixels * channels / (CHAIN * 4 * max(THREADS, channels // math.gcd(channels, 4))))
    need = lib.adop_group_norm_workspace_bytes(C.byref(p), gated, backward)
    assert need >= 8 * batch * parts * (groups + (channels if backward else 0))
    # and it stays a small part of the image: at least half of 384 threads have something to do, and 148 blocks have one part each that is not full
    assert need <= 8 * batch * (groups + (channels if backward else 0)) * (2 * 148 + 3 * parts) + 64


def test_ordinary_images_have_a_partial_sum_for_each_block(lib):
    """One 512 x 512 x 32 image of a batch of four, forward: 37 of 148 blocks, 56 or 111 vectors for each of their threads."""
    p = capi.AdopNormParams(4, 32, 512 * 512, 8, capi.TYPE_F16, capi.TYPE_F32, capi.ACTIVATION_ELU, 1e-5, None, None)
    assert lib.adop_group_norm_workspace_bytes(C.byref(p), 0, 0) == 8 * 4 * 8 * 37
