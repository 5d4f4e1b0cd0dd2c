"""Linear with softmax cross entropy: only an operand whose own rows miss 16 bytes is copied into the workspace."""
import ctypes

import pytest
import torch

from test_linear_xent import DTYPES, check, inputs

M, V, H = 40, 5000, 136


def size(api, x=4096, ldx=H, w=4096, ldw=H, backward=0, h=H, m=M):
    n = ctypes.c_size_t()
    p = ctypes.c_void_p
    assert api.lib().mp_linear_xent_workspace(api.MP_FP16, m, V, h, p(x), ldx, p(w), ldw, backward, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("backward", [0, 1])
def test_workspace_holds_copies_of_unaligned_operands_alone(api, backward):
    up = lambda b: (b + 255) // 256 * 256
    copy_x, copy_w = up(M * 192 * 2), up(V * 192 * 2)                     # rows are padded to whole blocks of 64
    none = size(api, backward=backward)
    for bad in (dict(x=4098), dict(ldx=H + 1), dict(x=4104, ldx=H + 4)):
        assert size(api, **bad, backward=backward) == none + copy_x, bad
    for bad in (dict(w=4098), dict(ldw=H + 1), dict(w=4104, ldw=H + 4)):
        assert size(api, **bad, backward=backward) == none + copy_w, bad
    assert size(api, x=4098, ldw=H + 1, backward=backward) == none + copy_x + copy_w
    assert size(api, ldx=H + 8, ldw=H + 16, backward=backward) == none


def test_python_asks_for_the_same_sizes(api):
    for ax in (True, False):
        for aw in (True, False):
            for backward in (0, 1):
                assert api._xent_workspace_bytes(api.MP_FP16, M, V, H, ax, aw, backward) == size(api, x=4096 if ax else 4098, w=4096 if aw else 4098, backward=backward)
                assert api._xent_workspace_bytes(api.MP_FP16, M, V, 63, ax, aw, backward) == size(api, x=4096 if ax else 4098, w=4096 if aw else 4098, ldx=64, ldw=64, h=63, backward=backward)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [136, 1111, 63])
def test_every_mixture_of_alignments_gives_the_same_bits(api, h, dtype):
    x, w, target, g = inputs(M, 700, h, dtype, seed=h)
    want = check(api, x, w, target, g)

    def at(t, offset, pad):
        rows, width = t.shape
        flat = torch.full((rows * (width + pad) + 16,), float("nan"), dtype=dtype, device="cuda")
        return flat[offset:offset + rows * (width + pad)].view(rows, width + pad)[:, :width].copy_(t)
    aligned = -h % 8
    for xo, xp in ((0, aligned), (1, aligned), (0, aligned + 1), (8, aligned + 8)):
        for wo, wp in ((0, aligned), (1, aligned), (0, aligned + 1), (8, aligned + 8)):
            xx, ww = at(x, xo, xp), at(w, wo, wp)
            loss, lse = api.linear_cross_entropy(xx, ww, target)
            got = (loss, lse) + api.linear_cross_entropy_grad(xx, ww, target, lse, g)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (xo, xp, wo, wp)
    assert api.device_status() == 0
