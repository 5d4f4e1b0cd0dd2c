"""The ring of packed weights in the tensor-core kernel of the 4-bit Linear, followed on the host.

Two groups of warps unpack in turns (two steps each, or the odd last step of a unit); turn T reads slot T % slots.  A wait for a
slot's fill passes by the parity of its phase, so it also passes, falsely, while the fill *before* the awaited one has not
landed.  That fill was turn T - slots.  It has certainly landed where the same group waited for it (an even number of slots), or
where the product of its first step is known to be done: the group's last stage of turn T - 2 became free only with the product
of the step `stages` before it."""
import ctypes

import pytest
import torch

from test_linear_w4 import DTYPES, make, tokens, weight, within


def turns_of(unit_steps):
    """[(first step, last step)] of the turns of consecutive units."""
    out, at = [], 0
    for steps in unit_steps:
        for s in range(0, steps, 2):
            out.append((at + s, at + min(s + 2, steps) - 1))
        at += steps
    return out


def false_passes(slots, stages, unit_steps):
    """Turns whose wait could pass before their fill has landed."""
    turns = turns_of(unit_steps)
    return [t for t in range(slots, len(turns))
            if slots % 2 == 1 and turns[t - 2][1] - stages < turns[t - slots][0]]


def launch(api, m, n, k, group=128, grad=0):
    out = (ctypes.c_int * 8)()
    assert api.lib().mp_debug_w4_launch(m, n, k, group, grad, out) == 0
    return dict(zip(("stream", "bn", "units", "split", "steps", "steps_per_split", "stages", "slots"), out))


def test_the_model_tells_safe_rings_from_unsafe_ones():
    for steps in range(1, 40):
        for slots in (2, 4, 5, 6):
            assert not false_passes(slots, 3, [steps] * 6), (slots, steps)
        assert bool(false_passes(3, 3, [steps] * 6)) == (steps % 2 == 1), steps
    for units in ([1] * 30, [3, 1, 2, 5, 1, 1, 1, 7, 2], [4, 1] * 9):
        assert not false_passes(5, 3, units) and not false_passes(2, 3, units)


@pytest.mark.parametrize("m,n,k,grad", [(180, 28672, 3456, 0), (380, 9728, 896, 0), (512, 9728, 896, 0), (540, 9728, 896, 0),
                                        (380, 11520, 2880, 0), (1537, 5760, 2880, 1), (192, 20000, 128, 0), (192, 128, 20000, 1)])
def test_many_units_of_an_odd_number_of_steps(api, m, n, k, grad):
    p = launch(api, m, n, k, grad=grad)
    assert p["steps"] % 2 == 1 and p["units"] > 74 and p["split"] == 1            # a pair of CTAs has a second unit
    assert not false_passes(p["slots"], p["stages"], [p["steps"]] * 6), p


def test_every_launch_keeps_its_ring_safe(api):
    seen = set()
    for m in list(range(17, 300, 5)) + [320, 380, 384, 500, 512, 768, 1001, 1537, 2047, 4096]:
        for n in (1, 256, 896, 5760, 9728, 11520, 28672, 70000):
            for k in (32, 128, 384, 896, 2880, 3456, 4096, 14336):
                for grad in (0, 1):
                    p = launch(api, m, n, k, 32, grad)
                    seen.add((p["bn"], p["slots"]))
                    assert not p["stream"] and p["stages"] >= 2 and p["slots"] >= 2
                    # what the ring, the stages and their barriers take of the shared memory of a CTA
                    assert 1024 + p["stages"] * (32768 + p["bn"] // 2 * 256) + p["slots"] * 16384 + 256 <= 232448
                    last = p["steps"] - (p["split"] - 1) * p["steps_per_split"]
                    for units in ([p["steps_per_split"]] * 6, [p["steps_per_split"], last] * 4):
                        assert not false_passes(p["slots"], p["stages"], units), (m, n, k, grad, p)
    assert {bn for bn, _ in seen} >= {32, 64, 96, 128, 160, 192, 224, 256}


def test_the_aid_refuses_bad_arguments(api):
    out = (ctypes.c_int * 8)()
    aid = api.lib().mp_debug_w4_launch
    assert launch(api, 16, 64, 64)["stream"] == 1 and launch(api, 16, 64, 64, grad=1)["stream"] == 0
    for args in ((0, 64, 64, 32, 0, out), (1, 0, 64, 32, 0, out), (1, 64, 0, 32, 0, out), (1, 64, 64, 16, 0, out),
                 ((1 << 28) + 1, 64, 64, 32, 0, out), (1, 64, 64, 32, 0, None)):
        assert aid(*args) != 0


def test_the_workspace_query_refuses_what_the_call_refuses(api):
    # a group size near 2^31 overflowed the number of groups, and sizes came back for calls that are refused
    n, p, z = ctypes.c_size_t(7), ctypes.c_void_p(4096), ctypes.c_void_p(0)
    L = api.lib()
    for group in (0, -1, 16, 33, 48, 2 ** 31 - 1, 2 ** 31 - 64):
        call = L.mp_linear_w4(api.MP_FP16, 100, 64, 4096, p, 4096, p, p, z, group, z, p, p, 1 << 30, z)
        assert call == 1 and L.mp_linear_w4_workspace(100, 64, 4096, group, p, 4096, 0, ctypes.byref(n)) == call, group
        assert L.mp_debug_w4_launch(100, 64, 4096, group, 0, (ctypes.c_int * 8)()) == call
    assert L.mp_linear_w4_workspace(100, 64, 4080, 32, p, 4080, 0, ctypes.byref(n)) == 3 and n.value == 7
    # one group per row: any size of at least K asks for the same
    sizes = set()
    for shift in range(12, 31):
        assert L.mp_linear_w4_workspace(300, 64, 4096, 1 << shift, p, 4096, 0, ctypes.byref(n)) == 0
        sizes.add(n.value)
    assert len(sizes) == 1


# ------------------------------------------------------------------------------------ many units per pair of CTAs (GPU)
MANY = [  # tokens, N, K, group: even and odd steps of 128 along the contraction, tiles of 160 to 256 tokens and of fewer
    (40, 20000, 256, 32), (40, 20000, 384, 64), (96, 20000, 128, 32), (120, 20000, 384, 128), (150, 19000, 640, 128), (150, 20000, 512, 32), (180, 28672, 3456, 128), (192, 20000, 128, 64),
    (380, 9728, 896, 128), (512, 9728, 896, 32), (380, 9728, 1024, 64), (700, 9000, 416, 256), (1100, 9728, 128, 128), (2047, 4100, 1056, 64)]


def zeros_to_63(q, s, z):
    """Zero points over their whole range, and a scale that keeps the weights' size."""
    gen = torch.Generator().manual_seed(7)
    z = torch.randint(0, 64, z.shape, generator=gen, dtype=torch.uint8).to(z.device)
    z.view(-1)[:2] = torch.tensor([0, 63], dtype=torch.uint8)
    return q, s, z


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,group", MANY)
def test_pairs_with_several_units(api, m, n, k, group, dtype):
    p = launch(api, m, n, k, group)
    assert p["units"] > 74 and p["split"] == 1
    q, s, z = zeros_to_63(*make(n, k, group, dtype, seed=m))
    x, pw = tokens(m, k, dtype), api.pack_w4(q)
    y = api.linear_w4(x, pw, s, z, group_size=group)
    assert api.device_status() == 0
    within(y, x, weight(q, s, z, group), None, True)
    assert all(torch.equal(api.linear_w4(x, pw, s, z, group_size=group), y) for _ in range(3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,group", [(40, 256, 20000, 32), (40, 300, 20000, 64), (192, 128, 20000, 32), (380, 896, 9728, 128),
                                         (512, 1000, 9728, 64), (1537, 5760, 2880, 128), (1001, 4096, 5120, 256), (2047, 33, 4128, 32)])
def test_pairs_with_several_units_of_the_gradient(api, m, n, k, group, dtype):
    p = launch(api, m, n, k, group, 1)
    assert p["units"] > 74 and p["split"] == 1
    q, s, z = zeros_to_63(*make(n, k, group, dtype, seed=m))
    dy, pw = tokens(m, n, dtype), api.pack_w4(q)
    dx = api.linear_w4_grad_input(dy, pw, s, z, group_size=group, in_features=k)
    assert api.device_status() == 0
    within(dx, dy, weight(q, s, z, group).t(), None, True)
    assert all(torch.equal(api.linear_w4_grad_input(dy, pw, s, z, group_size=group, in_features=k), dx) for _ in range(3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 7, 16, 17, 100])
def test_zero_points_over_their_whole_range(api, m, dtype):
    for group in (32, 128):
        q, s, z = zeros_to_63(*make(150, 672, group, dtype, seed=m))
        x = tokens(m, 672, dtype)
        within(api.linear_w4(x, api.pack_w4(q), s, z, group_size=group), x, weight(q, s, z, group), None, m > 16)
        dy = tokens(m, 150, dtype)
        dx = api.linear_w4_grad_input(dy, api.pack_w4(q), s, z, group_size=group, in_features=672)
        within(dx, dy, weight(q, s, z, group).t(), None, True)
