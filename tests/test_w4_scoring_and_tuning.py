"""The 4-bit Linear, the output layer's loss and their gradients together, as scoring and tuning a model with frozen 4-bit
projections use them, and the same operators through the torch extension and the serving path."""
import os
import sys

import pytest
import torch

from moonpoly_b200 import vllm_linear
from test_linear_w4 import make, tokens, weight, within
from test_linear_xent import bounds, exact, inputs

EXT_DIR = os.path.abspath(os.path.join(os.path.dirname(__file__), "..", "moonpoly-dev_b200", "torch_ext"))


@pytest.fixture(scope="module")
def ops():
    if EXT_DIR not in sys.path:
        sys.path.insert(0, EXT_DIR)
    import moonpoly                     # noqa: F401  registers torch.ops.moonpoly_ops
    return torch.ops.moonpoly_ops


def test_schemas_and_meta_kernels(ops):
    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")
    x, qw, s, z = meta(5, 160), meta(24, 32, dtype=torch.int32), meta(24, 5), meta(24, 5, dtype=torch.uint8)
    assert ops.pack_w4(meta(24, 160, dtype=torch.uint8)).shape == (24, 32)
    y = ops.linear_w4(x, qw, s, z, 32)
    assert y.shape == (5, 24) and y.dtype == torch.bfloat16
    assert ops.linear_w4_grad_input(y, qw, s, z, 32, 160).shape == (5, 160)
    assert ops.linear_w4_grad_input(y, qw, s, z, 32).shape == (5, 256)
    w, t = meta(300, 160), meta(5, dtype=torch.int64)
    loss, lse = ops.linear_cross_entropy(x, w, t)
    assert loss.shape == lse.shape == (5,) and loss.dtype == lse.dtype == torch.float32
    dx, dw = ops.linear_cross_entropy_grad(x, w, t, lse, loss)
    assert dx.shape == (5, 160) and dw.shape == (300, 160)
    assert ops.linear_cross_entropy_grad(x, w, t, lse, loss, -100, True, False)[1].shape == (0, 160)


def test_extension_refuses_host_tensors(ops):
    x, qw, s = torch.zeros(2, 64).half(), torch.zeros(8, 16, dtype=torch.int32), torch.zeros(8, 2).half()
    for call in (lambda: ops.linear_w4(x, qw, s, None, 32), lambda: ops.linear_cross_entropy(x, x, torch.zeros(2, dtype=torch.int64))):
        with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
            call()


def test_serving_path_declines_without_a_gpu(monkeypatch):
    x, qw, s = torch.zeros(2, 64).half(), torch.zeros(8, 16, dtype=torch.int32), torch.zeros(8, 2).half()
    monkeypatch.delenv("VLLM_USE_MOONPOLY_LINEAR", raising=False)
    assert vllm_linear.apply_moonpoly_linear_w4(x, qw, s, None, 32) is None
    monkeypatch.setenv("VLLM_USE_MOONPOLY_LINEAR", "1")
    assert vllm_linear.apply_moonpoly_linear_w4(x, qw, s, None, 32) is None

    class Layer:
        weight = torch.ones(8, 64).half()
        moonpoly_w4 = (qw, s, None, 32)
    assert vllm_linear.apply(Layer(), x, fallback=lambda la, xx, bb: "engine") == "engine"


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_extension_gives_the_same_bits(api, ops, m):
    q, s, z = make(130, 288, 32, torch.float16, seed=m)
    x, dy = tokens(m, 288, torch.float16), tokens(m, 130, torch.float16)
    bias = torch.randn(130, device="cuda").half()
    pw = ops.pack_w4(q)
    assert torch.equal(pw, api.pack_w4(q))
    assert torch.equal(ops.linear_w4(x, pw, s, z, 32, bias), api.linear_w4(x, pw, s, z, 32, bias))
    assert torch.equal(ops.linear_w4_grad_input(dy, pw, s, z, 32, 288), api.linear_w4_grad_input(dy, pw, s, z, 32, 288))
    x, w, t, g = inputs(m, 500, 96, torch.bfloat16, seed=m)
    loss, lse = ops.linear_cross_entropy(x, w, t)
    want = api.linear_cross_entropy(x, w, t)
    assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
    for a, b in zip(ops.linear_cross_entropy_grad(x, w, t, lse, g), api.linear_cross_entropy_grad(x, w, t, lse, g)):
        assert torch.equal(a, b)
    with pytest.raises(ValueError):
        ops.linear_w4(x, pw, s, z, 32)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(x, w[:, :90], t)


@pytest.mark.gpu
def test_serving_path_runs_a_4_bit_layer(ops, monkeypatch):
    monkeypatch.setenv("VLLM_USE_MOONPOLY_LINEAR", "1")
    vllm_linear.reset_stats()
    q, s, z = make(96, 256, 64, torch.bfloat16, seed=4)
    layer = torch.nn.Module()
    layer.moonpoly_w4 = (ops.pack_w4(q), s, z, 64)
    bias = torch.randn(96, device="cuda").bfloat16()
    x = tokens(6, 256, torch.bfloat16)
    out = vllm_linear.apply(layer, x.view(2, 3, 256), bias)
    assert out.shape == (2, 3, 96) and vllm_linear.STATS["linear_w4"] == 1
    within(out.view(6, 96), x, weight(q, s, z, 64), bias, False)
    # a layer of another type of weight falls back
    assert vllm_linear.apply(layer, x.float(), None, fallback=lambda la, xx, bb: "engine") == "engine"
    assert vllm_linear.STATS["declined"] == 1


class W4Linear(torch.autograd.Function):
    """A frozen 4-bit projection in a training graph."""

    @staticmethod
    def forward(ctx, x, api, qweight, scales, zeros, group):
        ctx.args = (api, qweight, scales, zeros, group, x.shape[1])
        return api.linear_w4(x, qweight, scales, zeros, group)

    @staticmethod
    def backward(ctx, dy):
        api, qweight, scales, zeros, group, k = ctx.args
        return api.linear_w4_grad_input(dy, qweight, scales, zeros, group, k), None, None, None, None, None


class LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, target, api):
        loss, lse = api.linear_cross_entropy(x, w, target)
        ctx.save_for_backward(x, w, target, lse)
        ctx.api = api
        return loss

    @staticmethod
    def backward(ctx, grad_loss):
        x, w, target, lse = ctx.saved_tensors
        dx, dw = ctx.api.linear_cross_entropy_grad(x, w, target, lse, grad_loss, need_dx=ctx.needs_input_grad[0], need_dw=ctx.needs_input_grad[1])
        return dx, dw, None, None


@pytest.mark.gpu
@pytest.mark.parametrize("m", [7, 200])
def test_scoring_and_tuning_through_autograd(api, m):
    """hidden -> 4-bit projection -> output layer's mean loss -> gradients; every stage is held to the bounds of its own
    formula on the inputs that it really had."""
    dtype, k, h, v, group = torch.bfloat16, 416, 192, 1500, 32
    q, s, z = make(h, k, group, dtype, seed=m)
    pw = api.pack_w4(q)
    x = tokens(m, k, dtype).requires_grad_()
    _, w, target, _ = inputs(m, v, h, dtype, seed=m)
    w.requires_grad_()
    kept = (target >= 0).sum()
    hidden = W4Linear.apply(x, api, pw, s, z, group)
    hidden.retain_grad()
    loss = LinearCrossEntropy.apply(hidden, w, target, api).sum() / kept
    loss.backward()
    assert api.device_status() == 0
    wq = weight(q, s, z, group)
    within(hidden.detach(), x.detach(), wq, None, m > 16)
    e = exact(hidden.detach(), w.detach(), target, torch.full((m,), 1.0 / float(kept), device="cuda"))
    fwd, bx, bw = bounds(hidden.detach(), w.detach(), e)
    assert abs(float(loss.detach()) - float(e["loss"].sum() / kept)) <= float(fwd.mean()) + 1e-6
    assert ((hidden.grad.double() - e["dx"]).abs() <= bx).all()
    assert ((w.grad.double() - e["dw"]).abs() <= bw).all()
    within(x.grad, hidden.grad, wq.t(), None, True)


@pytest.mark.gpu
def test_a_tuning_step_captured_while_an_eager_one_lives(api):
    """The explicit gradients of one step captured in a graph, with eager results of the same tensors alive."""
    dtype, m, k, h, v = torch.float16, 90, 256, 128, 700
    q, s, z = make(h, k, 64, dtype, seed=1)
    pw, x = api.pack_w4(q), tokens(m, k, dtype)
    _, w, target, g = inputs(m, v, h, dtype, seed=2)

    def step():
        hidden = api.linear_w4(x, pw, s, z, 64)
        loss, lse = api.linear_cross_entropy(hidden, w, target)
        dh, dw = api.linear_cross_entropy_grad(hidden, w, target, lse, g)
        return loss, dw, api.linear_w4_grad_input(dh, pw, s, z, 64, k)
    want = step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x2 = tokens(m, k, dtype, seed=9)
    eager = x.clone()
    x.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    new = step()
    assert all(torch.equal(a, b) for a, b in zip(out, new)) and not torch.equal(out[0], want[0])
    x.copy_(eager)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
