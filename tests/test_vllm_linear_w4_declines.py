"""What becomes of a layer with a 4-bit weight when the operator's path declines: never another weight's numbers without a word,
never an error about something else, and no error of the device swallowed."""
import types
import warnings

import pytest
import torch

from moonpoly_b200 import vllm_linear


def cuda_like(*shape):
    """What the path looks at of a CUDA tensor."""
    t = types.SimpleNamespace(device=torch.device("cuda", 0), dtype=torch.float16, shape=torch.Size(shape))
    t.reshape = lambda *a: t
    return t


def layer(weight=None):
    la = torch.nn.Module()
    la.moonpoly_w4 = (cuda_like(8, 16), None, None, 32)
    if weight is not None:
        la.weight = torch.nn.Parameter(weight)
    return la


@pytest.fixture
def refusing(monkeypatch):
    def with_error(error):
        def linear_w4(*args):
            raise error
        monkeypatch.setenv("VLLM_USE_MOONPOLY_LINEAR", "1")
        monkeypatch.setattr(vllm_linear, "_ops", lambda: types.SimpleNamespace(linear=None, linear_w4=linear_w4))
        vllm_linear.reset_stats()
    return with_error


@pytest.mark.parametrize("weight", [None, torch.ones(8, 64).half()])
def test_a_refusal_without_a_fallback_is_the_operators_own(refusing, weight):
    refusing(ValueError("linear_w4: K must be a multiple of 32"))
    with pytest.raises(ValueError, match="multiple of 32"):
        vllm_linear.apply(layer(weight), cuda_like(2, 64))
    assert vllm_linear.STATS["declined"] == 1 and vllm_linear.STATS["linear"] == 0


@pytest.mark.parametrize("weight", [None, torch.ones(8, 64).half()])
def test_other_declines_without_a_fallback_say_why(monkeypatch, weight):
    monkeypatch.delenv("VLLM_USE_MOONPOLY_LINEAR", raising=False)
    with pytest.raises(RuntimeError, match="VLLM_USE_MOONPOLY_LINEAR"):
        vllm_linear.apply(layer(weight), cuda_like(2, 64))
    monkeypatch.setenv("VLLM_USE_MOONPOLY_LINEAR", "1")
    monkeypatch.setattr(vllm_linear, "_ops", lambda: None)
    with pytest.raises(RuntimeError, match="not registered"):
        vllm_linear.apply(layer(weight), torch.ones(2, 64).half())
    monkeypatch.setattr(vllm_linear, "_ops", lambda: types.SimpleNamespace(linear_w4=None))
    with pytest.raises(RuntimeError, match="CUDA"):
        vllm_linear.apply(layer(weight), torch.ones(2, 64).half())


def test_a_given_fallback_runs_and_the_reason_is_told(refusing):
    refusing(ValueError("linear_w4: scales must be [N, ceil(K / group_size)]"))
    with pytest.warns(RuntimeWarning, match="scales must be"):
        assert vllm_linear.apply(layer(), cuda_like(2, 64), fallback=lambda la, x, b: "engine") == "engine"


@pytest.mark.parametrize("fallback", [None, lambda la, x, b: "engine"])
def test_errors_of_the_device_are_not_caught(refusing, fallback):
    refusing(RuntimeError("cudaLaunchKernelExC failed: out of memory"))
    with pytest.raises(RuntimeError, match="out of memory"):
        vllm_linear.apply(layer(torch.ones(8, 64).half()), cuda_like(2, 64), fallback=fallback)
    with pytest.raises(RuntimeError, match="out of memory"):
        vllm_linear.apply_moonpoly_linear_w4(cuda_like(2, 64), *layer().moonpoly_w4)
    assert vllm_linear.STATS["declined"] == 0


def test_an_installed_path_without_another_weight_says_why(refusing, monkeypatch):
    class UnquantizedLinearMethod:
        def apply(self, la, x, bias=None):
            return la.weight

    module = types.SimpleNamespace(UnquantizedLinearMethod=UnquantizedLinearMethod)
    assert vllm_linear.install(module)
    refusing(ValueError("linear_w4: refused"))
    with pytest.raises(ValueError, match="refused"):
        UnquantizedLinearMethod().apply(layer(), cuda_like(2, 64))
    held = layer(torch.ones(8, 64).half())
    with pytest.warns(RuntimeWarning, match="refused"):                   # the engine's own weight, not without a word
        assert UnquantizedLinearMethod().apply(held, cuda_like(2, 64)) is held.weight
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        monkeypatch.setattr(vllm_linear, "_ops", lambda: None)            # not there at all: the engine's own, as it was
        assert UnquantizedLinearMethod().apply(held, cuda_like(2, 64)) is held.weight


@pytest.mark.gpu
def test_a_refusal_of_the_real_operator(api, monkeypatch):
    import os
    import sys
    ext = os.path.abspath(os.path.join(os.path.dirname(__file__), "..", "moonpoly-dev_b200", "torch_ext"))
    if ext not in sys.path:
        sys.path.insert(0, ext)
    import moonpoly                     # noqa: F401  registers torch.ops.moonpoly_ops
    monkeypatch.setenv("VLLM_USE_MOONPOLY_LINEAR", "1")
    la = torch.nn.Module()
    la.moonpoly_w4 = (torch.zeros(8, 16, dtype=torch.int32, device="cuda"), torch.zeros(8, 3, device="cuda").half(), None, 32)
    with pytest.raises(ValueError, match="scales must be"):
        vllm_linear.apply(la, torch.ones(2, 64, device="cuda").half())
    assert vllm_linear.apply_moonpoly_linear_w4(torch.ones(2, 64, device="cuda").half(), *la.moonpoly_w4) is None
