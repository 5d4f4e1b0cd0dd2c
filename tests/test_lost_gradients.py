"""The functions of api.py return results without an autograd graph, and say so where that loses a gradient."""
import warnings

import pytest
import torch

from test_linear_w4 import make, tokens
from test_linear_xent import inputs
from test_w4_scoring_and_tuning import LinearCrossEntropy, W4Linear


@pytest.mark.gpu
def test_a_lost_gradient_is_told(api):
    q, s, z = make(96, 128, 32, torch.float16)
    pw, x = api.pack_w4(q), tokens(5, 128, torch.float16)
    h, w, target, _ = inputs(5, 300, 96, torch.float16)

    def calls(xx, hh, ww):
        return (lambda: api.linear_w4(xx, pw, s, z, 32)), (lambda: api.linear_cross_entropy(hh, ww, target))
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for call in calls(x, h, w):
            call()
    want = [calls(x, h, w)[0](), *calls(x, h, w)[1]()]
    xg, hg, wg = (t.clone().requires_grad_() for t in (x, h, w))
    for call in (*calls(xg, hg, w), calls(x, h, wg)[1]):
        with pytest.warns(RuntimeWarning, match="carries no autograd graph"):
            call()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with torch.no_grad():
            for call in calls(xg, hg, wg):
                call()
        hidden = W4Linear.apply(xg, api, pw, s, z, 32)                     # as a training graph uses them
        loss = LinearCrossEntropy.apply(hidden, wg, target, api)
        loss.sum().backward()
    with pytest.warns(RuntimeWarning):
        assert torch.equal(calls(xg, hg, wg)[0](), want[0])
    assert xg.grad is not None and wg.grad is not None
