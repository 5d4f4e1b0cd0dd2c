"""Linear with softmax cross entropy where its arithmetic is strained: infinite logits beside large finite ones."""
import pytest
import torch

from test_linear_xent import DTYPES, IGNORE, exact, inputs

NINF, INF, NAN = float("-inf"), float("inf"), float("nan")


@pytest.mark.gpu
@pytest.mark.parametrize("v", [300, 9001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_logits_beside_large_ones(api, v, dtype):
    # every pair of 128-entry pieces, joined early or late, either one first: the infinity wins, whatever the other's size
    x = torch.ones((8, 64), dtype=dtype, device="cuda")
    target = torch.full((8,), 1, dtype=torch.int64, device="cuda")
    for at, large in ((5, v - 1), (v - 1, 5), (5, 140), (140, 5), (200, 201)) + (((5, 4101), (4101, 5), (8200, 9000)) if v > 9000 else ()):
        for size in (2.0, 100.0, -100.0):                                  # logits of 128 and of +- 6400
            w = torch.zeros((v, 64), dtype=dtype, device="cuda")
            w[large], w[at] = size, INF
            loss, lse = api.linear_cross_entropy(x, w, target)
            assert (lse == INF).all() and (loss == INF).all(), (at, large, size, lse, loss)
            w[at] = NINF                                                   # masked out: the others decide
            loss, lse = api.linear_cross_entropy(x, w, target)
            z = x.double() @ w.double().t()
            assert torch.allclose(lse.double(), torch.logsumexp(z, 1), rtol=1e-6) and torch.isfinite(loss).all()
            w[at] = NAN
            loss, lse = api.linear_cross_entropy(x, w, target)
            assert torch.isnan(lse).all() and torch.isnan(loss).all()
            w[large], w[at] = NAN, INF
            assert torch.isnan(api.linear_cross_entropy(x, w, target)[1]).all()
    assert api.device_status() == 0
