"""Linear with softmax cross entropy where its arithmetic is strained: infinite logits beside large finite ones, rows whose
target is nearly certain, long contractions.

The tensor cores drop what an addition shifts out, towards zero.  One addition takes 16 products; it loses half a unit of the
running sum on average, a unit being 2^-24 to 2^-23 of it.  A sum that grows evenly over n additions thus ends short by
n / 2 * 2^-24 of itself at most (the running sum is half the final one on average)."""
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


def confident(m, v, h, dtype, level, gap):
    """Rows of h elements whose target's logit is near `level` and the others' `gap` below, the same way for every row."""
    gen = torch.Generator().manual_seed(3)
    half = h // 2
    b = torch.randn((m, half), generator=gen)
    x = torch.cat([torch.ones(m, half), b], 1)                             # the first half carries what the logits share
    w = torch.randn((v, h), generator=gen) * 0.5 / half ** 0.5
    w[:, :half] = w[:, :half] * 0.1 + (level - gap) / half
    target = torch.randperm(v, generator=gen)[:m]
    w[target, half:] = gap * b / (b * b).sum(1, keepdim=True)
    return x.to(dtype).cuda(), w.to(dtype).cuda(), target.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("v", [2000, 70000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_loss_of_confident_rows(api, v, dtype):
    # The loss is log(1 + r) with an r of many terms, each below half a unit of the 1: added to it one by one they all vanish.
    # Added in pairs, a sum of 128 terms passes 7 additions, that of the pieces one for every 32 of them and 5 more; each is off by
    # half a unit of a number between 1 and 2, 2^-24.  r itself moves by exp (2^-21 with the rounding of its argument) and by the
    # truncation of the gap between the logits.
    level, gap = 22.0, 17.3
    x, w, target = confident(90, v, 2048, dtype, level, gap)
    loss, _ = api.linear_cross_entropy(x, w, target)
    e = exact(x, w, target, torch.ones(90, device="cuda"))
    r = e["loss"].expm1()
    assert (r / v > 2.0 ** -27).all() and (r / v < 2.0 ** -23).all()
    off = (loss.double() - e["loss"]).abs()
    tol = (12 + v // 4096) * 2.0 ** -24 + r * (2.0 ** -21 + 64 * 2.0 ** -23 * 2 * level)
    print(float((off / tol).max()), float(off.max()), float((loss.double() - e["loss"]).mean()), float(r.mean()))
    assert (off <= tol).all(), (off, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("level", [22.0, -22.0])
@pytest.mark.parametrize("h", [4096, 8192])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_confident_rows(api, h, level, dtype):
    # d at the target is -(1 - p), the difference of two numbers near one: the logits of the gradient have to be those that lse was
    # summed from.  lse in fp32 is off by 2^-24 of itself, its sum of exponentials by 12 additions of 2^-24 (test_loss_of_confident_rows),
    # exp by 2^-22: 2^-24 |lse| + 2^-20 in all, measured against 1 - p.  d and the result are rounded to 16 bits, u each.  The
    # others' probabilities move by the truncation of the gap between the logits.
    x, w, target = confident(60, 2000, h, dtype, level, 18.0)
    g = torch.full((60,), 1024.0, device="cuda")
    _, lse = api.linear_cross_entropy(x, w, target)
    dx, dw = api.linear_cross_entropy_grad(x, w, target, lse, g)
    e = exact(x, w, target, g)
    rest = -e["d"].gather(1, target[:, None]).squeeze(1) / g               # 1 - p
    assert (rest > 1e-5).all() and (rest < 1e-3).all()
    u = torch.finfo(dtype).eps / 2
    off = (dx.double() - e["dx"]).norm(dim=1) / e["dx"].norm(dim=1)
    # w at the target is the longest of what the row sums up: an error of d there counts by |w_t| / |w_t - mean of the others|
    lever = w[target].double().norm(dim=1) * rest * g / e["dx"].norm(dim=1)
    tol = 2 * u + lever * (2.0 ** -24 * e["lse"].abs() + 2.0 ** -20) / rest + 64 * 2.0 ** -23 * 2 * abs(level)
    print(float(off.max()), float((off / tol).max()), float(rest.max()), float(lever.max()))
    assert (off <= tol).all(), (off, tol)
    # the same through dw: row t of it is d_t x
    off = (dw.double() - e["dw"])[target].norm(dim=1) / e["dw"][target].norm(dim=1)
    assert (off <= 2 * u + (2.0 ** -24 * e["lse"].abs() + 2.0 ** -20) / rest + 64 * 2.0 ** -23 * 2 * abs(level)).all(), off


@pytest.mark.gpu
@pytest.mark.parametrize("m,v,h", [(1024, 131072, 4096), (131072, 1024, 256)])
def test_long_sums_of_the_gradients_are_not_short(api, m, v, h):
    # dx is summed over the vocabulary, dw over the rows: 8192 additions of 16 products each.  In one accumulator such a sum ends short
    # by up to 8192 / 2 * 2^-24 = 2.4e-4 (what it loses comes to 0.5 to 1 of that, as the unit is 2^-24 to 2^-23 of the sum).  In
    # chunks of 512 additions it is 512 / 2 * 2^-24.  Measured along the exact gradient, where the roundings of d and of the result do
    # not add up: d at the m targets, u / sqrt(3) each, leaves u / sqrt(3 m); the logits' own shortness, of chunks of 64 additions,
    # moves p by 64 / 2 * 2^-24 (z - mean z), |z - mean z| < 20 here.
    x, w, target, g = inputs(m, v, h, torch.float16, seed=2, skip=0.0)
    g = torch.ones_like(g)
    _, lse = api.linear_cross_entropy(x, w, target)
    grads = api.linear_cross_entropy_grad(x, w, target, lse, g)
    e = exact(x, w, target, g)
    tol = 256 * 2.0 ** -24 + 20 * 32 * 2.0 ** -24 + 4 * 2.0 ** -11 / (3 * m) ** 0.5
    for name, got in zip(("dx", "dw"), grads):
        short = float((got.double() * e[name]).sum() / (e[name] ** 2).sum()) - 1.0
        print(name, short, tol)
        assert abs(short) <= tol, (name, short, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("h", [1024, 4096, 16384])
@pytest.mark.parametrize("dtype", DTYPES)
def test_mean_and_rms_errors_over_a_long_hidden_size(api, h, dtype):
    # A chunk of 64 additions leaves its part of a logit short by f <= 64 / 2 * 2^-24 of it, so a logit by f of itself, whatever h,
    # and lse by f E[z] (the mean under the softmax), loss by f (E[z] - z_target).  With a single accumulator f would be 128 * 2^-24 at
    # h = 4096, and never below half of that.  lse in fp32 is rounded by 2^-24 of itself at random; exp moves it by 2^-22 at
    # most; single additions scatter by half a unit each, 2 sqrt(h / 16) 2^-24 max |z| over a row's logits.
    m, v = 512, 8192
    x, w, target, g = inputs(m, v, h, dtype, seed=h, skip=0.0)
    loss, lse = api.linear_cross_entropy(x, w, target)
    dx, dw = api.linear_cross_entropy_grad(x, w, target, lse, g)
    e = exact(x, w, target, g)
    z = x.double() @ w.double().t()
    mean_z = ((z - e["lse"][:, None]).exp() * z).sum(1)
    f = 32 * 2.0 ** -24
    for name, got, part in (("lse", lse, mean_z), ("loss", loss, mean_z - (e["lse"] - e["loss"]))):
        off = got.double() - e[name]
        mean, rms = float(off.mean()), float(off.square().mean().sqrt())
        # the means of the random parts: over m rows
        noise = 2.0 ** -24 * float(e["lse"].abs().max()) + 2 * (h / 16) ** 0.5 * 2.0 ** -24 * float(z.abs().max()) / 8
        tol = f * abs(float(part.mean())) + 2.0 ** -22 + 4 * noise / m ** 0.5
        print(h, name, mean, rms, tol, float(part.mean()))
        assert abs(mean) <= tol, (name, mean, tol)
        assert rms <= f * float(part.square().mean().sqrt()) + 2.0 ** -22 + noise, (name, rms)
    # d and the result are rounded once each: a relative error of u at most, u / sqrt(3) in the mean square if spread evenly
    u = torch.finfo(dtype).eps / 2
    for name, got in (("dx", dx), ("dw", dw)):
        off = float((got.double() - e[name]).norm() / e[name].norm())
        print(h, name, off / u)
        assert off <= (2.0 / 3.0) ** 0.5 * u + 2e-5, (name, off)
