"""Linear with softmax cross entropy: loss, logsumexp and both gradients against a 64-bit implementation of the formulas.

Tolerances, derived before the first run.  Products of two 16-bit numbers are exact in fp32, so a logit is off by at most
H additions of one unit each, 2^-23 of the running sum of |x w|:  dz = H 2^-23 max sum|x w|.  loss and lse move by at most
2 dz plus a few fp32 units of their own size and of exp / log.  Of the gradients' terms, d = g (p - onehot) moves by
g p (dz + its exponent's rounding), and is rounded once to 16 bits (half a step, u = eps / 2, relative); its products are
summed in fp32 and the result is rounded once more."""
import pytest
import torch

IGNORE = -100
DTYPES = [torch.float16, torch.bfloat16]


def inputs(m, v, h, dtype, seed=0, device="cuda", skip=0.2, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((m, h), generator=gen).to(dtype)
    w = (torch.randn((v, h), generator=gen) * spread / h ** 0.5).to(dtype)
    target = torch.randint(0, v, (m,), generator=gen)
    target[torch.rand((m,), generator=gen) < skip] = IGNORE
    g = torch.rand((m,), generator=gen) + 0.25
    return [t.to(device) for t in (x, w, target, g)]


def exact(x, w, target, g, ignore=IGNORE):
    x, w, g = x.double(), w.double(), g.double()
    z = x @ w.t()
    lse = torch.logsumexp(z, 1)
    kept = target != ignore
    idx = torch.where(kept, target, 0).long().clamp(0, z.shape[1] - 1)
    loss = torch.where(kept, lse - z.gather(1, idx[:, None]).squeeze(1), 0.0)
    p = (z - lse[:, None]).exp()
    hot = torch.zeros_like(p).scatter_(1, idx[:, None], 1.0)
    g = torch.where(kept, g, 0.0)[:, None]
    d = g * (p - hot)
    return {"loss": loss, "lse": lse, "dx": d @ w, "dw": d.t() @ x, "d": d, "gp": g.abs() * p}


def bounds(x, w, e):
    xa, wa = x.double().abs(), w.double().abs()
    h, (m, v) = x.shape[1], e["d"].shape
    dz = h * 2.0 ** -23 * float((xa @ wa.t()).max())
    u = torch.finfo(x.dtype).eps / 2
    tiny = float(torch.finfo(x.dtype).smallest_normal) * torch.finfo(x.dtype).eps      # the step of subnormal outputs
    fwd = 2 * dz + 2.0 ** -20 * (1 + e["lse"].abs())
    dd = e["d"].abs() * (u + 2.0 ** -21) + e["gp"] * (2 * dz + 2.0 ** -20 * (1 + float(e["lse"].abs().max()))) \
        + 2.0 ** -39 * float(e["gp"].sum(1).max())                                      # fp16: d is scaled into its normal range
    bx = dd @ wa + v * 2.0 ** -23 * (e["d"].abs() @ wa) + u * e["dx"].abs() * 1.01 + tiny
    bw = dd.t() @ xa + m * 2.0 ** -23 * (e["d"].abs().t() @ xa) + u * e["dw"].abs() * 1.01 + tiny
    return fwd, bx, bw


def check(api, x, w, target, g, ignore=IGNORE):
    loss, lse = api.linear_cross_entropy(x, w, target, ignore_index=ignore)
    dx, dw = api.linear_cross_entropy_grad(x, w, target, lse, g, ignore_index=ignore)
    assert api.device_status() == 0
    e = exact(x, w, target, g, ignore)
    fwd, bx, bw = bounds(x, w, e)
    assert loss.dtype == lse.dtype == torch.float32 and dx.dtype == x.dtype and dw.dtype == w.dtype
    assert ((lse.double() - e["lse"]).abs() <= fwd).all()
    assert ((loss.double() - e["loss"]).abs() <= fwd).all()
    assert (loss[target == ignore] == 0).all()
    assert ((dx.double() - e["dx"]).abs() <= bx).all(), float(((dx.double() - e["dx"]).abs() / bx).max())
    assert ((dw.double() - e["dw"]).abs() <= bw).all(), float(((dw.double() - e["dw"]).abs() / bw).max())
    return loss, lse, dx, dw


# ---------------------------------------------------------------------------------------------------- refusals (host)
def test_refusals_name_their_argument(api):
    x, w, target, g = inputs(4, 32, 16, torch.float16, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        api.linear_cross_entropy(x, w, target)
    xm, wm = x.to("meta"), w.to("meta")
    for bad in (lambda: api.linear_cross_entropy(xm[0], wm, target), lambda: api.linear_cross_entropy(xm, wm[:, :8], target),
                lambda: api.linear_cross_entropy_grad(x, w, target, g, g)):
        with pytest.raises(ValueError):
            bad()


def test_extents_beyond_32_bits_are_refused(api):
    # 2^32 + 10 entries would reach the library as 10
    big = 2 ** 32 + 10
    meta = lambda *shape, t=torch.float16: torch.empty(shape, dtype=t, device="meta")
    for m, v in ((4, big), (big, 4)):
        x, w, target, g = meta(m, 1), meta(v, 1), meta(m, t=torch.int64), meta(m, t=torch.float32)
        for call in (lambda: api.linear_cross_entropy(x, w, target), lambda: api.linear_cross_entropy_grad(x, w, target, g, g)):
            with pytest.raises(ValueError, match="32 bits"):
                call()


def test_abi_refusals_need_no_gpu(api):
    import ctypes
    L, n = api.lib(), ctypes.c_size_t()
    p = ctypes.c_void_p(4096)
    ok = [api.MP_BF16, 8, 1000, 64, p, 64, p, 64]

    def workspace(**change):
        a = list(ok)
        for k, v in change.items():
            a[["dtype", "M", "V", "H", "X", "ldx", "W", "ldw"].index(k)] = v
        return L.mp_linear_xent_workspace(*a, 0, ctypes.byref(n))
    assert workspace() == 0 and n.value > 0
    for change in (dict(dtype=api.MP_FP32), dict(dtype=api.MP_INT8), dict(M=-1), dict(V=0), dict(H=0), dict(ldx=63), dict(ldw=1),
                   dict(W=ctypes.c_void_p(0)), dict(V=(1 << 30) + 1)):
        assert workspace(**change) == 1, change
    assert workspace(M=0) == 0 and n.value == 0
    # an unaligned row stride asks for room for the aligned copies
    aligned = L.mp_linear_xent_workspace(*ok, 1, ctypes.byref(n)) or n.value
    assert workspace(H=63, ldx=63, ldw=63) == 0
    assert L.mp_linear_xent_workspace(api.MP_BF16, 8, 1000, 63, p, 63, p, 63, 1, ctypes.byref(n)) == 0 and n.value > aligned
    z = ctypes.c_void_p(0)
    tail = [p, 8, -100, p, p]
    assert L.mp_linear_xent(*ok, *tail, z, 0, z) == 5                      # no workspace
    assert L.mp_linear_xent(*ok, *tail, ctypes.c_void_p(4096 + 16), 1 << 30, z) == 5      # unaligned workspace
    assert L.mp_linear_xent(*ok, p, 2, -100, p, p, p, 1 << 30, z) == 1     # targets of another width
    assert L.mp_linear_xent(*ok, p, 8, -100, z, p, p, 1 << 30, z) == 1     # no output
    assert L.mp_linear_xent(*ok, z, 8, -100, p, p, p, 1 << 30, z) == 1
    assert L.mp_linear_xent_grad(*ok, p, 8, -100, z, p, p, p, p, 1 << 30, z) == 1         # no lse
    assert L.mp_linear_xent_grad(*ok, p, 8, -100, p, p, z, z, z, 0, z) == 0               # nothing wanted


# ------------------------------------------------------------------------------------------------------------ results
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,v,h", [(1, 1, 8), (1, 257, 64), (3, 1000, 72), (128, 256, 128), (129, 513, 64), (255, 2047, 200),
                                   (257, 300, 1024), (300, 5003, 264)])
def test_against_64_bits(api, m, v, h, dtype):
    check(api, *inputs(m, v, h, dtype, seed=m + v + h))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_pieces_of_the_vocabulary(api, dtype):
    # 33000 rows: a piece holds 4096 entries, so 9001 entries are three pieces and dx is summed over them
    check(api, *inputs(33000, 9001, 64, dtype, seed=5))


@pytest.mark.gpu
def test_many_pieces_and_slices(api):
    # 1000 rows: a piece holds 131072 entries, so 140001 entries are two pieces, and dx's few tiles are cut into slices of the
    # vocabulary that the short second piece does not fill
    check(api, *inputs(1000, 140001, 64, torch.float16, seed=6))


@pytest.mark.gpu
def test_many_short_units(api):
    # 5 rows: 274 x 6 tiles of dw of one short product each, some twenty for every pair of CTAs, the last of 24 columns
    check(api, *inputs(5, 70013, 1304, torch.bfloat16, seed=12))


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1, 4, 8])
@pytest.mark.parametrize("h", [264, 315, 332])
def test_outputs_keep_to_their_elements(api, h, offset):
    # gradients that start at any element of a larger buffer: the same values, and nothing around them is written
    import ctypes
    m, v = 37, 1003
    x, w, target, g = inputs(m, v, h, torch.float16, seed=h)
    lse = api.linear_cross_entropy(x, w, target)[1]
    want = api.linear_cross_entropy_grad(x, w, target, lse, g)
    bufs = [torch.full((r * h + 64,), 7.0, dtype=x.dtype, device="cuda") for r in (m, v)]
    views = [b[16 + offset:16 + offset + r * h].view(r, h) for b, r in zip(bufs, (m, v))]
    n, p = ctypes.c_size_t(), lambda t: ctypes.c_void_p(t.data_ptr())
    common = [api.MP_FP16, m, v, h, p(x), h, p(w), h]
    assert api.lib().mp_linear_xent_workspace(*common, 1, ctypes.byref(n)) == 0
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert api.lib().mp_linear_xent_grad(*common, p(target), 8, IGNORE, p(lse), p(g), p(views[0]), p(views[1]), p(ws), n.value, stream) == 0
    torch.cuda.synchronize()
    for b, t, r, e in zip(bufs, views, (m, v), want):
        assert torch.equal(t, e)
        assert (b[:16 + offset] == 7.0).all() and (b[16 + offset + r * h:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("h", [1, 7, 63, 100, 333])
def test_rows_that_miss_16_bytes(api, h):
    check(api, *inputs(37, 400, h, torch.bfloat16, seed=h))


@pytest.mark.gpu
def test_strides_and_offsets(api):
    x, w, target, g = inputs(70, 500, 136, torch.float16, seed=3)
    want = check(api, x, w, target, g)
    wide = torch.randn(70, 200, device="cuda", dtype=torch.float16)
    wide[:, 8:144] = x
    wide_w = torch.randn(500, 144, device="cuda", dtype=torch.float16)
    wide_w[:, 8:] = w
    odd = torch.empty(70 * 136 + 1, device="cuda", dtype=torch.float16)[1:].view(70, 136).copy_(x)       # base off by 2 bytes
    for xx, ww in ((wide[:, 8:144], wide_w[:, 8:]), (x.t().contiguous().t(), w.t().contiguous().t()), (odd, w)):
        got = check(api, xx, ww, target.int(), g)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    one = x[:1].expand(70, 136)                       # rows that share their memory
    check(api, one, w, target, g)


@pytest.mark.gpu
@pytest.mark.parametrize("ignore", [-100, -1, 3, 10 ** 12])
def test_ignored_and_impossible_targets(api, ignore):
    x, w, target, g = inputs(40, 100, 64, torch.bfloat16, seed=9, skip=0.0)
    if ignore == 3:
        target[target == 3] = 4                       # an entry that doubles as the mark
    target[::4] = ignore
    g[::4] = float("nan")                             # never looked at
    loss, lse, dx, dw = check(api, x, w, target, torch.where(target == ignore, 0.0, g), ignore)
    dx2, dw2 = api.linear_cross_entropy_grad(x, w, target, lse, g, ignore_index=ignore)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and (dx[::4] == 0).all()
    # all rows ignored
    target[:] = ignore
    loss, lse = api.linear_cross_entropy(x, w, target, ignore_index=ignore)
    dx, dw = api.linear_cross_entropy_grad(x, w, target, lse, g, ignore_index=ignore)
    assert (loss == 0).all() and torch.isfinite(lse).all() and (dx == 0).all() and (dw == 0).all()
    # a target that is no entry: NaN in its own row, the others untouched
    target[:] = 5
    want, _ = api.linear_cross_entropy(x, w, target, ignore_index=ignore)
    for bad in (100, 101, 255, -7, 2 ** 40):
        target[11] = bad
        loss, lse = api.linear_cross_entropy(x, w, target, ignore_index=ignore)
        assert torch.isnan(loss[11]) and torch.isfinite(lse).all()
        assert torch.equal(loss[:11], want[:11]) and torch.equal(loss[12:], want[12:])
        dx, dw = api.linear_cross_entropy_grad(x, w, target, lse, g.nan_to_num(1.0), ignore_index=ignore)
        assert torch.isnan(dx[11]).all() and torch.isfinite(dx[:11]).all() and torch.isfinite(dx[12:]).all()


@pytest.mark.gpu
def test_infinities(api):
    x, w, target, g = inputs(8, 300, 64, torch.bfloat16, seed=2, skip=0.0)
    x[:] = x.abs() + 0.5
    w[7] = float("-inf")                               # an entry that is masked out
    w[299] = float("-inf")
    target[:] = 100
    loss, lse = api.linear_cross_entropy(x, w, target)
    z = x.double() @ w.double().t()
    assert torch.allclose(lse.double(), torch.logsumexp(z, 1), atol=1e-4)
    target[0] = 7
    loss, _ = api.linear_cross_entropy(x, w, target)
    assert torch.isinf(loss[0]) and loss[0] > 0 and torch.isfinite(loss[1:]).all()
    w[:] = float("-inf")                               # nothing left in any row
    _, lse = api.linear_cross_entropy(x, w, target)
    assert (lse == float("-inf")).all()
    w[:] = 0
    w[3] = float("inf")
    _, lse = api.linear_cross_entropy(x, w, target)
    assert (lse == float("inf")).all()
    w[3] = float("nan")
    loss, lse = api.linear_cross_entropy(x, w, target)
    assert torch.isnan(lse).all() and torch.isnan(loss).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_confident_rows_and_large_logits(api, dtype):
    x, w, target, g = inputs(64, 777, 64, dtype, seed=4, skip=0.0, spread=1.0)
    w[target] = x / 2                                  # the target's logit is far above the rest
    check(api, x, w, target, g)
    x = (x.float() * 8).to(dtype)
    check(api, x, w, target, g * 1e-6)


@pytest.mark.gpu
def test_upstream_gradients_of_every_size(api):
    x, w, target, g = inputs(50, 300, 64, torch.float16, seed=6, skip=0.0)
    for scale in (0.0, 1e-9, 1.0 / 50, 1e4):
        loss, lse = api.linear_cross_entropy(x, w, target)
        dx, dw = api.linear_cross_entropy_grad(x, w, target, lse, torch.full_like(g, scale))
        e = exact(x, w, target, torch.full_like(g, scale))
        _, bx, bw = bounds(x, w, e)
        assert ((dx.double() - e["dx"]).abs() <= bx).all() and ((dw.double() - e["dw"]).abs() <= bw).all()
    g[3] = float("inf")
    dx, _ = api.linear_cross_entropy_grad(x, w, target, lse, g, need_dw=False)
    assert not torch.isfinite(dx[3]).any() and torch.isfinite(dx[4:]).all()


@pytest.mark.gpu
def test_either_gradient_alone_and_no_tokens(api):
    x, w, target, g = inputs(90, 700, 72, torch.bfloat16, seed=8)
    loss, lse, dx, dw = check(api, x, w, target, g)
    only_x, none = api.linear_cross_entropy_grad(x, w, target, lse, g, need_dw=False)
    assert none is None and torch.equal(only_x, dx)
    none, only_w = api.linear_cross_entropy_grad(x, w, target, lse, g, need_dx=False)
    assert none is None and torch.equal(only_w, dw)
    assert api.linear_cross_entropy_grad(x, w, target, lse, g, need_dx=False, need_dw=False) == (None, None)
    e = x[:0]
    loss, lse = api.linear_cross_entropy(e, w, target[:0])
    dx, dw = api.linear_cross_entropy_grad(e, w, target[:0], lse, g[:0])
    assert loss.shape == lse.shape == (0,) and dx.shape == (0, 72) and (dw == 0).all() and dw.shape == w.shape


@pytest.mark.gpu
def test_gradient_against_differences(api):
    # central differences of the 64-bit loss along random directions, against the returned gradients
    x, w, target, g = inputs(33, 211, 64, torch.bfloat16, seed=12)
    loss, lse, dx, dw = check(api, x, w, target, g)
    gen = torch.Generator().manual_seed(1)
    for t, d in (("x", dx), ("w", dw)):
        u = torch.randn(d.shape, generator=gen).cuda().double()
        eps = 1e-5

        def total(sign):
            xx, ww = x.double() + sign * eps * u if t == "x" else x.double(), w.double() + sign * eps * u if t == "w" else w.double()
            return (exact(xx, ww, target, g)["loss"] * g.double()).sum()
        slope = float((total(1) - total(-1)) / (2 * eps))
        # the gradient's own rounding: u |d| per element, against a random direction
        assert abs(slope - float((d.double() * u).sum())) <= 3 * 2.0 ** -8 * float((d.double() * u).norm()) + 1e-6


@pytest.mark.gpu
def test_other_streams_and_captured_graphs(api):
    x, w, target, g = inputs(200, 3000, 128, torch.bfloat16, seed=20)
    want = check(api, x, w, target, g)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (s1, s2):                                 # two calls at once
        with torch.cuda.stream(s):
            loss, lse = api.linear_cross_entropy(x, w, target)
            outs.append((loss, lse) + api.linear_cross_entropy_grad(x, w, target, lse, g))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            loss, lse = api.linear_cross_entropy(x, w, target)
            outs.append((loss, lse) + api.linear_cross_entropy_grad(x, w, target, lse, g))
        graphs.append(gr)
    for _ in range(3):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for gr, s in zip(graphs, (s1, s2)):            # replayed side by side
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, want))
    assert api.device_status() == 0
