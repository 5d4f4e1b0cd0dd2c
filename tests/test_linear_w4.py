"""Linear with 4-bit weights and the gradient of its input, against 64-bit products of the unpacked weight.

Tolerances, derived before the first run.  x * (q - zero) and (q - zero) * scale are exact before rounding.  fp32 sums of C
terms: at most C steps of 2^-23 of sum |x w|.  The result is rounded once (half a step: u = eps / 2, relative).  Where the
weight itself is rounded to 16 bits (more than 16 tokens, and the gradient) every term moves by u, or by half a subnormal
step of the type."""
import ctypes

import pytest
import torch

DTYPES = [torch.float16, torch.bfloat16]


def make(n, k, group, dtype, zeros=True, seed=0, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.uint8)
    groups = -(-k // group)
    s = (torch.rand((n, groups), generator=gen) * 0.02 + 0.002).to(dtype)
    z = torch.randint(0, 17, (n, groups), generator=gen, dtype=torch.uint8) if zeros else None
    return [None if t is None else t.to(device) for t in (q, s, z)]


def weight(q, s, z, group):
    each = torch.arange(q.shape[1], device=q.device) // group
    return (q.double() - (8.0 if z is None else z.double()[:, each])) * s.double()[:, each]


def within(got, x, w, bias, rounded_weight):
    """got against x @ w.T (+ bias) in 64 bits."""
    xd = x.double()
    want, size = xd @ w.t(), xd.abs() @ w.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    info = torch.finfo(got.dtype)
    u, sub = info.eps / 2, float(info.smallest_normal) * info.eps / 2
    tol = w.shape[1] * 2.0 ** -23 * size + 1.01 * u * want.abs() + sub
    if rounded_weight:
        tol = tol + u * size + sub * xd.abs().sum(1, keepdim=True)
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (off <= tol).all(), (float((off / tol).max()), int((off > tol).sum()))


def tokens(m, k, dtype, seed=1):
    return torch.randn((m, k), generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# ---------------------------------------------------------------------------------------------------- refusals (host)
def test_refusals_need_no_gpu(api):
    L, p, z, n = api.lib(), ctypes.c_void_p(4096), ctypes.c_void_p(0), ctypes.c_size_t()

    def fwd(dtype=api.MP_FP16, M=64, N=64, K=64, X=p, ldx=64, W=p, S=p, Z=z, group=32, Y=p, ws=p, size=1 << 30):
        return L.mp_linear_w4(dtype, M, N, K, X, ldx, W, S, Z, group, z, Y, ws, size, z)
    for change in (dict(dtype=api.MP_FP32), dict(dtype=api.MP_INT8), dict(M=-1), dict(N=0), dict(K=0), dict(ldx=63), dict(X=z),
                   dict(W=z), dict(S=z), dict(group=16), dict(group=48), dict(group=0), dict(group=-1), dict(Y=z),
                   dict(W=ctypes.c_void_p(4104))):
        assert fwd(**change) == 1, change
    assert fwd(K=48) == 3                                                 # not a multiple of 32
    assert fwd(M=0) == 0
    assert fwd(M=40, K=4096, ldx=4096, ws=z, size=0) == 5                 # split sums need room
    assert L.mp_linear_w4_workspace(40, 64, 4096, 32, p, 4096, 0, ctypes.byref(n)) == 0 and n.value > 0
    assert fwd(M=40, K=4096, ldx=4096, size=n.value - 1) == 5 and fwd(M=40, K=4096, ldx=4096, ws=ctypes.c_void_p(4096 + 64)) == 5
    assert L.mp_linear_w4_workspace(1, 64, 4096, 32, p, 4096, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert L.mp_linear_w4_workspace(1, 64, 4096, 32, p, 4097, 0, ctypes.byref(n)) == 0 and n.value > 0      # an aligned copy
    assert L.mp_linear_w4_workspace(1, 64, 4096, 32, p, 4096, 0, None) == 1
    assert L.mp_w4_pack(4, 64, z, 64, p, z) == 1 and L.mp_w4_pack(4, 64, p, 63, p, z) == 1 and L.mp_w4_pack(0, 64, z, 64, z, z) == 0


def test_argument_checks(api):
    x = torch.zeros((2, 64), dtype=torch.float16)
    w, s = torch.zeros((8, 16), dtype=torch.int32), torch.zeros((8, 2), dtype=torch.float16)
    for call in (lambda: api.linear_w4(x[0], w, s, group_size=32), lambda: api.linear_w4(x.float(), w, s, group_size=32),
                 lambda: api.linear_w4(x, w[:, :8], s, group_size=32), lambda: api.linear_w4(x, w, s, group_size=64),
                 lambda: api.linear_w4(x, w, s.bfloat16(), group_size=32), lambda: api.linear_w4(x, w, s, s, group_size=32),
                 lambda: api.linear_w4(x[:, :48], w, s, group_size=32), lambda: api.linear_w4(x, w, s, group_size=24),
                 lambda: api.linear_w4(x, w, s, group_size=32), lambda: api.pack_w4(torch.zeros((8, 64), dtype=torch.uint8)),
                 lambda: api.linear_w4_grad_input(x, w, s, group_size=32)):
        with pytest.raises(ValueError):
            call()


def test_extents_above_the_limit_are_refused(api):
    L, p, z, n, big = api.lib(), ctypes.c_void_p(4096), ctypes.c_void_p(0), ctypes.c_size_t(), (1 << 28) + 32
    assert L.mp_w4_pack(1, big, p, big, p, z) == 1 and L.mp_w4_pack(big, 1, p, 1, p, z) == 1
    for m, rows, k in ((big, 8, 64), (8, big, 64), (8, 8, big)):
        assert L.mp_linear_w4_workspace(m, rows, k, 32, p, k, 0, ctypes.byref(n)) == 1


def test_extents_beyond_32_bits_are_refused(api):
    # 2^32 + 8 rows would reach the library as 8
    big = 2 ** 32 + 8
    meta = lambda *shape, t=torch.float16: torch.empty(shape, dtype=t, device="meta")
    w, s = meta(8, 16, t=torch.int32), meta(8, 2)
    for call in (lambda: api.linear_w4(meta(big, 64), w, s, group_size=32), lambda: api.linear_w4(meta(2, 64), meta(big, 16, t=torch.int32), meta(big, 2), group_size=32),
                 lambda: api.linear_w4(meta(2, 64), w, meta(8, 1), group_size=2 ** 40), lambda: api.linear_w4_grad_input(meta(big, 8), w, s, group_size=32, in_features=64),
                 lambda: api.pack_w4(meta(big, 1, t=torch.uint8))):
        with pytest.raises(ValueError, match="32 bits"):
            call()


# ------------------------------------------------------------------------------------------------------------ results
@pytest.mark.gpu
@pytest.mark.parametrize("n,k", [(1, 32), (3, 160), (17, 128), (64, 4096), (5, 100), (2, 1)])
def test_packed_layout(api, n, k):
    q = torch.randint(0, 16, (n, k), dtype=torch.uint8, device="cuda")
    got = api.pack_w4(q).cpu().to(torch.int64) & 0xFFFFFFFF
    full = torch.zeros((n, -(-k // 128) * 128), dtype=torch.int64)
    full[:, :k] = q.cpu()
    for b in range(full.shape[1] // 128):
        for t in range(4):
            for i in range(4):
                word = sum(full[:, b * 128 + 32 * i + 8 * t + e] << (4 * (e // 2) + 16 * (e % 2)) for e in range(8))
                assert torch.equal(got[:, b * 16 + 4 * t + i], word)
    assert torch.equal(api.pack_w4(q + 16), api.pack_w4(q))              # the low four bits count
    wide = torch.randint(0, 16, (n, k + 7), dtype=torch.uint8, device="cuda")
    assert torch.equal(api.pack_w4(wide[:, 3:3 + k]), api.pack_w4(wide[:, 3:3 + k].contiguous()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("m", [1, 2, 8, 9, 16, 17, 32, 33, 65, 130, 300])
def test_forward_against_64_bits(api, m, group, dtype):
    n, k = (200, 544) if m % 2 else (129, 1024)                          # 544 = 4 blocks and one run of 32
    q, s, z = make(n, k, group, dtype, zeros=m % 3 != 0, seed=m)
    x = tokens(m, k, dtype)
    bias = torch.randn(n, device="cuda").to(dtype) if m % 2 else None
    y = api.linear_w4(x, api.pack_w4(q), s, z, group_size=group, bias=bias)
    assert api.device_status() == 0
    within(y, x, weight(q, s, z, group), bias, m > 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,group", [(1, 1, 32, 32), (5, 37, 96, 32), (40, 1, 32, 32), (33, 9473, 256, 64), (1, 9500, 256, 128),
                                         (20, 9500, 160, 32), (257, 515, 2080, 128), (64, 300, 4096, -1), (3, 300, 4096, -1), (700, 260, 288, 32),
                                         (1, 40, 80000, 32), (16, 70000, 64, 32), (3, 30000, 2048, 32), (9, 2400, 1056, 64)])
def test_forward_sizes(api, m, n, k, group, dtype):
    real = group if group > 0 else 4096
    q, s, z = make(n, k, real, dtype, seed=n)
    x = tokens(m, k, dtype)
    y = api.linear_w4(x, api.pack_w4(q), s, z, group_size=group)
    assert api.device_status() == 0
    within(y, x, weight(q, s, z, real), None, m > 16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k,group", [(1, 1, 32, 32), (1, 300, 544, 128), (7, 129, 96, 32), (33, 1000, 4096, 64), (65, 127, 160, 128),
                                         (130, 515, 608, 32), (300, 2049, 1056, 256), (1001, 130, 288, 128), (2, 4100, 64, 64)])
def test_gradient_against_64_bits(api, m, n, k, group, dtype):
    q, s, z = make(n, k, group, dtype, zeros=n % 2 == 1, seed=k)
    dy = tokens(m, n, dtype)
    dx = api.linear_w4_grad_input(dy, api.pack_w4(q), s, z, group_size=group, in_features=k)
    assert api.device_status() == 0 and dx.shape == (m, k)
    within(dx, dy, weight(q, s, z, group).t(), None, True)


@pytest.mark.gpu
def test_gradient_against_differences(api):
    q, s, z = make(96, 256, 64, torch.float16, seed=3)
    x, dy, u = tokens(40, 256, torch.float16, 1), tokens(40, 96, torch.float16, 2), tokens(40, 256, torch.float16, 3).double()
    dx = api.linear_w4_grad_input(dy, api.pack_w4(q), s, z, group_size=64)
    w = weight(q, s, z, 64)
    slope = float((((x.double() + u) @ w.t() - (x.double() - u) @ w.t()) * dy.double()).sum() / 2)       # linear: exact differences
    # each dx is off by u (sum |dy w| + |dx|) at most, at random signs along u
    off = 2 * 2.0 ** -11 * float(((dy.double().abs() @ w.abs()) * u.abs()).norm()) * 4
    assert abs(slope - float((dx.double() * u).sum())) <= off


@pytest.mark.gpu
def test_strides_offsets_and_no_tokens(api):
    q, s, z = make(70, 192, 64, torch.bfloat16, seed=5)
    pw = api.pack_w4(q)
    for m in (3, 50):
        x = tokens(m, 192, torch.bfloat16)
        want = api.linear_w4(x, pw, s, z, group_size=64)
        wide = torch.randn(m, 300, device="cuda").bfloat16()
        wide[:, 8:200] = x
        odd = torch.empty(m * 192 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(m, 192).copy_(x)
        shifted = torch.empty(pw.numel() + 1, dtype=torch.int32, device="cuda")[1:].view_as(pw).copy_(pw)
        for xx, ww in ((wide[:, 8:200], pw), (odd, pw), (x.t().contiguous().t(), pw), (x, shifted)):
            assert torch.equal(api.linear_w4(xx, ww, s, z, group_size=64), want)
        assert torch.equal(api.linear_w4(x, pw, s.t().contiguous().t(), z.t().contiguous().t(), group_size=64), want)
        assert torch.equal(api.linear_w4(x[:1].expand(m, 192), pw, s, z, group_size=64)[0], api.linear_w4(x[:1].expand(m, 192).contiguous(), pw, s, z, group_size=64)[0])
    assert api.linear_w4(x[:0], pw, s, z, group_size=64).shape == (0, 70)
    assert api.linear_w4_grad_input(tokens(4, 70, torch.bfloat16)[:0], pw, s, z, group_size=64, in_features=192).shape == (0, 192)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 100])
def test_padding_bits_and_rows_behind_the_end(api, m):
    # bits behind K and memory behind the last row and token must not reach the result, nor be written
    q, s, z = make(33, 160, 32, torch.float16, seed=8)
    pw = api.pack_w4(q)
    x = tokens(m, 160, torch.float16)
    want = api.linear_w4(x, pw, s, z, group_size=32)
    dy = tokens(m, 33, torch.float16)
    dwant = api.linear_w4_grad_input(dy, pw, s, z, group_size=32, in_features=160)
    dirty = pw.clone().view(33, 2, 4, 4)
    dirty[:, 1, :, 1:] = -1                                              # runs 1..3 of the second block do not exist
    dirty = dirty.view_as(pw)
    assert torch.equal(api.linear_w4(x, dirty, s, z, group_size=32), want)
    assert torch.equal(api.linear_w4_grad_input(dy, dirty, s, z, group_size=32, in_features=160), dwant)
    big = torch.full((m + 5, 168), float("nan"), device="cuda", dtype=torch.float16)
    big[:m, :160] = x
    assert torch.equal(api.linear_w4(big[:m, :160], pw, s, z, group_size=32), want)
    out = torch.full((m + 2, 33), 7.0, device="cuda", dtype=torch.float16)
    L, n = api.lib(), ctypes.c_size_t()
    assert L.mp_linear_w4_workspace(m, 33, 160, 32, ctypes.c_void_p(x.data_ptr()), 160, 0, ctypes.byref(n)) == 0
    ws = torch.empty(n.value + 256, dtype=torch.uint8, device="cuda")
    api._check(L.mp_linear_w4(api.MP_FP16, m, 33, 160, x.data_ptr(), 160, pw.data_ptr(), s.data_ptr(), z.data_ptr(), 32, None, out.data_ptr(),
                              ws.data_ptr(), n.value, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert torch.equal(out[:m], want) and (out[m:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 48])
def test_infinite_and_nan_tokens_stay_in_their_rows(api, m):
    q, s, z = make(40, 160, 32, torch.bfloat16, seed=9)
    pw, x = api.pack_w4(q), tokens(m, 160, torch.bfloat16)
    want = api.linear_w4(x, pw, s, z, group_size=32)
    x[1, 5] = float("nan")
    y = api.linear_w4(x, pw, s, z, group_size=32)
    assert torch.isnan(y[1]).all() and torch.equal(y[:1], want[:1]) and torch.equal(y[2:], want[2:])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 90])
def test_other_streams_and_captured_graphs(api, m):
    q, s, z = make(520, 4096, 128, torch.float16, seed=10)
    pw, x, dy = api.pack_w4(q), tokens(m, 4096, torch.float16), tokens(m, 520, torch.float16)

    def both():
        return api.linear_w4(x, pw, s, z), api.linear_w4_grad_input(dy, pw, s, z)
    want = both()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append(both())
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(both())
        graphs.append(gr)
    for _ in range(3):
        for gr, st in zip(graphs, streams):                              # two graphs side by side
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    assert api.device_status() == 0
