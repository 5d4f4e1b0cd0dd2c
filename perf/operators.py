"""Cases of the 4-bit Linear and of the Linear with a softmax cross entropy: their inputs, a plain form in elementary
torch operations, the exact values in 64 bits, and the calls a user makes.

The 4-bit weight format (`qweight`, int32 [N, 16 * ceil(K / 128)]): every row is cut into blocks of 128 weights, a block
is 16 words, and word 4 t + i of a block holds the 8 weights k = 32 i + 8 t ... + 7 of the block, weight 2 j in bits
4 j ... 4 j + 3 and weight 2 j + 1 in bits 16 + 4 j ... 19 + 4 j.  A weight is (q - zero) * scale with one scale (and
zero, 8 where none is given) for every `group` consecutive k of a row."""
import math
import os
import sys

import torch

own = False

IGNORE = -100          # target of a token that has no loss (padding, prompt tokens)
_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoded token through a square projection: the smallest call, latency counts
        dict(name="w4_m1_4096x4096", op="w4", m=1, n=4096, k=4096, group=128, zeros=False, bias=False, dtype="fp16"),
        # a small decode batch through the widest projection, asymmetric weights
        dict(name="w4_m4_28672x4096", op="w4", m=4, n=28672, k=4096, group=64, zeros=True, bias=False, dtype="bf16"),
        # a ragged decode batch through the down projection with the finest groups and a bias
        dict(name="w4_m37_4096x14336", op="w4", m=37, n=4096, k=14336, group=32, zeros=True, bias=True, dtype="fp16"),
        # a short prompt or a large decode batch
        dict(name="w4_m200_6144x4096", op="w4", m=200, n=6144, k=4096, group=128, zeros=False, bias=False, dtype="bf16"),
        # a prefill chunk with an odd number of tokens
        dict(name="w4_m2047_28672x4096", op="w4", m=2047, n=28672, k=4096, group=128, zeros=True, bias=False, dtype="fp16"),
        # the gradient that a frozen 4-bit projection hands back, an odd batch
        dict(name="w4_grad_m1001_4096x14336", op="w4_grad", m=1001, n=4096, k=14336, group=128, zeros=True, bias=False, dtype="bf16"),
        # the same for a full training batch and the widest projection
        dict(name="w4_grad_m4096_28672x4096", op="w4_grad", m=4096, n=28672, k=4096, group=64, zeros=False, bias=False, dtype="fp16"),
        # the log-probability of one decoded token over an odd vocabulary
        dict(name="xent_m1_v50021", op="xent", m=1, v=50021, h=4096, skip=0.0, dtype="bf16"),
        # scoring a prompt, part of it without a loss
        dict(name="xent_m1023_v32768", op="xent", m=1023, v=32768, h=4096, skip=0.25, dtype="fp16"),
        # tuning with a frozen output layer: the loss and the hidden states' gradient, ragged on every side
        dict(name="xent_dx_m300_v50021", op="xent_train", m=300, v=50021, h=2040, skip=0.5, dw=False, dtype="fp16"),
        # a training step of a small model: loss and both gradients
        dict(name="xent_train_m2048_v32768", op="xent_train", m=2048, v=32768, h=1024, skip=0.1, dw=True, dtype="bf16"),
        # a training step's largest call: a full batch over a large vocabulary
        dict(name="xent_train_m4096_v131072", op="xent_train", m=4096, v=131072, h=4096, skip=0.0, dw=True, dtype="bf16"),
    ]


def _between(rng, lo, hi):
    """A whole number whose logarithm is spread evenly over the range."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["w4", "w4", "w4_grad", "xent", "xent_train", "xent_train"])
    dtype = rng.choice(["fp16", "bf16"])
    if op in ("w4", "w4_grad"):
        m = _between(rng, 1, 4096)
        n = _between(rng, 256, 28672)
        k = 32 * _between(rng, 8, 448)
        return dict(op=op, m=m, n=n, k=k, group=rng.choice([32, 64, 128, 128, 256]), zeros=rng.random() < 0.5,
                    bias=op == "w4" and rng.random() < 0.3, dtype=dtype)
    m = _between(rng, 1, 4096)
    v = _between(rng, 1000, 131072)
    h = 8 * _between(rng, 32, 512)
    case = dict(op=op, m=m, v=v, h=h, skip=rng.choice([0.0, 0.1, 0.5]), dtype=dtype)
    if op == "xent_train":
        case["dw"] = rng.random() < 0.7
    return case


def work(case):
    m = case["m"]
    if case["op"] in ("w4", "w4_grad"):
        n, k, groups = case["n"], case["k"], -(-case["k"] // case["group"])
        weight = n * k // 2 + n * groups * (3 if case["zeros"] else 2)
        return {"bytes": weight + 2 * m * (n + k) + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    v, h = case["v"], case["h"]
    read = 2 * h * (m + v) + 16 * m                    # hidden states, weight, targets, loss and normaliser
    if case["op"] == "xent":
        return {"bytes": read, "flops": 2 * m * v * h}
    # the logits' product, the hidden states' gradient and, where it is wanted, the weight's
    return {"bytes": read + 4 * m + 2 * h * m + (2 * h * v if case["dw"] else 0), "flops": (6 if case["dw"] else 4) * m * v * h}


# ----------------------------------------------------------------------------------------------------------- inputs
def _pack(q):
    """q [N, K] of whole numbers 0 ... 15 -> the int32 words described above."""
    n, k = q.shape
    blocks = -(-k // 128)
    full = torch.zeros((n, blocks * 128), dtype=torch.int64, device=q.device)
    full[:, :k] = q
    full = full.view(n, blocks, 4, 4, 4, 2)                        # [row, block, i, t, j, odd]
    shift = torch.tensor([[4 * j, 16 + 4 * j] for j in range(4)], device=q.device)
    words = (full << shift).sum(dim=(4, 5)).transpose(2, 3)        # [row, block, t, i]
    words = torch.where(words >= 1 << 31, words - (1 << 32), words)
    return words.to(torch.int32).reshape(n, blocks * 16)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = _DT[case["dtype"]]
    m = case["m"]

    def normal(shape, std):
        return torch.empty(shape, dtype=torch.float32, device=dev).normal_(0.0, std, generator=gen)

    if case["op"] in ("w4", "w4_grad"):
        n, k, group = case["n"], case["k"], case["group"]
        groups = -(-k // group)
        # a weight of a projection, quantised group by group as a checkpoint holds it
        q = (normal((n, k), 2.6) + 8.0).round_().clamp_(0, 15).to(torch.uint8)
        state = {"case": case, "qweight": _pack(q), "group": group, "k": k, "bias": None, "zeros": None}
        state["scales"] = (normal((n, groups), 0.001).abs_() + 0.006).to(dt)
        if case["zeros"]:
            state["zeros"] = torch.randint(5, 11, (n, groups), dtype=torch.uint8, device=dev, generator=gen)
        if case["bias"]:
            state["bias"] = normal((n,), 0.5).to(dt)
        state["x"] = normal((m, k if case["op"] == "w4" else n), 1.0).to(dt)
        return state
    v, h = case["v"], case["h"]
    state = {"case": case, "x": normal((m, h), 1.0).to(dt), "w": normal((v, h), 2.0 / math.sqrt(h)).to(dt)}
    target = torch.randint(0, v, (m,), device=dev, generator=gen)
    skip = torch.rand((m,), device=dev, generator=gen) < case["skip"]
    state["target"] = torch.where(skip, torch.full_like(target, IGNORE), target)
    if case["op"] == "xent_train":
        # the mean over the tokens that have a loss, each with a weight of its own
        kept = (~skip).float()
        weight = 0.5 + torch.rand((m,), device=dev, generator=gen)
        state["grad_loss"] = weight * kept / kept.sum().clamp(min=1.0)
    return state


# ------------------------------------------------------------------------------------------------------- plain form
def _unpack(qweight, k):
    """The whole numbers 0 ... 15 of the packed words, [N, K]."""
    n = qweight.shape[0]
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32, device=qweight.device)
    nib = (qweight.view(n, -1, 4, 4, 1) >> shift) & 15             # [row, block, t, i, weight]
    return nib.transpose(2, 3).reshape(n, -1)[:, :k]


def _weight(s):
    q = _unpack(s["qweight"], s["k"]).float()
    each = torch.arange(s["k"], device=q.device) // s["group"]     # the group of every k
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[:, each]
    return (q - zero) * s["scales"].float()[:, each]


def _plain(s):
    case, x = s["case"], s["x"]
    if case["op"] == "w4":
        y = x.float() @ _weight(s).t()
        if s["bias"] is not None:
            y = y + s["bias"].float()
        return y.to(x.dtype)
    if case["op"] == "w4_grad":
        return (x.float() @ _weight(s)).to(x.dtype)
    w, target = s["w"], s["target"]
    kept = target != IGNORE
    safe = torch.where(kept, target, torch.zeros_like(target))
    logits = x.float() @ w.float().t()
    top = logits.amax(dim=1, keepdim=True)
    e = (logits - top).exp()
    total = e.sum(dim=1, keepdim=True)
    lse = (top + total.log()).squeeze(1)
    loss = total.log().squeeze(1) + (top - logits.gather(1, safe[:, None])).squeeze(1)
    loss = torch.where(kept, loss, torch.zeros_like(loss))
    if case["op"] == "xent":
        return {"loss": loss, "lse": lse}
    d = e / total
    d.scatter_add_(1, safe[:, None], torch.full_like(total, -1.0))
    d = d * torch.where(kept, s["grad_loss"], torch.zeros_like(lse))[:, None]
    out = {"loss": loss, "lse": lse, "dx": (d @ w.float()).to(x.dtype)}
    if case["dw"]:
        out["dw"] = (d.t() @ x.float()).to(w.dtype)
    return out


# ------------------------------------------------------------------------------------------------------------- runs
def _api():
    path = os.path.abspath(os.path.join("moonpoly-dev_b200", "py"))
    if path not in sys.path:
        sys.path.insert(0, path)
    from moonpoly_b200 import api
    return api


def run(state):
    if not own:
        return _plain(state)
    api, case, s = _api(), state["case"], state
    if case["op"] == "w4":
        return api.linear_w4(s["x"], s["qweight"], s["scales"], s["zeros"], group_size=s["group"], bias=s["bias"])
    if case["op"] == "w4_grad":
        return api.linear_w4_grad_input(s["x"], s["qweight"], s["scales"], s["zeros"], group_size=s["group"], in_features=s["k"])
    loss, lse = api.linear_cross_entropy(s["x"], s["w"], s["target"], ignore_index=IGNORE)
    if case["op"] == "xent":
        return {"loss": loss, "lse": lse}
    dx, dw = api.linear_cross_entropy_grad(s["x"], s["w"], s["target"], lse, s["grad_loss"], ignore_index=IGNORE,
                                           need_dw=case["dw"])
    out = {"loss": loss, "lse": lse, "dx": dx}
    if case["dw"]:
        out["dw"] = dw
    return out


# ------------------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] in ("w4", "w4_grad"):
        n, k, group = case["n"], case["k"], case["group"]
        words = s["qweight"].to(torch.int64) & 0xFFFFFFFF
        w = torch.empty((n, words.shape[1] * 8), dtype=torch.float64, device=x.device)
        for pos in range(16):                                      # word `pos` of every block of 128
            base = 32 * (pos % 4) + 8 * (pos // 4)
            for e in range(8):                                     # weight e of the word
                w[:, base + e::128] = ((words[:, pos::16] >> (4 * (e // 2) + 16 * (e % 2))) & 15).double()
        w = w[:, :k].clone()
        for g in range(-(-k // group)):
            zero = 8.0 if s["zeros"] is None else s["zeros"][:, g:g + 1].double()
            part = w[:, g * group:(g + 1) * group]
            part.sub_(zero).mul_(s["scales"][:, g:g + 1].double())
        if case["op"] == "w4_grad":
            return torch.matmul(x, w)
        y = torch.matmul(x, w.t())
        return y if s["bias"] is None else y + s["bias"].double()
    w = s["w"].double()
    z = torch.matmul(x, w.t())
    lse = torch.logsumexp(z, dim=1)
    rows = torch.arange(case["m"], device=x.device)
    kept = s["target"] >= 0
    loss = torch.zeros_like(lse)
    loss[kept] = lse[kept] - z[rows[kept], s["target"][kept]]
    out = {"loss": loss, "lse": lse}
    if case["op"] == "xent_train":
        g = s["grad_loss"].double()
        g[~kept] = 0.0
        z.sub_(lse[:, None]).exp_()
        z[rows[kept], s["target"][kept]] -= 1.0
        z.mul_(g[:, None])
        out["dx"] = torch.matmul(z, w)
        if case["dw"]:
            out["dw"] = torch.matmul(z.t(), x)
    return out
