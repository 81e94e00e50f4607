"""Microscaled 4-bit floating point (MXFP4) and the balance of a router's experts, as cases to be timed.

MXFP4: 32 consecutive values along the last dimension share a scale 2**(byte - 127); a value is an e2m1 code
(sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two codes in a byte, the even index in
the low four bits.

* ``quantize``: a tensor to MXFP4 and back, as the values that the codes stand for;
* ``gemm``: a linear layer with MXFP4 weights; its 16-bit input is quantised on the way in;
* ``moe``: the gated MLP of a mixture of experts with MXFP4 stacks, the routing given;
* ``balance``: the load-balancing loss of a router with the routes per expert, and the logits' gradient.
"""
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _quantize(name, rows, cols, dtype):
    return {"name": name, "kind": "quantize", "rows": rows, "cols": cols, "dtype": dtype}


def _gemm(name, m, n, k, dtype="bf16", bias=False):
    return {"name": name, "kind": "gemm", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias}


def _moe(name, tokens, experts=64, topk=8, hidden=2048, inter=1024, dtype="bf16", activation="silu"):
    return {"name": name, "kind": "moe", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "inter": inter,
            "dtype": dtype, "activation": activation}


def _balance(name, tokens, experts, topk, dtype, grad, padding):
    return {"name": name, "kind": "balance", "tokens": tokens, "experts": experts, "topk": topk, "dtype": dtype, "grad": grad,
            "padding": padding}


def listed():
    return [
        # the activations of a long prompt in front of the down projection
        _quantize("quantize-prompt", 2048, 12288, "bf16"),
        # one projection of a 32-bit checkpoint, converted when it is loaded; an odd number of blocks in a row
        _quantize("quantize-weight", 11008, 4128, "f32"),
        # one token through gate and up of a decoder layer
        _gemm("gemm-1", 1, 24576, 4096),
        # a small ragged batch through the down projection, with a bias
        _gemm("gemm-13-bias", 13, 4096, 12288, "f16", True),
        # a serving batch through QKV
        _gemm("gemm-57", 57, 6144, 4096),
        # a part of a prompt through an output projection whose width fits no tile
        _gemm("gemm-200-odd", 200, 5001, 4128, "f16"),
        # a long prompt through gate and up
        _gemm("gemm-4096", 4096, 24576, 4096),
        # a decode batch through 64 experts
        _moe("moe-4", 4),
        # a prompt through 64 experts
        _moe("moe-2048", 2048, dtype="f16"),
        # a decode batch: how the experts are loaded
        _balance("balance-33", 33, 64, 8, "f32", False, 0.0),
        # a training step of a router, padded sequences among its tokens
        _balance("balance-16384", 16384, 64, 8, "bf16", True, 0.2),
        # many tokens over many experts
        _balance("balance-65536", 65536, 160, 6, "f32", True, 0.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("quantize", "gemm", "gemm", "moe", "balance"))
    if kind == "quantize":
        while True:
            rows, cols = _log_int(rng, 1, 16384), 32 * _log_int(rng, 1, 512)
            if rows * cols <= 11008 * 4128:
                break
        c = _quantize("", rows, cols, rng.choice(("f16", "bf16", "f32")))
    elif kind == "gemm":
        while True:
            m, n, k = _log_int(rng, 1, 4096), _log_int(rng, 200, 24576), 32 * _log_int(rng, 8, 384)
            if m * n * k <= 4096 * 24576 * 4096:
                break
        c = _gemm("", m, n, k, rng.choice(("f16", "bf16")), rng.random() < 0.3)
    elif kind == "moe":
        c = _moe("", _log_int(rng, 1, 2048), rng.choice((8, 24, 32, 64)), rng.choice((1, 2, 4, 8)), 32 * rng.randint(16, 64),
                 32 * rng.randint(4, 32), rng.choice(("f16", "bf16")), rng.choice(("silu", "gelu_pytorch_tanh")))
    else:
        while True:
            tokens, experts = _log_int(rng, 1, 65536), _log_int(rng, 4, 512)
            if tokens * experts <= 65536 * 160:
                break
        c = _balance("", tokens, experts, rng.randint(1, min(8, experts)), rng.choice(("f16", "bf16", "f32")), rng.random() < 0.7,
                     rng.choice((0.0, 0.0, 0.1, 0.5)))
    del c["name"]
    return c


# ------------------------------------------------------------------ the plain form
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _rounded(x):
    """x [..., K] in 32 bits as the values of its MXFP4 form."""
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)  # frexp's mantissa is in [0.5, 1): floor(log2) is one less
    e = torch.where(top > 0, e, torch.full_like(e, -127))
    q = torch.ldexp(torch.ldexp(b, -(e // 2)), e // 2 - e)  # in two steps: 2**127 times a small value passes no limit
    size = q.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    q = torch.copysign((torch.round(size / step) * step).clamp(max=6.0), q)
    return torch.ldexp(torch.ldexp(q, e // 2), e - e // 2).flatten(-2)


def _values(codes, scales):
    """The 32-bit values of codes [..., K/2] with scales [..., K/32]."""
    table = torch.tensor(_E2M1, device=codes.device)
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).flatten(-2)
    return (v.unflatten(-1, (-1, 32)) * torch.exp2(scales.float() - 127).unsqueeze(-1)).flatten(-2)


def _packed(w):
    """codes and scales of a 32-bit matrix, for the weights that prepare() makes."""
    b = w.unflatten(-1, (-1, 32))
    e = (torch.frexp(b.abs().amax(-1)).exponent - 3).clamp(-127, 127)
    v = (_rounded(w).unflatten(-1, (-1, 32)) * torch.exp2(-e.float()).unsqueeze(-1)).flatten(-2)
    code = torch.bucketize(v.abs(), torch.tensor(_E2M1[1:8], device=w.device) - 0.1).to(torch.uint8) | ((v < 0).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _activated(g, activation):
    if activation == "silu":
        return g / (1 + torch.exp(-g))
    return g / (1 + torch.exp(-2 * 0.7978845608028654 * (g + 0.044715 * g * g * g)))


def _plain_moe(s):
    case, x, ids = s["case"], s["x"], s["ids"]
    t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inter"]
    w1 = _values(s["gate_up"], s["gate_up_scales"]).reshape(e * 2 * i, h)
    gu = (_rounded(x.float()) @ w1.t()).reshape(t, e, 2 * i)
    mid = _rounded(_activated(gu[..., :i], case["activation"]) * gu[..., i:])
    slot = (ids.unsqueeze(-1) == torch.arange(e, device=ids.device)).float()  # [T, k, E]
    mid = mid * (s["weights"].float().unsqueeze(-1) * slot).sum(1).unsqueeze(-1)
    w2 = _values(s["down"], s["down_scales"]).permute(0, 2, 1).reshape(e * i, h)
    return (mid.reshape(t, e * i) @ w2).to(x.dtype)


def _plain_balance(s):
    case, z, ids = s["case"], s["logits"].detach().float(), s["ids"]
    e, k = case["experts"], case["topk"]
    kept = s["mask"].float() if s["mask"] is not None else torch.ones(case["tokens"], device=z.device)
    n = kept.sum(dtype=torch.float64).clamp(min=1)
    hit = (ids.unsqueeze(-1) == torch.arange(e, device=ids.device)).sum(1) * kept.int().unsqueeze(-1)
    counts = hit.sum(0)
    f = counts.double() / (n * k)
    p = torch.exp(z - z.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    loss = e * (f * ((p * kept.unsqueeze(-1)).sum(0, dtype=torch.float64) / n)).sum()
    out = {"loss": loss.float(), "counts": counts.int()}
    if case["grad"]:
        f = f.float()
        g = p * (f - (p * f).sum(1, keepdim=True)) * kept.unsqueeze(-1)
        out["grad"] = (g * (s["upstream"] * e / n).float()).to(s["logits"].dtype)
    return out


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "quantize":
        return _rounded(s["x"].float()).to(s["x"].dtype)
    if kind == "gemm":
        y = _rounded(s["x"].float()) @ _values(s["codes"], s["scales"]).t()
        return (y + s["bias"].float() if s["bias"] is not None else y).to(s["x"].dtype)
    return _plain_moe(s) if kind == "moe" else _plain_balance(s)


# ------------------------------------------------------------------ the framework's calls
def _calls(s):
    import litevllm_amd as fw
    case, kind = s["case"], s["case"]["kind"]
    if kind == "quantize":
        codes, scales = fw.mxfp4_quantize(s["x"])
        return fw.mxfp4_dequantize(codes, scales, s["x"].dtype)
    if kind == "gemm":
        return fw.mxfp4_gemm(s["x"], s["codes"], s["scales"], bias=s["bias"])
    if kind == "moe":
        return fw.mxfp4_moe(s["x"], s["weights"], s["ids"], fw.MXFP4Experts(s["gate_up"], s["gate_up_scales"]),
                            fw.MXFP4Experts(s["down"], s["down_scales"]), activation=case["activation"])
    loss, counts = fw.moe_balance_loss(s["logits"], s["ids"], s["mask"])
    out = {"loss": loss.detach(), "counts": counts}
    if case["grad"]:
        out["grad"], = torch.autograd.grad(loss, s["logits"], s["upstream"])
    return out


def run(state):
    if own:
        return _calls(state)
    return _plain(state)


# ------------------------------------------------------------------ inputs
def _activations(g, rows, cols, dtype):
    """N(0, 1) with 0.1 % of the channels 20 times as large, as in trained models."""
    x = torch.randn((rows, cols), generator=g, device=DEVICE)
    x[:, torch.randperm(cols, generator=g, device=DEVICE)[: max(1, cols // 1000)]] *= 20.0
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind == "quantize":
        s["x"] = _activations(g, case["rows"], case["cols"], dt)
    elif kind == "gemm":
        s["x"] = _activations(g, case["m"], case["k"], dt)
        s["codes"], s["scales"] = _packed(torch.randn((case["n"], case["k"]), generator=g, device=DEVICE) * 0.02)
        s["bias"] = torch.randn(case["n"], generator=g, device=DEVICE).to(dt) if case["bias"] else None
    elif kind == "moe":
        t, e, h, i = case["tokens"], case["experts"], case["hidden"], case["inter"]
        s["x"] = torch.randn((t, h), generator=g, device=DEVICE).to(dt)
        s["gate_up"], s["gate_up_scales"] = _packed(torch.randn((e, 2 * i, h), generator=g, device=DEVICE) * 0.02)
        s["down"], s["down_scales"] = _packed(torch.randn((e, h, i), generator=g, device=DEVICE) * 0.02)
        # popular experts and rare ones
        logits = torch.randn((t, e), generator=g, device=DEVICE) + torch.randn(e, generator=g, device=DEVICE)
        p, ids = torch.softmax(logits, 1).topk(case["topk"], dim=1)
        s["weights"], s["ids"] = p / p.sum(1, keepdim=True), ids.int()
    else:
        t, e = case["tokens"], case["experts"]
        z = (torch.randn((t, e), generator=g, device=DEVICE) + torch.randn(e, generator=g, device=DEVICE)).to(dt)
        s["ids"] = z.float().topk(case["topk"], dim=1).indices.int()
        s["mask"] = torch.rand(t, generator=g, device=DEVICE) >= case["padding"] if case["padding"] else None
        s["logits"] = z.requires_grad_(case["grad"])
        # the loss' coefficient, times a loss scale where the gradient's type needs one
        s["upstream"] = torch.tensor(0.01 * (65536.0 if dt is torch.float16 else 1.0), device=DEVICE)
    return s


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind == "quantize":
        v = case["rows"] * case["cols"]
        return {"bytes": v * (2 * size + 2 * 17 / 32), "flops": 4 * v}
    if kind == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k * 17 / 32 + (m * (n + k) + (n if case["bias"] else 0)) * 2, "flops": 2 * m * n * k}
    if kind == "moe":
        t, e, k, h, i = case["tokens"], case["experts"], case["topk"], case["hidden"], case["inter"]
        reached = e * (1.0 - (1.0 - k / e) ** t)  # by a uniform router
        return {"bytes": reached * 3 * h * i * 17 / 32 + t * (2 * h * 2 + 8 * k), "flops": 2 * t * k * 3 * h * i}
    t, e, k = case["tokens"], case["experts"], case["topk"]
    return {"bytes": t * (e * size * (2 if case["grad"] else 1) + 4 * k) + 4 * e, "flops": t * e * (10 if case["grad"] else 5)}


# ------------------------------------------------------------------ 64-bit answers
def _exact_rounded(x):
    """The MXFP4 value nearest to each of x's, ties to the even code."""
    rows = x.reshape(-1, 32)
    top = rows.abs().max(1, keepdim=True).values
    scale = torch.pow(2.0, torch.floor(torch.log2(top.clamp(min=2.0 ** -126))).clamp(min=-125) - 2)
    a = rows.abs() / scale
    n = (a > 0.25).long() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    size = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)[n]
    return (torch.sign(rows) * size * scale).reshape(x.shape)


def _exact_values(codes, scales):
    nib = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    field, half = ((nib >> 1) & 3).double(), (nib & 1).double()
    size = torch.where(field == 0, half / 2, (1 + half / 2) * torch.pow(2.0, field - 1))
    size = torch.where(nib >= 8, -size, size)
    return size * torch.pow(2.0, scales.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "quantize":
        return _exact_rounded(s["x"].double())
    if kind == "gemm":
        y = torch.matmul(_exact_rounded(s["x"].double()), _exact_values(s["codes"], s["scales"]).t())
        return y if s["bias"] is None else y + s["bias"].double()
    if kind == "moe":
        x, i = _exact_rounded(s["x"].double()), case["inter"]
        out = torch.zeros_like(x)
        for e in range(case["experts"]):
            rows, slot = (s["ids"] == e).nonzero(as_tuple=True)
            gu = x[rows] @ _exact_values(s["gate_up"][e], s["gate_up_scales"][e]).t()
            g, u = gu[:, :i], gu[:, i:]
            act = g * torch.sigmoid(g) if case["activation"] == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
            y = _exact_rounded(act * u) @ _exact_values(s["down"][e], s["down_scales"][e]).t()
            out.index_add_(0, rows, y * s["weights"][rows, slot].double().unsqueeze(1))
        return out
    e, k = case["experts"], case["topk"]
    z = s["logits"].detach().double().requires_grad_(True)
    rows = torch.arange(case["tokens"], device=z.device) if s["mask"] is None else s["mask"].nonzero()[:, 0]
    n = max(1, rows.numel())
    counts = torch.bincount(s["ids"][rows].reshape(-1).long(), minlength=e)
    loss = e * (counts.double() / (n * k) * (torch.softmax(z[rows], 1).sum(0) / n)).sum()
    out = {"loss": loss.detach(), "counts": counts.int()}
    if case["grad"]:
        out["grad"] = torch.autograd.grad(loss, z, s["upstream"].double())[0]
    return out
