"""Rows dealt out by an index that each of them carries, as cases to be timed.

* ``sort``: the tokens' rows in the order of the experts that a router chose, and where every route went;
  with its gradient, the tokens' sums over their routes;
* ``unsort``: the experts' rows back at their tokens, weighted and summed; with the gradients of rows and weights;
* ``lora``: the low-rank adapters of many requests added to what a shared projection gave:
  ``out[m] = base[m] + s_l (x[m] A_l^T) B_l^T`` with ``l = ids[m]``, ``base[m]`` alone where ``ids[m]`` is no adapter.
"""
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _routes(kind, name, tokens, experts=64, topk=8, hidden=2048, dtype="bf16", grad=False, dropped=0.0):
    return {"name": name, "kind": kind, "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "dtype": dtype,
            "grad": grad, "dropped": dropped}


def _lora(name, rows, requests, k, n, rank, adapters, dtype="bf16", without=0.0):
    return {"name": name, "kind": "lora", "rows": rows, "requests": requests, "k": k, "n": n, "rank": rank, "adapters": adapters,
            "dtype": dtype, "without": without}


def listed():
    return [
        # a decode batch in front of 64 experts
        _routes("sort", "sort-4", 4),
        # a prompt in front of 64 experts
        _routes("sort", "sort-2048", 2048, dtype="f16"),
        # 32-bit rows of no round width; a third of the routes go to experts of other devices
        _routes("sort", "sort-700-odd", 700, 160, 6, 1001, "f32", True, 0.3),
        # a training step
        _routes("sort", "sort-16384-grad", 16384, grad=True),
        # a decode batch behind the experts
        _routes("unsort", "unsort-4", 4),
        # a prompt behind 128 experts of a wider model
        _routes("unsort", "unsort-1000", 1000, 128, 8, 4096, "f16"),
        # a training step
        _routes("unsort", "unsort-16384-grad", 16384, grad=True),
        # one token of one request, an output projection
        _lora("lora-1", 1, 1, 4096, 4096, 16, 8),
        # a ragged batch of single tokens, the down projection of a width that fits no tile, some requests without an adapter
        _lora("lora-29-odd", 29, 29, 12288, 5001, 12, 16, "f16", 0.2),
        # a decode batch through QKV, adapters of many customers
        _lora("lora-64", 64, 64, 4096, 6144, 32, 64),
        # the prompts of five requests
        _lora("lora-777", 777, 5, 4128, 4096, 8, 20, "f16", 0.2),
        # long prompts through gate and up
        _lora("lora-4096", 4096, 6, 4096, 24576, 64, 32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("sort", "unsort", "lora", "lora"))
    if kind == "lora":
        while True:
            rows, k, n = _log_int(rng, 1, 4096), _log_int(rng, 256, 12288), _log_int(rng, 200, 24576)
            if rng.random() < 0.8:
                k, n = -(-k // 32) * 32, -(-n // 16) * 16
            rank, adapters = rng.choice((4, 8, 8, 12, 16, 16, 32, 64)), rng.randint(1, 64)
            if rows * (k + 2 * n) <= 4096 * (4096 + 2 * 24576) and rank * adapters <= 32 * 64:
                break
        requests = rows if rows <= 128 and rng.random() < 0.7 else rng.randint(1, min(rows, 12))
        c = _lora("", rows, requests, k, n, rank, adapters, rng.choice(("f16", "bf16")), rng.choice((0.0, 0.0, 0.3)))
    else:
        while True:
            tokens, topk, hidden = _log_int(rng, 1, 16384), rng.choice((1, 2, 4, 6, 8)), _log_int(rng, 256, 8192)
            dtype = rng.choice(("f16", "bf16", "bf16", "f32"))
            if rng.random() < 0.7:
                hidden = -(-hidden // 64) * 64
            if tokens * topk * hidden * (2 if dtype == "f32" else 1) <= 16384 * 8 * 2048:
                break
        c = _routes(kind, "", tokens, _log_int(rng, 8, 512), topk, hidden, dtype, rng.random() < 0.5, rng.choice((0.0, 0.0, 0.3)))
    del c["name"]
    return c


# ------------------------------------------------------------------ the plain form
def _plain_places(ids, experts):
    """offsets [E + 1], the expert of every place and the place of every route (-1: none), routes of an expert in their order."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    order = torch.argsort(key, stable=True)
    placed = key[order]
    hit = torch.zeros(experts + 1, dtype=torch.long, device=ids.device).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([torch.zeros_like(hit[:1]), torch.cumsum(hit[:experts], 0)])
    places = torch.empty_like(flat)
    places[order] = torch.arange(flat.numel(), device=ids.device)
    places = torch.where(key < experts, places, torch.full_like(places, -1))
    return (offsets.int(), torch.where(placed < experts, placed, torch.full_like(placed, -1)).int(), places.int().reshape(ids.shape),
            order)


def _gathered(rows, places):
    """rows [places] in 32 bits, [T, k, H], zero where there is no place."""
    g = rows[places.reshape(-1).clamp(min=0).long()].float() if rows.dtype != torch.float32 else rows[places.reshape(-1).clamp(min=0).long()]
    return (g * (places.reshape(-1, 1) >= 0).float()).reshape(*places.shape, rows.shape[1])


def _plain_sort(s):
    x, k = s["x"].detach(), s["ids"].shape[1]
    offsets, experts, places, order = _plain_places(s["ids"], s["case"]["experts"])
    rows = x[order // k] * (experts >= 0).unsqueeze(1).to(x.dtype)
    out = {"rows": rows, "offsets": offsets, "experts": experts, "places": places}
    if s["case"]["grad"]:
        out["grad"] = _gathered(s["upstream"], places).sum(1).to(x.dtype)
    return out


def _plain_unsort(s):
    rows, w, places = s["rows"].detach(), s["weights"].detach(), s["places"]
    g = _gathered(rows, places)
    out = {"out": (g * w.unsqueeze(-1)).sum(1).to(rows.dtype)}
    if s["case"]["grad"]:
        up = s["upstream"].float()
        out["grad_weights"] = (g * up.unsqueeze(1)).sum(2)
        flat = places.reshape(-1).long()
        at = torch.where(flat >= 0, flat, torch.full_like(flat, rows.shape[0]))
        grad = torch.zeros((rows.shape[0] + 1, rows.shape[1]), dtype=rows.dtype, device=rows.device)
        grad[at] = (w.unsqueeze(-1) * up.unsqueeze(1)).to(rows.dtype).reshape(flat.numel(), -1)
        out["grad_rows"] = grad[:-1]
    return out


def _plain_lora(s):
    a, b, ids = s["a"].float(), s["b"].float(), s["ids"]
    (adapters, rank, k), n = a.shape, b.shape[1]
    mine = (ids.unsqueeze(1) == torch.arange(adapters, device=ids.device)).float() * s["scales"]  # [M, L]
    v = (s["x"].float() @ a.reshape(adapters * rank, k).t()).reshape(-1, adapters, rank) * mine.unsqueeze(-1)
    delta = v.reshape(-1, adapters * rank) @ b.permute(0, 2, 1).reshape(adapters * rank, n)
    return (s["base"].float() + delta).to(s["base"].dtype)


# ------------------------------------------------------------------ the framework's calls
def _calls(s):
    import litevllm_amd as fw
    case, kind = s["case"], s["case"]["kind"]
    if kind == "lora":
        return fw.lora_add(s["base"], s["x"], s["a"], s["b"], s["ids"], s["scales"])
    if kind == "sort":
        rows, routes = fw.moe_sort(s["x"], s["ids"], case["experts"])
        out = {"rows": rows.detach(), "offsets": routes.offsets, "experts": routes.experts, "places": routes.places}
        if case["grad"]:
            out["grad"], = torch.autograd.grad(rows, s["x"], s["upstream"])
        return out
    y = fw.moe_unsort(s["rows"], s["weights"], fw.MoERoutes(s["offsets"], s["experts"], s["places"]))
    out = {"out": y.detach()}
    if case["grad"]:
        out["grad_rows"], out["grad_weights"] = torch.autograd.grad(y, (s["rows"], s["weights"]), s["upstream"])
    return out


def run(state):
    if own:
        return _calls(state)
    return {"sort": _plain_sort, "unsort": _plain_unsort, "lora": _plain_lora}[state["case"]["kind"]](state)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEVICE)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=DEVICE)

    if kind == "lora":
        m, k, n, rank, adapters = case["rows"], case["k"], case["n"], case["rank"], case["adapters"]
        x = normal(m, k)
        # 0.1 % of the channels 20 times as large, as in trained models
        x[:, torch.randperm(k, generator=g, device=DEVICE)[: max(1, k // 1000)]] *= 20.0
        s["x"], s["base"] = x.to(dt), normal(m, n).to(dt)
        s["a"] = (normal(adapters, rank, k) * k ** -0.5).to(dt)
        s["b"] = (normal(adapters, n, rank) * 0.05).to(dt)
        s["scales"] = 0.5 + 2.0 * uniform(adapters)  # alpha / rank
        # the rows of a request lie together; some requests have no adapter
        which = torch.randint(adapters, (case["requests"],), generator=g, device=DEVICE)
        which[uniform(case["requests"]) < case["without"]] = -1
        cuts = torch.randperm(m - 1, generator=g, device=DEVICE)[: case["requests"] - 1] + 1 if m > 1 else torch.empty(0, device=DEVICE)
        request = (torch.arange(m, device=DEVICE).unsqueeze(1) >= cuts).sum(1)
        s["ids"] = which[request].int()
        return s
    t, e, k, h = case["tokens"], case["experts"], case["topk"], case["hidden"]
    # popular experts and rare ones
    p, ids = torch.softmax(normal(t, e) + normal(e), 1).topk(k, dim=1)
    ids = torch.where(uniform(t, k) < case["dropped"], torch.full_like(ids, -1), ids).int()
    if kind == "sort":
        s["x"], s["ids"] = normal(t, h).to(dt).requires_grad_(case["grad"]), ids
        s["upstream"] = normal(t * k, h).to(dt) if case["grad"] else None
        return s
    s["offsets"], s["experts"], s["places"], _ = _plain_places(ids, e)
    s["rows"] = normal(t * k, h).to(dt).requires_grad_(case["grad"])
    s["weights"] = (p / p.sum(1, keepdim=True)).contiguous().requires_grad_(case["grad"])
    s["upstream"] = normal(t, h).to(dt) if case["grad"] else None
    return s


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "lora":
        m, k, n, rank = case["rows"], case["k"], case["n"], case["rank"]
        reached = case["adapters"] * (1.0 - (1.0 - (1.0 - case["without"]) / case["adapters"]) ** case["requests"])
        return {"bytes": (reached * rank * (k + n) + m * (k + 2 * n)) * 2 + 4 * m,
                "flops": 2 * m * (1.0 - case["without"]) * rank * (k + n)}
    t, k, h, kept = case["tokens"], case["topk"], case["hidden"], 1.0 - case["dropped"]
    tokens, rows = t * h * size, t * k * h * size
    if case["kind"] == "sort":
        moved = tokens + rows + t * k * 12 + (rows * kept + tokens if case["grad"] else 0)
        return {"bytes": moved, "flops": t * k * h * kept if case["grad"] else 0}
    moved = rows * kept + tokens + t * k * 8 + (rows * kept + rows + tokens + t * k * 12 if case["grad"] else 0)
    return {"bytes": moved, "flops": t * k * h * kept * (5 if case["grad"] else 2)}


# ------------------------------------------------------------------ 64-bit answers
def _exact_lora(s):
    x, out = s["x"].double(), s["base"].double()
    for l in torch.unique(s["ids"]).tolist():
        if l >= 0:
            at = (s["ids"] == l).nonzero()[:, 0]
            low = torch.matmul(x[at], s["a"][l].double().t().contiguous())
            out[at] += s["scales"][l].double() * torch.matmul(low, s["b"][l].double().t().contiguous())
    return out


def _exact_sort(s):
    case, ids = s["case"], s["ids"]
    t, k = ids.shape
    x = s["x"].detach().double()
    rows, experts = torch.zeros((t * k, x.shape[1]), dtype=torch.float64, device=x.device), torch.full((t * k,), -1, device=x.device)
    places, offsets, at = torch.full((t * k,), -1, device=x.device), [0], 0
    grad = torch.zeros_like(x) if case["grad"] else None
    for e in range(case["experts"]):
        token, slot = (ids == e).nonzero(as_tuple=True)  # by token, then by slot
        end = at + token.numel()
        rows[at:end], experts[at:end] = x[token], e
        places[token * k + slot] = torch.arange(at, end, device=x.device)
        if grad is not None:
            grad.index_add_(0, token, s["upstream"][at:end].double())
        at = end
        offsets.append(at)
    out = {"rows": rows, "offsets": torch.tensor(offsets, device=x.device).int(), "experts": experts.int(),
           "places": places.int().reshape(t, k)}
    if grad is not None:
        out["grad"] = grad
    return out


def _exact_unsort(s):
    places, w, rows = s["places"], s["weights"].detach().double(), s["rows"].detach()
    up = s["upstream"].double() if s["case"]["grad"] else None
    out = torch.zeros((places.shape[0], rows.shape[1]), dtype=torch.float64, device=rows.device)
    gw = torch.zeros_like(w)
    gr = torch.zeros(rows.shape, dtype=torch.float64, device=rows.device) if up is not None else None
    for j in range(places.shape[1]):
        token = (places[:, j] >= 0).nonzero()[:, 0]
        at = places[token, j].long()
        part = rows[at].double()
        out[token] += part * w[token, j].unsqueeze(1)
        if up is not None:
            gw[token, j] = torch.linalg.vecdot(part, up[token])
            gr[at] = up[token] * w[token, j].unsqueeze(1)
    return {"out": out} if up is None else {"out": out, "grad_weights": gw, "grad_rows": gr}


def exact(case, seed):
    s = prepare(case, seed)
    return {"sort": _exact_sort, "unsort": _exact_unsort, "lora": _exact_lora}[case["kind"]](s)
