"""Rows sorted by expert and back, and their gradients, against plain 64-bit forms."""
import ctypes

import pytest
import torch

from litevllm_amd import _lib as L

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _places(ids, experts):
    """offsets, the expert of every place, places, by a loop over the routes on the host."""
    flat = [i if 0 <= i < experts else experts for i in ids.flatten().tolist()]
    order = sorted(range(len(flat)), key=lambda r: flat[r])  # stable
    places, of, offsets = [-1] * len(flat), [-1] * len(flat), [0] * (experts + 1)
    for p, r in enumerate(order):
        if flat[r] < experts:
            places[r], of[p] = p, flat[r]
            offsets[flat[r] + 1] += 1
    for e in range(experts):
        offsets[e + 1] += offsets[e]
    return torch.tensor(offsets), torch.tensor(of), torch.tensor(places).reshape(ids.shape)


def _ids(seed, t, e, k, dropped=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(e, (t, k), generator=g)
    if dropped:
        out = torch.tensor([-1, e, 2 ** 31 - 1, -2 ** 31])[torch.randint(4, (t, k), generator=g)]
        ids = torch.where(torch.rand(t, k, generator=g) < dropped, out, ids)
    return ids.int().cuda()


def _whole(seed, *shape, size=4):
    """Small whole numbers: their sums in fp32 are exact, so results have one right value."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-size, size + 1, shape, generator=g).float().cuda()


# one launch and three, few and many experts, rows of one element, of odd widths, of several blocks
CASES = [(1, 1, 1, 1, 0.0), (1, 8, 2, 7, 0.0), (4, 64, 8, 256, 0.0), (3, 5, 11, 33, 0.5), (37, 160, 6, 1001, 0.3), (511, 7, 8, 24, 0.0),
         (512, 1024, 8, 8, 0.1), (513, 64, 8, 130, 0.2), (4097, 33, 1, 5, 1.0), (9000, 200, 3, 40, 0.4), (20, 16, 2, 9000, 0.2),
         (40000, 1024, 4, 12, 0.0), (2048, 64, 8, 96, 0.0), (2049, 5, 4, 40, 0.2), (60, 40, 130, 20, 0.1), (9, 30, 700, 16, 0.1),
         (70, 30, 600, 16, 0.1), (11, 1024, 1024, 3, 0.0), (4096, 513, 8, 10, 0.05), (4097, 512, 8, 9, 0.05), (700, 300, 9, 2056, 0.1)]


def _check_sort(x, ids, experts):
    from litevllm_amd import moe_sort
    rows, routes = moe_sort(x, ids, experts)
    offsets, of, places = _places(ids, experts)
    assert routes.offsets.dtype == routes.experts.dtype == routes.places.dtype == torch.int32
    assert torch.equal(routes.offsets.cpu().long(), offsets)
    assert torch.equal(routes.experts.cpu().long(), of)
    assert torch.equal(routes.places.cpu().long(), places)
    want = torch.zeros_like(rows)
    at = (places >= 0).nonzero()
    want[places[at[:, 0], at[:, 1]].cuda()] = x.detach()[at[:, 0].cuda()]
    assert rows.dtype == x.dtype and torch.equal(rows.detach(), want)
    return rows, routes


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("t,e,k,h,dropped", CASES)
def test_sort_and_its_gradient(t, e, k, h, dropped, dtype):
    ids = _ids(t + e, t, e, k, dropped)
    x = _whole(1, t, h).to(DTYPES[dtype]).requires_grad_(True)
    rows, routes = _check_sort(x, ids, e)
    up = _whole(2, t * k, h).to(DTYPES[dtype])
    want = torch.zeros(t, h, device="cuda", dtype=torch.float64)
    for j in range(k):
        p = routes.places[:, j].long()
        want += up[p.clamp(min=0)].double() * (p >= 0).unsqueeze(1)
    up[int(routes.offsets[-1]):] = float("nan")  # behind the last row: not read
    grad, = torch.autograd.grad(rows, x, up)
    assert grad.dtype == x.dtype and torch.equal(grad, want.to(x.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("t,e,k,h,dropped", CASES)
def test_unsort_and_its_gradients(t, e, k, h, dropped, dtype):
    """Whole numbers and weights of quarters: every sum is exact, results are rounded once."""
    from litevllm_amd import moe_sort, moe_unsort
    ids, dt = _ids(t + e + 1, t, e, k, dropped), DTYPES[dtype]
    _, routes = moe_sort(torch.zeros(t, 1, device="cuda"), ids, e)
    rows, up = _whole(3, t * k, h).to(dt), _whole(4, t, h).to(dt)
    last = int(routes.offsets[-1])
    rows[last:] = float("nan")
    rows.requires_grad_(True)
    w = (_whole(5, t, k) / 4).requires_grad_(True)
    out = moe_unsort(rows, w, routes)
    grads = torch.autograd.grad(out, (rows, w), up)
    want, want_rows = torch.zeros(t, h, dtype=torch.float64, device="cuda"), torch.zeros(t * k, h, dtype=torch.float64, device="cuda")
    want_w = torch.zeros(t, k, dtype=torch.float64, device="cuda")
    for j in range(k):
        token = (routes.places[:, j] >= 0).nonzero()[:, 0]
        p = routes.places[token, j].long()
        r, f = rows.detach()[p].double(), w.detach()[token, j].double().unsqueeze(1)
        want[token] += f * r
        want_rows[p] = f * up[token].double()
        want_w[token, j] = (up[token].double() * r).sum(1)
    assert out.dtype == dt and torch.equal(out.detach(), want.to(dt))
    assert grads[0].dtype == dt and torch.equal(grads[0], want_rows.to(dt))
    assert grads[1].dtype == torch.float32 and torch.equal(grads[1], want_w.float())
    # each gradient alone, and no weights
    assert torch.equal(torch.autograd.grad(moe_unsort(rows, w.detach(), routes), rows, up)[0], grads[0])
    assert torch.equal(torch.autograd.grad(moe_unsort(rows.detach(), w, routes), w, up)[0], grads[1])
    ones = torch.ones_like(w)
    plain = moe_unsort(rows, None, routes)
    assert torch.equal(plain, moe_unsort(rows, ones, routes))
    assert torch.equal(torch.autograd.grad(plain, rows, up)[0], torch.autograd.grad(moe_unsort(rows, ones, routes), rows, up)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("wtype", list(DTYPES))
def test_random_values_and_weight_types(dtype, wtype):
    """k products and sums in fp32 (2 k half steps of the sum of magnitudes at most) and one rounding of the result."""
    from litevllm_amd import moe_sort, moe_unsort
    t, e, k, h = 130, 24, 5, 513
    g, dt, wt = torch.Generator().manual_seed(6), DTYPES[dtype], DTYPES[wtype]
    _, routes = moe_sort(torch.zeros(t, 1, device="cuda"), _ids(7, t, e, k, 0.2), e)
    rows = torch.randn(t * k, h, generator=g).to(dt).cuda().requires_grad_(True)
    w = torch.rand(t, k, generator=g).to(wt).cuda().requires_grad_(True)
    up = torch.randn(t, h, generator=g).to(dt).cuda()
    out = moe_unsort(rows, w, routes)
    gr, gw = torch.autograd.grad(out, (rows, w), up)
    assert gr.dtype == dt and gw.dtype == wt
    p = routes.places.long()
    there = (p >= 0).unsqueeze(2).double()
    r = rows.detach().double()[p.clamp(min=0)] * there
    terms = r * w.detach().double().unsqueeze(2)
    tiny, f = 2.0 ** -24, torch.finfo

    def near(got, want, magnitude, roundings):
        tol = magnitude * roundings * tiny + want.abs() * f(got.dtype).eps / 2 + f(got.dtype).smallest_normal * f(got.dtype).eps
        assert bool(((got.double() - want).abs() <= tol).all())
    near(out.detach(), terms.sum(1), terms.abs().sum(1), 2 * k)
    dots = r * up.double().unsqueeze(1)
    near(gw, dots.sum(2), dots.abs().sum(2), 2 * h)
    back = (w.detach().double().unsqueeze(2) * up.double().unsqueeze(1)).expand_as(r)
    want = torch.zeros(t * k + 1, h, dtype=torch.float64, device="cuda")
    want[torch.where(p >= 0, p, torch.full_like(p, t * k)).flatten()] = back.reshape(-1, h)
    near(gr, want[:-1], want[:-1].abs(), 1)


@pytest.mark.gpu
def test_gradients_against_differences():
    """The operator is bilinear: out(rows + d, w) - out(rows - d, w) over 2 is its derivative along d, and the gradients' dot
    product with d is the same number; whole numbers make both exact."""
    from litevllm_amd import moe_sort, moe_unsort
    t, e, k, h = 19, 6, 3, 40
    x, dx = _whole(8, t, h).requires_grad_(True), _whole(9, t, h)
    w, dw = _whole(10, t, k).requires_grad_(True), _whole(11, t, k)
    up = _whole(12, t, h)
    ids = _ids(13, t, e, k, 0.2)

    def f(x, w):
        rows, routes = moe_sort(x, ids, e)
        return (moe_unsort(rows * 2.0, w, routes) * up).sum(dtype=torch.float64)
    gx, gw = torch.autograd.grad(f(x, w), (x, w))
    with torch.no_grad():
        assert float((f(x + dx, w) - f(x - dx, w)) / 2) == float((gx.double() * dx).sum())
        assert float((f(x, w + dw) - f(x, w - dw)) / 2) == float((gw.double() * dw).sum())


@pytest.mark.gpu
def test_strides_types_of_ids_and_infinities():
    from litevllm_amd import moe_sort, moe_unsort
    t, e, k, h = 50, 9, 4, 70
    x, ids = _whole(14, t, h).bfloat16(), _ids(15, t, e, k, 0.3)
    x[3, 5], x[4, 6] = float("inf"), float("nan")
    want, routes = moe_sort(x, ids, e)
    wide = torch.zeros(2 * t, 99, dtype=torch.bfloat16, device="cuda")
    wide[::2, 7:77] = x
    for y, i in ((wide[::2, 7:77], ids.long() - (ids.long() < 0).long() * 2 ** 40), (x.t().contiguous().t(), ids.t().contiguous().t())):
        got, other = moe_sort(y, i, e)
        assert torch.equal(got.view(torch.int16), want.view(torch.int16)) and all(torch.equal(a, b) for a, b in zip(other, routes))
    w = _whole(16, t, k).t().contiguous().t()
    out = moe_unsort(want, w, routes)
    assert torch.equal(out.view(torch.int16), moe_unsort(want.t().contiguous().t(), w.contiguous(), routes).view(torch.int16))
    keep = torch.ones(t, dtype=torch.bool, device="cuda")
    keep[3:5] = False
    assert bool(torch.isfinite(out[keep]).all())
    leaf = wide.clone().nan_to_num(0, 0, 0).requires_grad_(True)
    up = torch.randn(1, 1, device="cuda").bfloat16().expand(t * k, h)  # as sum() passes it
    grad, = torch.autograd.grad(moe_sort(leaf[::2, 7:77], ids, e)[0], leaf, up)
    assert torch.equal(grad[::2, 7:77], (up[0, 0].double() * (routes.places >= 0).sum(1, keepdim=True)).expand(t, h).bfloat16())
    assert int((grad[1::2] != 0).sum()) == 0


@pytest.mark.gpu
def test_no_tokens_and_empty_rows():
    from litevllm_amd import moe_sort, moe_unsort
    rows, routes = moe_sort(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 5)
    assert rows.shape == (0, 8) and routes.places.shape == (0, 2) and routes.offsets.tolist() == [0] * 6
    assert moe_unsort(rows, None, routes).shape == (0, 8)
    for t in (3, 5000):
        ids = _ids(17, t, 5, 2, 0.2)
        rows, routes = moe_sort(torch.zeros(t, 0, device="cuda"), ids, 5)
        offsets, of, places = _places(ids, 5)
        assert rows.shape == (2 * t, 0) and torch.equal(routes.places.cpu().long(), places) and torch.equal(routes.offsets.cpu().long(), offsets)
        w = torch.ones(t, 2, device="cuda", requires_grad=True)
        out = moe_unsort(rows, w, routes)
        assert out.shape == (t, 0) and torch.equal(torch.autograd.grad(out, w, out)[0], torch.zeros(t, 2, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("t,k,h", [(1023, 8, 16), (1025, 8, 16), (13000, 8, 1100), (26000, 8, 1100), (9000, 2, 8200)])
def test_many_rows(t, k, h):
    """Around the numbers of routes and bytes from which on other launches do the work."""
    from litevllm_amd import moe_unsort
    x = _whole(50 + k, t, h).half().requires_grad_(True)
    rows, routes = _check_sort(x, _ids(51 + k, t, 37, k, 0.2), 37)
    kept = (routes.places >= 0).sum(1, keepdim=True)
    assert torch.equal(moe_unsort(rows, None, routes), (x * kept).half())
    assert torch.equal(torch.autograd.grad(rows, x, torch.ones_like(rows))[0], kept.half().expand(t, h))


@pytest.mark.gpu
def test_rows_past_4_gib():
    from litevllm_amd import moe_sort, moe_unsort
    t, e, k, h = 66000, 16, 8, 4104
    x = torch.randint(-3, 4, (t, h), device="cuda", dtype=torch.int8).bfloat16().requires_grad_(True)
    ids = _ids(18, t, e, k, 0.1)
    rows, routes = moe_sort(x, ids, e)
    assert rows.numel() * 2 > 2 ** 32
    w = torch.ones(t, k, device="cuda", requires_grad=True)
    out = moe_unsort(rows, w, routes)
    many = (routes.places >= 0).sum(1, keepdim=True)
    assert torch.equal(out.detach(), x.detach() * many)
    gx, gw = torch.autograd.grad(out, (x, w), x.detach())
    assert torch.equal(gx, x.detach() * many)
    assert torch.equal(gw, (x.detach().float() ** 2).sum(1, keepdim=True) * (routes.places >= 0))


@pytest.mark.gpu
def test_routes_that_are_written_over():
    """The adapters' ids may be made of routes.experts in place; places that a backward needs may not change unnoticed."""
    from litevllm_amd import moe_sort, moe_unsort
    x, w, ids = _whole(60, 6, 8).requires_grad_(True), _whole(61, 6, 2).requires_grad_(True), _ids(62, 6, 4, 2)
    want = None
    for touch in (lambda r: None, lambda r: r.experts.clamp_(min=0), lambda r: r.offsets.zero_(), lambda r: r.places.zero_()):
        rows, routes = moe_sort(x, ids, 4)
        touch(routes)
        grad = lambda: torch.autograd.grad(rows, x, torch.ones_like(rows))[0]
        if int(routes.places.max()) == 0:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                grad()
        else:
            got = grad()
            want = got if want is None else want
            assert torch.equal(got, want)
    rows, routes = moe_sort(x, ids, 4)
    out = moe_unsort(rows, w, routes)
    routes.experts.zero_()
    torch.autograd.grad(out, w, torch.ones_like(out), retain_graph=True)
    routes.offsets.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, w, torch.ones_like(out))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [30, 3000, 9000])
def test_two_calls_at_once(t):
    from litevllm_amd import moe_sort, moe_unsort
    h, e, k = 264, 40, 4
    x, w = _whole(70, t, h).bfloat16(), _whole(71, t, k)
    ids = [_ids(72, t, e, k, 0.1), _ids(73, t, e, k, 0.3)]

    def step(ids):
        rows, routes = moe_sort(x, ids, e)
        return [rows, *routes, moe_unsort(rows, w, routes)]
    want, got, streams = [step(i) for i in ids], [[], []], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for s, i, to in zip(streams, ids, got):
            with torch.cuda.stream(s):
                to.append(step(i))
    torch.cuda.synchronize()
    for to, ref in zip(got, want):
        assert all(torch.equal(a, b) for outs in to for a, b in zip(outs, ref))


@pytest.mark.gpu
def test_the_most_tokens():
    from litevllm_amd import moe_sort, moe_unsort
    t, h = 1 << 23, 2
    x = (torch.arange(t, device="cuda") % 97).half().unsqueeze(1).repeat(1, h).requires_grad_(True)
    ids = (torch.arange(t, device="cuda") % 5).unsqueeze(1) - 1
    rows, routes = moe_sort(x, ids, 4)
    assert torch.equal(routes.offsets.cpu(), torch.tensor([0, *(int((ids <= e).sum() - (ids < 0).sum()) for e in range(4))], dtype=torch.int32))
    w = (torch.arange(t, device="cuda") % 3).float().unsqueeze(1).requires_grad_(True)
    out = moe_unsort(rows, w, routes)
    kept = (ids >= 0).float()
    assert torch.equal(out, (x * w * kept).half())
    dx, dw = torch.autograd.grad(out, (x, w), torch.ones_like(out))
    assert torch.equal(dx, (w * kept).half().expand(t, h)) and torch.equal(dw, x.float().sum(1, keepdim=True) * kept)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [30, 3000])
def test_replays_and_another_stream(t):
    from litevllm_amd import moe_sort, moe_unsort
    e, k, h = 40, 4, 264
    x, ids, w, up = _whole(19, t, h).bfloat16(), _ids(20, t, e, k, 0.1), _whole(21, t, k), _whole(22, t, h).bfloat16()

    def step(x, w, ids):
        rows, routes = moe_sort(x, ids, e)
        out = moe_unsort(rows, w, routes)
        return [out.detach(), *torch.autograd.grad(out, (x, w), up), *routes]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x.clone().requires_grad_(True), w.clone().requires_grad_(True), ids)
        lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        with torch.cuda.graph(graph, stream=side):
            got = step(lx, lw, ids)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        with torch.no_grad():
            lx.copy_(x * (1 + i))
            ids.copy_((ids + 3) % (e + 2))
        graph.replay()
        torch.cuda.synchronize()
        want = step(lx.detach().clone().requires_grad_(True), lw.detach().clone().requires_grad_(True), ids)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("back", [lambda t: t.cpu(), lambda t: t[:1], lambda t: t.double()])
def test_saved_tensors_that_come_back_as_others_are_refused(back):
    from litevllm_amd import moe_sort, moe_unsort
    x, w, ids = _whole(23, 6, 8).requires_grad_(True), _whole(24, 6, 2).requires_grad_(True), _ids(25, 6, 4, 2)
    rows, routes = moe_sort(x.detach(), ids, 4)
    for f in (lambda: moe_sort(x, ids, 4)[0], lambda: moe_unsort(rows, w, routes)):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            y = f()
        with pytest.raises(RuntimeError, match="came back"):
            y.sum().backward()


@pytest.mark.gpu
def test_gradient_under_hooks_that_copy():
    from litevllm_amd import moe_sort, moe_unsort
    x, w, ids, up = _whole(26, 60, 24).requires_grad_(True), _whole(27, 60, 3).requires_grad_(True), _ids(28, 60, 7, 3, 0.2), _whole(29, 60, 24)

    def f():
        rows, routes = moe_sort(x, ids, 7)
        return moe_unsort(rows, w, routes)
    want = torch.autograd.grad(f(), (x, w), up)
    apart = lambda t: torch.stack([t, t], -1)[..., 0]
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.saved_tensors_hooks(lambda t: t, apart)):
        with hooks:
            y = f()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), up), want))


@pytest.mark.gpu
def test_refusals():
    from litevllm_amd import MoERoutes, moe_sort, moe_unsort
    x, ids, w = _whole(30, 6, 8), _ids(31, 6, 4, 2), _whole(32, 6, 2)
    rows, routes = moe_sort(x, ids, 4)
    o, of, p = routes
    for bad in (lambda: moe_sort(x[0], ids, 4), lambda: moe_sort(x, ids[:5], 4), lambda: moe_sort(x, ids[0], 4), lambda: moe_sort(x, ids[:, :0], 4),
                lambda: moe_sort(x, ids, 0), lambda: moe_sort(x, ids.repeat(1, 513), 4), lambda: moe_sort(x, ids, 1025), lambda: moe_sort(x.cpu(), ids, 4), lambda: moe_sort(x.cpu(), ids.cpu(), 4),
                lambda: moe_unsort(rows[:11], w, routes), lambda: moe_unsort(rows[0], w, routes), lambda: moe_unsort(rows, w[:5], routes),
                lambda: moe_unsort(rows, w.cpu(), routes), lambda: moe_unsort(rows, w, MoERoutes(o, of, p[0])),
                lambda: moe_unsort(rows, w, MoERoutes(o[:1], of, p)), lambda: moe_unsort(rows, w, MoERoutes(o, of, p[:, :0]))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: moe_sort(x.double(), ids, 4), lambda: moe_sort(x, ids.short(), 4), lambda: moe_unsort(rows.double(), w, routes),
                lambda: moe_unsort(rows, w.double(), routes), lambda: moe_unsort(rows, w, MoERoutes(o, of, p.long())),
                lambda: moe_unsort(rows, w, MoERoutes(o.long(), of, p))):
        with pytest.raises(TypeError):
            bad()
    x.requires_grad_(True)
    w.requires_grad_(True)
    up = _whole(33, 12, 8).requires_grad_(True)
    g, = torch.autograd.grad(moe_sort(x, ids, 4)[0], x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    g, = torch.autograd.grad(moe_unsort(rows, w, routes).sum(), w, create_graph=True)
    rows.requires_grad_(True)
    g = torch.autograd.grad(moe_unsort(rows, w, routes).sum(), (rows, w), create_graph=True)
    for one in g:
        with pytest.raises(RuntimeError, match="twice"):
            one.sum().backward(retain_graph=True)


@pytest.mark.gpu
def test_places_outside_the_rows_are_not_followed():
    from litevllm_amd import MoERoutes, moe_sort, moe_unsort
    x, ids, w = _whole(34, 6, 8), _ids(35, 6, 4, 2), _whole(36, 6, 2).requires_grad_(True)
    rows, routes = moe_sort(x, ids, 4)
    wild = routes.places.clone()
    wild[0], wild[1] = torch.tensor([12, 2 ** 31 - 1]), torch.tensor([-7, -2 ** 31])
    out = moe_unsort(rows.requires_grad_(True), w, MoERoutes(routes.offsets - 100, routes.experts, wild))
    gr, gw = torch.autograd.grad(out, (rows, w), x)
    assert bool((out[:2] == 0).all()) and bool((gw[:2] == 0).all())
    assert torch.equal(out[2:], moe_unsort(rows, w, routes)[2:])


def test_entries_refuse():
    lib = L.load()
    p = (ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p).value + 255) & ~255

    def sort(x=p, ld=8, ids=p, bits=32, rows=p, off=p, t=2, h=8, e=8, k=2, dt=L.DTYPE_F16, ws=None, wsb=0):
        return lib.awq_w4a16_moe_sort(x, ld, ids, bits, rows, off, p, p, t, h, e, k, dt, ws, wsb, None)
    assert sort(x=None) == sort(ids=None) == sort(rows=None) == sort(off=None) == L.ERR_NULL
    assert sort(t=-1) == sort(h=-1) == sort(e=0) == sort(k=0) == L.ERR_SHAPE
    assert sort(dt=0) == sort(bits=16) == sort(e=1025) == sort(k=1025) == sort(t=(1 << 30) + 1) == sort(t=1 << 29, k=3) == L.ERR_UNSUPPORTED
    assert sort(h=(1 << 24) + 1, ld=1 << 25) == L.ERR_UNSUPPORTED
    assert sort(t=(1 << 23) + 1, k=1) == L.ERR_UNSUPPORTED and lib.awq_w4a16_moe_sort_workspace_bytes((1 << 23) + 1, 8, 1) == 0
    assert sort(ld=7) == sort(x=p + 1) == sort(rows=p + 2, dt=L.DTYPE_F32) == L.ERR_STRIDE
    need = lib.awq_w4a16_moe_sort_workspace_bytes(50000, 8, 2)
    assert need > 0 and sort(t=50000) == sort(t=50000, ws=p, wsb=need - 1) == L.ERR_WORKSPACE
    assert sort(t=50000, ws=p + 4, wsb=need) == L.ERR_STRIDE
    for t, e, k in ((0, 8, 2), (-1, 8, 2), (5, 0, 2), (5, 1025, 2), (5000, 8, 1025), (5, 8, 0), ((1 << 30) + 1, 8, 1), (1 << 62, 8, 8)):
        assert lib.awq_w4a16_moe_sort_workspace_bytes(t, e, k) == 0

    def unsort(rows=p, places=p, w=p, wdt=L.DTYPE_F32, out=p, ld=8, t=2, h=8, k=2, dt=L.DTYPE_F16):
        return lib.awq_w4a16_moe_unsort(rows, places, w, wdt, out, ld, t, h, k, dt, None)
    assert unsort(rows=None) == unsort(places=None) == unsort(out=None) == L.ERR_NULL
    assert unsort(t=-1) == unsort(h=-1) == unsort(k=0) == L.ERR_SHAPE
    assert unsort(dt=0) == unsort(wdt=0) == unsort(w=None) == unsort(t=1 << 30) == L.ERR_UNSUPPORTED
    assert unsort(t=(1 << 23) + 1, k=1) == L.ERR_UNSUPPORTED
    assert unsort(ld=7) == unsort(rows=p + 1) == unsort(out=p + 1) == L.ERR_STRIDE
    assert unsort(t=0) == unsort(h=0) == L.OK

    def grad(up=p, ld=8, rows=p, places=p, total=p, w=p, wdt=L.DTYPE_F32, gr=p, gw=p, t=2, h=8, k=2, dt=L.DTYPE_F16):
        return lib.awq_w4a16_moe_unsort_grad(up, ld, rows, places, total, w, wdt, gr, gw, t, h, k, dt, None)
    assert grad(up=None) == grad(rows=None) == grad(places=None) == grad(total=None) == L.ERR_NULL
    assert grad(t=-1) == grad(h=-1) == grad(k=0) == L.ERR_SHAPE
    assert grad(dt=0) == grad(wdt=0) == grad(w=None, wdt=0) == grad(w=None, gw=None) == grad(t=1 << 30) == L.ERR_UNSUPPORTED
    assert grad(t=(1 << 23) + 1, k=1) == L.ERR_UNSUPPORTED
    assert grad(ld=7) == grad(up=p + 1) == grad(gr=p + 1) == L.ERR_STRIDE
    assert grad(t=0) == grad(gr=None, gw=None) == L.OK


@pytest.mark.gpu
@pytest.mark.parametrize("t", [9, 900])
def test_a_routed_layer_with_adapters_of_its_experts(t):
    """Router, sort, dense experts, adapters of the experts on the sorted rows, weights, sum: against a 64-bit loop over tokens.
    bf16 roundings, each at most half a step: the expert's product (K + 1 half steps of fp32 among its terms aside), the adapters'
    sum, the output."""
    from litevllm_amd import lora_add, moe_balance_loss, moe_route, moe_sort, moe_unsort
    e, k, h, r = 12, 3, 96, 8
    g = torch.Generator().manual_seed(t)
    rnd = lambda *s: torch.randn(*s, generator=g).cuda()
    x, logits, w1 = rnd(t, h).bfloat16(), rnd(t, e), (rnd(e, h, h) / 10).bfloat16()
    a, b, s = (rnd(e, r, h) / 10).bfloat16(), (rnd(e, h, r) / 3).bfloat16(), torch.rand(e, generator=g).cuda() + 0.5
    w, ids = moe_route(logits, k)
    rows, routes = moe_sort(x, ids, e)
    mid, at = torch.zeros_like(rows), routes.offsets.tolist()
    for i in range(e):
        mid[at[i]:at[i + 1]] = rows[at[i]:at[i + 1]] @ w1[i].t()
    mid = lora_add(mid, rows, a, b, routes.experts, s, out=mid)
    out = moe_unsort(mid, w, routes)
    loss, counts = moe_balance_loss(logits, ids)
    assert torch.equal(counts, routes.offsets.diff()) and bool(torch.isfinite(loss))
    want = torch.zeros(t, h, dtype=torch.float64, device="cuda")
    tol, half = torch.zeros_like(want), 2.0 ** -8
    for j in range(k):
        i = ids[:, j].long()
        xd, f = x.double().unsqueeze(2), w[:, j].double().unsqueeze(1)
        dense = (w1[i].double() @ xd).squeeze(2)
        low = a[i].double() @ xd * s[i].double().reshape(-1, 1, 1)
        delta = (b[i].double() @ low).squeeze(2)
        want += f * (dense + delta)
        terms = (w1[i].double().abs() @ xd.abs()).squeeze(2) + (b[i].double().abs() @ (a[i].double().abs() @ xd.abs())).squeeze(2) * 1.5
        tol += f * (dense.abs() * half + (dense + delta).abs() * half * (1 + half) + terms * (3 * h * 2.0 ** -24 + 2.0 ** -16))
    tol = tol + want.abs() * half + 1e-6
    assert bool(((out.double() - want).abs() <= tol).all()), float(((out.double() - want).abs() / tol).max())


@pytest.mark.gpu
def test_a_training_step_of_a_routed_layer():
    """Gradients of router, experts and input through sort and unsort against 64-bit autograd of the plain form; fp32 products
    of whole numbers and weights of 1/8: exact."""
    from litevllm_amd import moe_sort, moe_unsort
    t, e, k, h = 33, 5, 2, 16
    x, w1 = _whole(40, t, h, size=2).requires_grad_(True), _whole(41, e, h, h, size=1).requires_grad_(True)
    w = (_whole(42, t, k) / 8).requires_grad_(True)
    ids, up = _ids(43, t, e, k, 0.15), _whole(44, t, h, size=1)
    rows, routes = moe_sort(x, ids, e)
    at = routes.offsets.tolist()
    mid = torch.cat([rows[at[i]:at[i + 1]] @ w1[i].t() for i in range(e)] + [rows[at[e]:]])
    out = moe_unsort(mid, w, routes)
    got = [out.detach(), *torch.autograd.grad(out, (x, w1, w), up)]
    xd, wd, gd = (v.detach().double().requires_grad_(True) for v in (x, w1, w))
    kept = ((ids >= 0) & (ids < e))
    y = torch.matmul(wd[ids.clamp(0, e - 1).long()], xd.unsqueeze(1).unsqueeze(3).expand(t, k, h, 1)).squeeze(3)
    ref = (y * (gd * kept).unsqueeze(2)).sum(1)
    want = [ref.detach(), *torch.autograd.grad(ref, (xd, wd, gd), up.double())]
    for a, b in zip(got, want):
        assert torch.equal(a.double(), b)


@pytest.mark.gpu
def test_a_backward_in_the_weights_alone_needs_only_the_rows():
    """dw = <dout, rows>: weights and offsets may change in front of it, as beside any product whose other factor is constant."""
    from litevllm_amd import moe_sort, moe_unsort
    x, w, ids, up = _whole(80, 30, 24), _whole(81, 30, 3).requires_grad_(True), _ids(82, 30, 7, 3, 0.2), _whole(83, 30, 24)
    rows, routes = moe_sort(x, ids, 7)
    want, = torch.autograd.grad(moe_unsort(rows, w, routes), w, up)
    out = moe_unsort(rows, w, routes)
    with torch.no_grad():
        w.mul_(3)
        routes.offsets.zero_()
    got, = torch.autograd.grad(out, w, up)
    assert torch.equal(got, want)
    rows, routes = moe_sort(x, ids, 7)
    out = moe_unsort(rows.requires_grad_(True), w, routes)  # rows' gradient needs them
    with torch.no_grad():
        w.mul_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, w, up)
