"""Low-rank adapters of many requests against 64-bit products."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from litevllm_amd import _lib as L

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _whole(g, *shape, size=2):
    return torch.randint(-size, size + 1, shape, generator=g).float().cuda()


def _ids(g, m, adapters, requests, without):
    """Ids of the rows: requests one after another; some without an adapter, by negative ids or ids past the last."""
    which = torch.randint(adapters, (requests,), generator=g)
    none = torch.tensor([-1, adapters, 2 ** 31 - 1, -2 ** 31])[torch.randint(4, (requests,), generator=g)]
    which = torch.where(torch.rand(requests, generator=g) < without, none, which)
    cuts = torch.randperm(max(m - 1, 1), generator=g)[:requests - 1] + 1
    return which[(torch.arange(m).unsqueeze(1) >= cuts).sum(1)].int().cuda()


def _reference(base, x, a, b, ids, scales):
    out = torch.zeros(*x.shape[:-1], b.shape[1], dtype=torch.float64, device=x.device) if base is None else base.double()
    for l in torch.unique(ids).tolist():
        if 0 <= l < a.shape[0]:
            low = x[ids == l].double() @ a[l].double().t().contiguous()
            out[ids == l] += (1.0 if scales is None else scales[l].double()) * (low @ b[l].double().t().contiguous())
    return out


def _check_exact(base, x, a, b, ids, scales):
    """Whole numbers whose sums fp32 holds, and whose 16-bit halves are exact: one right value."""
    from litevllm_amd import lora_add
    want = _reference(base, x, a, b, ids, scales)
    for l in torch.unique(ids).tolist():
        if 0 <= l < a.shape[0]:
            assert float((x[ids == l].double() @ a[l].double().t().contiguous()).abs().max()) * (1.0 if scales is None else float(scales[l])) < 2 ** 15
    assert float(want.abs().max()) < 2 ** 15
    got = lora_add(base, x, a, b, ids, scales)
    assert got.dtype == x.dtype and got.shape == want.shape
    bad = got != want.to(x.dtype)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist())
    return got


CASES = [  # rows, requests, K, N, rank, adapters, without
    (1, 1, 64, 64, 8, 1, 0.0), (1, 1, 4096, 4096, 16, 8, 0.0), (1, 1, 33, 17, 1, 2, 0.0), (1, 1, 5, 3, 3, 1, 0.0), (2, 2, 100, 130, 64, 4, 0.0),
    (7, 7, 72, 520, 16, 9, 0.3), (16, 16, 1024, 255, 32, 16, 0.0), (17, 3, 257, 300, 12, 5, 0.4), (29, 29, 2001, 501, 12, 16, 0.2),
    (64, 64, 512, 640, 32, 64, 0.1), (128, 20, 200, 96, 100, 7, 0.2), (129, 129, 130, 70, 24, 40, 0.2), (300, 5, 640, 333, 8, 20, 0.2),
    (513, 4, 96, 1100, 16, 3, 0.3), (600, 9, 128, 256, 256, 4, 0.2), (700, 700, 64, 48, 20, 30, 0.3), (1500, 6, 328, 700, 64, 4, 0.2),
    (2049, 3, 1000, 80, 130, 2, 0.4), (40, 40, 12288, 64, 16, 3, 0.0), (5, 5, 64, 24580, 16, 6, 0.2),
    (100, 2, 4096, 520, 64, 4, 0.3), (96, 1, 12288, 300, 16, 1, 0.0), (33, 2, 9000, 1030, 40, 2, 0.0), (128, 128, 5000, 40, 24, 5, 0.2),
    (16, 1, 12288, 4100, 128, 1, 0.0), (100, 3, 7, 90, 5, 2, 0.2), (20, 2, 6, 300, 200, 2, 0.2), (200, 200, 300, 200, 64, 30, 0.1),
    (1100, 1100, 64, 72, 64, 50, 0.1), (64, 1, 600, 24600, 16, 1, 0.0),
    (512, 512, 128, 256, 256, 9, 0.1), (511, 2, 5000, 70, 40, 3, 0.1), (520, 520, 300, 200, 64, 30, 0.1), (600, 3, 7, 90, 5, 2, 0.2),
    (700, 3, 6, 50, 200, 2, 0.2), (514, 3, 1025, 65, 64, 3, 0.2),
    (300, 300, 40, 24, 8, 1024, 0.1), (300, 300, 40, 27, 8, 1025, 0.1), (400, 400, 64, 40, 16, 1, 0.5), (512, 512, 64, 100, 16, 2, 0.3),
    (129, 129, 64, 33, 64, 3, 0.3), (257, 40, 1000, 65, 8, 600, 0.1), (500, 500, 7, 30, 20, 3, 0.3), (480, 480, 4100, 300, 64, 30, 0.1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,requests,k,n,r,adapters,without", CASES)
def test_whole_numbers(m, requests, k, n, r, adapters, without, dtype):
    g, dt = torch.Generator().manual_seed(m + k + n + r), DTYPES[dtype]
    x, base = _whole(g, m, k, size=1).to(dt), _whole(g, m, n, size=100).to(dt)
    # few values that are not zero: |x A^T| stays below 2^8
    a = (_whole(g, adapters, r, k, size=1) * (torch.rand(adapters, r, k, generator=g) < 1500 / k).cuda()).to(dt)
    b = (_whole(g, adapters, n, r, size=1) * (torch.rand(adapters, n, r, generator=g) < 0.5).cuda()).to(dt)
    ids = _ids(g, m, adapters, requests, without)
    scales = 2.0 ** torch.randint(0, 3, (adapters,), generator=g).float().cuda()
    _check_exact(base, x, a, b, ids, scales)
    got = _check_exact(None, x, a, b, ids.long(), None)
    assert bool((got[(ids < 0) | (ids >= adapters)] == 0).all())


def _check_random(base, x, a, b, ids, scales):
    """fp32 sums of K and R terms, products of the scale and the two halves (16 bits for bf16), and one rounding."""
    from litevllm_amd import lora_add
    want = _reference(base, x, a, b, ids, scales)
    terms = _reference(None, x.abs(), a.abs(), b.abs(), ids, scales)
    f, k, r = torch.finfo(x.dtype), a.shape[2], a.shape[1]
    halves = 2.0 ** -17 if x.dtype == torch.bfloat16 else 2.0 ** -22
    tol = terms * ((k + r + 8) * 2.0 ** -23 + halves) + want.abs() * f.eps / 2 + f.smallest_normal * f.eps
    got = lora_add(base, x, a, b, ids, scales)
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,requests,k,n,r,adapters,without", [(3, 3, 200, 300, 16, 4, 0.0), (50, 50, 96, 200, 40, 9, 0.2), (640, 4, 130, 99, 8, 4, 0.2)])
def test_random_values(m, requests, k, n, r, adapters, without, dtype):
    g, dt = torch.Generator().manual_seed(m), DTYPES[dtype]
    rnd = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    ids, scales = _ids(g, m, adapters, requests, without), torch.rand(adapters, generator=g).cuda() + 0.3
    _check_random(rnd(m, n), rnd(m, k), rnd(adapters, r, k), rnd(adapters, n, r), ids, scales)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_ranges_of_the_low_rank_values(dtype):
    """x A^T past fp16's largest value, below its smallest, and both in one row."""
    dt, g = DTYPES[dtype], torch.Generator().manual_seed(1)
    m, k, n, r = 20, 64, 70, 16
    rnd = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    ids = torch.zeros(m, dtype=torch.int32, device="cuda")
    x, a, b = rnd(m, k), rnd(1, r, k), rnd(1, n, r)
    _check_random(None, x * 500, a * 500, b * 2.0 ** -12, ids, None)
    _check_random(None, x * 2.0 ** -10, a * 2.0 ** -10, b * 500, ids, None)
    mixed = a.clone()
    mixed[0, ::2] *= 400
    mixed[0, 1::2] *= 2.0 ** -7
    _check_random(None, x * 400, mixed, b * 2.0 ** -10, ids, None)
    _check_random(None, x, a, b, ids, torch.tensor([2.0 ** 20], device="cuda") if dt == torch.bfloat16 else torch.tensor([2.0 ** 5], device="cuda"))
    _check_random(rnd(m, n), torch.zeros_like(x), a, b, ids, None)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [4, 64])
@pytest.mark.parametrize("m", [2, 100, 200, 600])
def test_low_rank_values_above_the_largest_bf16(m, k):
    """1.9996 * 2^127 rounds to infinity in bf16 but not in fp32; B takes it down again."""
    from litevllm_amd import lora_add
    x, a, b = torch.zeros(m, k), torch.zeros(1, 2, k), torch.zeros(1, 24, 2)
    x[:, 0], a[0, 0, 0], a[0, 1, 0], b[:, :, 0], b[:, ::2, 1] = 1.4140625 * 2.0 ** 63, 1.4140625 * 2.0 ** 64, -2.0 ** -60, 2.0 ** -100, 8.0
    x, a, b = (t.bfloat16().cuda() for t in (x, a, b))
    for sign in (1, -1):
        got = lora_add(None, x * sign, a, b, torch.zeros(m, dtype=torch.int32, device="cuda"))
        low = x.double() * sign @ a[0].double().t().contiguous()
        assert torch.equal(got, (low @ b[0].double().t().contiguous()).bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [30, 700])
def test_infinities_and_nan_stay_in_their_rows(m):
    from litevllm_amd import lora_add
    g = torch.Generator().manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()
    x, a, b, base = rnd(m, 72), rnd(3, 16, 72), rnd(3, 90, 16), rnd(m, 90)
    ids = torch.arange(m, dtype=torch.int32, device="cuda") % 4 - 1  # -1: no adapter
    want = lora_add(base, x, a, b, ids)
    x[5, 3], x[9, 70], base[6, 2] = float("inf"), float("nan"), float("inf")
    x[8] = float("nan")                    # a row without an adapter: x is not needed
    bad_a, bad_b = a.clone(), b.clone()
    bad_a[2], bad_b[2] = float("nan"), float("inf")
    got = lora_add(base, x, bad_a, bad_b, ids)
    assert int(ids[8]) == -1
    clean = (ids != 2)
    clean[[5, 6, 9]] = False
    assert torch.equal(got[clean], want[clean])
    assert not bool(torch.isfinite(got[5]).any()) or int(ids[5]) == -1
    assert bool(torch.isnan(got[9]).all()) == (int(ids[9]) >= 0)
    assert got[6, 2] == float("inf") or int(ids[6]) == 2
    assert not bool(torch.isfinite(got[ids == 2]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [20, 600])
def test_in_place_slices_and_strides(m):
    from litevllm_amd import lora_add
    g = torch.Generator().manual_seed(3)
    k, n, r, adapters = 100, 90, 12, 5
    x, base = _whole(g, m, k).half(), _whole(g, m, n, size=50).half()
    a, b = _whole(g, adapters, r, k, size=1).half(), _whole(g, adapters, n, r, size=1).half()
    ids = _ids(g, m, adapters, min(m, 30), 0.3)
    want = _check_exact(base, x, a, b, ids, None)
    y = base.clone()
    assert lora_add(y, x, a, b, ids, out=y) is y and torch.equal(y, want)
    # columns of one projection's output, parts of stacked adapters
    wide = torch.full((m, 3 * n + 1), 7.0, dtype=torch.float16, device="cuda")
    q = wide[:, n + 1:2 * n + 1]
    q.copy_(base)
    stack_a, stack_b = torch.cat([a * 3, a, a], 1), torch.cat([b, b * 3], 1)
    lora_add(q, x, stack_a[:, r:2 * r], stack_b[:, :n], ids, out=q)
    assert torch.equal(q, want) and bool((wide[:, :n + 1] == 7).all()) and bool((wide[:, 2 * n + 1:] == 7).all())
    # another part of the same memory
    wide[:, :n].copy_(base)
    lora_add(wide[:, :n], x, a, b, ids, out=wide[:, 5:n + 5])
    assert torch.equal(wide[:, 5:n + 5], want)
    # over x
    both = torch.zeros(m, 128, dtype=torch.float16, device="cuda")
    both[:, 20:120].copy_(x)
    lora_add(base, both[:, 20:120], a, b, ids, out=both[:, :n])
    assert torch.equal(both[:, :n], want)
    spread = torch.zeros(2 * m, 2 * k, dtype=torch.float16, device="cuda")
    spread[::2, ::2] = x
    t = lambda v: v.transpose(-1, -2).contiguous().transpose(-1, -2)
    assert torch.equal(lora_add(t(base), spread[::2, ::2], t(a), t(b), ids.repeat_interleave(2)[::2], None), want)
    assert torch.equal(lora_add(base, x, a[:1].expand(adapters, r, k), b[:1].expand(adapters, n, r), ids), lora_add(base, x, a[:1], b[:1], torch.where((ids >= 0) & (ids < adapters), 0, -1).int()))
    assert torch.equal(lora_add(base.view(2, m // 2, n), x.view(2, m // 2, k), a, b, ids.view(2, m // 2)), want.view(2, m // 2, n))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 100, 200, 1000])
@pytest.mark.parametrize("n,r", [(1, 1), (1, 256), (7, 16), (8, 9), (8, 1), (15, 1), (16, 40)])
def test_few_columns(m, n, r):
    """Fewer columns than a piece has, or than B's last piece reaches over."""
    g = torch.Generator().manual_seed(20 + m + n + r)
    x, a, b, base = _whole(g, m, 40).half(), _whole(g, 3, r, 40, size=1).half(), _whole(g, 3, n, r, size=1).half(), _whole(g, m, n).half()
    ids = _ids(g, m, 3, min(m, 5), 0.2)
    _check_exact(base, x, a, b, ids, None)
    _check_exact(None, x, a, b, ids, None)


@pytest.mark.gpu
def test_no_rows_no_columns():
    from litevllm_amd import lora_add
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
    ids = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert lora_add(z(0, 8), z(0, 16), z(2, 4, 16), z(2, 8, 4), ids).shape == (0, 8)
    assert lora_add(z(3, 0), z(3, 16), z(2, 4, 16), z(2, 0, 4), torch.zeros(3, dtype=torch.int32, device="cuda")).shape == (3, 0)
    assert lora_add(z(8) + 3, z(16), z(2, 4, 16), z(2, 8, 4), torch.tensor(-1, device="cuda")).tolist() == [3.0] * 8


@pytest.mark.gpu
def test_operands_past_4_gib():
    from litevllm_amd import lora_add
    g = torch.Generator().manual_seed(4)
    adapters, r, k, n = 1100, 256, 8200, 16
    a = torch.zeros(adapters, r, k, dtype=torch.float16, device="cuda")
    assert a.numel() * 2 > 2 ** 32
    a[-1], a[0] = _whole(g, r, k, size=1).half(), 1.0
    b = torch.zeros(adapters, n, r, dtype=torch.float16, device="cuda")
    b[-1] = 1.0
    x = torch.zeros(3, k, dtype=torch.float16, device="cuda")
    x[:, ::97] = 1.0
    ids = torch.tensor([adapters - 1, 0, adapters - 1], dtype=torch.int32, device="cuda")
    want = a[-1][:, ::97].double().sum()
    got = lora_add(None, x, a, b, ids)
    assert torch.equal(got.double(), torch.stack([want, want * 0, want]).unsqueeze(1).expand(3, n))
    del a, b
    m, n = 80000, 32768  # the result
    x, a, b = _whole(g, m, 32, size=1).half(), _whole(g, 2, 4, 32, size=1).half(), _whole(g, 2, n, 4, size=1).half()
    ids = (torch.arange(m, device="cuda") >= 70000).int()
    got = lora_add(None, x, a, b, ids)
    assert got.numel() * 2 > 2 ** 32
    for rows in (slice(0, 200), slice(69900, 70100), slice(m - 200, m)):
        assert torch.equal(got[rows], _reference(None, x[rows], a, b, ids[rows], None).half())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 50, 600])
def test_the_same_bits_replays_and_another_stream(m):
    from litevllm_amd import lora_add
    g = torch.Generator().manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()
    x, base, a, b = rnd(m, 520), rnd(m, 300), rnd(4, 16, 520), rnd(4, 300, 16)
    ids, scales = _ids(g, m, 4, m, 0.2), torch.rand(4, generator=g).cuda()
    want = lora_add(base, x, a, b, ids, scales)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(lora_add(base, x, a, b, ids, scales), want)
        with torch.cuda.graph(graph, stream=side):
            got = lora_add(base, x, a, b, ids, scales)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        x.mul_(0.5)
        ids.copy_((ids + 1).clamp(-1, 3))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, lora_add(base, x, a, b, ids, scales))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 100, 600])
def test_two_calls_at_once_and_replays_in_place(m):
    from litevllm_amd import LoRAAdapters
    g = torch.Generator().manual_seed(30)
    x, a, b, base = _whole(g, m, 5000, size=1).half(), _whole(g, 4, 80, 5000, size=1).half(), _whole(g, 4, 600, 80, size=1).half(), _whole(g, m, 600).half()
    x[:, torch.rand(5000, generator=g).cuda() > 0.02] = 0
    layer, ids = LoRAAdapters(a, b), _ids(g, m, 4, m, 0.2)
    others = (ids + 1).clamp(-1, 3)
    want = [_check_exact(base, x, a, b, i, None) for i in (ids, others)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    with torch.inference_mode():
        for _ in range(8):
            for s, i, to in zip(streams, (ids, others), got):
                with torch.cuda.stream(s):
                    to.append(layer.add(base, x, i))
    torch.cuda.synchronize()
    for to, w in zip(got, want):
        assert all(torch.equal(t, w) for t in to)
    y, graph = base.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.add(y, x, ids, out=y)
    for _ in range(3):
        again = layer.add(y, x, ids)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, again)


@pytest.mark.gpu
def test_a_row_does_not_depend_on_its_neighbours_adapters():
    from litevllm_amd import lora_add
    g = torch.Generator().manual_seed(6)
    rnd = lambda *s: torch.randn(*s, generator=g).half().cuda()
    x, a, b, ids = rnd(48, 300), rnd(6, 16, 300), rnd(6, 100, 16), _ids(g, 48, 6, 48, 0.0)
    want, order = lora_add(None, x, a, b, ids), torch.randperm(48, generator=g).cuda()
    assert torch.equal(lora_add(None, x[order], a, b, ids[order]), want[order])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["awq", "symmetric", "mxfp4", "dense"])
def test_layers_with_adapters(kind):
    """AWQConfig.apply adds a layer's adapters to what it gives without them: half a step of the result's type beside the sums."""
    from litevllm_amd import AWQConfig, LoRAAdapters, mxfp4_quantize
    from oracle.gen import make_awq_problem
    m, k, n, adapters = 24, 256, 384, 3
    g = torch.Generator().manual_seed(7)
    rnd = lambda *s: torch.randn(*s, generator=g).half().cuda()
    cfg, layer = AWQConfig(group_size=128, layout="autoawq"), SimpleNamespace(prefix="model.layers.0.self_attn.o_proj", bias=None)
    if kind in ("awq", "symmetric"):
        p = make_awq_problem(M=m, K=k, N=n, group_size=128, seed=5)
        layer.qweight, layer.scales = (torch.from_numpy(p[i]).cuda() for i in ("qweight", "scales"))
        layer.qzeros = torch.from_numpy(p["qzeros"]).cuda() if kind == "awq" else None
    elif kind == "mxfp4":
        layer.qweight, layer.scales = mxfp4_quantize(rnd(n, k))
    else:
        layer.qweight, layer.weight = None, rnd(n, k) * 0.05
    layer.lora_adapters = LoRAAdapters.stack([(rnd(r, k) * 0.05, rnd(n, r), s) for r, s in ((8, 2.0), (16, 0.5), (5, 1.0))])
    assert layer.lora_adapters.lora_a.shape == (adapters, 16, k) and layer.lora_adapters.scales.tolist() == [2.0, 0.5, 1.0]
    x, ids = rnd(2, m // 2, k), _ids(g, m, adapters, m, 0.3).view(2, m // 2)
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            plain = cfg.apply(layer, x)
            got = cfg.apply(layer, x, lora_ids=ids)
        a, b, s = layer.lora_adapters.lora_a.data, layer.lora_adapters.lora_b.data, layer.lora_adapters.scales.data
        want = _reference(plain, x, a, b, ids, s)
        terms = _reference(None, x.abs(), a.abs(), b.abs(), ids, s)
        assert got.shape == plain.shape
        assert bool(((got.double() - want).abs() <= want.abs() * 2.0 ** -11 + terms * ((k + 24) * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -25).all())
        assert torch.equal(got[(ids < 0) | (ids >= adapters)], plain[(ids < 0) | (ids >= adapters)])
    layer.lora_adapters = layer.lora_adapters.half()  # scales as well: these are the same numbers in fp16
    assert torch.equal(cfg.apply(layer, x, lora_ids=ids), got)
    layer.lora_adapters = None
    assert torch.equal(cfg.apply(layer, x, lora_ids=ids), plain)


@pytest.mark.gpu
def test_derivatives_are_refused():
    from litevllm_amd import lora_add
    g = torch.Generator().manual_seed(8)
    t = [_whole(g, 6, 40).half(), _whole(g, 6, 32).half(), _whole(g, 2, 4, 32).half(), _whole(g, 2, 40, 4).half(), torch.ones(2, device="cuda")]
    ids = torch.zeros(6, dtype=torch.int32, device="cuda")
    want = lora_add(*t[:4], ids, t[4])
    for i in range(5):
        u = [v.clone().requires_grad_(j == i) for j, v in enumerate(t)]
        y = lora_add(*u[:4], ids, u[4])
        assert torch.equal(y, want) and y.requires_grad
        with pytest.raises(RuntimeError, match="not differentiable"):
            y.sum().backward()
        with pytest.raises(RuntimeError):
            lora_add(*u[:4], ids, u[4], out=torch.empty_like(want))
        with torch.no_grad():
            assert not lora_add(*u[:4], ids, u[4]).requires_grad


@pytest.mark.gpu
def test_a_backward_notices_what_out_overwrote():
    from litevllm_amd import lora_add
    g = torch.Generator().manual_seed(10)
    x, y, a, b = _whole(g, 6, 32).half(), _whole(g, 6, 40).half(), _whole(g, 2, 4, 32).half(), _whole(g, 2, 40, 4).half()
    w = torch.ones(6, 40, dtype=torch.float16, device="cuda", requires_grad=True)
    loss = (w * y).sum()
    lora_add(y, x, a, b, torch.zeros(6, dtype=torch.int32, device="cuda"), out=y)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():
        z = y.clone()
        assert lora_add(z, x, a, b, torch.zeros(6, dtype=torch.int32, device="cuda"), out=z) is z


@pytest.mark.gpu
def test_refusals():
    from litevllm_amd import LoRAAdapters, lora_add
    g = torch.Generator().manual_seed(9)
    base, x, a, b = _whole(g, 6, 40).half(), _whole(g, 6, 32).half(), _whole(g, 2, 4, 32).half(), _whole(g, 2, 40, 4).half()
    ids, s = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda")
    big = torch.zeros(1, 257, 32, dtype=torch.float16, device="cuda")
    for bad in (lambda: lora_add(base, x, a[0], b, ids), lambda: lora_add(base, x, a, b[0], ids), lambda: lora_add(base, x, a[:1], b, ids),
                lambda: lora_add(base, x, a[:, :3], b, ids), lambda: lora_add(base, x[:, :31], a, b, ids), lambda: lora_add(base[:5], x, a, b, ids),
                lambda: lora_add(base[:, :39], x, a, b, ids), lambda: lora_add(base, x, a, b, ids[:5]), lambda: lora_add(base, x, a, b, ids.unsqueeze(1)),
                lambda: lora_add(base, x, a, b, ids, s.half()), lambda: lora_add(base, x, a, b, ids, s[:1]), lambda: lora_add(base, x, a[:0], b[:0], ids),
                lambda: lora_add(base, x, big, torch.zeros(1, 40, 257, dtype=torch.float16, device="cuda"), ids),
                lambda: lora_add(base, x, a[:, :0], b[:, :, :0], ids), lambda: lora_add(base, x[:, :0], a[:, :, :0], b, ids),
                lambda: lora_add(base, x.cpu(), a, b, ids), lambda: lora_add(base, x, a, b, ids.cpu()),
                lambda: lora_add(base, x, a, b, ids, out=base[:5]), lambda: lora_add(base, x, a, b, ids, out=torch.empty(40, 6, dtype=torch.float16, device="cuda").t()),
                lambda: lora_add(base, x, a, b, ids, out=torch.empty(1, 40, dtype=torch.float16, device="cuda").expand(6, 40)),
                lambda: lora_add(base.view(2, 3, 40), x.view(2, 3, 32), a, b, ids.view(2, 3), out=torch.empty(3, 2, 40, dtype=torch.float16, device="cuda").transpose(0, 1)),
                lambda: LoRAAdapters.stack([]), lambda: LoRAAdapters.stack([(a[0], b[0], 1.0), (a[0, :, :8], b[0], 1.0)])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: lora_add(base, x.float(), a, b, ids), lambda: lora_add(base.bfloat16(), x, a, b, ids), lambda: lora_add(base, x, a.float(), b, ids),
                lambda: lora_add(base, x, a, b.bfloat16(), ids), lambda: lora_add(base, x, a, b, ids.float()),
                lambda: lora_add(base, x, a, b, ids, out=base.float())):
        with pytest.raises(TypeError):
            bad()


def test_entry_refuses():
    lib = L.load()
    p = (ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p).value + 255) & ~255

    def call(base=p, ldb=8, x=p, ldx=8, a=p, sa=32, b=p, sb=32, ids=p, bits=32, out=p, ldo=8, m=2, n=8, k=8, r=4, l=2, dt=L.DTYPE_F16, ws=p, wsb=1 << 20):
        return lib.awq_w4a16_lora_add(base, ldb, x, ldx, a, sa, b, sb, ids, bits, None, out, ldo, m, n, k, r, l, dt, ws, wsb, None)
    assert call(x=None) == call(a=None) == call(b=None) == call(ids=None) == call(out=None) == L.ERR_NULL
    assert call(m=-1) == call(n=-1) == call(k=0) == call(r=0) == call(l=0) == L.ERR_SHAPE
    assert call(dt=L.DTYPE_F32) == call(bits=8) == call(r=257, sa=1 << 20, sb=1 << 20) == L.ERR_UNSUPPORTED
    assert call(m=(1 << 30) + 1) == call(n=(1 << 24) + 1, ldo=1 << 25, ldb=1 << 25, sb=1 << 40) == L.ERR_UNSUPPORTED
    assert call(m=(1 << 24) + 1) == L.ERR_UNSUPPORTED and lib.awq_w4a16_lora_workspace_bytes((1 << 24) + 1, 8, 4) == 0
    assert call(ldx=7) == call(ldo=7) == call(ldb=7) == call(sa=31) == call(sb=31) == call(x=p + 1) == call(out=p + 1) == L.ERR_STRIDE
    need = lib.awq_w4a16_lora_workspace_bytes(600, 8, 4)
    assert need > 0 and call(m=600, ws=None) == call(m=600, wsb=need - 1) == L.ERR_WORKSPACE
    assert call(m=600, ws=p + 4) == L.ERR_STRIDE
    assert call(m=0) == call(n=0) == L.OK
    for m, k, r in ((0, 8, 4), (-1, 8, 4), (2, 0, 4), (2, 8, 0), (2, 8, 257), ((1 << 30) + 1, 8, 4), (2, (1 << 24) + 1, 4)):
        assert lib.awq_w4a16_lora_workspace_bytes(m, k, r) == 0


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.float16),
                                  lambda m: torch.nn.ModuleList([m]).bfloat16()[0], lambda m: m.double().half(), lambda m: m.half().float()])
def test_scales_keep_their_bits_when_the_module_is_cast(cast):
    """16 / 12 is not a bf16 number, and 2^20 is past fp16's range."""
    from litevllm_amd import LoRAAdapters
    layer = LoRAAdapters.stack([(torch.ones(12, 8), torch.ones(10, 12), 16 / 12), (torch.ones(4, 8), torch.ones(10, 4), 2.0 ** 20)])
    want, state = layer.scales.detach().clone(), {k: v.clone() for k, v in layer.state_dict().items()}
    got = cast(layer)
    assert got.scales.dtype == torch.float32 and torch.equal(got.scales, want) and not got.scales.requires_grad
    assert isinstance(got.scales, torch.nn.Parameter) and [k for k, _ in got.named_parameters()] == ["lora_a", "lora_b", "scales"]
    got.load_state_dict(state)
    assert torch.equal(got.scales, want)
    assert cast(LoRAAdapters(torch.ones(1, 4, 8), torch.ones(1, 10, 4))).scales is None


def test_scales_follow_the_module_to_another_device():
    from litevllm_amd import LoRAAdapters
    layer = LoRAAdapters(torch.ones(1, 4, 8), torch.ones(1, 10, 4), torch.ones(1)).to("meta", torch.bfloat16)
    assert layer.scales.is_meta and layer.scales.dtype == torch.float32 and layer.lora_a.dtype == torch.bfloat16
    assert layer.to_empty(device="cpu").scales.shape == (1,)


@pytest.mark.gpu
def test_out_that_a_backward_goes_through_is_refused():
    """A result that a graph already holds would keep the derivative of what was there before."""
    from litevllm_amd import lora_add
    g = torch.Generator().manual_seed(11)
    x, base, a, b = _whole(g, 6, 32).half(), _whole(g, 6, 40).half(), _whole(g, 2, 4, 32).half(), _whole(g, 2, 40, 4).half()
    ids, w = torch.zeros(6, dtype=torch.int32, device="cuda"), torch.ones(6, 40, dtype=torch.float16, device="cuda", requires_grad=True)
    want, y = lora_add(base, x, a, b, ids), w * 2
    for out in (w, y, y[:]):
        before = out.detach().clone()
        with pytest.raises(RuntimeError, match="require a gradient"):
            lora_add(base, x, a, b, ids, out=out)
        assert torch.equal(out.detach(), before)
    y.sum().backward()
    assert bool((w.grad == 2).all())
    with torch.no_grad():
        assert torch.equal(lora_add(base, x, a, b, ids, out=w), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("r", [16, 40])
@pytest.mark.parametrize("m,k", [(3, 64), (100, 4200), (600, 64), (1, 5), (600, 5)])
def test_low_rank_values_far_apart(m, k, r, dtype):
    """Values of v a factor of up to 2^34 apart in a row, columns of B that are zero at the large ones.  Each is off by
    2^-17 of itself in bf16; in fp16 by 2^-22 of itself or 2^-38 of the largest of the 16 or 32 ranks beside it (its low half
    ends at 2^-24 where that largest is 2^13 at least), whichever is more.  Every rank has an input of its own, so v is one product."""
    from litevllm_amd import lora_add
    g, dt, n = torch.Generator().manual_seed(m + r), DTYPES[dtype], 90
    at = torch.arange(r) % k                                 # a rank's input
    steps = (torch.arange(r) * 7 % 18).double()
    mantissa = lambda *s: 1 + torch.rand(*s, generator=g, dtype=torch.float64)
    x, a, b = torch.zeros(m, k, dtype=torch.float64), torch.zeros(1, r, k, dtype=torch.float64), torch.zeros(1, n, r, dtype=torch.float64)
    scale = torch.zeros(k, dtype=torch.float64)
    scale[at] = 9 - steps                                     # ranks that share an input (k < r) have one exponent of it
    x[:] = mantissa(m, k) * 2.0 ** scale
    a[0, torch.arange(r), at] = mantissa(r) * 2.0 ** (9 - steps)
    one = torch.arange(n) % r                                 # a column's rank; some have more
    b[0, torch.arange(n), one] = mantissa(n) * 2.0 ** (steps - 11 - scale[at])[one]  # v B is about 1/4
    b[0, ::5, :] += (torch.rand(n, r, generator=g, dtype=torch.float64) < 0.1)[::5] * 2.0 ** -18
    x, a, b = (t.to(dt).cuda() for t in (x, a, b))
    ids = torch.zeros(m, dtype=torch.int32, device="cuda")
    want = _reference(None, x, a, b, ids, None)
    v = (x.double() @ a[0].double().t().contiguous()).abs()
    w, f = 16 if r <= 16 else 32, torch.finfo(dt)
    top = torch.cat([v[:, i:i + w].amax(1, keepdim=True).expand(m, min(w, r - i)) for i in range(0, r, w)], 1)
    off = v * 2.0 ** -17 if dt == torch.bfloat16 else torch.maximum(v * 2.0 ** -22, top * 2.0 ** -38)
    weight = b[0].double().abs().t().contiguous()
    terms = v @ weight
    tol = off @ weight + terms * (r + 8) * 2.0 ** -23 + want.abs() * f.eps / 2 + f.smallest_normal * f.eps
    got = lora_add(None, x, a, b, ids)
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,k,r", [(29, 12288, 12), (100, 4096, 64), (300, 5000, 40)])
def test_a_row_among_other_neighbours(m, k, r, dtype):
    """Two launches: which blocks share K, and so the order of fp32 sums, follows the adapters of the batch.  A row keeps its
    value but for those sums, each within _check_random's bound of the exact value."""
    from litevllm_amd import lora_add
    g, dt, n = torch.Generator().manual_seed(m), DTYPES[dtype], 72
    rnd = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    x, base, a, b = rnd(m, k), rnd(m, n), rnd(m, r, k), rnd(m, n, r)
    own, shared = torch.arange(m, device="cuda"), torch.full((m,), 5, device="cuda")
    shared[m // 2:] = 3
    for ids in (own, shared, own.flip(0), torch.where(own == 5, 5, -1)):
        got = _check_random(base, x, a, b, ids, None)
        assert torch.equal(lora_add(base, x, a, b, ids), got)
    order = torch.randperm(m, generator=g).cuda()
    _check_random(base[order], x[order], a, b, shared[order], None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("m,requests,n,r", [(1400, 5, 24581, 20), (1401, 60, 24576, 64), (530, 3, 65003, 130), (1100, 2, 32011, 16), (9000, 40, 4100, 7)])
def test_results_that_pass_the_caches(m, requests, n, r, dtype):
    """2^25 results and more from a base, with rows of no adapter and odd columns; in place the same."""
    from litevllm_amd import lora_add
    g, dt, adapters, k = torch.Generator().manual_seed(m), DTYPES[dtype], 7, 64
    assert m * n >= 2 ** 25
    x, a, b = _whole(g, m, k, size=1).to(dt), _whole(g, adapters, r, k, size=1).to(dt), _whole(g, adapters, n, r, size=1).to(dt)
    base, ids = _whole(g, m, n, size=100).to(dt), _ids(g, m, adapters, requests, 0.3)
    got = _check_exact(base, x, a, b, ids, None)
    assert torch.equal(lora_add(base, x, a, b, ids, out=base), got)
    wide = torch.full((m, n + 9), 7.0, dtype=dt, device="cuda")  # rows apart, at other alignments
    lora_add(None, x, a, b, ids, out=wide[:, 4:n + 4])
    assert bool((wide[:, :4] == 7).all()) and bool((wide[:, n + 4:] == 7).all())
    want = _reference(None, x, a, b, ids, None)
    assert torch.equal(wide[:, 4:n + 4], want.to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["awq", "symmetric", "mxfp4", "dense"])
def test_layers_with_adapters_take_the_types_of_the_adapters(kind):
    """bf16 as fp16; rows of 32 bits, which dense layers and unpacked int4 take, are refused instead of rounded, and so are
    adapters of another type than the rows."""
    from litevllm_amd import AWQConfig, LoRAAdapters, mxfp4_quantize
    from oracle.gen import make_awq_problem
    m, k, n = 24, 256, 384
    g = torch.Generator().manual_seed(12)
    rnd = lambda *s: torch.randn(*s, generator=g).cuda()
    cfg, layer = AWQConfig(group_size=128, layout="autoawq"), SimpleNamespace(prefix="model.layers.0.self_attn.o_proj", bias=None)
    if kind in ("awq", "symmetric"):
        p = make_awq_problem(M=m, K=k, N=n, group_size=128, seed=5)
        layer.qweight, layer.scales = (torch.from_numpy(p[i]).cuda() for i in ("qweight", "scales"))
        layer.qzeros = torch.from_numpy(p["qzeros"]).cuda() if kind == "awq" else None
    elif kind == "mxfp4":
        layer.qweight, layer.scales = mxfp4_quantize(rnd(n, k))
    else:
        layer.qweight, layer.weight = None, (rnd(n, k) * 0.05).bfloat16()
    layer.lora_adapters = LoRAAdapters.stack([(rnd(8, k) * 0.05, rnd(n, 8), 2.0), (rnd(12, k) * 0.05, rnd(n, 12), 0.7)]).bfloat16()
    x, ids = rnd(m, k).bfloat16(), _ids(g, m, 2, m, 0.3)
    with torch.no_grad():
        plain = cfg.apply(layer, x)
        got = cfg.apply(layer, x, lora_ids=ids)
    assert plain.dtype == got.dtype == torch.bfloat16
    a, b, s = layer.lora_adapters.lora_a.data, layer.lora_adapters.lora_b.data, layer.lora_adapters.scales.data
    want, terms = _reference(plain, x, a, b, ids, s), _reference(None, x.abs(), a.abs(), b.abs(), ids, s)
    tol = want.abs() * 2.0 ** -8 + terms * ((k + 20) * 2.0 ** -23 + 2.0 ** -17) + 2.0 ** -130
    assert bool(((got.double() - want).abs() <= tol).all())
    for rows in (x.float(), x.half()):
        if kind == "dense":
            layer.weight = layer.weight.to(rows.dtype)
        if kind != "mxfp4" or rows.dtype == torch.float16:
            cfg.apply(layer, rows)  # without ids it is taken
            with pytest.raises(TypeError):
                cfg.apply(layer, rows, lora_ids=ids)


def test_calls_without_ids_do_not_look_for_adapters():
    """A missing attribute of a module costs a call about 1 us."""
    from litevllm_amd import AWQConfig

    class Layer(torch.nn.Module):
        bias, looked = None, 0

        @property
        def lora_adapters(self):
            self.looked += 1
    layer = Layer()
    layer._quant_weight = SimpleNamespace(matmul=lambda x, bias, config: x)
    x = torch.ones(1, 8)
    assert AWQConfig().apply(layer, x) is x and layer.looked == 0
    assert AWQConfig().apply(layer, x, lora_ids=torch.zeros(1, dtype=torch.int32)) is x and layer.looked == 1
