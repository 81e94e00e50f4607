"""The router's balance loss and its gradient against 64-bit formulas and differences."""
import ctypes

import pytest
import torch

from litevllm_amd import _lib as L

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _reference(z, ids, mask=None):
    """loss, counts, gradient, probabilities and F (the gradient is p (F - sum F p)) in 64 bits."""
    z, (t, e) = z.detach().double(), z.shape
    kept = torch.ones(t, dtype=torch.bool, device=z.device) if mask is None else mask
    n = max(1, int(kept.sum()))
    hit = ids[kept].flatten()
    hit = hit[(hit >= 0) & (hit < e)].long()
    counts = torch.zeros(e, dtype=torch.int64, device=z.device).index_add_(0, hit, torch.ones_like(hit))
    f = counts.double() / (n * ids.shape[1])
    empty = (z == -float("inf")).all(1)
    p = torch.softmax(torch.where(empty[:, None], torch.zeros_like(z), z), 1)
    p = torch.where((kept & ~empty)[:, None], p, torch.zeros_like(p))
    loss = e * (f * p.sum(0) / n).sum()
    F = e * f / n
    return loss, counts, p * (F - (p * F).sum(1, keepdim=True)), p, F


def _prob_error(z, mask=None):
    """Relative error of an fp32 softmax's values per row: exp2(x log2 e) carries 2 |x| + 8 half steps for x =
    z - max (the difference, the product, the function), the sum's relative error is at most the largest of
    its terms', plus the sum's and the quotient's own roundings (at most 32)."""
    z = z.detach().double()
    x = (z.amax(1, keepdim=True) - z).nan_to_num(0, 0, 0).clamp(max=110)
    return (2 * (2 * x.amax(1, keepdim=True) + 8) + 32) * 2.0 ** -24


def _case(seed, t, e, k, dtype, padding=0.0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(t, e, generator=g) * scale).to(DTYPES[dtype]).cuda()
    ids = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(t)]).int().cuda() if t else torch.zeros(0, k, dtype=torch.int32, device="cuda")
    mask = (torch.rand(t, generator=g) >= padding).cuda() if padding else None
    return z, ids, mask


def _check(z, ids, mask, upstream=1.0):
    from litevllm_amd import moe_balance_loss
    z = z.detach().requires_grad_(True)
    loss, counts = moe_balance_loss(z, ids, mask)
    rl, rc, rg, p, F = _reference(z, ids, mask)
    assert torch.equal(counts.long(), rc) and counts.dtype == torch.int32
    rel = _prob_error(z) if z.shape[0] else torch.zeros(1, 1)
    worst = float(rel.max()) if z.shape[0] else 0.0
    # a wave adds its rows' values in fp32: at most 512 of them
    assert abs(float(loss.detach()) - float(rl)) <= float(rl) * (worst + 516 * 2.0 ** -24)
    grad, = torch.autograd.grad(loss, z, torch.tensor(upstream, device="cuda"))
    assert grad.dtype == z.dtype and grad.shape == z.shape
    if not z.shape[0]:
        return grad
    dot = (p * F).sum(1, keepdim=True)
    # the hardware's exp2 gives 0 below the smallest normal number, 2^-126: a p = exp / sum with sum >= 1 is off
    # by at most that, and the gradient is p times at most F + dot
    tol = (p * (2 * rel.to(p.device) + 16 * 2.0 ** -24) + 2.0 ** -126) * (F + dot) * abs(upstream)
    f = torch.finfo(z.dtype)
    want = rg * upstream
    tol = tol + want.abs() * f.eps / 2 + f.smallest_normal * f.eps
    bad = (grad.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((grad.double() - want).abs() / tol).max()))
    if mask is not None:
        assert bool((grad[~mask] == 0).all())
    return grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("t,e,k,padding", [
    (1, 1, 1, 0.0), (1, 8, 2, 0.0), (3, 5, 5, 0.0), (64, 64, 8, 0.0), (65, 63, 3, 0.3), (130, 128, 2, 0.0), (200, 160, 6, 0.5),
    (515, 256, 8, 0.1), (33, 300, 4, 0.0), (40, 513, 2, 0.2), (9, 1024, 7, 0.0), (3000, 64, 8, 0.2), (20000, 60, 4, 0.0), (0, 8, 2, 0.0)])
def test_loss_counts_and_gradient(t, e, k, padding, dtype):
    z, ids, mask = _case(t + e, t, e, k, dtype, padding)
    _check(z, ids, mask, 1024.0 if dtype == "f16" else 0.37)


@pytest.mark.gpu
def test_masked_rows_are_not_read_and_a_mask_of_nothing():
    from litevllm_amd import moe_balance_loss
    z, ids, mask = _case(1, 90, 20, 3, "f32", 0.4)
    want = _check(z, ids, mask)
    dirty, wild = z.clone(), ids.clone()
    dirty[~mask] = float("nan")
    wild[~mask] = 12345678
    assert torch.equal(_check(dirty.masked_fill(torch.isnan(dirty), 0.0), ids, mask), want)
    d = dirty.requires_grad_(True)
    loss, counts = moe_balance_loss(d, wild, mask)
    assert torch.equal(loss, moe_balance_loss(z, ids, mask)[0]) and torch.equal(counts, moe_balance_loss(z, ids, mask)[1])
    assert torch.equal(torch.autograd.grad(loss, d)[0], want)
    none = torch.zeros_like(mask)
    loss, counts = moe_balance_loss(d, wild, none)
    assert float(loss.detach()) == 0.0 and int(counts.sum()) == 0
    assert bool((torch.autograd.grad(loss, d)[0] == 0).all())


@pytest.mark.gpu
def test_infinities_nan_large_logits_and_ids_out_of_range():
    from litevllm_amd import moe_balance_loss
    z, ids, _ = _case(2, 50, 70, 4, "f32", scale=20.0)
    z[3, 10:60] = -float("inf")   # experts that are switched off
    z[4] = -float("inf")          # nothing left
    z[5] = 3.0e38
    z[6] = -3.0e38
    z[7, 1:] = -float("inf")
    ids[8] = torch.tensor([-1, 70, 2 ** 31 - 1, 5])
    ids[9] = 6                    # one expert in every slot
    grad = _check(z, ids, None)
    assert bool((grad[4] == 0).all()) and bool((grad[3, 10:60] == 0).all())
    _check(z, ids.long() + (ids.long() < 0) * -(2 ** 40), None)
    for bad in (float("nan"), float("inf")):
        y = z.clone()
        y[2, 2] = bad
        y.requires_grad_(True)
        loss, counts = moe_balance_loss(y, ids)
        assert torch.isnan(loss) and torch.equal(counts.long(), _reference(z, ids)[1])
        g, = torch.autograd.grad(loss, y)
        keep = torch.arange(50, device="cuda") != 2
        assert torch.isnan(g[2]).all() and torch.equal(g[keep], _check(z, ids, None)[keep])


@pytest.mark.gpu
def test_the_gradient_against_differences():
    """The kernel's loss at z +- h d against the 64-bit loss there, and the 64-bit formula's gradient against
    the 64-bit differences: a loss near 1 carries its tolerance / h into a difference."""
    from litevllm_amd import moe_balance_loss
    z, ids, _ = _case(3, 6, 10, 2, "f32")
    ids[:4] = torch.tensor([1, 2], dtype=torch.int32)
    d = torch.randn(6, 10, generator=torch.Generator().manual_seed(4)).cuda()
    grad = _check(z, ids, None).double()
    h = 2.0 ** -6
    mine = (moe_balance_loss(z + h * d, ids)[0].double() - moe_balance_loss(z - h * d, ids)[0].double()) / (2 * h)
    far = [_reference(z + s * h * d, ids)[0] for s in (1, -1)]
    loss_tol = 2 * float(far[0]) * (float(_prob_error(z).max()) * 2 + 516 * 2.0 ** -24)
    assert abs(float(mine - (far[0] - far[1]) / (2 * h))) <= loss_tol / (2 * h)
    tiny = 2.0 ** -13
    q = (_reference(z.double() + tiny * d, ids)[0] - _reference(z.double() - tiny * d, ids)[0]) / (2 * tiny)
    # differences: third derivatives of at most 6 |d|^3 per row, over 6, times tiny^2
    slack = tiny ** 2 * float((d.abs().amax(1) ** 3).sum()) * float(_reference(z, ids)[4].max()) * 8
    assert abs(float((grad * d).sum() - q)) <= slack + 1e-5 * float((grad * d).abs().sum())


@pytest.mark.gpu
def test_strides_types_of_ids_and_no_gradient():
    from litevllm_amd import moe_balance_loss
    z, ids, mask = _case(5, 40, 24, 3, "bf16", 0.2)
    want = moe_balance_loss(z, ids, mask)
    wide = torch.zeros(80, 31, dtype=torch.bfloat16, device="cuda")
    wide[::2, 5:29] = z
    assert all(torch.equal(a, b) for a, b in zip(moe_balance_loss(wide[::2, 5:29], ids.long(), mask), want))
    assert all(torch.equal(a, b) for a, b in zip(moe_balance_loss(z.t().contiguous().t(), ids.t().contiguous().t(), mask), want))
    assert not want[0].requires_grad and not moe_balance_loss(z.requires_grad_(True), ids, mask)[1].requires_grad
    v = wide.requires_grad_(True)
    a, = torch.autograd.grad(moe_balance_loss(v[::2, 5:29], ids, mask)[0], v)
    b, = torch.autograd.grad(moe_balance_loss(z, ids, mask)[0], z)
    assert torch.equal(a[::2, 5:29], b) and int((a != 0).sum()) == int((b != 0).sum())


@pytest.mark.gpu
def test_upstream_accumulation_and_the_same_bits():
    from litevllm_amd import moe_balance_loss
    z, ids, mask = _case(6, 700, 96, 4, "f32", 0.3)
    z.requires_grad_(True)
    (3.0 * moe_balance_loss(z, ids, mask)[0] + moe_balance_loss(z, ids)[0]).backward()
    a, = torch.autograd.grad(moe_balance_loss(z, ids, mask)[0], z, torch.tensor(3.0, device="cuda"))
    b, = torch.autograd.grad(moe_balance_loss(z, ids)[0], z)
    assert torch.equal(z.grad, a + b) or torch.equal(z.grad, b + a)
    for _ in range(3):
        assert torch.equal(moe_balance_loss(z, ids, mask)[0], moe_balance_loss(z, ids, mask)[0])


@pytest.mark.gpu
def test_replays_and_another_stream():
    from litevllm_amd import moe_balance_loss
    z, ids, mask = _case(7, 900, 64, 8, "bf16", 0.2)
    graph = torch.cuda.CUDAGraph()
    up = torch.tensor(0.5, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = z.clone().requires_grad_(True)  # a leaf of its own: no eager graph of the captured one
        torch.autograd.grad(moe_balance_loss(warm, ids, mask)[0], warm, up)
        leaf = z.clone().requires_grad_(True)
        with torch.cuda.graph(graph, stream=side):
            loss, counts = moe_balance_loss(leaf, ids, mask)
            grad, = torch.autograd.grad(loss, leaf, up)
            loss = loss.detach()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(4):
        with torch.no_grad():
            leaf.copy_(z * (1 + i))
            mask.logical_not_()
        graph.replay()
        torch.cuda.synchronize()
        own = leaf.detach().clone().requires_grad_(True)
        want, c = moe_balance_loss(own, ids, mask)
        assert torch.equal(loss, want) and torch.equal(counts, c)
        assert torch.equal(grad, torch.autograd.grad(want, own, up)[0])


@pytest.mark.gpu
def test_refusals():
    from litevllm_amd import moe_balance_loss
    z, ids, mask = _case(8, 6, 8, 2, "f32", 0.5)
    for bad in (lambda: moe_balance_loss(z[0], ids), lambda: moe_balance_loss(z, ids[:5]), lambda: moe_balance_loss(z, ids[0]),
                lambda: moe_balance_loss(z, ids[:, :0]), lambda: moe_balance_loss(z, ids, mask[:5]),
                lambda: moe_balance_loss(z, ids, mask.int()), lambda: moe_balance_loss(z.cpu(), ids), lambda: moe_balance_loss(z[:, :0], ids),
                lambda: moe_balance_loss(torch.zeros(6, 1025, device="cuda"), ids)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: moe_balance_loss(z.double(), ids), lambda: moe_balance_loss(z, ids.short())):
        with pytest.raises(TypeError):
            bad()
    z.requires_grad_(True)
    loss, _ = moe_balance_loss(z, ids)
    g, = torch.autograd.grad(loss, z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_entries_refuse():
    lib = L.load()
    p = (ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p).value + 255) & ~255

    def call(z=p, ld=8, dt=L.DTYPE_F32, ids=p, bits=32, t=2, e=8, k=2, loss=p, ws=p, wsb=1 << 20):
        return lib.awq_w4a16_moe_balance(z, ld, dt, ids, bits, None, t, e, k, loss, p, p, ws, wsb, None)
    assert call(z=None) == call(ids=None) == call(loss=None) == L.ERR_NULL
    assert call(t=-1) == call(e=0) == call(k=0) == L.ERR_SHAPE
    assert call(dt=0) == call(bits=8) == call(e=1025, ld=1025) == L.ERR_UNSUPPORTED
    assert call(ld=7) == L.ERR_STRIDE
    assert call(ws=None) == call(wsb=4) == L.ERR_WORKSPACE

    def grad(z=p, ld=8, dt=L.DTYPE_F32, t=2, e=8, g=p):
        return lib.awq_w4a16_moe_balance_grad(z, ld, dt, None, p, p, g, t, e, None)
    assert grad(z=None) == grad(g=None) == L.ERR_NULL
    assert grad(t=-1) == grad(e=0) == L.ERR_SHAPE
    assert grad(dt=9) == grad(e=1025, ld=1025) == L.ERR_UNSUPPORTED
    assert grad(ld=3) == L.ERR_STRIDE
    assert grad(t=0) == L.OK


def test_entries_refuse_more_tokens_than_they_number():
    lib = L.load()
    p = (ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p).value + 255) & ~255
    for t, k in (((1 << 30) + 1, 1), ((1 << 31) - 1, 1), (1 << 29, 3)):
        need = lib.awq_w4a16_moe_balance_workspace_bytes(t, 1)
        assert lib.awq_w4a16_moe_balance(p, 1, L.DTYPE_F16, p, 32, None, t, 1, k, p, p, p, p, need, None) == L.ERR_UNSUPPORTED
        if t > 1 << 30:
            assert lib.awq_w4a16_moe_balance_grad(p, 1, L.DTYPE_F16, None, p, p, p, t, 1, None) == L.ERR_UNSUPPORTED


class _Hooks(torch.autograd.graph.saved_tensors_hooks):
    """Gives saved tensors back as copies made by `copy`."""

    def __init__(self, copy):
        super().__init__(lambda t: t, lambda t: copy(t) if t.dim() == 2 else t)


def _every_second_column(t):
    """A copy whose rows are not dense."""
    wide = torch.zeros(t.shape[0], 2 * t.shape[1], dtype=t.dtype, device=t.device)
    wide[:, ::2] = t
    return wide[:, ::2]


# copies of other strides than the original's
COPIES = {"dense": lambda t: t.contiguous().clone(), "wide": lambda t: torch.cat([t, t, t], 1)[:, t.shape[1]:2 * t.shape[1]],
          "transposed": lambda t: t.t().contiguous().t(), "apart": _every_second_column}


@pytest.mark.parametrize("copy", list(COPIES))
def test_the_backward_reads_saved_logits_by_their_own_strides(copy, monkeypatch):
    """Without a GPU, the launches replaced: hooks may give the logits back with other strides than they had."""
    from litevllm_amd import moe_balance as B
    calls = []
    monkeypatch.setattr(B, "_call", lambda dev, name, *args: calls.append((name, args)))
    monkeypatch.setattr(B.ops, "_require_device", lambda *t: torch.device("cpu"))
    seen = []

    def back(t):
        seen.append(COPIES[copy](t))
        return seen[-1]
    wide = torch.randn(6, 31, requires_grad=True)
    ids = torch.zeros(6, 2, dtype=torch.int32)
    with _Hooks(back):
        loss, _ = B.moe_balance_loss(wide[:, 5:29], ids)
    grad, = torch.autograd.grad(loss, wide)
    assert grad.shape == (6, 31)
    (first, forward), (second, backward) = calls
    assert first == "awq_w4a16_moe_balance" and forward[1] == 31
    assert second == "awq_w4a16_moe_balance_grad"
    z, ld = backward[0], backward[1]
    if copy in ("dense", "wide"):
        assert z == seen[0].data_ptr() and ld == seen[0].stride(0)
    else:
        assert ld == 24  # a dense copy of what came back


@pytest.mark.gpu
@pytest.mark.parametrize("copy", [*COPIES, "save_on_cpu"])
def test_gradient_under_saved_tensor_hooks(copy):
    from litevllm_amd import moe_balance_loss
    z, ids, mask = _case(15, 40, 24, 3, "f32", 0.2)
    wide = torch.zeros(80, 31, device="cuda")
    wide[::2, 5:29] = z
    wide.requires_grad_(True)
    kept = torch.stack([mask, ~mask], 1)[:, 0]  # every second byte
    want, = torch.autograd.grad(moe_balance_loss(wide[::2, 5:29], ids, kept)[0], wide)
    assert torch.equal(want[::2, 5:29], _check(z, ids, mask))
    with torch.autograd.graph.save_on_cpu() if copy == "save_on_cpu" else _Hooks(COPIES[copy]):
        loss, _ = moe_balance_loss(wide[::2, 5:29], ids, kept)
    assert torch.equal(torch.autograd.grad(loss, wide)[0], want)


@pytest.mark.gpu
def test_saved_tensors_that_come_back_elsewhere_or_as_others_are_refused():
    from litevllm_amd import moe_balance_loss
    z, ids, _ = _case(16, 6, 8, 2, "f32")
    z.requires_grad_(True)
    for back in (lambda t: t.cpu(), lambda t: t[:1], lambda t: t.half() if t.dim() == 1 else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            loss, _ = moe_balance_loss(z, ids)
        with pytest.raises((RuntimeError, ValueError)):
            loss.backward()


@pytest.mark.gpu
def test_sums_over_many_tokens():
    """2^27 equal rows.  Their probability, just below the middle between two fp32 numbers next to sums past 1024, is rounded
    down in every addition to such a sum: one chain of a lane's 8192 rows is off by 1.2e-4.  The bound: chains of 512, the 16 of
    them, the 16 waves, and the blocks' sums in fp64."""
    import math

    from litevllm_amd import moe_balance_loss
    t = 1 << 27
    p = 0.25 + 0.49 * 2.0 ** -13
    row = torch.tensor([math.log(p / (1 - p)), 0.0], device="cuda")
    z = row.expand(t, 2).contiguous()
    loss, counts = moe_balance_loss(z, torch.zeros(t, 1, dtype=torch.int32, device="cuda"))
    assert counts.tolist() == [t, 0]
    want = 2 * float(torch.softmax(row.double(), 0)[0])
    tol = float(_prob_error(row.unsqueeze(0)).max()) + (512 + 16 + 16 + 2) * 2.0 ** -24
    assert abs(float(loss) - want) <= want * tol, (float(loss) / want - 1, tol)
