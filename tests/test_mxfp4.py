"""MXFP4 quantisation, linear layers and expert stacks against plain 64-bit implementations."""
import ctypes

import pytest
import torch

import mx_reference as R
from litevllm_amd import _lib as L

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _made(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _weight(seed, *shape):
    """codes, scales (GPU) of a random matrix, and its 64-bit values."""
    c, s = R.quantize(_made(seed, *shape, scale=0.05).cuda())
    return c, s, R.values(c, s)


def _close(y, ref, off, dtype):
    err, tol = (y.double() - ref).abs(), off + R.half_step(ref.abs() + off, dtype)
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp(min=1e-300)).max()):.3f} of the tolerance"


# ------------------------------------------------------------------ the C entry points, before any launch
def _fake(n=4096):
    return (ctypes.cast(ctypes.create_string_buffer(n), ctypes.c_void_p).value + 255) & ~255


def test_quantize_entries_refuse():
    lib, p = L.load(), _fake()
    for fn, extra in ((lib.awq_w4a16_mxfp4_quantize, (32,)), (lib.awq_w4a16_mxfp4_dequantize, None)):
        def call(a=p, b=p, c=p, m=1, k=32, dt=L.DTYPE_F16):
            return fn(a, 32, b, c, m, k, dt, None) if extra else fn(a, b, c, m, k, dt, None)
        assert call(a=None) == L.ERR_NULL
        assert call(k=48) == L.ERR_SHAPE
        assert call(m=-1) == L.ERR_SHAPE
        assert call(dt=L.DTYPE_NONE) == L.ERR_UNSUPPORTED
        assert call(a=p + 8) == L.ERR_STRIDE
        assert call(m=0) == L.OK
        assert call(k=0) == L.OK
    assert lib.awq_w4a16_mxfp4_quantize(p, 33, p, p, 2, 32, L.DTYPE_F16, None) == L.ERR_STRIDE


def test_gemm_entry_refuses():
    lib, p = L.load(), _fake()

    def call(a=p, lda=64, sa=None, w=p, sw=p, bias=None, c=p, ldc=16, m=20, n=16, k=64, dt=L.DTYPE_BF16, bdt=L.DTYPE_NONE, ws=p, wsb=4096):
        return lib.awq_w4a16_mxfp4_gemm(a, lda, sa, w, sw, bias, c, ldc, m, n, k, dt, bdt, ws, wsb, None)
    assert call(a=None) == call(w=None) == call(sw=None) == call(c=None) == L.ERR_NULL
    assert call(k=48) == call(k=0) == call(m=-1) == L.ERR_SHAPE
    assert call(dt=L.DTYPE_F32) == call(bdt=L.DTYPE_F16) == call(bias=p) == L.ERR_UNSUPPORTED
    assert call(ldc=8) == call(lda=60) == call(lda=32) == call(w=p + 4) == call(ws=p + 16) == L.ERR_STRIDE
    assert call(ws=None) == call(wsb=8) == L.ERR_WORKSPACE
    assert call(m=0) == call(n=0) == L.OK


def test_moe_entry_refuses():
    lib, p = L.load(), _fake()

    def call(x=p, ldx=64, ids=p, bits=32, wdt=L.DTYPE_F32, gu=p, dn=p, out=p, ldo=64, t=2, h=64, i=32, e=4, k=2, act=0,
             dt=L.DTYPE_F16, ws=p, wsb=1 << 20):
        return lib.awq_w4a16_mxfp4_moe(x, ldx, ids, bits, p, wdt, gu, p, dn, p, out, ldo, t, h, i, e, k, act, dt, ws, wsb, None)
    assert call(x=None) == call(ids=None) == call(gu=None) == call(out=None) == L.ERR_NULL
    assert call(h=48) == call(i=48) == call(e=0) == call(k=0) == L.ERR_SHAPE
    assert call(bits=16) == call(wdt=0) == call(act=7) == call(dt=L.DTYPE_F32) == call(e=1025) == L.ERR_UNSUPPORTED
    assert call(ldx=60) == call(ldo=32) == call(gu=p + 8) == L.ERR_STRIDE
    assert call(ws=None) == call(wsb=64) == L.ERR_WORKSPACE
    assert call(t=0) == L.OK


def test_the_reference_rounds_to_nearest_even():
    x = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -5.0, 0.2501, 4.0] + [0.0] * 20)
    c, s = R.quantize(x)
    assert s.tolist() == [127]
    assert R.values(c, s)[:12].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, 0, -4, 0.5, 4]


# ------------------------------------------------------------------ quantisation
def _hard_rows(dtype):
    """Rows of 64 whose blocks hold ties, saturation, subnormals, zeros, one value, the largest values."""
    f = torch.finfo(dtype)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0, 7.9, 4.0, 0.0, -0.0, 0.1, 2.0, 3.0]).repeat(2)
    rows = [ties.repeat(2), torch.zeros(64), torch.full((64,), f.max), torch.full((64,), f.smallest_normal * f.eps),
            ties.repeat(2) * f.smallest_normal, -ties.repeat(2) * 2.0 ** 10]
    one = torch.zeros(64)
    one[37] = -3.3
    return torch.stack([*rows, one, torch.full((64,), f.smallest_normal)]).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (1, 4096), (257, 1056), (2, 3, 64), (64,), (0, 64), (5, 0), (4000, 32)])
def test_quantize_is_the_nearest_code(dtype, shape):
    from litevllm_amd import mxfp4_dequantize, mxfp4_quantize
    x = _made(1, *shape, scale=3.0).to(DTYPES[dtype])
    if x.numel() and x.dim() > 1:
        x.view(-1, x.shape[-1])[::3] *= 2.0 ** -13
    x = x.cuda()
    codes, scales = mxfp4_quantize(x)
    c, s = R.quantize(x) if x.numel() else (codes, scales)
    assert torch.equal(scales, s) and torch.equal(codes, c)
    for out in DTYPES.values():
        assert torch.equal(mxfp4_dequantize(codes, scales, out), R.values(c, s).to(out))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_quantize_hard_values(dtype):
    from litevllm_amd import mxfp4_dequantize, mxfp4_quantize
    x = _hard_rows(DTYPES[dtype]).cuda()
    codes, scales = mxfp4_quantize(x)
    c, s = R.quantize(x)
    assert torch.equal(scales, s) and torch.equal(codes, c)
    assert torch.equal(mxfp4_dequantize(codes, scales, torch.float32), R.values(c, s).float())


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_nan_or_infinity_stands_for_nan(bad):
    from litevllm_amd import mxfp4_dequantize, mxfp4_quantize
    x = _made(2, 3, 96).cuda()
    x[1, 40] = bad
    codes, scales = mxfp4_quantize(x)
    assert scales[1].tolist()[1] == 255 and int((scales == 255).sum()) == 1
    c, s = R.quantize(x)
    assert torch.equal(codes, c) and torch.equal(scales, s)
    v = mxfp4_dequantize(codes, scales, torch.float32)
    assert torch.isnan(v[1, 32:64]).all() and int(torch.isnan(v).sum()) == 32


@pytest.mark.gpu
def test_dequantize_every_code_and_scale():
    from litevllm_amd import mxfp4_dequantize
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1).cuda()
    codes = (torch.arange(16, dtype=torch.uint8) * 17).repeat(256, 1).cuda()
    v = R.values(codes, scales)
    for dt in DTYPES.values():
        got = mxfp4_dequantize(codes, scales, dt)
        assert torch.equal(torch.isnan(got), torch.isnan(v))
        assert torch.equal(torch.nan_to_num(got, 0, 1, -1), torch.nan_to_num(v.float().to(dt), 0, 1, -1))


@pytest.mark.gpu
def test_quantize_strided_and_unaligned():
    from litevllm_amd import mxfp4_quantize
    big = _made(3, 20, 200).cuda()
    for x in (big[:, :96], big[:, 8:104], big[:, 3:99], big[::2, :64], big.t()[:, :0], big[:, :32].t().contiguous().t(), big[4:5, 5:69]):
        codes, scales = mxfp4_quantize(x)
        if not x.numel():
            assert codes.numel() == 0
            continue
        c, s = R.quantize(x.contiguous())
        assert torch.equal(codes, c) and torch.equal(scales, s)


@pytest.mark.gpu
def test_quantize_refuses():
    from litevllm_amd import mxfp4_dequantize, mxfp4_quantize
    with pytest.raises(ValueError):
        mxfp4_quantize(torch.zeros(4, 48, device="cuda"))
    with pytest.raises(TypeError):
        mxfp4_quantize(torch.zeros(4, 64, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError):
        mxfp4_quantize(torch.zeros(4, 64))
    c, s = mxfp4_quantize(torch.zeros(4, 64, device="cuda"))
    with pytest.raises(ValueError):
        mxfp4_dequantize(c, s[:, :1])
    with pytest.raises(ValueError):
        mxfp4_dequantize(c[:3], s)
    with pytest.raises(TypeError):
        mxfp4_dequantize(c.int(), s)
    with pytest.raises(TypeError):
        mxfp4_dequantize(c, s, torch.int32)


# ------------------------------------------------------------------ the product
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k,bias", [
    (1, 16, 32, None), (1, 1, 64, "f32"), (1, 4096, 4096, None), (2, 333, 1056, "f16"), (5, 48, 96, None), (13, 1000, 2048, "bf16"),
    (16, 256, 12288, None), (17, 128, 512, None), (33, 517, 160, "f32"), (57, 1024, 4096, None), (64, 256, 1024, None),
    (65, 130, 2080, "f16"), (128, 512, 384, None), (200, 5001, 288, "bf16"), (300, 256, 4128, None), (513, 771, 1024, None),
    (1030, 2048, 512, "f32"), (2100, 1100, 256, None), (2100, 2111, 288, "f16"), (4100, 4203, 96, None), (4000, 4300, 800, "bf16"), (8, 20000, 256, None), (129, 1, 32, None), (64, 300, 4096, "f16"), (40, 5000, 12320, None), (15, 16500, 96, None), (12, 9000, 4128, "f32"), (600, 900, 2080, None),
    (700, 24010, 96, "bf16"), (690, 24000, 544, None), (2500, 20007, 64, "f32"),
    (300, 4001, 5152, "f16"), (630, 4100, 1056, None),
    (17, 1, 32, None), (100, 500, 2080, "bf16"), (33, 4096, 992, None), (250, 257, 4128, "f32"), (1000, 64, 544, "f16"), (31, 2000, 8224, None)])
def test_gemm(m, n, k, bias, dtype):
    from litevllm_amd import mxfp4_gemm
    dt = DTYPES[dtype]
    x = _made(m + 1, m, k).to(dt).cuda()
    c, s, w = _weight(n, n, k)
    b = _made(7, n, scale=2.0).to(DTYPES[bias]).cuda() if bias else None
    y = mxfp4_gemm(x, c, s, bias=b)
    assert y.dtype == dt and y.shape == (m, n)
    ref, off = R.gemm(R.rounded(x), w, b)
    _close(y, ref, off, dt)
    assert torch.equal(y, mxfp4_gemm(x, c, s, bias=b))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 7, 40, 100, 700])
def test_gemm_of_quantised_activations_equals_that_of_the_activations(m):
    from litevllm_amd import MXFP4Weight, mxfp4_gemm, mxfp4_quantize
    x = _made(5, m, 544).half().cuda()
    c, s, _ = _weight(6, 300, 544)
    qa, sa = mxfp4_quantize(x)
    y = mxfp4_gemm(x, c, s)
    assert torch.equal(mxfp4_gemm(qa, c, s, a_scales=sa, out_dtype=torch.float16), y)
    assert torch.equal(MXFP4Weight(c, s).matmul(x.view(1, m, 544)), y.view(1, m, 300))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 9, 48, 260])
def test_gemm_far_apart_scales_and_nan(m):
    """Scales 2^-60 .. 2^60 (an operand in 16 bits between would lose them), and NaN blocks, whose row or
    column alone is NaN."""
    from litevllm_amd import mxfp4_gemm
    n, k = 70, 416
    g = torch.Generator().manual_seed(9)
    a, w = (torch.randint(0, 256, (r, k // 2), generator=g).to(torch.uint8).cuda() for r in (m, n))
    sa, sw = (torch.randint(60, 64, (r, k // 32), generator=g).to(torch.uint8).cuda() for r in (m, n))
    sw = sw + 126
    ref, off = R.gemm(R.values(a, sa), R.values(w, sw))
    y = mxfp4_gemm(a, w, sw, a_scales=sa, out_dtype=torch.bfloat16)
    _close(y, ref, off, torch.bfloat16)
    sa[m // 2, 5] = 255
    sw[33, 12] = 255
    y2 = mxfp4_gemm(a, w, sw, a_scales=sa, out_dtype=torch.bfloat16)
    nan = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    nan[m // 2], nan[:, 33] = True, True
    assert torch.equal(torch.isnan(y2), nan)
    assert torch.equal(y2[~nan], y[~nan])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 4, 31, 90, 520])
def test_gemm_strides_and_what_lies_around_the_output(m):
    from litevllm_amd import mxfp4_gemm
    n, k = 203, 128
    big = _made(11, 2 * m + 2, 400).half().cuda()
    c, s, w = _weight(12, n, k)
    for x in (big[:m, :k], big[1:m + 1, 5:5 + k], big[::2, 16:16 + k][:m], big[:m, :k].t().contiguous().t()):
        room = torch.full((m + 2, n + 9), -7.0, dtype=torch.float16, device="cuda")
        out = room[1:m + 1, 4:4 + n]
        got = mxfp4_gemm(x, c, s, out=out)
        assert got is out
        _close(out, *R.gemm(R.rounded(x.contiguous()), w), torch.float16)
        room[1:m + 1, 4:4 + n] = -7.0
        assert bool((room == -7.0).all())
    # weights behind another matrix, and as a slice of columns
    wide = torch.cat([c, c], 1)
    assert torch.equal(mxfp4_gemm(big[:m, :k], wide[:, k // 2:], s), mxfp4_gemm(big[:m, :k], c, s))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 3, 16, 80])
def test_gemm_over_its_own_input_and_beside_it(m):
    from litevllm_amd import mxfp4_gemm, mxfp4_quantize
    g = torch.Generator().manual_seed(11)
    k = n = 1024
    w, ws = mxfp4_quantize(torch.randn(n, k, generator=g).cuda())
    x = torch.randn(m, k, generator=g).to(torch.bfloat16).cuda()
    want = mxfp4_gemm(x, w, ws)
    for _ in range(4):
        a = x.clone()
        assert mxfp4_gemm(a, w, ws, out=a) is a and torch.equal(a, want)
        both = torch.cat([x, x], 1)
        mxfp4_gemm(both[:, :k], w, ws, out=both[:, k:])
        assert torch.equal(both[:, :k], x) and torch.equal(both[:, k:], want)


@pytest.mark.gpu
def test_gemm_over_a_part_of_its_input_held_by_another_tensor():
    from litevllm_amd import mxfp4_gemm, mxfp4_quantize
    g = torch.Generator().manual_seed(13)
    w, ws = mxfp4_quantize(torch.randn(1024, 1024, generator=g).cuda())
    x = torch.randn(5, 1024, generator=g).to(torch.bfloat16).cuda()
    want = mxfp4_gemm(x[1:], w, ws)
    for _ in range(4):
        buf = x.clone()
        out = torch.from_dlpack(buf[:4])
        mxfp4_gemm(buf[1:], w, ws, out=out)
        assert torch.equal(buf[:4], want) and torch.equal(buf[4], x[4])


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 8, 60])
def test_moe_over_its_own_input(t):
    from litevllm_amd import MXFP4Experts, mxfp4_moe, mxfp4_quantize
    g = torch.Generator().manual_seed(12)
    e, k, h, i = 4, 2, 512, 256
    gu = MXFP4Experts(*mxfp4_quantize(torch.randn(e, 2 * i, h, generator=g).cuda()))
    dn = MXFP4Experts(*mxfp4_quantize(torch.randn(e, h, i, generator=g).cuda()))
    x = torch.randn(t, h, generator=g).to(torch.bfloat16).cuda()
    ids = torch.randint(0, e, (t, k), generator=g).cuda()
    w = torch.rand(t, k, generator=g).cuda()
    want = mxfp4_moe(x, w, ids, gu, dn)
    assert torch.equal(mxfp4_moe(x, w, ids, gu, dn, out=x), want) and torch.equal(x, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 40, 300])
def test_gemm_with_a_weight_past_4_gib(m):
    """The columns at the weight's end, whose codes lie past 2^32 bytes; the rest of it is zeros."""
    from litevllm_amd import mxfp4_gemm
    n, k, last = 530000, 16384, 70
    w = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    ws = torch.full((n, k // 32), 127, dtype=torch.uint8, device="cuda")
    assert w.numel() > 1 << 32
    c, s, wv = _weight(31, last, k)
    w[-last:], ws[-last:] = c, s
    x = _made(32, m, k, dtype=torch.bfloat16).cuda()
    y = mxfp4_gemm(x, w, ws)
    ref, off = R.gemm(R.rounded(x), wv)
    _close(y[:, -last:], ref, off, torch.bfloat16)
    assert not bool(y[:, :-last].any())


@pytest.mark.gpu
def test_activations_past_4_gib():
    """Rows at the end of an input whose codes pass 2^32 bytes: quantised, multiplied and brought back."""
    from litevllm_amd import mxfp4_dequantize, mxfp4_gemm, mxfp4_quantize
    m, n, k, last = 530000, 48, 16384, 300
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-last:] = _made(33, last, k, dtype=torch.bfloat16).cuda()
    codes, scales = mxfp4_quantize(x)
    c, s = R.quantize(x[-last:])
    assert codes.numel() > 1 << 32 and torch.equal(codes[-last:], c) and torch.equal(scales[-last:], s)
    wc, wsc, wv = _weight(34, n, k)
    ref, off = R.gemm(R.values(c, s), wv)
    for y in (mxfp4_gemm(x, wc, wsc), mxfp4_gemm(codes, wc, wsc, a_scales=scales, out_dtype=torch.bfloat16)):
        _close(y[-last:], ref, off, torch.bfloat16)
        assert not bool(y[:-last].any())
    back = mxfp4_dequantize(codes, scales, torch.bfloat16)
    assert torch.equal(back[-last:].double(), R.values(c, s)) and not bool(back[:-last].any())


@pytest.mark.gpu
def test_gemm_refuses_and_empty():
    from litevllm_amd import mxfp4_gemm, mxfp4_quantize
    c, s, _ = _weight(1, 32, 64)
    x = torch.zeros(3, 64, device="cuda", dtype=torch.float16)
    for bad in (lambda: mxfp4_gemm(x[:, :32], c, s), lambda: mxfp4_gemm(x[0], c, s), lambda: mxfp4_gemm(x, c, s[:, :1]),
                lambda: mxfp4_gemm(x, c, s, bias=torch.zeros(31, device="cuda")), lambda: mxfp4_gemm(x.cpu(), c, s),
                lambda: mxfp4_gemm(x, c, s, out=torch.empty(3, 31, device="cuda", dtype=torch.float16)),
                lambda: mxfp4_gemm(x, c, s, out=torch.empty(32, 3, device="cuda", dtype=torch.float16).t()),
                lambda: mxfp4_gemm(x, c, s, out=torch.empty(3, 32, device="cuda")),
                lambda: mxfp4_gemm(x, c, s, out_dtype=torch.bfloat16),
                lambda: mxfp4_gemm(*([mxfp4_quantize(x)[0], c, s] + [mxfp4_quantize(x)[1]]))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: mxfp4_gemm(x.float(), c, s), lambda: mxfp4_gemm(x, c.int(), s)):
        with pytest.raises(TypeError):
            bad()
    assert mxfp4_gemm(x[:0], c, s).shape == (0, 32)
    assert mxfp4_gemm(x, c[:0], s[:0]).shape == (3, 0)


@pytest.mark.gpu
def test_gemm_other_stream_and_replays():
    """Two captured graphs, replayed in turn with eager work between, and a side stream."""
    from litevllm_amd import mxfp4_gemm
    c, s, _ = _weight(21, 512, 1024)
    xs = [_made(30 + m, m, 1024).half().cuda() for m in (1, 20, 150)]
    want = [mxfp4_gemm(x, c, s) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [mxfp4_gemm(x, c, s) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = mxfp4_gemm(x, c, s)
        graphs.append((g, y))
    for i in range(4):
        for x, (g, y) in zip(xs, graphs):
            x.mul_(-1.5 if i % 2 else 2.0)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, mxfp4_gemm(x, c, s))


# ------------------------------------------------------------------ experts
def _experts(seed, e, i, h):
    from litevllm_amd import MXFP4Experts
    c1, s1, w1 = _weight(seed, e, 2 * i, h)
    c2, s2, w2 = _weight(seed + 1, e, h, i)
    return MXFP4Experts(c1, s1), MXFP4Experts(c2, s2), w1 * 1.0, w2


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("t,e,k,h,i,kind", [
    (1, 8, 2, 64, 32, "silu"), (1, 1, 1, 32, 32, "gelu"), (5, 8, 8, 160, 96, "silu"), (17, 4, 2, 256, 128, "gelu_pytorch_tanh"),
    (40, 64, 4, 512, 64, "silu"), (70, 3, 2, 96, 160, "silu"), (150, 2, 1, 128, 32, "silu"), (3, 5, 4, 4128, 64, "silu"), (16, 1, 8, 64, 64, "gelu"), (2, 300, 3, 96, 32, "silu"), (128, 7, 1, 64, 32, "silu"),
    (43, 1000, 3, 64, 32, "silu"), (6, 9, 3, 4096, 288, "silu"), (2, 4, 2, 4224, 32, "gelu"), (1400, 3, 3, 32, 32, "silu"), (260, 5, 3, 64, 288, "gelu"),
    (600, 64, 8, 1024, 320, "silu"), (1200, 40, 8, 544, 608, "silu"), (900, 5, 8, 1056, 96, "gelu"),
    (32, 1, 1, 96, 64, "silu"), (30, 1, 1, 4128, 32, "silu"), (8, 2, 4, 288, 320, "gelu"), (33, 4, 1, 64, 96, "silu"), (700, 6, 8, 64, 32, "silu"),
    (8, 64, 8, 2048, 544, "silu"), (5, 33, 11, 2112, 96, "gelu"), (9, 20, 4, 1056, 1824, "silu"), (40, 16, 11, 96, 64, "silu"),
    (70000, 20, 4, 64, 32, "silu")])
def test_moe(t, e, k, h, i, kind, dtype):
    from litevllm_amd import mxfp4_moe
    dt = DTYPES[dtype]
    gu, dn, w1, w2 = _experts(t, e, i, h)
    x = (_made(t + 3, t, h) * 4).to(dt).cuda()
    g = torch.Generator().manual_seed(t)
    ids = torch.randint(0, e, (t, k), generator=g)
    weights = torch.rand(t, k, generator=g)
    y = mxfp4_moe(x, weights.cuda(), ids.int().cuda(), gu, dn, activation=kind)
    ref, off = R.moe(x, weights, ids, w1, w2, "silu" if kind == "silu" else "gelu")
    _close(y, ref, off, dt)
    for _ in range(3):  # the places of the routes may differ, the result may not
        assert torch.equal(y, mxfp4_moe(x, weights.cuda(), ids.cuda(), gu, dn, activation=kind))


@pytest.mark.gpu
def test_moe_ids_without_an_expert_an_expert_twice_and_an_idle_token():
    from litevllm_amd import mxfp4_moe
    gu, dn, w1, w2 = _experts(50, 6, 64, 128)
    x = _made(51, 6, 128).half().cuda() * 4
    ids = torch.tensor([[0, 0, 0], [-1, 6, 2], [-1, -1, 99], [5, 4, 5], [2 ** 40, 1, -2 ** 40], [3, 3, -7]])
    weights = torch.tensor([[0.5, 0.25, 0.25]] * 6).half()
    weights[2] = float("nan")  # without an expert a weight is not read
    y = mxfp4_moe(x, weights.cuda(), ids.cuda(), gu, dn)
    ref, off = R.moe(x, weights, ids, w1, w2, "silu")
    _close(y, ref, off, torch.float16)
    assert bool((y[2] == 0).all())
    none = mxfp4_moe(x, weights.cuda(), torch.full_like(ids, -1).cuda(), gu, dn)
    assert bool((none == 0).all())
    big = _made(52, 12, 200).half().cuda()
    room = torch.full((8, 131), -7.0, dtype=torch.float16, device="cuda")
    xs = big[::2, 8:136]
    mxfp4_moe(xs, weights[:6].cuda(), ids[[0, 1, 0, 3, 4, 5]].int().cuda().clamp(-1, 6), gu, dn, out=room[1:7, 2:130])
    want = mxfp4_moe(xs.contiguous(), weights.cuda(), ids[[0, 1, 0, 3, 4, 5]].int().cuda().clamp(-1, 6), gu, dn)
    assert torch.equal(torch.nan_to_num(room[1:7, 2:130]), torch.nan_to_num(want))
    room[1:7, 2:130] = -7.0
    assert bool((room == -7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,i", [(40, 64, 1, 96, 64), (20, 40, 3, 4128, 32), (7, 50, 9, 2080, 96), (300, 12, 2, 64, 64), (64, 32, 1, 288, 544)])
def test_moe_all_routes_to_one_expert_and_none_to_any(t, e, k, h, i):
    from litevllm_amd import mxfp4_moe
    gu, dn, w1, w2 = _experts(61, e, i, h)
    x = _made(62, t, h, dtype=torch.bfloat16).cuda()
    weights = torch.rand(t, k, generator=torch.Generator().manual_seed(63)).cuda()
    ids = torch.full((t, k), e - 2, dtype=torch.int32, device="cuda")
    y = mxfp4_moe(x, weights, ids, gu, dn)
    ref, off = R.moe(x, weights, ids, w1, w2, "silu")
    _close(y, ref, off, torch.bfloat16)
    assert torch.equal(y, mxfp4_moe(x, weights, ids.long(), gu, dn))
    for none in (-1, e):
        out = torch.full_like(x, 7.0)
        mxfp4_moe(x, weights, torch.full_like(ids, none), gu, dn, out=out)
        assert not bool(out.any())


@pytest.mark.gpu
def test_moe_nan_stays_with_its_token():
    from litevllm_amd import mxfp4_moe
    gu, dn, _, _ = _experts(60, 4, 64, 96)
    x = _made(61, 40, 96).bfloat16().cuda()
    ids = torch.randint(0, 4, (40, 2), generator=torch.Generator().manual_seed(1)).cuda()
    w = torch.rand(40, 2).cuda()
    y = mxfp4_moe(x, w, ids, gu, dn)
    x[7, 50] = float("inf")
    z = mxfp4_moe(x, w, ids, gu, dn)
    assert torch.isnan(z[7]).all()
    keep = torch.arange(40, device="cuda") != 7
    assert torch.equal(z[keep], y[keep])


@pytest.mark.gpu
def test_moe_refuses_and_empty():
    from litevllm_amd import MXFP4Experts, mxfp4_moe
    gu, dn, _, _ = _experts(70, 4, 32, 64)
    x = torch.zeros(3, 64, device="cuda", dtype=torch.float16)
    ids, w = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, 2, device="cuda")
    for bad in (lambda: mxfp4_moe(x[:, :32], w, ids, gu, dn), lambda: mxfp4_moe(x, w[:2], ids, gu, dn),
                lambda: mxfp4_moe(x, w, ids[:2], gu, dn), lambda: mxfp4_moe(x, w, ids, dn, gu),
                lambda: mxfp4_moe(x, w, ids, gu, MXFP4Experts(dn.qweight[:3], dn.scales[:3])),
                lambda: mxfp4_moe(x, w, ids, gu, dn, activation="relu"),
                lambda: mxfp4_moe(x, w, ids, gu, dn, out=torch.empty(3, 32, device="cuda", dtype=torch.float16))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: mxfp4_moe(x.float(), w, ids, gu, dn), lambda: mxfp4_moe(x, w, ids.short(), gu, dn),
                lambda: mxfp4_moe(x, w.double(), ids, gu, dn)):
        with pytest.raises(TypeError):
            bad()
    assert mxfp4_moe(x[:0], w[:0], ids[:0], gu, dn).shape == (0, 64)
    assert bool((mxfp4_moe(x, w[:, :0], ids[:, :0], gu, dn) == 0).all())


@pytest.mark.gpu
def test_moe_replays_and_streams():
    from litevllm_amd import mxfp4_moe
    gu, dn, _, _ = _experts(80, 16, 64, 256)
    graphs = []
    for t in (2, 90):
        x = _made(t, t, 256).half().cuda()
        g = torch.Generator().manual_seed(t)
        ids, w = torch.randint(0, 16, (t, 4), generator=g).cuda(), torch.rand(t, 4, generator=g).cuda()
        mxfp4_moe(x, w, ids, gu, dn)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mxfp4_moe(x, w, ids, gu, dn)
        graphs.append((graph, x, ids, w, y))
    for i in range(4):
        for graph, x, ids, w, y in graphs:
            x.mul_(1.25)
            ids.add_(1).remainder_(16)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, mxfp4_moe(x, w, ids, gu, dn))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = mxfp4_moe(graphs[1][1], graphs[1][3], graphs[1][2], gu, dn)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, graphs[1][4])


@pytest.mark.gpu
@pytest.mark.parametrize("t", [3, 100])
def test_fused_moe_takes_mxfp4_stacks(t):
    from litevllm_amd import AWQExperts, fused_moe, moe_route, mxfp4_moe
    gu, dn, _, _ = _experts(90, 8, 96, 128)
    x = _made(91, t, 128).bfloat16().cuda()
    logits = _made(92, t, 8).bfloat16().cuda()
    w, ids = moe_route(logits, 2, True, flow="logits")
    assert torch.equal(fused_moe(x, gu, dn, logits, 2), mxfp4_moe(x, w, ids, gu, dn, activation="silu"))
    with pytest.raises(TypeError):
        fused_moe(x, gu, dn.qweight, logits, 2)
    with pytest.raises(TypeError):
        fused_moe(x, gu, AWQExperts(dn.qweight, dn.scales), logits, 2)


# ------------------------------------------------------------------ together
@pytest.mark.gpu
@pytest.mark.parametrize("t", [2, 130])
def test_a_layer_of_router_balance_experts_and_projection(t):
    """Route, watch the balance, run the experts, project: each step on the output of the one before."""
    from litevllm_amd import MXFP4Weight, moe_balance_loss, moe_route, mxfp4_moe
    h, e, k, i = 192, 12, 3, 64
    x = _made(100, t, h).half().cuda() * 4
    logits = (x.float() @ _made(101, h, e).cuda() * 0.05).requires_grad_(True)
    w, ids = moe_route(logits.detach(), k, True)
    loss, counts = moe_balance_loss(logits, ids)
    loss.backward()
    gu, dn, w1, w2 = _experts(102, e, i, h)
    y = mxfp4_moe(x, w, ids, gu, dn)
    dense = _made(104, 80, h, scale=0.05).cuda()
    proj = MXFP4Weight.from_dense(dense)
    z = proj.matmul(y)
    assert torch.equal(counts.cpu().long(), torch.bincount(ids.flatten().cpu(), minlength=e))
    p = torch.softmax(logits.detach().double(), 1)
    f = counts.double() / (t * k)
    assert abs(float(loss.detach()) - float(e * (f * p.mean(0)).sum())) < 1e-5
    grad = e / t * p * (f - (p * f).sum(1, keepdim=True))
    assert float((logits.grad.double() - grad).abs().max()) <= 1e-5 * float(grad.abs().max())
    _close(y, *R.moe(x, w.cpu(), ids.cpu(), w1, w2, "silu"), torch.float16)
    _close(z, *R.gemm(R.rounded(y), R.rounded(dense)), torch.float16)


def test_gemm_entry_refuses_columns_that_a_block_cannot_number():
    """A block's columns, also those behind the last, are numbered in 32 bits: up to 2^31 - 256."""
    lib, p = L.load(), _fake()

    def call(n, m):
        return lib.awq_w4a16_mxfp4_gemm(p, 64, None, p, p, None, p, n, m, n, 64, L.DTYPE_BF16, L.DTYPE_NONE, None, 0, None)
    for m in (20, 300):
        assert call((1 << 31) - 256, m) == L.ERR_WORKSPACE  # what it has to say next
    for n in ((1 << 31) - 255, (1 << 31) - 8, (1 << 31) - 1, 1 << 31):
        for m in (1, 20, 300):
            assert call(n, m) == L.ERR_UNSUPPORTED


# ------------------------------------------------------------------ the framework's linear method
def _layer(**tensors):
    from litevllm_amd.awq import AWQConfig
    layer = torch.nn.Module()
    cfg = AWQConfig.from_config({"config_groups": {"group_0": {"weights": {"num_bits": 4, "group_size": 32}}}})
    cfg.init_layer(layer)
    cfg.load_weights(layer, tensors.items())
    return cfg, layer


def test_the_linear_method_calls_the_product(monkeypatch):
    """Without a GPU, the product replaced: what ``AWQConfig.apply`` hands it, for a weight that the layer holds and for
    one that it builds of the layer's tensors."""
    from litevllm_amd import MXFP4Weight, mxfp4
    calls = []

    def gemm(a, qweight, scales, a_scales=None, bias=None, **kw):
        calls.append((a, qweight, scales, bias, kw))
        return a.new_zeros(a.shape[0], qweight.shape[0])
    monkeypatch.setattr(mxfp4, "mxfp4_gemm", gemm)
    c, s = R.quantize(_made(110, 48, 64))
    x, bias = torch.zeros(2, 3, 64, dtype=torch.bfloat16), torch.ones(48)
    cfg, layer = _layer(qweight=c, scales=s, bias=bias)
    held = torch.nn.Module()
    held._quant_weight, held.bias = MXFP4Weight(c, s, prefix="p"), None
    for on, b in ((layer, layer.bias), (held, None)):
        for kw in ({}, {"config": {"kernel_policy": {}}}, {"inf_config": object()}):
            assert cfg.apply(on, x, **kw).shape == (2, 3, 48)
            a, qweight, scales, got, rest = calls.pop()
            assert a.shape == (6, 64) and torch.equal(qweight, c) and torch.equal(scales, s) and got is b and not rest
    assert isinstance(layer._quant_weight, MXFP4Weight)
    # like the other weights a module, whose tensors move and are saved with the layer's
    assert set(held.state_dict()) == {"_quant_weight.qweight", "_quant_weight.scales"}
    assert not any(p.requires_grad for p in held.parameters())


def test_the_loader_knows_the_format():
    from litevllm_amd import MXFP4Weight, loader
    c, s = R.quantize(_made(111, 48, 128))
    w = loader.make_awq_weight(loader.awq_components({"m.weight_packed": c, "m.weight_scale": s}, "m"), prefix="m")
    assert type(w) is MXFP4Weight and w.prefix == "m" and torch.equal(w.qweight, c) and torch.equal(w.scales, s)
    with pytest.raises(ValueError):
        loader.make_awq_weight({"qweight": c, "scales": s[:, :2]})
    with pytest.raises(ValueError):  # the format has no zero points
        loader.make_awq_weight({"qweight": c, "scales": s, "qzeros": torch.zeros(48, 4, dtype=torch.uint8)})


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40])
def test_the_linear_method_on_mxfp4_tensors(m):
    from litevllm_amd import loader, mxfp4_gemm
    from litevllm_amd.awq import AWQConfig
    c, s = R.quantize(_made(112, 80, 128))
    b = _made(113, 80)
    x = _made(114, m, 1, 128, dtype=torch.bfloat16).cuda()
    want = mxfp4_gemm(x.view(m, 128), c.cuda(), s.cuda(), bias=b.cuda()).view(m, 1, 80)
    cfg, layer = _layer(weight_packed_qweight=c, scales=s, bias=b)
    assert torch.equal(cfg.apply(layer.cuda(), x, inf_config=None), want)
    held = torch.nn.Module()
    held._quant_weight, held.bias = loader.make_awq_weight({"qweight": c, "scales": s}), b.cuda()
    assert torch.equal(AWQConfig().apply(held.cuda(), x), want)


# ------------------------------------------------------------------ derivatives
def _without_launches(monkeypatch):
    """The operators on CPU tensors, nothing launched."""
    from litevllm_amd import moe_balance, mxfp4
    monkeypatch.setattr(mxfp4, "_call", lambda *a: None)
    monkeypatch.setattr(moe_balance, "_call", lambda *a: None)
    monkeypatch.setattr(mxfp4.ops, "_require_device", lambda *t: torch.device("cpu"))


def _leaves():
    return (torch.randn(3, 64, dtype=torch.bfloat16, requires_grad=True), torch.randn(48, requires_grad=True),
            torch.rand(3, 2, requires_grad=True))


def _calls(x, bias, weights):
    """Name -> a call with a floating result, and the leaves that it depends on."""
    from litevllm_amd import MXFP4Experts, MXFP4Weight, mxfp4_gemm, mxfp4_moe
    dev = x.device
    c, s = (t.to(dev) for t in R.quantize(_made(120, 48, 64)))
    gu, dn = (MXFP4Experts(*(t.to(dev) for t in R.quantize(_made(121, 4, *shape)))) for shape in ((64, 64), (64, 32)))
    ids = torch.zeros(3, 2, dtype=torch.int32, device=dev)
    return {"gemm": (lambda: mxfp4_gemm(x, c, s), [x]), "bias": (lambda: mxfp4_gemm(x.detach(), c, s, bias=bias), [bias]),
            "weight": (lambda: MXFP4Weight(c, s).matmul(x, bias), [x, bias]),
            "moe": (lambda: mxfp4_moe(x, weights, ids, gu, dn), [x, weights]),
            "routing": (lambda: mxfp4_moe(x.detach(), weights, ids, gu, dn), [weights])}


@pytest.mark.parametrize("name", ["gemm", "bias", "weight", "moe", "routing"])
def test_a_derivative_is_refused_and_not_dropped(name, monkeypatch):
    _without_launches(monkeypatch)
    x, bias, weights = _leaves()
    call, leaves = _calls(x, bias, weights)[name]
    y = call()
    assert y.requires_grad and y.dtype == torch.bfloat16
    with pytest.raises(RuntimeError, match="not differentiable"):
        y.float().sum().backward()
    for leaf in leaves:  # also where the leaf has another way into the result
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(call().float().sum() + (2 * leaf.float()).sum(), leaf)
    with torch.no_grad():
        assert not call().requires_grad
    for leaf in (x, bias, weights):
        leaf.requires_grad_(False)
    assert not call().requires_grad


def test_where_a_result_cannot_carry_the_refusal_the_call_is_refused(monkeypatch):
    import torch.autograd.forward_ad as fwd

    from litevllm_amd import MXFP4Experts, MXFP4Weight, moe_balance_loss, mxfp4_gemm, mxfp4_moe, mxfp4_quantize
    _without_launches(monkeypatch)
    x, bias, weights = _leaves()
    with pytest.raises(RuntimeError, match="not differentiable"):
        mxfp4_quantize(x)
    with torch.no_grad():
        mxfp4_quantize(x)
    assert not MXFP4Weight.from_dense(x).scales.requires_grad  # a weight's conversion takes its values
    c, s = R.quantize(_made(120, 48, 64))
    gu, dn = (MXFP4Experts(*R.quantize(_made(121, 4, *shape))) for shape in ((64, 64), (64, 32)))
    ids = torch.zeros(3, 2, dtype=torch.int32)
    for call in (lambda out: mxfp4_gemm(x, c, s, out=out[:, :48]), lambda out: mxfp4_moe(x, weights, ids, gu, dn, out=out)):
        out = torch.zeros(3, 64, dtype=torch.bfloat16)
        with pytest.raises(RuntimeError, match="out="):
            call(out)
        with torch.no_grad():
            call(out)
    x, bias, weights = (t.detach() for t in (x, bias, weights))
    logits = torch.randn(3, 4)
    with fwd.dual_level():
        dx, db, dw, dl = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, bias, weights, logits))
        for call in (lambda: mxfp4_quantize(dx), lambda: mxfp4_gemm(dx, c, s), lambda: mxfp4_gemm(x, c, s, bias=db),
                     lambda: mxfp4_moe(dx, weights, ids, gu, dn), lambda: mxfp4_moe(x, dw, ids, gu, dn), lambda: moe_balance_loss(dl, ids)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        mxfp4_gemm(x, c, s, bias=bias)
        moe_balance_loss(logits, ids)


def test_a_second_derivative_of_the_balance_loss_is_refused_and_not_dropped(monkeypatch):
    from litevllm_amd import moe_balance_loss
    _without_launches(monkeypatch)
    z, up = torch.randn(3, 4, requires_grad=True), torch.tensor(2.0, requires_grad=True)
    loss, _ = moe_balance_loss(z, torch.zeros(3, 2, dtype=torch.int32))
    g, = torch.autograd.grad(loss, z, up, create_graph=True)
    for leaf in (z, up):  # also where the leaf has another way into the result
        with pytest.raises(RuntimeError, match="twice"):
            torch.autograd.grad(g.sum() + (2 * leaf).sum(), leaf, retain_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


@pytest.mark.gpu
def test_results_that_refuse_a_derivative_are_the_same():
    x, bias, weights = (t.detach().cuda().requires_grad_(True) for t in _leaves())
    for call, _ in _calls(x, bias, weights).values():
        y = call()
        with torch.no_grad():
            assert torch.equal(y, call())
        assert y.requires_grad
        with pytest.raises(RuntimeError, match="not differentiable"):
            y.float().sum().backward()


def test_workspace_queries_answer_nothing_for_what_the_calls_refuse():
    lib = L.load()
    big = (1 << 31, 1 << 40, 1 << 62, (1 << 63) - 1)
    for t in ((1 << 30) + 1, *big):
        assert lib.awq_w4a16_moe_balance_workspace_bytes(t, 8) == 0
    assert lib.awq_w4a16_moe_balance_workspace_bytes(1 << 30, 8) > 0 < lib.awq_w4a16_moe_balance_workspace_bytes(0, 8)
    assert lib.awq_w4a16_moe_balance_workspace_bytes(4, 1025) == 0
    for n in big:
        assert lib.awq_w4a16_mxfp4_gemm_workspace_bytes(n, 64, 64) == 0 == lib.awq_w4a16_mxfp4_gemm_workspace_bytes(64, 64, n)
        assert lib.awq_w4a16_mxfp4_gemm_workspace_bytes(64, n, 64) == 0
        assert lib.awq_w4a16_mxfp4_moe_workspace_bytes(n, 64, 64, 8, 1) == 0 == lib.awq_w4a16_mxfp4_moe_workspace_bytes(2, n, 64, 8, 1)
        assert lib.awq_w4a16_mxfp4_moe_workspace_bytes(2, 64, n, 8, 1) == 0
    assert lib.awq_w4a16_mxfp4_moe_workspace_bytes(1 << 20, 64, 64, 8, 1 << 12) == 0 == lib.awq_w4a16_mxfp4_moe_workspace_bytes(2, 64, 64, 1025, 1)
    # 2^31 - 1 rows, and their codes and scales
    assert lib.awq_w4a16_mxfp4_gemm_workspace_bytes((1 << 31) - 1, 64, 1 << 24) >= ((1 << 31) - 1) * ((1 << 23) + (1 << 19))


# ------------------------------------------------------------------ scales far apart inside one sum
@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 70, 416), (9, 300, 1280), (48, 70, 2080), (260, 130, 4128), (700, 4100, 1056), (2100, 2100, 288)])
def test_gemm_blocks_of_one_sum_far_apart(m, n, k):
    """Blocks of both operands 2^-25 to 2^25: terms up to 2^100 apart meet in a sum."""
    from litevllm_amd import mxfp4_gemm
    g = torch.Generator().manual_seed(m)
    a, w = (torch.randint(0, 256, (r, k // 2), generator=g).to(torch.uint8).cuda() for r in (m, n))
    sa, sw = (torch.randint(102, 153, (r, k // 32), generator=g).to(torch.uint8).cuda() for r in (m, n))
    y = mxfp4_gemm(a, w, sw, a_scales=sa, out_dtype=torch.bfloat16)
    _close(y, *R.gemm(R.values(a, sa), R.values(w, sw)), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 70, 416), (9, 300, 1280), (48, 70, 2080), (260, 130, 4128), (700, 4100, 1056), (2100, 2100, 288)])
def test_gemm_smallest_and_largest_scales(m, n, k):
    """Scale bytes 0 and 254 in both operands: the other one of a block is near 254 and 0, so the products are near 1."""
    from litevllm_amd import mxfp4_gemm
    g = torch.Generator().manual_seed(m + 1)
    a, w = (torch.randint(0, 256, (r, k // 2), generator=g).to(torch.uint8).cuda() for r in (m, n))
    ends = torch.randint(0, 2, (k // 32,), generator=g) * 254
    ends[:2] = torch.tensor([0, 254])
    near = torch.randint(0, 4, (n, k // 32), generator=g)
    sa = ends.expand(m, -1).to(torch.uint8).cuda()
    sw = torch.where(ends == 0, 254 - near, near).to(torch.uint8).cuda()
    y = mxfp4_gemm(a, w, sw, a_scales=sa, out_dtype=torch.bfloat16)
    ref = R.gemm(R.values(a, sa), R.values(w, sw))
    _close(y, *ref, torch.bfloat16)
    if n == m:  # the operands' places changed
        z = mxfp4_gemm(w, a, sa, a_scales=sw, out_dtype=torch.bfloat16)
        _close(z, ref[0].t(), ref[1].t(), torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k,h,i", [(2, 9, 3, 160, 64), (9, 2, 2, 416, 96), (40, 16, 4, 256, 64), (500, 5, 4, 288, 96)])
def test_moe_blocks_of_one_sum_far_apart(t, e, k, h, i):
    """The gate and up stack's blocks 2^-20 to 2^20 times their size, the tokens' the other way round, block by block but for 2^3:
    the sums stay in the range that the activation is tested in."""
    from litevllm_amd import MXFP4Experts, mxfp4_moe
    g = torch.Generator().manual_seed(t)
    c1, s1, _ = _weight(t, e, 2 * i, h)
    c2, s2, _ = _weight(t + 1, e, h, i)
    by = torch.randint(-20, 21, (h // 32,), generator=g)
    s1 = (s1.int() + by.cuda() + torch.randint(-1, 2, s1.shape, generator=g).cuda()).to(torch.uint8)
    x = (_made(t, t, h) * torch.pow(2.0, -by.float()).repeat_interleave(32)).bfloat16().cuda()
    ids, weights = torch.randint(0, e, (t, k), generator=g), torch.rand(t, k, generator=g)
    y = mxfp4_moe(x, weights.cuda(), ids.cuda(), MXFP4Experts(c1, s1), MXFP4Experts(c2, s2))
    # on the CPU: the GPU's powers of two are not exact at all of these exponents, and a tie is then none
    whole = torch.arange(-127, 128, dtype=torch.float64)
    assert torch.pow(2.0, whole).tolist() == [2.0 ** n for n in range(-127, 128)]
    _close(y.cpu(), *R.moe(x.cpu(), weights, ids, R.values(c1.cpu(), s1.cpu()), R.values(c2.cpu(), s2.cpu()), "silu"), torch.bfloat16)


@pytest.mark.parametrize("name", ["gemm", "moe"])
def test_a_result_that_refuses_a_derivative_can_be_written_to(name, monkeypatch):
    _without_launches(monkeypatch)
    call, (leaf, *_) = _calls(*_leaves())[name]
    y = call()
    assert not y._is_view()
    y.zero_().add_(1.0)
    y[0] = 3.0
    assert y.detach().sum() == 2 * y.shape[1] + 3 * y.shape[1]
    z = call()
    z.add_(1.0)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(z.float().sum() + leaf.float().sum(), leaf)
