"""8-bit block matrices, their product and fp8_linear against plain implementations in 64 bits.

Tolerances: quantised values and scales are exact.  A product's terms are exact in fp32; the sum over k takes k / 32
accumulator steps of 32 terms, each step's rounding (or truncation) at most 2^-23 of the magnitudes added so far and
the 32 terms inside a step at most 2^-23 each of the largest: (k / 32 + 32) * 2^-23 of the sum of magnitudes in all,
then half an ulp of the result's type (2^-8 of the value in bf16, 2^-11 in fp16).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def plain_quantize(x, br, bc):
    """(values, exponents of each block) of x in 64 bits by the definition, on the CPU."""
    x = x.detach().double().cpu()
    rows, cols = x.shape
    values, exps = torch.empty_like(x), torch.empty(-(-rows // br), -(-cols // bc), dtype=torch.int32)
    for i in range(exps.shape[0]):
        for j in range(exps.shape[1]):
            t = x[i * br:(i + 1) * br, j * bc:(j + 1) * bc]
            finite = t[torch.isfinite(t)].abs()
            top = finite.max().item() if finite.numel() else 0.0
            e = 0
            if top > 0:
                e = max(-126, math.frexp(top / 448)[1] - (math.frexp(top / 448)[0] == 0.5))
            v = t / 2.0 ** e
            step = 2.0 ** (torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
            v = torch.round(v / step) * step * 2.0 ** e
            values[i * br:(i + 1) * br, j * bc:(j + 1) * bc] = torch.where(torch.isfinite(t), v, math.nan)
            exps[i, j] = e
    return values, exps


def make(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * std
    return (x * torch.exp2(torch.randint(-6, 7, shape[-1:], generator=g).float())).to(dtype)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=1e30), torch.nan_to_num(b, nan=1e30))


SHAPES = [(1, 1), (1, 2048), (3, 100), (130, 257), (200, 1001), (128, 128), (129, 640), (300, 1100)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantize_is_exact(cuda_device, shape, dtype):
    from pack3d_b200 import quantize, quantize_weight
    from pack3d_b200.fp8 import _quantize
    x = make(shape, dtype, 3)
    x[0, 0] = 0
    xd = x.to(cuda_device)
    rows, cols = shape
    v, e = plain_quantize(x, 1, 128)
    q = quantize(xd)
    assert q.shape == shape and torch.equal(q.exponents().cpu(), e) and same(q.dequantize(torch.float64).cpu(), v)
    v2, e2 = plain_quantize(x, 128, 128)
    w = quantize_weight(xd)
    assert torch.equal(w.exponents().cpu(), e2.repeat_interleave(128, 0)[:rows])
    assert same(w.dequantize(torch.float64).cpu(), v2)
    vt, et = plain_quantize(x.t(), 1, 128)
    sums = torch.empty(cols, device=cuda_device)
    a, at = _quantize(xd, transposed=True, sums=sums)
    assert same(a.dequantize(torch.float64).cpu(), v) and torch.equal(at.exponents().cpu(), et)
    assert same(at.dequantize(torch.float64).cpu(), vt)
    # fp32 sums of `rows` terms
    limit = x.double().abs().sum(0) * rows * 2.0 ** -24
    assert ((sums.cpu().double() - x.double().sum(0)).abs() <= limit).all()
    _, wt = _quantize(xd, square=True, rows=False, transposed=True)
    assert same(wt.dequantize(torch.float64).cpu(), v2.t())


def test_quantize_special_blocks(cuda_device):
    """Zeros, NaN and infinities, the edges of a power of two, subnormal and huge blocks."""
    from pack3d_b200 import quantize
    x = torch.ones(12, 256)
    x[0] = 0
    x[1, 5], x[1, 200] = math.nan, math.inf
    x[2, :128] = math.inf
    x[3, 0] = 448.0
    x[4, 0] = 448.0 * (1 + 2.0 ** -23)
    x[5] = 2.0 ** -149
    x[6, 0] = 3.4e38
    x[7] = -3.4e38
    x[8, 0] = 449.0
    x[9] = 2.0 ** -126 * 448
    x[10] = 2.0 ** -126 * 224
    x[11, 1] = -1e-30
    q = quantize(x.to(cuda_device))
    v, e = plain_quantize(x, 1, 128)
    assert torch.equal(q.exponents().cpu(), e)
    assert same(q.dequantize(torch.float64).cpu(), v)
    assert e[0].tolist() == [0, 0] and e[3, 0] == 0 and e[4, 0] == 1 and e[5, 0] == -126


def test_quantize_views(cuda_device):
    from pack3d_b200 import quantize
    base = make((40, 300), torch.bfloat16, 5).to(cuda_device)
    for view in (base[:, 1:257], base.t(), base[::2], base[3:, 8:]):
        assert same(quantize(view).dequantize(), quantize(view.contiguous().clone()).dequantize())
    odd = torch.empty(40 * 256 + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(40, 256)
    odd.copy_(base[:, :256])
    assert same(quantize(odd).dequantize(), quantize(base[:, :256].contiguous()).dequantize())


def check_product(got, a, b, bias=None):
    """got against a b^T (+ bias) of 64-bit matrices."""
    a, b = a.double(), b.double()
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    k = a.shape[1]
    limit = size * (k / 32 + 32) * 2.0 ** -23 + want.abs() * ULP[got.dtype] * 1.01
    if got.dtype == torch.float16:
        limit = limit + 2.0 ** -25
    bad = (got.double() - want).abs() - limit
    assert bad.max().item() <= 0, (bad.max().item(), want.abs().max().item())


PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 1000, 2048), (2, 257, 640), (16, 300, 129), (17, 128, 4096), (33, 513, 1100),
            (64, 200, 300), (65, 128, 128), (128, 128, 128), (130, 250, 260), (256, 512, 1024), (1000, 392, 520),
            (4097, 1096, 192), (129, 8, 8200), (700, 5000, 64)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_matmul(cuda_device, m, n, k, dtype):
    from pack3d_b200 import _native, fp8_matmul, quantize, quantize_weight
    a = quantize(make((m, k), torch.float32, m + k, 0.05).to(cuda_device))
    b = quantize(make((n, k), torch.float32, n + k, 0.05).to(cuda_device))   # another scale for every row
    bias = make((n,), dtype, 7).to(cuda_device)
    got = fp8_matmul(a, b, bias=bias, dtype=dtype)
    assert got.shape == (m, n) and got.dtype == dtype
    check_product(got, a.dequantize(torch.float64), b.dequantize(torch.float64), bias)
    assert torch.equal(fp8_matmul(a, b, bias=bias, dtype=dtype), got)
    w = quantize_weight(make((n, k), torch.bfloat16, n, 0.05).to(cuda_device))
    check_product(fp8_matmul(a, w, dtype=dtype), a.dequantize(torch.float64), w.dequantize(torch.float64))
    assert _native.device_errors() == 0


def test_matmul_large_k_and_extreme_scales(cuda_device):
    """A long sum in slices, and scales at both ends of their range."""
    from pack3d_b200 import fp8_matmul, quantize
    a = quantize(make((24, 40000), torch.float32, 1).to(cuda_device))
    b = quantize(make((136, 40000), torch.float32, 2).to(cuda_device))
    check_product(fp8_matmul(a, b, dtype=torch.float32), a.dequantize(torch.float64), b.dequantize(torch.float64))
    a = quantize((make((70, 512), torch.float32, 3) * 2.0 ** -90).to(cuda_device))
    b = quantize((make((70, 512), torch.float32, 4) * 2.0 ** 100).to(cuda_device))
    check_product(fp8_matmul(a, b, dtype=torch.float32), a.dequantize(torch.float64), b.dequantize(torch.float64))


def test_matmul_nan_stays_in_its_row(cuda_device):
    from pack3d_b200 import fp8_matmul, quantize
    x = make((100, 256), torch.float32, 6)
    w = make((90, 256), torch.float32, 8)
    clean = fp8_matmul(quantize(x.to(cuda_device)), quantize(w.to(cuda_device)), dtype=torch.float32)
    x[7, 3], w[11, 200] = math.nan, math.inf
    got = fp8_matmul(quantize(x.to(cuda_device)), quantize(w.to(cuda_device)), dtype=torch.float32)
    assert got[7].isnan().all() and got[:, 11].isnan().all()
    # inf raised no scale: the row's other blocks and every other row keep their bits
    keep_r, keep_c = [i for i in range(100) if i != 7], [i for i in range(90) if i != 11]
    assert torch.equal(got[keep_r][:, keep_c], clean[keep_r][:, keep_c])


LINEARS = [(1, 64, 96), (5, 100, 257), (64, 128, 128), (70, 520, 392), (300, 257, 1001), (1025, 192, 768)]


@pytest.mark.parametrize("m,k,n", LINEARS)
@pytest.mark.parametrize("dtype,wtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                         (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("bias", [True, False])
def test_linear_and_gradients(cuda_device, m, k, n, dtype, wtype, bias):
    from pack3d_b200 import fp8_linear, quantize_weight
    x, w = make((m, k), dtype, m), make((n, k), wtype, n, 0.05)
    b = make((n,), wtype, 5) if bias else None
    dy = make((m, n), dtype, 9, 0.01)
    xd, wd = x.to(cuda_device).requires_grad_(), w.to(cuda_device).requires_grad_()
    bd = b.to(cuda_device).requires_grad_() if bias else None
    y = fp8_linear(xd, wd, bd)
    leaves = [xd, wd] + ([bd] if bias else [])
    grads = torch.autograd.grad(y, leaves, dy.to(cuda_device))
    xq, wq, dq = plain_quantize(x, 1, 128)[0], plain_quantize(w, 128, 128)[0], plain_quantize(dy, 1, 128)[0]
    xt, dt = plain_quantize(x.t(), 1, 128)[0], plain_quantize(dy.t(), 1, 128)[0]
    check_product(y.detach().cpu(), xq, wq, b)
    assert [g.dtype for g in grads] == [t.dtype for t in leaves]
    check_product(grads[0].cpu(), dq, wq.t())
    check_product(grads[1].cpu(), dt, xt)
    if bias:
        want = dy.double().sum(0)
        limit = dy.double().abs().sum(0) * m * 2.0 ** -24 + want.abs() * ULP[wtype] * 1.01 + 2.0 ** -25
        assert ((grads[2].cpu().double() - want).abs() <= limit).all()
    with torch.no_grad():
        assert torch.equal(fp8_linear(xd, wd, bd), y)
        assert torch.equal(fp8_linear(xd, quantize_weight(wd), bd), y)      # the kept weight gives the same bits
    again = torch.autograd.grad(fp8_linear(xd, wd, bd), leaves, dy.to(cuda_device))
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    only_w, = torch.autograd.grad(fp8_linear(xd.detach(), wd, None), [wd], dy.to(cuda_device))
    assert torch.equal(only_w, grads[1])
    only_x, = torch.autograd.grad(fp8_linear(xd, wd.detach(), None), [xd], dy.to(cuda_device))
    assert torch.equal(only_x, grads[0])


def test_linear_gradients_against_differences(cuda_device):
    """Small whole numbers are exact in e4m3 whatever the blocks' scales, so the layer is exactly linear on them and
    differences of its outputs are its gradients."""
    from pack3d_b200 import fp8_linear
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-4, 5, (37, 150), generator=g).float().to(cuda_device).requires_grad_()
    w = torch.randint(-4, 5, (70, 150), generator=g).float().to(cuda_device).requires_grad_()
    dy = torch.randint(-4, 5, (37, 70), generator=g).float().to(cuda_device)
    dx, dw = torch.autograd.grad(fp8_linear(x, w), [x, w], dy)
    px = torch.randint(-3, 4, x.shape, generator=g).float().to(cuda_device)
    pw = torch.randint(-3, 4, w.shape, generator=g).float().to(cuda_device)
    with torch.no_grad():
        along_x = ((fp8_linear(x + px, w) - fp8_linear(x - px, w)) * dy).double().sum() / 2
        along_w = ((fp8_linear(x, w + pw) - fp8_linear(x, w - pw)) * dy).double().sum() / 2
    assert along_x == (dx * px).double().sum() and along_w == (dw * pw).double().sum()


def test_linear_shapes_streams_and_empty(cuda_device):
    from pack3d_b200 import fp8_linear, quantize_weight
    x = make((2, 3, 5, 64), torch.bfloat16, 1).to(cuda_device)
    w = make((40, 64), torch.bfloat16, 2).to(cuda_device)
    y = fp8_linear(x, w)
    assert y.shape == (2, 3, 5, 40) and torch.equal(y.view(-1, 40), fp8_linear(x.view(-1, 64), w))
    assert torch.equal(fp8_linear(x.transpose(0, 1), w), y.transpose(0, 1))
    assert torch.equal(fp8_linear(x[0, 0, 0], w), y[0, 0, 0])
    kept = quantize_weight(w)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = fp8_linear(x, kept)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, y)
    assert fp8_linear(x[:0], kept).shape == (0, 3, 5, 40)
    wg, xg = w.clone().requires_grad_(), x[:0].clone().requires_grad_()
    dx, dw = torch.autograd.grad(fp8_linear(xg, wg).sum(), [xg, wg])
    assert dx.shape == xg.shape and (dw == 0).all()
    assert fp8_linear(torch.randn(5, 64, device=cuda_device), w[:1].float()).shape == (5, 1)


def test_linear_in_a_captured_graph(cuda_device):
    from pack3d_b200 import fp8_linear, quantize_weight
    x = make((9, 640), torch.bfloat16, 1).to(cuda_device)
    kept = quantize_weight(make((384, 640), torch.bfloat16, 2).to(cuda_device))
    want = fp8_linear(x, kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp8_linear(x, kept)
    y.zero_()
    graph.replay()
    assert torch.equal(y, want)


def test_refusals(cuda_device):
    from pack3d_b200 import fp8_linear, fp8_matmul, quantize, quantize_weight
    x, w = torch.randn(4, 64, device=cuda_device), torch.randn(32, 64, device=cuda_device)
    kept = quantize_weight(w)
    with pytest.raises(ValueError, match="weight must be"):
        fp8_linear(x, w[:, :32])
    with pytest.raises(ValueError, match="weight must be"):
        fp8_linear(x, w.double())
    with pytest.raises(ValueError, match="CUDA"):
        fp8_linear(x.double(), w)
    with pytest.raises(ValueError, match="same device"):
        fp8_linear(x, w.cpu())
    with pytest.raises(ValueError, match="bias"):
        fp8_linear(x, w, torch.zeros(31, device=cuda_device))
    with pytest.raises(ValueError, match="no gradients"):
        fp8_linear(x.clone().requires_grad_(), kept)
    with pytest.raises(ValueError, match="matrix"):
        quantize(x[0])
    with pytest.raises(ValueError, match="matrix"):
        quantize_weight(w[:0])
    with pytest.raises(ValueError, match="CUDA"):
        quantize(x.cpu())
    with pytest.raises(ValueError, match="same columns"):
        fp8_matmul(quantize(x), quantize_weight(w[:, :32]))
    with pytest.raises(ValueError, match="two Fp8Matrix"):
        fp8_matmul(x, kept)
    with pytest.raises(ValueError, match="dtype"):
        fp8_matmul(quantize(x), kept, dtype=torch.float64)


def test_linear_offsets_past_32_bits(cuda_device):
    """More than 2^31 outputs: the last rows are those of a call with these rows alone, in both directions."""
    from pack3d_b200 import fp8_linear
    m, k, n, tail = 2 ** 20 + 1000, 136, 2048, 1000
    g = torch.Generator(device=cuda_device).manual_seed(4)
    x = torch.empty(m, k, dtype=torch.bfloat16, device=cuda_device).normal_(generator=g).requires_grad_()
    w = torch.randn(n, k, dtype=torch.bfloat16, device=cuda_device, generator=g)
    y = fp8_linear(x, w)
    dy = torch.empty_like(y).normal_(generator=g)
    y.backward(dy)
    last = x.detach()[-tail:].clone().requires_grad_()
    want = fp8_linear(last, w)
    want.backward(dy[-tail:].clone())
    assert torch.equal(y[-tail:], want) and torch.equal(x.grad[-tail:], last.grad)


def test_changed_parts_of_a_matrix_are_refused(cuda_device):
    """An Fp8Matrix whose attributes no longer fit together, and tensors off a 16-byte boundary, reach no kernel."""
    from pack3d_b200 import Fp8Matrix, fp8_linear, fp8_matmul, quantize, quantize_weight
    x = torch.randn(4, 64, device=cuda_device)
    qx, w = quantize(x), quantize_weight(torch.randn(130, 64, device=cuda_device))
    changes = {"values": [w.values.cpu(), w.values[:129], w.values.view(torch.uint8), w.values.t(), w.values[:, :32]],
               "scales": [w.scales.cpu(), w.scales[:512], w.scales.view(torch.int8), w.scales.repeat(2)[::2]],
               "rows": [129, 131, 258], "cols": [80]}
    for name, bads in changes.items():
        for bad in bads:
            other = Fp8Matrix(w.values, w.scales, w.rows, w.cols)
            setattr(other, name, bad)
            for call in (lambda: fp8_linear(x, other), lambda: fp8_matmul(qx, other), lambda: fp8_matmul(other, qx)):  # noqa: B023
                with pytest.raises(ValueError):
                    call()
    odd = torch.empty(130 * 64 + 1, dtype=torch.uint8, device=cuda_device)[1:].view(torch.float8_e4m3fn).view(130, 64)
    for call in (lambda m: fp8_linear(x, m), lambda m: fp8_matmul(qx, m)):
        with pytest.raises(ValueError, match="16"):
            call(Fp8Matrix(odd, w.scales, 130, 64))


def test_matmul_has_no_gradients(cuda_device):
    from pack3d_b200 import fp8_matmul, quantize
    a = quantize(torch.randn(5, 64, device=cuda_device))
    bias = torch.randn(5, device=cuda_device, requires_grad=True)
    with pytest.raises(ValueError, match="no gradients"):
        fp8_matmul(a, a, bias=bias)
    with torch.no_grad():
        got = fp8_matmul(a, a, bias=bias)
    assert torch.equal(got, fp8_matmul(a, a, bias=bias.detach()))
