"""norm, residual_norm and dropout against plain implementations in 64 bits.

Tolerances: the kernels compute in fp32 and round each output once to its type, so an element may be off by half an
ulp of its type (2^-8 of the value in bf16, with its 8-bit significand, 2^-11 in fp16, 2^-24 in fp32) plus fp32's own
error, a few ulps of the terms that make it up: the terms here are of order one, up to eight, and 64 ulps of that
(2^-18 * 8) cover the ten or so operations and the row sums.  Sums over R rows of fp32 terms add independent
roundings: sqrt(R) * 2^-22 of the terms' norm, which is sqrt(R) times their size (four).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LOW = 0xFFFFFFFF


def philox_fields(block, rng):
    """The eight 16-bit fields of one block, in Python integers."""
    seed, offset = rng
    c = [block & LOW, block >> 32, offset & LOW, (offset >> 32) & LOW]
    k = [seed & LOW, (seed >> 32) & LOW]
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & LOW, (p0 >> 32) ^ c[3] ^ k[1], p0 & LOW]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return [f for w in c for f in (w & 0xFFFF, w >> 16)]


def keep_mask(rows, dim, p, rng):
    blocks = -(-dim // 8)
    t = round(65536 * p)
    m = torch.empty(rows, dim, dtype=torch.bool)
    for r in range(rows):
        fields = [f for b in range(blocks) for f in philox_fields(r * blocks + b, rng)]
        m[r] = torch.tensor(fields[:dim]) >= t
    return m


def test_philox_known_answers():
    """The published known-answer vectors of philox4x32-10 (counter and key all zeros, all ones)."""
    def words(fields):
        return [fields[2 * i] | fields[2 * i + 1] << 16 for i in range(4)]
    assert words(philox_fields(0, (0, 0))) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFFFFFFFFFF
    assert words(philox_fields(ones, (ones, ones))) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


@pytest.mark.parametrize("shape", [(1,), (7,), (3, 5), (2, 3, 8), (33, 64), (5, 195), (4, 1000), (1, 8192 + 3)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout_matches_its_definition(cuda_device, shape, dtype, p):
    from pack3d_b200 import dropout
    rng = (0x123456789ABCDEF, (1 << 40) + 5)
    x = torch.randn(shape, generator=torch.Generator().manual_seed(1)).to(dtype)
    keep = keep_mask(x.numel() // shape[-1], shape[-1], p, rng).view(shape)
    t = round(65536 * p)
    want = torch.where(keep, x.double() * (65536 / (65536 - t) if t < 65536 else 0.0), 0.0)
    xd = x.to(cuda_device).requires_grad_()
    y = dropout(xd, p, rng)
    assert y.dtype == dtype and y.shape == shape
    assert torch.equal(y.cpu() != 0, (want != 0))
    subnormal = 2.0 ** -25 if dtype == torch.float16 else 0.0      # half a step of fp16 below 2^-14
    assert ((y.cpu().double() - want).abs() <= want.abs() * (ULP[dtype] + 2.0 ** -23) + subnormal).all()
    dy = torch.randn(shape, generator=torch.Generator().manual_seed(2)).to(dtype)
    dx, = torch.autograd.grad(y, [xd], dy.to(cuda_device))
    back = torch.where(keep, dy.double() * (65536 / (65536 - t) if t < 65536 else 0.0), 0.0)
    assert ((dx.cpu().double() - back).abs() <= back.abs() * (ULP[dtype] + 2.0 ** -23) + subnormal).all()
    device_rng = torch.tensor(rng, dtype=torch.int64, device=cuda_device)
    assert torch.equal(dropout(xd, p, device_rng), y)


def test_dropout_drops_what_is_not_finite(cuda_device):
    from pack3d_b200 import dropout
    x = torch.full((64, 96), float("nan"), device=cuda_device)
    x[::2] = float("inf")
    rng = (3, 4)
    keep = keep_mask(64, 96, 0.5, rng).to(cuda_device)
    y = dropout(x, 0.5, rng)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()


def test_dropout_strides_alignment_and_streams(cuda_device):
    from pack3d_b200 import dropout
    rng = (9, 1)
    base = torch.randn(40, 65, device=cuda_device, dtype=torch.bfloat16)
    want = dropout(base[:, 1:].contiguous(), 0.3, rng)
    assert torch.equal(dropout(base[:, 1:], 0.3, rng), want)
    odd = torch.empty(40 * 64 + 1, device=cuda_device, dtype=torch.bfloat16)[1:].view(40, 64)
    odd.copy_(base[:, 1:])
    assert odd.data_ptr() % 16 and torch.equal(dropout(odd, 0.3, rng), want)
    t = torch.randn(64, 40, device=cuda_device, dtype=torch.bfloat16)
    assert torch.equal(dropout(t.t(), 0.3, rng), dropout(t.t().contiguous(), 0.3, rng))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = dropout(odd, 0.3, rng)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, want)
    assert dropout(base[:0], 0.3, rng).shape == (0, 65)


def test_dropout_rate(cuda_device):
    from pack3d_b200 import dropout
    n = 1 << 20
    y = dropout(torch.ones(n, device=cuda_device), 0.1, (11, 12))
    dropped = (y == 0).double().mean().item()
    assert abs(dropped - 0.1) < 6 * (0.1 * 0.9 / n) ** 0.5 + 2.0 ** -17
    again = dropout(torch.ones(n, device=cuda_device), 0.1, (11, 13))
    both = ((y == 0) & (again == 0)).double().mean().item()     # another offset: independent bits
    assert abs(both - 0.01) < 6 * (0.01 * 0.99 / n) ** 0.5 + 2.0 ** -17


# ------------------------------------------------------------------------------- norms
def plain_norm(z, spec):
    if spec is None:
        return z
    w, b, kind, eps = spec
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    z = z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)
    z = z if w is None else z * w
    return z if b is None else z + b


ACT = {"identity": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}


def plain_residual(x, h, post, gate, act, scale, nxt, keep, keep_scale):
    u = plain_norm(h, post)
    if gate is not None:
        u = u * ACT[act](gate)
    if keep is not None:
        u = torch.where(keep, u * keep_scale, torch.zeros_like(u))
    out = x + (u if scale is None else scale * u)
    return out, (None if nxt is None else plain_norm(out, nxt))


def close(got, want, dtype, summed=1):
    """Whether got is want rounded to dtype after fp32 arithmetic; `summed`: how many rows or columns were added up."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    slack = 2.0 ** -18 * 8 + (summed * 2.0 ** -22 * 4 if summed > 1 else 0) + (2.0 ** -25 if dtype == torch.float16 else 0)
    worst = ((got - want).abs() - want.abs() * (ULP[dtype] * 1.01 + 2.0 ** -20) - slack).max().item() if got.numel() else 0
    assert worst <= 0, worst


def make(shape, dtype, device, seed, mean=0.0, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype).to(device)


def check_residual(device, shape, dtype, kind="rms", gate=None, act="identity", p=0.0, post=True, nxt=True, scale=True,
                   bias=True, pdtype=None, seed=0, use_y=True, use_out=True):
    from pack3d_b200 import NormSpec, residual_norm
    pdtype = pdtype or dtype
    dim = shape[-1]
    x, h = make(shape, dtype, device, seed, 0.3, 1.5), make(shape, dtype, device, seed + 1, -0.2, 0.7)
    gate_shape = {None: None, "element": shape, "token": (*shape[:-1], 1), "sample": (shape[0], *(1,) * (len(shape) - 2), dim),
                  "all": (dim,)}[gate]
    leaves = {"x": x, "h": h}
    if gate_shape is not None:
        leaves["gate"] = make(gate_shape, dtype, device, seed + 2)
    if post:
        leaves["pw"] = make((dim,), pdtype, device, seed + 3, 1.0, 0.2)
        if bias:
            leaves["pb"] = make((dim,), pdtype, device, seed + 4, 0.0, 0.2)
    if scale is True:
        leaves["scale"] = make((dim,), pdtype, device, seed + 5, 0.5, 0.2)
    if nxt:
        leaves["nw"] = make((dim,), pdtype, device, seed + 6, 1.0, 0.2)
        if bias:
            leaves["nb"] = make((dim,), pdtype, device, seed + 7, 0.0, 0.2)
    for t in leaves.values():
        t.requires_grad_()
    exact = {k: t.detach().double().requires_grad_() for k, t in leaves.items()}
    rng = (seed + 77, seed + 5)
    t = round(65536 * p)
    rows = x.numel() // dim
    keep = keep_mask(rows, dim, p, rng).view(shape).to(device) if t else None
    eps = 1e-5

    def spec(w, b, of, cls):
        return cls((of.get(w), of.get(b), kind, eps)) if cls is tuple else cls(of.get(w), of.get(b), kind, eps)

    value = scale if not isinstance(scale, bool) else None
    out, y = residual_norm(x, h, post_norm=spec("pw", "pb", leaves, NormSpec) if post else None, gate=leaves.get("gate"),
                           gate_activation=act, scale=leaves.get("scale", value),
                           next_norm=spec("nw", "nb", leaves, NormSpec) if nxt else None, p=p, rng=rng)
    want_out, want_y = plain_residual(exact["x"], exact["h"], spec("pw", "pb", exact, tuple) if post else None,
                                      exact.get("gate"), act, exact.get("scale", value),
                                      spec("nw", "nb", exact, tuple) if nxt else None, keep,
                                      65536 / (65536 - t) if t < 65536 else 0.0)
    close(out, want_out, dtype)
    if nxt:
        close(y, want_y, dtype)
    else:
        assert y is None
    dout, dy = make(shape, dtype, device, seed + 8), make(shape, dtype, device, seed + 9)
    got_of, want_of, up = [], [], []
    if use_out:
        got_of, want_of, up = [out], [want_out], [dout]
    if nxt and use_y:
        got_of, want_of, up = got_of + [y], want_of + [want_y], up + [dy]
    names = [n for n in leaves if nxt and use_y or n not in ("nw", "nb")]
    got = torch.autograd.grad(got_of, [leaves[n] for n in names], up)
    want = torch.autograd.grad(want_of, [exact[n] for n in names], [u.double() for u in up])
    for name, a, b in zip(names, got, want):
        assert a.dtype == leaves[name].dtype and a.shape == leaves[name].shape, name
        summed = rows if name in ("pw", "pb", "scale", "nw", "nb") else dim if gate == "token" and name == "gate" else \
            rows // shape[0] if gate == "sample" and name == "gate" else rows if name == "gate" and gate == "all" else 1
        close(a, b, a.dtype, summed)
    again = torch.autograd.grad(
        [v for v, u in zip(residual_norm(x, h, post_norm=spec("pw", "pb", leaves, NormSpec) if post else None,
                                         gate=leaves.get("gate"), gate_activation=act, scale=leaves.get("scale", value),
                                         next_norm=spec("nw", "nb", leaves, NormSpec) if nxt else None, p=p, rng=rng),
                           (use_out, nxt and use_y)) if u], [leaves[n] for n in names], up)
    assert all(torch.equal(a, b) for a, b in zip(got, again))    # bitwise repeatable


SHAPES = [(1, 1), (1, 2048), (3, 7), (2, 5, 8), (2, 9, 192), (5, 33, 200), (37, 255), (3, 1001), (2, 3, 4096), (3, 4104),
          (2, 8193), (2, 16384), (2, 16383)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_shapes(cuda_device, shape, dtype, kind):
    check_residual(cuda_device, shape, dtype, kind, gate="element", act="sigmoid", p=0.25 if shape[-1] < 300 else 0.0)


@pytest.mark.parametrize("gate,act", [(None, "identity"), ("element", "tanh"), ("token", "sigmoid"), ("sample", "identity"),
                                      ("all", "tanh")])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("nxt", [True, False])
@pytest.mark.parametrize("scale", [True, False, 0.5])
@pytest.mark.parametrize("dim", [96, 101])
def test_residual_forms(cuda_device, gate, act, post, nxt, scale, dim):
    check_residual(cuda_device, (3, 50, dim), torch.bfloat16, "layer", gate, act, 0.1, post, nxt, scale, seed=dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bias", [True, False])
def test_residual_fp32_parameters(cuda_device, dtype, bias):
    check_residual(cuda_device, (4, 130, 320), dtype, "layer", "sample", "sigmoid", bias=bias, pdtype=torch.float32)
    check_residual(cuda_device, (4, 130, 321), dtype, "rms", "token", "tanh", bias=bias, pdtype=torch.float32)


@pytest.mark.parametrize("use_out,use_y", [(True, False), (False, True)])
def test_residual_one_output_used(cuda_device, use_out, use_y):
    check_residual(cuda_device, (7, 11, 136), torch.bfloat16, "layer", "element", "sigmoid", 0.2, use_out=use_out,
                   use_y=use_y)


@pytest.mark.parametrize("batch,tokens", [(1, 5000), (700, 3), (40, 130), (1300, 1)])
def test_residual_many_rows_and_samples(cuda_device, batch, tokens):
    check_residual(cuda_device, (batch, tokens, 40), torch.float32, "layer", "sample", "identity", seed=batch)


def test_residual_large_offset_mean(cuda_device):
    """A mean a thousand deviations away: squares about the mean, not a difference of squares."""
    from pack3d_b200 import NormSpec, norm
    z = 1000 + torch.randn(9, 512, generator=torch.Generator().manual_seed(3))
    y = norm(z.to(cuda_device), NormSpec(kind="layer", eps=0.0)).cpu().double()
    want = plain_norm(z.double(), (None, None, "layer", 0.0))
    assert (y - want).abs().max() < 1000 * 2.0 ** -23 * 8      # the mean's own rounding, over a deviation of one


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_of_zeros_infinity_and_nan(cuda_device, kind):
    """A row of zeros norms to its bias; a row with NaN or infinities touches no other row."""
    from pack3d_b200 import NormSpec, norm, residual_norm
    x = torch.randn(6, 72, device=cuda_device)
    x[1] = 0
    w, b = torch.rand(72, device=cuda_device), torch.rand(72, device=cuda_device)
    spec = NormSpec(w, b, kind)
    clean = norm(x, spec)
    assert torch.equal(clean[1], b)
    bad = x.clone()
    bad[2, 5], bad[4, 70] = float("nan"), float("inf")
    y = norm(bad, spec)
    good = [0, 1, 3, 5]
    assert torch.equal(y[good], clean[good]) and y[2].isnan().all() and not y[4].isfinite().all()
    out, y2 = residual_norm(x, bad, post_norm=spec, next_norm=spec)
    ref, ref2 = residual_norm(x, x, post_norm=spec, next_norm=spec)
    assert torch.equal(out[good], ref[good]) and torch.equal(y2[good], ref2[good])


def test_residual_dropout_is_dropout(cuda_device):
    """With nothing else asked for, the fused call adds exactly what dropout() gives."""
    from pack3d_b200 import dropout, residual_norm
    for dim in (64, 77):
        h = torch.randn(21, dim, device=cuda_device)
        out, _ = residual_norm(torch.zeros_like(h), h, p=0.4, rng=(5, 6))
        assert torch.equal(out, dropout(h, 0.4, (5, 6)))


def test_residual_strides_alignment_and_empty(cuda_device):
    from pack3d_b200 import NormSpec, residual_norm
    big = torch.randn(12, 2 * 80 + 2, device=cuda_device, dtype=torch.bfloat16)
    x, h = big[:, :80], big[:, 81:161]
    w = torch.rand(81, device=cuda_device, dtype=torch.bfloat16)[1:]
    spec = NormSpec(w)
    want = residual_norm(x.contiguous(), h.contiguous(), post_norm=NormSpec(w.clone()), next_norm=NormSpec(w.clone()))
    got = residual_norm(x, h, post_norm=spec, next_norm=spec)
    for a, b in zip(got, want):
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -8 * b.float().abs().max()   # other summation order
    e = torch.empty(0, 3, 80, device=cuda_device, requires_grad=True)
    w32 = torch.ones(80, device=cuda_device, requires_grad=True)
    out, y = residual_norm(e, e * 1, post_norm=NormSpec(w32), next_norm=NormSpec(w32))
    g = torch.autograd.grad(out.sum() + y.sum(), [e, w32])
    assert out.shape == y.shape == (0, 3, 80) and g[0].shape == (0, 3, 80) and (g[1] == 0).all()


def test_norm_matches_residual_and_gradient_by_differences(cuda_device):
    """norm() by itself, and its gradient against central differences in 64 bits of the plain form."""
    from pack3d_b200 import NormSpec, norm
    for kind in ("rms", "layer"):
        x = make((5, 40), torch.float32, cuda_device, 4).requires_grad_()
        w = make((40,), torch.float32, cuda_device, 5, 1.0, 0.3).requires_grad_()
        dy = make((5, 40), torch.float32, cuda_device, 6)
        y = norm(x, NormSpec(w, None, kind))
        close(y, plain_norm(x.double(), (w.double(), None, kind, 1e-6)), torch.float32)
        dx, dw = torch.autograd.grad(y, [x, w], dy)

        def loss(xd, wd):
            return (plain_norm(xd, (wd, None, kind, 1e-6)) * dy.double()).sum()

        for t, d in ((x, dx), (w, dw)):
            probe = torch.randn(t.shape, generator=torch.Generator().manual_seed(8)).double().to(cuda_device)
            step = 1e-5
            xs, ws = x.detach().double(), w.detach().double()
            at = [(xs + s * probe, ws) if t is x else (xs, ws + s * probe) for s in (step, -step)]
            numeric = (loss(*at[0]) - loss(*at[1])) / (2 * step)
            analytic = (d.double() * probe).sum()
            # central differences err by step^2, the gradient by fp32 roundings of 200 terms of order one
            assert abs(numeric - analytic) < 1e-3


def test_second_derivative_is_refused(cuda_device):
    from pack3d_b200 import NormSpec, dropout, fp8_linear, norm
    x = torch.randn(6, 32, device=cuda_device, requires_grad=True)
    w = torch.randn(16, 32, device=cuda_device, requires_grad=True)
    for f in (lambda t: dropout(t, 0.5, (1, 2)), lambda t: norm(t, NormSpec()), lambda t: fp8_linear(t, w)):
        y = f(x)
        dy = torch.ones_like(y, requires_grad=True)
        dx, = torch.autograd.grad(y, [x], dy, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            dx.sum().backward()


def test_changed_input_is_noticed(cuda_device):
    from pack3d_b200 import NormSpec, norm
    x = torch.randn(6, 32, device=cuda_device, requires_grad=True) * 1
    y = norm(x, NormSpec())
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals(cuda_device):
    from pack3d_b200 import NormSpec, dropout, norm, residual_norm
    x = torch.randn(4, 6, 32, device=cuda_device)
    w = torch.ones(32, device=cuda_device)
    with pytest.raises(ValueError, match="between 0 and 1"):
        dropout(x, 1.5, (1, 2))
    with pytest.raises(ValueError, match="between 0 and 1"):
        dropout(x, float("nan"), (1, 2))
    for rng in (None, 3, (1,), torch.zeros(2, device=cuda_device), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="rng"):
            dropout(x, 0.5, rng)
    with pytest.raises(ValueError, match="CUDA"):
        dropout(x.double(), 0.5, (1, 2))
    with pytest.raises(ValueError, match="shape"):
        norm(x, NormSpec(w[:16]))
    with pytest.raises(ValueError, match="kind"):
        norm(x, NormSpec(w, None, "batch"))
    with pytest.raises(ValueError, match="eps"):
        norm(x, NormSpec(w, None, "rms", -1.0))
    with pytest.raises(ValueError, match="parameters must be"):
        norm(x, NormSpec(w.half()))
    with pytest.raises(ValueError, match="same device"):
        norm(x, NormSpec(w.cpu()))
    with pytest.raises(ValueError, match="last dimension"):
        norm(torch.randn(2, 16385, device=cuda_device), NormSpec())
    with pytest.raises(ValueError, match="NormSpec"):
        norm(x, w)
    with pytest.raises(ValueError, match="h must"):
        residual_norm(x, x[:2])
    with pytest.raises(ValueError, match="gate must"):
        residual_norm(x, x, gate=torch.ones(4, 6, 16, device=cuda_device))
    with pytest.raises(ValueError, match="gate must"):
        residual_norm(x, x, gate=torch.ones(2, 1, 32, device=cuda_device))
    with pytest.raises(ValueError, match="gate_activation"):
        residual_norm(x, x, gate=x, gate_activation="relu")
    with pytest.raises(ValueError, match="rng"):
        residual_norm(x, x, p=0.5)


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 elements: the last rows, forward and backward, are those of a call with these rows alone, and
    their dropout is not that of the rows 2^31 elements before."""
    from pack3d_b200 import NormSpec, dropout, norm
    rows, dim, tail = 2 ** 19 + 200, 4096, 200
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device=cuda_device).normal_(generator=g).requires_grad_()
    w = torch.randn(dim, device=cuda_device, generator=g)
    y = norm(x, NormSpec(w))
    dy = torch.empty_like(y).normal_(generator=g)
    y.backward(dy)
    last = x.detach()[-tail:].clone().requires_grad_()
    want = norm(last, NormSpec(w))
    want.backward(dy[-tail:].clone())
    assert torch.equal(y[-tail:], want) and torch.equal(x.grad[-tail:], last.grad)
    ones = x.detach().fill_(1.0)
    kept = dropout(ones, 0.5, (5, 2)) != 0
    same = (kept[-tail:] == kept[:tail]).float().mean().item()
    assert abs(same - 0.5) < 5 * 0.5 / (tail * dim) ** 0.5      # five deviations of that many fair coins


@pytest.mark.parametrize("dim", [8200, 8960, 10248, 12296])
@pytest.mark.parametrize("nxt", [True, False])
def test_sample_gate_of_rows_over_uneven_clusters(cuda_device, dim, nxt):
    """fp32 widths whose rows fill fewer than eight CTAs of whole warps, with a gate whose last vector ends the tensor."""
    check_residual(cuda_device, (3, 5, dim), torch.float32, "layer", "sample", "tanh", nxt=nxt, seed=dim)


@pytest.mark.parametrize("dim", [1, 2, 3, 7])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_shorter_than_a_copied_piece(cuda_device, dim, dtype):
    check_residual(cuda_device, (2, 301, dim), dtype, "rms", "element", "sigmoid", 0.25, seed=dim)


@pytest.mark.parametrize("gate", [None, "element", "token", "sample"])
@pytest.mark.parametrize("dim", [64, 1024, 77])
@pytest.mark.parametrize("p,nxt", [(0.0, False), (0.5, False), (0.5, True)])
@pytest.mark.parametrize("scale", [True, False])
def test_gradients_beside_infinity_and_nan_in_the_block(cuda_device, gate, dim, p, nxt, scale):
    """Without a post norm the block's output enters no gradient but the gate's and the scale's: where it is infinite or
    NaN, its own gradient is as finite as elsewhere, and what is dropped adds nothing to any.  Compared wherever the
    plain form's gradient is finite; with a next norm only dropped places hold infinities and NaN."""
    from pack3d_b200 import NormSpec, residual_norm
    shape, rng, dtype = (2, 6, dim), (7, 8), torch.float32
    keep = keep_mask(12, dim, p, rng).view(shape).to(cuda_device) if p else None
    h = make(shape, dtype, cuda_device, 1)
    bad = torch.zeros(shape, dtype=torch.bool, device=cuda_device)
    bad[0, 1, 3::9], bad[1, 4, 5::7], bad[1, 2, ::11] = True, True, True
    if nxt:
        bad &= ~keep
    h[bad] = float("inf")
    h[1, 2][bad[1, 2]] = float("nan")
    leaves = {"x": make(shape, dtype, cuda_device, 2), "h": h}
    gate_shape = {None: None, "element": shape, "token": (2, 6, 1), "sample": (2, 1, dim)}[gate]
    if gate_shape:
        leaves["gate"] = make(gate_shape, dtype, cuda_device, 3)
    if scale:
        leaves["scale"] = make((dim,), dtype, cuda_device, 4, 0.5, 0.2)
    if nxt:
        leaves["nw"] = make((dim,), dtype, cuda_device, 5, 1.0, 0.2)
    for t in leaves.values():
        t.requires_grad_()
    exact = {k: t.detach().double().requires_grad_() for k, t in leaves.items()}
    out, y = residual_norm(leaves["x"], leaves["h"], gate=leaves.get("gate"), gate_activation="tanh",
                           scale=leaves.get("scale"), next_norm=NormSpec(leaves["nw"]) if nxt else None, p=p, rng=rng)
    want_out, want_y = plain_residual(exact["x"], exact["h"], None, exact.get("gate"), "tanh", exact.get("scale"),
                                      (exact["nw"], None, "rms", 1e-6) if nxt else None, keep, 1 / (1 - p))
    up = [make(shape, dtype, cuda_device, 6 + i) for i in range(1 + nxt)]
    got = torch.autograd.grad([out, y][:1 + nxt], list(leaves.values()), up)
    want = torch.autograd.grad([want_out, want_y][:1 + nxt], list(exact.values()), [u.double() for u in up])
    for name, a, b in zip(leaves, got, want):
        at = torch.isfinite(b)
        assert name not in ("x", "h") or at.all()
        close(a[at], b[at], dtype, {"x": 1, "h": 1, "gate": dim if gate == "token" else 6}.get(name, 12))


@pytest.mark.parametrize("gate", [None, "element", "token", "sample"])
@pytest.mark.parametrize("dim", [64, 1024, 77])
def test_dropped_infinity_under_an_rms_norm(cuda_device, gate, dim):
    """An RMS norm takes a row with an infinity to zeros beside it: dropped, the infinity leaves out and the scale's
    gradient finite."""
    from pack3d_b200 import NormSpec, residual_norm
    shape, rng = (2, 6, dim), (7, 8)
    keep = keep_mask(12, dim, 0.5, rng).view(shape).to(cuda_device)
    h = make(shape, torch.float32, cuda_device, 1)
    bad = torch.zeros(shape, dtype=torch.bool, device=cuda_device)
    bad[0, 1, 3::9], bad[1, 4, 5::7] = True, True
    h[bad & ~keep] = float("inf")
    x, w = make(shape, torch.float32, cuda_device, 2), make((dim,), torch.float32, cuda_device, 3, 1.0, 0.2)
    s, nw = make((dim,), torch.float32, cuda_device, 4, 0.5, 0.2), make((dim,), torch.float32, cuda_device, 5, 1.0, 0.2)
    gate_shape = {None: None, "element": shape, "token": (2, 6, 1), "sample": (2, 1, dim)}[gate]
    g = make(gate_shape, torch.float32, cuda_device, 9) if gate_shape else None
    up = [make(shape, torch.float32, cuda_device, 6 + i) for i in range(2)]

    def grads(run, *leaves):
        leaves = [t.requires_grad_() for t in leaves]
        out, y = run(*leaves)
        return (out, *torch.autograd.grad([out, y], leaves, [u.to(out.dtype) for u in up]))

    got = grads(lambda x, s, nw: residual_norm(x, h.requires_grad_(), post_norm=NormSpec(w), gate=g, gate_activation="tanh", scale=s,
                                               next_norm=NormSpec(nw), p=0.5, rng=rng), x.clone(), s.clone(), nw.clone())
    want = grads(lambda x, s, nw: plain_residual(x, h.double(), (w.double(), None, "rms", 1e-6), None if g is None else g.double(),
                                                 "tanh", s, (nw, None, "rms", 1e-6), keep, 2.0),
                 x.double(), s.double(), nw.double())
    for a, b, rows in zip(got, want, (1, 1, 12, 12)):
        assert torch.isfinite(b).all()
        close(a, b, torch.float32, rows)


@pytest.mark.parametrize("dim", [64, 1024, 77])
@pytest.mark.parametrize("act", ["identity", "sigmoid", "tanh"])
@pytest.mark.parametrize("post", [None, "rms", "layer"])
def test_dropped_infinity_and_nan_in_the_gate(cuda_device, dim, act, post):
    """A gate value that is infinite or NaN where the element is dropped reaches neither out, y nor any gradient."""
    from pack3d_b200 import NormSpec, residual_norm
    shape, rng, dtype = (2, 6, dim), (7, 8), torch.float32
    keep = keep_mask(12, dim, 0.5, rng).view(shape).to(cuda_device)
    gate = make(shape, dtype, cuda_device, 1)
    bad = torch.zeros(shape, dtype=torch.bool, device=cuda_device)
    bad[0, 1, 3::9], bad[1, 4, 5::7], bad[1, 2, ::11] = True, True, True
    gate[bad & ~keep] = float("inf")
    gate[1, 2][(bad & ~keep)[1, 2]] = float("nan")
    leaves = {"x": make(shape, dtype, cuda_device, 2), "h": make(shape, dtype, cuda_device, 3), "gate": gate,
              "scale": make((dim,), dtype, cuda_device, 4, 0.5, 0.2), "nw": make((dim,), dtype, cuda_device, 5, 1.0, 0.2)}
    if post:
        leaves["pw"] = make((dim,), dtype, cuda_device, 6, 1.0, 0.2)
    for t in leaves.values():
        t.requires_grad_()
    exact = {k: t.detach().double() for k, t in leaves.items()}
    exact["gate"] = torch.where(keep, exact["gate"], 0.5)     # any finite value: it is dropped
    exact = {k: t.requires_grad_() for k, t in exact.items()}
    spec = (lambda of, cls: cls(of["pw"], None, post, 1e-6)) if post else lambda of, cls: None  # noqa: E731
    out, y = residual_norm(leaves["x"], leaves["h"], post_norm=spec(leaves, NormSpec), gate=leaves["gate"], gate_activation=act,
                           scale=leaves["scale"], next_norm=NormSpec(leaves["nw"]), p=0.5, rng=rng)
    want_out, want_y = plain_residual(exact["x"], exact["h"], spec(exact, lambda *a: a), exact["gate"], act, exact["scale"],
                                      (exact["nw"], None, "rms", 1e-6), keep, 2.0)
    close(out, want_out, dtype)
    close(y, want_y, dtype)
    up = [make(shape, dtype, cuda_device, 7 + i) for i in range(2)]
    got = torch.autograd.grad([out, y], list(leaves.values()), up)
    want = torch.autograd.grad([want_out, want_y], list(exact.values()), [u.double() for u in up])
    for name, a, b in zip(leaves, got, want):
        close(a, b, dtype, 1 if name in ("x", "h", "gate") else 12)


def test_tangents_are_refused(cuda_device):
    """Forward-mode derivatives, in any argument and in the upstream gradients: refused with and without reverse mode."""
    import torch.autograd.forward_ad as forward_ad
    from pack3d_b200 import NormSpec, dropout, fp8_linear, norm, quantize_weight, residual_norm
    x, w = torch.randn(6, 32, device=cuda_device), torch.randn(32, device=cuda_device)
    m = torch.randn(16, 32, device=cuda_device)
    kept = quantize_weight(m)
    with forward_ad.dual_level():
        for grad in (False, True):
            def dual(t):
                return forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))  # noqa: B023
            for call in (lambda: dropout(dual(x), 0.5, (1, 2)), lambda: norm(dual(x), NormSpec()),
                         lambda: norm(x, NormSpec(dual(w))), lambda: norm(x, NormSpec(w, dual(w))),
                         lambda: residual_norm(dual(x), x), lambda: residual_norm(x, dual(x)),
                         lambda: residual_norm(x, x, gate=dual(x)), lambda: residual_norm(x, x, scale=dual(w)),
                         lambda: residual_norm(x, x, post_norm=NormSpec(dual(w))),
                         lambda: residual_norm(x, x, next_norm=NormSpec(None, dual(w))),
                         lambda: fp8_linear(dual(x), m), lambda: fp8_linear(x, dual(m)),
                         lambda: fp8_linear(x, m, dual(m[:, 0])), lambda: fp8_linear(dual(x).detach(), kept, dual(m[:, 0]))):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        leaf = x.clone().requires_grad_()
        for f in (lambda t: dropout(t, 0.5, (1, 2)), lambda t: norm(t, NormSpec()), lambda t: residual_norm(t, t)[0],
                  lambda t: fp8_linear(t, m)):
            y = f(leaf)
            up = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, [leaf], up)
    for transform in (lambda f: torch.func.jvp(f, (x,), (x,)),):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            transform(lambda t: norm(t, NormSpec()))


def keep_mask_at_once(rows, dim, p, rng):
    """keep_mask over arrays."""
    import numpy as np
    seed, offset = rng
    n = rows * -(-dim // 8)
    block = np.arange(n, dtype=np.uint64)
    low, half = np.uint64(LOW), np.uint64(32)
    c = [block & low, block >> half, np.full(n, offset & LOW, np.uint64), np.full(n, offset >> 32 & LOW, np.uint64)]
    k = [seed & LOW, seed >> 32 & LOW]
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> half) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> half) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    fields = np.stack([f for w in c for f in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1)
    return torch.from_numpy(fields.reshape(rows, -1)[:, :dim] >= round(65536 * p))


def test_keep_masks_agree():
    assert torch.equal(keep_mask_at_once(7, 43, 0.3, (1 << 40, 5)), keep_mask(7, 43, 0.3, (1 << 40, 5)))


# Samples of so many rows that the forward multiplies a sample's gate into the norm's parameters: few samples, each over
# many CTAs, and many, several to a CTA; one group of rows a CTA and eight.
FOLDED = [(2, 160001, 40), (1184, 257, 40), (2, 100001, 37), (1184, 260, 37), (1184, 131, 200), (2, 40003, 195), (1184, 9, 2056),
          (3, 2401, 4096), (5, 3001, 1001)]


@pytest.mark.parametrize("shape", FOLDED)
@pytest.mark.parametrize("act,kind,post,p,scale", [("sigmoid", "layer", True, 0.25, True), ("tanh", "rms", True, 0.0, 0.5),
                                                   ("sigmoid", "rms", False, 0.25, False), ("identity", "layer", False, 0.0, True)])
def test_folded_sample_gate(cuda_device, monkeypatch, shape, act, kind, post, p, scale):
    import sys
    monkeypatch.setattr(sys.modules[__name__], "keep_mask", keep_mask_at_once)
    dtype = torch.bfloat16 if shape[1] % 2 else torch.float32
    check_residual(cuda_device, shape, dtype, kind, "sample", act, p, post, scale=scale, seed=shape[1])


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
@pytest.mark.parametrize("dim", [40, 37, 200, 4096])
def test_folded_sample_gate_is_the_gate_of_each_row(cuda_device, act, dim):
    """The same rows with the gate given for each element: only the order of two multiplications differs."""
    from pack3d_b200 import NormSpec, residual_norm
    batch, tokens = (2, 80000) if dim < 300 else (2, 6000)
    g = torch.Generator(device=cuda_device).manual_seed(dim)
    x, h = (torch.randn(batch, tokens, dim, device=cuda_device, generator=g) for _ in range(2))
    gate = torch.randn(batch, 1, dim, device=cuda_device, generator=g)
    w, s = (torch.randn(dim, device=cuda_device, generator=g) for _ in range(2))
    run = lambda gate: residual_norm(x, h, post_norm=NormSpec(w), gate=gate, gate_activation=act, scale=s,  # noqa: E731
                                     next_norm=NormSpec(), p=0.25, rng=(3, 4))
    for a, b in zip(run(gate), run(gate.expand(x.shape).contiguous())):
        # eight fp32 roundings of values up to the size of either, and as much again in the deviation that divides y
        assert ((a - b).abs() <= 2.0 ** -20 * (b.abs() + x.abs() + 1)).all()


@pytest.mark.parametrize("post,nxt", [("rms", "layer"), ("layer", "rms")])
@pytest.mark.parametrize("dim", [96, 101, 1032])
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_norms_of_two_kinds(cuda_device, post, nxt, dim, p):
    from pack3d_b200 import NormSpec, residual_norm
    shape, rng = (3, 7, dim), (5, 6)
    keep = keep_mask(21, dim, p, rng).view(shape).to(cuda_device) if p else None
    leaves = [make(shape, torch.float32, cuda_device, 1, 0.3, 1.5), make(shape, torch.float32, cuda_device, 2, -0.2, 0.7)]
    leaves += [make((dim,), torch.float32, cuda_device, 3 + i, 1.0, 0.2) for i in range(3)]
    leaves = [t.requires_grad_() for t in leaves]
    exact = [t.detach().double().requires_grad_() for t in leaves]
    x, h, pw, nw, s = leaves
    got = residual_norm(x, h, post_norm=NormSpec(pw, None, post), scale=s, next_norm=NormSpec(nw, None, nxt), p=p, rng=rng)
    x, h, pw, nw, s = exact
    want = plain_residual(x, h, (pw, None, post, 1e-6), None, None, s, (nw, None, nxt, 1e-6), keep, 1 / (1 - p))
    up = [make(shape, torch.float32, cuda_device, 7 + i) for i in range(2)]
    for a, b in zip(got, want):
        close(a, b, torch.float32)
    for i, (a, b) in enumerate(zip(torch.autograd.grad(got, leaves, up),
                                   torch.autograd.grad(want, exact, [u.double() for u in up]))):
        close(a, b, torch.float32, 1 if i < 2 else 21)
