"""Packed-sequence attention and the norms with rotation over values that are not finite, small gradients and long sums, against
their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAN, INF = math.nan, math.inf


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    """No bounded wait of a kernel gave up."""
    yield
    from pack3d_b200 import _native
    assert _native.device_errors() == 0


def offsets_of(lengths, device):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


def randn(*shape, device, seed, dtype, scale=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device=device) * scale).to(dtype)


# ------------------------------------------------------------------------------- scores that are infinite
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 128), (BF16, 128), (F16, 48)])
@pytest.mark.parametrize("keys", [64, 128, 256])
@pytest.mark.parametrize("causal", [False, True])
def test_infinite_scores(cuda_device, dtype, dim, keys, causal):
    """A key with an infinity in one column, at every place of the last 64, one to a sequence: queries with a positive, a negative or both
    signs in that column. NaN exactly where the 64-bit softmax is, and its value elsewhere."""
    from pack3d_b200 import sequence_attention
    rows, heads, last = 160, 2, 64
    q = randn(last, rows, heads, dim, device=cuda_device, seed=1, dtype=dtype)
    k = randn(last, keys, 1, dim, device=cuda_device, seed=2, dtype=dtype)
    v = randn(last, keys, 1, dim, device=cuda_device, seed=3, dtype=dtype)
    at = torch.arange(last, device=cuda_device)
    k[at, keys - last + at, 0, 3] = INF
    for sign in (1, -1, 0):
        x = q.clone()
        x[..., 3] = q[..., 3].abs() * sign if sign else q[..., 3]
        x[..., 3] += 0.125 * torch.where(x[..., 3] < 0, -1, 1)    # not 0
        got = sequence_attention(x.flatten(0, 1), k.flatten(0, 1), v.flatten(0, 1), offsets_of([rows] * last, cuda_device),
                                 offsets_of([keys] * last, cuda_device), causal=causal).view(last, rows, heads, dim)
        s = torch.einsum("bihd,bjd->bhij", x.double(), k[:, :, 0].double()) * dim ** -0.5
        if causal:
            s = torch.where(torch.ones(rows, keys, dtype=torch.bool, device=cuda_device).tril(keys - rows), s, -INF)
        p = torch.softmax(s, -1)
        nothing = s.new_zeros(rows, dtype=torch.bool)
        if causal and rows > keys:
            nothing[:rows - keys] = True
            p = torch.where(nothing[:, None], 0.0, p)
        want = torch.einsum("bhij,bjd->bihd", p, v[:, :, 0].double())
        assert torch.equal(got.isnan(), want.isnan())
        # weights and results rounded (half a step each), exponentials to 2^-13, sums in fp32
        u = torch.finfo(dtype).eps / 2
        tol = (2 * u + 2.0 ** -13 + 2.0 ** -15) * torch.einsum("bhij,bjd->bihd", p, v[:, :, 0].double().abs()) + 2.0 ** -24
        there = ~want.isnan()
        assert there.any() or sign == 1
        assert ((got.double() - want).abs() <= tol)[there].all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("keys", [64, 128, 192])
def test_every_score_minus_infinity(cuda_device, dtype, keys):
    """The softmax of nothing but -inf is NaN, and so are the gradients that come of it; the sequence beside it keeps its own."""
    from pack3d_b200 import sequence_attention
    rows, dim = 128, 64
    q = randn(2 * rows, 1, dim, device=cuda_device, seed=1, dtype=dtype)
    k, v = (randn(2 * keys, 1, dim, device=cuda_device, seed=s, dtype=dtype) for s in (2, 3))
    q[:rows, :, 3] = 1
    qo, ko = offsets_of([rows, rows], cuda_device), offsets_of([keys, keys], cuda_device)

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = sequence_attention(*leaves, qo, ko, causal=False)
        return [out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))]
    clean = run()
    k[:keys, :, 3] = -INF
    for got, before, n in zip(run(), clean, (rows, rows, keys, keys)):
        assert got[:n].isnan().all() and torch.equal(got[n:], before[n:])


# ------------------------------------------------------------------------------- values that nobody before them sees
def step(q, k, v, dout, offsets, causal=True, k_offsets=None):
    """(out, dq, dk, dv) and the milliseconds that they took."""
    from pack3d_b200 import sequence_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    out = sequence_attention(*leaves, offsets, k_offsets, causal=causal)
    grads = torch.autograd.grad(out, leaves, dout)
    end.record()
    end.synchronize()
    return [out.detach(), *grads], start.elapsed_time(end)


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("at", [0, 63, 64, 100, 255, 290])
@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 64), (3, 3, 128), (8, 1, 48)])
def test_later_values_keep_out_of_earlier_rows(cuda_device, value, at, heads, kv, dim):
    """A value, key, query or gradient row that is not finite: what does not see it keeps its bits, in every column."""
    n = 300
    offsets = offsets_of([n], cuda_device)
    clean = [randn(n, h, dim, device=cuda_device, seed=s, dtype=BF16) for s, h in enumerate((heads, kv, kv, heads))]
    want, _ = step(*clean, offsets)
    for which in range(4):
        tensors = [t.clone() for t in clean]
        tensors[which][at, 0, 3] = value
        got, _ = step(*tensors, offsets)
        assert torch.equal(got[0][:at], want[0][:at]) and torch.equal(got[1][:at], want[1][:at])
        if which in (0, 3):
            assert all(torch.equal(got[i][at + 1:], want[i][at + 1:]) for i in (2, 3))
        if which == 2:
            # weights are positive: the column of every query that sees it, and no other
            column = torch.full_like(got[0][at:, :heads // kv, 3], value)
            assert torch.equal(got[0][at:, :heads // kv, 3].nan_to_num(7.0), column.nan_to_num(7.0))
            keep = torch.arange(dim, device=cuda_device) != 3
            assert torch.equal(got[0][at:][..., keep], want[0][at:][..., keep])
        if which == 3:
            # dv of every key that the row sees has the weight's sign in that column; the row's own score gradient is not finite
            seen = got[3][:at + 1, 0, 3]
            assert seen.isnan().all() if math.isnan(value) else (seen == value).all()
            keep = torch.arange(dim, device=cuda_device) != 3
            assert torch.equal(got[3][..., keep], want[3][..., keep])
            assert (at == 0 or got[1][at, 0].isnan().any()) and not got[2][:at + 1, 0].isfinite().all()


@pytest.mark.parametrize("n", [130, 256, 300])
@pytest.mark.parametrize("at", [0, 1, 63, 64, 127, 129])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(2, 1, 64, BF16), (3, 3, 128, F16)])
@pytest.mark.parametrize("causal", [True, False])
def test_a_key_without_weight_that_is_infinite(cuda_device, n, at, heads, kv, dim, dtype, causal):
    """A key whose score is -inf for every query has no weight, and its score gradient is 0: times the infinity, NaN in that column of dq for
    every query that sees it, whole tile or not; all else as if the key were not seen."""
    offsets = offsets_of([n], cuda_device)
    q, k, v, dout = (randn(n, h, dim, device=cuda_device, seed=s, dtype=dtype) for s, h in enumerate((heads, kv, kv, heads)))
    q[:, :, 3] = 1
    k[at, :, 3] = -INF
    (out, dq, dk, dv), _ = step(q, k, v, dout, offsets, causal=causal)
    sees = torch.ones(n, dtype=torch.bool, device=cuda_device)
    if causal:
        sees[:at] = False
    nothing = sees.clone()
    nothing[1 if causal and at == 0 else 0:] = False        # a query that sees that key alone
    keep = torch.arange(dim, device=cuda_device) != 3
    assert dq[sees][..., 3].isnan().all() and dq[~sees].isfinite().all()
    assert out[~nothing].isfinite().all() and dq[~nothing][..., keep].isfinite().all()
    if not nothing.any():
        assert not dk[at].any() and not dv[at].any() and dk.isfinite().all() and dv.isfinite().all()
    other = torch.arange(n, device=cuda_device) != at
    if not causal:
        want, _ = step(q, k[other], v[other], dout, offsets, causal=False, k_offsets=offsets_of([n - 1], cuda_device))
        u = torch.finfo(dtype).eps / 2
        # the same sums in another order of tiles: weights and score gradients round alike, the accumulations in fp32 do not
        for a, b in ((out, want[0]), (dq[..., keep], want[1][..., keep]), (dk[other], want[2]), (dv[other], want[3])):
            assert (a.double() - b.double()).norm() <= 8 * u * b.double().norm()


def test_signs_that_meet(cuda_device):
    """A column with infinities of both signs is NaN from the second on, and the first one's sign in between; the same of gradients, from
    the other end."""
    n, dim = 400, 64
    offsets = offsets_of([n], cuda_device)
    q, k, v, dout = (randn(n, 1, dim, device=cuda_device, seed=s, dtype=BF16) for s in range(4))
    for first, second in ((10, 50), (130, 140), (130, 300), (383, 390)):
        x, d = v.clone(), dout.clone()
        x[first, 0, 5], x[second, 0, 5], x[second, 0, 6] = INF, -INF, -INF
        out = step(q, k, x, dout, offsets)[0][0][:, 0]
        assert out[:first].isfinite().all() and (out[first:second, 5] == INF).all() and out[second:, 5].isnan().all()
        assert out[:second, 6].isfinite().all() and (out[second:, 6] == -INF).all() and out[:, 7:].isfinite().all()
        d[first, 0, 5], d[second, 0, 5], d[first, 0, 6] = INF, -INF, -INF
        dv = step(q, k, v, d, offsets)[0][3][:, 0]
        assert dv[second + 1:].isfinite().all() and (dv[first + 1:second + 1, 5] == -INF).all() and dv[:first + 1, 5].isnan().all()
        assert dv[first + 1:, 6].isfinite().all() and (dv[:first + 1, 6] == -INF).all() and dv[:, 7:].isfinite().all()


@pytest.mark.parametrize("prefix", [0, 70, -40])
@pytest.mark.parametrize("heads,kv", [(4, 1), (3, 3)])
def test_prefix_with_values_that_are_not_finite(cuda_device, prefix, heads, kv):
    """Keys of other lengths than the queries: masks that begin anywhere in a tile, and rows that see nothing."""
    lengths = [129, 1, 64, 200]
    keys = [max(0, n + prefix) for n in lengths]
    offsets, k_offsets = offsets_of(lengths, cuda_device), offsets_of(keys, cuda_device)
    clean = [randn(sum(r), h, 80, device=cuda_device, seed=s, dtype=F16) for s, (h, r) in enumerate(((heads, lengths), (kv, keys), (kv, keys), (heads, lengths)))]
    want, _ = step(*clean, offsets, k_offsets=k_offsets)
    at = sum(lengths[:3]) + 100
    key = sum(keys[:3]) + 100 + prefix            # what query 100 of the last sequence sees last
    for which in range(4):
        tensors = [t.clone() for t in clean]
        tensors[which][at if which in (0, 3) else key, 0, 2] = NAN if which == 1 else INF   # -inf scores would have no weight
        got, _ = step(*tensors, offsets, k_offsets=k_offsets)
        if which in (1, 2):                        # earlier queries, and all of the other sequences
            assert torch.equal(got[0][:at], want[0][:at]) and torch.equal(got[1][:at], want[1][:at])
            assert not got[0][at, 0].isfinite().all()
        else:                                      # later keys, and the other sequences' ones
            for i in (2, 3):
                assert torch.equal(got[i][key + 1:], want[i][key + 1:])
                assert torch.equal(got[i][:sum(keys[:3])], want[i][:sum(keys[:3])])
                assert not got[i][key, 0].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("what", ["dout nan", "dout inf", "dout one inf a row", "v channel", "v nan", "k channel", "q nan"])
def test_many_that_are_not_finite(cuda_device, what, dtype):
    """A step whose values have overflown, at a length where work that grows with its square would show: as every value is looked at a
    bounded number of times, it stays within 30 ms (all finite: about one)."""
    n, heads, kv, dim = 8192, 8, 2, 128
    offsets = offsets_of([n], cuda_device)
    q, k, v, dout = (randn(n, h, dim, device=cuda_device, seed=s, dtype=dtype) for s, h in enumerate((heads, kv, kv, heads)))
    clean, _ = step(q, k, v, dout, offsets)
    if what == "dout nan":
        dout[:] = NAN
    elif what == "dout inf":
        dout[:] = INF
    elif what == "dout one inf a row":
        dout[:, :, 9] = INF
    elif what == "v channel":
        v[:, :, 9] = INF
    elif what == "v nan":
        v[:] = NAN
    elif what == "k channel":
        k[:, :, 9] = INF
    else:
        q[:] = NAN
    (out, dq, dk, dv), ms = step(q, k, v, dout, offsets)
    assert ms < 30
    keep = torch.arange(dim, device=cuda_device) != 9
    if what.startswith("dout"):
        assert torch.equal(out, clean[0])
        if what == "dout one inf a row":
            assert (dv[..., 9] == INF).all() and torch.equal(dv[..., keep], clean[3][..., keep])
        elif what == "dout nan":
            assert dv.isnan().all() and dq.isnan().all() and dk.isnan().all()
        else:
            assert (dv == INF).all()
    elif what == "v channel":
        assert (out[..., 9] == INF).all() and torch.equal(out[..., keep], clean[0][..., keep])
    elif what == "v nan":
        assert out.isnan().all()
    elif what == "q nan":
        assert out.isnan().all() and dq.isnan().all() and dk.isnan().all() and dv.isnan().all()
    else:
        # queries see an infinite key of either sign: NaN where any score is +inf, and where all are -inf
        assert out.isnan().all() and dq.isnan().all()


@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 64), (3, 3, 128), (8, 1, 48), (16, 4, 128)])
def test_a_value_reaches_every_row_that_sees_it(cuda_device, value, heads, kv, dim):
    """Two tiles of queries share what is cleared of their values, in any order: at every place of a tile, over many sequences."""
    from pack3d_b200 import sequence_attention
    n, count = 256, 64
    offsets = offsets_of([n] * count, cuda_device)
    q, k, v = (randn(n * count, h, dim, device=cuda_device, seed=s, dtype=BF16) for s, h in enumerate((heads, kv, kv)))
    clean = sequence_attention(q, k, v, offsets).view(count, n, heads, dim)
    at = torch.arange(count, device=cuda_device) * 4 + 1
    v.view(count, n, kv, dim)[torch.arange(count, device=cuda_device), at, 0, 3] = value
    sees = (torch.arange(n, device=cuda_device) >= at[:, None])[..., None]
    want = clean.clone()
    want[..., :heads // kv, 3] = torch.where(sees, value, want[..., :heads // kv, 3])
    for _ in range(5):
        out = sequence_attention(q, k, v, offsets).view(count, n, heads, dim)
        assert torch.equal(out.nan_to_num(3.25), want.nan_to_num(3.25))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("value", [NAN, INF, -INF])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (3, 3, 64)])
def test_a_channel_of_values_that_are_not_finite(cuda_device, dtype, value, heads, kv, dim):
    """One column of every value: the other columns keep their bits, and it takes no longer than a few times the usual (below 1 ms)."""
    from pack3d_b200 import sequence_attention
    n = 8192
    offsets = offsets_of([n - 900, 900], cuda_device)
    q, k, v = (randn(n, h, dim, device=cuda_device, seed=s, dtype=dtype) for s, h in enumerate((heads, kv, kv)))
    clean = sequence_attention(q, k, v, offsets)
    v[:, :, 9] = value
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    out = sequence_attention(q, k, v, offsets)
    end.record()
    end.synchronize()
    assert start.elapsed_time(end) < 15
    keep = torch.arange(dim, device=cuda_device) != 9
    assert torch.equal(out[..., keep], clean[..., keep])
    assert out[..., 9].isnan().all() if math.isnan(value) else (out[..., 9] == value).all()


@pytest.mark.parametrize("heads,kv", [(2, 1), (1, 1)])
def test_infinite_value_at_the_end_of_a_long_sequence(cuda_device, heads, kv):
    """200,000 tokens, the last ones' values infinite: the rows before keep their bits, as do sequences behind it, in bounded time."""
    from pack3d_b200 import sequence_attention
    lengths = [200000, 5, 700]
    offsets = offsets_of(lengths, cuda_device)
    q, k, v = (randn(sum(lengths), h, 64, device=cuda_device, seed=s, dtype=BF16) for s, h in enumerate((heads, kv, kv)))
    clean = sequence_attention(q, k, v, offsets)
    v[199990:200000] = INF
    out = sequence_attention(q, k, v, offsets)
    assert torch.equal(out[:199990], clean[:199990]) and torch.equal(out[200000:], clean[200000:])
    assert (out[199990:200000] == INF).all()


# ------------------------------------------------------------------------------- gradients and weights of any size
def coherent(n, heads, kv, dim, up, device, small=1.0):
    """Queries, keys, values and upstream gradients whose score gradients are about 1 / n each and add up to results of the order of
    `up`: V_j and K_j have a common sign each, dO one direction for all rows, and scores are near 0."""
    def noise(h, s):
        return randn(n, h, dim, device=device, seed=s, dtype=F32) * 0.1
    gen = torch.Generator(device=device).manual_seed(9)
    sign = torch.randint(0, 2, (n, kv, 1), generator=gen, device=device) * 2.0 - 1
    g = torch.randint(0, 2, (dim,), generator=gen, device=device) * 2.0 - 1
    half = torch.ones(dim, device=device)
    half[dim // 2:] = -1
    q = (0.5 * half + noise(heads, 1)) * small
    k = (sign + noise(kv, 2)) * small
    return q.half(), k.half(), (sign * g + noise(kv, 3)).half(), ((g + noise(heads, 4)) * up).half()


def definition(q, k, v, dout, causal, scale):
    """(out, dq, dk, dv) in 64 bits of one sequence, and how far a kernel may be off: weights p and score gradients ds are rounded to the
    dtype before a product, half a step u relative, or half of the smallest f16 number beside 2^10 for p and beside 2^11 for the
    largest that a row's (a key's) ds can be; exponentials are off by 2^-13, sums in fp32 by 2^-15 of magnitudes, out (which delta
    comes from) by what its own rounding and its weights' make, results by half a step, or half of the smallest number."""
    u, e, least = torch.finfo(q.dtype).eps / 2, 2.0 ** -13 + 2.0 ** -15, 2.0 ** -25
    q, k, v, d = (t.double() for t in (q, k, v, dout))
    n, h, g = q.shape[0], q.shape[1], k.shape[1]
    out, grads, tols = torch.zeros_like(q), [torch.zeros_like(t) for t in (q, k, v)], [torch.zeros_like(t) for t in (q, k, v)]
    for i in range(h):
        j = i // (h // g)
        s = q[:, i] @ k[:, j].t() * scale
        if causal:
            s = torch.where(torch.ones_like(s, dtype=torch.bool).tril(), s, -INF)
        p = torch.softmax(s, -1)
        o = p @ v[:, j]
        out[:, i] = o
        out_tol = u * o.abs() + (u + e) * (p @ v[:, j].abs())
        dp = d[:, i] @ v[:, j].t()
        delta = (d[:, i] * o).sum(-1, keepdim=True)
        ds = p * (dp - delta) * scale
        # the largest that ds of a row can be, by Cauchy and Schwarz, for the power of two that it is held in
        most = scale * (d[:, i].norm(dim=-1, keepdim=True) * v[:, j].norm(dim=-1).max() + delta.abs())
        wrong = scale * p * (e * (dp.abs() + delta.abs() + d[:, i].abs() @ v[:, j].abs().t()) + (d[:, i].abs() * out_tol).sum(-1, keepdim=True)) + u * ds.abs()
        floor = least * 2.0 ** -11
        grads[0][:, i] = ds @ k[:, j]
        tols[0][:, i] = (wrong + e * ds.abs()) @ k[:, j].abs() + floor * most * k[:, j].abs().sum(0)
        grads[1][:, j] += ds.t() @ q[:, i]
        tols[1][:, j] += (wrong + e * ds.abs()).t() @ q[:, i].abs() + floor * most.max() * q[:, i].abs().sum(0)
        grads[2][:, j] += p.t() @ d[:, i]
        tols[2][:, j] += (u + 2 * e) * (p.t() @ d[:, i].abs()) + least * 2.0 ** -10 * d[:, i].abs().sum(0)
        del s, p, dp, ds, wrong
    return out, grads, [t + u * x.abs() + least for t, x in zip(tols, grads)]


@pytest.mark.parametrize("causal,n", [(False, 12000), (True, 9001)])
@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 64), (1, 1, 128)])
@pytest.mark.parametrize("up,small", [(2e-5, 1.0), (1e-3, 1.0), (2e4, 0.01)])
def test_f16_gradients_of_any_size(cuda_device, causal, n, heads, kv, dim, up, small):
    """Score gradients below what f16 holds that add up to results well within it, and above it with results that are not."""
    q, k, v, dout = coherent(n, heads, kv, dim, up, cuda_device, small)
    got, _ = step(q, k, v, dout, offsets_of([n], cuda_device), causal=causal)
    _, want, tols = definition(q, k, v, dout, causal, dim ** -0.5)
    for name, g, w, t in zip("qkv", got[1:], want, tols):
        # the first keys' values have gradients of up to 2 * 2e4 * (1 + 1/2 + ..), past the largest f16 number: infinite, as rounded;
        # where the error may carry them over that border, either
        past = w.abs() >= 65520 + t
        assert (g.double() == w.sign() * INF)[past].all() and (name == "v" or not past.any())
        past |= (w.abs() > 65520 - t) & (g.double() == w.sign() * INF)
        off = torch.where(past, 0.0, (g.double() - w).abs())
        assert (off <= t).all(), f"d{name}: {float((off / t).max()):.2f} x the tolerance, {float(off.norm() / w.norm()):.2e} of the norm"


@pytest.mark.parametrize("causal", [False, True])
def test_f16_value_gradients_of_small_weights(cuda_device, causal):
    """One key has nearly all of each query's weight, the others 2^-26 each, and their values' gradients are sums over many queries."""
    n, dim = 9000, 64
    q = torch.zeros(n, 1, dim, device=cuda_device, dtype=F16)
    k, v = torch.zeros_like(q), randn(n, 1, dim, device=cuda_device, seed=1, dtype=F16)
    q[..., 0] = 1
    k[0, 0, 0] = 18.0                      # e^18 is 2^26
    dout = (randn(n, 1, dim, device=cuda_device, seed=2, dtype=F32) * 0.1 + 1).half()
    from pack3d_b200 import sequence_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = sequence_attention(*leaves, offsets_of([n], cuda_device), causal=causal, scale=1.0)
    got = torch.autograd.grad(out, leaves, dout)
    _, want, tols = definition(q, k, v, dout, causal, 1.0)
    for g, w, t in zip(got, want, tols):
        assert ((g.double() - w).abs() <= t).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("first", [True, False])
def test_many_small_weights(cuda_device, dtype, first):
    """One loud key whose value is 0 and 65,536 of 2^-26 of its weight: what they add up to is not lost."""
    from pack3d_b200 import sequence_attention
    n, rows, dim = 65537, 130, 64
    at = 0 if first else n - 1
    q, k = torch.zeros(rows, 2, dim, device=cuda_device, dtype=dtype), torch.zeros(n, 1, dim, device=cuda_device, dtype=dtype)
    q[..., 0] = 1
    k[at, 0, 0] = 18.0
    v = (randn(n, 1, dim, device=cuda_device, seed=1, dtype=F32) * 0.25 + 1).to(dtype)
    v[at] = 0
    out = sequence_attention(q, k, v, offsets_of([rows], cuda_device), offsets_of([n], cuda_device), causal=False, scale=1.0)
    p = torch.softmax(k[:, 0, 0].double(), 0)
    want = (p[:, None] * v[:, 0].double()).sum(0)
    # weights: half a step, and for f16 half its smallest number beside 2^10 for the largest; exponentials and sums as everywhere
    u = torch.finfo(dtype).eps / 2
    tol = (2 * u + 2.0 ** -13 + 2.0 ** -15) * want.abs() + (2.0 ** -35 * v[:, 0].double().abs().sum(0) if dtype is F16 else 0)
    assert ((out.double() - want).abs() <= tol).all()


# ------------------------------------------------------------------------------- norms with rotation
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,pairs", [(64, (5,)), (48, (3, 0, 2)), (10, (2,)), (16, (0,))])
@pytest.mark.parametrize("value", [NAN, INF])
def test_columns_past_the_last_pair_stand_alone(cuda_device, dtype, dim, pairs, value):
    """They are not rotated: what is not finite in one of them reaches no other, nor does a gradient."""
    from pack3d_b200 import norm_rotate
    axes = len(pairs)
    positions = torch.arange(40, device=cuda_device) if axes == 1 else torch.arange(40 * axes, device=cuda_device).view(40, axes)
    x = randn(40, 3, dim, device=cuda_device, seed=1, dtype=dtype)
    up = randn(40, 3, dim, device=cuda_device, seed=2, dtype=dtype)

    def run(x, up):
        leaf = x.clone().requires_grad_()
        y, _ = norm_rotate(leaf, None, positions, pairs=pairs)
        return y.detach(), torch.autograd.grad(y, leaf, up)[0]
    clean = run(x, up)
    for column in (2 * sum(pairs), dim - 1):
        bad = [x.clone(), up.clone()]
        for t in bad:
            t[7, 1, column] = value
        for got, want, given in zip(run(*bad), clean, bad):
            expected = want.clone()
            expected[7, 1, column] = given[7, 1, column]
            assert torch.equal(got.nan_to_num(3.25), expected.nan_to_num(3.25))


@pytest.mark.parametrize("tokens,heads,kv,dim,kind", [(4097, 3, 1, 64, "rms"), (1000, 32, 8, 128, "layer"), (263, 4, 4, 48, "layer"), (1, 1, 1, 8, "rms"),
                                                      (5000, 1, 7, 250, "rms")])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_every_row_counts_in_the_parameters_gradients(cuda_device, tokens, heads, kv, dim, kind, dtype):
    """Upstream gradients in one row alone (the first and last token, head, of each input), and in all: sums to 2^-18 of their magnitudes."""
    from pack3d_b200 import NormSpec, norm_rotate
    x = [randn(tokens, h, dim, device=cuda_device, seed=s, dtype=dtype, scale=2.0) for s, h in enumerate((heads, kv))]
    positions = torch.arange(tokens, device=cuda_device) * 7 + 100000
    params = [[(1 + 0.2 * randn(dim, device=cuda_device, seed=5 + i, dtype=F32)).requires_grad_(), randn(dim, device=cuda_device, seed=7 + i, dtype=F32).requires_grad_()]
              for i in range(2)]
    spec = [NormSpec(*p, kind, 1e-5) for p in params]
    leaves = [t for p in params for t in p]
    y = norm_rotate(*x, positions, q_norm=spec[0], k_norm=spec[1])
    angle = positions.double()[:, None] * 10000.0 ** (-torch.arange(dim // 2, device=cuda_device).double() / (dim // 2))
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    for where in [None] + [(i, t, h) for i, n in enumerate((heads, kv)) for t in sorted({0, tokens - 1}) for h in sorted({0, n - 1})]:
        up = [randn(tokens, h, dim, device=cuda_device, seed=20 + i, dtype=dtype) for i, h in enumerate((heads, kv))]
        if where is not None:
            i, t, h = where
            kept = up[i][t, h].clone()
            for u in up:
                u.zero_()
            up[i][t, h] = kept
        got = torch.autograd.grad(y, leaves, up, retain_graph=True)
        for i in range(2):
            z = x[i].double()
            top = z.abs().amax(-1, keepdim=True)
            if kind == "layer":
                z = z - z.mean(-1, keepdim=True)
            r = 1 / torch.sqrt(z.square().mean(-1, keepdim=True) + 1e-5)
            z, own = z * r, top * r if kind == "layer" else 0
            a, b = up[i].double()[..., 0::2], up[i].double()[..., 1::2]
            g = torch.stack((a * cos + b * sin, b * cos - a * sin), -1).flatten(-2)
            # sine and cosine to 2^-21 and a product in fp32, of both columns of a pair; the deviation and sums in fp32
            size = torch.stack((a.abs() + b.abs(),) * 2, -1).flatten(-2)
            # a mean in fp32 is off by 2^-21 of the row's largest magnitude (eight levels of additions, the division), however near
            # to it the column lies: z is off by as much of that over the deviation
            wrong = size * (2.0 ** -18 * z.abs() + 2.0 ** -21 * own)
            for have, want, most in ((got[2 * i], (g * z).sum((0, 1)), wrong.sum((0, 1))), (got[2 * i + 1], g.sum((0, 1)), 2.0 ** -18 * size.sum((0, 1)))):
                assert ((have.double() - want).abs() <= most + 2.0 ** -24 * want.abs()).all()
