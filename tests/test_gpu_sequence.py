"""Packed-sequence attention and the norms with rotation, against their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    """No bounded wait of a kernel gave up."""
    yield
    from pack3d_b200 import _native
    assert _native.device_errors() == 0


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def offsets_of(lengths, device):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device=device)


# ------------------------------------------------------------------------------- packed sequences
def reference(q, k, v, q_len, k_len, causal, scale, dout=None):
    """out, and with dout (dq, dk, dv), in 64 bits with bounds of their errors.

    A kernel rounds weights p and score gradients ds to the tensors' dtype before a product (u relative each), sums in fp32,
    takes exponentials to 2^-13 relative, and rounds its results (u).  fp32 sums of up to a few hundred terms add under
    2^-15 of the sums of magnitudes.  delta = dout . out comes from the rounded out.
    """
    u, e = half_step(q.dtype), 2.0 ** -13 + 2.0 ** -15
    q, k, v = q.double(), k.double(), v.double()
    h, g = q.shape[1], k.shape[1]
    out, out_tol = torch.zeros_like(q), torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    tols = [torch.zeros_like(t) for t in (q, k, v)]
    q0 = k0 = 0
    for nq, nk in zip(q_len, k_len):
        sq, sk = slice(q0, q0 + nq), slice(k0, k0 + nk)
        q0, k0 = q0 + nq, k0 + nk
        if not nq or not nk:
            continue
        seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            seen = seen.tril(nk - nq)
        for i in range(h):
            qi, ki, vi = q[sq, i], k[sk, i // (h // g)], v[sk, i // (h // g)]
            s = torch.where(seen, qi @ ki.t() * scale, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)      # rows that see nothing
            o = p @ vi
            a = p @ vi.abs()
            out[sq, i] = o
            out_tol[sq, i] = u * o.abs() + (u + e) * a
            if dout is None:
                continue
            d = dout[sq, i].double()
            dp = torch.where(seen, d @ vi.t(), 0.0)
            delta = (d * o).sum(-1, keepdim=True)
            ds = p * (dp - delta) * scale
            wrong = scale * p * (e * (dp.abs() + (d.abs() * o.abs()).sum(-1, keepdim=True)) + e * (d.abs() @ vi.abs().t())
                                 + (d.abs() * out_tol[sq, i]).sum(-1, keepdim=True)) + u * ds.abs()
            grads[0][sq, i] = ds @ ki
            tols[0][sq, i] = wrong @ ki.abs() + e * (ds.abs() @ ki.abs())
            grads[1][sk, i // (h // g)] += ds.t() @ qi
            tols[1][sk, i // (h // g)] += wrong.t() @ qi.abs() + e * (ds.abs().t() @ qi.abs())
            grads[2][sk, i // (h // g)] += p.t() @ d
            tols[2][sk, i // (h // g)] += (u + 2 * e) * (p.t() @ d.abs())
    return out, out_tol, grads, [t + u * x.abs() + 2.0 ** -24 for t, x in zip(tols, grads)]


def make(q_len, k_len, heads, kv, dim, dtype, device, seed=0, extra=0, spread=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device=device)  # noqa: E731
    q = (rand(sum(q_len) + extra, heads, dim) * spread).to(dtype)
    k = (rand(sum(k_len) + extra, kv, dim) * spread).to(dtype)
    v, dout = rand(sum(k_len) + extra, kv, dim).to(dtype), rand(sum(q_len) + extra, heads, dim).to(dtype)
    return q, k, v, dout


def check(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol + 2.0 ** -24)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - want).abs() / (tol + 1e-30))[bad].max()):.2f} x the tolerance"


def run(q, k, v, dout, q_len, k_len, causal, scale=None):
    from pack3d_b200 import sequence_attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    qo = offsets_of(q_len, q.device)
    ko = None if k_len is q_len else offsets_of(k_len, q.device)
    out = sequence_attention(*leaves, qo, ko, causal=causal, scale=scale)
    return out.detach(), torch.autograd.grad(out, leaves, dout)


LENGTHS = {
    "one": ([1], None), "short": ([5, 0, 17, 1], None), "tiles": ([128, 256, 64], None), "odd": ([129, 1, 257, 0, 63], None),
    "prefix": ([1, 40, 130], [200, 41, 389]), "empty rows": ([150, 7, 30], [20, 0, 30]), "no keys": ([3, 2], [0, 0]),
    "long": ([700], None), "few queries": ([2, 3], [300, 513]),
}


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim,dtype", [(4, 2, 64, BF16), (2, 2, 128, F16), (3, 1, 48, BF16), (5, 1, 8, F16)])
def test_attention(cuda_device, lengths, causal, heads, kv, dim, dtype):
    q_len, k_len = LENGTHS[lengths]
    k_len = q_len if k_len is None else k_len
    q, k, v, dout = make(q_len, k_len, heads, kv, dim, dtype, cuda_device)
    out, grads = run(q, k, v, dout, q_len, k_len, causal)
    want, tol, want_grads, grad_tols = reference(q, k, v, q_len, k_len, causal, dim ** -0.5, dout)
    check(out, want, tol, "out")
    for name, g, w, t in zip("qkv", grads, want_grads, grad_tols):
        assert g.dtype == dtype and g.is_contiguous()
        check(g, w, t, "d" + name)


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 56, 72, 80, 88, 96, 104, 112, 120, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_head_dims(cuda_device, dim, dtype):
    lengths = [131, 70]
    q, k, v, dout = make(lengths, lengths, 2, 1, dim, dtype, cuda_device, seed=dim)
    out, grads = run(q, k, v, dout, lengths, lengths, True)
    want, tol, want_grads, grad_tols = reference(q, k, v, lengths, lengths, True, dim ** -0.5, dout)
    check(out, want, tol, "out")
    for name, g, w, t in zip("qkv", grads, want_grads, grad_tols):
        check(g, w, t, "d" + name)


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (7, 7), (8, 1), (12, 3), (16, 2)])
def test_head_groups(cuda_device, heads, kv):
    q_len, k_len = [140, 3, 0, 33], [150, 3, 9, 20]
    q, k, v, dout = make(q_len, k_len, heads, kv, 32, BF16, cuda_device, seed=heads)
    out, grads = run(q, k, v, dout, q_len, k_len, True, 0.3)
    want, tol, want_grads, grad_tols = reference(q, k, v, q_len, k_len, True, 0.3, dout)
    check(out, want, tol, "out")
    for name, g, w, t in zip("qkv", grads, want_grads, grad_tols):
        check(g, w, t, "d" + name)


@pytest.mark.parametrize("spread", [8.0, 60.0])
def test_scores_of_any_size(cuda_device, spread):
    """Scores of hundreds and thousands: the running maximum has to move, and weights underflow.  Without gradients of
    fp32 scores' own errors (|s| 2^-24 a weight) mattering: their share is added to the tolerance."""
    lengths = [300, 129]
    q, k, v, dout = make(lengths, lengths, 2, 1, 64, BF16, cuda_device, spread=spread)
    out, _ = run(q, k, v, dout, lengths, lengths, True)
    want, tol, _, _ = reference(q, k, v, lengths, lengths, True, 0.125)
    # |s| <= |q| |k| / 8, about 8 spread^2 at the most; 64 products of fp32 and the scaling: 2^-21 of it, twice in a difference
    slack = 2 * 2.0 ** -21 * 20 * spread ** 2
    check(out, want, tol + min(2.0, slack) * v.double().abs().max(), "out")
    assert torch.isfinite(out).all()


def test_extreme_rows(cuda_device):
    """A maximum that rises by the most a tile after another, and one that never moves after the first key."""
    n, dim = 520, 64
    for sign in (1.0, -1.0):
        q = torch.ones(n, 1, dim, device=cuda_device, dtype=BF16)
        k = (sign * torch.arange(n, device=cuda_device, dtype=torch.float32)[:, None, None].expand(n, 1, dim) / 16).to(BF16).contiguous()
        v = torch.randn(n, 1, dim, device=cuda_device, dtype=BF16)
        out, _ = run(q, k, v, v, [n], [n], True)
        want, tol, _, _ = reference(q, k, v, [n], [n], True, 0.125)
        check(out, want, tol + 2.0 ** -14 * v.double().abs().max(), "out")   # |s| up to 260: 2^-16 in fp32


def test_strides(cuda_device):
    """Views into one projection's rows, head-major memory, heads that share memory, and rows off their alignment."""
    lengths, dim = [77, 130], 64
    n = sum(lengths)
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    row = torch.randn(n, (4 + 2 + 2) * dim, generator=gen, device=cuda_device).to(BF16)
    q, k, v = row[:, :4 * dim].view(n, 4, dim), row[:, 4 * dim:6 * dim].view(n, 2, dim), row[:, 6 * dim:].view(n, 2, dim)
    dout = torch.randn(n, 4, dim, generator=gen, device=cuda_device).to(BF16)
    plain = run(q.contiguous(), k.contiguous(), v.contiguous(), dout, lengths, lengths, True)
    views = [(q, k, v, dout),
             (q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1), v,
              dout.transpose(0, 1).contiguous().transpose(0, 1))]
    off = torch.empty(n * 4 * dim + 1, dtype=BF16, device=cuda_device)[1:].view(n, 4, dim)
    views.append((off.copy_(q), k, v, off.clone()))
    views[-1] = (off, k, v, dout)
    wide = torch.zeros(n, 4, 2 * dim, dtype=BF16, device=cuda_device)
    wide[..., ::2] = q
    views.append((wide[..., ::2], k, v, dout))
    for case in views:
        got = run(*case, lengths, lengths, True)
        assert torch.equal(got[0], plain[0])
        for a, b in zip(got[1], plain[1]):
            assert torch.equal(a, b)
    shared = k[:, :1].expand(n, 2, dim)
    want = run(q.contiguous(), shared.contiguous(), v.contiguous(), dout, lengths, lengths, True)
    got = run(q, shared, v, dout, lengths, lengths, True)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [48, 128])
def test_what_nobody_sees_changes_nothing(cuda_device, value, dim):
    """Rows behind the last sequence, and other sequences' rows, may hold anything."""
    lengths = [60, 129, 5]
    n = sum(lengths)
    q, k, v, dout = make(lengths, lengths, 4, 2, dim, BF16, cuda_device, extra=70)
    clean, clean_grads = run(q[:n], k[:n], v[:n], dout[:n], lengths, lengths, True)
    for t in (q, k, v, dout):
        t[n:] = value
    out, grads = run(q, k, v, dout, lengths, lengths, True)
    assert torch.equal(out[:n], clean) and not out[n:].any()
    for a, b in zip(grads, clean_grads):
        assert torch.equal(a[:n], b) and not a[n:].any()
    # the middle sequence poisoned: its neighbours keep their bits
    for t in (q, k, v, dout):
        t[60:189] = value
    out, grads = run(q, k, v, dout, lengths, lengths, True)
    for at in (slice(0, 60), slice(189, n)):
        assert torch.equal(out[at], clean[at])
        assert all(torch.equal(a[at], b[at]) for a, b in zip(grads, clean_grads))


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("at", [0, 100, 127, 128, 290])
@pytest.mark.parametrize("dim", [64, 128])
def test_what_comes_later_is_not_seen(cuda_device, which, value, at, dim):
    """Causal: a key or value that is not finite reaches the queries from its own on, and none before: bit for bit, but in the value's own
    column of the queries whose tile of keys it lies in, which is made another way."""
    n = 300
    q, k, v, dout = make([n], [n], 2, 1, dim, BF16, cuda_device)
    clean, _ = run(q, k, v, dout, [n], [n], True)
    want, tol, _, _ = reference(q, k, v, [n], [n], True, dim ** -0.5)
    (k if which == "k" else v)[at, 0, 3] = value
    out, _ = run(q, k, v, dout, [n], [n], True)
    keep = torch.arange(dim, device=cuda_device) != 3
    assert torch.equal(out[:at][..., keep], clean[:at][..., keep])
    check(out[:at], want[:at], tol[:at], "out")
    if which == "v":
        filled = torch.full_like(out[at:, :, 3], value)
        assert torch.equal(out[at:, :, 3].isnan(), filled.isnan())
        assert math.isnan(value) or torch.equal(out[at:, :, 3], filled)
        assert torch.equal(out[at:][..., keep], clean[at:][..., keep])
    else:
        assert torch.equal(out[:at], clean[:at])
        assert not math.isnan(value) or out[at:].isnan().all()


@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("at", [0, 100, 255])
@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 64), (2, 2, 128)])
def test_gradients_of_queries_before_a_nan(cuda_device, which, at, heads, kv, dim):
    n = 300
    tensors = dict(zip(("q", "k", "v", "dout"), make([n], [n], heads, kv, dim, BF16, cuda_device)))
    _, clean = run(*tensors.values(), [n], [n], True)
    _, _, want, tol = reference(tensors["q"], tensors["k"], tensors["v"], [n], [n], True, dim ** -0.5, tensors["dout"])
    tensors[which][at] = math.nan
    _, grads = run(*tensors.values(), [n], [n], True)
    tile = at // 128 * 128
    assert torch.equal(grads[0][:tile], clean[0][:tile])
    check(grads[0][:at], want[0][:at], tol[0][:at], "dq")
    # keys after a query's own see nothing of it; those up to it get NaN
    if which in ("q", "dout"):
        for i in (1, 2):
            assert torch.equal(grads[i][tile + 128:], clean[i][tile + 128:])
            check(grads[i][at + 1:], want[i][at + 1:], tol[i][at + 1:], "dk, dv")
            assert grads[i][:at + 1].isnan().any(-1).all()


def test_all_nan(cuda_device):
    """Nothing but NaN: quick, and NaN."""
    n = 3000
    q, k, v, dout = (torch.full_like(t, math.nan) for t in make([n], [n], 4, 2, 64, BF16, cuda_device))
    out, grads = run(q, k, v, dout, [n], [n], True)
    assert out.isnan().all() and all(g.isnan().all() for g in grads)


def test_gradients_against_differences(cuda_device):
    """Central differences of the 64-bit definition along random directions."""
    q_len, k_len = [37, 60], [50, 55]
    q, k, v, dout = make(q_len, k_len, 4, 2, 32, BF16, cuda_device, seed=5)
    _, grads = run(q, k, v, dout, q_len, k_len, True)
    value = lambda a, b, c: (reference(a, b, c, q_len, k_len, True, 32 ** -0.5)[0] * dout.double()).sum()  # noqa: E731
    x = [t.double() for t in (q, k, v)]
    _, _, _, tols = reference(q, k, v, q_len, k_len, True, 32 ** -0.5, dout)
    for i in range(3):
        d = torch.randn(x[i].shape, device=cuda_device, dtype=torch.float64)
        step = 1e-4
        # `reference` takes its inputs' dtype for tolerances only: 64-bit inputs give the definition itself
        up, down = ([t + sign * step * d if j == i else t for j, t in enumerate(x)] for sign in (1, -1))
        slope = (value(*up) - value(*down)) / (2 * step)
        # each element is off by at most its tolerance; differences themselves by step^2 times third derivatives
        assert abs((grads[i].double() * d).sum() - slope) <= (tols[i] * d.abs()).sum() + 1e-4 * d.numel() ** 0.5


def test_repeatable_and_on_other_streams(cuda_device):
    lengths = [400, 90, 0, 333]
    q, k, v, dout = make(lengths, lengths, 8, 2, 128, BF16, cuda_device)
    first = run(q, k, v, dout, lengths, lengths, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(q, k, v, dout, lengths, lengths, True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], second[0]) and all(torch.equal(a, b) for a, b in zip(first[1], second[1]))


def test_captured_step_follows_its_inputs(cuda_device):
    """A training step in a graph, replayed for other values and other lengths in the same buffers."""
    from pack3d_b200 import sequence_attention
    lengths = [100, 30, 70]
    q, k, v, dout = make(lengths, lengths, 4, 2, 64, BF16, cuda_device)
    offsets = offsets_of(lengths, cuda_device)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(sequence_attention(*leaves, offsets), leaves, dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sequence_attention(*leaves, offsets)
        grads = torch.autograd.grad(out, leaves, dout)
    for seed, other in ((1, [100, 30, 70]), (2, [3, 190, 5]), (3, [0, 200, 0])):
        fresh = make(other, other, 4, 2, 64, BF16, cuda_device, seed=seed, extra=200 - sum(other))
        with torch.no_grad():
            for leaf, t in zip(leaves, fresh):
                leaf.copy_(t)
            dout.copy_(fresh[3])
            offsets.copy_(offsets_of(other, cuda_device))
        graph.replay()
        want = run(*fresh, other, other, True)
        assert torch.equal(out, want[0]) and all(torch.equal(a, b) for a, b in zip(grads, want[1]))


def test_offsets_are_cut_to_the_rows(cuda_device):
    """Offsets past the rows or decreasing reach no memory outside the tensors."""
    from pack3d_b200 import sequence_attention
    q, k, v, dout = make([50], [50], 2, 1, 32, BF16, cuda_device)
    want = run(q, k, v, dout, [50], [50], True)
    for bad in ([0, 1 << 30], [7, 60], [-5, 50]):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = sequence_attention(*leaves, torch.tensor(bad, dtype=torch.int32, device=cuda_device))
        assert torch.equal(out, want[0])
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, dout), want[1]))
    for bad in ([0, 40, 10], [0, -3, 1 << 30, 5], [0, 50, 0, 50]):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = sequence_attention(*leaves, torch.tensor(bad, dtype=torch.int32, device=cuda_device))
        torch.autograd.grad(out, leaves, dout)
    torch.cuda.synchronize()


def test_many_sequences(cuda_device):
    q_len = [i % 5 for i in range(700)]
    q, k, v, dout = make(q_len, q_len, 2, 2, 16, F16, cuda_device)
    out, grads = run(q, k, v, dout, q_len, q_len, True)
    want, tol, want_grads, grad_tols = reference(q, k, v, q_len, q_len, True, 0.25, dout)
    check(out, want, tol, "out")
    for g, w, t in zip(grads, want_grads, grad_tols):
        check(g, w, t, "gradients")


@pytest.mark.parametrize("count", [31, 32, 126, 127, 128])
@pytest.mark.parametrize("heads,kv", [(2, 1), (3, 3)])
@pytest.mark.parametrize("causal", [True, False])
def test_order_of_tiles(cuda_device, count, heads, kv, causal):
    """Sequences of none to three tiles, more keys or more queries, on both sides of the count up to which tiles are sorted, and rows
    behind them all."""
    q_len = [(37 * i) % 301 if i % 4 else 0 for i in range(count)]
    k_len = [max(0, n + (53 * i) % 200 - 60) for i, n in enumerate(q_len)]
    q, k, v, dout = make(q_len, k_len, heads, kv, 16, BF16, cuda_device, extra=200)
    out, grads = run(q, k, v, dout, q_len, k_len, causal)
    want, tol, want_grads, grad_tols = reference(q, k, v, q_len, k_len, causal, 0.25, dout)
    check(out, want, tol, "out")
    for g, w, t in zip(grads, want_grads, grad_tols):
        check(g, w, t, "gradients")
    assert not out[sum(q_len):].any() and not grads[0][sum(q_len):].any()
    assert not grads[1][sum(k_len):].any() and not grads[2][sum(k_len):].any()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 64), (5, 1, 128), (3, 3, 48)])
def test_single_keys_have_no_score_gradient(cuda_device, dtype, heads, kv, dim):
    """Where a query sees one key its weight is 1 whatever the score: its gradient is 0 exactly, and a key's of a sequence of one."""
    for q_len, k_len, causal in (([1, 0, 1, 1], None, True), ([4, 300, 1], [1, 1, 1], False), ([4, 300, 1], [1, 1, 1], True),
                                 ([1, 2], [1, 2], True)):
        k_len = q_len if k_len is None else k_len
        q, k, v, dout = make(q_len, k_len, heads, kv, dim, dtype, cuda_device)
        out, (dq, dk, dv) = run(q, k, v, dout, q_len, k_len, causal)
        want, tol, want_grads, grad_tols = reference(q, k, v, q_len, k_len, causal, dim ** -0.5, dout)
        check(out, want, tol, "out")
        check(dv, want_grads[2], grad_tols[2], "dv")
        if k_len[-1] == 1:
            assert not dq.any() and not dk.any()
        else:   # the second sequence's first query sees one key, its second two
            assert not dq[:2].any() and not dk[:1].any() and dq[2].any()


def test_some_gradients_only(cuda_device):
    from pack3d_b200 import sequence_attention
    lengths = [200, 40]
    q, k, v, dout = make(lengths, lengths, 2, 1, 64, BF16, cuda_device)
    _, want = run(q, k, v, dout, lengths, lengths, True)
    for chosen in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.clone().requires_grad_(i in chosen) for i, t in enumerate((q, k, v))]
        out = sequence_attention(*leaves, offsets_of(lengths, cuda_device))
        for i, g in zip(chosen, torch.autograd.grad(out, [leaves[i] for i in chosen], dout)):
            assert torch.equal(g, want[i])


def test_attention_refuses_what_it_cannot_do(cuda_device):
    import torch.autograd.forward_ad as forward_ad
    from pack3d_b200 import sequence_attention
    q, k, v, dout = make([20], [20], 4, 2, 64, BF16, cuda_device)
    o = offsets_of([20], cuda_device)
    for bad, text in (((q.float(), k.float(), v.float(), o), "fp16 or bf16"), ((q, k.half(), v, o), "same dtype"),
                      ((q[:, :3], k, v, o), "divisible"), ((q[..., :60], k[..., :60], v[..., :60], o), "multiple of 8"),
                      ((q, k, v[:10], o), r"\[rows"), ((q, k, v, o.long()), "int32"), ((q, k, v, o[None]), "int32"),
                      ((q, k, v, o.cpu()), "int32"), ((q, k, v, o[:1]), "at least one"), ((q, k[:10], v[:10], o), "k_offsets"),
                      ((q, k, v, o, offsets_of([10, 10], cuda_device)), "as many"), ((q[0], k, v, o), r"\[rows"),
                      ((q.cpu(), k, v, o), "CUDA"), ((q, k.cpu(), v, o), "device")):
        with pytest.raises(ValueError, match=text):
            sequence_attention(*bad)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            sequence_attention(q, k, v, o, scale=scale)
    with pytest.raises(ValueError, match="causal"):
        sequence_attention(q, k, v, o, causal=1)
    leaf = q.clone().requires_grad_()
    g, = torch.autograd.grad(sequence_attention(leaf, k, v, o), leaf, dout.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        sequence_attention(forward_ad.make_dual(q, q), k, v, o)


def test_no_rows(cuda_device):
    from pack3d_b200 import sequence_attention
    q = torch.zeros(0, 4, 64, device=cuda_device, dtype=BF16).requires_grad_()
    k = torch.randn(9, 2, 64, device=cuda_device, dtype=BF16).requires_grad_()
    out = sequence_attention(q, k, k, offsets_of([0], cuda_device), offsets_of([9], cuda_device))
    assert out.shape == (0, 4, 64)
    dq, dk = torch.autograd.grad(out, (q, k), torch.zeros_like(out))
    assert dq.shape == q.shape and not dk.any()


# ------------------------------------------------------------------------------- norms with rotation
def rotated(x, positions, pairs, base=10000.0):
    """x [.., tokens, heads, dim] in 64 bits."""
    positions = positions.double() if positions.ndim == 2 else positions.double()[:, None]
    angle = torch.cat([positions[:, a:a + 1] * base ** (-torch.arange(n, device=x.device).double() / max(n, 1))
                       for a, n in enumerate(pairs)], -1)[:, None]
    y, n = x.clone(), 2 * sum(pairs)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    y[..., 0:n:2], y[..., 1:n:2] = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    return y


def normed(x, spec):
    if spec is None:
        return x
    if spec.kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + spec.eps)
    if spec.weight is not None:
        y = y * spec.weight.double()
    return y if spec.bias is None else y + spec.bias.double()


def norm_rotate_case(cuda_device, dim, dtype, tokens=33, heads=3, kv=2, kind="rms", bias=False, param=None, axes=1, batch=(),
                     far=100000, pairs=None, weight=True):
    from pack3d_b200 import NormSpec, norm_rotate
    gen = torch.Generator(device=cuda_device).manual_seed(dim)
    rand = lambda *s: torch.randn(*s, generator=gen, device=cuda_device)  # noqa: E731
    param = param or dtype
    x = [(rand(*batch, tokens, n, dim) * 2 + 0.5).to(dtype).requires_grad_() for n in (heads, kv)]
    params = [[(1 + 0.2 * rand(dim)).to(param).requires_grad_() if weight else None,
               rand(dim).to(param).requires_grad_() if bias else None] for _ in range(2)]
    specs = [NormSpec(*p, kind, 1e-5) if kind else None for p in params]
    positions = torch.randint(-far, far + 1, (tokens,) if axes == 1 else (tokens, axes), generator=gen, device=cuda_device)
    up = [rand(*batch, tokens, n, dim).to(dtype) for n in (heads, kv)]
    got = norm_rotate(*x, positions, q_norm=specs[0], k_norm=specs[1], pairs=pairs)
    leaves = x + [p for ps in params for p in ps if p is not None and kind]
    grads = torch.autograd.grad(got, leaves, up)
    if pairs is None:
        share, extra = divmod(dim // 2, axes)
        pairs = tuple(share + (a < extra) for a in range(axes))
    wide = [t.detach().double().requires_grad_() for t in leaves]
    it = iter(wide[2:])
    ref_specs = [None if s is None else NormSpec(next(it) if s.weight is not None else None, next(it) if s.bias is not None else None,
                                                 s.kind, s.eps) for s in specs]
    want = [rotated(normed(t, s), positions, pairs) for t, s in zip(wide[:2], ref_specs)]
    want_grads = torch.autograd.grad(want, wide, [t.double() for t in up])
    u = half_step(dtype)
    for g, w in zip(got, want):
        assert g.dtype == dtype and g.is_contiguous()
        # one rounding; sine and cosine to 2^-21, statistics and products in fp32: 2^-19 of a pair's size
        size = w.abs().amax(-1, keepdim=True)
        assert ((g.double() - w).abs() <= u * w.abs() + 2.0 ** -19 * size + 2.0 ** -25).all()
    for leaf, g, w in zip(leaves, grads, want_grads):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        if leaf.ndim == 1:
            # a sum of rows' products: each in fp32 with sine and cosine to 2^-21, of magnitudes whose sum is at most this
            rows = sum(t.numel() // dim for t in x)
            slack = 2.0 ** -18 * rows * 6 * 4
            assert ((g.double() - w).abs() <= half_step(leaf.dtype) * w.abs() + slack).all()
        else:
            size = w.abs().amax(-1, keepdim=True) + 1
            assert ((g.double() - w).abs() <= u * w.abs() + 2.0 ** -17 * size).all()


@pytest.mark.parametrize("dim", [2, 4, 8, 10, 16, 32, 48, 64, 80, 96, 128, 130, 200, 256])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_rotate(cuda_device, dim, dtype):
    norm_rotate_case(cuda_device, dim, dtype)


@pytest.mark.parametrize("kind,bias,weight", [("layer", True, True), ("layer", False, True), ("rms", True, True), ("rms", False, False),
                                              ("layer", True, False), (None, False, True)])
@pytest.mark.parametrize("dtype,param", [(BF16, F32), (F32, F32), (F16, F16)])
def test_norm_rotate_kinds(cuda_device, kind, bias, weight, dtype, param):
    norm_rotate_case(cuda_device, 48, dtype, kind=kind, bias=bias, param=param, weight=weight)


@pytest.mark.parametrize("axes,pairs", [(3, None), (2, None), (3, (4, 0, 9)), (1, (5,)), (1, (0,)), (2, (16, 16)), (3, (24, 0, 0))])
def test_norm_rotate_axes(cuda_device, axes, pairs):
    norm_rotate_case(cuda_device, 64, F32, axes=axes, pairs=pairs)


@pytest.mark.parametrize("tokens,heads,kv,batch", [(1, 1, 1, ()), (1, 16, 4, ()), (1000, 32, 8, ()), (5, 1, 7, (3,)), (64, 4, 4, (2, 2)),
                                                   (4097, 3, 1, ())])
def test_norm_rotate_shapes(cuda_device, tokens, heads, kv, batch):
    norm_rotate_case(cuda_device, 64, BF16, tokens=tokens, heads=heads, kv=kv, batch=batch)


def test_norm_rotate_positions_are_exact(cuda_device):
    """At positions of 2^50 an angle in fp32 or even fp64 says nothing: against whole-number arithmetic."""
    from fractions import Fraction
    from pack3d_b200 import norm_rotate
    dim, base = 16, 10000.0
    for at in (2 ** 50 + 12345, -(2 ** 50) - 77):
        q = torch.zeros(1, 1, dim, device=cuda_device)
        q[..., 0::2] = 1
        y, none = norm_rotate(q, None, torch.tensor([at], device=cuda_device), base=base)
        assert none is None
        for i in range(dim // 2):
            # the frequency as the definition has it in fp64, in turns to 2^-64
            turns = round(Fraction(base ** (-i / (dim // 2))) / Fraction(6283185307179586476925286766559005768394, 10 ** 39) * 2 ** 64)
            angle = float(Fraction(at * turns % 2 ** 64, 2 ** 64)) * 2 * math.pi
            # a frequency's last bit of 2^-64 turns is 2^-14 turns here: 4e-4 radians, and as much for the division's rounding
            assert abs(y[0, 0, 2 * i].item() - math.cos(angle)) < 1e-3 and abs(y[0, 0, 2 * i + 1].item() - math.sin(angle)) < 1e-3


def test_norm_rotate_views(cuda_device):
    from pack3d_b200 import NormSpec, norm_rotate
    row = torch.randn(50, 6 * 64 + 1, device=cuda_device).to(BF16)
    positions = torch.arange(100, device=cuda_device, dtype=torch.int32)[::2]
    spec = NormSpec(torch.rand(64, device=cuda_device))
    for at in (0, 1):   # aligned (never, with an odd row) and not
        q, k = row[:, at:at + 4 * 64].unflatten(-1, (4, 64)), row[:, at + 256:at + 384].unflatten(-1, (2, 64))
        got = norm_rotate(q, k, positions, q_norm=spec, k_norm=spec)
        want = norm_rotate(q.contiguous(), k.contiguous(), positions.long().contiguous(), q_norm=spec, k_norm=spec)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = torch.randn(4, 50, 64, device=cuda_device).to(BF16).transpose(0, 1)
    assert torch.equal(norm_rotate(q, None, positions)[0], norm_rotate(q.contiguous(), None, positions)[0])


def test_norm_rotate_some_gradients(cuda_device):
    from pack3d_b200 import NormSpec, norm_rotate
    q, k = (torch.randn(9, n, 32, device=cuda_device) for n in (4, 2))
    w = torch.rand(32, device=cuda_device)
    positions = torch.arange(9, device=cuda_device)

    def grads(*wanted, outputs=2):
        t = [x.clone().requires_grad_(i in wanted) for i, x in enumerate((q, k, w))]
        y = norm_rotate(t[0], t[1], positions, q_norm=NormSpec(t[2]), k_norm=NormSpec(t[2]))
        return torch.autograd.grad([x.square().sum() for x in y[:outputs]], [t[i] for i in wanted])
    every = grads(0, 1, 2)
    for wanted in ((0,), (1,), (2,), (0, 2)):
        for i, g in zip(wanted, grads(*wanted)):
            assert torch.equal(g, every[i])
    dq, dk = torch.autograd.grad(norm_rotate(*(leaves := [q.clone().requires_grad_(), k.clone().requires_grad_()]), positions)[0].sum(),
                                 leaves, allow_unused=True)
    assert dk is None or not dk.any()
    assert dq.abs().sum() > 0


def test_norm_rotate_no_tokens(cuda_device):
    from pack3d_b200 import NormSpec, norm_rotate
    w = torch.ones(16, device=cuda_device, requires_grad=True)
    q = torch.zeros(0, 2, 16, device=cuda_device, requires_grad=True)
    y, _ = norm_rotate(q, None, torch.zeros(0, dtype=torch.long, device=cuda_device), q_norm=NormSpec(w))
    dq, dw = torch.autograd.grad(y.sum(), (q, w))
    assert y.shape == q.shape and not dw.any()


def test_norm_rotate_refusals(cuda_device):
    from pack3d_b200 import NormSpec, norm_rotate
    q, k, p = torch.randn(9, 4, 32, device=cuda_device), torch.randn(9, 2, 32, device=cuda_device), torch.arange(9, device=cuda_device)
    for args, more, text in (((q[..., :31], None, p), {}, "even"), ((q, k[:8], p), {}, "shape of q"), ((q, k.half(), p), {}, "dtype"),
                             ((q, k, p[:8]), {}, "positions"), ((q, k, p.float()), {}, "positions"), ((q, k, p.cpu()), {}, "positions"),
                             ((q, k, p), {"pairs": (17,)}, "pairs"), ((q, k, p), {"pairs": (4, 4)}, "pairs"), ((q, k, p), {"pairs": (-1,)}, "pairs"),
                             ((q, k, p), {"base": 0.5}, "base"), ((q, k, p), {"base": math.nan}, "base"),
                             ((q, k, p), {"q_norm": NormSpec(torch.ones(16, device=cuda_device))}, r"\[32\]"),
                             ((q, k, p), {"k_norm": 3}, "NormSpec"), ((q, None, p), {"k_norm": NormSpec()}, "without k"),
                             ((q.cpu(), None, p), {}, "CUDA"), ((q[0], None, p), {}, "shape")):
        with pytest.raises(ValueError, match=text):
            norm_rotate(*args, **more)


def test_capture_behind_a_living_graph(cuda_device):
    """While a graph from the default stream holds a leaf, a captured step over it is refused; without it the step is captured,
    and its replay follows its inputs."""
    from pack3d_b200 import NormSpec, norm_rotate, sequence_attention
    torch.manual_seed(12)
    x = torch.randn(40, 2, 64, device=cuda_device, dtype=BF16, requires_grad=True)
    w = torch.randn(64, device=cuda_device, requires_grad=True)
    at = torch.arange(40, device=cuda_device)
    offsets = torch.tensor([0, 11, 40], dtype=torch.int32, device=cuda_device)

    def step(x, w):
        q, k = norm_rotate(x, x, at, q_norm=NormSpec(w, None, "rms", 1e-6))
        y = sequence_attention(q, k, x, offsets)
        return y, torch.autograd.grad(y.float().square().sum(), (x, w))

    alive = step(x, w)[0]
    for call in (lambda: norm_rotate(x, None, at), lambda: norm_rotate(x.detach(), None, at, q_norm=NormSpec(w, None, "rms", 1e-6)),
                 lambda: sequence_attention(x.detach(), x.detach(), x, offsets)):
        with pytest.raises(ValueError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    del alive
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step(x, w)                        # lives on, from another stream than the default one
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = step(x, w)
    with torch.no_grad():
        x.mul_(-0.5).add_(0.25)
    graph.replay()
    want, ref = step(x.detach().requires_grad_(), w.detach().requires_grad_())
    assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(grads, ref))
    assert not torch.equal(other[0], want)
