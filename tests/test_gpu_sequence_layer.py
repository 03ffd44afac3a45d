"""Attention over sequences as a layer: the operators together, in training and over a cache."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def offsets_of(lengths, device):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=device)


def positions_of(lengths, device, starts=None):
    return torch.cat([torch.arange(s, s + n) for n, s in zip(lengths, starts or [0] * len(lengths))]).to(device)


def by_hand(m, x, positions, lengths, gradients=True):
    """The layer in fp32, its heads rotated as complex numbers."""
    x, at = x.float(), 0
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + m.eps) * m.pre_weight.float()
    row = y @ m.to_qkv.weight.float().t()
    h, g, d = m.heads, m.kv_heads, m.head_dim
    q, k, v = (t.unflatten(-1, (-1, d)) for t in row.split((h * d, g * d, g * d), -1))
    angle = positions[:, None].double() * m.base ** (-torch.arange(d // 2, device=x.device).double() / (d // 2))
    turn = torch.polar(torch.ones_like(angle), angle).to(torch.complex64)[:, None]
    q, k = (torch.view_as_real(torch.view_as_complex((t * torch.rsqrt(t.square().mean(-1, keepdim=True) + m.eps) * w.float())
                                                     .unflatten(-1, (-1, 2)).contiguous()) * turn).flatten(-2)
            for t, w in ((q, m.q_weight), (k, m.k_weight)))
    out = []
    for n in lengths:
        s = slice(at, at + n)
        at += n
        kk, vv = (t[s].repeat_interleave(h // g, 1) for t in (k, v))
        score = torch.einsum("ihd,jhd->hij", q[s], kk) * d ** -0.5
        score = score.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), float("-inf"))
        out.append(torch.einsum("hij,jhd->ihd", score.softmax(-1), vv))
    return x + torch.cat(out).flatten(-2) @ m.to_out.weight.float().t()


def layer(device, dtype, head_dim=64, heads=8, kv_heads=2, dim=256, seed=0):
    from pack3d_b200 import SequenceAttention
    torch.manual_seed(seed)
    return SequenceAttention(dim, heads=heads, kv_heads=kv_heads, head_dim=head_dim).to(device, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("head_dim,heads,kv_heads", [(64, 8, 2), (128, 2, 2), (48, 3, 1)])
def test_layer_is_its_definition(cuda_device, dtype, head_dim, heads, kv_heads):
    m = layer(cuda_device, dtype, head_dim, heads, kv_heads)
    lengths = [70, 1, 0, 200]
    x = torch.randn(sum(lengths), m.dim, device=cuda_device).to(dtype).requires_grad_()
    positions = positions_of(lengths, cuda_device)
    out, y = m(x, positions, offsets_of(lengths, cuda_device), next_norm=m.pre_norm)
    want = by_hand(m, x, positions, lengths)
    u = torch.finfo(dtype).eps / 2
    # six roundings on the way (norm, projection, heads' norm, weights, attention, output) and the result's: each of u on values whose
    # sums through the next matrix keep their relative size in the 2-norm
    assert (out.float() - want).norm() <= 8 * u * want.norm()
    assert y.shape == out.shape
    leaves = [x, *m.parameters()]
    up = torch.randn_like(want)
    got = torch.autograd.grad((out.float() * up).sum(), leaves)
    ref = torch.autograd.grad((want * up).sum(), leaves)
    for g, r in zip(got, ref):
        # as many roundings again on the way back, and sums of unlike signs that lose up to a few times that
        assert g.shape == r.shape and (g.float() - r.float()).norm() <= 40 * u * r.float().norm() + 1e-6


def test_stack_hands_the_norm_on(cuda_device):
    from pack3d_b200 import FeedForward
    a, b = layer(cuda_device, BF16), layer(cuda_device, BF16, seed=1)
    f = FeedForward(256, 512, norm="rms").to(cuda_device, BF16)
    lengths = [33, 90]
    x = torch.randn(123, 256, device=cuda_device, dtype=BF16)
    positions, offsets = positions_of(lengths, cuda_device), offsets_of(lengths, cuda_device)
    with torch.no_grad():
        h, y = a(x, positions, offsets, next_norm=f.pre_norm)
        h, y = f(h, normed=y, next_norm=b.pre_norm)
        got, none = b(h, positions, offsets, normed=y)
        plain = b(f(a(x, positions, offsets)[0])[0], positions, offsets)[0]
    assert none is None
    # the norm handed on is of the sum before its rounding: two roundings of 2^-8 more or less
    assert (got.float() - plain.float()).norm() <= 4 * 2.0 ** -8 * plain.float().norm()


def table_of(sequences, width, device, seed=0):
    order = torch.randperm(sequences * width + 2, generator=torch.Generator().manual_seed(seed))[:sequences * width]
    return order.view(sequences, width).to(torch.int32).to(device), sequences * width + 2


@pytest.mark.parametrize("stored", [BF16, E4M3])
@pytest.mark.parametrize("page", [16, 24])
def test_serving_is_the_forward_pass(cuda_device, stored, page):
    """A prompt, a second prompt behind it and single tokens over the cache, against the forward pass of the whole."""
    m = layer(cuda_device, BF16)
    first, second, steps = [40, 7, 129], [5, 60, 1], 6
    total = [a + b + steps for a, b in zip(first, second)]
    x = [torch.randn(n, 256, device=cuda_device, dtype=BF16) for n in total]
    table, pages = table_of(3, -(-max(total) // page), cuda_device)
    cache = m.new_cache(pages, page, dtype=stored)
    lengths = torch.zeros(3, dtype=torch.int32, device=cuda_device)
    got = [[] for _ in total]

    def keep(out, parts):
        for g, t in zip(got, out.split(parts)):
            g.append(t)
    with torch.no_grad():
        whole = m(torch.cat(x), positions_of(total, cuda_device), offsets_of(total, cuda_device))[0].split(total)
        out, _ = m.prefill(torch.cat([t[:n] for t, n in zip(x, first)]), positions_of(first, cuda_device), offsets_of(first, cuda_device),
                           cache, table, lengths)
        keep(out, first)
        lengths += offsets_of(first, cuda_device).diff()
        out, _ = m.prefill(torch.cat([t[n:n + k] for t, n, k in zip(x, first, second)]), positions_of(second, cuda_device, first),
                           offsets_of(second, cuda_device), cache, table, lengths, cached_rows=sum(first) + sum(second))
        keep(out, second)
        lengths += offsets_of(second, cuda_device).diff()
        for _ in range(steps):
            at = lengths.tolist()
            out, _ = m.decode(torch.stack([t[n] for t, n in zip(x, at)]), lengths.long(), cache, table, lengths)
            keep(out, [1, 1, 1])
            lengths += 1
        v = m._qkv(torch.cat(x), positions_of(total, cuda_device), None)[2].float().abs().max()
    # 16 bits: two ways to the same sums, each with weights and results rounded to 2^-8 of at most |v|. 8 bits: keys off by 2^-4 of
    # themselves move a weight by exp of |q| |k| 2^-4 / 8, both of norm 8 on average: e^0.5 - 1 in the worst case, values 2^-4.
    off = (4 * 2.0 ** -8 if stored is BF16 else 0.65 + 2.0 ** -4 + 4 * 2.0 ** -8) * v
    bound = off * m.to_out.weight.float().abs().sum(1)
    for g, w in zip(got, whole):
        g = torch.cat(g).float()
        assert ((g - w.float()).abs() <= bound + 2.0 ** -7 * w.float().abs()).all()
        # and on the whole far nearer: errors of random sign
        assert (g - w.float()).norm() <= (0.02 if stored is BF16 else 0.1) * w.float().norm()


def test_captured_decode_steps(cuda_device):
    """Steps replayed from a graph, lengths advancing on the device, are the eager steps bit for bit."""
    m = layer(cuda_device, BF16)
    table, pages = table_of(4, 8, cuda_device)
    tokens = torch.randn(20, 4, 256, device=cuda_device, dtype=BF16)
    results = []
    for captured in (False, True):
        cache, lengths = m.new_cache(pages, 16, dtype=E4M3), torch.zeros(4, dtype=torch.int32, device=cuda_device)
        x = tokens[0].clone()

        def step():
            out, _ = m.decode(x, lengths.long(), cache, table, lengths)
            lengths.add_(1)
            return out
        outs = []
        with torch.no_grad():
            if captured:
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    step()
                torch.cuda.current_stream().wait_stream(side)
                lengths.zero_()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = step()
            for t in tokens:
                x.copy_(t)
                if captured:
                    graph.replay()
                    outs.append(out.clone())
                else:
                    outs.append(step())
        assert lengths.tolist() == [20] * 4
        results.append(torch.stack(outs))
    assert torch.equal(*results)


def test_layer_refusals(cuda_device):
    from pack3d_b200 import SequenceAttention
    for bad in ({"heads": 3, "kv_heads": 2, "head_dim": 64}, {"heads": 2, "kv_heads": 2, "head_dim": 60},
                {"heads": 2, "kv_heads": 2, "head_dim": 136}, {"heads": 0, "kv_heads": 1, "head_dim": 64}):
        with pytest.raises(ValueError):
            SequenceAttention(64, **bad)
    m = layer(cuda_device, BF16)
    offsets = offsets_of([3], cuda_device)
    with pytest.raises(ValueError, match="rows"):
        m(torch.zeros(1, 3, 256, device=cuda_device, dtype=BF16), torch.arange(3, device=cuda_device), offsets)
    with pytest.raises(ValueError, match="no gradients"):
        table, pages = table_of(1, 2, cuda_device)
        m.decode(torch.zeros(1, 256, device=cuda_device, dtype=BF16), torch.zeros(1, dtype=torch.long, device=cuda_device),
                 m.new_cache(pages, 16), table, torch.zeros(1, dtype=torch.int32, device=cuda_device))


@pytest.mark.parametrize("had,n", [([3, 0], [30, 9]), ([0, 1], [30, 9]), ([0, 0], [30, 9]), ([7, 0], [0, 9]), ([0, 5], [30, 0])])
def test_a_second_prompt_needs_the_cached_rows(cuda_device, had, n):
    """Without `cached_rows` a sequence begins with its new tokens: where one that has some had others already, the results say so."""
    m = layer(cuda_device, BF16)
    x = torch.randn(sum(n), 256, device=cuda_device, dtype=BF16)
    table, pages = table_of(2, 4, cuda_device)
    offsets, lengths = offsets_of(n, cuda_device), torch.tensor(had, dtype=torch.int32, device=cuda_device)
    cache = m.new_cache(pages, 16)
    with torch.no_grad():
        got, _ = m.prefill(x, positions_of(n, cuda_device), offsets, cache, table, lengths)
        want, _ = m(x, positions_of(n, cuda_device), offsets)
    assert got.isnan().all() if any(a and b for a, b in zip(had, n)) else torch.equal(got, want)
