"""The feed-forward block: the operators in one module, behind the attention layer, in training and serving."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def by_hand(m, x, gate, p, rng):
    from pack3d_b200 import dropout, fp8_linear, norm
    y = norm(x, m.pre_norm)
    h = fp8_linear(torch.nn.functional.gelu(fp8_linear(y, m.w1, m.b1)), m.w2, m.b2)
    u = norm(h, m.post_norm).float()
    if gate is not None:
        u = u * torch.sigmoid(gate.float())
    if p:
        u = dropout(u, p, rng)
    return x.float() + m.scale.float() * u


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gated", [False, True])
def test_block_is_its_operators(cuda_device, kind, dtype, gated):
    from pack3d_b200 import FeedForward
    torch.manual_seed(3)
    m = FeedForward(72, 200, norm=kind, dropout=0.2, gate_activation="sigmoid").to(cuda_device, dtype)
    x = torch.randn(2, 33, 72, device=cuda_device).to(dtype).requires_grad_()
    gate = torch.randn(2, 1, 72, device=cuda_device).to(dtype).requires_grad_() if gated else None
    out, y = m(x, gate=gate, rng=(5, 6))
    want = by_hand(m, x, gate, 0.2, (5, 6))
    assert y is None and out.dtype == dtype
    # the norm of h is rounded to 16 bits by hand and not inside the kernel, and both round out once: 2^-8 (bf16) or 2^-11
    # each of values up to |x| + scale * |u| / (1 - p), u at most eight
    ulp = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    assert ((out.float() - want).abs() <= ulp * (want.abs() + 0.1 * 8 / 0.8) + 2.0 ** -12).all()
    leaves = [x, *m.parameters()] + ([gate] if gated else [])
    got = torch.autograd.grad(out.float().square().sum(), leaves)
    ref = torch.autograd.grad(want.square().sum(), leaves)
    for g, r in zip(got, ref):
        assert g.shape == r.shape and torch.isfinite(g).all()
        # the two differ by roundings to 16 bits, and where one crosses a step of e4m3, by 2^-4 of an element:
        # a few percent of the whole in the 2-norm
        assert (g.float() - r.float()).norm() <= 0.05 * r.float().norm() + 1e-3


def test_stack_hands_the_norm_on(cuda_device):
    from pack3d_b200 import FeedForward
    torch.manual_seed(4)
    layers = [FeedForward(64, 128).to(cuda_device) for _ in range(3)]
    x = torch.randn(17, 64, device=cuda_device)
    a, y = x, None
    for i, layer in enumerate(layers):
        a, y = layer(a, normed=y, next_norm=layers[i + 1].pre_norm if i < 2 else None)
    b = x
    for layer in layers:
        b, _ = layer(b)
    assert y is None
    # in fp32 the handed-on norm is the norm of the same values: only the order of its sums can differ
    assert (a - b).abs().max() <= 1e-4 * b.abs().max()


def test_serving_from_kept_weights(cuda_device):
    from pack3d_b200 import FeedForward
    torch.manual_seed(5)
    m = FeedForward(192, 768).to(cuda_device, torch.bfloat16).eval()
    for tokens in (1, 7, 300):
        x = torch.randn(tokens, 192, device=cuda_device, dtype=torch.bfloat16)
        with torch.no_grad():
            want, want_y = m(x, next_norm=m.pre_norm)
            m.keep_8bit()
            got, got_y = m(x, next_norm=m.pre_norm)
            m.keep_8bit(False)
        assert torch.equal(got, want) and torch.equal(got_y, want_y)


def test_training_behind_the_attention_layer(cuda_device):
    """A few steps of attention and feed-forward together bring a small regression's loss down, and with the same seeds
    the run repeats bit for bit."""
    from pack3d_b200 import FeedForward, PACK3DAttention, build_layout

    def run():
        torch.manual_seed(0)
        layout = build_layout((8, 8, 8), (4, 4, 4), radius=2, pool_size=1).to(cuda_device)
        attention = PACK3DAttention(96, heads=2, kv_heads=2, head_dim=48, block_volume=64).to(cuda_device, torch.bfloat16)
        block = FeedForward(96, 256, dropout=0.1, residual_scale=0.5).to(cuda_device, torch.bfloat16)
        x = torch.randn(1, 512, 96, device=cuda_device, dtype=torch.bfloat16)
        goal = torch.randn(1, 512, 96, device=cuda_device, dtype=torch.bfloat16)
        params = [*attention.parameters(), *block.parameters()]
        losses = []
        for step in range(12):
            out, _ = block(attention(x, layout), rng=(9, step))
            loss = (out.float() - goal.float()).square().mean()
            grads = torch.autograd.grad(loss, params)
            with torch.no_grad():
                for p, g in zip(params, grads):
                    p.sub_((g.float() * 2.0).to(p.dtype))
            losses.append(loss.item())
        return losses

    losses = run()
    assert losses[-1] < 0.97 * losses[0], losses
    assert run() == losses


def test_refusals(cuda_device):
    from pack3d_b200 import FeedForward
    for kwargs in ({"norm": "batch"}, {"dropout": 1.0}, {"dropout": -0.1}, {"residual_scale": float("inf")}):
        with pytest.raises(ValueError):
            FeedForward(32, 64, **kwargs)
    with pytest.raises(ValueError, match="positive"):
        FeedForward(0, 64)
    m = FeedForward(32, 64, dropout=0.1).to(cuda_device)
    x = torch.randn(3, 32, device=cuda_device)
    with pytest.raises(ValueError, match="rng"):
        m(x)
    m.keep_8bit()
    with pytest.raises(ValueError, match="no_grad"):
        m(x)


def test_kept_weights_follow_the_parameters(cuda_device):
    """Served after the weights have changed, by whatever way PyTorch counts, the block answers as with 8-bit weights
    kept anew; untouched, it quantises nothing."""
    import copy
    from pack3d_b200 import FeedForward

    def block(seed):
        torch.manual_seed(seed)
        return FeedForward(64, 160).to(cuda_device, torch.bfloat16).eval()

    x = torch.randn(9, 64, device=cuda_device, dtype=torch.bfloat16)
    m, other = block(1).keep_8bit(), block(2)
    with torch.no_grad():
        first = m(x)[0]
        assert torch.equal(first, block(1)(x)[0])
        values = m._kept[0].values
        assert torch.equal(m(x)[0], first) and m._kept[0].values is values

        def same():
            want = copy.deepcopy(m).keep_8bit(False)(x)[0]
            got = m(x)[0]
            return torch.equal(got, want) and not torch.equal(got, first)

        m.load_state_dict(other.state_dict())
        assert same() and m._kept[0].values.data_ptr() == values.data_ptr()
        m.w1.mul_(-0.5)
        assert same()
        m.w2.copy_(block(3).w2)
        assert same()
        torch._foreach_add_([m.w1, m.w2], 0.01)
        assert same()
        m.load_state_dict(block(4).state_dict(), assign=True)
        assert same()
        m.w1 = torch.nn.Parameter(block(5).w1.detach().clone())
        assert same()
        m.half().to(torch.bfloat16)
        assert same()
        m.float()
        x = x.float()
        assert same()
        assert torch.equal(copy.deepcopy(m)(x)[0], m(x)[0])
        served = m(x)[0]
        m.w1 = None                                   # the full weight is given up: served as before
        m.w2.data = torch.empty(0, device=cuda_device)
        assert torch.equal(m(x)[0], served)


def test_graph_over_kept_weights(cuda_device):
    """A captured forward reads the kept weights' memory: after a change and one forward its replay is the new answer;
    capturing over weights that have changed is refused."""
    from pack3d_b200 import FeedForward
    torch.manual_seed(6)
    m = FeedForward(64, 160).to(cuda_device, torch.bfloat16).eval().keep_8bit()
    x = torch.randn(3, 64, device=cuda_device, dtype=torch.bfloat16)
    stream = torch.cuda.Stream()
    with torch.no_grad():
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            m(x)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)[0]
        m.w1.mul_(-0.5)
        want = m(x)[0]
        graph.replay()
        assert torch.equal(out, want)
        m.w1.mul_(-0.5)
        with pytest.raises(ValueError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                m(x)
