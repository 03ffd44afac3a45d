"""Operators of the feed-forward half of a transformer block, in real sizes.

``norm`` and ``residual_norm`` (the norms before and after a block with its gate, dropout and
residual scale), ``dropout`` (counter-based, the mask never stored) and ``fp8_linear`` (a linear
layer in 8-bit floating point with one power-of-two scale for each block of 128).  Each is
written out in elementary torch operations in 32 bits, and, where ``own`` is set, called from
``pack3d_b200``.  ``exact`` is the same definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------- cases
def _residual(name, batch, tokens, dim, dtype, train, kind, gate, act, p, post=True, nxt=True, scale=True):
    return {"name": name, "op": "residual", "batch": batch, "tokens": tokens, "dim": dim, "dtype": dtype,
            "train": train, "kind": kind, "gate": gate, "act": act, "p": p, "post": post, "next": nxt,
            "scale": scale}


def _norm(name, tokens, dim, dtype, train, kind):
    return {"name": name, "op": "norm", "tokens": tokens, "dim": dim, "dtype": dtype, "train": train, "kind": kind}


def _dropout(name, tokens, dim, dtype, train, p):
    return {"name": name, "op": "dropout", "tokens": tokens, "dim": dim, "dtype": dtype, "train": train, "p": p}


def _linear(name, tokens, k, n, dtype, train, bias):
    return {"name": name, "op": "linear", "tokens": tokens, "k": k, "n": n, "dtype": dtype, "train": train,
            "bias": bias}


def listed():
    return [
        # one token of an autoregressive pass: the block's tail and the next block's norm
        _residual("residual_token", 1, 1, 2048, "bf16", False, "rms", "none", "identity", 0.0),
        # a training step on two 64^3 fields, each modulated by one gate vector, with dropout
        _residual("residual_field_train", 2, 262144, 192, "bf16", True, "layer", "sample", "identity", 0.1),
        # a training step at a language model's width, one gate value for each token
        _residual("residual_wide_train", 4, 2048, 4096, "bf16", True, "rms", "token", "tanh", 0.0),
        # odd rows and an odd width in 32 bits, a gate for every element
        _residual("residual_ragged_train", 3, 1337, 1001, "f32", True, "layer", "element", "sigmoid", 0.25),
        # the norm before the first block: a handful of drafted tokens, and a training step
        _norm("norm_tokens", 5, 2048, "f16", False, "rms"),
        _norm("norm_wide_train", 16384, 4096, "bf16", True, "rms"),
        # dropout of a small odd batch in inference-like fine-tuning, and of the 128^3 layer's width in training
        _dropout("dropout_small", 77, 195, "f16", False, 0.1),
        _dropout("dropout_field_train", 262144, 384, "bf16", True, 0.2),
        # one token through a kept 8-bit weight
        _linear("linear_token", 1, 2048, 8192, "bf16", False, False),
        # the 64^3 field through the first feed-forward weight
        _linear("linear_field", 262144, 192, 768, "bf16", False, True),
        # a training step on an odd number of tokens between widths that no tile divides
        _linear("linear_ragged_train", 5003, 520, 1096, "f16", True, True),
        # a training step at a language model's width
        _linear("linear_wide_train", 16384, 2048, 8192, "bf16", True, False),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm, and often odd."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    r = rng.random()
    if r < 0.35:
        v = max(lo, v // 64 * 64)
    elif r < 0.6:
        v = max(lo, v // 8 * 8)
    return v + 8 if v == 3072 else v


def draw(rng):
    op = rng.choice(["residual", "residual", "norm", "dropout", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.6
    if op == "linear":
        while True:
            tokens, k, n = _log(rng, 1, 65536), _log(rng, 32, 8192), _log(rng, 32, 8192)
            if tokens * k * n <= 2.5e11 and tokens * (k + n) <= 2.5e8:
                break
        c = _linear("", tokens, k, n, rng.choice(["bf16", "f16"]), train, rng.random() < 0.5)
    else:
        while True:
            tokens, dim = _log(rng, 1, 262144), _log(rng, 16, 16384)
            if tokens * dim <= 6e7:
                break
        if op == "norm":
            c = _norm("", tokens, dim, dtype, train, rng.choice(["rms", "layer"]))
        elif op == "dropout":
            c = _dropout("", tokens, dim, dtype, train, rng.choice([0.05, 0.1, 0.3, 0.5]))
        else:
            batch = rng.choice([1, 2, 5]) if tokens >= 5 else 1
            c = _residual("", batch, tokens // batch, dim, dtype, train, rng.choice(["rms", "layer"]),
                          rng.choice(["none", "element", "sample", "token"]),
                          rng.choice(["identity", "sigmoid", "tanh"]), rng.choice([0.0, 0.1, 0.4]),
                          rng.random() < 0.8, rng.random() < 0.8, rng.random() < 0.8)
    c.pop("name")
    return c


# ------------------------------------------------------------------------------- inputs
def _make(case, seed):
    """The inputs of a case as plain tensors."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dt)

    s = {}
    op = case["op"]
    if op == "linear":
        m, k, n = case["tokens"], case["k"], case["n"]
        # activations with a few channels far above the others, and padded tokens that are all zero
        loud = 1 + 15 * (torch.rand(k, generator=g, device="cuda") < 0.01).float()
        x = torch.randn(m, k, generator=g, device="cuda") * loud
        if m > 16:
            x[torch.rand(m, generator=g, device="cuda") < 0.02] = 0
        s["x"] = x.to(dt)
        s["w"] = normal(n, k, scale=1 / math.sqrt(k))
        s["bias"] = normal(n, scale=0.1) if case["bias"] else None
        s["dy"] = normal(m, n, scale=0.02) if case["train"] else None
        return s
    if op == "dropout":
        s["x"] = normal(case["tokens"], case["dim"])
        s["dy"] = normal(case["tokens"], case["dim"]) if case["train"] else None
        s["rng"] = (seed * 7919 + 12345, seed + (1 << 33))
        return s
    dim = case["dim"]
    shape = (case["tokens"], dim) if op == "norm" else (case["batch"], case["tokens"], dim)
    s["x"] = normal(*shape, scale=1.5, mean=0.2)
    s["next_w"] = normal(dim, scale=0.2, mean=1.0)
    s["next_b"] = normal(dim, scale=0.1) if case["kind"] == "layer" else None
    s["dy"] = normal(*shape) if case["train"] else None
    if op == "norm":
        return s
    s["h"] = normal(*shape, scale=0.7, mean=-0.1)
    s["post_w"] = normal(dim, scale=0.2, mean=1.0)
    s["post_b"] = normal(dim, scale=0.1) if case["kind"] == "layer" else None
    s["scale"] = normal(dim, scale=0.1, mean=0.5) if case["scale"] else None
    gate_shape = {"none": None, "element": shape, "sample": (shape[0], 1, dim), "token": (*shape[:2], 1)}[case["gate"]]
    s["gate"] = normal(*gate_shape) if gate_shape else None
    s["dout"] = normal(*shape) if case["train"] else None
    s["rng"] = (seed * 7919 + 12345, seed + (1 << 33))
    if not case["post"]:
        s["post_w"] = s["post_b"] = None
    if not case["next"]:
        s["next_w"] = s["next_b"] = s["dy"] = None
    return s


#: what a training step returns gradients of, in this order
LEAVES = ("x", "h", "gate", "scale", "post_w", "post_b", "next_w", "next_b")


def prepare(case, seed):
    s = _make(case, seed)
    s["case"] = case
    if case["op"] == "linear":
        if case["train"]:
            for name in ("x", "w", "bias"):
                if s[name] is not None:
                    s[name].requires_grad_()
        elif own:
            import pack3d_b200
            s["kept"] = pack3d_b200.quantize_weight(s["w"])
        else:
            # a serving program holds the weight in 8 bits, with its scales
            q, scale = _quantize(s["w"].float(), 128, 128)
            s["kept"] = (q.to(torch.float8_e4m3fn), scale)
        return s
    if case["train"]:
        for name in LEAVES:
            if s.get(name) is not None:
                s[name].requires_grad_()
    if own:
        import pack3d_b200
        if s.get("next_w") is not None:
            s["next"] = pack3d_b200.NormSpec(s["next_w"], s["next_b"], case["kind"])
        if s.get("post_w") is not None:
            s["post"] = pack3d_b200.NormSpec(s["post_w"], s["post_b"], case["kind"])
    return s


# --------------------------------------------------------------------- plain forms, 32 bits
EPS = 1e-6
LOW = 0xFFFFFFFF


def _product(a, b):
    """High and low 32 bits of a * b, a < 2^32 a number, b < 2^32 in int64."""
    low, high = a * (b & 0xFFFF), a * (b >> 16)
    return (high + (low >> 16)) >> 16, (low + ((high & 0xFFFF) << 16)) & LOW


def _keep(rows, dim, p, rng, device):
    """Whether each element of [rows, dim] is kept: 16-bit field c % 8 of Philox-4x32-10 (Salmon et al.,
    SC 2011) at counter (row * ceil(dim / 8) + c // 8, offset) under the key seed, against round(65536 p)."""
    seed, offset = rng
    blocks = -(-dim // 8)
    at = torch.arange(rows * blocks, device=device)
    c0, c1 = at & LOW, at >> 32
    c2, c3 = torch.full_like(at, offset & LOW), torch.full_like(at, (offset >> 32) & LOW)
    k0, k1 = seed & LOW, (seed >> 32) & LOW
    for _ in range(10):
        h0, l0 = _product(0xD2511F53, c0)
        h1, l1 = _product(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    fields = torch.stack([c0 & 0xFFFF, c0 >> 16, c1 & 0xFFFF, c1 >> 16, c2 & 0xFFFF, c2 >> 16, c3 & 0xFFFF, c3 >> 16], -1)
    return fields.view(rows, blocks * 8)[:, :dim] >= round(65536 * p)


def _drop(x, p, rng):
    keep = _keep(x.numel() // x.shape[-1], x.shape[-1], p, rng, x.device).view(x.shape)
    return torch.where(keep, x * (65536 / (65536 - round(65536 * p))), torch.zeros_like(x))


def _normed(z, w, b, kind):
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) * w
    return z if b is None else z + b


def _block_max(x, br, bc):
    """The largest finite magnitude of each br x bc block of x, spread over the block's elements."""
    rows, cols = x.shape
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    a = torch.nn.functional.pad(a, (0, -cols % bc, 0, -rows % br))
    m = a.view(a.shape[0] // br, br, a.shape[1] // bc, bc).amax((1, 3))
    return m


def _spread(s, br, bc, rows, cols):
    return s.repeat_interleave(br, 0)[:rows].repeat_interleave(bc, 1)[:, :cols]


def _quantize(x, br, bc):
    """e4m3 values of x (in 32 bits, as the numbers 8 bits hold) and the power-of-two scale of each block."""
    m = _block_max(x, br, bc)
    frac, e = torch.frexp(m)                       # m = frac * 2^e, frac in [0.5, 1)
    e = e - 9 + (frac > 0.875).to(e.dtype)         # 448 = 0.875 * 2^9
    e = torch.where(m > 0, e.clamp_min(-126), torch.zeros_like(e))
    scale = ((e + 127) << 23).view(torch.float32)  # 2^e from its bits
    v = x * _spread(((127 - e) << 23).view(torch.float32), br, bc, *x.shape)
    v = torch.where(torch.isfinite(x), v, torch.full_like(v, math.nan))
    return v.to(torch.float8_e4m3fn).float(), scale


def _through(x, br, bc):
    """x as its 8-bit blocks stand for it."""
    q, scale = _quantize(x, br, bc)
    return q * _spread(scale, br, bc, *x.shape)


def _act(gate, act):
    return torch.sigmoid(gate) if act == "sigmoid" else torch.tanh(gate) if act == "tanh" else gate


def _plain_residual(s, case, f):
    """out and y of residual_norm; `f` takes an input to the width that is computed in."""
    u = f(s["h"])
    if s["post_w"] is not None:
        u = _normed(u, f(s["post_w"]), None if s["post_b"] is None else f(s["post_b"]), case["kind"])
    if s["gate"] is not None:
        u = u * _act(f(s["gate"]), case["act"])
    if case["p"]:
        u = _drop(u, case["p"], s["rng"])
    if s["scale"] is not None:
        u = u * f(s["scale"])
    out = f(s["x"]) + u
    if s["next_w"] is None:
        return out, None
    return out, _normed(out, f(s["next_w"]), None if s["next_b"] is None else f(s["next_b"]), case["kind"])


def _gradients(s, outputs, upstream):
    leaves = [s[n] for n in LEAVES if s.get(n) is not None]
    return torch.autograd.grad(outputs, leaves, upstream)


def _float(t):
    return t.float()


def _run_plain(s):
    case = s["case"]
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "linear":
        x = s["x"].detach().float()
        if case["train"]:
            w = _through(s["w"].detach().float(), 128, 128)
        else:
            q, scale = s["kept"]
            w = q.float() * _spread(scale, 128, 128, *q.shape)
        y = _through(x, 1, 128) @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"].detach().float()
        if not case["train"]:
            return [y.to(dt)]
        dy = s["dy"].float()
        dx = _through(dy, 1, 128) @ w
        dw = _through(dy, 128, 1).t() @ _through(x, 128, 1)
        return [y.to(dt), dx.to(dt), dw.to(dt)] + ([dy.sum(0).to(dt)] if s["bias"] is not None else [])
    if op == "dropout":
        y = _drop(s["x"].float(), case["p"], s["rng"]).to(dt)
        return [y] if not case["train"] else [y, *torch.autograd.grad(y, [s["x"]], s["dy"])]
    if op == "norm":
        b = s["next_b"]
        y = _normed(s["x"].float(), s["next_w"].float(), None if b is None else b.float(), case["kind"]).to(dt)
        return [y] if not case["train"] else [y, *_gradients(s, [y], [s["dy"]])]
    out, y = _plain_residual(s, case, _float)
    outputs = [out.to(dt)] + ([y.to(dt)] if y is not None else [])
    if not case["train"]:
        return outputs
    return outputs + list(_gradients(s, outputs, [s["dout"]] + ([s["dy"]] if y is not None else [])))


# ------------------------------------------------------------------- the framework's calls
def _run_own(s):
    import pack3d_b200 as p3d
    case = s["case"]
    op = case["op"]
    if op == "linear":
        if not case["train"]:
            return [p3d.fp8_linear(s["x"], s["kept"], s["bias"])]
        y = p3d.fp8_linear(s["x"], s["w"], s["bias"])
        leaves = [s["x"], s["w"]] + ([s["bias"]] if s["bias"] is not None else [])
        return [y, *torch.autograd.grad(y, leaves, s["dy"])]
    if op == "dropout":
        y = p3d.dropout(s["x"], case["p"], s["rng"])
        return [y] if not case["train"] else [y, *torch.autograd.grad(y, [s["x"]], s["dy"])]
    if op == "norm":
        y = p3d.norm(s["x"], s["next"])
        return [y] if not case["train"] else [y, *_gradients(s, [y], [s["dy"]])]
    out, y = p3d.residual_norm(s["x"], s["h"], post_norm=s.get("post"), gate=s["gate"], gate_activation=case["act"],
                               scale=s["scale"], next_norm=s.get("next"), p=case["p"], rng=s["rng"])
    outputs = [out] + ([y] if y is not None else [])
    if not case["train"]:
        return outputs
    return outputs + list(_gradients(s, outputs, [s["dout"]] + ([s["dy"]] if y is not None else [])))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------- floors
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    op, train = case["op"], case["train"]
    if op == "linear":
        m, k, n = case["tokens"], case["k"], case["n"]
        flops = 2 * m * k * n
        if not train:
            return {"bytes": size * (m * k + m * n) + n * k, "flops": flops}
        return {"bytes": 2 * size * (m * k + m * n + n * k), "flops": 3 * flops}
    if op in ("dropout", "norm"):
        e = case["tokens"] * case["dim"]
        return {"bytes": (4 if train else 2) * e * size, "flops": (8 if op == "norm" else 2) * e * (3 if train else 1)}
    rows = case["batch"] * case["tokens"]
    e = rows * case["dim"]
    gate = {"none": 0, "element": e, "sample": case["batch"] * case["dim"], "token": rows}[case["gate"]]
    words = 3 * e + (e if case["next"] else 0) + gate
    if train:   # dout and dy; dx, dh and the gate's gradient
        words += 3 * e + (e if case["next"] else 0) + gate
    return {"bytes": words * size, "flops": 16 * e * (3 if train else 1)}


# ------------------------------------------------------------- the definitions in 64 bits
def _exact_norm(z, w, b, kind):
    """(N(z) * w + b, N(z), 1 / deviation)."""
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS)
    n = z * r
    return (n * w if b is None else n * w + b), n, r


def _exact_norm_back(g, n, r, kind):
    """The gradient of z from the gradient of N(z)."""
    d = g - n * (g * n).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(-1, keepdim=True)
    return r * d


def _two_to(e):
    """2^e for whole e in 64 bits, from its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_blocks(x, br, bc):
    """x in 64 bits as e4m3 numbers with a power-of-two scale for each br x bc block stand for it."""
    rows, cols = x.shape
    padded = torch.zeros(-(-rows // br) * br, -(-cols // bc) * bc, dtype=torch.float64, device=x.device)
    padded[:rows, :cols] = x
    t = padded.view(padded.shape[0] // br, br, padded.shape[1] // bc, bc)
    top = t.abs().amax((1, 3), keepdim=True)
    e = torch.where(top > 0, torch.ceil(torch.log2(top / 448)), torch.zeros_like(top))
    e = torch.where(top > 448 * _two_to(e), e + 1, e)                          # log2 may be off in its last place
    e = torch.where((top > 0) & (top <= 448 * _two_to(e - 1)), e - 1, e).clamp_min(-126)
    v = t / _two_to(e)
    # e4m3: three fraction bits, smallest exponent -6; ties to even
    step = _two_to(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    v = torch.round(v / step) * step
    return (v * _two_to(e)).view_as(padded)[:rows, :cols]


def exact(case, seed):
    s = _make(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    op, train = case["op"], case["train"]
    if op == "linear":
        w = _exact_blocks(d["w"], 128, 128)
        y = _exact_blocks(d["x"], 1, 128) @ w.t()
        if d["bias"] is not None:
            y += d["bias"]
        if not train:
            return [y]
        dx = _exact_blocks(d["dy"], 1, 128) @ w
        dw = _exact_blocks(d["dy"], 128, 1).t() @ _exact_blocks(d["x"], 128, 1)
        return [y, dx, dw] + ([d["dy"].sum(0)] if d["bias"] is not None else [])
    if op == "dropout":
        keep = _keep(case["tokens"], case["dim"], case["p"], s["rng"], "cuda").double()
        keep *= 65536 / (65536 - round(65536 * case["p"]))
        return [d["x"] * keep] + ([d["dy"] * keep] if train else [])
    kind = case["kind"]
    if op == "norm":
        y, n, r = _exact_norm(d["x"], d["next_w"], d["next_b"], kind)
        if not train:
            return [y]
        grads = [_exact_norm_back(d["dy"] * d["next_w"], n, r, kind), (d["dy"] * n).sum(0)]
        return [y, *grads] + ([d["dy"].sum(0)] if kind == "layer" else [])
    rows, dim = case["batch"] * case["tokens"], case["dim"]
    shape = d["x"].shape
    u = d["h"]
    if d["post_w"] is not None:
        u, hn, hr = _exact_norm(d["h"], d["post_w"], d["post_b"], kind)
    a = slope = torch.ones((), dtype=torch.float64, device="cuda")
    if d["gate"] is not None:
        a, slope = {"identity": lambda t: (t, torch.ones_like(t)),
                    "sigmoid": lambda t: (1 / (1 + torch.exp(-t)), torch.exp(-t) / (1 + torch.exp(-t)).square()),
                    "tanh": lambda t: (torch.tanh(t), 1 - torch.tanh(t).square())}[case["act"]](d["gate"])
    keep = 1.0
    if case["p"]:
        keep = _keep(rows, dim, case["p"], s["rng"], "cuda").view(shape).double()
        keep *= 65536 / (65536 - round(65536 * case["p"]))
    scale = d["scale"] if d["scale"] is not None else 1.0
    dropped = u * a * keep
    out = d["x"] + dropped * scale
    answer = [out]
    if d["next_w"] is not None:
        y, on, orr = _exact_norm(out, d["next_w"], d["next_b"], kind)
        answer.append(y)
    if not train:
        return answer
    g = d["dout"]
    if d["next_w"] is not None:
        g = g + _exact_norm_back(d["dy"] * d["next_w"], on, orr, kind)
    dv = g * scale * keep
    du = dv * a
    answer += [g, du if d["post_w"] is None else _exact_norm_back(du * d["post_w"], hn, hr, kind)]
    if d["gate"] is not None:
        dgate = dv * u * slope
        over = [i for i in range(3) if d["gate"].shape[i] != shape[i]]
        answer.append(dgate.sum(over, keepdim=True) if over else dgate)
    if d["scale"] is not None:
        answer.append((g * dropped).sum((0, 1)))
    if d["post_w"] is not None:
        answer.append((du * hn).sum((0, 1)))
        if d["post_b"] is not None:
            answer.append(du.sum((0, 1)))
    if d["next_w"] is not None:
        answer.append((d["dy"] * on).sum((0, 1)))
        if d["next_b"] is not None:
            answer.append(d["dy"].sum((0, 1)))
    return answer
