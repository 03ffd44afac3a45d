"""Operators of attention over ordered sequences, in real sizes.

``norm_rotate`` (norms of queries and keys for each head with the rotation of their positions),
``sequence_attention`` (attention over packed prompts of different lengths with grouped heads, both
directions), ``PagedCache.append`` / ``PagedCache.read`` (keys and values written into pages, in 8 bits with a
power-of-two scale for each token and head or as they are, and read back) and ``paged_attention`` (one new
token of each sequence over its pages).  Each is written out in elementary torch operations in 32 bits,
and, where ``own`` is set, called from ``pack3d_b200``.  ``exact`` is the same definition in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
BASE = 10000.0


# ------------------------------------------------------------------------------- cases
def _rotate(name, tokens, heads, kv_heads, dim, dtype, train, kind, axes, far):
    return {"name": name, "op": "rotate", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "train": train, "kind": kind, "axes": axes, "far": far}


def _attention(name, tokens, sequences, heads, kv_heads, dim, dtype, train, causal=True, prefix=0, cut=1):
    return {"name": name, "op": "attention", "tokens": tokens, "sequences": sequences, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "train": train, "causal": causal, "prefix": prefix,
            "cut": cut}


def _cache(name, old, new, sequences, kv_heads, dim, page, dtype, bits, cut=1):
    return {"name": name, "op": "cache", "old": old, "new": new, "sequences": sequences, "kv_heads": kv_heads,
            "dim": dim, "page": page, "dtype": dtype, "bits": bits, "cut": cut}


def _decode(name, tokens, sequences, heads, kv_heads, dim, page, dtype, bits, cut=1):
    return {"name": name, "op": "decode", "tokens": tokens, "sequences": sequences, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "bits": bits, "cut": cut}


def listed():
    return [
        # one token of an autoregressive pass, far into its sequence
        _rotate("rotate_token", 1, 16, 4, 128, "bf16", False, "rms", 1, 100000),
        # a training step on the 64^3 field, positions in three axes
        _rotate("rotate_field_train", 262144, 4, 4, 48, "bf16", True, "rms", 3, 0),
        # a training step on packed prompts at a language model's width, far positions
        _rotate("rotate_prompt_train", 16384, 32, 8, 128, "bf16", True, "rms", 1, 100000),
        # the smallest prompts that one call sees
        _attention("attention_short", 203, 3, 4, 4, 48, "bf16", False),
        # prompts of different lengths in a serving batch
        _attention("attention_prompts", 20011, 8, 16, 4, 128, "bf16", False),
        # a training step on many odd pieces, some of them empty, each after a cached prefix
        _attention("attention_pieces_train", 5003, 41, 6, 3, 48, "f16", True, True, 65),
        # a training step on packed documents
        _attention("attention_documents_train", 16384, 6, 16, 4, 128, "bf16", True),
        # one token of each of 24 sequences written in 8 bits, and the cache read back
        _cache("cache_step", 150, 24, 24, 4, 64, 16, "bf16", 8),
        # the prompts of a serving batch written in 8 bits behind what is there, and read back
        _cache("cache_prompts", 10000, 40001, 16, 8, 128, 64, "bf16", 8),
        # one token of four short sequences
        _decode("decode_short", 700, 4, 4, 2, 64, 16, "f16", 16),
        # one token of a serving batch over 8-bit pages
        _decode("decode_batch", 262144, 64, 32, 8, 128, 64, "bf16", 8),
        # one token of a single long sequence
        _decode("decode_long", 200003, 1, 32, 8, 128, 64, "bf16", 16),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm, and often odd."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    r = rng.random()
    return max(lo, v // 64 * 64) if r < 0.3 else max(lo, v // 8 * 8) if r < 0.5 else v


def _heads(rng, most=32):
    kv = rng.choice([1, 2, 3, 4, 8])
    return kv * rng.choice([r for r in (1, 2, 3, 4, 5, 8) if kv * r <= most]), kv


def draw(rng):
    op = rng.choice(["rotate", "attention", "attention", "cache", "decode", "decode"])
    heads, kv = _heads(rng)
    dim = rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    cut = rng.randrange(1 << 30)
    if op == "rotate":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        tokens = _log(rng, 1, 262144)
        while tokens * (heads + kv) * dim > 1.0e8:
            tokens = tokens * 5 // 8
        c = _rotate("", tokens, heads, kv, dim, dtype, rng.random() < 0.6, rng.choice(["rms", "layer"]),
                    rng.choice([1, 3]), rng.choice([0, 5000, 1000000]))
    elif op == "attention":
        while True:
            tokens, sequences = _log(rng, 1, 16384), _log(rng, 1, 64)
            c = _attention("", tokens, sequences, heads, kv, dim, dtype, rng.random() < 0.5, rng.random() < 0.75,
                           rng.choice([0, 0, 0, 40, 300, -20]), cut)
            q, k = _lengths(c)
            if sequences * heads * max(q) * max(k + [1]) * (2 if c["train"] else 1) <= 2.0e9:
                break
    elif op == "cache":
        while True:
            sequences = _log(rng, 1, 128)
            c = _cache("", _log(rng, 1, 65536), sequences if rng.random() < 0.4 else _log(rng, 1, 40000), sequences, kv, dim,
                       rng.choice([16, 32, 64, 64, 128, 24]), dtype, rng.choice([8, 8, 16]), cut)
            if (c["old"] + c["new"]) * kv * dim <= 5.0e7:
                break
    else:
        while True:
            c = _decode("", _log(rng, 1, 400000), _log(rng, 1, 128), heads, kv, dim, rng.choice([16, 32, 64, 64, 128, 24]),
                        dtype, rng.choice([8, 16]), cut)
            if c["tokens"] * kv * dim <= 2.0e8 and c["tokens"] * heads * dim <= 8.0e8:
                break
    c.pop("name")
    return c


def _cut(total, parts, seed):
    """`total` cut into `parts` lengths, unevenly; where there are many, every seventh is empty."""
    r = random.Random(seed)
    w = [0.0 if parts > 8 and i % 7 == 3 else r.uniform(0.2, 1.0) for i in range(parts)]
    edges = [0]
    for x in w:
        edges.append(edges[-1] + x)
    at = [round(total * e / edges[-1]) for e in edges]
    return [b - a for a, b in zip(at, at[1:])]


def _lengths(case):
    """Queries and keys of each sequence: a prefix of up to `prefix` more keys (or fewer, where it is below zero)."""
    q = _cut(case["tokens"], case["sequences"], case["cut"])
    r = random.Random(case["cut"] + 1)
    p = case["prefix"]
    return q, [max(0, n + (r.randrange(p + 1) if p > 0 else -r.randrange(1 - p))) for n in q]


def _cache_lengths(case):
    """Tokens of each sequence in the cache before the call, and new ones."""
    old = _cut(case["old"], case["sequences"], case["cut"])
    if case["new"] == case["sequences"]:
        return old, [1] * case["sequences"]
    return old, _cut(case["new"], case["sequences"], case["cut"] + 1)


# ------------------------------------------------------------------------------- inputs
def _offsets(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _pages(lengths, page, g):
    """A page table [sequences, most pages] over shuffled pages, some of which nobody has, and the number of pages."""
    need = [-(-n // page) for n in lengths]
    total, width = sum(need) + 3, max(max(need), 1)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), width, dtype=torch.int32, device="cuda")
    columns = torch.arange(width, device="cuda")
    starts = _offsets(need)[:-1]
    used = columns[None] < torch.tensor(need, device="cuda", dtype=torch.int32)[:, None]
    table[used] = order[(starts[:, None] + columns[None])[used]]
    return table, total


def _make(case, seed):
    """The inputs of a case as plain tensors."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, dim = DTYPES[case["dtype"]], case["dim"]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)

    s = {"case": case}
    if case["op"] == "rotate":
        n, h, kv = case["tokens"], case["heads"], case["kv_heads"]
        # queries and keys as a projection gives them, side by side in one row of a token
        row = normal(n, (h + kv) * dim, scale=1.5)
        s["q"], s["k"] = row[:, :h * dim].view(n, h, dim), row[:, h * dim:].view(n, kv, dim)
        s["q_w"], s["k_w"] = normal(dim, scale=0.2, mean=1.0), normal(dim, scale=0.2, mean=1.0)
        layer = case["kind"] == "layer"
        s["q_b"], s["k_b"] = (normal(dim, scale=0.1), normal(dim, scale=0.1)) if layer else (None, None)
        if case["axes"] == 3:
            side = max(1, round(n ** (1 / 3)))
            i = torch.arange(n, device="cuda")
            s["positions"] = torch.stack((i // (side * side), i // side % side, i % side), -1) + case["far"]
        else:
            s["positions"] = torch.arange(n, device="cuda") % 4096 + case["far"]
        s["dq"], s["dk"] = (normal(n, h, dim), normal(n, kv, dim)) if case["train"] else (None, None)
        return s
    if case["op"] == "attention":
        q_len, k_len = _lengths(case)
        s["q"] = normal(sum(q_len), case["heads"], dim, scale=1.3)
        s["k"] = normal(sum(k_len), case["kv_heads"], dim, scale=1.3)
        s["v"] = normal(sum(k_len), case["kv_heads"], dim)
        s["q_offsets"], s["k_offsets"] = _offsets(q_len), _offsets(k_len)
        s["longest"] = (max(q_len), max(k_len))
        s["dout"] = normal(sum(q_len), case["heads"], dim) if case["train"] else None
        return s
    kv, page = case["kv_heads"], case["page"]
    old, new = _cache_lengths(case) if case["op"] == "cache" else (_cut(case["tokens"], case["sequences"], case["cut"]), [])
    lengths = [a + b for a, b in zip(old, new)] if new else old
    s["table"], pages = _pages(lengths, page, g)
    s["lengths"] = torch.tensor(old, dtype=torch.int32, device="cuda")
    shape = (pages, kv, page, dim)
    # keys with a few channels above the others, values of changing size
    loud = 1 + 7 * (torch.rand(dim, generator=g, device="cuda") < 0.03).float()
    k = normal(*shape, dtype=torch.float32) * loud
    v = normal(*shape, dtype=torch.float32) * torch.exp2(torch.randn(*shape[:3], 1, generator=g, device="cuda"))
    if case["bits"] == 8:
        s["k_pages"], s["k_scales"] = _quantize(k)
        s["v_pages"], s["v_scales"] = _quantize(v)
    else:
        s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"] = k.to(dt), v.to(dt), None, None
    if case["op"] == "decode":
        s["q"] = normal(case["sequences"], case["heads"], dim, scale=0.6)
        return s
    s["new_k"] = normal(sum(new), kv, dim) * loud.to(dt)
    s["new_v"] = normal(sum(new), kv, dim)
    if sum(new) > 16:
        s["new_v"][torch.rand(sum(new), generator=g, device="cuda") < 0.02] = 0       # a padded token's values
    s["new_offsets"], s["all_offsets"] = _offsets(new), _offsets(lengths)
    s["all_lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["total"] = sum(lengths)
    return s


#: what a training step returns gradients of, in this order
LEAVES = ("q", "k", "v", "q_w", "q_b", "k_w", "k_b")


def prepare(case, seed):
    s = _make(case, seed)
    if case.get("train"):
        for name in LEAVES:
            if s.get(name) is not None:
                s[name] = s[name].detach().requires_grad_()
    if own:
        import pack3d_b200 as p3d
        if case["op"] == "rotate":
            s["q_norm"] = p3d.NormSpec(s["q_w"], s["q_b"], case["kind"], EPS)
            s["k_norm"] = p3d.NormSpec(s["k_w"], s["k_b"], case["kind"], EPS)
        elif case["op"] in ("cache", "decode"):
            s["cache"] = p3d.PagedCache(*s["k_pages"].shape, dtype=s["k_pages"].dtype, device="cuda")
            s["cache"].k.copy_(s["k_pages"])
            s["cache"].v.copy_(s["v_pages"])
            if case["bits"] == 8:
                s["cache"].k_scales.copy_(s["k_scales"])
                s["cache"].v_scales.copy_(s["v_scales"])
            s["k_pages"] = s["v_pages"] = s["k_scales"] = s["v_scales"] = None
    return s


# --------------------------------------------------------------------- plain forms, 32 bits
def _two_to(byte):
    """2^(byte - 127) of an int32 tensor, from its bits."""
    return (byte << 23).view(torch.float32)


def _quantize(x):
    """e4m3 values of x [.., dim] and a byte e + 127 of the power-of-two scale of each row."""
    m = x.abs().amax(-1)
    frac, e = torch.frexp(m)                       # m = frac * 2^e, frac in [0.5, 1)
    e = e - 9 + (frac > 0.875).to(e.dtype)         # 448 = 0.875 * 2^9
    e = torch.where(m > 0, e.clamp_min(-126), torch.zeros_like(e))
    return (x * _two_to(127 - e)[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _turned(z, positions, dim):
    """z [n, heads, dim] with pair i of an axis turned by position * BASE^(-i / pairs); angles in 64 bits."""
    if positions.ndim == 1:
        positions = positions[:, None]
    axes, half = positions.shape[1], dim // 2
    pairs = [half // axes + (1 if a < half % axes else 0) for a in range(axes)]
    angle = torch.cat([positions[:, a:a + 1].double() * BASE ** (-torch.arange(p, device=z.device, dtype=torch.float64) / max(p, 1))
                       for a, p in enumerate(pairs)], -1)
    cos, sin = angle.cos().to(z.dtype)[:, None], angle.sin().to(z.dtype)[:, None]
    a, b = z[..., 0::2], z[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _normed(z, w, b, kind):
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) * w
    return z if b is None else z + b


def _float(t):
    return None if t is None else t.float()


def _padded(offsets, longest):
    """Rows [sequences, longest] of the packed tensor that each padded place stands for, and which places are there."""
    i = torch.arange(longest, device=offsets.device)
    there = i[None] < (offsets[1:] - offsets[:-1])[:, None]
    return torch.where(there, offsets[:-1, None] + i[None], torch.zeros_like(offsets[:-1, None])).long(), there


def _plain_attention(s, case):
    h, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    lq, lk = s["longest"]
    if s["k"].shape[0] == 0 or s["q"].shape[0] == 0:
        return s["q"].float() * 0 + s["k"].float().sum() + s["v"].float().sum()
    rows, q_there = _padded(s["q_offsets"], lq)
    keys, k_there = _padded(s["k_offsets"], lk)
    b = rows.shape[0]
    q = s["q"].float()[rows].view(b, lq, kv, h // kv, dim).permute(0, 2, 3, 1, 4)          # [b, kv, group, lq, dim]
    k, v = (s[n].float()[keys].permute(0, 2, 1, 3)[:, :, None] for n in ("k", "v"))        # [b, kv, 1, lk, dim]
    seen = q_there[:, :, None] & k_there[:, None, :]
    if case["causal"]:
        # the last query sees the last key
        shift = (s["k_offsets"].diff() - s["q_offsets"].diff())[:, None, None]
        seen = seen & (torch.arange(lk, device=q.device)[None, None] <= torch.arange(lq, device=q.device)[None, :, None] + shift)
    seen = seen[:, None, None]
    score = (q @ k.transpose(-1, -2)) * (1 / math.sqrt(dim))
    score = torch.where(seen, score, torch.full_like(score, -math.inf))
    top = score.detach().amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))                   # a row that sees nothing: 0
    return out.permute(0, 3, 1, 2, 4).reshape(b, lq, h, dim)[q_there]


def _places(table, lengths, starts, offsets, page, total):
    """Page and place in it of each packed token: token i of sequence b is at starts[b] + i."""
    sequence = torch.repeat_interleave(torch.arange(len(lengths), device=table.device), lengths.long(), output_size=total)
    at = torch.arange(total, device=table.device) - offsets[sequence] + starts[sequence]
    return table[sequence, at // page].long(), at % page


def _kept(pages, scales):
    return pages.float() if scales is None else pages.float() * _two_to(scales.to(torch.int32))[..., None]


def _run_plain(s):
    case = s["case"]
    op, dt, dim = case["op"], DTYPES[case["dtype"]], case["dim"]
    if op == "rotate":
        out = [_turned(_normed(s[n].float(), s[n + "_w"].float(), _float(s[n + "_b"]), case["kind"]), s["positions"], dim).to(dt)
               for n in ("q", "k")]
        return out + (_gradients(s, out, [s["dq"], s["dk"]]) if case["train"] else [])
    if op == "attention":
        out = _plain_attention(s, case).to(dt)
        return [out] + (_gradients(s, [out], [s["dout"]]) if case["train"] else [])
    if op == "cache":
        page, at = _places(s["table"], s["all_lengths"] - s["lengths"], s["lengths"], s["new_offsets"], case["page"],
                           s["new_k"].shape[0])
        for name in ("k", "v"):
            new = s["new_" + name]
            if case["bits"] == 8:
                new, scale = _quantize(new.float())
                s[name + "_scales"][page, :, at] = scale
                s[name + "_pages"].view(torch.uint8)[page, :, at] = new.view(torch.uint8)
            else:
                s[name + "_pages"][page, :, at] = new
        page, at = _places(s["table"], s["all_lengths"], torch.zeros_like(s["lengths"]), s["all_offsets"], case["page"],
                           s["total"])
        return [_kept(s[n + "_pages"].view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn) if case["bits"] == 8
                      else s[n + "_pages"][page, :, at],
                      None if case["bits"] != 8 else s[n + "_scales"][page, :, at]).to(dt) for n in ("k", "v")]
    # decode: padded to the width of the page table
    h, kv, b = case["heads"], case["kv_heads"], case["sequences"]
    i = torch.arange(s["table"].shape[1] * case["page"], device="cuda")
    where, at = s["table"][:, i // case["page"]].long(), (i % case["page"]).expand(b, -1)
    take = (lambda t: t.view(torch.uint8)[where, :, at].view(t.dtype)) if case["bits"] == 8 else (lambda t: t[where, :, at])
    k, v = (_kept(take(s[n + "_pages"]), None if case["bits"] != 8 else s[n + "_scales"][where, :, at]).permute(0, 2, 1, 3)
            for n in ("k", "v"))                                                             # [b, kv, longest, dim]
    score = (s["q"].float().view(b, kv, h // kv, dim) @ k.transpose(-1, -2)) * (1 / math.sqrt(dim))
    score = torch.where((i < s["lengths"][:, None])[:, None, None], score, torch.full_like(score, -math.inf))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))                    # an empty sequence: 0
    return [out.reshape(b, h, dim).to(dt)]


def _gradients(s, outputs, upstream):
    leaves = [s[n] for n in LEAVES if s.get(n) is not None]
    return list(torch.autograd.grad(outputs, leaves, upstream))


# ------------------------------------------------------------------- the framework's calls
def _run_own(s):
    import pack3d_b200 as p3d
    case = s["case"]
    op = case["op"]
    if op == "rotate":
        out = list(p3d.norm_rotate(s["q"], s["k"], s["positions"], q_norm=s["q_norm"], k_norm=s["k_norm"], base=BASE))
        return out + (_gradients(s, out, [s["dq"], s["dk"]]) if case["train"] else [])
    if op == "attention":
        out = p3d.sequence_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], causal=case["causal"])
        return [out] + (_gradients(s, [out], [s["dout"]]) if case["train"] else [])
    if op == "cache":
        s["cache"].append(s["new_k"], s["new_v"], s["table"], s["lengths"], s["new_offsets"])
        return list(s["cache"].read(s["table"], s["all_offsets"], s["total"], dtype=DTYPES[case["dtype"]]))
    return [p3d.paged_attention(s["q"], s["cache"], s["table"], s["lengths"])]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------- floors
def _seen(case):
    """Pairs of a query and a key that it sees."""
    total = 0
    for q, k in zip(*_lengths(case)):
        if not case["causal"]:
            total += q * k
        else:   # row i sees min(k, max(0, k - q + i + 1)) keys
            first = max(0, q - k)
            n = q - first
            total += n * (k - q + first + 1 + k) // 2 if n > 0 else 0
    return total


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    dim, kv, op = case["dim"], case["kv_heads"], case["op"]
    if op == "rotate":
        e = case["tokens"] * (case["heads"] + kv) * dim
        return {"bytes": (4 if case["train"] else 2) * e * size + 8 * case["tokens"] * case["axes"],
                "flops": 12 * e * (3 if case["train"] else 1)}
    if op == "attention":
        q, k = _lengths(case)
        e = sum(q) * case["heads"] * dim * 2 + sum(k) * kv * dim * 2
        flops = 4 * _seen(case) * case["heads"] * dim
        # a training step: two products forward, five backward
        return {"bytes": size * e * (2 if case["train"] else 1), "flops": flops * (3.5 if case["train"] else 1)}
    row = dim + 1 if case["bits"] == 8 else size * dim
    if op == "cache":
        return {"bytes": 2 * kv * (case["new"] * (size * dim + row) + (case["old"] + case["new"]) * (row + size * dim)),
                "flops": 4 * kv * dim * (case["old"] + 2 * case["new"])}
    return {"bytes": 2 * kv * row * case["tokens"] + 2 * case["sequences"] * case["heads"] * dim * size,
            "flops": 4 * case["tokens"] * case["heads"] * dim}


# ------------------------------------------------------------- the definitions in 64 bits
def _exact_norm(z, w, b, kind):
    """(N(z) * w + b, N(z), 1 / deviation)."""
    if kind == "layer":
        z = z - z.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS)
    n = z * r
    return (n * w if b is None else n * w + b), n, r


def _exact_turn(z, positions, back):
    """Pairs as complex numbers times exp(i angle), or its conjugate."""
    half = z.shape[-1] // 2
    where = positions.double() if positions.ndim == 2 else positions.double()[:, None]
    columns = []
    for a in range(where.shape[1]):
        count = half // where.shape[1] + (1 if a < half % where.shape[1] else 0)
        columns += [where[:, a] * math.pow(BASE, -i / count) for i in range(count)]
    angle = torch.stack(columns, -1)[:, None]
    return torch.view_as_real(torch.view_as_complex(z.reshape(*z.shape[:-1], half, 2).contiguous())
                              * torch.polar(torch.ones_like(angle), -angle if back else angle)).flatten(-2)


def _exact_rotate(d, case):
    outs, grads, params = [], [], []
    for name in ("q", "k"):
        w, b, z = d[name + "_w"], d[name + "_b"], d[name]
        y, n, r = _exact_norm(z, w, b, case["kind"])
        outs.append(_exact_turn(y, d["positions"], False))
        if case["train"]:
            up = _exact_turn(d["d" + name], d["positions"], True)
            g = up * w
            dz = g - n * (g * n).mean(-1, keepdim=True)
            if case["kind"] == "layer":
                dz = dz - g.mean(-1, keepdim=True)
            grads.append(r * dz)
            params.append((up * n).sum((0, 1)))
            if b is not None:
                params.append(up.sum((0, 1)))
    return outs + grads + params


def _exact_attention(d, case):
    h, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    out, dq = torch.zeros_like(d["q"]), torch.zeros_like(d["q"])
    dk, dv = torch.zeros_like(d["k"]), torch.zeros_like(d["v"])
    q0 = k0 = 0
    for nq, nk in zip(*_lengths(case)):
        sq, sk = slice(q0, q0 + nq), slice(k0, k0 + nk)
        q0, k0 = q0 + nq, k0 + nk
        if not nq or not nk:
            continue
        hidden = torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1) if case["causal"] else None
        empty = hidden.all(-1) if hidden is not None else None
        for head in range(h):
            q, k, v = d["q"][sq, head], d["k"][sk, head // (h // kv)], d["v"][sk, head // (h // kv)]
            score = q @ k.t() / math.sqrt(dim)
            if hidden is not None:
                score.masked_fill_(hidden, -math.inf)
            p = torch.softmax(score, -1)
            if hidden is not None:
                p[empty] = 0
            o = p @ v
            out[sq, head] = o
            if case["train"]:
                up = d["dout"][sq, head]
                dv[sk, head // (h // kv)] += p.t() @ up
                ds = p * (up @ v.t() - (up * o).sum(-1, keepdim=True)) / math.sqrt(dim)
                dq[sq, head] = ds @ k
                dk[sk, head // (h // kv)] += ds.t() @ q
    return [out, dq, dk, dv] if case["train"] else [out]


def _exact_pow2(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_8bit(x):
    """Rows of x in 64 bits as e4m3 numbers with the smallest power-of-two scale that brings them to 448 stand for them."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.ceil(torch.log2(top / 448)), torch.zeros_like(top))
    e = torch.where(top > 448 * _exact_pow2(e), e + 1, e)                     # log2 may be off in its last place
    e = torch.where((top > 0) & (top <= 448 * _exact_pow2(e - 1)), e - 1, e).clamp_min(-126)
    v = x / _exact_pow2(e)
    # e4m3: three fraction bits, smallest exponent -6; ties to even
    step = _exact_pow2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step * _exact_pow2(e)


def _exact_pages(s, name):
    pages = s[name + "_pages"].double()
    return pages if s[name + "_scales"] is None else pages * _exact_pow2(s[name + "_scales"].to(torch.int64) - 127)[..., None]


def exact(case, seed):
    s = _make(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.dtype in DTYPES.values() else v for k, v in s.items()}
    if case["op"] == "rotate":
        return _exact_rotate(d, case)
    if case["op"] == "attention":
        return _exact_attention(d, case)
    table, page, kv, dim = s["table"].tolist(), case["page"], case["kv_heads"], case["dim"]
    if case["op"] == "cache":
        old, new = _cache_lengths(case)
        result = []
        for name in ("k", "v"):
            pages, rows, at = _exact_pages(s, name), [], 0
            fresh = _exact_8bit(d["new_" + name]) if case["bits"] == 8 else d["new_" + name]
            for b, (n, more) in enumerate(zip(old, new)):
                own_pages = pages[table[b]].permute(0, 2, 1, 3).reshape(-1, kv, dim)
                rows += [own_pages[:n], fresh[at:at + more]]
                at += more
            result.append(torch.cat(rows))
        return result
    k_pages, v_pages = _exact_pages(s, "k"), _exact_pages(s, "v")
    out = torch.zeros_like(d["q"])
    for b, n in enumerate(_cut(case["tokens"], case["sequences"], case["cut"])):
        if n:
            k, v = (t[table[b]].permute(1, 0, 2, 3).reshape(kv, -1, dim)[:, :n] for t in (k_pages, v_pages))
            q = d["q"][b].view(kv, -1, dim)
            out[b] = (torch.softmax(q @ k.transpose(1, 2) / math.sqrt(dim), -1) @ v).reshape(-1, dim)
    return [out]
