"""The paged cache and the attention of one new token over it, against their definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def offsets_of(lengths, device):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return ints(at, device)


def table_of(lengths, page, device, seed=0, width=None, spare=3):
    """A table over shuffled pages; places that no token uses hold a page number far outside."""
    need = [-(-n // page) for n in lengths]
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(need) + spare, generator=gen).tolist()
    width = max(need + [1]) if width is None else width
    rows = []
    for n in need:
        rows.append([order.pop() for _ in range(n)] + [1 << 30] * (width - n))
    return ints(rows, device).view(len(lengths), width), sum(need) + spare


def two_to(e):
    """2^e in 64 bits for whole e, from its bits: the device's pow is off by its last place."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def in_8_bits(x):
    """What 8 bits hold of x [.., dim] in 64 bits, by the definition; not finite: NaN."""
    x = x.double()
    finite = torch.isfinite(x)
    top = torch.where(finite, x.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp_min(1e-300) / 448)), -126.0)
    e = torch.where(top > 448 * two_to(e), e + 1, e)
    e = torch.where((top > 0) & (top <= 448 * two_to(e - 1)), e - 1, e).clamp_min(-126)
    v = x / two_to(e)
    step = two_to(torch.floor(torch.log2(torch.where(finite, v, 0.0).abs().clamp_min(2.0 ** -6))) - 3)
    return torch.where(finite, torch.round(v / step) * step * two_to(e), math.nan)


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(torch.where(a.isnan(), 0, a), torch.where(b.isnan(), 0, b))


# ------------------------------------------------------------------------------- written and read back
@pytest.mark.parametrize("dtype,stored", [(BF16, E4M3), (F16, E4M3), (F32, E4M3), (BF16, BF16), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("dim,kv,page", [(8, 1, 1), (48, 3, 16), (64, 2, 24), (128, 8, 64), (256, 1, 7)])
def test_append_and_read(cuda_device, dtype, stored, dim, kv, page):
    from pack3d_b200 import PagedCache
    old, new = [3, 0, 70, 16, 1], [1, 0, 33, 64, 130]
    both = [a + b for a, b in zip(old, new)]
    table, pages = table_of(both, page, cuda_device)
    cache = PagedCache(pages, kv, page, dim, dtype=stored, device=cuda_device)
    gen = torch.Generator(device=cuda_device).manual_seed(dim)
    kept = [torch.zeros(len(old), max(both), kv, dim, dtype=torch.float64, device=cuda_device) for _ in range(2)]
    for lengths, more in (([0] * len(old), old), (old, new)):
        rows = [(torch.randn(sum(more) + 2, kv, dim, generator=gen, device=cuda_device)
                 * torch.exp2(6 * torch.randn(sum(more) + 2, kv, 1, generator=gen, device=cuda_device))).to(dtype) for _ in range(2)]
        for t in rows:
            t[::5] = 0                                     # tokens of zeros
            t[-2:] = math.nan                              # rows of no sequence
        before = [x.clone() for x in (cache.k.view(torch.uint8), cache.v.view(torch.uint8))]
        cache.append(*rows, table, ints(lengths, cuda_device), offsets_of(more, cuda_device))
        at = 0
        for b, (n, m) in enumerate(zip(lengths, more)):
            for t, r in zip(kept, rows):
                t[b, n:n + m] = in_8_bits(r[at:at + m]) if stored is E4M3 else r[at:at + m].double()
            at += m
        # places that belong to no new token keep their bytes
        written = torch.zeros(pages, page, dtype=torch.bool, device=cuda_device)
        for b, (n, m) in enumerate(zip(lengths, more)):
            for i in range(n, n + m):
                written[table[b, i // page].item(), i % page] = True
        keep = ~written[:, None, :, None]
        for now, then in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8)), before):
            assert torch.equal(torch.where(keep, now, 0), torch.where(keep, then, 0))
    want = [torch.cat([t[b, :n] for b, n in enumerate(both)]) for t in kept]
    for out in (F32, BF16, F16):
        got = cache.read(table, offsets_of(both, cuda_device), sum(both) + 3, dtype=out)
        for g, w in zip(got, want):
            assert g.dtype == out and not g[sum(both):].any()
            assert same(g[:sum(both)], w.float().to(out))   # f16 inputs past its range are infinite
    starts = [min(n, 5) for n in both]
    part = cache.read(table, offsets_of([n - s for n, s in zip(both, starts)], cuda_device), sum(both) - sum(starts),
                      starts=ints(starts, cuda_device), dtype=F32)
    for g, t in zip(part, kept):
        assert same(g, torch.cat([t[b, s:n] for b, (s, n) in enumerate(zip(starts, both))]).float())
    assert cache.read(table, offsets_of(both, cuda_device), 4)[0].dtype == (BF16 if stored is E4M3 else stored)


def test_rounding_borders(cuda_device):
    """Values on and beside the borders of a scale and of an e4m3 step, the largest and smallest."""
    from pack3d_b200 import PagedCache
    x = torch.tensor([[448, 1, 0.0009765625, 17, 18, 19, 1 / 3, 0], [448.1, 449, 25, 26, 27, 1e-3, 1e-6, 0], [2 ** -133, 2 ** -130, 0, 0, 0, 0, 0, 0],
                      [3e38, 1e38, -3.3e38, 1e30, 1, 0, 0, 0], [0] * 8, [math.inf, 5, -math.inf, math.nan, 448, 1, 2, 3],
                      [math.nan] * 8, [-0.0, 1e-20, 224, 225, 240, 248, 464, -464]], device=cuda_device, dtype=F32)[:, None]
    cache = PagedCache(2, 1, 8, 8, dtype=E4M3, device=cuda_device)
    table, offsets = ints([[1]], cuda_device), ints([0, 8], cuda_device)
    cache.append(x, x, table, ints([0], cuda_device), offsets)
    got, _ = cache.read(table, offsets, 8, dtype=F32)
    want = in_8_bits(x).float()
    assert same(got, want)
    assert not cache.k.view(torch.uint8)[0].any()


def test_strided_new_rows(cuda_device):
    from pack3d_b200 import PagedCache
    row = torch.randn(20, 2 * 2 * 64 + 8, device=cuda_device).to(BF16)
    k, v = row[:, :128].view(20, 2, 64), row[:, 128:256].view(20, 2, 64)
    off = torch.empty(20 * 128 + 1, dtype=BF16, device=cuda_device)[1:].view(20, 2, 64).copy_(v)
    table, offsets = ints([[2, 0]], cuda_device), ints([0, 20], cuda_device)
    results = []
    for a, b in ((k.contiguous(), v.contiguous()), (k, v), (k, off), (k.transpose(0, 1).contiguous().transpose(0, 1), v)):
        cache = PagedCache(3, 2, 16, 64, device=cuda_device)
        cache.append(a, b, table, ints([0], cuda_device), offsets)
        results.append(cache.read(table, offsets, 20))
    for r in results:
        assert torch.equal(r[0], k) and torch.equal(r[1], v)


def test_bad_pages_are_never_followed(cuda_device):
    from pack3d_b200 import PagedCache, _native, paged_attention
    _native.device_errors()
    cache = PagedCache(4, 1, 8, 64, device=cuda_device)
    table = ints([[0, -1, 2], [1, 1 << 30, 3]], cuda_device)
    x = torch.randn(40, 1, 64, device=cuda_device).to(BF16)
    offsets = ints([0, 20, 40], cuda_device)
    cache.append(x, x, table, ints([0, 0], cuda_device), offsets)
    assert _native.device_errors() == 64
    k, _ = cache.read(table, offsets, 40)
    assert _native.device_errors() == 64
    bad = torch.zeros(40, dtype=torch.bool, device=cuda_device)
    bad[8:16] = bad[28:36] = True
    assert k[bad].isnan().all() and torch.equal(k[~bad], x[~bad])
    # past the table's width, and before its first place
    cache.append(x[:2], x[:2], table[:1], ints([23], cuda_device), ints([0, 2], cuda_device))
    assert _native.device_errors() == 64
    cache.append(x[:2], x[:2], table[:1], ints([-1], cuda_device), ints([0, 2], cuda_device))
    assert _native.device_errors() == 64
    q = torch.randn(2, 2, 64, device=cuda_device).to(BF16)
    out = paged_attention(q, cache, table, ints([8, 20], cuda_device))
    assert torch.isfinite(out[0]).all() and out[1].isnan().all() and _native.device_errors() == 64
    assert paged_attention(q, cache, table, ints([25, 3], cuda_device))[0].isnan().all()
    _native.device_errors()


# ------------------------------------------------------------------------------- one new token
def filled(lengths, kv, dim, page, stored, device, seed=0, heads=None, dtype=BF16, loud=1.0):
    """A cache whose free places hold NaN, its table, what it stands for, and queries."""
    from pack3d_b200 import PagedCache
    gen = torch.Generator(device=device).manual_seed(seed)
    table, pages = table_of(lengths, page, device, seed)
    cache = PagedCache(pages, kv, page, dim, dtype=stored, device=device)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x7f if stored is E4M3 else 0xff)
    n = sum(lengths)
    k = (torch.randn(n, kv, dim, generator=gen, device=device) * 1.5).to(dtype)
    v = (torch.randn(n, kv, dim, generator=gen, device=device)
         * torch.exp2(loud * torch.randn(n, kv, 1, generator=gen, device=device))).to(dtype)
    cache.append(k, v, table, ints([0] * len(lengths), device), offsets_of(lengths, device))
    held = cache.read(table, offsets_of(lengths, device), n, dtype=F32)
    q = torch.randn(len(lengths), heads or kv, dim, generator=gen, device=device).to(dtype)
    return cache, table, held, q


def decode_reference(q, held, lengths, scale):
    """out in 64 bits and a bound of its error: weights rounded to the storage dtype (u; f16 over 8 bits, whose
    weights are relative to the largest product), exponentials to 2^-13, and the result's own rounding."""
    u = torch.finfo(q.dtype).eps / 2
    out, tol = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    h, g, at = q.shape[1], held[0].shape[1], 0
    for b, n in enumerate(lengths):
        k, v = (t[at:at + n].double() for t in held)
        at += n
        if not n:
            continue
        for i in range(h):
            p = torch.softmax(k[:, i // (h // g)] @ q[b, i].double() * scale, 0)
            out[b, i] = p @ v[:, i // (h // g)]
            # 2^-24 of the largest weighted value, for each token: what f16 weights lose below their smallest normal
            most = (p[:, None] * v[:, i // (h // g)].abs().amax(-1, keepdim=True)).max()
            tol[b, i] = u * out[b, i].abs() + (u + 2.0 ** -13 + 2.0 ** -15) * (p @ v[:, i // (h // g)].abs()) + n * 2.0 ** -24 * most
    return out, tol + 2.0 ** -24


@pytest.mark.parametrize("stored", [BF16, F16, E4M3])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 2, 128), (5, 1, 48), (16, 1, 128), (20, 1, 32), (33, 1, 8), (6, 3, 80), (2, 1, 120)])
@pytest.mark.parametrize("page", [16, 5, 64])
def test_decode(cuda_device, stored, heads, kv, dim, page):
    from pack3d_b200 import paged_attention
    lengths = [1, 0, 63, 64, 65, 300, 7, 16, 129]
    dtype = BF16 if stored is E4M3 else stored
    cache, table, held, q = filled(lengths, kv, dim, page, stored, cuda_device, heads=heads, dtype=dtype)
    got = paged_attention(q, cache, table, ints(lengths, cuda_device))
    want, tol = decode_reference(q, held, lengths, dim ** -0.5)
    assert not got[1].any()
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("stored", [BF16, E4M3])
def test_decode_long(cuda_device, stored):
    """One sequence over all of the device, and lengths that share it unevenly."""
    from pack3d_b200 import paged_attention
    for lengths, heads, kv, dim in (([70001], 8, 2, 128), ([9000, 1, 0, 20000, 17], 4, 4, 64)):
        cache, table, held, q = filled(lengths, kv, dim, 64, stored, cuda_device, heads=heads)
        got = paged_attention(q, cache, table, ints(lengths, cuda_device))
        want, tol = decode_reference(q, held, lengths, dim ** -0.5)
        assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decode_over_8_bits_of_any_size(cuda_device, dtype):
    """Values whose scales lie far apart, and queries of any size: nothing overflows on the way through f16."""
    from pack3d_b200 import paged_attention
    lengths = [200, 33]
    cache, table, held, q = filled(lengths, 2, 64, 16, E4M3, cuda_device, heads=8, dtype=dtype, loud=4.0 if dtype == BF16 else 2.0)
    for size in (1.0, 1e-3, 30.0):
        got = paged_attention(q * size, cache, table, ints(lengths, cuda_device))
        want, tol = decode_reference(q * size, held, lengths, 0.125)
        # scores of up to 30 x 100: fp32 products to 2^-20 of them
        assert ((got.double() - want).abs() <= tol + 2.0 ** -20 * 100 * size * tol.new_tensor(held[1].abs().max().item())).all()
    huge = torch.full_like(q, 3e38 if dtype == BF16 else 6e4)
    assert paged_attention(huge, cache, table, ints(lengths, cuda_device), scale=1e-38).isfinite().all()


@pytest.mark.parametrize("stored", [BF16, E4M3])
def test_decode_passes_on_what_is_not_finite(cuda_device, stored):
    """NaN in a seen key reaches the heads that read it; places past the length hold NaN in every test here."""
    from pack3d_b200 import paged_attention
    lengths = [100, 40]
    cache, table, held, q = filled(lengths, 2, 64, 16, stored, cuda_device, heads=4)
    want = paged_attention(q, cache, table, ints(lengths, cuda_device))
    assert want.isfinite().all()
    x = torch.full((1, 2, 64), math.nan, dtype=BF16, device=cuda_device)
    x[:, 1] = 0.5
    cache.append(x, x, table, ints([50, 0], cuda_device), ints([0, 1, 1], cuda_device))
    got = paged_attention(q, cache, table, ints(lengths, cuda_device))
    assert got[0, :2].isnan().all() and got[0, 2:].isfinite().all() and torch.equal(got[1], want[1])
    q[1] = math.nan
    got = paged_attention(q, cache, table, ints(lengths, cuda_device))
    assert got[1].isnan().all() and got[0, 2:].isfinite().all()


def test_decode_strides_streams_and_graphs(cuda_device):
    from pack3d_b200 import paged_attention
    lengths = [300, 4, 150]
    cache, table, held, q = filled(lengths, 2, 64, 16, E4M3, cuda_device, heads=8)
    n = ints(lengths, cuda_device)
    want = paged_attention(q, cache, table, n)
    wide = torch.zeros(3, 10, 128, dtype=BF16, device=cuda_device)
    wide[:, 1:9, 64:] = q
    assert torch.equal(paged_attention(wide[:, 1:9, 64:], cache, table, n), want)
    assert torch.equal(paged_attention(q.transpose(0, 1).contiguous().transpose(0, 1), cache, table, n), want)
    widened = torch.cat([table, torch.full((3, 40), -7, dtype=torch.int32, device=cuda_device)], 1)
    assert torch.equal(paged_attention(q, cache, widened[:, :table.shape[1]], n), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = paged_attention(q, cache, table, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, want)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(q, cache, table, n))
        graphs.append(graph)
    for seed in (1, 2):
        q.copy_(torch.randn(q.shape, generator=torch.Generator(device=cuda_device).manual_seed(seed), device=cuda_device))
        n.copy_(ints([20 * seed, 1, 70 * seed], cuda_device))
        for graph in graphs:
            graph.replay()
        fresh = paged_attention(q, cache, table, n)
        assert all(torch.equal(o, fresh) for o in outs)


def test_places_past_32_bits(cuda_device):
    """A cache of more than 2^32 bytes and 2^31 elements: its last pages are written, read and attended to."""
    from pack3d_b200 import PagedCache, paged_attention
    pages = (1 << 31) // (8 * 64 * 128) + 40
    cache = PagedCache(pages, 8, 64, 128, dtype=BF16, device=cuda_device)
    table = ints([[pages - 1, 0, pages - 30]], cuda_device)
    k, v = (torch.randn(150, 8, 128, device=cuda_device).to(BF16) for _ in range(2))
    cache.append(k, v, table, ints([0], cuda_device), ints([0, 150], cuda_device))
    got = cache.read(table, ints([0, 150], cuda_device), 150)
    assert torch.equal(got[0], k) and torch.equal(got[1], v)
    assert torch.equal(cache.k[pages - 1], k[:64].transpose(0, 1))
    q = torch.randn(1, 16, 128, device=cuda_device).to(BF16)
    out = paged_attention(q, cache, table, ints([150], cuda_device))
    want, tol = decode_reference(q, (k, v), [150], 128 ** -0.5)
    assert ((out.double() - want).abs() <= tol).all()


def test_cache_refusals(cuda_device):
    from pack3d_b200 import PagedCache, paged_attention
    for bad in ((0, 1, 1, 8), (1, 1, 1, 9), (1, 1, 1, 264), (1, 1.0, 1, 8)):
        with pytest.raises(ValueError):
            PagedCache(*bad, device=cuda_device)
    with pytest.raises(ValueError, match="dtype"):
        PagedCache(1, 1, 1, 8, dtype=torch.int8, device=cuda_device)
    cache = PagedCache(4, 2, 8, 64, device=cuda_device)
    table, lengths, offsets = ints([[0, 1]], cuda_device), ints([0], cuda_device), ints([0, 3], cuda_device)
    x = torch.randn(3, 2, 64, device=cuda_device).to(BF16)
    for args, text in (((x[:, :1], x, table, lengths, offsets), "new k and v"), ((x.half(), x.half(), table, lengths, offsets), "dtype"),
                       ((x, x, table.long(), lengths, offsets), "table"), ((x, x, table[0], lengths, offsets), "table"),
                       ((x, x, table, lengths.cpu(), offsets), "lengths"), ((x, x, table, lengths, lengths), "offsets"),
                       ((x.clone().requires_grad_(), x, table, lengths, offsets), "no gradients")):
        with pytest.raises(ValueError, match=text):
            cache.append(*args)
    for rows, dtype in ((-1, None), (1.5, None), (3, torch.int32)):
        with pytest.raises(ValueError):
            cache.read(table, offsets, rows, dtype=dtype)
    q = torch.randn(1, 4, 64, device=cuda_device).to(BF16)
    for args, text in (((q.float(), cache, table, lengths), "fp16 or bf16"), ((q.half(), cache, table, lengths), "cache's dtype"),
                       ((q[:, :3], cache, table, lengths), "divisible"), ((q[..., :32], cache, table, lengths), "q must be"),
                       ((q.expand(2, 4, 64), cache, table, lengths), "q must be"), ((q, cache, table, offsets), "lengths"),
                       ((q.clone().requires_grad_(), cache, table, lengths), "no gradients"), ((q, (cache,), table, lengths), "PagedCache")):
        with pytest.raises(ValueError, match=text):
            paged_attention(*args)
    cache.k = cache.k.transpose(0, 1)
    with pytest.raises(ValueError, match="contiguous"):
        cache.append(x, x, table, lengths, offsets)
    eight = PagedCache(4, 2, 8, 64, dtype=E4M3, device=cuda_device)
    eight.k_scales = None
    with pytest.raises(ValueError, match="scales"):
        eight.append(x, x, table, lengths, offsets)


def test_no_sequences_and_no_rows(cuda_device):
    from pack3d_b200 import PagedCache, paged_attention
    cache = PagedCache(4, 2, 8, 64, device=cuda_device)
    none, empty = ints([], cuda_device).view(0, 3), torch.zeros(0, 2, 64, dtype=BF16, device=cuda_device)
    cache.append(empty, empty, none, ints([], cuda_device), ints([0], cuda_device))
    assert cache.read(none, ints([0], cuda_device), 2)[0].shape == (2, 2, 64)
    assert paged_attention(empty.expand(0, 2, 64), cache, none, ints([], cuda_device)).shape == (0, 2, 64)
    assert not paged_attention(torch.ones(1, 2, 64, dtype=BF16, device=cuda_device), cache, ints([[0]], cuda_device)[:, :0],
                               ints([0], cuda_device)).any()


@pytest.mark.parametrize("stored,dtype", [(F16, F16), (E4M3, F16), (E4M3, BF16), (BF16, BF16)])
@pytest.mark.parametrize("first", [True, False])
def test_many_small_weights(cuda_device, stored, dtype, first):
    """One loud token whose values are 0 but for one and 65,535 of 2^-26 of its weight: what they add up to is not lost.  400 sequences over
    the same pages, so that a block has whole sequences."""
    from pack3d_b200 import PagedCache, paged_attention
    n, dim, page, sequences = 65536, 64, 64, 400
    at = 0 if first else n - 1
    cache = PagedCache(n // page, 1, page, dim, dtype=stored, device=cuda_device)
    table = torch.arange(n // page, dtype=torch.int32, device=cuda_device)[None]
    k = torch.zeros(n, 1, dim, dtype=dtype, device=cuda_device)
    v = (torch.randn(n, 1, dim, generator=torch.Generator(device=cuda_device).manual_seed(1), device=cuda_device) * 0.25 + 1).to(dtype)
    k[at, 0, 0], v[at], v[at, 0, 0] = 18.0, 0, 1     # e^18 is 2^26; a value of about the others' scale
    cache.append(k, v, table, ints([0], cuda_device), ints([0, n], cuda_device))
    held = cache.read(table, ints([0, n], cuda_device), n, dtype=F32)
    q = torch.zeros(sequences, 3, dim, dtype=dtype, device=cuda_device)
    q[..., 0] = 1
    out = paged_attention(q, cache, table.expand(sequences, -1), ints([n] * sequences, cuda_device), scale=1.0)
    assert held[0][at, 0, 0] == 18
    p = torch.softmax(held[0][:, 0, 0].double(), 0)
    values = held[1][:, 0].double()
    want = (p[:, None] * values).sum(0)
    # weights and results: half a step each; f16 weights half of its smallest number, beside 2^10 for the largest weight times scale
    # (values lie below 4, their scales below 2^-6); exponentials to 2^-13, fp32 sums of a thread's thousands of tokens to 2^-13
    u = torch.finfo(dtype).eps / 2
    tol = (2 * u + 2 * 2.0 ** -13) * want.abs() + (0 if stored is BF16 else 2.0 ** -35 * n * 448 * 2.0 ** -6)
    assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("stored,dim", [(BF16, 64), (BF16, 128), (E4M3, 128)])
def test_wider_tables(cuda_device, stored, dim):
    """The same lengths under tables of any width, on both sides of the one from which work is cut over sequences: the same result up to the
    order of its sums, whatever the columns that no token reaches hold."""
    from pack3d_b200 import paged_attention
    lengths, page = [100, 0, 256, 1, 200], 16
    cache, table, held, q = filled(lengths, 2, dim, page, stored, cuda_device, heads=4)
    want, tol = decode_reference(q, held, lengths, dim ** -0.5)
    n = ints(lengths, cuda_device)
    seen = {}
    unit = 4 * (16 if dim == 128 and stored is not E4M3 else 32)
    for width in (table.shape[1], 4 * unit // page, 4 * unit // page + 1, 10 * unit // page, 2000):
        more = width - table.shape[1]
        wide = torch.cat([table, torch.full((len(lengths), max(more, 0)), -7, dtype=torch.int32, device=cuda_device)], 1)
        got = paged_attention(q, cache, wide, n)
        assert torch.equal(got, paged_attention(q, cache, wide, n))
        assert ((got.double() - want).abs() <= tol).all()
        # the order depends on which side of four units the table is, and on no more of its width
        side = wide.shape[1] * page > 4 * unit
        assert torch.equal(got, seen.setdefault(side, got))
    assert len(seen) == 2
