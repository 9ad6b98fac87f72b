"""Latent attention against its formulas in 64 bits: the cache append, the
absorbed form over the paged cache, the expanded form over ragged prompts.

Tolerance of an attention output, u half a step of the operands' type: the
weights of the softmax may be rounded to the type before their product with
the values (u of sum p |v|), the output is rounded once (u of itself), a score
of d products summed in float32 is off by at most d 2^-23 sum |q k| (a matrix
instruction may cut off where an addition rounds), which changes a weight, and
its share of the sum, by that ratio each, and the exponential, the sums and
the joining of parts add up to 64 steps of 2^-23.  Float16 weights below the
normal range are off by 2^-25 of the largest weight at most."""

import math

import pytest

from helpers import torch_dtype

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23


def _attend(q, k, v, seen, scale, half):
    """(output, tolerance, lse) in float64 of q [t, d] over k [n, d], v [n, e]; seen [t] keys each."""
    import torch

    # a key that nobody sees keeps the reductions defined where there is no other
    q, k, v = (torch.nn.functional.pad(x.double(), (0, 0, 0, n)) for x, n in ((q, 0), (k, 1), (v, 1)))
    mask = torch.arange(k.shape[0], device=q.device)[None] < seen[:, None]
    s = (q @ k.t() * scale).masked_fill(~mask, -math.inf)
    off = (q.abs() @ k.abs().t() * abs(scale) * (q.shape[1] * STEP)).masked_fill(~mask, 0.0).amax(1, keepdim=True)
    top = s.amax(1, keepdim=True).clamp_min(-1e300)
    p = torch.exp(s - top)
    total = p.sum(1, keepdim=True)
    out = p @ v / total.clamp_min(1e-300)
    weight = p @ v.abs() / total.clamp_min(1e-300)
    tol = weight * (half * 1.01 + 2 * off + 64 * STEP) + out.abs() * half * 1.01 + 1e-30
    tol = tol + 2.0 ** -25 * (mask.double() @ v.abs()) / total.clamp_min(1e-300) * (half > 2.0 ** -12) * (half < 2.0 ** -10)
    tol = tol + 2.0 ** -25
    lse = torch.where(total[:, 0] > 0, top[:, 0] + total[:, 0].clamp_min(1e-300).log(), torch.full_like(top[:, 0], -math.inf))
    return out, tol, lse, off[:, 0] + 64 * STEP * (1 + top[:, 0].abs() + lse.abs().nan_to_num(posinf=0.0))


def _close(got, expected, tol):
    assert bool(((got.double() - expected).abs() <= tol).all()), float(((got.double() - expected).abs() - tol).max())


# ---- append -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens, rank, heads, page, norm, rope, interleaved", [
    (1, 512, 64, 64, True, True, True), (33, 128, 1, 16, True, True, False), (7, 384, 20, 32, False, True, True),
    (300, 256, 3, 48, True, False, True), (5, 512, 0, 128, False, False, False),
])
def test_append_matches_the_formula(dtype, tokens, rank, heads, page, norm, rope, interleaved):
    import torch

    from mlxlr8_b200.latent import latent_append, rope_table

    g = torch.Generator(device="cuda").manual_seed(tokens + rank)
    td = torch_dtype(dtype)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(td)

    kv, cache = normal(tokens, rank + 64), normal(40, page, rank + 64)
    joint = normal(tokens, max(heads, 1), 192)
    q = joint[..., 128:] if heads else None
    slots = torch.randperm(40 * page, generator=g, device="cuda")[:tokens]
    if tokens > 4:
        slots[1], slots[3] = -1, 40 * page
    w = (1 + 0.1 * torch.randn(rank, generator=g, device="cuda")).to(td) if norm else None
    table = rope_table(900) if rope else None
    at = torch.randint(0, 900, (tokens,), generator=g, device="cuda", dtype=torch.int32) if rope else None
    before = cache.clone()
    got = latent_append(kv[:, :rank], kv[:, rank:], cache, slots, weight=w, cos_sin=table, positions=at, q_rope=q,
                        interleaved=interleaved)

    def rotated(v):
        v = v.double()
        if not rope:
            return v, v.abs()
        c, n = (table[at.long()][..., i].double() for i in (0, 1))
        if v.dim() == 3:
            c, n = c[:, None], n[:, None]
        a, b = (v[..., 0::2], v[..., 1::2]) if interleaved else (v[..., :32], v[..., 32:])
        x, y = a * c - b * n, a * n + b * c
        size = a.abs() + b.abs()
        if interleaved:
            return torch.stack([x, y], -1).flatten(-2), torch.stack([size, size], -1).flatten(-2)
        return torch.cat([x, y], -1), torch.cat([size, size], -1)

    latent = kv[:, :rank].double()
    if norm:
        latent = latent / (latent.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    key, size = rotated(kv[:, rank:])
    expected = before.double().view(-1, rank + 64)
    kept = (slots >= 0) & (slots < 40 * page)
    half = torch.finfo(td).eps / 2
    tol = torch.zeros_like(expected)
    expected[slots[kept]] = torch.cat([latent, key], 1)[kept]
    tol[slots[kept]] = torch.cat([latent.abs() * (half + 64 * STEP), key.abs() * half + size * 4 * STEP], 1)[kept] + 2.0 ** -25
    _close(cache.view(-1, rank + 64), expected, tol)
    if heads:
        e, size = rotated(q)
        assert got.shape == (tokens, heads, 64)
        _close(got, e, e.abs() * half + size * 4 * STEP + 2.0 ** -25)
    else:
        assert got is None


def test_append_positions_outside_the_table():
    import torch

    from mlxlr8_b200.latent import latent_append, rope_table

    cache = torch.zeros(2, 16, 192, device="cuda", dtype=torch.bfloat16)
    kv = torch.ones(4, 192, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([0, -1, 8, 7], device="cuda", dtype=torch.int32)
    q = latent_append(kv[:, :128], kv[:, 128:], cache, torch.arange(4, device="cuda"), cos_sin=rope_table(8), positions=at,
                      q_rope=kv[:, None, 128:])
    assert q.isnan().all(-1)[:, 0].tolist() == [False, True, True, False]
    assert (cache[0, :4] != 0).any(-1).tolist() == [True, False, False, True]
    assert not bool(cache.isnan().any())


def test_append_refusals():
    import torch

    from mlxlr8_b200.latent import latent_append

    cache = torch.zeros(2, 16, 576, device="cuda", dtype=torch.bfloat16)
    kv = torch.zeros(3, 576, device="cuda", dtype=torch.bfloat16)
    slots = torch.arange(3, device="cuda")
    a, b = kv[:, :512], kv[:, 512:]
    table, at = torch.zeros(4, 32, 2, device="cuda"), slots.int()
    latent_append(a[:0], b[:0], cache, slots[:0])
    for call in (lambda: latent_append(a[:, :500], b, cache, slots), lambda: latent_append(a, b[:2], cache, slots),
                 lambda: latent_append(a.half(), b, cache, slots), lambda: latent_append(a, b, cache, slots.int()),
                 lambda: latent_append(a, b, cache[:, :8], slots), lambda: latent_append(a, b, cache.float(), slots),
                 lambda: latent_append(a, b, cache[..., :500], slots), lambda: latent_append(a, b, cache[0], slots),
                 lambda: latent_append(a, b, cache, slots, weight=kv[0, :511]),
                 lambda: latent_append(a, b, cache, slots, cos_sin=table),
                 lambda: latent_append(a, b, cache, slots, positions=at),
                 lambda: latent_append(a, b, cache, slots, cos_sin=table.half(), positions=at),
                 lambda: latent_append(a, b, cache, slots, q_rope=kv[:, None, :32]),
                 lambda: latent_append(a, b, cache, slots, q_rope=b),
                 lambda: latent_append(a, b, cache.transpose(0, 1), slots),
                 lambda: latent_append(a.cpu(), b, cache, slots)):
        with pytest.raises(ValueError):
            call()


# ---- absorbed form ----------------------------------------------------------


def _paged(g, lengths, rank, page, dtype, spare=5, extra=0, garbage=None):
    """(cache, table): pages in random order; rows past a length hold ``garbage`` where given."""
    import torch

    width = max(1, -(-max(lengths + [1]) // page) + extra)
    total = len(lengths) * width + spare
    order = torch.randperm(total, generator=g, device="cuda")[: len(lengths) * width].view(-1, width).int()
    cache = torch.randn(total, page, rank + 64, generator=g, device="cuda").to(dtype)
    if garbage is not None:
        kept = torch.zeros(total, page, dtype=torch.bool, device="cuda")
        for b, n in enumerate(lengths):
            rows = order[b].long().repeat_interleave(page)[:n]
            kept[rows, torch.arange(n, device="cuda") % page] = True
        cache[~kept] = garbage
    return cache, order


def _absorbed(ql, qr, cache, table, lengths, scale, **more):
    import torch

    from mlxlr8_b200.latent import latent_attention

    got, lse = latent_attention(ql, qr, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale,
                                return_lse=True, **more)
    batch, queries, heads, rank = ql.shape
    half = torch.finfo(cache.dtype).eps / 2
    for b in range(batch):
        n = max(lengths[b], 0)
        rows = cache[table[b].long()].flatten(0, 1)[:n]
        seen = (n - queries + 1 + torch.arange(queries, device="cuda")).clamp_min(0).repeat_interleave(heads)
        q = torch.cat([ql[b], qr[b]], -1).flatten(0, 1)
        out, tol, e_lse, lse_tol = _attend(q, rows, rows[:, :rank], seen, scale, half)
        _close(got[b].flatten(0, 1), out, tol)
        empty = seen == 0
        flat = lse[b].flatten().double()
        assert bool((flat[empty] == -math.inf).all()) and bool((got[b].flatten(0, 1)[empty] == 0).all())
        _close(flat[~empty], e_lse[~empty], lse_tol[~empty])
    return got


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("lengths, queries, heads, rank, page", [
    ([1], 1, 1, 128, 16), ([1], 1, 64, 512, 64), ([0], 1, 16, 512, 64), ([129], 1, 16, 512, 64),
    ([127, 128, 129, 0, 1, 2], 1, 20, 512, 16), ([700, 3, 64], 3, 20, 512, 16), ([5, 1, 0], 4, 8, 256, 32),
    ([1500], 1, 64, 512, 64), ([260, 255], 2, 64, 384, 48), ([900, 40], 5, 33, 128, 256), ([513], 1, 128, 512, 128),
    ([4096, 17], 1, 64, 512, 64), ([300], 40, 7, 512, 64), ([20000], 1, 16, 512, 64),
])
def test_absorbed_matches_the_formula(dtype, lengths, queries, heads, rank, page):
    import torch

    g = torch.Generator(device="cuda").manual_seed(sum(lengths) + heads)
    td = torch_dtype(dtype)
    cache, table = _paged(g, lengths, rank, page, td)
    ql = torch.randn(len(lengths), queries, heads, rank, generator=g, device="cuda").to(td)
    qr = torch.randn(len(lengths), queries, heads, 64, generator=g, device="cuda").to(td)
    _absorbed(ql, qr, cache, table, lengths, 2.0 * (rank + 64) ** -0.5)


@pytest.mark.parametrize("lengths, queries, heads, rank, page", [
    ([7000, 1, 0, 64, 9000, 4500, 130], 2, 40, 128, 64), ([500 + 7 * i for i in range(70)], 1, 64, 128, 16),
    ([3000] * 20 + [0, 1] * 9, 1, 16, 256, 48), ([65] * 160, 3, 48, 128, 80), ([200] * 150, 1, 8, 384, 32),
])
def test_absorbed_shares_of_many_segments(lengths, queries, heads, rank, page):
    """Enough tiles that the segments' own cost is evened out over the CTAs:
    shares that begin and end inside, between and behind sequences."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(sum(lengths) + heads)
    cache, table = _paged(g, lengths, rank, page, torch.bfloat16, garbage=float("nan"))
    ql = torch.randn(len(lengths), queries, heads, rank, generator=g, device="cuda").bfloat16()
    qr = torch.randn(len(lengths), queries, heads, 64, generator=g, device="cuda").bfloat16()
    scale = 2.0 * (rank + 64) ** -0.5
    got = _absorbed(ql, qr, cache, table, lengths, scale)
    assert torch.equal(_absorbed(ql, qr, cache, table, lengths, scale), got)


@pytest.mark.parametrize("garbage", [float("nan"), float("inf"), -3e38])
def test_absorbed_ignores_what_lies_past_a_length(garbage):
    import torch

    g = torch.Generator(device="cuda").manual_seed(77)
    lengths = [1, 15, 16, 17, 130, 0, 250]
    for dtype in (torch.bfloat16, torch.float16):
        cache, table = _paged(g, lengths, 512, 32, dtype, extra=2, garbage=garbage)
        ql = torch.randn(7, 2, 10, 512, generator=g, device="cuda").to(dtype)
        qr = torch.randn(7, 2, 10, 64, generator=g, device="cuda").to(dtype)
        got = _absorbed(ql, qr, cache, table, lengths, 0.05)
        assert bool(got.isfinite().all())


def test_absorbed_scores_of_every_size():
    """Sharp and flat softmax, rising and falling scores, negative scales: the
    running maximum moves late, early and often."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(78)
    n = 1100
    for dtype in (torch.bfloat16, torch.float16):
        cache, table = _paged(g, [n], 256, 64, dtype)
        flat = table[0].long().repeat_interleave(64)[:n], torch.arange(n, device="cuda") % 64
        ramp = torch.linspace(-6, 6, n, device="cuda")
        for order in (ramp, ramp.flip(0), ramp[torch.randperm(n, generator=g, device="cuda")]):
            cache[flat[0], flat[1], 0] = order.to(dtype)
            ql = torch.randn(1, 1, 24, 256, generator=g, device="cuda")
            ql[..., 0] = 8.0
            qr = torch.randn(1, 1, 24, 64, generator=g, device="cuda")
            for scale in (1.0, -1.0, 0.001, 0.0):
                _absorbed(ql.to(dtype), qr.to(dtype), cache, table, [n], scale)


def test_absorbed_tables_with_pages_outside_the_cache():
    """An entry outside the cache holds no tokens; a length past the table's
    room counts as the room; a negative length as none."""
    import torch

    from mlxlr8_b200.latent import latent_attention

    g = torch.Generator(device="cuda").manual_seed(79)
    cache, table = _paged(g, [256, 256, 256], 512, 64, torch.bfloat16)
    ql = torch.randn(3, 1, 16, 512, generator=g, device="cuda").bfloat16()
    qr = torch.randn(3, 1, 16, 64, generator=g, device="cuda").bfloat16()
    lengths = torch.tensor([256, 100000, -5], dtype=torch.int32, device="cuda")
    broken = table.clone()
    broken[0, 1], broken[0, 3] = -1, cache.shape[0]
    got = latent_attention(ql, qr, cache, broken, lengths, 0.05)
    rows = torch.cat([cache[table[0, 0].long()], cache[table[0, 2].long()]])
    half = torch.finfo(torch.bfloat16).eps / 2
    seen = torch.full((16,), 128, device="cuda")
    out, tol, _, _ = _attend(torch.cat([ql[0, 0], qr[0, 0]], -1), rows, rows[:, :512], seen, 0.05, half)
    _close(got[0, 0], out, tol)
    full = latent_attention(ql, qr, cache, table, torch.full_like(lengths, 256), 0.05)
    assert torch.equal(got[1], full[1]) and bool((got[2] == 0).all())
    broken[0] = 1 << 30
    assert bool((latent_attention(ql, qr, cache, broken, lengths, 0.05)[0] == 0).all())
    assert bool((latent_attention(ql, qr, cache, table[:, :0], lengths, 0.05) == 0).all())


def test_absorbed_parts_join_by_their_lse():
    import torch

    from mlxlr8_b200.latent import latent_attention

    g = torch.Generator(device="cuda").manual_seed(80)
    cache, table = _paged(g, [512], 512, 64, torch.float16)
    ql = torch.randn(1, 1, 32, 512, generator=g, device="cuda").half()
    qr = torch.randn(1, 1, 32, 64, generator=g, device="cuda").half()

    def part(t, n):
        o, lse = latent_attention(ql, qr, cache, t.contiguous(), torch.tensor([n], dtype=torch.int32, device="cuda"), 0.08,
                                  return_lse=True)
        return o.double(), lse.double()

    (a, la), (b, lb), (whole, lw) = part(table[:, :3], 192), part(table[:, 3:], 320), part(table, 512)
    both = torch.logaddexp(la, lb)
    joined = a * (la - both).exp()[..., None] + b * (lb - both).exp()[..., None]
    assert float((both - lw).abs().max()) < 1e-4
    assert float((joined - whole).abs().max()) < 4 * 2.0 ** -11 * float(whole.abs().max())


def test_absorbed_same_bits_on_streams_replays_and_shared_graphs():
    import torch

    from mlxlr8_b200 import _lib
    from mlxlr8_b200.latent import latent_attention

    g = torch.Generator(device="cuda").manual_seed(81)
    lengths = torch.tensor([3000, 70], dtype=torch.int32, device="cuda")
    cache, table = _paged(g, [3000, 70], 512, 64, torch.bfloat16)
    ql = torch.randn(2, 1, 64, 512, generator=g, device="cuda").bfloat16()
    qr = torch.randn(2, 1, 64, 64, generator=g, device="cuda").bfloat16()
    first = latent_attention(ql, qr, cache, table, lengths, 0.05)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(latent_attention(ql, qr, cache, table, lengths, 0.05), first)
    side.synchronize()
    # two graphs over one workspace, one after the other; the lengths change between replays
    ws = torch.full((_lib.lib().exlr8_latent_attention_workspace(2, 1, 64, 512) + 256,), 255, dtype=torch.uint8,
                    device="cuda")
    outs, graphs = [torch.empty_like(ql) for _ in range(2)], []
    for out in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            latent_attention(ql, qr, cache, table, lengths, 0.05, out=out, workspace=ws)
        graphs.append(graph)
    for n in (3000, 129, 0, 2999, 3000):
        lengths[0] = n
        expected = latent_attention(ql, qr, cache, table, lengths, 0.05)
        for graph, out in zip(graphs, outs):
            graph.replay()
            assert torch.equal(out, expected)
    assert torch.equal(outs[1], first)


def test_absorbed_rows_far_behind_2_to_the_31st_byte():
    """Page numbers whose rows lie past 4 GB of the cache."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(82)
    pages = (5 << 30) // (64 * 576 * 2)
    cache = torch.zeros(pages, 64, 576, device="cuda", dtype=torch.bfloat16)
    table = torch.tensor([[pages - 1, 3, pages - 2, pages // 2]], device="cuda", dtype=torch.int32)
    cache[table[0].long()] = torch.randn(4, 64, 576, generator=g, device="cuda").bfloat16()
    ql = torch.randn(1, 1, 16, 512, generator=g, device="cuda").bfloat16()
    qr = torch.randn(1, 1, 16, 64, generator=g, device="cuda").bfloat16()
    _absorbed(ql, qr, cache, table, [250], 0.05)


def test_absorbed_refusals():
    import torch

    from mlxlr8_b200.latent import latent_attention

    cache = torch.zeros(4, 16, 576, device="cuda", dtype=torch.bfloat16)
    table = torch.zeros(2, 2, device="cuda", dtype=torch.int32)
    lengths = torch.ones(2, device="cuda", dtype=torch.int32)
    ql, qr = (torch.zeros(2, 1, 8, n, device="cuda", dtype=torch.bfloat16) for n in (512, 64))
    assert latent_attention(ql[:0], qr[:0], cache, table[:0], lengths[:0], 1.0).shape == (0, 1, 8, 512)
    for call in (lambda: latent_attention(ql, qr[..., :32], cache, table, lengths, 1.0),
                 lambda: latent_attention(ql.half(), qr, cache, table, lengths, 1.0),
                 lambda: latent_attention(ql, qr, cache, table.long(), lengths, 1.0),
                 lambda: latent_attention(ql, qr, cache, table[:1], lengths, 1.0),
                 lambda: latent_attention(ql, qr, cache, table, lengths[:1], 1.0),
                 lambda: latent_attention(ql, qr, cache, table, lengths, float("nan")),
                 lambda: latent_attention(ql[:, :0], qr[:, :0], cache, table, lengths, 1.0),
                 lambda: latent_attention(ql[0], qr[0], cache, table, lengths, 1.0),
                 lambda: latent_attention(ql, qr, cache[..., :560], table, lengths, 1.0),
                 lambda: latent_attention(ql, qr, cache, table, lengths, 1.0, out=ql[..., :256]),
                 lambda: latent_attention(ql, qr, cache, table, lengths, 1.0, out=ql),
                 lambda: latent_attention(ql, qr, cache, table, lengths, 1.0,
                                          out=cache.view(-1)[:8192].view(2, 1, 8, 512)),
                 lambda: latent_attention(ql, qr, cache, table, lengths, 1.0,
                                          workspace=torch.empty(1 << 26, 2, device="cuda", dtype=torch.uint8)[:, 0]),
                 lambda: latent_attention(ql, qr, cache, table.cpu(), lengths, 1.0)):
        with pytest.raises((ValueError, RuntimeError)):
            call()


# ---- expanded form ------------------------------------------------------------


def _prompt(q, k, kr, v, queries, keys, scale, **more):
    import torch

    from mlxlr8_b200.latent import latent_prompt_attention

    def starts(n):
        return torch.tensor([0] + list(torch.tensor(n).cumsum(0)), dtype=torch.int32, device="cuda")

    got, lse = latent_prompt_attention(q, k, kr, v, starts(queries), starts(keys), scale, return_lse=True, **more)
    half = torch.finfo(q.dtype).eps / 2
    a = c = 0
    for n, m in zip(queries, keys):
        seen = (m - n + 1 + torch.arange(n, device="cuda")).clamp_min(0)
        for h in range(q.shape[1]):
            key = torch.cat([k[c:c + m, h], kr[c:c + m]], 1)
            out, tol, e_lse, lse_tol = _attend(q[a:a + n, h], key, v[c:c + m, h], seen, scale, half)
            _close(got[a:a + n, h], out, tol)
            flat, empty = lse[a:a + n, h].double(), seen == 0
            assert bool((flat[empty] == -math.inf).all()) and bool((got[a:a + n, h][empty] == 0).all())
            _close(flat[~empty], e_lse[~empty], lse_tol[~empty])
        a, c = a + n, c + m
    return got


def _operands(g, queries, keys, heads, nope, value, dtype):
    import torch

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    return (normal(sum(queries), heads, nope + 64), normal(sum(keys), heads, nope), normal(sum(keys), 64),
            normal(sum(keys), heads, value))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("queries, keys, heads, nope, value", [
    ([1], [1], 1, 64, 64), ([1], [300], 3, 128, 128), ([129], [129], 2, 128, 128), ([128, 127], [128, 127], 2, 192, 256),
    ([64, 0, 65, 1], [64, 7, 200, 1], 3, 64, 128), ([300], [300], 1, 128, 256), ([257], [700], 2, 192, 192),
    ([100, 30], [60, 0], 2, 128, 128), ([5, 700, 33], [5, 700, 500], 4, 128, 128), ([520], [520], 2, 64, 256),
    ([385], [513], 1, 192, 64),
])
def test_prompt_matches_the_formula(dtype, queries, keys, heads, nope, value):
    import torch

    g = torch.Generator(device="cuda").manual_seed(sum(queries) + sum(keys) + nope)
    td = torch_dtype(dtype)
    _prompt(*_operands(g, queries, keys, heads, nope, value, td), queries, keys, 1.5 * (nope + 64) ** -0.5)


def test_prompt_scores_of_every_size():
    import torch

    g = torch.Generator(device="cuda").manual_seed(90)
    for dtype in (torch.bfloat16, torch.float16):
        q, k, kr, v = _operands(g, [700], [700], 2, 128, 128, dtype)
        ramp = torch.linspace(-6, 6, 700, device="cuda")
        for order in (ramp, ramp.flip(0), ramp[torch.randperm(700, generator=g, device="cuda")]):
            k[:, :, 0] = order.to(dtype)[:, None]
            q[..., 0] = 8.0
            for scale in (1.0, -1.0, 0.001, 0.0):
                _prompt(q, k, kr, v, [700], [700], scale)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("queries, keys, heads, nope, value", [
    ([165], [2165], 3, 192, 256), ([900], [900], 4, 64, 64), ([5, 260, 0], [1900, 2260, 900], 2, 128, 192),
    ([40], [1200], 1, 128, 128), ([700], [600], 1, 128, 64), ([256, 1], [2050, 1], 2, 64, 128),
])
def test_prompt_with_keys_shared_by_several_ctas(dtype, queries, keys, heads, nope, value):
    """Few tiles of queries and many keys: two, four or eight CTAs to a tile."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(sum(queries) + heads)
    q, k, kr, v = _operands(g, queries, keys, heads, nope, value, torch_dtype(dtype))
    got = _prompt(q, k, kr, v, queries, keys, 1.5 * (nope + 64) ** -0.5)
    # a score that outgrows all before it, in the last share and in the first
    for at in (0, keys[0] - queries[0]):
        if at >= 0:
            k2 = k.clone()
            k2[at] *= 30.0
            _prompt(q, k2, kr, v, queries, keys, 0.2)
    assert torch.equal(_prompt(q, k, kr, v, queries, keys, 1.5 * (nope + 64) ** -0.5), got)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("queries, keys, heads, nope, value", [
    ([128], [640], 2, 128, 128), ([17, 100], [700, 900], 2, 192, 192), ([1, 1, 1], [129, 256, 2000], 3, 64, 256),
    ([384, 60], [384, 60], 30, 64, 64),
])
def test_prompt_lone_tiles_of_queries(dtype, queries, keys, heads, nope, value):
    """At most 128 queries in a tile of 256: its keys go to two groups in turn,
    whose maxima differ with rising, falling and mixed scores."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(sum(keys) + heads)
    q, k, kr, v = _operands(g, queries, keys, heads, nope, value, torch_dtype(dtype))
    _prompt(q, k, kr, v, queries, keys, 1.5 * (nope + 64) ** -0.5)
    n = sum(keys)
    q[..., 0] = 8.0
    ramp = torch.linspace(-6, 6, n, device="cuda")
    for order in (ramp, ramp.flip(0), ramp[torch.randperm(n, generator=g, device="cuda")]):
        k[:, :, 0] = order.to(k.dtype)[:, None]
        _prompt(q, k, kr, v, queries, keys, 0.5)


def test_prompt_takes_views_and_leaves_other_rows():
    import torch

    g = torch.Generator(device="cuda").manual_seed(91)
    queries, keys, heads = [70, 130], [70, 260], 3
    joint = torch.randn(sum(keys) + 9, heads, 128 + 128, generator=g, device="cuda").bfloat16()
    kr = torch.randn(sum(keys) + 9, 576, generator=g, device="cuda").bfloat16()[:, 512:]
    q = torch.randn(heads, sum(queries) + 11, 192, generator=g, device="cuda").bfloat16().transpose(0, 1)
    out = torch.full((sum(queries) + 11, heads, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    # rows past the sequences may hold anything, in the operands too
    joint[sum(keys):] = float("nan")
    kr[sum(keys):] = float("inf")
    q[sum(queries):] = float("nan")
    got = _prompt(q, joint[..., :128], kr, joint[..., 128:], queries, keys, 0.1, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[sum(queries):] == 7.0).all())
    odd = torch.randn(200, heads, 193, generator=g, device="cuda").bfloat16()[..., 1:]
    one = torch.randn(330, 1, 128, generator=g, device="cuda").bfloat16().expand(330, heads, 128)
    _prompt(odd, one, kr[:330], one, queries, keys, 0.1)


def test_prompt_values_of_other_sequences_and_later_keys_do_not_leak():
    """NaN and infinite keys and values of a neighbouring sequence stay there."""
    import torch

    from mlxlr8_b200.latent import latent_prompt_attention

    g = torch.Generator(device="cuda").manual_seed(92)
    q, k, kr, v = _operands(g, [60, 50, 70], [60, 50, 70], 2, 128, 128, torch.bfloat16)
    starts = torch.tensor([0, 60, 110, 180], dtype=torch.int32, device="cuda")
    clean = latent_prompt_attention(q, k, kr, v, starts, starts, 0.1)
    for bad in (float("nan"), float("inf")):
        k2, v2 = k.clone(), v.clone()
        k2[60:110], v2[60:110] = bad, bad
        got = latent_prompt_attention(q, k2, kr, v2, starts, starts, 0.1)
        assert torch.equal(got[:60], clean[:60]) and torch.equal(got[110:], clean[110:])


def test_prompt_same_bits_on_streams_and_replays():
    import torch

    from mlxlr8_b200.latent import latent_prompt_attention

    g = torch.Generator(device="cuda").manual_seed(93)
    q, k, kr, v = _operands(g, [200, 300], [200, 800], 4, 128, 128, torch.bfloat16)
    qs = torch.tensor([0, 200, 500], dtype=torch.int32, device="cuda")
    ks = torch.tensor([0, 200, 1000], dtype=torch.int32, device="cuda")
    first = latent_prompt_attention(q, k, kr, v, qs, ks, 0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert torch.equal(latent_prompt_attention(q, k, kr, v, qs, ks, 0.1), first)
    side.synchronize()
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        latent_prompt_attention(q, k, kr, v, qs, ks, 0.1, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, first)


def test_prompt_refusals():
    import torch

    from mlxlr8_b200.latent import latent_prompt_attention

    g = torch.Generator(device="cuda").manual_seed(94)
    q, k, kr, v = _operands(g, [6], [6], 2, 128, 128, torch.float16)
    s = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    assert latent_prompt_attention(q[:0], k[:0], kr[:0], v[:0], s * 0, s * 0, 1.0).shape == (0, 2, 128)
    for call in (lambda: latent_prompt_attention(q[..., :128], k, kr, v, s, s, 1.0),
                 lambda: latent_prompt_attention(q, k.bfloat16(), kr, v, s, s, 1.0),
                 lambda: latent_prompt_attention(q, k[..., :96], kr, v, s, s, 1.0),
                 lambda: latent_prompt_attention(q, k, kr[:5], v, s, s, 1.0),
                 lambda: latent_prompt_attention(q, k, kr, v[:, :1], s, s, 1.0),
                 lambda: latent_prompt_attention(q, k, kr, v, s.long(), s, 1.0),
                 lambda: latent_prompt_attention(q, k, kr, v, s, s[:1], 1.0),
                 lambda: latent_prompt_attention(q, k, kr, v, s[:1], s[:1], 1.0),
                 lambda: latent_prompt_attention(q.float(), k.float(), kr.float(), v.float(), s, s, 1.0),
                 lambda: latent_prompt_attention(q, k, kr, v, s, s, 1.0, out=q[..., :128]),
                 lambda: latent_prompt_attention(q, k, kr, v, s, s, 1.0, out=v),
                 lambda: latent_prompt_attention(q, k, kr, v, s, s, float("inf")),
                 lambda: latent_prompt_attention(q, k, kr, v, s.cpu(), s, 1.0)):
        with pytest.raises((ValueError, RuntimeError)):
            call()


def test_prompt_starts_outside_the_operands():
    """Starts past either end count as that end; descending ones hold no query."""
    import torch

    from mlxlr8_b200.latent import latent_prompt_attention

    g = torch.Generator(device="cuda").manual_seed(95)
    q, k, kr, v = _operands(g, [300], [300], 2, 128, 128, torch.bfloat16)
    low, high = -2 ** 31, 2 ** 31 - 1

    def run(qs, ks):
        qs, ks = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (qs, ks))
        out = torch.full((300, 2, 128), 7.0, device="cuda").bfloat16()
        return latent_prompt_attention(q, k, kr, v, qs, ks, 0.1, out=out)

    whole = run([0, 300], [0, 300])
    assert torch.equal(run([low, high], [low, high]), whole)
    assert torch.equal(run([0, 300, high, low, -5, 0], [0, 300, high, low, low, 0]), whole)
    assert bool((run([high, high], [0, 300]) == 7.0).all()) and bool((run([300, 0], [0, 300]) == 7.0).all())


def test_absorbed_many_short_sequences():
    """More sequences than CTAs, most of them empty or of one token."""
    import torch

    from mlxlr8_b200.latent import latent_attention

    g = torch.Generator(device="cuda").manual_seed(96)
    batch, heads, rank = 5003, 2, 128
    cache = torch.randn(64, 16, rank + 64, generator=g, device="cuda").bfloat16()
    ql, qr = (torch.randn(batch, 1, heads, n, generator=g, device="cuda").bfloat16() for n in (rank, 64))
    table = torch.randint(0, 64, (batch, 2), generator=g, device="cuda", dtype=torch.int32)
    lengths = torch.tensor([0, 1, 0, 17, 1], device="cuda", dtype=torch.int32).repeat(1001)[:batch]
    lengths[-1] = 32
    got = latent_attention(ql, qr, cache, table, lengths, 0.1)
    rows = cache[table.long()].view(batch, 32, rank + 64).double()
    s = torch.einsum("bhd,bnd->bhn", torch.cat([ql, qr], -1)[:, 0].double(), rows) * 0.1
    mask = torch.arange(32, device="cuda") < lengths[:, None]
    p = torch.softmax(s.masked_fill(~mask[:, None], -1e300), -1) * (lengths > 0)[:, None, None]
    rows = rows[..., :rank]
    half = 2.0 ** -8  # rounded weights, rounded output; scores and sums in float32 are far below
    expected, weight = (torch.einsum("bhn,bnd->bhd", p, r) for r in (rows, rows.abs()))
    _close(got[:, 0], expected, 1.02 * half * (weight + expected.abs()) + 2.0 ** -25)


def test_attention_forms_side_by_side_on_two_streams():
    """Calls that overlap on the GPU, each with its own workspace."""
    import torch

    from mlxlr8_b200.latent import latent_attention, latent_prompt_attention

    g = torch.Generator(device="cuda").manual_seed(97)
    q, k, kr, v = _operands(g, [165], [2165], 4, 128, 128, torch.bfloat16)
    qs, ks = (torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (165, 2165))
    cache, table = _paged(g, [5000, 900], 512, 64, torch.bfloat16)
    lengths = torch.tensor([5000, 900], dtype=torch.int32, device="cuda")
    ql, qr = (torch.randn(2, 1, 64, n, generator=g, device="cuda").bfloat16() for n in (512, 64))

    def prompt():
        return latent_prompt_attention(q, k, kr, v, qs, ks, 0.1)

    def absorbed():
        return latent_attention(ql, qr, cache, table, lengths, 0.05)

    first = prompt(), absorbed()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for stream, call in zip(streams, (prompt, absorbed, absorbed)):
            with torch.cuda.stream(stream):
                got.append((call is absorbed, call()))
    torch.cuda.synchronize()
    assert all(torch.equal(out, first[which]) for which, out in got)


def test_many_calls_of_both_forms_repeat_their_bits():
    """Several segments a CTA, clusters whose rows are no multiple of a warp,
    lone tiles: call after call."""
    import torch

    from mlxlr8_b200.latent import latent_attention, latent_prompt_attention

    g = torch.Generator(device="cuda").manual_seed(100)
    calls = []
    for queries, keys in (([165], [2165]), ([17, 100], [700, 900]), ([300, 1, 40], [300, 129, 500])):
        operands = _operands(g, queries, keys, 3, 128, 192, torch.bfloat16)
        starts = [torch.tensor([0] + list(torch.tensor(n).cumsum(0)), dtype=torch.int32, device="cuda") for n in (queries, keys)]
        calls.append(lambda o=operands, s=starts: latent_prompt_attention(*o, *s, 0.1))
    for lengths in ([3000, 70, 0, 1], [200 + i for i in range(200)]):
        cache, table = _paged(g, lengths, 256, 16, torch.bfloat16)
        ql, qr = (torch.randn(len(lengths), 2, 24, n, generator=g, device="cuda").bfloat16() for n in (256, 64))
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        calls.append(lambda a=(ql, qr, cache, table, n): latent_attention(*a, 0.05))
    first = [call() for call in calls]
    assert all(bool(out.isfinite().all()) for out in first)
    for _ in range(60):
        assert all(torch.equal(call(), out) for call, out in zip(calls, first))


# ---- append without rotation, and views that no vector load fits -------------------


@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("interleaved", [True, False])
def test_append_without_a_table_copies_what_it_is_given(offset, interleaved):
    """Infinities, NaN and signed zeros of a key and of queries stay in their channel."""
    import torch

    from mlxlr8_b200.latent import latent_append

    g = torch.Generator(device="cuda").manual_seed(98)
    for dtype in (torch.bfloat16, torch.float16):
        kv = torch.randn(5, 192 + offset, generator=g, device="cuda").to(dtype)[:, offset:]
        q = torch.randn(5, 3, 64 + offset, generator=g, device="cuda").to(dtype)[..., offset:]
        for at, value in ((0, math.inf), (7, -math.inf), (33, math.nan), (40, 0.0), (41, -0.0)):
            kv[:, 128 + at], kv[:, at], q[..., at] = value, value, value
        cache = torch.zeros(1, 16, 192, device="cuda", dtype=dtype)
        got = latent_append(kv[:, :128], kv[:, 128:], cache, torch.arange(5, device="cuda"), q_rope=q,
                            interleaved=interleaved)
        for copy, given in ((cache[0, :5], kv), (got, q)):
            assert torch.equal(copy.isnan(), given.isnan())
            kept = ~given.isnan()
            assert torch.equal(copy[kept].view(torch.int16), given[kept].view(torch.int16))
        assert not bool(cache[0, 5:].any())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens, rank, heads, norm, rope, interleaved, odd", [
    (1, 512, 64, True, True, True, "latent"), (33, 128, 1, True, True, False, "key"), (70, 384, 20, False, True, True, "head"),
    (300, 256, 3, True, False, True, "latent"), (5, 512, 0, True, True, False, "weight"), (9, 256, 5, True, True, False, "token"),
    (12, 128, 40, False, False, False, "key"), (8, 512, 7, True, True, True, "table"),
])
def test_append_of_unaligned_views_matches_the_formula(dtype, tokens, rank, heads, norm, rope, interleaved, odd):
    """One operand off its 16 bytes, or with rows that are."""
    import torch

    from mlxlr8_b200.latent import latent_append, rope_table

    g = torch.Generator(device="cuda").manual_seed(tokens + rank + heads)
    td = torch_dtype(dtype)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(td)

    latent = normal(tokens, rank + 9)[:, 1 : 1 + rank] if odd == "latent" else normal(tokens, rank)
    key = normal(tokens + 1, 65)[1:, :64] if odd == "key" else normal(tokens, 64)
    q = None
    if heads:
        q = {"head": lambda: normal(tokens, heads, 67)[..., :64],
             "token": lambda: normal(tokens, heads * 64 + 2)[:, 2:].view(tokens, heads, 64)}.get(
                 odd, lambda: normal(heads, tokens, 64).transpose(0, 1))()
    flat = (1 + 0.1 * torch.randn(rank + 1, generator=g, device="cuda")).to(td)
    w = (flat[1:] if odd == "weight" else flat[:rank]) if norm else None
    table = None
    if rope:
        table = rope_table(901)[1:].contiguous()
        if odd == "table":
            shifted = torch.empty(table.numel() + 1, device="cuda")
            shifted[1:] = table.flatten()
            table = shifted[1:].view(table.shape)
    cache = normal(40, 16, rank + 64)
    slots = torch.randperm(640, generator=g, device="cuda")[:tokens]
    at = torch.randint(0, 900, (tokens,), generator=g, device="cuda", dtype=torch.int32) if rope else None
    if tokens > 4:
        slots[1], slots[3] = -1, 640
        if rope:
            at[2], at[0] = -1, 900
    before = cache.clone()
    got = latent_append(latent, key, cache, slots, weight=w, cos_sin=table, positions=at, q_rope=q, interleaved=interleaved)
    known = (at >= 0) & (at < 900) if rope else torch.ones(tokens, dtype=torch.bool, device="cuda")

    def rotated(v):
        v = v.double()
        if not rope:
            return v, torch.zeros_like(v)
        cs = table[at.long().clamp(0, 899)].double()
        c, n = (cs[..., i].reshape((tokens,) + (1,) * (v.dim() - 2) + (32,)) for i in (0, 1))
        a, b = (v[..., 0::2], v[..., 1::2]) if interleaved else (v[..., :32], v[..., 32:])
        size = a.abs() + b.abs()

        def back(x, y):
            return torch.stack([x, y], -1).flatten(-2) if interleaved else torch.cat([x, y], -1)

        return back(a * c - b * n, a * n + b * c), back(size, size)

    e = latent.double()
    if norm:
        e = e / (e.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    k, size = rotated(key)
    half = torch.finfo(td).eps / 2
    expected = before.double().view(-1, rank + 64)
    tol = torch.zeros_like(expected)
    kept = (slots >= 0) & (slots < 640) & known
    expected[slots[kept]] = torch.cat([e, k], 1)[kept]
    tol[slots[kept]] = torch.cat([e.abs() * (half + 64 * STEP), k.abs() * half + size * 4 * STEP], 1)[kept] + 2.0 ** -25
    _close(cache.view(-1, rank + 64), expected, tol)
    if heads:
        e, size = rotated(q)
        assert got.is_contiguous() and bool(got[~known].isnan().all())
        _close(got[known], e[known], (e.abs() * half + size * 4 * STEP + 2.0 ** -25)[known])


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_absorbed_queries_that_see_nothing_beside_a_token_that_is_not_finite(bad):
    """Zeros, whole and joined from parts, whatever the cache holds."""
    import torch

    from mlxlr8_b200.latent import latent_attention

    g = torch.Generator(device="cuda").manual_seed(99)
    for lengths, queries, heads in (([1, 2, 40], 4, 10), ([70], 90, 16), ([1, 300], 5, 40), ([150], 200, 3)):
        cache, table = _paged(g, lengths, 512, 16, torch.bfloat16)
        for b in range(len(lengths)):
            cache[table[b, 0].long(), 0] = bad
        batch = len(lengths)
        ql, qr = (torch.randn(batch, queries, heads, n, generator=g, device="cuda").bfloat16() for n in (512, 64))
        got, lse = latent_attention(ql, qr, cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 0.05,
                                    return_lse=True)
        for b, n in enumerate(lengths):
            none = max(queries - n, 0)
            assert bool((got[b, :none] == 0).all()) and bool((lse[b, :none] == -math.inf).all())
            assert bool(got[b, none:].isnan().all())


def test_caches_and_workspaces_over_other_operands_are_refused():
    import torch

    from mlxlr8_b200.latent import latent_append, latent_attention

    cache = torch.zeros(4, 16, 576, device="cuda", dtype=torch.bfloat16)
    rows = cache.view(64, 576)
    kv = torch.ones(3, 576, device="cuda", dtype=torch.bfloat16)
    slots = torch.arange(3, device="cuda")
    for call in (lambda: latent_append(rows[8:11, :512], kv[:, 512:], cache, slots),
                 lambda: latent_append(kv[:, :512], rows[61:, 512:], cache, slots),
                 lambda: latent_append(kv[:, :512], kv[:, 512:], cache, slots, weight=rows[0, :512]),
                 lambda: latent_append(kv[:, :512], kv[:, 512:], cache, slots, q_rope=rows[:3, None, :64])):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    assert not bool(cache.any())
    table, lengths = (torch.zeros(n, device="cuda", dtype=torch.int32) for n in ((2, 2), (2,)))
    ql, qr = (torch.zeros(2, 1, 8, n, device="cuda", dtype=torch.bfloat16) for n in (512, 64))
    big = torch.zeros(64 << 20, device="cuda", dtype=torch.uint8)
    half = big[: 4 * 16 * 576 * 2].view(torch.bfloat16).view(4, 16, 576)
    out = big[: 2 * 8 * 512 * 2].view(torch.bfloat16).view(2, 1, 8, 512)
    for more in (dict(cache=half), dict(cache=cache, out=out)):
        with pytest.raises(ValueError, match="overlaps"):
            latent_attention(ql, qr, more.pop("cache"), table, lengths, 1.0, workspace=big, **more)
