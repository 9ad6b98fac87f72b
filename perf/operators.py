"""Cases, plain forms and 64-bit values of the operators of a decoder block's attention half.

Five operators of ``mlxlr8_b200``: the residual add + RMS norm with an 8-bit
output, the linear layer with 4-bit weights and group scales, the write into
the paged latent cache (rotary embedding, latent norm), attention over that
cache (absorbed form) and attention over expanded keys and values (prompts).
``own`` selects the framework's calls; otherwise ``run`` is elementary torch
arithmetic in float32, rounded once at the end.
"""

import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # one token of a decoding user, between two blocks of the stack
        dict(name="norm8 token", op="norm8", rows=1, hidden=6144, group=128, dtype="bf16", residual=True),
        # a chunk of a prompt in front of 8-bit products
        dict(name="norm8 prompt", op="norm8", rows=8192, hidden=6144, group=128, dtype="bf16", residual=True),
        # a narrow projection for one token: latency counts
        dict(name="linear4 narrow", op="linear4", rows=1, inner=6144, outer=576, group=64, dtype="bf16", scales="bf16",
             biases=True, x_group=0),
        # a wide projection for one token, weights of a 16-bit float checkpoint
        dict(name="linear4 wide", op="linear4", rows=1, inner=16384, outer=6144, group=128, dtype="f16", scales="f16",
             biases=True, x_group=0),
        # eight users' tokens from the 8-bit norm into the widest projection
        dict(name="linear4 batch", op="linear4", rows=8, inner=6144, outer=36864, group=128, dtype="bf16",
             scales="f16", biases=False, x_group=128),
        # a decode step of a batch: one token of each user enters the cache
        dict(name="append step", op="append", tokens=32, heads=64, rank=512, page=64, pages=512, dtype="bf16",
             norm=True, interleaved=True),
        # a prompt chunk enters the cache
        dict(name="append prompt", op="append", tokens=8192, heads=64, rank=512, page=64, pages=512, dtype="bf16",
             norm=True, interleaved=True),
        # one user, a long conversation: the split over the cache's length has to fill the GPU
        dict(name="absorbed one user", op="absorbed", batch=1, queries=1, heads=64, rank=512, longest=16000, page=64,
             dtype="bf16"),
        # verification of two drafted tokens for a few short conversations
        dict(name="absorbed draft", op="absorbed", batch=5, queries=3, heads=20, rank=512, longest=700, page=16,
             dtype="f16"),
        # a full decode batch with long contexts
        dict(name="absorbed batch", op="absorbed", batch=64, queries=1, heads=64, rank=512, longest=12000, page=64,
             dtype="bf16"),
        # short prompts of several users, one of them with a history
        dict(name="prompt ragged", op="prompt", seqs=5, total=1300, history=500, heads=16, nope=128, value=128,
             dtype="f16"),
        # one long prompt
        dict(name="prompt long", op="prompt", seqs=1, total=8192, history=0, heads=32, nope=128, value=128,
             dtype="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm8", "linear4", "linear4", "append", "absorbed", "absorbed", "prompt", "prompt"])
    if op == "norm8":
        group = rng.choice([32, 64, 128, 0])
        hidden = _spread(rng, 2, 64) * 128 if group else _spread(rng, 200, 8000)
        return dict(op=op, rows=_spread(rng, 1, 6000), hidden=hidden, group=group,
                    dtype=rng.choice(["f32", "f16", "bf16"]), residual=rng.random() < 0.7)
    if op == "linear4":
        group = rng.choice([32, 64, 128])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        inner = _spread(rng, 512 // group, 16384 // group) * group
        outer = _spread(rng, 100, 12000)
        x_group = rng.choice([0, 0, group, -1]) if dtype != "f32" else 0
        return dict(op=op, rows=_spread(rng, 1, 40), inner=inner, outer=outer, group=group, dtype=dtype,
                    scales=rng.choice(["f16", "bf16", "f32"]), biases=rng.random() < 0.6, x_group=x_group)
    if op == "append":
        return dict(op=op, tokens=_spread(rng, 1, 6000), heads=rng.choice([1, 8, 16, 20, 32, 64]),
                    rank=rng.choice([128, 256, 384, 512]), page=rng.choice([16, 32, 64, 128]), pages=600,
                    dtype=rng.choice(["bf16", "f16"]), norm=rng.random() < 0.7, interleaved=rng.random() < 0.5)
    if op == "absorbed":
        batch = _spread(rng, 1, 60)
        return dict(op=op, batch=batch, queries=rng.choice([1, 1, 1, 2, 3, 5]),
                    heads=rng.choice([4, 8, 16, 20, 32, 48, 64]), rank=rng.choice([128, 256, 384, 512, 512, 512]),
                    longest=_spread(rng, 1, 6000 if batch > 8 else 30000), page=rng.choice([16, 32, 64, 128, 256, 48]),
                    dtype=rng.choice(["bf16", "f16"]))
    total = _spread(rng, 40, 6000)
    return dict(op=op, seqs=rng.choice([1, 1, 2, 3, 6]), total=total, history=rng.choice([0, 0, 100, 2000]),
                heads=rng.choice([4, 8, 12, 16, 24]), nope=rng.choice([64, 128, 192]),
                value=rng.choice([64, 128, 192, 256]), dtype=rng.choice(["bf16", "f16"]))


ROPE = 64


def _fixed(case):
    """Random numbers that the case alone decides (lengths: the work depends on them)."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _cache_lengths(case):
    """Ragged lengths up to the longest; one sequence of a larger batch has nothing cached yet."""
    rng, longest = _fixed(case), case["longest"]
    lengths = [longest] + [rng.randint((longest + 1) // 2, longest) for _ in range(case["batch"] - 1)]
    if case["batch"] >= 10:
        lengths[rng.randrange(1, case["batch"])] = 0
    return lengths


def _prompt_lengths(case):
    """Queries of each sequence (their sum is the total; one of six sequences has none) and keys."""
    rng, n, total = _fixed(case), case["seqs"], case["total"]
    cuts = sorted(rng.randint(0, total) for _ in range(n - 1))
    queries = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    if n >= 6:
        queries[0], queries[1] = 0, queries[0] + queries[1]
    keys = [q + (case["history"] if i % 2 == 0 else 0) for i, q in enumerate(queries)]
    return queries, keys


def _starts(lengths, device):
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    return torch.tensor(ends, dtype=torch.int32, device=device)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype)

    op, t = case["op"], DTYPES[case["dtype"]]
    if op == "norm8":
        rows, hidden = case["rows"], case["hidden"]
        x = normal(rows, hidden)
        x[:, :: max(1, hidden // 7)] *= 20.0  # a residual stream has a few channels far above the others
        return dict(op=op, x=x.to(t), r=normal(rows, hidden, dtype=t) if case["residual"] else None,
                    w=(1.0 + 0.1 * normal(hidden)).to(t), group=case["group"] or hidden)
    if op == "linear4":
        rows, inner, outer, group = case["rows"], case["inner"], case["outer"], case["group"]
        ts = DTYPES[case["scales"]]
        codes = torch.randint(-(1 << 31), 1 << 31, (outer, inner // 8), generator=g, device=device, dtype=torch.int32)
        scales = ((0.5 + torch.rand(outer, inner // group, generator=g, device=device)) * 0.01).to(ts)
        biases = (-7.5 * scales.float() + normal(outer, inner // group, scale=0.002)).to(ts) if case["biases"] else None
        x, x_scales = normal(rows, inner), None
        if case["x_group"]:
            xg = case["x_group"] if case["x_group"] > 0 else inner
            blocks = x.view(rows, inner // xg, xg)
            x_scales = blocks.abs().amax(-1) / 448.0
            x = (blocks / x_scales[..., None]).reshape(rows, inner).to(torch.float8_e4m3fn)
        else:
            x = x.to(t)
        return dict(op=op, x=x, x_scales=x_scales, codes=codes, scales=scales, biases=biases, out=t)
    if op == "append":
        n, heads, rank, page, pages = case["tokens"], case["heads"], case["rank"], case["page"], case["pages"]
        kv = normal(n, rank + ROPE, dtype=t)
        slots = torch.randperm(page * pages, generator=g, device=device)[:n]
        slots[n - 1] = -1 if n > 2 else slots[n - 1]  # a padding row of the batch: nothing is written for it
        positions = torch.randint(0, 8192, (n,), generator=g, device=device, dtype=torch.int32)
        angles = torch.arange(8192, device=device, dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(0, ROPE, 2, device=device, dtype=torch.float64) / ROPE))
        table = torch.stack([angles.cos(), angles.sin()], -1).float()
        return dict(op=op, latent=kv[:, :rank], rope_key=kv[:, rank:], cache=normal(pages, page, rank + ROPE, dtype=t),
                    slots=slots, positions=positions, cos_sin=table,
                    w=(1.0 + 0.1 * normal(rank)).to(t) if case["norm"] else None,
                    q_rope=normal(n, heads, ROPE, dtype=t), interleaved=case["interleaved"])
    if op == "absorbed":
        batch, queries, heads, rank, page = (case[k] for k in ("batch", "queries", "heads", "rank", "page"))
        lengths = _cache_lengths(case)
        width = -(-max(lengths) // page)
        total = batch * width + 3
        table = torch.randperm(total, generator=g, device=device)[:batch * width].view(batch, width).int()
        cache = torch.empty(total, page, rank + ROPE, dtype=t, device=device)
        cache.normal_(generator=g)
        return dict(op=op, ql=normal(batch, queries, heads, rank, dtype=t), qr=normal(batch, queries, heads, ROPE, dtype=t),
                    cache=cache, table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device=device),
                    scale=2.0 * (rank + ROPE) ** -0.5)
    queries, keys = _prompt_lengths(case)
    heads, nope, value = case["heads"], case["nope"], case["value"]
    return dict(op=op, q=normal(sum(queries), heads, nope + ROPE, dtype=t), k=normal(sum(keys), heads, nope, dtype=t),
                kr=normal(sum(keys), ROPE, dtype=t), v=normal(sum(keys), heads, value, dtype=t),
                q_starts=_starts(queries, device), k_starts=_starts(keys, device), scale=1.5 * (nope + ROPE) ** -0.5)


def run(s):
    return (_own if own else _plain)[s["op"]](s)


# ---- the framework's calls ---------------------------------------------------


def _own_norm8(s):
    from mlxlr8_b200.stack import residual_rms_norm_q8

    if s["r"] is None:
        return residual_rms_norm_q8(s["x"], s["w"], EPS, group=s["group"])
    return residual_rms_norm_q8(s["x"], s["w"], EPS, residual=s["r"], group=s["group"], return_sum=True)


def _own_linear4(s):
    from mlxlr8_b200.affine4 import affine4_linear

    return affine4_linear(s["x"], s["codes"], s["scales"], s["biases"], x_scales=s["x_scales"], out_dtype=s["out"])


def _own_append(s):
    from mlxlr8_b200.latent import latent_append

    q = latent_append(s["latent"], s["rope_key"], s["cache"], s["slots"], weight=s["w"], eps=EPS, cos_sin=s["cos_sin"],
                      positions=s["positions"], q_rope=s["q_rope"], interleaved=s["interleaved"])
    return q, s["cache"]


def _own_absorbed(s):
    from mlxlr8_b200.latent import latent_attention

    return latent_attention(s["ql"], s["qr"], s["cache"], s["table"], s["lengths"], s["scale"])


def _own_prompt(s):
    from mlxlr8_b200.latent import latent_prompt_attention

    return latent_prompt_attention(s["q"], s["k"], s["kr"], s["v"], s["q_starts"], s["k_starts"], s["scale"])


_own = dict(norm8=_own_norm8, linear4=_own_linear4, append=_own_append, absorbed=_own_absorbed, prompt=_own_prompt)


# ---- plain forms -------------------------------------------------------------


def _plain_norm8(s):
    x, r, group = s["x"], s["r"], s["group"]
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * s["w"].float()
    blocks = y.view(y.shape[0], -1, group)
    scales = blocks.abs().amax(-1) / 448.0
    codes = (blocks / scales[..., None].clamp_min(1e-38)).reshape(y.shape).to(torch.float8_e4m3fn)
    return (codes, scales) if r is None else (h, codes, scales)


def _plain_linear4(s):
    codes, scales, biases = s["codes"], s["scales"].float(), s["biases"]
    outer, groups = scales.shape
    nibbles = (codes[..., None] >> torch.arange(0, 32, 4, device=codes.device, dtype=torch.int32)) & 15
    q = nibbles.view(outer, groups, -1).float()
    b = -8.0 * scales if biases is None else biases.float()
    w = (q * scales[..., None] + b[..., None]).view(outer, -1)
    x = s["x"].float()
    if s["x_scales"] is not None:
        xs = s["x_scales"]
        x = (x.view(x.shape[0], xs.shape[1], -1) * xs[..., None]).view(x.shape)
    return (x @ w.t()).to(s["out"])


def _rotated(v, cs, interleaved):
    """The rotary embedding of v [..., 64] with cs [..., 32, 2], in v's precision."""
    c, n = cs[..., 0], cs[..., 1]
    if interleaved:
        a, b = v[..., 0::2], v[..., 1::2]
        return torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)
    a, b = v[..., : ROPE // 2], v[..., ROPE // 2 :]
    return torch.cat([a * c - b * n, a * n + b * c], -1)


def _plain_append(s):
    latent, cache = s["latent"].float(), s["cache"]
    if s["w"] is not None:
        latent = latent * torch.rsqrt(latent.square().mean(-1, keepdim=True) + EPS) * s["w"].float()
    cs = s["cos_sin"][s["positions"].long()]
    row = torch.cat([latent, _rotated(s["rope_key"].float(), cs, s["interleaved"])], -1).to(cache.dtype)
    flat = cache.view(-1, cache.shape[-1])
    kept = s["slots"] >= 0
    flat[s["slots"][kept]] = row[kept]
    return _rotated(s["q_rope"].float(), cs[:, None], s["interleaved"]).to(cache.dtype), cache


def _plain_absorbed(s):
    ql, cache, table, lengths = s["ql"], s["cache"], s["table"], s["lengths"]
    batch, queries, heads, rank = ql.shape
    rows = cache[table.long()].view(batch, -1, cache.shape[-1]).float()
    q = torch.cat([ql, s["qr"]], -1).float().view(batch, queries * heads, -1)
    scores = torch.matmul(q, rows.transpose(1, 2)).view(batch, queries, heads, -1) * s["scale"]
    last = lengths[:, None] - queries + 1 + torch.arange(queries, device=ql.device)
    seen = torch.arange(rows.shape[1], device=ql.device) < last[..., None]
    scores = scores.masked_fill(~seen[:, :, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return torch.matmul(p.view(batch, queries * heads, -1), rows[..., :rank]).view(ql.shape).to(ql.dtype)


def _plain_prompt(s):
    q, k, kr, v = (s[n].float() for n in ("q", "k", "kr", "v"))
    qs, ks = s["q_starts"].long(), s["k_starts"].long()
    scores = torch.matmul(q.transpose(0, 1), torch.cat([k, kr[:, None].expand(-1, k.shape[1], -1)], -1).permute(1, 2, 0))
    rows, cols = (torch.arange(n, device=q.device) for n in (q.shape[0], k.shape[0]))
    row_seq, col_seq = torch.searchsorted(qs, rows, right=True) - 1, torch.searchsorted(ks, cols, right=True) - 1
    row_at = rows - qs[row_seq] + (ks[row_seq + 1] - ks[row_seq]) - (qs[row_seq + 1] - qs[row_seq])
    seen = (row_seq[:, None] == col_seq) & (cols - ks[col_seq] <= row_at[:, None])
    scores.mul_(s["scale"]).masked_fill_(~seen, float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    scores.div_(scores.sum(-1, keepdim=True).clamp_min(1e-30))
    return torch.matmul(scores, v.transpose(0, 1)).transpose(0, 1).to(s["q"].dtype).contiguous()


_plain = dict(norm8=_plain_norm8, linear4=_plain_linear4, append=_plain_append, absorbed=_plain_absorbed,
              prompt=_plain_prompt)


# ---- work ---------------------------------------------------------------------


def work(case):
    op = case["op"]
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if op == "norm8":
        n = case["rows"] * case["hidden"]
        groups = case["hidden"] // (case["group"] or case["hidden"])
        return {"bytes": n * size * (3 if case["residual"] else 1) + n + 4 * case["rows"] * groups
                + case["hidden"] * size, "flops": 6 * n}
    if op == "linear4":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        groups = inner // case["group"]
        per = torch.finfo(DTYPES[case["scales"]]).bits // 8 * (2 if case["biases"] else 1)
        x_bytes = rows * inner * (1 if case["x_group"] else size)
        if case["x_group"]:
            x_bytes += 4 * rows * (inner // case["x_group"] if case["x_group"] > 0 else 1)
        return {"bytes": outer * (inner // 2 + groups * per) + x_bytes + rows * outer * size,
                "flops": 2 * rows * inner * outer}
    if op == "append":
        per = 2 * (case["rank"] + ROPE) + 2 * case["heads"] * ROPE
        return {"bytes": case["tokens"] * (per * size + 8 + 4 + 4 * ROPE), "flops": case["tokens"] * per * 3}
    if op == "absorbed":
        seen = sum(_cache_lengths(case))
        rows = case["queries"] * case["heads"]
        return {"bytes": seen * (case["rank"] + ROPE) * size + case["batch"] * rows * (2 * case["rank"] + ROPE) * size,
                "flops": 2 * rows * seen * (2 * case["rank"] + ROPE)}
    queries, keys = _prompt_lengths(case)
    pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(queries, keys))
    heads, nope, value = case["heads"], case["nope"], case["value"]
    return {"bytes": size * (sum(queries) * heads * (nope + ROPE + value) + sum(keys) * (heads * (nope + value) + ROPE)),
            "flops": 2 * pairs * heads * (nope + ROPE + value)}


# ---- values in 64 bits -------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm8": _exact_norm8, "linear4": _exact_linear4, "append": _exact_append, "absorbed": _exact_absorbed,
            "prompt": _exact_prompt}[case["op"]](s)


def _exact_norm8(s):
    total = s["x"].double()
    if s["r"] is not None:
        total = total + s["r"].double()
    # the norm is taken of the rounded sum, which is an output of its own
    h = total.to(s["x"].dtype).double()
    length = (h * h).sum(1) / h.shape[1] + EPS
    y = h / length.sqrt()[:, None] * s["w"].double()[None, :]
    biggest = torch.stack([part.abs().max(1).values for part in y.split(s["group"], 1)], 1)
    wide = biggest.repeat_interleave(s["group"], 1) / 448.0
    # the codes' values before their rounding to 8 bits
    codes = torch.where(wide > 0, y / wide, torch.zeros_like(y))
    return (codes, biggest / 448.0) if s["r"] is None else (total, codes, biggest / 448.0)


def _exact_linear4(s):
    x = s["x"].double()
    inner = x.shape[1]
    if s["x_scales"] is not None:
        x = x * s["x_scales"].double().repeat_interleave(inner // s["x_scales"].shape[1], 1)
    out = []
    per = inner // s["scales"].shape[1]
    words = s["codes"].long() & 0xFFFFFFFF
    for at in range(0, words.shape[0], 4096):
        part = words[at : at + 4096]
        w = torch.empty(part.shape[0], inner, dtype=torch.float64, device=x.device)
        for j in range(8):
            w[:, j::8] = ((part // 16**j) % 16).double()
        sc = s["scales"][at : at + 4096].double().repeat_interleave(per, 1)
        if s["biases"] is None:
            w = (w - 8.0) * sc
        else:
            w = w * sc + s["biases"][at : at + 4096].double().repeat_interleave(per, 1)
        out.append(x.mm(w.t()))
    return torch.cat(out, 1)


def _exact_append(s):
    cache = s["cache"].double()
    rank, page = s["latent"].shape[1], cache.shape[1]
    table = s["cos_sin"].double()[s["positions"].long()]
    turn = torch.complex(table[..., 0], table[..., 1])

    def rotate(v, by):
        v = v.double()
        if s["interleaved"]:
            return torch.view_as_real(torch.complex(v[..., ::2].contiguous(), v[..., 1::2].contiguous()) * by).flatten(-2)
        turned = torch.complex(v[..., : ROPE // 2].contiguous(), v[..., ROPE // 2 :].contiguous()) * by
        return torch.cat([turned.real, turned.imag], -1)

    latent = s["latent"].double()
    if s["w"] is not None:
        latent = latent / (latent.pow(2).sum(1, keepdim=True) / rank + EPS).sqrt() * s["w"].double()
    key = rotate(s["rope_key"], turn)
    slots = s["slots"]
    for i in (slots >= 0).nonzero()[:, 0].split(4096):
        cache[slots[i] // page, slots[i] % page, :rank] = latent[i]
        cache[slots[i] // page, slots[i] % page, rank:] = key[i]
    return rotate(s["q_rope"], turn[:, None]), cache


def _exact_absorbed(s):
    ql, qr, cache = s["ql"], s["qr"], s["cache"]
    batch, queries, heads, rank = ql.shape
    out = torch.zeros(ql.shape, dtype=torch.float64, device=ql.device)
    for b, n in enumerate(s["lengths"].tolist()):
        rows = cache[s["table"][b].long()].flatten(0, 1)[:n].double()
        for t in range(queries):
            m = n - (queries - 1 - t)
            if m <= 0:
                continue
            seen = rows[:m]
            weight = (ql[b, t].double() @ seen[:, :rank].t() + qr[b, t].double() @ seen[:, rank:].t()) * s["scale"]
            out[b, t] = torch.softmax(weight, -1) @ seen[:, :rank]
    return out


def _exact_prompt(s):
    q, v = s["q"], s["v"]
    out = torch.zeros(q.shape[0], q.shape[1], v.shape[2], dtype=torch.float64, device=q.device)
    qs, ks = s["q_starts"].tolist(), s["k_starts"].tolist()
    for a, b, c, d in zip(qs, qs[1:], ks, ks[1:]):
        if a == b:
            continue
        hidden = torch.ones(b - a, d - c, dtype=torch.bool, device=q.device).triu(d - c - (b - a) + 1)
        for h in range(q.shape[1]):
            keys = torch.cat([s["k"][c:d, h], s["kr"][c:d]], 1).double()
            weight = (q[a:b, h].double() @ keys.t() * s["scale"]).masked_fill(hidden, float("-inf"))
            out[a:b, h] = torch.softmax(weight, 1) @ v[c:d, h].double()
    return out
