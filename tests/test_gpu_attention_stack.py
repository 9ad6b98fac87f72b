"""The attention half of a decoder block as one run: 8-bit norm, 4-bit layers,
cache append, absorbed attention, and a stack whose blocks have it.

The oracle repeats the stages in 64 bits and rounds where the operators round
(the codes and scales of the norm are the operator's own: it is tested by
itself).  From there to the block's r lie roundings to bfloat16 of the key row,
the queries, the softmax's weights, the attention's output and r: five half
steps of 2^-8, independent and even, each 2^-8 / sqrt(3) of its value in the
mean square; the score's roundings act through the softmax by less than the
scores' spread (below 2 here) times the same.  Their root sum is below
2^-8 / sqrt(3) * sqrt(5 + 2 * 4) = 8.2e-3."""

import pytest

from helpers import rel_l2

pytestmark = pytest.mark.gpu

TOL = 8.2e-3
HIDDEN, HEADS, RANK, SCALE = 256, 4, 128, 0.06


def _linear(g, outer, inner, group=64):
    import torch

    from mlxlr8_b200.affine4 import Affine4Linear

    codes = torch.randint(-(1 << 31), 1 << 31, (outer, inner // 8), generator=g, device="cuda", dtype=torch.int32)
    scales = torch.full((outer, inner // group), 0.22 * inner ** -0.5, device="cuda", dtype=torch.float16)
    return Affine4Linear(codes, scales, (-7.5 * scales.float()).half())


def _dense(layer):
    import torch

    words = layer.codes.long() & 0xFFFFFFFF
    q = torch.stack([(words >> (4 * j)) & 15 for j in range(8)], -1).flatten(1).double()
    s, b = (t.double().repeat_interleave(layer.group, 1) for t in (layer.scales, layer.biases))
    return q * s + b


def _attention(seed, pages=12, page=16):
    import torch

    from mlxlr8_b200.latent import LatentSelfAttention, rope_table

    g = torch.Generator(device="cuda").manual_seed(seed)
    norm = (1 + 0.1 * torch.randn(HIDDEN, generator=g, device="cuda")).bfloat16()
    key_norm = (1 + 0.1 * torch.randn(RANK, generator=g, device="cuda")).bfloat16()
    cache = torch.full((pages, page, RANK + 64), float("nan"), device="cuda", dtype=torch.bfloat16)
    return LatentSelfAttention(norm, _linear(g, HEADS * RANK, HIDDEN), _linear(g, HEADS * 64, HIDDEN),
                               _linear(g, RANK + 64, HIDDEN), key_norm, _linear(g, HIDDEN, HEADS * RANK), cache, HEADS, SCALE,
                               rope_table(256))


class _Oracle:
    """One block's attention in float64, with every token's cache row kept."""

    def __init__(self, attention):
        self.a, self.rows = attention, {}

    def __call__(self, h, sequences, step):
        import torch

        from mlxlr8_b200.stack import residual_rms_norm_q8

        a = self.a

        def rounded(v):
            return v.to(torch.bfloat16).double()

        codes, scales = residual_rms_norm_q8(h, a.input_norm, a.eps, group=a.group)
        x = codes.float().double() * scales.double().repeat_interleave(a.group, 1)
        kv, ql, qr = (rounded(x @ _dense(layer).t()) for layer in (a.key, a.query_latent, a.query_rope))
        cs = a.cos_sin.double()[step.positions.long()]

        def rotated(v):
            c, n = (cs[..., i].reshape((-1,) + (1,) * (v.dim() - 2) + (32,)) for i in (0, 1))
            p, q = v[..., 0::2], v[..., 1::2]
            return rounded(torch.stack([p * c - q * n, p * n + q * c], -1).flatten(-2))

        latent = kv[:, :RANK]
        latent = rounded(latent / (latent.square().mean(1, keepdim=True) + a.eps).sqrt() * a.key_norm.double())
        row = torch.cat([latent, rotated(kv[:, RANK:])], 1)
        q = torch.cat([ql.view(-1, HEADS, RANK), rotated(qr.view(-1, HEADS, 64))], -1)
        out = []
        for i, s in enumerate(sequences):
            for t in range(step.queries):
                n = i * step.queries + t
                self.rows[s] = torch.cat([self.rows[s], row[n:n + 1]]) if s in self.rows else row[n:n + 1]
                p = torch.softmax(q[n] @ self.rows[s].t() * SCALE, -1)
                out.append((p @ self.rows[s][:, :RANK]).flatten())
        return rounded(torch.stack(out)) @ _dense(a.output).t()


@pytest.mark.parametrize("queries", [1, 2])
def test_decode_steps_match_the_formulas(queries):
    import torch

    from mlxlr8_b200.latent import LatentPages

    g = torch.Generator(device="cuda").manual_seed(5)
    attention = _attention(6)
    oracle, pages = _Oracle(attention), LatentPages(12, 16)
    for n in range(20):
        sequences = ["a", "b", "c"] if n % 3 else ["c", "a"]
        step = pages.step(sequences, queries)
        h = torch.randn(len(sequences) * queries, HIDDEN, generator=g, device="cuda").bfloat16()
        got = attention(h, step)
        expected = oracle(h, sequences, step)
        assert rel_l2(got.double().cpu().numpy(), expected.cpu().numpy()) < TOL
    pages.release("b")
    oracle.rows.pop("b")
    step = pages.step(["b", "c"], queries)
    h = torch.randn(2 * queries, HIDDEN, generator=g, device="cuda").bfloat16()
    assert rel_l2(attention(h, step).double().cpu().numpy(), oracle(h, ["b", "c"], step).cpu().numpy()) < TOL


def test_stack_with_attention_is_its_parts():
    """A stack whose blocks have an attention: h + r, its norm, the MoE layer,
    bit for bit the operators' own results; blocks without one as before."""
    import torch

    from mlxlr8_b200.latent import LatentPages
    from mlxlr8_b200.moe import MoELayer
    from mlxlr8_b200.stack import MoEStack, residual_rms_norm
    from mlxlr8_b200.synthetic import make_layer

    made = [make_layer(seed=20 + i, hidden=HIDDEN, intermediate=128, device="cuda") for i in range(3)]
    layers = [MoELayer(m.gate_weight, m.bias, m.experts) for m in made]
    norm = torch.ones(HIDDEN, device="cuda", dtype=torch.bfloat16)
    pair = [_attention(30), _attention(31)]
    twin = [_attention(30), _attention(31)]
    stack = MoEStack([(norm, layers[0], pair[0]), (norm, layers[1]), (norm, layers[2], pair[1])])
    pages, pages_twin = LatentPages(12, 16), LatentPages(12, 16)
    h, _ = made[0].tokens(2)
    other = h.clone()
    for _ in range(3):
        h, steps = stack(h, trace=True, step=pages.step([1, 2]))
        step = pages_twin.step([1, 2])
        for i, attention in ((0, twin[0]), (1, None), (2, twin[1])):
            if attention is not None:
                other = attention(other, step) + other
            xn = residual_rms_norm(other, norm)
            assert torch.equal(steps[i][0], other) and torch.equal(steps[i][1], xn)
            other = layers[i](xn, other)
            assert torch.equal(steps[i][2], other)
        assert torch.equal(h, other) and bool(h.isfinite().all())


def test_decode_step_in_a_graph():
    """One captured step replayed while the lengths, slots and positions change
    in place."""
    import torch

    from mlxlr8_b200.latent import LatentPages, LatentStep

    g = torch.Generator(device="cuda").manual_seed(8)
    eager, captured = _attention(40), _attention(40)
    pages = LatentPages(12, 16)
    h = torch.zeros(2, HIDDEN, device="cuda", dtype=torch.bfloat16)
    fixed = LatentStep(torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"),
                       torch.full((2, 4), -1, dtype=torch.int32, device="cuda"),
                       torch.zeros(2, dtype=torch.int32, device="cuda"), 1)
    captured(h, fixed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = captured(h, fixed)
    for _ in range(40):
        step = pages.step(["x", "y"])
        h.copy_(torch.randn(2, HIDDEN, generator=g, device="cuda"))
        fixed.slots.copy_(step.slots)
        fixed.positions.copy_(step.positions)
        fixed.lengths.copy_(step.lengths)
        fixed.block_table[:, : step.block_table.shape[1]].copy_(step.block_table)
        graph.replay()
        assert torch.equal(out, eager(h, step))
    with pytest.raises(ValueError, match="of the step"):
        eager(h[:1], step)


def test_hidden_state_keeps_its_type_beside_an_attention_of_another():
    import torch

    from mlxlr8_b200.stack import MoEStack, residual_rms_norm

    g = torch.Generator(device="cuda").manual_seed(50)
    h, r = (torch.randn(3, HIDDEN, generator=g, device="cuda") for _ in range(2))
    h, w = h.bfloat16(), torch.ones(HIDDEN, device="cuda", dtype=torch.bfloat16)
    out, steps = MoEStack([(w, lambda xn, h: xn + h, lambda h, step: r)])(h, trace=True)
    total, xn = residual_rms_norm(h, w, residual=r.bfloat16(), return_sum=True)
    assert out.dtype == torch.bfloat16 and torch.equal(steps[0][0], total) and torch.equal(steps[0][1], xn)
    for other in (w.cpu(), w[:-1]):
        with pytest.raises(ValueError):
            residual_rms_norm(h, other)
    with pytest.raises(ValueError):
        residual_rms_norm(h, w, residual=r.cpu())
