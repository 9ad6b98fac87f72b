"""Host-side checks of the attention half's C entry points (nothing is
launched: every call is refused or empty) and the page bookkeeping."""

import ctypes

import pytest

from mlxlr8_b200 import _lib

P = 1 << 20  # a 16-byte aligned address that no refused call touches


def _norm(x=P, w=P, dtype=2, rows=1, hidden=256, group=128, eps=1e-5, codes=P, scales=P):
    return _lib.load().exlr8_residual_rms_norm_q8(x, None, w, dtype, rows, hidden, group, eps, None, codes, scales, None)


@pytest.mark.parametrize("change, status", [
    (dict(rows=0), 0), (dict(rows=0, x=None), 0), (dict(dtype=3), 8), (dict(dtype=7), 8), (dict(rows=-1), 16),
    (dict(hidden=0), 16), (dict(group=48), 16), (dict(group=0), 16), (dict(hidden=200), 16), (dict(rows=1 << 40), 16),
    (dict(x=None), 11), (dict(w=None), 11), (dict(codes=None), 11), (dict(scales=None), 11),
    (dict(eps=float("nan")), 11), (dict(eps=-1.0), 11),
])
def test_norm_refusals(change, status):
    assert _norm(**change) == status


def _linear(x=P, x_dtype=2, xs=None, xg=0, rows=1, inner=256, outer=8, codes=P, scales=P, sdt=1, group=64, out=P, odt=2):
    return _lib.load().exlr8_affine4_linear(x, x_dtype, xs, xg, rows, inner, outer, codes, scales, None, sdt, group, out,
                                            odt, None)


@pytest.mark.parametrize("change, status", [
    (dict(rows=0), 0), (dict(x_dtype=4), 8), (dict(sdt=3), 8), (dict(odt=3), 8), (dict(inner=0), 16),
    (dict(inner=224), 16), (dict(group=16), 16), (dict(group=256), 16), (dict(outer=0), 16), (dict(rows=-3), 16),
    (dict(rows=(1 << 20) + 1), 16), (dict(rows=(1 << 19) + 1), 16), (dict(x_dtype=3, xs=P, xg=96), 16), (dict(x_dtype=3, xs=P, xg=0), 16),
    (dict(x_dtype=3, xg=128), 11), (dict(xs=P), 11), (dict(x=None), 11), (dict(codes=None), 11), (dict(out=None), 11),
    (dict(x=P + 8), 9), (dict(codes=P + 4), 9),
])
def test_linear_refusals(change, status):
    assert _linear(**change) == status


def _append(latent=P, tokens=1, rank=512, dtype=2, cos=None, cos_rows=0, positions=None, slots=P, cache=P, pages=4,
            page=16, q=None, heads=0, q_out=None, eps=1e-5):
    return _lib.load().exlr8_latent_append(latent, rank, P, 64, tokens, rank, dtype, None, eps, cos, cos_rows, positions,
                                           1, slots, cache, pages, page, q, 64, 64, heads, q_out, None)


@pytest.mark.parametrize("change, status", [
    (dict(tokens=0), 0), (dict(dtype=0), 8), (dict(rank=192), 16), (dict(rank=640), 16), (dict(rank=0), 16),
    (dict(page=8), 16), (dict(page=0), 16), (dict(page=24), 16), (dict(pages=-1), 16), (dict(pages=1 << 60), 16),
    (dict(tokens=-1), 16), (dict(latent=None), 11), (dict(slots=None), 11), (dict(cache=None), 11), (dict(cos=P), 11),
    (dict(q=P, heads=0), 16), (dict(q=P, heads=2), 11), (dict(eps=float("nan")), 11), (dict(cos_rows=-1), 16),
])
def test_append_refusals(change, status):
    assert _append(**change) == status


def _attend(ql=P, batch=1, queries=1, heads=8, rank=512, dtype=2, cache=P, pages=4, page=16, table=P, width=4, lengths=P,
            scale=0.1, out=P, ws=P, ws_bytes=1 << 40):
    return _lib.load().exlr8_latent_attention(ql, P, batch, queries, heads, rank, dtype, cache, pages, page, table, width,
                                              lengths, scale, out, None, ws, ws_bytes, None)


@pytest.mark.parametrize("change, status", [
    (dict(batch=0), 0), (dict(dtype=0), 8), (dict(dtype=3), 8), (dict(rank=100), 16), (dict(queries=0), 16),
    (dict(heads=0), 16), (dict(page=20), 16), (dict(batch=-1), 16), (dict(batch=1 << 30), 16), (dict(width=-1), 16),
    (dict(pages=1 << 40), 16), (dict(width=1 << 30), 16), (dict(width=(1 << 26) + 1), 16), (dict(queries=1 << 30, heads=1 << 16), 16),
    (dict(ql=None), 11), (dict(table=None), 11), (dict(lengths=None), 11), (dict(cache=None), 11), (dict(out=None), 11),
    (dict(scale=float("inf")), 11), (dict(scale=float("nan")), 11), (dict(ql=P + 2), 9), (dict(cache=P + 8), 9),
])
def test_attention_refusals(change, status):
    assert _attend(**change) == status


def test_attention_workspace_refuses_unusable_sizes():
    query = _lib.load().exlr8_latent_attention_workspace
    bad = ctypes.c_size_t(-1).value
    for args in ((-1, 1, 8, 512), (1, 0, 8, 512), (1, 1, 0, 512), (1, 1, 8, 500), (1 << 20, 1 << 20, 1 << 15, 512)):
        assert query(*args) == bad
    assert query(0, 1, 8, 512) != bad and query(4, 2, 64, 512) != bad


def _prompt(q=P, qs=(192 * 4, 192), k=P, ks=(128 * 4, 128), rs=64, vs=(128 * 4, 128), total_q=5, total_k=7, heads=4,
            nope=128, value=128, dtype=1, starts=P, seqs=1, scale=0.1, out=P):
    return _lib.load().exlr8_latent_prompt_attention(q, *qs, k, *ks, P, rs, P, *vs, total_q, total_k, heads, nope, value,
                                                     dtype, starts, P, seqs, scale, out, None, None)


@pytest.mark.parametrize("change, status", [
    (dict(total_q=0), 0), (dict(dtype=0), 8), (dict(nope=96), 16), (dict(nope=256), 16), (dict(value=320), 16),
    (dict(value=0), 16), (dict(heads=0), 16), (dict(heads=70000), 16), (dict(seqs=0), 16), (dict(seqs=5000), 16),
    (dict(total_q=-1), 16), (dict(total_k=1 << 33), 16), (dict(qs=(770, 192)), 16), (dict(ks=(512, 4)), 16),
    (dict(rs=65), 16), (dict(vs=(-8, 128)), 16), (dict(q=None), 11), (dict(k=None), 11), (dict(starts=None), 11),
    (dict(out=None), 11), (dict(scale=float("nan")), 11), (dict(q=P + 2), 9), (dict(out=P + 4), 9),
])
def test_prompt_refusals(change, status):
    assert _prompt(**change) == status


def test_shape_status_is_a_value_error():
    with pytest.raises(ValueError, match="sizes or strides"):
        _lib.check(16)


def test_pages_are_handed_out_and_given_back():
    from mlxlr8_b200.latent import LatentPages

    pages = LatentPages(6, 16, device="cpu")
    step = pages.step(["a", "b"], 10)
    assert step.lengths.tolist() == [10, 10] and step.queries == 10
    assert step.positions.tolist() == 2 * list(range(10))
    a, b = step.block_table[:, 0].tolist()
    assert a != b and step.slots.tolist() == [16 * a + i for i in range(10)] + [16 * b + i for i in range(10)]
    step = pages.step(["b"], 7)
    assert step.lengths.tolist() == [17] and step.block_table.shape == (1, 2)
    assert step.slots.tolist()[:6] == [16 * b + i for i in range(10, 16)] and step.slots[6] % 16 == 0
    step = pages.step(["a", "b"])
    assert step.block_table.tolist()[0][1] == -1 and step.lengths.tolist() == [11, 18]
    with pytest.raises(ValueError, match="no free pages"):
        pages.step(["c", "b"], 40)
    assert pages.length("c") == 0 and pages.length("b") == 18
    pages.release("b")
    assert pages.length("b") == 0
    step = pages.step(["c"], 80)
    assert sorted(step.block_table[0].tolist()) == sorted(set(range(6)) - {a})
    for bad in (lambda: pages.step([]), lambda: pages.step(["a", "a"]), lambda: pages.step(["a"], 0),
                lambda: LatentPages(4, 24)):
        with pytest.raises(ValueError):
            bad()


# ---- outputs and workspaces over other operands: refused before any launch ---------
# Operands lie a MB apart from each other; every case puts one over another.

MB = 1 << 20


def _apart(names):
    return {name: (i + 1) * (16 * MB) for i, name in enumerate(names)}


@pytest.mark.parametrize("change", [
    ("h", "x", 0), ("h", "residual", 2 * 512 - 2), ("codes", "x", 3 * 512 * 2 - 8), ("scales", "w", 0), ("codes", "residual", 8),
    ("scales", "codes", 3 * 512 - 4), ("h", "scales", -3 * 512 * 2 + 4),
])
def test_norm_outputs_over_other_operands(change):
    at = _apart(["x", "residual", "w", "h", "codes", "scales"])
    at[change[0]] = at[change[1]] + change[2]
    assert _lib.load().exlr8_residual_rms_norm_q8(at["x"], at["residual"], at["w"], 2, 3, 512, 128, 1e-5, at["h"], at["codes"],
                                                  at["scales"], None) == 17


@pytest.mark.parametrize("other, by", [("x", 0), ("x", 2 * 3 * 512 - 4), ("codes", 40 * 256 - 4), ("scales", -3 * 40 * 2 + 2),
                                       ("biases", 40 * 8 * 2 - 2)])
def test_linear_output_over_other_operands(other, by):
    at = _apart(["x", "codes", "scales", "biases"])
    assert _lib.load().exlr8_affine4_linear(at["x"], 2, None, 0, 3, 512, 40, at["codes"], at["scales"], at["biases"], 1, 64,
                                            at[other] + by, 2, None) == 17


def test_linear_output_over_the_activations_scales():
    assert _lib.load().exlr8_affine4_linear(MB, 3, 2 * MB, 128, 3, 512, 40, 3 * MB, 4 * MB, None, 1, 64, 2 * MB + 44, 2, None) == 17


@pytest.mark.parametrize("name, by", [
    ("latent", 0), ("latent", 4 * 16 * 192 * 2 - 2), ("latent", -(4 * 200 + 128) * 2 + 2), ("key", 64), ("weight", 0),
    ("cos", 4096), ("positions", -16), ("slots", -36), ("q", -(4 * 300 + 64 + 64) * 2 + 2), ("q_out", 8),
])
def test_append_cache_over_other_operands(name, by):
    at = _apart(["cache", "latent", "key", "weight", "cos", "positions", "slots", "q", "q_out"])
    at[name] = at["cache"] + by
    assert _lib.load().exlr8_latent_append(at["latent"], 200, at["key"], 200, 5, 128, 2, at["weight"], 1e-5, at["cos"], 40,
                                           at["positions"], 1, at["slots"], at["cache"], 4, 16, at["q"], 300, 64, 2, at["q_out"],
                                           None) == 17


def test_append_rows_with_negative_strides_over_the_cache():
    at = _apart(["cache", "latent", "key", "slots"])
    latent = at["cache"] + 4 * 16 * 192 * 2 + 3 * 200 * 2  # the last of five rows ends over the cache
    assert _lib.load().exlr8_latent_append(latent, -200, at["key"], 64, 5, 128, 2, None, 1e-5, None, 0, None, 1, at["slots"],
                                           at["cache"], 4, 16, None, 0, 0, 0, None, None) == 17


@pytest.mark.parametrize("name, other, by", [
    ("out", "ql", 0), ("out", "cache", 4 * 16 * 576 * 2 - 16), ("out", "lengths", 0), ("lse", "out", 3 * 8 * 512 * 2 - 16),
    ("ws", "ql", 1024), ("ws", "qr", 0), ("ws", "cache", 0), ("ws", "table", -16), ("ws", "out", 0), ("ws", "lse", -16),
    ("lse", "qr", 0), ("table", "out", 16),
])
def test_attention_outputs_and_workspace_over_other_operands(name, other, by):
    names = ["ql", "qr", "cache", "table", "lengths", "out", "lse", "ws"]
    at = _apart(names)
    at[name] = at[other] + by
    assert _lib.load().exlr8_latent_attention(at["ql"], at["qr"], 3, 1, 8, 512, 2, at["cache"], 4, 16, at["table"], 4, at["lengths"],
                                              0.1, at["out"], at["lse"], at["ws"], 1 << 40, None) == 17


@pytest.mark.parametrize("name, other, by", [
    ("out", "q", (4 * 768 + 3 * 192 + 192) * 2 - 16), ("out", "k", 16), ("out", "kr", 0), ("out", "v", 0), ("out", "qs", 0),
    ("out", "ks", 0), ("lse", "out", 0), ("lse", "v", (6 * 512 + 3 * 128 + 128) * 2 - 4),
])
def test_prompt_outputs_over_other_operands(name, other, by):
    at = _apart(["q", "k", "kr", "v", "qs", "ks", "out", "lse"])
    at[name] = at[other] + by
    assert _lib.load().exlr8_latent_prompt_attention(at["q"], 768, 192, at["k"], 512, 128, at["kr"], 64, at["v"], 512, 128, 5, 7, 4,
                                                     128, 128, 1, at["qs"], at["ks"], 1, 0.1, at["out"], at["lse"], None) == 17


def test_overlap_status_is_a_value_error():
    with pytest.raises(ValueError, match="overlaps"):
        _lib.check(17)


def test_stack_blocks_stay_as_they_are_given(monkeypatch):
    """Pairs are pairs, as callers walk and extend them; a third entry is the
    block's attention."""
    from mlxlr8_b200 import stack

    def norm(x, weight, eps, residual=0, return_sum=False):
        return (x + residual, (x + residual) * weight) if return_sum else x * weight

    monkeypatch.setattr(stack, "residual_rms_norm", norm)
    made = stack.MoEStack((w, lambda xn, h: xn + h) for w in (2, 3))
    assert [w for w, layer in made.blocks] == [2, 3] and len(made) == 2
    made.blocks.append((5, lambda xn, h: xn - h))
    assert made(1) == 3 * 4 * 4
    made = stack.MoEStack([[2, lambda xn, h: xn + h, lambda h, step: h * step], (3, lambda xn, h: xn + h, None)])
    assert made(1, step=10) == 11 * 3 * 4
    for bad in ((1,), (1, 2, 3, 4)):
        with pytest.raises(ValueError):
            stack.MoEStack([bad])


def test_residuals_of_another_size_are_refused():
    """As what an attention returns: the kernel would read past one of the two."""
    import torch

    from mlxlr8_b200 import stack

    x, w = torch.zeros(4, 128), torch.ones(128)
    for rows in (3, 5):
        with pytest.raises(ValueError, match="size of x"):
            stack.residual_rms_norm(x, w, residual=torch.zeros(rows, 128))
        made = stack.MoEStack([(w, lambda xn, h: h, lambda h, step: torch.zeros(rows, 128))])
        with pytest.raises(ValueError, match="size of x"):
            made(x)


def test_weights_of_a_layer_lie_on_one_device():
    import torch

    from mlxlr8_b200.affine4 import Affine4Linear

    codes, scales = torch.zeros(8, 32, dtype=torch.int32), torch.ones(8, 4)
    assert Affine4Linear(codes, scales, scales).group == 64
    for parts in ((scales.to("meta"), None), (scales, scales.to("meta"))):
        with pytest.raises(ValueError, match="different devices"):
            Affine4Linear(codes, *parts)
