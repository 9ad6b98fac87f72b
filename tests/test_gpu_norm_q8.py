"""The residual RMS norm with E4M3 output against its formula in 64 bits.

Tolerances: the rounded sum h is exact; a scale carries the float32 error of
the sum of squares (pairwise over a row: well under 32 half steps), the root,
two products and the maximum's division; a code is off by half an E4M3 step of
the quotient (2^-4 of the value, 2^-10 below the normal range) and the same
float32 errors."""

import pytest

from helpers import torch_dtype

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24


def _expected(x, w, residual, group, eps, dtype):
    import torch

    h = x.double() if residual is None else (x.double() + residual.double()).to(dtype).double()
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()
    blocks = y.reshape(y.shape[0], -1, group)
    return h, blocks, blocks.abs().amax(-1) / 448.0


def _check(x, w, residual, group, eps=1e-5):
    import torch

    from mlxlr8_b200.stack import residual_rms_norm_q8

    h, codes, scales = residual_rms_norm_q8(x, w, eps, residual=residual, group=group, return_sum=True)
    eh, blocks, es = _expected(x.reshape(-1, x.shape[-1]), w, None if residual is None else residual.reshape(
        -1, x.shape[-1]), group, eps, x.dtype)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape
    assert scales.shape == x.shape[:-1] + (x.shape[-1] // group,)
    assert torch.equal(h.double().reshape(eh.shape), eh)
    s = scales.double().reshape(es.shape)
    assert bool(((s - es).abs() <= 48 * F32 * es + 1e-44).all())
    q = codes.float().double().reshape(blocks.shape)
    ratio = torch.where(es[..., None] > 0, blocks / es[..., None].clamp_min(1e-300), torch.zeros_like(blocks))
    assert bool(((q - ratio).abs() <= ratio.abs() * (2.0 ** -4 + 96 * F32) + 2.0 ** -10).all())
    return codes, scales


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows, hidden, group", [
    (1, 6144, 128), (3, 6144, 64), (5, 256, 32), (2, 128, 128), (7, 1000, 1000), (2, 1, 1), (3, 33, 33),
    (4, 8192, 8192), (2, 20480, 128), (1, 20001, 20001), (300, 512, 64),
    (2, 30001, 30001), (3, 33280, 128), (40, 4099, 4099),
])
@pytest.mark.parametrize("with_residual", [False, True])
def test_codes_and_scales_match_the_formula(dtype, rows, hidden, group, with_residual):
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows * hidden + group)
    td = torch_dtype(dtype)
    x = torch.randn(rows, hidden, generator=g, device="cuda")
    x[:, :: max(1, hidden // 5)] *= 30.0
    r = torch.randn(rows, hidden, generator=g, device="cuda").to(td) if with_residual else None
    w = (1.0 + 0.2 * torch.randn(hidden, generator=g, device="cuda")).to(td)
    _check(x.to(td), w, r, group)


@pytest.mark.parametrize("group", [32, 64, 128, 512])
def test_groups_of_zeros_and_rows_that_are_not_finite(group):
    import torch

    from mlxlr8_b200.stack import residual_rms_norm_q8

    x = torch.randn(6, 512, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    w = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    x[0] = 0
    x[1, :group] = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    codes, scales = residual_rms_norm_q8(x, w, group=group)
    values = codes.float().reshape(6, -1, group) * scales[..., None]
    assert bool((scales[0] == 0).all()) and bool((codes[0].float() == 0).all())
    assert float(scales[1, 0]) == 0.0 and bool((codes[1, :group].float() == 0).all())
    assert bool(values[2].isnan().all())
    # an infinite channel: the norm makes the others 0 and itself NaN
    assert bool(values[3, 0].isnan().all()) and bool((values[3, 1:] == 0).all())
    # a weight that is not finite touches its own group alone
    w[300] = float("inf")
    _, scales = residual_rms_norm_q8(x[4:], w, group=group)
    assert bool(scales[:, 300 // group].isnan().all())
    assert int(scales.isnan().sum()) == 2


def test_views_shapes_and_an_unaligned_start():
    import torch

    g = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randn(384, generator=g, device="cuda").bfloat16()
    _check(torch.randn(2, 3, 384, generator=g, device="cuda").bfloat16(), w, None, 128)
    _check(torch.randn(384, 5, generator=g, device="cuda").bfloat16().t(), w, None, 128)
    flat = torch.randn(5 * 384 + 1, generator=g, device="cuda").bfloat16()
    _check(flat[1:].view(5, 384), w, flat[:-1].view(5, 384), 64)
    wide = torch.randn(385, generator=g, device="cuda").bfloat16()
    _check(flat[: 5 * 384].view(5, 384), wide[1:], None, 384)


def test_no_rows_and_refusals():
    import torch

    from mlxlr8_b200.stack import residual_rms_norm_q8

    x = torch.randn(2, 256, device="cuda").bfloat16()
    w = torch.ones(256, device="cuda", dtype=torch.bfloat16)
    codes, scales = residual_rms_norm_q8(x[:0], w)
    assert codes.shape == (0, 256) and scales.shape == (0, 2)
    for bad in (dict(group=16), dict(group=96), dict(group=0), dict(residual=x[:1])):
        with pytest.raises(ValueError):
            residual_rms_norm_q8(x, w, **bad)
    with pytest.raises(ValueError, match="one entry per hidden channel"):
        residual_rms_norm_q8(x, w[:-1])
    for none in (x[:, :0], x[0, 0]):
        with pytest.raises(ValueError, match="needs a channel"):
            residual_rms_norm_q8(none, w[:0])
    with pytest.raises(ValueError, match="dtype"):
        residual_rms_norm_q8(x.double(), w)
    with pytest.raises(ValueError, match="CUDA"):
        residual_rms_norm_q8(x.cpu(), w)


def _small_or_large(x, w, group, eps=1e-5):
    """Codes and scales by the formula where a group's values are small or
    large: a scale below the smallest float32 is 0, and its codes with it."""
    import torch

    from mlxlr8_b200.stack import residual_rms_norm_q8

    codes, scales = residual_rms_norm_q8(x, w, eps, group=group)
    _, blocks, es = _expected(x, w, None, group, eps, x.dtype)
    s = scales.double().reshape(es.shape)
    # float32 errors, and half a step of the smallest float32
    assert bool(((s - es).abs() <= 48 * F32 * es + 2.0 ** -149).all())
    q = codes.float().double().reshape(blocks.shape)
    ratio = torch.where(s[..., None] > 0, blocks / es[..., None].clamp_min(1e-300), torch.zeros_like(blocks))
    assert bool(((q - ratio).abs() <= ratio.abs() * (2.0 ** -4 + 96 * F32) + 2.0 ** -10).all())
    return s


TINY = (1e-44, 1e-42, 1e-40, 1e-38, 1e-37, 1e-36, 1.3e-36, 1.4e-36, 1e-33, 1e-30, 1e-24)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hidden, group, offset", [
    (512, 32, 0), (1024, 128, 0), (20480, 64, 0), (512, 64, 1), (33280, 128, 0),  # a group of an ordinary row
    (512, 512, 0), (8192, 8192, 0), (333, 333, 0), (30001, 30001, 0), (512, 512, 1),  # the row
])
def test_groups_of_values_down_to_the_smallest(dtype, hidden, group, offset):
    import torch

    g = torch.Generator(device="cuda").manual_seed(hidden + group)
    td = torch_dtype(dtype)
    x = torch.randn(len(TINY), hidden, generator=g, device="cuda")
    for i, top in enumerate(TINY):
        part = x[i, : group]
        part /= part.abs().max()
        part[::3] = 0.0
        part[1] = -1.0
        # (products with the least values are formed without a flush to zero)
        x[i, : group] = (part.double() * top).float()
    w = (1.0 + 0.2 * torch.randn(hidden, generator=g, device="cuda")).to(td)
    flat = torch.empty(x.numel() + offset, device="cuda", dtype=td)
    flat[offset:] = x.to(td).flatten()
    scales = _small_or_large(flat[offset:].view(x.shape), w, group)
    assert bool((scales[3:, 0] > 0).all())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("hidden, group, offset", [(512, 32, 0), (512, 512, 0), (333, 333, 0), (512, 64, 1), (30001, 30001, 0)])
def test_products_with_the_weight_past_the_largest_float(dtype, hidden, group, offset):
    """h * w overflows, the normed h * w does not."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(hidden + group)
    td = torch_dtype(dtype)
    flat = (torch.randn(3 * hidden + offset, generator=g, device="cuda") * 1e12).to(td)
    w = (1.0 + 0.2 * torch.randn(hidden, generator=g, device="cuda"))
    w[: 16] *= 1e28
    scales = _small_or_large(flat[offset:].view(3, hidden), w.to(td), group)
    assert bool(scales.isfinite().all()) and bool((scales > 0).all())
