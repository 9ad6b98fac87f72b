"""The 4-bit affine linear layer against its formula in 64 bits.

Tolerance of an output: half a step of its type, and the float32 error of the
sums.  The kernel adds products of q - 8 (and of the folded bias) with x; a
chain of n additions is off by at most n 2^-23 of the sum of their magnitudes
(2^-23, a whole step: matrix instructions cut off where a float addition
rounds), and no chain is longer than in / 8 + 64."""

import pytest

from helpers import torch_dtype

pytestmark = pytest.mark.gpu


def _weights(g, outer, inner, group, dtype, biases):
    import torch

    codes = torch.randint(-(1 << 31), 1 << 31, (outer, inner // 8), generator=g, device="cuda", dtype=torch.int32)
    scales = (torch.randn(outer, inner // group, generator=g, device="cuda") * 0.02).to(dtype)
    b = (torch.randn(outer, inner // group, generator=g, device="cuda") * 0.1).to(dtype) if biases else None
    return codes, scales, b


def _values(codes):
    import torch

    words = codes.view(torch.int32).long() & 0xFFFFFFFF
    return torch.stack([(words >> (4 * j)) & 15 for j in range(8)], -1).flatten(1).double()


def _check(x, codes, scales, biases, x_scales=None, out_dtype=None, out=None):
    import torch

    from mlxlr8_b200.affine4 import affine4_linear

    got = affine4_linear(x, codes, scales, biases, x_scales=x_scales, out_dtype=out_dtype, out=out)
    inner = codes.shape[1] * 8
    group = inner // scales.shape[1]
    xv = x.float().double().reshape(-1, inner)
    if x_scales is not None:
        xs = x_scales.double().reshape(xv.shape[0], -1)
        xv = xv * xs.repeat_interleave(inner // xs.shape[1], 1)
    s = scales.double().repeat_interleave(group, 1)
    b = -8.0 * s if biases is None else biases.double().repeat_interleave(group, 1)
    q = _values(codes)
    expected = xv @ (q * s + b).t()
    magnitude = xv.abs() @ (((q - 8.0) * s).abs() + (b + 8.0 * s).abs()).t()
    tol = expected.abs() * torch.finfo(got.dtype).eps / 2 * 1.001 + (inner / 8 + 64) * 2.0 ** -23 * magnitude + 1e-30
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert got.shape == x.shape[:-1] + (codes.shape[0],)
    assert bool(((got.double().reshape(expected.shape) - expected).abs() <= tol).all())
    return got


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("rows, inner, outer, group, biases", [
    (1, 6144, 576, 64, True), (1, 512, 1000, 128, False), (2, 32, 1, 32, True), (3, 96, 33, 32, True),
    (8, 2080, 130, 32, False), (9, 1024, 64, 128, True), (16, 1152, 257, 64, True), (17, 640, 48, 128, False),
    (33, 256, 31, 64, True), (1, 128, 5, 128, True), (5, 64, 16, 64, False), (4, 16384, 70, 128, True),
    (8, 8192, 4000, 32, True), (16, 12288, 300, 32, False), (3, 6144, 5000, 64, True),
])
def test_float_activations(dtype, rows, inner, outer, group, biases):
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows + inner + outer)
    td = torch_dtype(dtype)
    x = torch.randn(rows, inner, generator=g, device="cuda").to(td)
    for scale_dtype in (torch.float16, torch.bfloat16, torch.float32):
        _check(x, *_weights(g, outer, inner, group, scale_dtype, biases))


@pytest.mark.parametrize("x_group", [32, 64, 128, 0])
@pytest.mark.parametrize("rows, inner, outer, group", [(1, 1536, 100, 128), (8, 768, 65, 64), (11, 384, 40, 32),
                                                       (2, 6144, 576, 128)])
def test_8_bit_activations(x_group, rows, inner, outer, group):
    import torch

    g = torch.Generator(device="cuda").manual_seed(rows * inner + x_group)
    x = (torch.randn(rows, inner, generator=g, device="cuda") * 100).to(torch.float8_e4m3fn)
    xs = torch.rand(rows, inner // (x_group or inner), generator=g, device="cuda") + 0.1
    for biases, out_dtype in ((True, torch.bfloat16), (False, torch.float32), (True, torch.float16)):
        _check(x, *_weights(g, outer, inner, group, torch.float16, biases), x_scales=xs, out_dtype=out_dtype)


@pytest.mark.parametrize("x_dtype, out_dtype", [("bfloat16", "float32"), ("float16", "bfloat16"), ("float32", "float16")])
def test_other_output_types(x_dtype, out_dtype):
    import torch

    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(3, 512, generator=g, device="cuda").to(torch_dtype(x_dtype))
    _check(x, *_weights(g, 77, 512, 64, torch.bfloat16, True), out_dtype=torch_dtype(out_dtype))


def test_all_codes_in_every_place():
    """Each nibble of a word reaches its own channel: one channel of x at a time."""
    import torch

    from mlxlr8_b200.affine4 import affine4_linear

    codes = torch.randint(-(1 << 31), 1 << 31, (16, 32), device="cuda", dtype=torch.int32)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.eye(256, device="cuda", dtype=dtype)
        for group in (32, 64, 128):
            scales = torch.ones(16, 256 // group, device="cuda")
            got = affine4_linear(x, codes, scales, out_dtype=torch.float32)
            assert torch.equal(got.t().double(), _values(codes) - 8.0)


def test_large_and_small_channels_and_infinities():
    import torch

    from mlxlr8_b200.affine4 import affine4_linear

    g = torch.Generator(device="cuda").manual_seed(9)
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(2, 1024, generator=g, device="cuda")
        x[:, 7] = 1e30
        x[:, 500:600] = 1e-30
        weights = _weights(g, 40, 1024, 64, torch.float32, True)
        _check(x.to(dtype), *weights)
        x[1, 900] = float("nan")
        got = affine4_linear(x.to(dtype), *weights)
        assert bool(got[0].isfinite().all()) and bool(got[1].isnan().all())


def test_views_out_streams_and_leading_dimensions():
    import torch

    g = torch.Generator(device="cuda").manual_seed(10)
    weights = _weights(g, 96, 256, 64, torch.float16, True)
    x = torch.randn(256, 6, generator=g, device="cuda").bfloat16().t()
    _check(x, *weights)
    _check(torch.randn(2, 3, 256, generator=g, device="cuda").bfloat16(), *weights)
    _check(torch.randn(256, generator=g, device="cuda").half(), *weights)
    flat = torch.randn(3 * 256 + 1, generator=g, device="cuda").bfloat16()
    _check(flat[1:].view(3, 256), *weights)
    out = torch.empty(6, 96, device="cuda", dtype=torch.float32)
    assert _check(x, *weights, out=out).data_ptr() == out.data_ptr()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _check(x, *weights)
    side.synchronize()
    codes = weights[0].repeat(1, 2)[:, ::2].contiguous()
    wide = torch.stack([codes, codes], -1)[..., 0]
    _check(x, wide, *weights[1:])
    _check(x, weights[0].view(torch.uint32), *weights[1:])


def test_results_do_not_change_between_runs_and_replays():
    import torch

    from mlxlr8_b200.affine4 import Affine4Linear

    g = torch.Generator(device="cuda").manual_seed(11)
    layer = Affine4Linear(*_weights(g, 4096, 2048, 64, torch.bfloat16, True))
    x = torch.randn(3, 2048, generator=g, device="cuda").bfloat16()
    out = torch.empty(3, 4096, device="cuda", dtype=torch.bfloat16)
    first = layer(x).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, out=out)
    for _ in range(5):
        out.zero_()
        graph.replay()
        assert torch.equal(out, first) and torch.equal(layer(x), first)


def test_no_rows_and_refusals():
    import torch

    from mlxlr8_b200.affine4 import Affine4Linear, affine4_linear

    g = torch.Generator(device="cuda").manual_seed(12)
    codes, scales, biases = _weights(g, 8, 256, 64, torch.float16, True)
    x = torch.randn(2, 256, device="cuda").bfloat16()
    assert affine4_linear(x[:0], codes, scales, biases).shape == (0, 8)
    x8, xs = x.to(torch.float8_e4m3fn), torch.ones(2, 2, device="cuda")
    for call in (lambda: affine4_linear(x[:, :128], codes, scales, biases),
                 lambda: affine4_linear(x, codes.long(), scales, biases),
                 lambda: affine4_linear(x, codes, scales[:, :3], biases),
                 lambda: affine4_linear(x, codes, scales, biases.float()),
                 lambda: affine4_linear(x, codes, scales[:, :1], biases[:, :1]),
                 lambda: affine4_linear(x, codes, scales, biases, x_scales=xs),
                 lambda: affine4_linear(x8, codes, scales, biases),
                 lambda: affine4_linear(x8, codes, scales, biases, x_scales=xs.half()),
                 lambda: affine4_linear(x8, codes, scales, biases, x_scales=torch.ones(2, 16, device="cuda")),
                 lambda: affine4_linear(x.double(), codes, scales, biases),
                 lambda: affine4_linear(x, codes, scales, biases, out=torch.empty(2, 7, device="cuda")),
                 lambda: affine4_linear(x, codes, scales, biases, out=x[:, :8].reshape(-1)[:0]),
                 lambda: affine4_linear(x.view(-1)[:256], codes, scales, biases, out=x.view(-1)[100:108]),
                 lambda: affine4_linear(x[0, 0], codes, scales, biases),
                 lambda: affine4_linear(x, codes, scales, biases, out_dtype=torch.int8),
                 lambda: affine4_linear(x, codes, scales.cpu(), biases),
                 lambda: Affine4Linear(codes, scales[:4])):
        with pytest.raises(ValueError):
            call()


def _bound(xv, q, s, b, inner):
    """What the sums of a bfloat16 or float32 row may be off by: 16 s v x with v =
    1 + q / 16, and (b - 16 s) x beside it, in chains of at most in / 8 + 64
    additions that are off by a whole step each (the float16 and E4M3 sums, of
    q s x and b x, have smaller terms)."""
    terms = ((16.0 + q) * s).abs() + (b - 16.0 * s).abs()
    return (inner / 8 + 64) * 2.0 ** -23 * (xv.abs() @ terms.t())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32", "e4m3"])
@pytest.mark.parametrize("low, high", [(7, 9), (8, 8), (0, 0), (15, 15)])
@pytest.mark.parametrize("rows, inner, outer, group", [(1, 4096, 130, 128), (9, 1024, 33, 32), (3, 512, 600, 64)])
def test_codes_of_a_narrow_range_with_a_float32_output(dtype, low, high, rows, inner, outer, group):
    """Weights near zero, whose terms cancel, and weights of one value."""
    import torch

    from mlxlr8_b200.affine4 import affine4_linear

    g = torch.Generator(device="cuda").manual_seed(low * 31 + inner)
    q = torch.randint(low, high + 1, (outer, inner), generator=g, device="cuda")
    words = (q.view(outer, -1, 8) << torch.arange(0, 32, 4, device="cuda")).sum(-1)
    codes = torch.where(words >= 1 << 31, words - (1 << 32), words).int()
    scales = (torch.randn(outer, inner // group, generator=g, device="cuda") * 0.02).half()
    x = torch.randn(rows, inner, generator=g, device="cuda") + 1.0
    xs = None
    if dtype == "e4m3":
        x, xs = x.to(torch.float8_e4m3fn), torch.ones(rows, 1, device="cuda")
    else:
        x = x.to(torch_dtype(dtype))
    for biases in (None, (-7.5 * scales.float()).half()):
        got = affine4_linear(x, codes, scales, biases, x_scales=xs, out_dtype=torch.float32)
        s = scales.double().repeat_interleave(group, 1)
        b = -8.0 * s if biases is None else biases.double().repeat_interleave(group, 1)
        xv = x.float().double()
        expected = xv @ (q.double() * s + b).t()
        tol = expected.abs() * 2.0 ** -24 + _bound(xv, q.double(), s, b, inner) + 1e-30
        assert bool(((got.double() - expected).abs() <= tol).all())


def test_infinite_channels_leave_no_finite_output():
    """An infinite channel: infinities or NaN in its row, the other rows as they were."""
    import torch

    from mlxlr8_b200.affine4 import affine4_linear

    g = torch.Generator(device="cuda").manual_seed(13)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = torch.randn(3, 1024, generator=g, device="cuda").to(dtype)
        for biases in (False, True):
            weights = _weights(g, 300, 1024, 64, torch.float16, biases)
            clean = affine4_linear(x, *weights)
            for bad in (float("inf"), float("-inf"), float("nan")):
                y = x.clone()
                y[1, 900] = bad
                got = affine4_linear(y, *weights)
                assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
                assert not bool(got[1].isfinite().any())


@pytest.mark.parametrize("outer", [1, 31, 129, 4100, 5001])
def test_widths_that_end_inside_a_warp_share_channels(outer):
    """A cluster's last barrier behind rows that only some lanes store."""
    import torch

    from mlxlr8_b200.affine4 import Affine4Linear

    g = torch.Generator(device="cuda").manual_seed(outer)
    weights = _weights(g, outer, 8192, 128, torch.float16, True)
    layer = Affine4Linear(*weights)
    for rows in (1, 8, 16):
        x = torch.randn(rows, 8192, generator=g, device="cuda").half()
        first = _check(x, *weights)
        for _ in range(20):
            assert torch.equal(layer(x), first)
