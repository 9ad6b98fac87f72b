"""Linear layers with 4-bit affine weights and group scales (the affine4 dense
format of ``exlr8/dense.py``; the layout of MLX ``quantize(bits=4)``).

A weight row is ``in / 8`` words of eight codes, low nibble first, and one
scale and bias per group of 32, 64 or 128 channels: ``w = scale * q + bias``.
Without biases the format is symmetric, ``w = scale * (q - 8)``.  Activations
are 16- or 32-bit floats, or the E4M3 codes and scales that
``stack.residual_rms_norm_q8`` writes.  The kernel streams the codes once for
up to 16 rows of activations: it is made for decoding.
"""

from __future__ import annotations

import torch

from . import _lib

_GROUPS = (32, 64, 128)


def _check_weights(codes, scales, biases):
    """(in_features, out_features, group) of one layer's weights."""
    if codes.dim() != 2 or codes.dtype not in (torch.int32, torch.uint32):
        raise ValueError("codes must be a [out, in / 8] tensor of 32-bit words")
    out_features, words = codes.shape
    if scales.dim() != 2 or scales.shape[0] != out_features or scales.shape[1] == 0 or (8 * words) % scales.shape[1]:
        raise ValueError("scales must be [out, in / group]")
    group = 8 * words // scales.shape[1]
    if group not in _GROUPS:
        raise ValueError("the weights' group must be 32, 64 or 128 channels")
    if biases is not None and (biases.shape != scales.shape or biases.dtype != scales.dtype):
        raise ValueError("biases must have the shape and dtype of the scales")
    if scales.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"unsupported scale dtype {scales.dtype}")
    return 8 * words, out_features, group


def affine4_linear(x, codes, scales, biases=None, *, x_scales=None, out_dtype=None, out=None):
    """``x @ w.T`` for ``x [..., in]`` -> ``[..., out]``, summed in float32 and
    rounded once to ``out_dtype`` (x's; bfloat16 for E4M3 codes).

    An infinite channel leaves infinities or NaN in its row.  The sums round
    like sums of ``scale * (16 + q) * x``, also where weights are near zero.
    ``x_scales [..., in / g]`` (float32, ``g`` 32, 64, 128 or ``in``) belongs to
    ``x`` of dtype float8_e4m3fn.  ``out`` (optional) receives the result."""
    device = _lib.require_cuda(x, codes, scales, biases, x_scales, out)
    in_features, out_features, group = _check_weights(codes, scales, biases)
    if x.dim() == 0 or x.shape[-1] != in_features:
        raise ValueError("activation width does not match in_features")
    lead = x.shape[:-1]
    x_group = in_features
    if x.dtype == torch.float8_e4m3fn:
        if x_scales is None or x_scales.dtype != torch.float32 or x_scales.shape[:-1] != lead \
                or x_scales.shape[-1] == 0 or in_features % x_scales.shape[-1]:
            raise ValueError("E4M3 activations take float32 x_scales [..., in / group]")
        x_group = in_features // x_scales.shape[-1]
        if x_group != in_features and x_group not in _GROUPS:
            raise ValueError("the activations' group must be 32, 64, 128 or the row's width")
        x_code, x_scales = _lib.E4M3_CODE, x_scales.contiguous()
    elif x_scales is not None:
        raise ValueError("x_scales belong to float8_e4m3fn activations")
    else:
        x_code = _lib.act_code(x)
    if out is None:
        dtype = out_dtype or (torch.bfloat16 if x_scales is not None else x.dtype)
        out = scales.new_empty(lead + (out_features,), dtype=dtype)
    elif out.shape != lead + (out_features,) or not out.is_contiguous() or out_dtype not in (None, out.dtype):
        raise ValueError("out must be a contiguous [..., out] tensor")
    else:
        _lib.refuse_overlap(out, x, codes, scales, biases, x_scales)
    x, codes, scales = _lib.aligned(x), _lib.aligned(codes), scales.contiguous()
    biases = biases.contiguous() if biases is not None else None
    _lib.call(device, _lib.lib().exlr8_affine4_linear, x.data_ptr(), x_code, _lib.ptr(x_scales), x_group,
              x.numel() // in_features, in_features, out_features, codes.data_ptr(), scales.data_ptr(),
              _lib.ptr(biases), _lib.act_code(scales), group, out.data_ptr(), _lib.act_code(out))
    return out


class Affine4Linear:
    """One layer's weights, checked and laid out once."""

    def __init__(self, codes, scales, biases=None):
        self.in_features, self.out_features, self.group = _check_weights(codes, scales, biases)
        if any(t is not None and t.device != codes.device for t in (scales, biases)):
            raise ValueError("operands are on different devices")
        self.codes, self.scales = _lib.aligned(codes), scales.contiguous()
        self.biases = biases.contiguous() if biases is not None else None

    def __call__(self, x, x_scales=None, out_dtype=None, out=None):
        return affine4_linear(x, self.codes, self.scales, self.biases, x_scales=x_scales, out_dtype=out_dtype, out=out)
