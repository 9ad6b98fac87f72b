"""A stack of MoE decoder blocks (exlr8 model.py:373-418).

Each block of the reference decoder layer is

    r, _ = self_attn(rms_norm(x, input_norm))       a block's attention (without one: r = 0)
    h = x + r
    x = rms_norm(h, post_norm, eps)                  exlr8_residual_rms_norm
    return h + moe(x)                                the MoE layer, residual h

A block's attention is any callable ``attention(h, step) -> r`` that norms its
own input, such as ``latent.LatentSelfAttention``, and ``step`` is what the
stack's call hands to every block's attention (``latent.LatentStep``).  With
the attention stubbed the stack threads the hidden state through
``rms_norm`` and one MoE layer per block: ``MoELayer`` (one GPU, resident
trellis experts), ``JoinedMoELayer`` (MXFP4) or ``ExpertParallelMoE``
(experts sharded over the node's GPUs).  The reference model runs layers
3-77 this way (the first three are dense) plus the layer-78 block whose
experts are K3; any callable ``layer(x, residual) -> h + moe(x)`` fits.
"""

from __future__ import annotations

import torch

from . import _lib


def residual_rms_norm(x, weight, eps: float = 1e-5, residual=None, return_sum: bool = False):
    """``rms_norm(x + residual, weight, eps)`` in x's dtype
    (model.py:383-384; fast_norm.residual_rms_pair).  With ``return_sum`` the
    rounded sum ``h`` is returned as well."""
    if residual is not None and residual.numel() != x.numel():
        raise ValueError("the residual must have the size of x")
    device = _lib.require_cuda(x, weight, residual)
    hidden = x.shape[-1]
    if weight.shape != (hidden,):
        raise ValueError("norm weight must have one entry per hidden channel")
    x = x.contiguous()
    rows = x.numel() // hidden
    w = weight.to(x.dtype).contiguous()
    out = torch.empty_like(x)
    h = torch.empty_like(x) if return_sum else None
    res = residual.to(x.dtype).contiguous() if residual is not None else None
    _lib.check(_lib.lib().exlr8_residual_rms_norm(x.data_ptr(), res.data_ptr() if res is not None else None,
                                                  w.data_ptr(), _lib.act_code(x), rows, hidden, float(eps),
                                                  h.data_ptr() if h is not None else None, out.data_ptr(),
                                                  _lib.stream_handle(device)))
    return (h, out) if return_sum else out


def residual_rms_norm_q8(x, weight, eps: float = 1e-5, residual=None, group: int = 128, return_sum: bool = False):
    """``rms_norm(x + residual, weight, eps)`` as E4M3 codes with a float32
    scale per ``group`` channels (32, 64, 128 or all of a row's): the input of
    a product that takes 8-bit activations (``affine4.affine4_linear``).

    Returns ``(codes float8_e4m3fn [..., hidden], scales float32 [..., hidden
    // group])``, with ``return_sum`` the rounded sum ``h`` in front of them.
    The norm of ``h`` stays in float32 until ``code = e4m3(y / scale)``, ``scale
    = max|y| / 448``.  A group of zeros, or whose scale lies below the smallest
    float32, has scale 0; a group with a value that is not finite has scale NaN
    and codes 0.  The residual and the weight are taken in x's dtype."""
    device = _lib.require_cuda(x, weight, residual)
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError("the norm needs a channel")
    hidden = shape[-1]
    if weight.shape != (hidden,):
        raise ValueError("norm weight must have one entry per hidden channel")
    if residual is not None and residual.shape != shape:
        raise ValueError("the residual must have the shape of x")
    if group != hidden and (group not in (32, 64, 128) or hidden % group):
        raise ValueError("group must be 32, 64, 128 or the row's width, and divide it")
    code = _lib.act_code(x)
    x = x.contiguous()
    w, res = _lib.like(weight, x.dtype), _lib.like(residual, x.dtype)
    codes = torch.empty_like(x, dtype=torch.float8_e4m3fn)
    scales = x.new_empty((*shape[:-1], hidden // group), dtype=torch.float32)
    h = torch.empty_like(x) if return_sum else None
    _lib.call(device, _lib.lib().exlr8_residual_rms_norm_q8, x.data_ptr(), _lib.ptr(res), w.data_ptr(), code,
              x.numel() // hidden, hidden, group, float(eps), _lib.ptr(h), codes.data_ptr(), scales.data_ptr())
    return (h, codes, scales) if return_sum else (codes, scales)


class MoEStack:
    """Blocks of (post-attention norm weight [hidden], MoE layer) or (weight,
    MoE layer, attention) applied in order to the hidden state [tokens,
    hidden]."""

    def __init__(self, blocks, eps: float = 1e-5):
        self.blocks = [tuple(block) for block in blocks]
        if any(len(block) not in (2, 3) for block in self.blocks):
            raise ValueError("a block is (norm weight, MoE layer) or (norm weight, MoE layer, attention)")
        self.eps = eps

    def __len__(self):
        return len(self.blocks)

    def __call__(self, h, trace: bool = False, step=None):
        """The hidden state after every block; with ``trace`` also the list of
        (MoE residual, normalised input, block output) per block.  ``step`` is
        passed to the blocks' attentions."""
        steps = []
        for w, layer, *attention in self.blocks:
            attention = attention[0] if attention else None
            if attention is None:
                xn = residual_rms_norm(h, w, self.eps)
            else:
                h, xn = residual_rms_norm(h, w, self.eps, residual=attention(h, step), return_sum=True)
            out = layer(xn, h)
            if trace:
                steps.append((h, xn, out))
            h = out
        return (h, steps) if trace else h
