"""Latent attention: keys and values from one shared latent vector a token
(``exlr8/model.py:186-343``).

A token leaves one row ``[latent (rank), rotary key (64)]`` in a paged cache
``[pages, page_size, rank + 64]``.  ``latent_append`` writes it;
``latent_attention`` attends it in the absorbed form, where every head's query
already lives in the latent space and all heads read the same rows (decoding,
drafts); ``latent_prompt_attention`` is the expanded form over per-head keys and
values (prompts).  ``LatentPages`` hands out pages, and
``LatentSelfAttention`` is a decoder block's attention made of these and the
4-bit layers, which ``stack.MoEStack`` calls.
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch

from . import _lib
from .stack import residual_rms_norm_q8

ROPE = 64
_HALVES = (torch.float16, torch.bfloat16)


def _half(name, t, dtype=None):
    if t.dtype not in _HALVES or (dtype is not None and t.dtype != dtype):
        raise ValueError(f"{name} must be float16 or bfloat16 like the other operands")


def _check_cache(cache):
    """(pages, page size, rank) of a cache."""
    shape = cache.shape
    if len(shape) != 3 or shape[2] - ROPE not in (128, 256, 384, 512):
        raise ValueError("the cache is [pages, page_size, rank + 64] with rank 128, 256, 384 or 512")
    pages, size, width = shape
    if size == 0 or size % 16:
        raise ValueError("the page size must be a multiple of 16")
    if not cache.is_contiguous():
        raise ValueError("the cache must be contiguous")
    _half("the cache", cache)
    return pages, size, width - ROPE


@lru_cache(maxsize=4096)
def _workspace_bytes(device_index, queries, heads, rank):
    """Of one call, whatever its batch."""
    with torch.cuda.device(device_index):
        return _lib.lib().exlr8_latent_attention_workspace(1, queries, heads, rank)


def _index(name, t, shape, dtype):
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} of shape {list(shape)}")
    return t.contiguous()


def _rows(t):
    """``t`` with contiguous channels (a copy if they are not)."""
    return t if t.stride(-1) == 1 else t.contiguous()


def latent_append(latent, rope_key, cache, slots, *, weight=None, eps: float = 1e-5, cos_sin=None, positions=None,
                  q_rope=None, interleaved: bool = True):
    """Write ``latent [tokens, rank]`` and ``rope_key [tokens, 64]`` to the rows
    ``slots`` (int64 [tokens], ``page * page_size + offset``) of ``cache``.

    With ``weight [rank]`` (taken in the cache's type) the latent is RMS-normed
    first.  With ``cos_sin``
    (float32 [positions, 32, 2]) and ``positions`` (int32 [tokens]) the key, and
    ``q_rope [tokens, heads, 64]`` where given, are rotated: channel pairs (2i, 2i
    + 1) when ``interleaved``, else (i, i + 32).  A slot outside the cache (-1
    for padding rows) writes nothing; so does a position outside the table,
    whose rotated queries are NaN.  The slots inside the cache have to differ: a
    row that two tokens write holds some of either.  No other operand may lie
    in the cache.  Returns the rotated queries (a new tensor), or None."""
    device = _lib.require_cuda(latent, rope_key, cache, slots, weight, cos_sin, positions, q_rope)
    pages, page_size, rank = _check_cache(cache)
    dtype = cache.dtype
    tokens = slots.numel()
    if latent.shape != (tokens, rank) or rope_key.shape != (tokens, ROPE):
        raise ValueError("latent must be [tokens, rank] and rope_key [tokens, 64], with a slot a token")
    _half("latent", latent, dtype)
    _half("rope_key", rope_key, dtype)
    slots = _index("slots", slots, (tokens,), torch.int64)
    if weight is not None:
        if weight.shape != (rank,):
            raise ValueError("the latent norm's weight must have one entry per latent channel")
        weight = _lib.like(weight, dtype)
    if (cos_sin is None) != (positions is None):
        raise ValueError("cos_sin and positions go together")
    if cos_sin is not None:
        if cos_sin.dtype != torch.float32 or cos_sin.shape != (len(cos_sin), ROPE // 2, 2):
            raise ValueError("cos_sin must be float32 [positions, 32, 2]")
        cos_sin = _lib.aligned(cos_sin)
        positions = _index("positions", positions, (tokens,), torch.int32)
    latent, rope_key = _rows(latent), _rows(rope_key)
    q_out, heads, q_strides = None, 0, (0, 0)
    if q_rope is not None:
        heads = q_rope.shape[1] if q_rope.dim() == 3 else 0
        if heads == 0 or q_rope.shape != (tokens, heads, ROPE):
            raise ValueError("q_rope must be [tokens, heads, 64]")
        _half("q_rope", q_rope, dtype)
        q_rope = _rows(q_rope)
        q_strides = q_rope.stride()[:2]
        q_out = torch.empty_like(q_rope, memory_format=torch.contiguous_format)
    _lib.call(device, _lib.lib().exlr8_latent_append, latent.data_ptr(), latent.stride(0), rope_key.data_ptr(),
              rope_key.stride(0), tokens, rank, _lib.act_code(cache), _lib.ptr(weight), float(eps), _lib.ptr(cos_sin),
              0 if cos_sin is None else cos_sin.shape[0], _lib.ptr(positions), interleaved, slots.data_ptr(),
              cache.data_ptr(), pages, page_size, _lib.ptr(q_rope), *q_strides, heads, _lib.ptr(q_out))
    return q_out


def latent_attention(q_latent, q_rope, cache, block_table, lengths, scale: float, *, out=None, return_lse: bool = False,
                     workspace=None):
    """Attention over the paged latent cache: ``softmax(scale * [q_latent,
    q_rope] . row) @ row[:rank]`` for ``q_latent [batch, queries, heads, rank]``
    and ``q_rope [batch, queries, heads, 64]``.

    Sequence ``b`` has ``lengths[b]`` (int32) tokens in the pages ``block_table[b]``
    (int32 [batch, width]); its last query sees all of them, an earlier one
    fewer by its distance from the last.  A query that sees none gives zeros.
    Rows past a length are not used, whatever they hold; a row that is not
    finite reaches every query of its sequence, earlier ones too.  With
    ``return_lse`` also float32 ``[batch, queries, heads]``, the logarithm of the
    softmax's sum (-inf where nothing was seen), by which results over parts
    of a context can be joined.  ``workspace`` (optional uint8 tensor) is used
    when it is large enough; calls that overlap need one each, and no operand
    may lie in it."""
    device = _lib.require_cuda(q_latent, q_rope, cache, block_table, lengths, out, workspace)
    pages, page_size, rank = _check_cache(cache)
    batch, queries, heads, width = q_latent.shape if q_latent.dim() == 4 else (0, 0, 0, 0)
    if width != rank or q_rope.shape != (batch, queries, heads, ROPE):
        raise ValueError("q_latent must be [batch, queries, heads, rank] and q_rope [batch, queries, heads, 64]")
    _half("q_latent", q_latent, cache.dtype)
    _half("q_rope", q_rope, cache.dtype)
    if queries == 0 or heads == 0:
        raise ValueError("latent attention needs a query and a head")
    if block_table.dim() != 2:
        raise ValueError("block_table must be int32 [batch, pages]")
    table_width = block_table.shape[1]
    block_table = _index("block_table", block_table, (batch, table_width), torch.int32)
    lengths = _index("lengths", lengths, (batch,), torch.int32)
    q_latent, q_rope = _lib.aligned(q_latent), _lib.aligned(q_rope)
    if cache.data_ptr() % 16:
        raise ValueError("the cache must start on a 16-byte boundary")
    if out is None:
        out = torch.empty_like(q_latent)
    elif out.shape != q_latent.shape or out.dtype != cache.dtype or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous tensor like q_latent")
    else:
        _lib.refuse_overlap(out, q_latent, q_rope, cache, block_table, lengths)
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous")
    lse = q_latent.new_empty((batch, queries, heads), dtype=torch.float32) if return_lse else None
    need = _workspace_bytes(device.index, queries, heads, rank)
    if need >= 1 << 62:
        raise ValueError("operand sizes or strides are outside what the operator takes")
    if workspace is None or workspace.nbytes < need:
        workspace = q_latent.new_empty(need, dtype=torch.uint8)
    _lib.call(device, _lib.lib().exlr8_latent_attention, q_latent.data_ptr(), q_rope.data_ptr(), batch, queries, heads,
              rank, _lib.act_code(cache), cache.data_ptr(), pages, page_size, block_table.data_ptr(), table_width,
              lengths.data_ptr(), float(scale), out.data_ptr(), _lib.ptr(lse), workspace.data_ptr(), workspace.nbytes)
    return (out, lse) if return_lse else out


def _heads_first(name, t, dtype):
    """``t [tokens, heads, channels]`` as the kernel takes it: contiguous
    channels, rows of their own on 16 bytes (a copy of any other view)."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, channels]")
    _half(name, t, dtype)
    a, b, c = t.stride()
    if c == 1 and a % 8 == 0 and b % 8 == 0 and (a > 0 or t.shape[0] < 2) and (b > 0 or t.shape[1] < 2) \
            and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def latent_prompt_attention(q, k, k_rope, v, q_starts, k_starts, scale: float, *, out=None, return_lse: bool = False):
    """Causal attention of ragged prompts in the expanded form: ``q [total_q,
    heads, nope + 64]``, ``k [total_k, heads, nope]``, ``k_rope [total_k, 64]``
    (shared by all heads) and ``v [total_k, heads, value]``, with ``nope`` 64, 128
    or 192 and ``value`` 64, 128, 192 or 256.  Views are taken as they are when
    their channels are contiguous (k and v of one joint projection).

    Sequence ``s`` has the queries ``q_starts[s] : q_starts[s + 1]`` and the keys
    ``k_starts[s] : k_starts[s + 1]`` (int32 [seqs + 1], ascending); its last
    query sees all its keys, an earlier one fewer by its distance from the
    last, so a chunk with a history is one call.  A query that sees none gives
    zeros.  A key or value that is not finite reaches every query of its
    sequence, earlier ones too.  Rows behind the last sequence are left as they were (in a new
    ``out``: undefined).  With ``return_lse`` also float32 ``[total_q, heads]``."""
    device = _lib.require_cuda(q, k, k_rope, v, q_starts, k_starts, out)
    _half("q", q)
    q, k, v = (_heads_first(name, t, q.dtype) for name, t in (("q", q), ("k", k), ("v", v)))
    _half("k_rope", k_rope, q.dtype)
    total_q, heads, width = q.shape
    total_k, _, nope = k.shape
    value = v.shape[2]
    if nope not in (64, 128, 192) or value not in (64, 128, 192, 256):
        raise ValueError("keys have 64, 128 or 192 channels beside the rotary ones, values 64, 128, 192 or 256")
    if width != nope + ROPE or heads == 0 or k.shape != (total_k, heads, nope) \
            or v.shape != (total_k, heads, value) or k_rope.shape != (total_k, ROPE):
        raise ValueError("q, k, k_rope and v do not match")
    if k_rope.stride(1) != 1 or k_rope.stride(0) % 8 or (k_rope.stride(0) == 0 and total_k > 1) \
            or k_rope.data_ptr() % 16:
        k_rope = k_rope.clone(memory_format=torch.contiguous_format)
    seqs = q_starts.numel() - 1
    if not 1 <= seqs <= 4096:
        raise ValueError("1 to 4096 sequences in one call")
    q_starts = _index("q_starts", q_starts, (seqs + 1,), torch.int32)
    k_starts = _index("k_starts", k_starts, (seqs + 1,), torch.int32)
    if out is None:
        out = q.new_empty((total_q, heads, value))
    elif out.shape != (total_q, heads, value) or out.dtype != q.dtype or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise ValueError("out must be a contiguous [total_q, heads, value] tensor")
    else:
        _lib.refuse_overlap(out, q, k, k_rope, v, q_starts, k_starts)
    lse = q.new_empty((total_q, heads), dtype=torch.float32) if return_lse else None
    _lib.call(device, _lib.lib().exlr8_latent_prompt_attention, q.data_ptr(), *q.stride()[:2], k.data_ptr(),
              *k.stride()[:2], k_rope.data_ptr(), k_rope.stride(0), v.data_ptr(), *v.stride()[:2], total_q, total_k,
              heads, nope, value, _lib.act_code(q), q_starts.data_ptr(), k_starts.data_ptr(), seqs, float(scale),
              out.data_ptr(), _lib.ptr(lse))
    return (out, lse) if return_lse else out


def rope_table(positions: int, base: float = 10000.0, device="cuda"):
    """float32 [positions, 32, 2] cosine and sine of ``position * base ** (-2i /
    64)``, the angles formed in float64."""
    i = torch.arange(0, ROPE, 2, dtype=torch.float64, device=device)
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / ROPE)
    return torch.stack([angles.cos(), angles.sin()], -1).float()


@dataclass
class LatentStep:
    """What one step of a batch hands to every block: where its tokens go and
    what they attend.  ``slots`` int64 and ``positions`` int32 [batch * queries],
    ``block_table`` int32 [batch, width], ``lengths`` int32 [batch] (with this
    step's tokens)."""

    slots: torch.Tensor
    positions: torch.Tensor
    block_table: torch.Tensor
    lengths: torch.Tensor
    queries: int


class LatentPages:
    """Pages of the sequences of one batch, shared by the caches of all blocks
    (each block's cache is its own tensor with the same page numbers)."""

    def __init__(self, pages: int, page_size: int = 64, device="cuda"):
        if page_size <= 0 or page_size % 16:
            raise ValueError("the page size must be a multiple of 16")
        self.page_size, self.device = page_size, torch.device(device)
        self._free = list(range(pages - 1, -1, -1))
        self._pages, self._lengths = {}, {}

    def length(self, sequence) -> int:
        return self._lengths.get(sequence, 0)

    def release(self, sequence) -> None:
        """Give a sequence's pages back."""
        self._free.extend(reversed(self._pages.pop(sequence, [])))
        self._lengths.pop(sequence, None)

    def step(self, sequences, queries: int = 1) -> LatentStep:
        """Room for ``queries`` further tokens of every listed sequence (new ones
        begin empty).  Raises before it changes anything when the pages do not
        suffice."""
        sequences = list(sequences)
        if queries < 1 or not sequences or len(set(sequences)) != len(sequences):
            raise ValueError("a step takes at least one token of distinct sequences")
        size = self.page_size
        wanted = {s: -(-(self.length(s) + queries) // size) - len(self._pages.get(s, ())) for s in sequences}
        if sum(wanted.values()) > len(self._free):
            raise ValueError("the latent cache has no free pages left")
        slots, positions, lengths = [], [], []
        for s in sequences:
            held, start = self._pages.setdefault(s, []), self.length(s)
            held.extend(self._free.pop() for _ in range(wanted[s]))
            for p in range(start, start + queries):
                positions.append(p)
                slots.append(held[p // size] * size + p % size)
            self._lengths[s] = start + queries
            lengths.append(start + queries)
        width = max(len(self._pages[s]) for s in sequences)
        table = [self._pages[s] + [-1] * (width - len(self._pages[s])) for s in sequences]

        def device(values, dtype):
            return torch.tensor(values, dtype=dtype).to(self.device)

        return LatentStep(device(slots, torch.int64), device(positions, torch.int32), device(table, torch.int32),
                          device(lengths, torch.int32), queries)


class LatentSelfAttention:
    """A decoder block's attention at decode, absorbed form: ``attention(h,
    step) -> r`` for ``h [batch * queries, hidden]``.

    ``query_latent`` (hidden -> heads * rank), ``query_rope`` (hidden -> heads * 64),
    ``key`` (hidden -> rank + 64) and ``output`` (heads * rank -> hidden) are
    ``affine4.Affine4Linear`` layers, or callables of that form; the first three
    share one 8-bit norm of ``h``.  ``cache`` is the block's own pages."""

    def __init__(self, input_norm, query_latent, query_rope, key, key_norm, output, cache, heads, scale, cos_sin,
                 eps: float = 1e-5, group: int = 128, interleaved: bool = True):
        self.rank = _check_cache(cache)[2]
        if heads < 1 or key_norm.shape != (self.rank,):
            raise ValueError("the latent norm's weight must have one entry per latent channel")
        self.input_norm, self.key_norm = input_norm, key_norm.to(cache.dtype)
        self.query_latent, self.query_rope, self.key, self.output = query_latent, query_rope, key, output
        self.cache, self.heads, self.scale, self.cos_sin = cache, heads, float(scale), cos_sin
        self.eps, self.group, self.interleaved = eps, group, interleaved

    def __call__(self, h, step: LatentStep):
        dtype, heads, rank = self.cache.dtype, self.heads, self.rank
        tokens = step.slots.numel()
        if h.dim() != 2 or h.shape[0] != tokens:
            raise ValueError("the hidden state must be [batch * queries, hidden] of the step")
        codes, scales = residual_rms_norm_q8(h, self.input_norm, self.eps, group=self.group)
        kv = self.key(codes, x_scales=scales, out_dtype=dtype)
        q_latent = self.query_latent(codes, x_scales=scales, out_dtype=dtype)
        q_rope = self.query_rope(codes, x_scales=scales, out_dtype=dtype)
        q_rope = latent_append(kv[:, :rank], kv[:, rank:], self.cache, step.slots, weight=self.key_norm, eps=self.eps,
                               cos_sin=self.cos_sin, positions=step.positions, q_rope=q_rope.view(tokens, heads, ROPE),
                               interleaved=self.interleaved)
        shape = (tokens // step.queries, step.queries, heads)
        out = latent_attention(q_latent.view(*shape, rank), q_rope.view(*shape, ROPE), self.cache, step.block_table,
                               step.lengths, self.scale)
        return self.output(out.view(tokens, heads * rank), out_dtype=h.dtype)
