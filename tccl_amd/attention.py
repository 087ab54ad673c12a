"""What the ranks of a language model do between their collectives, over the same W symmetric buffers:

* ``qk_norm_rope`` / ``qk_norm_rope_backward`` -- one-shot all-reduce of the ranks' partial query/key/value
  projections with the per-head norms and the position rotation in the same pass, and its gradients;
* ``PagedCache``, ``cache_write``, ``cache_read`` -- a paged key/value cache that spans the ranks, in bf16 or 8 bits;
* ``decode_attention`` -- one new token per sequence attends to pages on all ranks;
* ``attention_all_reduce`` -- where each rank attends to its own part of the tokens, the join of the W partial
  attentions: an all-reduce whose weights are a softmax over the ranks.

As in ``collectives``: arguments are checked on the host before anything is launched, outputs are allocated with
torch unless the caller passes them, kernels run on torch's current stream of the tensors' device, nothing
synchronises, and every call can be captured into a HIP graph.  Inside ``spmd.run`` every rank makes the call,
except ``cache_write``, which a rank may make alone.  None of these functions records anything for autograd.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
from typing import Optional, Tuple, Union

import torch

from . import _lib, spmd
from .collectives import _check_out, _refuse_remote, _stream, _sum_dtype
from .symm import rendezvous, SymmGroup

HEAD_DIMS = (64, 128, 256)
PAGE_SIZES = (16, 32, 64, 128, 256)
_STORES = {torch.bfloat16: _lib.TCCL_BF16, torch.float8_e4m3fn: _lib.TCCL_E4M3}


_HERE = contextlib.nullcontext()
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _collective():
    """``spmd.collective()`` where the caller is a rank of a per-rank program, else nothing to wait for."""
    return _HERE if spmd.current_rank() is None else spmd.collective()


def _on(device: torch.device):
    """Launches go to the device of the tensors, whichever is current."""
    if device.type != "cuda":
        raise ValueError(f"the kernels take tensors on a GPU, not on {device}")
    return _HERE if device.index == _current_device() else torch.cuda.device(device)


@functools.lru_cache(maxsize=1024)
def _attention_workspace(batch: int, q_heads: int, kv_heads: int, dim: int, most: int, device: torch.device) -> int:
    return _lib.load().tccl_decode_attention_workspace(batch, q_heads, kv_heads, dim, most)


@functools.lru_cache(maxsize=64)
def _grad_workspace(dim: int, device: torch.device) -> int:
    return _lib.load().tccl_qk_norm_rope_backward_workspace(dim)


def _need(condition: bool, text: str) -> None:
    if not condition:
        raise ValueError(text)


def _integers(t: torch.Tensor, dtype: torch.dtype, shape, device: torch.device, name: str) -> None:
    if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")


def _aligned(t: torch.Tensor, name: str) -> None:
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must start at a multiple of 16 bytes")


def _heads_first(t: torch.Tensor, name: str) -> Tuple[int, int]:
    """Strides (in elements) of a ``[tokens, heads, head_dim]`` tensor whose rows are whole and 16-byte aligned."""
    if t.numel() == 0:
        return 0, 0
    token, head, element = t.stride()
    if t.shape[0] == 1:                # (the stride of a dimension of one means nothing)
        token = 0
    if t.shape[1] == 1:
        head = 0
    vec = 16 // t.element_size()
    if element != 1 or token % vec or head % vec or t.data_ptr() % 16:
        raise ValueError(f"{name}: rows of head_dim elements must be contiguous and start at multiples of 16 bytes")
    return token, head


def _refuse_overlap(out: torch.Tensor, buffers: Tuple[int, ...], nbytes: int, in_place: bool) -> None:
    """``out`` must not lie over the first ``nbytes`` of the ranks' buffers, except from one's very start if ``in_place``."""
    start = out.data_ptr()
    stop = start + out.numel() * out.element_size()
    for p in buffers:
        if start < p + nbytes and p < stop and not (in_place and start == p):
            raise ValueError("out must not overlap what the ranks' launches read")


# ---------------------------------------------------------------- sum, per-head norm and rotation

def _norm_arguments(tensor, q_weight, k_weight, positions, inv_freq, heads, what):
    dtype = _sum_dtype(tensor)
    dim = q_weight.numel()
    device = tensor.device
    if dim not in HEAD_DIMS:
        raise ValueError(f"{what}: head_dim (the weights' length) must be one of {HEAD_DIMS}")
    if tensor.dim() != 2:
        raise ValueError(f"{what}: the projection must be [tokens, columns]")
    for w in (q_weight, k_weight):
        if w.dtype != tensor.dtype or w.shape != (dim,) or w.device != device or not w.is_contiguous() or w.data_ptr() % 16:
            raise ValueError(f"{what}: the weights must be contiguous {tensor.dtype} tensors of shape ({dim},) on {device} that "
                             "start at a multiple of 16 bytes")
    tokens, columns = tensor.shape
    if min(heads) < 0 or sum(heads) < 1 or sum(heads) * dim != columns:
        raise ValueError(f"{what}: {columns} columns are not {heads[0]} + {heads[1]} + {heads[2]} heads of {dim}")
    _integers(positions, torch.int64, (tokens,), device, "positions")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float64 or inv_freq.device != device or not inv_freq.is_contiguous():
        raise ValueError(f"{what}: inv_freq must be a contiguous float64 vector on {device}")
    rotary = 2 * inv_freq.numel()
    if rotary % 16 or rotary > dim:
        raise ValueError(f"{what}: 2 * len(inv_freq) must be a multiple of 16 and at most head_dim")
    return dtype, dim, rotary


def qk_norm_rope(tensor: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                 inv_freq: torch.Tensor, q_heads: int, k_heads: int, *, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """All-reduce (sum) of the ranks' partial projections, then each query and key head normed and rotated.

    ``tensor`` is this rank's ``[tokens, columns]`` buffer (bfloat16 or float32) of a symmetric group, columns holding
    ``q_heads`` query heads, ``k_heads`` key heads and, in what is left, value heads, of ``len(q_weight)`` elements
    each (64, 128 or 256).  A query or key head becomes ``R(position) (x / sqrt(mean(x^2) + eps) * weight)``, where R
    turns the first ``2 * len(inv_freq)`` elements (a multiple of 16) in pairs (i, i + half), or (2i, 2i + 1) if
    ``interleaved``, by ``positions[t] * inv_freq[i]``: positions are int64, inv_freq float64, and the angle is reduced
    in fp64, so that far positions keep their precision.  Value heads are only summed.  Everything is fp32 and rounded
    once.  ``eps`` may be 0, where a head of zeros has no norm and gives NaN.  A head whose sum of squares passes fp32's
    range (elements of about 2^61 and more) becomes 0, with gradients of 0; for eps = 0 one below it loses its norm.
    Returns q, k, v as ``[tokens, heads, head_dim]``.

    With a group of one rank it is the plain norm and rotation."""
    dim = q_weight.numel()
    v_heads = tensor.shape[-1] // max(dim, 1) - q_heads - k_heads
    heads = (q_heads, k_heads, v_heads)
    dtype, dim, rotary = _norm_arguments(tensor, q_weight, k_weight, positions, inv_freq, heads, "qk_norm_rope")
    lib = _lib.load()
    with _collective():
        tokens = tensor.shape[0]
        q, k, v = (tensor.new_empty((tokens, q_heads, dim)), tensor.new_empty((tokens, k_heads, dim)),
                   tensor.new_empty((tokens, v_heads, dim)))
        if tokens == 0:                # (an empty view has no address to find a group by)
            return q, k, v
        symm = rendezvous(tensor)
        _refuse_remote(symm.group, "qk_norm_rope")
        symm.group.check_signals()
        with _on(tensor.device):
            rc = lib.tccl_qk_norm_rope(symm.buffer_ptrs_host, symm.world_size, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                       q_weight.data_ptr(), k_weight.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(),
                                       tokens, q_heads, k_heads, v_heads, dim, rotary, interleaved, eps, dtype,
                                       _stream(tensor.device))
        _lib.check("tccl_qk_norm_rope", rc)
    return q, k, v


def qk_norm_rope_backward(dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, tensor: torch.Tensor,
                          q_weight: torch.Tensor, k_weight: torch.Tensor, positions: torch.Tensor,
                          inv_freq: torch.Tensor, *, eps: float = 1e-6, interleaved: bool = False
                          ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of ``qk_norm_rope`` from the gradients of its three outputs (contiguous ``[tokens, heads, head_dim]``
    in ``tensor``'s dtype) and its inputs, whose buffers must still hold the partial projections (the sum, norm and
    rotation angles are formed again; nothing is kept from the forward pass).

    Returns ``(dx, dq_weight, dk_weight)``: dx ``[tokens, columns]`` in ``tensor``'s dtype is the gradient of every
    rank's buffer alike; the weights' gradients are float32, summed in a fixed order."""
    heads = tuple(g.shape[1] if g.dim() == 3 else -1 for g in (dq, dk, dv))
    dtype, dim, rotary = _norm_arguments(tensor, q_weight, k_weight, positions, inv_freq, heads, "qk_norm_rope_backward")
    tokens = tensor.shape[0]
    for g, n in zip((dq, dk, dv), heads):
        if g.shape != (tokens, n, dim) or g.dtype != tensor.dtype or g.device != tensor.device or not g.is_contiguous() \
                or (g.data_ptr() % 16 and g.numel()):
            raise ValueError(f"dq, dk and dv must be contiguous {tensor.dtype} tensors of shape [{tokens}, heads, {dim}] on "
                             f"{tensor.device} that start at a multiple of 16 bytes")
    lib = _lib.load()
    with _collective():
        device = tensor.device
        dx = torch.empty_like(tensor)
        if tokens == 0:
            return dx, torch.zeros(dim, device=device), torch.zeros(dim, device=device)
        symm = rendezvous(tensor)
        _refuse_remote(symm.group, "qk_norm_rope_backward")
        symm.group.check_signals()
        dweights = tensor.new_empty((2, dim), dtype=torch.float32)
        with _on(device):
            nbytes = _grad_workspace(dim, device)
            workspace = tensor.new_empty(nbytes, dtype=torch.uint8)
            first = dweights.data_ptr()
            rc = lib.tccl_qk_norm_rope_backward(
                symm.buffer_ptrs_host, symm.world_size, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), q_weight.data_ptr(),
                k_weight.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), dx.data_ptr(), first, first + 4 * dim,
                workspace.data_ptr(), nbytes, tokens, *heads, dim, rotary, interleaved, eps, dtype, _stream(device))
        _lib.check("tccl_qk_norm_rope_backward", rc)
    return (dx, *dweights.unbind(0))


# ---------------------------------------------------------------- the paged cache

class PagedCache:
    """A paged key/value cache that spans the ranks: W symmetric buffers (``group``) of ``pages_per_rank`` pages of
    ``page_size`` tokens (16, 32, 64, 128 or 256).  Pages are numbered over all ranks, rank r holding pages
    ``[r * pages_per_rank, (r + 1) * pages_per_rank)``; a *slot* is ``page * page_size + place in the page``.  Which
    sequence has which pages, on which ranks, is the caller's table.

    ``dtype``: ``torch.bfloat16``, or ``torch.float8_e4m3fn`` with one power-of-two scale per token and head, formed as
    the token is written; stored values are bfloat16 numbers either way.  The layout inside a page is the library's own.
    A new cache holds zeros.

    Its buffers come from the current stream, which another stream has to wait for before it uses the cache.  It may be
    dropped while streams still work on it: the allocator keeps the buffers until those that it was used on have passed
    that point.  A captured graph holds their addresses only, so the cache has to live as long as the graph is replayed.

    The constructor makes all W buffers.  For a program under ``spmd.run`` the ranks' common cache is therefore made
    outside and handed to it; one that a rank makes inside is that rank's own."""

    def __init__(self, world_size: int, pages_per_rank: int, page_size: int, kv_heads: int, head_dim: int, *,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        _need(1 <= world_size <= _lib.MAX_WORLD, f"world_size must be 1 to {_lib.MAX_WORLD}")
        _need(dtype in _STORES, "a paged cache holds torch.bfloat16 or torch.float8_e4m3fn")
        _need(head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}")
        _need(page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}")
        _need(1 <= kv_heads <= 65535, "kv_heads must be 1 to 65535")
        _need(pages_per_rank >= 1 and pages_per_rank * world_size < 1 << 31, "page numbers must fit 31 bits")
        self.world_size, self.pages_per_rank, self.page_size = world_size, pages_per_rank, page_size
        self.kv_heads, self.head_dim, self.dtype = kv_heads, head_dim, dtype
        self.pages = world_size * pages_per_rank
        self.slots = self.pages * page_size
        desc = _lib.PagedCacheDesc()
        desc.world, desc.pages_per_rank, desc.page_size = world_size, pages_per_rank, page_size
        desc.kv_heads, desc.head_dim, desc.dtype = kv_heads, head_dim, _STORES[dtype]
        nbytes = _lib.load().tccl_paged_cache_bytes(ctypes.byref(desc))
        _need(nbytes > 0, "a rank's buffer must be under 2^63 bytes")
        # a group of its own, but not one that rendezvous finds: its buffers are no operand of a collective
        self.group = SymmGroup([torch.zeros(nbytes, dtype=torch.uint8, device=device) for _ in range(world_size)])
        self.group.handles.clear()     # (they point back at the group: the buffers would outlive the cache until a collection)
        self.device = self.group.tensors[0].device
        for r, p in enumerate(self.group.buffer_ptrs):
            desc.bufs[r] = p
        self._desc = desc
        self._ref = ctypes.byref(desc)
        self._streams = {_stream(self.device).value} if self.device.type == "cuda" else set()

    def _launch_stream(self) -> ctypes.c_void_p:
        """The current stream.  The first launch on one that the buffers do not come from tells the allocator of it."""
        stream = _stream(self.device)
        if stream.value not in self._streams and not torch.cuda.is_current_stream_capturing():    # (capturing runs nothing)
            current = torch.cuda.current_stream(self.device)
            for t in self.group.tensors:
                t.record_stream(current)
            self._streams.add(stream.value)
        return stream

    def _rows(self, tokens: int) -> Tuple[int, int, int]:
        return tokens, self.kv_heads, self.head_dim


def cache_write(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Write keys and values ``[tokens, kv_heads, head_dim]`` (bfloat16 or float32; any token and head strides of whole
    16-byte vectors) into the cache at ``slots`` (int64).  A negative slot, or one outside the cache, is not written
    (padding); the slots of one call must differ from each other."""
    dtype = _sum_dtype(k)
    tokens = slots.numel()
    rows, device = (tokens, cache.kv_heads, cache.head_dim), cache.device
    if k.shape != rows or v.shape != rows or v.dtype != k.dtype or k.device != device or v.device != device:
        raise ValueError(f"k and v must be tensors of one dtype, of shape {rows}, on {device}")
    strides = _heads_first(k, "k") + _heads_first(v, "v")
    _integers(slots, torch.int64, (tokens,), cache.device, "slots")
    if tokens == 0:
        return
    with _on(cache.device):
        rc = _lib.load().tccl_cache_write(cache._ref, k.data_ptr(), v.data_ptr(), *strides, slots.data_ptr(), tokens,
                                          dtype, cache._launch_stream())
    _lib.check("tccl_cache_write", rc)


def cache_read(cache: PagedCache, slots: torch.Tensor, *, dtype: torch.dtype = torch.bfloat16,
               out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values at ``slots`` (int64, any order, repeats allowed) as two ``[tokens, kv_heads, head_dim]`` tensors of
    ``dtype`` (bfloat16 or float32; both hold the stored values exactly): a gather over the ranks.  A negative slot, or
    one outside the cache, reads as zeros.  Slots that follow each other cost least: of every 8 (bfloat16) or 16 (8 bits)
    neighbouring tokens' values all are read for one."""
    tokens = slots.numel()
    _integers(slots, torch.int64, (tokens,), cache.device, "slots")
    _need(dtype in (torch.bfloat16, torch.float32), "cache_read returns bfloat16 or float32")
    if out is None:
        k, v = slots.new_empty((2, tokens, cache.kv_heads, cache.head_dim), dtype=dtype).unbind(0)     # one allocation
    else:
        k, v = out
        for t, name in ((k, "out[0]"), (v, "out[1]")):
            if t.shape != cache._rows(tokens) or t.dtype != dtype or t.device != cache.device or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {cache._rows(tokens)} on {cache.device}")
    code = _sum_dtype(k)
    with _collective():
        if tokens:
            _aligned(k, "out[0]")
            _aligned(v, "out[1]")
            with _on(cache.device):
                rc = _lib.load().tccl_cache_read(cache._ref, slots.data_ptr(), tokens, k.data_ptr(), v.data_ptr(), code,
                                                 cache._launch_stream())
            _lib.check("tccl_cache_read", rc)
    return k, v


# ---------------------------------------------------------------- attention

def decode_attention(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
                     scale: Optional[float] = None, max_length: Optional[int] = None, return_lse: bool = False,
                     out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None
                     ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of one new token per sequence over the cached tokens of all ranks.

    ``q``: ``[batch, q_heads, head_dim]`` bfloat16 (any strides of whole 16-byte vectors), q_heads a multiple of the
    cache's kv_heads; query head i reads key head ``i // (q_heads // kv_heads)``.  ``page_table``: int32 ``[batch, pages]``
    (rows may be strided), page numbers of each sequence in order; ``lengths``: int32 ``[batch]``, how many tokens each
    has.  Entries behind a sequence's last page are not looked at, and tokens on a page number outside the cache are
    left out.  ``max_length``: an upper bound of the lengths that the host knows (default: what the table has room for);
    the launch is shaped for it, and tokens beyond it are left out.

    Returns ``[batch, q_heads, head_dim]`` bfloat16 and, with ``return_lse`` or ``lse``, the logarithm of the softmax's
    sum, float32 ``[batch, q_heads]``: what ``attention_all_reduce`` joins parts with.  A sequence without tokens gives
    0 and -inf.  Scores, softmax and sums are fp32; an infinite cached value gives NaN, and so may finite ones whose sum,
    weighted by up to 1 each, passes fp32's range before it is divided.  ``out`` may be q itself where q is contiguous and
    no other rank's call reads it; otherwise outputs must not overlap inputs."""
    batch, dim, device = lengths.numel(), cache.head_dim, cache.device
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[0] != batch or q.shape[2] != dim or q.device != device:
        raise ValueError(f"q must be a bfloat16 tensor of shape [{batch}, q_heads, {dim}] on {device}")
    q_heads = q.shape[1]
    if q_heads < 1 or q_heads % cache.kv_heads:
        raise ValueError("q_heads must be a multiple of the cache's kv_heads")
    q_strides = _heads_first(q, "q")
    _integers(lengths, torch.int32, (batch,), device, "lengths")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != batch or page_table.device != device:
        raise ValueError(f"page_table must be an int32 tensor of shape [{batch}, pages] on {device}")
    width, (row, element) = page_table.shape[1], page_table.stride()
    if width > 1 and element != 1:
        raise ValueError("page_table: a row must be contiguous")
    most = width * cache.page_size
    if max_length is not None:
        if max_length < 0:
            raise ValueError("max_length must not be negative")
        most = min(most, max_length)
    if most > 1 << 30:
        raise ValueError("page_table has room for more than 2^30 tokens: give max_length")
    shape = (batch, q_heads, dim)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    else:
        _check_out(out, shape, q)
    if lse is not None:
        _integers(lse, torch.float32, (batch, q_heads), device, "lse")
    elif return_lse:
        lse = q.new_empty((batch, q_heads), dtype=torch.float32)
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    with _collective():
        if batch:
            _aligned(out, "out")
            with _on(device):
                nbytes = _attention_workspace(batch, q_heads, cache.kv_heads, dim, most, device)
                workspace = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
                rc = _lib.load().tccl_decode_attention(
                    cache._ref, q.data_ptr(), *q_strides, page_table.data_ptr(), row, lengths.data_ptr(), out.data_ptr(),
                    lse.data_ptr() if lse is not None else None, workspace.data_ptr() if nbytes else None, nbytes, batch, q_heads,
                    most, scale, cache._launch_stream())
            _lib.check("tccl_decode_attention", rc)
    return (out, lse) if lse is not None else out


def attention_all_reduce(tensor: torch.Tensor, lse: torch.Tensor, *, out: Optional[torch.Tensor] = None
                         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Join of the ranks' partial attentions over disjoint parts of the tokens: an all-reduce
    ``sum_i w_i tensor_i / sum_i w_i`` with ``w_i = exp(lse_i - max)``, beside ``one_shot_all_reduce``.

    ``tensor``: this rank's ``[..., head_dim]`` buffer (bfloat16 or float32, head_dim 64, 128 or 256) of one symmetric
    group, ``lse``: its float32 ``[...]`` buffer of another, both as ``decode_attention(out=, lse=)`` fills them.  Returns
    the joined output and its lse, the same on every rank.  A rank whose lse is -inf is left out, whatever its buffer
    holds; where all are, the output is 0 and lse -inf.  ``out`` may be a rank's buffer where this call is the only one (not
    inside ``spmd.run``, where other ranks' launches still read it); any other overlap is refused.  The weighted sum is fp32
    and divided at the end: finite values past 2^128 / world_size may give infinity."""
    dtype = _sum_dtype(tensor)
    if tensor.dim() < 1 or tensor.shape[-1] not in HEAD_DIMS:
        raise ValueError(f"attention_all_reduce: head_dim must be one of {HEAD_DIMS}")
    if lse.dtype != torch.float32 or lse.shape != tensor.shape[:-1] or lse.device != tensor.device:
        raise ValueError(f"lse must be a float32 tensor of shape {tuple(tensor.shape[:-1])} on {tensor.device}")
    lib = _lib.load()
    with _collective():
        if lse.numel() == 0:           # (an empty view has no address to find a group by)
            return torch.empty_like(tensor) if out is None else _check_out(out, tensor.shape, tensor), torch.empty_like(lse)
        symm, symm_lse = rendezvous(tensor), rendezvous(lse)
        _refuse_remote(symm.group, "attention_all_reduce")
        _refuse_remote(symm_lse.group, "attention_all_reduce")
        if symm.world_size != symm_lse.world_size or symm.rank != symm_lse.rank:
            raise ValueError("attention_all_reduce: tensor and lse must be the same rank's buffers of two groups of one world")
        symm.group.check_signals()
        symm_lse.group.check_signals()
        output = torch.empty_like(tensor) if out is None else _check_out(out, tensor.shape, tensor)
        if out is not None:
            _refuse_overlap(out, symm.buffer_ptrs, lse.numel() * tensor.shape[-1] * tensor.element_size(),
                            in_place=spmd.current_rank() is None or symm.world_size == 1)
            _refuse_overlap(out, symm_lse.buffer_ptrs, lse.numel() * 4, in_place=False)
        output_lse = torch.empty_like(lse)
        _aligned(output, "out")
        with _on(tensor.device):
            rc = lib.tccl_attention_all_reduce(symm.buffer_ptrs_host, symm_lse.buffer_ptrs_host, symm.world_size,
                                               output.data_ptr(), output_lse.data_ptr(), lse.numel(),
                                               tensor.shape[-1], dtype, _stream(tensor.device))
        _lib.check("tccl_attention_all_reduce", rc)
    return output, output_lse
