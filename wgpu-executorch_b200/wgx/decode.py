"""Text decoding over a paged key/value cache: direct calls on torch tensors.

One step of generation is ``kv_append`` (the new tokens' K and V rows enter the
cache), ``paged_attention`` (their attention over it), now and then
``cache_evict`` (the slots with the least accumulated attention weight leave),
and ``beam_search_step`` (the next tokens, with the cache's state reordered).
The same operators are recorded into a context's graph through
``wgx.shaders.kvAppend``, ``pagedAttention``, ``cacheEvict`` and
``beamSearchStep``; include/wgx.h has their definitions.

A cache is a pair of tensors ``[pages, kv_heads, page_size, head_dim]``, float16
or float32, with any strides but a unit last one (a slot-major pool is passed
as ``pool.transpose(1, 2)``). ``page_table[b, s // page_size]`` is the page of
slot ``s`` of sequence ``b``; ``lengths[b]`` slots are in use. Lengths and page
tables stay on the device: a call never waits for them. A page id or length
that lies outside the cache is left out and noted (``device_error``); the calls
that write leave a sequence of such a length as it is.

Calls are enqueued on the tensors' device's current stream. Outputs are
arguments; nothing is kept between calls. Scratch memory comes from torch's
allocator unless ``workspace`` (a uint8 tensor) is given. The operators are for
inference: results carry no gradient, whatever the inputs require; what a call
writes counts as modified in place.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._lib import WgxError

try:
    from . import _torch_binding as _binding
except ImportError as e:  # no fallback: nothing may run on another path unseen
    raise ImportError(f"wgx._torch_binding is not built: run `make -C {_lib.PKG_DIR}` ({e})") from e

_ENTRY_POINTS = ("wgx_last_error", "wgx_kv_append", "wgx_paged_attention_scratch_bytes", "wgx_paged_attention",
                 "wgx_cache_evict", "wgx_beam_search_scratch_bytes", "wgx_beam_search_step")
_binding.init(WgxError, {n: ctypes.cast(getattr(_lib.lib, n), ctypes.c_void_p).value for n in _ENTRY_POINTS})


def kv_append(k, v, k_cache, v_cache, page_table, lengths, lengths_out, *, seen=None, seen_out=None,
              positions=None, weights=None) -> None:
    """Writes ``k``, ``v`` [batch, tokens, kv_heads, head_dim] behind the slots
    in use; ``lengths_out = lengths + tokens`` (may be ``lengths``). With
    ``seen`` / ``seen_out`` [batch] and ``positions``, ``weights`` [batch,
    kv_heads, slots]: the new slots get position ``seen[b] + t`` and weight 0.
    A sequence whose page table has no room for all of them gets none."""
    _binding.kv_append(k, v, k_cache, v_cache, page_table, lengths, lengths_out, seen, seen_out, positions,
                       weights)


def paged_attention(q, k_cache, v_cache, page_table, lengths, out=None, *, scale: Optional[float] = None,
                    window: int = 0, mask=None, weights=None, weights_out=None, workspace=None):
    """Attention of one token per sequence, ``q`` [batch, q_heads, head_dim]
    (``q_heads`` a multiple of the cache's K/V heads), over the slots in use;
    returns ``out`` (allocated when not given). ``scale``: 1 / sqrt(head_dim)
    by default; ``window`` > 0: the last ``window`` slots only; ``mask``
    [batch, n] bool: slots to attend to. ``weights`` / ``weights_out``
    [batch, kv_heads, slots] float32 (may be the same tensor): ``weights_out =
    weights +`` the probabilities of each K/V head's query heads, summed."""
    return _binding.paged_attention(q, k_cache, v_cache, page_table, lengths, out, scale, window, mask, weights,
                                    weights_out, workspace)


def cache_evict(k_cache, v_cache, page_table, lengths, lengths_out, weights, weights_out, positions,
                positions_out, seen, *, budget: int, recent: int = 0, sinks: int = 0) -> None:
    """Shrinks every sequence of more than ``budget`` slots to ``budget``
    slots, per K/V head: those at positions >= ``seen[b] - recent`` or <
    ``sinks`` stay, then those with the largest ``weights`` [batch, kv_heads,
    slots] (equal ones: the lower slot). Survivors behind the budget move into
    the slots that became free before it; ``positions`` (int32) say which
    token a slot holds. Each ``_out`` may be its input."""
    _binding.cache_evict(k_cache, v_cache, page_table, lengths, lengths_out, weights, weights_out, positions,
                         positions_out, seen, budget, recent, sinks)


def beam_search_step(logits, scores, finished, scores_out, parents, tokens, finished_out, *, eos: int,
                     k_cache=None, v_cache=None, page_table=None, lengths=None, spare=None,
                     page_table_out=None, lengths_out=None, workspace=None) -> None:
    """The ``beams`` best continuations of each item: ``logits`` [batch, beams,
    vocab] (float16 or float32), ``scores`` [batch, beams] float32 (sums of log
    probabilities), ``finished`` [batch, beams] bool (such a beam continues
    with ``eos`` at no cost). Writes ``scores_out``, ``parents`` and ``tokens``
    (int32) and ``finished_out``, best first. With a cache ([pages, ...] or
    [layers, pages, ...]; sequence ``b * beams + w``) the children take their
    parents' ``page_table`` and ``lengths``, the used part of a partly filled
    last page copied into ``spare[sequence]``."""
    _binding.beam_search_step(logits, scores, finished, scores_out, parents, tokens, finished_out, eos, k_cache,
                              v_cache, page_table, lengths, spare, page_table_out, lengths_out, workspace)


def device_error(device: int = 0, clear: bool = True) -> int:
    """The device's error word (0: none): bit 5 says that a page id or length
    outside its cache was left out. Waits for the device."""
    torch.cuda.synchronize(device)
    code = ctypes.c_uint32()
    _lib.check(_lib.lib.wgx_device_error(device, ctypes.byref(code), int(clear)))
    return code.value
