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
that lies outside the cache is left out and noted (``device_error``).

Calls are enqueued on the tensors' device's current stream. Outputs are
arguments; nothing is kept between calls. Scratch memory comes from torch's
allocator unless ``workspace`` (a uint8 tensor) is given.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Dict, Optional

import torch

from ._lib import WGX_ERR_INVALID, WgxError, check, lib

_DTYPE = {torch.float32: 0, torch.float16: 1}
# wgx_kv_cache and the operators' argument structs, field by field
_CACHE = "3P9q8i"
_APPEND = struct.Struct("@" + _CACHE + "2P6q6Pq2i")
_ATTEND = struct.Struct("@" + _CACHE + "2P4q2Pq2PqPQ3if")
_EVICT = struct.Struct("@" + _CACHE + "7Pq4i")
_BEAM = struct.Struct("@" + _CACHE + "P2q11PQ6i")
_NO_CACHE = (0,) * 20
_scratch: Dict[tuple, int] = {}  # bytes by everything they depend on


def _fail(op: str, msg: str):
    raise WgxError(WGX_ERR_INVALID, f"{op}: {msg}")


def _need(op: str, what: str, t, dtype, shape, dev: int) -> int:
    """The address of a dense device tensor, checked."""
    if t.dtype != dtype:
        _fail(op, f"{what} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        _fail(op, f"{what} shape {list(t.shape)} !== expected {list(shape)}")
    if not t.is_contiguous():
        _fail(op, f"{what} must be contiguous")
    if t.get_device() != dev:
        _fail(op, f"{what} must be on the cache's device")
    return t.data_ptr()


def _rows(op: str, what: str, t, dtype, dev: int) -> None:
    if t.dtype != dtype:
        _fail(op, "Tensors must have matching float32 or float16 dtype")
    if t.get_device() != dev:
        _fail(op, f"{what} must be on the cache's device")
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        _fail(op, f"{what} must have a unit last stride")


def _flags(op: str, what: str, t):
    if t.dtype != torch.bool and t.dtype != torch.uint8:
        _fail(op, f"{what} must be bool or uint8, got {t.dtype}")
    return t.dtype


def _cache(op: str, k, v, table, layered: bool = False):
    """(the wgx_kv_cache fields, device)."""
    dev = k.get_device()
    if dev < 0:
        _fail(op, "tensors must be on a CUDA device")
    if k.dtype not in _DTYPE:
        _fail(op, "Tensors must have matching float32 or float16 dtype")
    _rows(op, "v_cache", v, k.dtype, dev)
    _rows(op, "k_cache", k, k.dtype, dev)
    if k.shape != v.shape:
        _fail(op, f"v_cache shape {list(v.shape)} !== expected {list(k.shape)}")
    ks, vs = k.stride(), v.stride()
    if k.dim() == 4:
        layers = 1
        pages, heads, size, dim = k.shape
        ks, vs = (0,) + ks, (0,) + vs
    elif layered and k.dim() == 5:
        layers, pages, heads, size, dim = k.shape
    else:
        _fail(op, "a cache is [pages, kv_heads, page_size, head_dim]")
    if table.dim() != 2 or table.dtype != torch.int32 or table.get_device() != dev:
        _fail(op, "page_table must be a 2-D int32 tensor on the cache's device")
    ts = table.stride()
    if ts[1] != 1 and table.shape[1] != 1:
        _fail(op, "page_table must have a unit last stride")
    return (k.data_ptr(), v.data_ptr(), table.data_ptr(), ks[0], ks[1], ks[2], ks[3],
            vs[0], vs[1], vs[2], vs[3], ts[0], table.shape[0], heads, dim, _DTYPE[k.dtype],
            pages, size, table.shape[1], layers), dev


def _call(fn, packed: bytes, dev: int) -> None:
    if dev == torch.cuda.current_device():
        code = fn(packed, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            code = fn(packed, torch._C._cuda_getCurrentRawStream(dev))
    if code:
        check(code)


def _scratch_bytes(fn, key: tuple, pack, dev: int) -> int:
    n = _scratch.get(key)
    if n is None:
        out = ctypes.c_uint64()
        with torch.cuda.device(dev):
            check(fn(pack(0, 0), ctypes.byref(out)))
        n = _scratch[key] = out.value
    return n


def _workspace(op: str, workspace, bytes: int, dev: int):
    if workspace is None:
        return torch.empty(bytes, dtype=torch.uint8, device=dev)
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous() or workspace.get_device() != dev:
        _fail(op, "workspace must be a contiguous uint8 tensor on the cache's device")
    return workspace


def kv_append(k, v, k_cache, v_cache, page_table, lengths, lengths_out, *, seen=None, seen_out=None,
              positions=None, weights=None) -> None:
    """Writes ``k``, ``v`` [batch, tokens, kv_heads, head_dim] behind the slots
    in use; ``lengths_out = lengths + tokens`` (may be ``lengths``). With
    ``seen`` / ``seen_out`` [batch] and ``positions``, ``weights`` [batch,
    kv_heads, slots]: the new slots get position ``seen[b] + t`` and weight 0.
    A sequence whose page table has no room for all of them gets none."""
    op = "kv_append"
    c, dev = _cache(op, k_cache, v_cache, page_table)
    B, H, D = c[12], c[13], c[14]
    dt = k_cache.dtype
    _rows(op, "k", k, dt, dev)
    _rows(op, "v", v, dt, dev)
    shape = k.shape
    if len(shape) != 4 or shape[0] != B or shape[2] != H or shape[3] != D or v.shape != shape:
        _fail(op, f"k and v must be [{B}, tokens, {H}, {D}], got {list(k.shape)} and {list(v.shape)}")
    i32, n = torch.int32, (B,)
    slots = 0
    pos = w = s = so = 0
    if positions is not None or weights is not None:
        slots = (positions if positions is not None else weights).shape[-1]
        if positions is not None:
            pos = _need(op, "positions", positions, i32, (B, H, slots), dev)
        if weights is not None:
            w = _need(op, "weights", weights, torch.float32, (B, H, slots), dev)
    if seen is not None:
        s = _need(op, "seen", seen, i32, n, dev)
    if seen_out is not None:
        so = _need(op, "seen_out", seen_out, i32, n, dev)
    ks, vs = k.stride(), v.stride()
    _call(lib.wgx_kv_append, _APPEND.pack(
        *c, k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        _need(op, "lengths", lengths, i32, n, dev), _need(op, "lengths_out", lengths_out, i32, n, dev),
        s, so, w, pos, slots, shape[1], 0), dev)


def paged_attention(q, k_cache, v_cache, page_table, lengths, out=None, *, scale: Optional[float] = None,
                    window: int = 0, mask=None, weights=None, weights_out=None, workspace=None):
    """Attention of one token per sequence, ``q`` [batch, q_heads, head_dim]
    (``q_heads`` a multiple of the cache's K/V heads), over the slots in use;
    returns ``out`` (allocated when not given). ``scale``: 1 / sqrt(head_dim)
    by default; ``window`` > 0: the last ``window`` slots only; ``mask``
    [batch, n] bool: slots to attend to. ``weights`` / ``weights_out``
    [batch, kv_heads, slots] float32 (may be the same tensor): ``weights_out =
    weights +`` the probabilities of each K/V head's query heads, summed."""
    op = "paged_attention"
    c, dev = _cache(op, k_cache, v_cache, page_table)
    B, H, D = c[12], c[13], c[14]
    dt = k_cache.dtype
    shape = q.shape
    if len(shape) != 3 or shape[0] != B or shape[2] != D:
        _fail(op, f"q must be [{B}, q_heads, {D}], got {list(shape)}")
    _rows(op, "q", q, dt, dev)
    if out is None:
        out = torch.empty(shape, dtype=dt, device=q.device)
    else:
        _rows(op, "out", out, dt, dev)
        if out.shape != shape:
            _fail(op, f"out shape {list(out.shape)} !== expected {list(shape)}")
    m = ms = mw = w = wo = slots = 0
    if mask is not None:
        _flags(op, "mask", mask)
        if mask.dim() != 2 or mask.shape[0] != B or mask.get_device() != dev or \
                (mask.stride(1) != 1 and mask.shape[1] != 1):
            _fail(op, f"mask must be [{B}, slots] with a unit last stride")
        m, ms, mw = mask.data_ptr(), mask.stride(0), mask.shape[1]
    if weights is not None or weights_out is not None:
        if weights is None or weights_out is None:
            _fail(op, "weights and weights_out come together")
        slots = weights.shape[-1]
        w = _need(op, "weights", weights, torch.float32, (B, H, slots), dev)
        wo = _need(op, "weights_out", weights_out, torch.float32, (B, H, slots), dev)
    qs, os_ = q.stride(), out.stride()
    head = (*c, q.data_ptr(), out.data_ptr(), qs[0], qs[1], os_[0], os_[1],
            _need(op, "lengths", lengths, torch.int32, (B,), dev), m, ms, w, wo, slots)
    tail = (shape[1], window, mw, D ** -0.5 if scale is None else scale)

    def pack(ptr, size):
        return _ATTEND.pack(*head, ptr, size, *tail)

    size = _scratch_bytes(lib.wgx_paged_attention_scratch_bytes,
                          (op, dev, c[12:], shape[1], wo != 0), pack, dev)
    ws = _workspace(op, workspace, size, dev)
    _call(lib.wgx_paged_attention, pack(ws.data_ptr(), ws.numel()), dev)
    return out


def cache_evict(k_cache, v_cache, page_table, lengths, lengths_out, weights, weights_out, positions,
                positions_out, seen, *, budget: int, recent: int = 0, sinks: int = 0) -> None:
    """Shrinks every sequence of more than ``budget`` slots to ``budget``
    slots, per K/V head: those at positions >= ``seen[b] - recent`` or <
    ``sinks`` stay, then those with the largest ``weights`` [batch, kv_heads,
    slots] (equal ones: the lower slot). Survivors behind the budget move into
    the slots that became free before it; ``positions`` (int32) say which
    token a slot holds. Each ``_out`` may be its input."""
    op = "cache_evict"
    c, dev = _cache(op, k_cache, v_cache, page_table)
    B, H = c[12], c[13]
    i32, f32 = torch.int32, torch.float32
    shape = (B, H, weights.shape[-1])
    _call(lib.wgx_cache_evict, _EVICT.pack(
        *c, _need(op, "lengths", lengths, i32, (B,), dev), _need(op, "lengths_out", lengths_out, i32, (B,), dev),
        _need(op, "seen", seen, i32, (B,), dev), _need(op, "weights", weights, f32, shape, dev),
        _need(op, "weights_out", weights_out, f32, shape, dev),
        _need(op, "positions", positions, i32, shape, dev),
        _need(op, "positions_out", positions_out, i32, shape, dev), shape[2], budget, recent, sinks, 0), dev)


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
    op = "beam_search_step"
    dev = logits.get_device()
    if dev < 0:
        _fail(op, "tensors must be on a CUDA device")
    if logits.dtype not in _DTYPE or logits.dim() != 3:
        _fail(op, "logits must be [batch, beams, vocab], float32 or float16")
    B, W, V = logits.shape
    ls = logits.stride()
    if ls[2] != 1 and V != 1:
        _fail(op, "logits must have a unit last stride")
    i32, f32, bw = torch.int32, torch.float32, (B, W)
    c = _NO_CACHE
    ln = sp = to = lo = 0
    if k_cache is not None:
        if v_cache is None or page_table is None or lengths is None or spare is None or \
                page_table_out is None or lengths_out is None:
            _fail(op, "the cache's arguments come together")
        c, cdev = _cache(op, k_cache, v_cache, page_table, layered=True)
        if cdev != dev:
            _fail(op, "logits must be on the cache's device")
        n = (B * W,)
        ln = _need(op, "lengths", lengths, i32, n, dev)
        sp = _need(op, "spare", spare, i32, n, dev)
        to = _need(op, "page_table_out", page_table_out, i32, (B * W, c[18]), dev)
        lo = _need(op, "lengths_out", lengths_out, i32, n, dev)
    head = (*c, logits.data_ptr(), ls[0], ls[1], _need(op, "scores", scores, f32, bw, dev),
            _need(op, "finished", finished, _flags(op, "finished", finished), bw, dev),
            _need(op, "scores_out", scores_out, f32, bw, dev), _need(op, "parents", parents, i32, bw, dev),
            _need(op, "tokens", tokens, i32, bw, dev),
            _need(op, "finished_out", finished_out, _flags(op, "finished_out", finished_out), bw, dev),
            ln, sp, to, lo)
    tail = (B, W, V, _DTYPE[logits.dtype], eos, 0)

    def pack(ptr, size):
        return _BEAM.pack(*head, ptr, size, *tail)

    size = _scratch_bytes(lib.wgx_beam_search_scratch_bytes, (op, dev, B, W, V), pack, dev)
    ws = _workspace(op, workspace, size, dev)
    _call(lib.wgx_beam_search_step, pack(ws.data_ptr(), ws.numel()), dev)


def device_error(device: int = 0, clear: bool = True) -> int:
    """The device's error word (0: none): bit 5 says that a page id or length
    outside its cache was left out. Waits for the device."""
    torch.cuda.synchronize(device)
    code = ctypes.c_uint32()
    check(lib.wgx_device_error(device, ctypes.byref(code), int(clear)))
    return code.value
