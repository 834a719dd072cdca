"""The decoding operators' C entry points refuse what they cannot do, with
messages, before any GPU is touched (the checks read host arguments only)."""
import ctypes
import struct

import pytest

import wgx
from wgx import _lib

# the argument structs of include/wgx.h, field by field
CACHE = ["k", "v", "page_table", "k_layer", "k_page", "k_head", "k_slot", "v_layer", "v_page", "v_head", "v_slot",
         "table_stride", "batch", "kv_heads", "head_dim", "dtype", "pages", "page_size", "table_width", "layers"]
FORMATS = {
    "append": ("3P9q8i2P6q6Pq2i", CACHE + ["new_k", "new_v", "kb", "kt", "kh", "vb", "vt", "vh", "lengths",
                                           "lengths_out", "seen", "seen_out", "weights", "positions", "slots",
                                           "tokens", "reserved"]),
    "attention": ("3P9q8i2P4q2Pq2PqPQ3if", CACHE + ["q", "out", "qb", "qh", "ob", "oh", "lengths", "mask",
                                                     "mask_stride", "weights", "weights_out", "slots", "scratch",
                                                     "scratch_bytes", "q_heads", "window", "mask_width", "scale"]),
    "evict": ("3P9q8i7Pq4i", CACHE + ["lengths", "lengths_out", "seen", "weights", "weights_out", "positions",
                                      "positions_out", "slots", "budget", "recent", "sinks", "reserved"]),
    "beam": ("3P9q8iP2q11PQ6i", CACHE + ["logits", "lb", "lw", "scores", "finished", "scores_out", "parents",
                                         "tokens", "finished_out", "lengths", "spare", "table_out", "lengths_out",
                                         "scratch", "scratch_bytes", "batch_items", "beams", "vocab", "logits_dtype",
                                         "eos", "reserved"]),
}
ENTRY = {"append": "wgx_kv_append", "attention": "wgx_paged_attention", "evict": "wgx_cache_evict",
         "beam": "wgx_beam_search_step"}
# addresses that are never followed: every call here is refused
GOOD_CACHE = dict(k=4096, v=8192, page_table=1024, k_page=2048, k_head=1024, k_slot=64, v_page=2048, v_head=1024,
                  v_slot=64, table_stride=4, batch=2, kv_heads=2, head_dim=64, dtype=1, pages=8, page_size=16,
                  table_width=4, layers=1)
GOOD = {
    "append": dict(GOOD_CACHE, new_k=4096, new_v=4096, lengths=1024, lengths_out=1024, tokens=1),
    "attention": dict(GOOD_CACHE, q=4096, out=4096, lengths=1024, q_heads=4, scale=0.125),
    "evict": dict(GOOD_CACHE, lengths=4, lengths_out=4, seen=4, weights=4, weights_out=4, positions=4,
                  positions_out=4, slots=64, budget=8),
    "beam": dict(logits=4096, scores=4, finished=4, scores_out=8, parents=4, tokens=4, finished_out=8, batch_items=1,
                 beams=2, vocab=100, logits_dtype=1),
}


def refuse(op, match, **changes):
    fmt, names = FORMATS[op]
    fields = dict(GOOD[op], **changes)
    assert set(fields) <= set(names), set(fields) - set(names)
    packed = struct.Struct("@" + fmt).pack(*(fields.get(n, 0.0 if n == "scale" else 0) for n in names))
    buf = ctypes.create_string_buffer(packed, len(packed))
    with pytest.raises(wgx.WgxError, match=match) as e:
        _lib.check(getattr(_lib.lib, ENTRY[op])(ctypes.addressof(buf), None))
    assert e.value.code == _lib.WGX_ERR_INVALID


@pytest.mark.parametrize("op", ["append", "attention", "evict"])
def test_cache_checks(op):
    refuse(op, "float32 or float16", dtype=2)
    refuse(op, "null cache", k=0)
    refuse(op, "null cache", page_table=0)
    refuse(op, "misaligned", k=4097)
    refuse(op, "misaligned", page_table=1026)
    refuse(op, "batch must be", batch=0)
    refuse(op, "batch must be", batch=70000)
    for field in ("kv_heads", "pages", "page_size", "table_width", "layers"):
        refuse(op, "must be positive", **{field: 0})
    refuse(op, "head size", head_dim=0)
    refuse(op, "head size", head_dim=257)
    refuse(op, "2\\^30 slots", page_size=1 << 20, table_width=1 << 20)
    refuse(op, "2\\^27 sequences", batch=60000, kv_heads=60000)
    refuse(op, "extents too large", page_size=1 << 29, table_width=1)
    refuse(op, "extents too large", layers=1 << 30)


def test_append_checks():
    refuse("append", "at least one token", tokens=0)
    refuse("append", "null pointer", new_k=0)
    refuse("append", "null pointer", lengths_out=0)
    refuse("append", "misaligned", new_v=4097)
    refuse("append", "come together", seen=4)
    refuse("append", "positions need seen", positions=4, slots=64)
    refuse("append", "cover every slot", weights=4, slots=63)


def test_attention_checks():
    refuse("attention", "null pointer", q=0)
    refuse("attention", "misaligned", out=4097)
    refuse("attention", "multiple of the K/V heads", q_heads=3)
    refuse("attention", "128 query heads", q_heads=258)
    refuse("attention", "batch must be", batch=2049)
    refuse("attention", "window", window=-1)
    refuse("attention", "NaN", scale=float("nan"))
    refuse("attention", "come together", weights=4, slots=64)
    refuse("attention", "cover every slot", weights=4, weights_out=4, slots=63)
    refuse("attention", "mask width", mask=4, mask_width=-1)
    refuse("attention", "2\\^30 sequences", batch=2048, kv_heads=5000, q_heads=128 * 5000)
    refuse("attention", "2\\^33 slots", batch=2048, page_size=1 << 20, table_width=8)
    refuse("attention", "2\\^25 slots", weights=4, weights_out=4, slots=1 << 40, page_size=1 << 20, table_width=64)


def test_evict_checks():
    refuse("evict", "null pointer", seen=0)
    refuse("evict", "budget must be positive", budget=0)
    refuse("evict", "recent \\+ sinks", recent=9)
    refuse("evict", "recent \\+ sinks", sinks=-1)
    refuse("evict", "recent \\+ sinks", recent=2 ** 31 - 1, sinks=2 ** 31 - 1)
    refuse("evict", "cover every slot", slots=63)


def test_beam_checks():
    refuse("beam", "logits must be", logits_dtype=6)
    refuse("beam", "null pointer", parents=0)
    refuse("beam", "misaligned", logits=4097)
    refuse("beam", "beams must be", beams=0)
    refuse("beam", "beams must be", beams=33)
    refuse("beam", "batch \\* beams", batch_items=40000)
    refuse("beam", "vocabulary", vocab=0)
    refuse("beam", "vocabulary", vocab=(1 << 24) + 1)
    refuse("beam", "overlap", scores_out=4)
    state = dict(GOOD_CACHE, lengths=4, spare=4, table_out=2048, lengths_out=8)
    refuse("beam", "batch \\* beams sequences", **dict(state, batch=3))
    refuse("beam", "null pointer", **dict(state, spare=0))
    refuse("beam", "overlap", **dict(state, table_out=1024))
    refuse("beam", "overlap", **dict(state, lengths_out=4))


def test_null_arguments():
    for entry in ENTRY.values():
        assert getattr(_lib.lib, entry)(None, None) == _lib.WGX_ERR_INVALID
        assert b"null arguments" in _lib.lib.wgx_last_error()


def test_the_operators_are_registered():
    names = {"wgx.kv_append.default", "wgx.paged_attention.default", "wgx.cache_evict.default",
             "wgx.beam_search_step.default"}
    assert names <= set(wgx.shaderRegistry)


def test_the_direct_calls_need_cuda_tensors():
    """wgx.decode imports and refuses without a GPU."""
    import torch
    import wgx.decode as dec
    t = torch.zeros(1, 1, 16, 64)
    with pytest.raises(wgx.WgxError, match="CUDA device"):
        dec.paged_attention(torch.zeros(1, 1, 64), t, t, torch.zeros(1, 1, dtype=torch.int32),
                            torch.zeros(1, dtype=torch.int32))
    with pytest.raises(wgx.WgxError, match="torch.Tensor"):
        dec.paged_attention(None, None, t, t, t)
    with pytest.raises(wgx.WgxError, match="CUDA device"):
        dec.beam_search_step(*[t] * 7, eos=0)
