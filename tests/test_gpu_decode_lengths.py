"""Lengths and page ids outside their cache, in the operators that write: an
invalid length names no slots. Such a sequence is left exactly as it is, pool,
weights, positions and length included, and the device error word says so."""
import numpy as np
import pytest
import torch

import decode_reference as ref
from test_gpu_decode import F16, F32, Cache, beam_inputs, dec, dev, host  # noqa: F401

pytestmark = pytest.mark.gpu

BAD = [-3, -2 ** 31, 2 ** 31 - 1]  # and one more than the table's slots


def bad_lengths(c):
    return BAD + [c.width * c.page + 1]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("T", [1, 400])  # one block a sequence, and several
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("order", ["head", "padded"])
def test_append_leaves_a_sequence_of_invalid_length_alone(dec, dtype, T, in_place, order):  # noqa: F811
    H, D = 2, 64
    c = Cache([20] * 5, H, D, 16, dtype, order, room=T, seed=T)
    lengths = np.array(bad_lengths(c) + [20], np.int32)
    rng = np.random.default_rng(T)
    k, v = (rng.standard_normal((5, T, H, D)).astype(c.k.dtype) for _ in range(2))
    slots = c.width * 16
    w, pos = np.ones((5, H, slots), np.float32), np.full((5, H, slots), -1, np.int32)
    seen = np.array([7, 8, 9, 10, 20], np.int32)
    k0, v0 = host(c.dk).copy(), host(c.dv).copy()
    dw, dp, ds, dl = dev(w), dev(pos), dev(seen), dev(lengths)
    so, lo = (ds, dl) if in_place else (torch.full_like(ds, -9), torch.full_like(dl, -9))
    dec.kv_append(dev(k), dev(v), c.dk, c.dv, c.dtable, dl, lo, seen=ds, seen_out=so, positions=dp, weights=dw)
    for t in range(T):
        for h in range(H):
            ref.slot_row(k0, c.table, 4, h, 20 + t)[:] = k[4, t, h]
            ref.slot_row(v0, c.table, 4, h, 20 + t)[:] = v[4, t, h]
    np.testing.assert_array_equal(host(c.dk), k0)
    np.testing.assert_array_equal(host(c.dv), v0)
    w[4, :, 20:20 + T], pos[4, :, 20:20 + T] = 0, 20 + np.arange(T)
    np.testing.assert_array_equal(host(dw), w)
    np.testing.assert_array_equal(host(dp), pos)
    np.testing.assert_array_equal(host(lo), np.append(lengths[:4], 20 + T))
    np.testing.assert_array_equal(host(so), np.append(seen[:4], 20 + T))
    assert dec.device_error(0) == 32


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("long", [False, True])  # one block a row, and a cluster
def test_evict_leaves_a_sequence_of_invalid_length_alone(dec, in_place, long):  # noqa: F811
    n = 5000 if long else 90
    H, D, budget = 2, 16, n // 2
    c = Cache([n] * 5, H, D, 16, F16, seed=3)
    table = np.where(c.table < 0, 0, c.table)  # every slot of the tables can be followed
    lengths = np.array(bad_lengths(c) + [n], np.int32)
    slots = c.width * 16
    rng = np.random.default_rng(1)
    w = rng.random((5, H, slots)).astype(np.float32)
    pos = np.stack([[rng.permutation(slots) for _ in range(H)] for _ in range(5)]).astype(np.int32)
    seen = np.full(5, slots, np.int32)
    dw, dp, dl = dev(w), dev(pos), dev(lengths)
    wo, po, lo = (dw, dp, dl) if in_place else (torch.full_like(dw, -9.0), torch.full_like(dp, -9),
                                                torch.full_like(dl, -9))
    k, v = c.k.copy(), c.v.copy()
    dec.cache_evict(c.dk, c.dv, dev(table), dl, lo, dw, wo, dp, po, dev(seen), budget=budget, recent=4, sinks=2)
    w0, p0 = w.copy(), pos.copy()
    ref.cache_evict(k, v, table, np.array([0, 0, 0, 0, n]), w, pos, seen, budget, 4, 2)
    np.testing.assert_array_equal(host(c.dk), k)
    np.testing.assert_array_equal(host(c.dv), v)
    np.testing.assert_array_equal(host(lo), np.append(lengths[:4], budget))
    gw, gp = host(wo), host(po)
    np.testing.assert_array_equal(gw[4, :, :budget], w[4, :, :budget])
    np.testing.assert_array_equal(gp[4, :, :budget], pos[4, :, :budget])
    np.testing.assert_array_equal(gw[:4], w0[:4] if in_place else np.full_like(w0[:4], -9))
    np.testing.assert_array_equal(gp[:4], p0[:4] if in_place else np.full_like(p0[:4], -9))
    assert dec.device_error(0) == 32


@pytest.mark.parametrize("bad", [0, 1, 2, 3])
def test_beams_of_invalid_length_copy_nothing_and_keep_it(dec, bad):  # noqa: F811
    c = Cache([21, 21], 1, 64, 16, F16, layers=1, extra=2)
    length = bad_lengths(c)[bad]
    x, s, f = beam_inputs(1, 2, 100, np.float16)
    k0, v0 = host(c.dk).copy(), host(c.dv).copy()
    i32 = dict(dtype=torch.int32, device="cuda")
    outs = [torch.empty(1, 2, device="cuda"), torch.empty(1, 2, **i32), torch.empty(1, 2, **i32),
            torch.empty(1, 2, dtype=torch.bool, device="cuda")]
    to, lo = torch.empty_like(c.dtable), torch.empty(2, **i32)
    dec.beam_search_step(dev(x), dev(s), dev(f), *outs, eos=2, k_cache=c.dk, v_cache=c.dv, page_table=c.dtable,
                         lengths=dev(np.full(2, length, np.int32)), spare=dev(c.free[:2]), page_table_out=to,
                         lengths_out=lo)
    np.testing.assert_array_equal(host(to), c.table[host(outs[1])[0]])
    assert host(lo).tolist() == [length] * 2
    np.testing.assert_array_equal(host(c.dk), k0)
    np.testing.assert_array_equal(host(c.dv), v0)
    assert dec.device_error(0) == 32


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("bad", ["source", "destination"])
def test_evict_moves_a_slots_label_only_with_its_row(dec, in_place, bad):  # noqa: F811
    """A page id outside the pool: the rows of that page do not move, so
    neither do their weights and positions; every other pair moves."""
    H, D, page, n, budget = 1, 16, 16, 64, 32
    c = Cache([n], H, D, page, F16, seed=5)
    table = c.table.copy()
    entry = 3 if bad == "source" else 0
    table[0, entry] = c.k.shape[0]
    rng = np.random.default_rng(2)
    w = rng.random((1, H, c.width * page)).astype(np.float32)
    pos = np.arange(c.width * page, dtype=np.int32)[None, None]
    dw, dp, dl = dev(w), dev(pos), c.dlengths
    wo, po, lo = (dw, dp, dl) if in_place else (torch.full_like(dw, -9.0), torch.full_like(dp, -9),
                                                torch.full_like(dl, -9))
    dec.cache_evict(c.dk, c.dv, dev(table), dl, lo, dw, wo, dp, po, dev(np.array([n], np.int32)), budget=budget)
    _, moves = ref.evict_plan(w[0, 0], pos[0, 0], n, n, budget, 0, 0)
    done = [(d, s) for d, s in moves if entry not in (d // page, s // page)]
    assert 0 < len(done) < len(moves)
    ww, pw = w[0, 0].copy(), pos[0, 0].copy()
    for d, s in done:
        for x in (c.k, c.v):
            ref.slot_row(x, c.table, 0, 0, d)[:] = ref.slot_row(x, c.table, 0, 0, s)
        ww[d], pw[d] = ww[s], pw[s]
    np.testing.assert_array_equal(host(c.dk), c.k)
    np.testing.assert_array_equal(host(c.dv), c.v)
    np.testing.assert_array_equal(host(wo)[0, 0, :budget], ww[:budget])
    np.testing.assert_array_equal(host(po)[0, 0, :budget], pw[:budget])
    assert host(lo).tolist() == [budget] and dec.device_error(0) == 32


@pytest.mark.parametrize("B", [1, 3])
def test_append_of_more_tokens_than_any_table_holds(dec, B):  # noqa: F811
    c = Cache([5] * B, 1, 16, 16, F16)
    k0, lo = host(c.dk).copy(), torch.zeros(B, dtype=torch.int32, device="cuda")
    new = torch.zeros(1, 1, 1, 16, dtype=F16, device="cuda").expand(B, 2 ** 31 - 1, 1, 16)
    dec.kv_append(new, new, c.dk, c.dv, c.dtable, c.dlengths, lo)
    assert host(lo).tolist() == [5] * B
    np.testing.assert_array_equal(host(c.dk), k0)
    assert dec.device_error(0) == 32
