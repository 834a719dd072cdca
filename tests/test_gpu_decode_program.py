"""The decoding operators as a Program's chain: operators that write their
inputs, next to views, clones and what stays from submit to submit."""
import numpy as np
import pytest

import decode_reference as ref
import wgx
from test_gpu_decode import F16, T, Cache, attention_close

pytestmark = pytest.mark.gpu

SIZE = {"float16": 2, "float32": 4, "int32": 4, "bool": 1}


class Builder:
    """A Program with one memory pool per value; `None` and numbers become
    null and scalar values."""

    def __init__(self):
        self.values, self.pools, self.chain = [], [], []

    def tensor(self, dtype, shape, planned=True):
        v = {"type": "tensor", "shape": [int(n) for n in shape], "dtype": dtype}
        if planned:
            v["memObjId"] = len(self.pools)
            self.pools.append({"id": len(self.pools), "size": max(4, int(np.prod(shape)) * SIZE[dtype])})
        self.values.append(v)
        return len(self.values) - 1

    def like(self, a):
        return self.tensor(a.dtype.name, a.shape)

    def op(self, name, *args):
        ids = []
        for x in args:
            if isinstance(x, int):
                ids.append(x)
                continue
            if x is None:
                self.values.append({"type": "null"})
            elif isinstance(x, list):
                self.values.append({"type": "list", "items": x})
            else:
                self.values.append({"type": "scalar", "value": x[0]})
            ids.append(len(self.values) - 1)
        self.chain.append({"name": name, "args": ids})

    def program(self, inputs, outputs):
        return {"version": "1", "chain": self.chain, "values": self.values, "inputIds": inputs,
                "outputIds": outputs, "memoryPlan": {"pools": self.pools}}


@pytest.mark.parametrize("depth", [1, 2])
@pytest.mark.parametrize("also_output", [False, True])
@pytest.mark.parametrize("planned", [False, True])
def test_a_view_of_a_program_input(ctx, depth, also_output, planned):
    """A Program that begins with a view of an input: its readers see the
    caller's tensor, on every submit."""
    B, H, D, page = 2, 2, 64, 16
    c = Cache([20, 9], H, D, page, F16)
    rng = np.random.default_rng(2)
    table = np.where(c.table < 0, 0, c.table)
    p = Builder()
    q4 = p.tensor("float16", [B, 1, H, D], planned)
    kc, vc, t, ln = (p.like(a) for a in (c.k, c.v, table, c.lengths))
    q = p.tensor("float16", [B, H, D], planned)
    if depth == 2:
        mid = p.tensor("float16", [B, H * D], planned)
        p.op("aten.view_copy.default", q4, [B, H * D], mid)
        p.op("aten.view_copy.default", mid, [B, H, D], q)
    else:
        p.op("aten.view_copy.default", q4, [B, H, D], q)
    out = p.tensor("float16", [B, H, D])
    p.op("wgx.paged_attention.default", q, kc, vc, t, ln, None, None, None, None, None, out)
    qt, ot = ctx.tensor("float16", [B, 1, H, D]), ctx.tensor("float16", [B, H, D])
    args = [qt, T(ctx, c.k), T(ctx, c.v), T(ctx, table), T(ctx, c.lengths), ot]
    # (a tensor that is an output too keeps its copies)
    ctx.recordProgram(p.program([q4, kc, vc, t, ln], [out, q4] if also_output else [out]), b"",
                      args + [qt] if also_output else args)
    for _ in range(2):
        hq = rng.standard_normal((B, 1, H, D)).astype(np.float16)
        qt.setData(hq)
        ctx.submit()
        ctx.sync()
        want, _ = ref.paged_attention(hq[:, 0], c.k, c.v, table, c.lengths, D ** -0.5)
        attention_close(ot.numpy(), want, 6.0, True)
        np.testing.assert_array_equal(qt.numpy(), hq)


COPIES = ["aten.clone.default", "aten.view_copy.default", "aten.alias_copy.default"]


def copy_args(name, shape):
    return {"aten.clone.default": [None], "aten.view_copy.default": [[int(n) for n in shape]]}.get(name, [])


@pytest.mark.parametrize("name", COPIES[:2])
@pytest.mark.parametrize("what", ["lengths", "k_cache"])
@pytest.mark.parametrize("chained", [False, True])
def test_a_copy_taken_before_an_append_keeps_the_old_values(ctx, name, what, chained):
    B, H, G, D, page = 2, 2, 2, 64, 16
    c = Cache([13, 5], H, D, page, F16, room=4)
    c.k, c.v = np.nan_to_num(c.k, posinf=1, neginf=-1), np.nan_to_num(c.v, posinf=1, neginf=-1)
    rng = np.random.default_rng(0)
    hk, hv = (rng.standard_normal((B, 1, H, D)).astype(np.float16) for _ in range(2))
    hq = rng.standard_normal((B, H * G, D)).astype(np.float16)
    table = np.where(c.table < 0, 0, c.table)
    p = Builder()
    k, v, q, kc, vc, t, ln = (p.like(a) for a in (hk, hv, hq, c.k, c.v, table, c.lengths))
    src = {"lengths": ln, "k_cache": kc}[what]
    old = p.like({"lengths": c.lengths, "k_cache": c.k}[what])
    p.op(name, src, *copy_args(name, p.values[src]["shape"]), old)
    if chained:  # a copy of the copy
        older = p.like({"lengths": c.lengths, "k_cache": c.k}[what])
        p.op("aten.clone.default", old, None, older)
        old = older
    p.op("wgx.kv_append.default", k, v, t, ln, None, None, None, kc, vc, None, ln)
    out = p.like(hq)
    p.op("wgx.paged_attention.default", q, old if what == "k_cache" else kc, vc, t,
         old if what == "lengths" else ln, None, None, None, None, None, out)
    kt, vt, lt, ot = T(ctx, c.k), T(ctx, c.v), T(ctx, c.lengths), ctx.tensor("float16", list(hq.shape))
    ctx.recordProgram(p.program([k, v, q, kc, vc, t, ln], [out]), b"",
                      [T(ctx, hk), T(ctx, hv), T(ctx, hq), kt, vt, T(ctx, table), lt, ot])
    ctx.submit()
    ctx.sync()
    k0 = c.k.copy()
    for b in range(B):
        for h in range(H):
            ref.slot_row(c.k, table, b, h, c.lengths[b])[:] = hk[b, 0, h]
            ref.slot_row(c.v, table, b, h, c.lengths[b])[:] = hv[b, 0, h]
    want, _ = ref.paged_attention(hq, k0 if what == "k_cache" else c.k, c.v, table,
                                  c.lengths if what == "lengths" else c.lengths + 1, D ** -0.5)
    attention_close(ot.numpy(), want, 6.0, True)
    np.testing.assert_array_equal(kt.numpy(), c.k)  # the caller's cache itself


@pytest.mark.parametrize("later", [False, True])
def test_a_copy_of_weights_next_to_their_update_in_place(ctx, later):
    """Taken before the attention adds to them, it holds the old weights; taken
    after it, the new ones."""
    B, H, D, page = 1, 2, 64, 16
    c = Cache([30], H, D, page, F16)
    slots = c.width * page
    rng = np.random.default_rng(1)
    hq = rng.standard_normal((B, H, D)).astype(np.float16)
    hw = rng.random((B, H, slots)).astype(np.float32)
    table = np.where(c.table < 0, 0, c.table)
    p = Builder()
    q, kc, vc, t, ln, w = (p.like(a) for a in (hq, c.k, c.v, table, c.lengths, hw))
    kept, out, out2, w2 = p.like(hw), p.like(hq), p.like(hq), p.like(hw)
    if not later:
        p.op("aten.clone.default", w, None, kept)
    p.op("wgx.paged_attention.default", q, kc, vc, t, ln, None, None, None, w, w, out)
    if later:
        p.op("aten.clone.default", w, None, kept)
    p.op("wgx.paged_attention.default", q, kc, vc, t, ln, None, None, None, kept, w2, out2)
    wt, w2t = T(ctx, hw), ctx.tensor("float32", list(hw.shape))
    ctx.recordProgram(p.program([q, kc, vc, t, ln, w], [out, out2, w2]), b"",
                      [T(ctx, hq), T(ctx, c.k), T(ctx, c.v), T(ctx, table), T(ctx, c.lengths), wt,
                       ctx.tensor("float16", list(hq.shape)), ctx.tensor("float16", list(hq.shape)), w2t])
    ctx.submit()
    ctx.sync()
    _, once = ref.paged_attention(hq, c.k, c.v, table, c.lengths, D ** -0.5, weights=hw)
    _, twice = ref.paged_attention(hq, c.k, c.v, table, c.lengths, D ** -0.5, weights=once)
    np.testing.assert_allclose(w2t.numpy()[..., :30], (twice if later else once)[..., :30], atol=8e-5)
    np.testing.assert_allclose(wt.numpy()[..., :30], once[..., :30], atol=8e-5)


@pytest.mark.parametrize("outputs", [False, True])
def test_state_written_in_place_stays_from_submit_to_submit(ctx, outputs):
    """Append, attend with accumulated weights and evict, all of whose state
    (caches, weights, positions, lengths, seen) is written in place: the
    caller's tensors hold it after every submit and the next one goes on from
    there, whether they are the Program's outputs too or not."""
    B, H, G, D, page, steps, budget = 2, 2, 2, 64, 16, 6, 24
    c = Cache([22, 10], H, D, page, F16, room=steps)
    rng = np.random.default_rng(3)
    table = np.where(c.table < 0, 0, c.table)
    slots = c.width * page
    hk, hv = (rng.standard_normal((B, 1, H, D)).astype(np.float16) for _ in range(2))
    hq = rng.standard_normal((B, H * G, D)).astype(np.float16)
    weights = rng.random((B, H, slots)).astype(np.float32)
    pos = np.tile(np.arange(slots, dtype=np.int32), (B, H, 1))
    lengths, seen = c.lengths.copy(), c.lengths.copy()
    p = Builder()
    k, v, q, kc, vc, t, ln, sn, w, ps = (p.like(a) for a in (hk, hv, hq, c.k, c.v, table, lengths, seen, weights, pos))
    out = p.like(hq)
    p.op("wgx.kv_append.default", k, v, t, ln, ps, sn, w, kc, vc, sn, ln)
    p.op("wgx.paged_attention.default", q, kc, vc, t, ln, None, None, None, w, w, out)
    p.op("wgx.cache_evict.default", t, ln, sn, w, ps, (budget,), (4,), (2,), kc, vc, w, ps, ln)
    kt, vt, qt = T(ctx, hk), T(ctx, hv), T(ctx, hq)
    state = [T(ctx, a) for a in (c.k, c.v, table, lengths, seen, weights, pos)]
    ot = ctx.tensor("float16", list(hq.shape))
    more = ([ln, sn, w, ps], state[3:]) if outputs else ([], [])
    ctx.recordProgram(p.program([k, v, q, kc, vc, t, ln, sn, w, ps], [out] + more[0]), b"",
                      [kt, vt, qt] + state + [ot] + more[1])
    for _ in range(steps):
        hk, hv = (rng.standard_normal((B, 1, H, D)).astype(np.float16) for _ in range(2))
        hq = rng.standard_normal((B, H * G, D)).astype(np.float16)
        kt.setData(hk), vt.setData(hv), qt.setData(hq)
        ctx.submit()
        ctx.sync()
        for b in range(B):
            for h in range(H):
                ref.slot_row(c.k, table, b, h, lengths[b])[:] = hk[b, 0, h]
                ref.slot_row(c.v, table, b, h, lengths[b])[:] = hv[b, 0, h]
            weights[b, :, lengths[b]], pos[b, :, lengths[b]] = 0, seen[b]
        lengths, seen = lengths + 1, seen + 1
        want, added = ref.paged_attention(hq, c.k, c.v, table, lengths, D ** -0.5, weights=weights)
        attention_close(ot.numpy(), want, 6.0, True)
        before = lengths
        weights = added.astype(np.float32)
        lengths = ref.cache_evict(c.k, c.v, table, lengths, weights, pos, seen, budget, 4, 2)
        assert state[3].numpy().tolist() == lengths.tolist() and state[4].numpy().tolist() == seen.tolist()
        gw, gp = state[5].numpy(), state[6].numpy()
        for b in range(B):
            n = lengths[b]
            np.testing.assert_array_equal(gp[b, :, :n], pos[b, :, :n])
            np.testing.assert_allclose(gw[b, :, :n], weights[b, :, :n], atol=4e-5 * G * steps)
        # (slots behind the lengths hold what the eviction left there)
        np.testing.assert_array_equal(state[0].numpy(), c.k)
        np.testing.assert_array_equal(state[1].numpy(), c.v)
    assert (before > lengths).any()


def test_two_programs_hand_state_over(ctx):
    """The lengths that one Program advances in place are another's input."""
    B, H, D, page = 1, 1, 64, 16
    c = Cache([3], H, D, page, F16, room=4)
    rng = np.random.default_rng(4)
    hk, hv = (rng.standard_normal((B, 1, H, D)).astype(np.float16) for _ in range(2))
    hq = rng.standard_normal((B, H, D)).astype(np.float16)
    kt, vt, tt, lt = T(ctx, c.k), T(ctx, c.v), T(ctx, np.where(c.table < 0, 0, c.table)), T(ctx, c.lengths)
    a = Builder()
    k, v, t, ln, kc, vc = (a.like(x) for x in (hk, hv, c.table, c.lengths, c.k, c.v))
    a.op("wgx.kv_append.default", k, v, t, ln, None, None, None, kc, vc, None, ln)
    ctx.recordProgram(a.program([k, v, t, ln, kc, vc], []), b"", [T(ctx, hk), T(ctx, hv), tt, lt, kt, vt])
    b = Builder()
    q, t, ln, kc, vc = (b.like(x) for x in (hq, c.table, c.lengths, c.k, c.v))
    out = b.like(hq)
    b.op("wgx.paged_attention.default", q, kc, vc, t, ln, None, None, None, None, None, out)
    ot = ctx.tensor("float16", [B, H, D])
    ctx.recordProgram(b.program([q, t, ln, kc, vc], [out]), b"", [T(ctx, hq), tt, lt, kt, vt, ot])
    for step in range(2):
        ctx.submit()
        ctx.sync()
        n = c.lengths + step
        for h in range(H):
            ref.slot_row(c.k, c.table, 0, h, n[0])[:] = hk[0, 0, h]
            ref.slot_row(c.v, c.table, 0, h, n[0])[:] = hv[0, 0, h]
        want, _ = ref.paged_attention(hq, c.k, c.v, c.table, n + 1, D ** -0.5)
        attention_close(ot.numpy(), want, 6.0, True)
        assert lt.numpy().tolist() == (n + 1).tolist()


def test_state_of_another_size_is_refused(ctx):
    c = Cache([3], 1, 64, 16, F16, room=4)
    new = np.zeros((1, 1, 1, 64), np.float16)
    p = Builder()
    k, v, t, ln, kc, vc = (p.like(x) for x in (new, new, c.table, c.lengths, c.k, c.v))
    p.op("wgx.kv_append.default", k, v, t, ln, None, None, None, kc, vc, None, ln)
    small = T(ctx, c.k[:1])
    with pytest.raises(wgx.WgxError, match="updated in place"):
        ctx.recordProgram(p.program([k, v, t, ln, kc, vc], []), b"", [T(ctx, new), T(ctx, new), T(ctx, c.table),
                                                                      T(ctx, c.lengths), small, T(ctx, c.v)])
    assert ctx.stats()["commands"] == 0
