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
