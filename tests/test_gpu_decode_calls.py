"""What the decoding operators' calls say beside their results: the launch counts
of recorded commands, the scratch they ask for, refusals at recording, and what autograd sees."""
import ctypes
import struct

import numpy as np
import pytest
import torch

import wgx
from test_decode_cpu import FORMATS, GOOD
from test_gpu_decode import F16, T, Cache, dec  # noqa: F401
from wgx import _lib

pytestmark = pytest.mark.gpu


def same_launches(ctx, want):
    before = ctx.stats()["kernel_launches"]
    ctx.submit()
    ctx.sync()
    assert ctx.stats()["kernel_launches"] == before == want


@pytest.mark.parametrize("width,launches", [(8, 1), (200, 2)])  # a row in one block; split and joined
@pytest.mark.parametrize("weights", [False, True])
def test_launch_count_of_a_recorded_attention(ctx, width, launches, weights):
    c = Cache([50, 20], 2, 64, 16, F16, width=width)
    q, out = T(ctx, np.zeros((2, 4, 64), np.float16)), ctx.tensor("float16", [2, 4, 64])
    w = T(ctx, np.zeros((2, 2, width * 16), np.float32)) if weights else None
    ctx.recordShader(wgx.shaders.pagedAttention, [q, T(ctx, c.k), T(ctx, c.v), T(ctx, c.table), T(ctx, c.lengths), None,
                                                 None, None, w, w, out])
    same_launches(ctx, launches)


@pytest.mark.parametrize("tokens,in_place,launches", [(1, True, 1), (1, False, 1), (900, True, 2), (900, False, 1)])
def test_launch_count_of_a_recorded_append(ctx, tokens, in_place, launches):
    c = Cache([5, 0], 2, 64, 16, F16, room=tokens)
    new = T(ctx, np.zeros((2, tokens, 2, 64), np.float16))
    ln = T(ctx, c.lengths)
    lo = ln if in_place else ctx.tensor("int32", [2])
    ctx.recordShader(wgx.shaders.kvAppend, [new, new, T(ctx, c.table), ln, None, None, None, T(ctx, c.k), T(ctx, c.v),
                                            None, lo])
    same_launches(ctx, launches)


@pytest.mark.parametrize("in_place,launches", [(True, 2), (False, 1)])
def test_launch_count_of_a_recorded_eviction(ctx, in_place, launches):
    c = Cache([50, 20], 2, 64, 16, F16)
    slots = c.width * 16
    w, pos = T(ctx, np.zeros((2, 2, slots), np.float32)), T(ctx, np.zeros((2, 2, slots), np.int32))
    ln = T(ctx, c.lengths)
    lo = ln if in_place else ctx.tensor("int32", [2])
    ctx.recordShader(wgx.shaders.cacheEvict, [T(ctx, c.table), ln, T(ctx, c.lengths), w, pos, 30, 0, 0, T(ctx, c.k),
                                              T(ctx, c.v), w, pos, lo])
    same_launches(ctx, launches)


def test_launch_count_of_a_recorded_beam_step(ctx):
    t = lambda a: T(ctx, a)  # noqa: E731
    e = lambda dt: ctx.tensor(dt, [1, 2])  # noqa: E731
    ctx.recordShader(wgx.shaders.beamSearchStep, [t(np.zeros((1, 2, 50), np.float16)), t(np.zeros((1, 2), np.float32)),
                                                 t(np.zeros((1, 2), bool)), 0, None, None, None, None, None,
                                                 e("float32"), e("int32"), e("int32"), e("bool"), None, None])
    same_launches(ctx, 2)


def scratch_bytes(**fields):
    fmt, names = FORMATS["attention"]
    fields = dict(GOOD["attention"], **fields)
    packed = struct.Struct("@" + fmt).pack(*(fields.get(n, 0.0 if n == "scale" else 0) for n in names))
    buf, n = ctypes.create_string_buffer(packed, len(packed)), ctypes.c_uint64()
    _lib.check(_lib.lib.wgx_paged_attention_scratch_bytes(ctypes.addressof(buf), ctypes.byref(n)))
    return n.value


def test_scratch_of_a_window_goes_by_the_window():
    """Scores are kept for the weights: of the slots a window can hold, not of
    all that a wide table can name."""
    case = dict(batch=64, kv_heads=8, q_heads=32, head_dim=128, page_size=16, table_width=8192, table_stride=8192,
                weights=4096, weights_out=4096, slots=131072)
    scores = 64 * 32 * 4096 * 4
    most = 1.02 * scores + 2 ** 24  # and the partial results of the cut rows
    assert scores <= scratch_bytes(window=4096, **case) <= most
    assert scratch_bytes(window=0, **case) >= 32 * scores
    assert scratch_bytes(window=4096, **dict(case, table_width=256, table_stride=256)) <= most


@pytest.mark.parametrize("dtype,G", [(torch.float16, 2), (torch.float32, 2), (torch.float32, 12)])
@pytest.mark.parametrize("window", [1, 17, 250, 1000, 4097])
def test_window_weights_within_their_scratch(dec, dtype, G, window):  # noqa: F811
    """The result with a workspace of exactly the size asked for, poisoned
    around it; slots on both sides of a step's edge."""
    import decode_reference as ref
    lengths = [3, 1000, 2063, 4100]
    c = Cache(lengths, 2, 64, 16, dtype, width=300)
    slots = c.width * 16
    rng = np.random.default_rng(window)
    q = rng.standard_normal((4, 2 * G, 64)).astype(c.k.dtype)
    w = rng.random((4, 2, slots)).astype(np.float32)
    dq, dw = torch.from_numpy(q).cuda(), torch.from_numpy(w).cuda()
    wo = torch.full_like(dw, -5.0)
    n = scratch_bytes(batch=4, kv_heads=2, q_heads=2 * G, head_dim=64, dtype=1 if dtype == torch.float16 else 0,
                      pages=c.k.shape[0], page_size=16, table_width=c.width, table_stride=c.width, window=window,
                      weights=4096, weights_out=8192, slots=slots)
    room = torch.full((n + 4096,), 0xff, dtype=torch.uint8, device="cuda")
    dec.paged_attention(dq, c.dk, c.dv, c.dtable, c.dlengths, window=window, weights=dw, weights_out=wo,
                        workspace=room[:n])
    _, want = ref.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.125, window, None, w)
    got = wo.cpu().numpy()
    for b, m in enumerate(lengths):
        np.testing.assert_allclose(got[b, :, :m], want[b, :, :m], rtol=1e-6, atol=4e-5 * G)
        assert (got[b, :, m:] == -5).all()
    assert (room[n:] == 0xff).all() and dec.device_error(0) == 0


def test_autograd_sees_what_the_calls_write(dec):  # noqa: F811
    """The operators are outside autograd (results carry no graph), but what
    they write counts as written: backward over a tensor saved before and
    overwritten since is refused instead of silently wrong."""
    c = Cache([20, 10], 2, 64, 16, F16)
    q = torch.zeros(2, 4, 64, dtype=F16, device="cuda", requires_grad=True)
    slots = c.width * 16
    w, wo = torch.zeros(2, 2, slots, device="cuda"), torch.zeros(2, 2, slots, device="cuda")
    out = torch.empty(2, 4, 64, dtype=F16, device="cuda")
    count = lambda *ts: [t._version for t in ts]  # noqa: E731
    v0 = count(out, wo)
    r = dec.paged_attention(q, c.dk, c.dv, c.dtable, c.dlengths, out, weights=w, weights_out=wo)
    assert r is out or r.data_ptr() == out.data_ptr()
    assert not r.requires_grad and r.grad_fn is None
    assert count(out, wo) == [n + 1 for n in v0]
    k = torch.zeros(2, 1, 2, 64, dtype=F16, device="cuda")
    lo, so, seen = torch.zeros_like(c.dlengths), torch.zeros_like(c.dlengths), torch.zeros_like(c.dlengths)
    pos = torch.zeros(2, 2, slots, dtype=torch.int32, device="cuda")
    written, read = [c.dk, c.dv, lo, so, pos, w], [k, c.dtable, c.dlengths, seen]
    v0, r0 = count(*written), count(*read)
    dec.kv_append(k, k, c.dk, c.dv, c.dtable, c.dlengths, lo, seen=seen, seen_out=so, positions=pos, weights=w)
    assert count(*written) == [n + 1 for n in v0] and count(*read) == r0
    po = torch.zeros_like(pos)
    written, read = [c.dk, c.dv, lo, wo, po], [c.dtable, c.dlengths, w, pos, seen]
    v0, r0 = count(*written), count(*read)
    dec.cache_evict(c.dk, c.dv, c.dtable, c.dlengths, lo, w, wo, pos, po, seen, budget=8)
    assert count(*written) == [n + 1 for n in v0] and count(*read) == r0
    x, s = torch.zeros(1, 2, 50, device="cuda"), torch.zeros(1, 2, device="cuda")
    f = torch.zeros(1, 2, dtype=torch.bool, device="cuda")
    outs = [torch.zeros(1, 2, device="cuda"), torch.zeros(1, 2, dtype=torch.int32, device="cuda"),
            torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, dtype=torch.bool, device="cuda")]
    table, to = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    spare = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    written, read = outs + [c.dk, c.dv, to, lo], [x, s, f, table, c.dlengths, spare]
    v0, r0 = count(*written), count(*read)
    dec.beam_search_step(x, s, f, *outs, eos=0, k_cache=c.dk, v_cache=c.dv, page_table=table, lengths=c.dlengths,
                         spare=spare, page_table_out=to, lengths_out=lo)
    assert count(*written) == [n + 1 for n in v0] and count(*read) == r0
    # a saved tensor that was overwritten
    a = torch.randn(2, 4, 64, device="cuda", requires_grad=True)
    saved = torch.randn(2, 4, 64, device="cuda")
    y = (a * saved).sum()
    dec.paged_attention(torch.zeros(2, 4, 64, device="cuda"), c.dk.float(), c.dv.float(), c.dtable, c.dlengths, saved)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    # tensors made under inference mode have no versions to count
    with torch.inference_mode():
        t = torch.zeros(2, 4, 64, dtype=F16, device="cuda")
        dec.paged_attention(t, c.dk, c.dv, c.dtable, c.dlengths, t.clone())
    dec.paged_attention(q.detach(), c.dk, c.dv, c.dtable, c.dlengths, t)


def test_an_eviction_of_too_many_slots_is_refused_when_recorded(ctx):
    """Not at the first submit: a recorded command can run."""
    t = lambda dt, *s: ctx.tensor(dt, list(s))  # noqa: E731

    def record(width):
        slots = width * 16
        w, pos, ln = t("float32", 1, 1, slots), t("int32", 1, 1, slots), t("int32", 1)
        ctx.recordShader(wgx.shaders.cacheEvict, [t("int32", 1, width), ln, ln, w, pos, 8, 0, 0, t("float16", 2, 1, 16, 8),
                                                  t("float16", 2, 1, 16, 8), w, pos, ln])
    with pytest.raises(wgx.WgxError, match="262144 slots"):
        record(16385)
    assert ctx.stats()["commands"] == 0
    record(16384)
    assert ctx.stats()["commands"] == 1
