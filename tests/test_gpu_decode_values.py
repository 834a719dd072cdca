"""What paged_attention's result and accumulated weights hold where scores are
far apart or not finite.

A row with one slot (a "sink", value zero) far above all others: its result is
the others' small probabilities times their values. Tolerance, relative to
that result, derived before the first run: probabilities of a step (16 slots)
enter the product to 2^-21 of themselves, or of the step's largest by 2^-25
where they are smaller; scores of up to 50 (base 2) are off by 2^-23 of
themselves, exp2 by 2^-22: below 1e-5 in all. The sums are fp32, which a tensor
core may cut instead of round: at most two additions per step of 16 slots, each
by 2^-23, below 2^-12 for the 16384 slots here. The up to 15 slots that share a
step with the sink are held to 2^-36 of the sink's probability. fp16's output
adds half a unit: 2^-11, or 2^-25 absolutely below its normal range."""
import numpy as np
import pytest
import torch

import decode_reference as ref
from test_gpu_decode import F16, F32, Cache, dec, dev, host  # noqa: F401

pytestmark = pytest.mark.gpu


def sink_rows(n, gap, D, H, G, dtype, at, rng):
    """(q, k, v): scores are `gap` nats for slot `at` and 0 for the others,
    with scale 1 (exact in fp16: the gap is a product of two numbers)."""
    npdt = np.float16 if dtype == F16 else np.float32
    k = np.zeros((n, D), npdt)
    k[at, 0] = 1
    q = np.zeros((H * G, D), npdt)
    q[:, 0] = gap
    v = (rng.random((n, D)) + 0.5).astype(npdt)
    v[at] = 0
    return q, k, v


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n,rows", [(300, 8), (4096, 1300), (16384, 1300), (16384, 2)])
@pytest.mark.parametrize("gap", [10, 14, 16, 17, 18, 20, 23])
@pytest.mark.parametrize("D,G", [(64, 1), (128, 4), (128, 12), (256, 16)])
def test_attention_keeps_the_tail_of_a_peaked_row(dec, dtype, n, rows, gap, D, G):  # noqa: F811
    """All sequences read the same pages, so that thousands of slots of a row
    lie in one warp's share without a large cache."""
    page, B = 16, rows
    rng = np.random.default_rng(gap)
    at = {300: 0, 4096: 37, 16384: 16383 if rows > 2 else 8000}[n]
    q, k, v = sink_rows(n, gap, D, 1, G, dtype, at, rng)
    pages = -(-n // page)
    pool = lambda x: dev(np.pad(x, ((0, pages * page - n), (0, 0))).reshape(pages, 1, page, D))  # noqa: E731
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].expand(B, pages)
    size = 1000.0  # values of this size: results stay far above fp16's smallest numbers
    out = dec.paged_attention(dev(q)[None].expand(B, G, D), pool(k), pool((v * size).astype(v.dtype)), table,
                              torch.full((B,), n, dtype=torch.int32, device="cuda"), scale=1.0)
    p = np.where(np.arange(n) == at, 1.0, np.exp(-float(gap)))
    vv = (v * size).astype(v.dtype).astype(np.float64)
    want = (p / p.sum()) @ vv
    got = out.double().cpu().numpy()
    tol = want * (1e-5 + 2.0 ** -12 + (2.0 ** -11 if dtype == F16 else 0)) + 15 * 2.0 ** -36 * vv.max() + \
        (2.0 ** -25 if dtype == F16 else 0)
    assert (np.abs(got - want) <= tol).all(), np.abs(got / want - 1).max()
    assert dec.device_error(0) == 0


@pytest.mark.parametrize("n", [4096, 16384, 131072])
@pytest.mark.parametrize("D,G", [(64, 1), (128, 4), (256, 16)])
def test_attention_of_equal_values_is_that_value(dec, n, D, G):  # noqa: F811
    """Every value 1: the result is 1 to within fp16's rounding, however many
    slots one warp adds up (sums cut by the tensor core would fall short)."""
    B, page = 1300, 64
    pages = n // page
    k = torch.randn(pages, 1, page, D, device="cuda").half()
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].expand(B, pages)
    q = torch.randn(B, G, D, device="cuda").half()
    out = dec.paged_attention(q, k, torch.ones_like(k), table,
                              torch.full((B,), n, dtype=torch.int32, device="cuda"))
    assert float((out.float() - 1).abs().max()) <= 2.0 ** -11


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("gap", [41, 80, 300])
@pytest.mark.parametrize("at", [0, 2000, 4095])
@pytest.mark.parametrize("G,rows", [(4, 700), (16, 700), (4, 2)])
def test_attention_of_a_row_that_one_slot_takes(dec, dtype, gap, at, G, rows):  # noqa: F811
    """Scores further apart than any reference follows, values near fp16's
    largest: the slot's own value and weight, in whatever order it comes.
    (exp(-41) * 4096 is below 2^-46.)"""
    n, D, page = 4096, 64, 16
    rng = np.random.default_rng(at)
    q, k, v = sink_rows(n, gap, D, 1, G, dtype, at, rng)
    v = ((rng.random((n, D)) - 0.5) * 1.2e5).astype(v.dtype)
    pages = n // page
    pool = lambda x: dev(x.reshape(pages, 1, page, D))  # noqa: E731
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].expand(rows, pages)
    w = torch.zeros(rows, 1, n, device="cuda")
    out = dec.paged_attention(dev(q)[None].expand(rows, G, D), pool(k), pool(v), table,
                              torch.full((rows,), n, dtype=torch.int32, device="cuda"), scale=1.0, weights=w,
                              weights_out=w)
    got = out.double().cpu().numpy()
    want = v[at].astype(np.float64)
    assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want) + 2.0 ** -20).all() if dtype == F32 else (got == want).all()
    weight = host(w)
    np.testing.assert_allclose(weight[:, 0, at], G, rtol=2e-6)
    rest = np.delete(weight, at, axis=2)
    np.testing.assert_allclose(rest, G * np.exp(-float(gap)), rtol=gap * 2e-6 + 1e-5, atol=1e-37)


NANS = {"quiet": 0x7fc00000, "canonical": 0x7fffffff, "negative": 0xffffffff}


@pytest.mark.parametrize("G", [1, 4, 12, 20])
@pytest.mark.parametrize("D,n", [(64, 20), (128, 300), (256, 700)])
@pytest.mark.parametrize("kind", list(NANS))
@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_of_a_live_nan_is_nan(dec, dtype, kind, D, n, G):  # noqa: F811
    """NaN of a live key or of a query reaches every result of its row, NaN of
    a live value its channel's, whatever bits the NaN has; nothing else."""
    if dtype == F32:
        nan = np.array([NANS[kind]], np.uint32).view(np.float32)[0]
    else:
        nan = np.array([NANS[kind] >> 16 if kind != "quiet" else 0x7e00], np.uint16).view(np.float16)[0]
    assert np.isnan(nan)
    c = Cache([n, n], 2, D, 16, dtype, seed=D)
    q = np.random.default_rng(0).standard_normal((2, 2 * G, D)).astype(c.k.dtype)
    clean = host(dec.paged_attention(dev(q), c.dk, c.dv, c.dtable, c.dlengths))
    assert np.isfinite(clean).all()

    def run(q=q, k=c.k, v=c.v):
        return host(dec.paged_attention(dev(q), dev(k), dev(v), c.dtable, c.dlengths))
    k = c.k.copy()
    ref.slot_row(k, c.table, 1, 0, n // 2)[D // 3] = nan
    out = run(k=k)
    assert np.isnan(out[1, :G]).all()
    np.testing.assert_array_equal(out[0], clean[0])
    np.testing.assert_array_equal(out[1, G:], clean[1, G:])
    v = c.v.copy()
    ref.slot_row(v, c.table, 1, 1, n // 2)[D // 3] = nan
    out = run(v=v)
    assert np.isnan(out[1, G:, D // 3]).all()
    out[1, G:, D // 3] = clean[1, G:, D // 3]
    np.testing.assert_array_equal(out, clean)
    qn = q.copy()
    qn[0, G, D - 1] = nan
    out = run(q=qn)
    assert np.isnan(out[0, G]).all()
    out[0, G] = clean[0, G]
    np.testing.assert_array_equal(out, clean)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("G", [2, 12, 20])
@pytest.mark.parametrize("width,n", [(8, 100), (40, 600), (400, 6000)])
@pytest.mark.parametrize("in_place", [True, False])
def test_weights_of_slots_that_are_not_live_stay(dec, dtype, G, width, n, in_place):  # noqa: F811
    """A row whose probabilities are NaN adds them to its live slots alone: what
    the mask or the window leaves out keeps its weight."""
    c = Cache([n, n], 2, 64, 16, dtype, width=width)
    slots, window = width * 16, n - 21
    rng = np.random.default_rng(0)
    mask = rng.random((2, slots)) < 0.6
    mask[1, n - 5] = True
    ref.slot_row(c.k, c.table, 1, 0, n - 5)[0] = np.nan
    w = rng.random((2, 2, slots)).astype(np.float32)
    q = rng.standard_normal((2, 2 * G, 64)).astype(c.k.dtype)
    dw = dev(w)
    wo = dw if in_place else torch.full_like(dw, -5.0)
    dec.paged_attention(dev(q), dev(c.k), c.dv, c.dtable, c.dlengths, window=window, mask=dev(mask), weights=dw,
                        weights_out=wo)
    got = host(wo)
    live = mask & (np.arange(slots) >= n - window) & (np.arange(slots) < n)
    assert np.isnan(got[1, 0][live[1]]).all()
    for b in range(2):
        for h in range(2):
            dead = ~live[b] & (np.arange(slots) < n)
            np.testing.assert_array_equal(got[b, h][dead], w[b, h][dead])
            if (b, h) != (1, 0):
                assert np.isfinite(got[b, h][:n]).all() and (got[b, h][live[b]] >= w[b, h][live[b]]).all()
    np.testing.assert_array_equal(got[:, :, n:], w[:, :, n:] if in_place else np.full_like(w[:, :, n:], -5))
