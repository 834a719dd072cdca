"""The text-decoding operators (wgx.decode and their recorded forms) against
the 64-bit statements of decode_reference.py.

Tolerances, fixed before the first run. A score s = scale * q.k is formed in
fp32 from products good to 2^-20 of themselves (fp32 caches: three tf32
products; fp16: exact), so it is off by at most about 2^-20 * sum |q_i k_i| *
scale, below 1.5e-5 for the sizes here (sum |q_i k_i| * scale <= 0.64 *
sqrt(256) for unit normals), and so is every probability's logarithm; the
weighted sum adds 2^-20 of |v|. Hence |out - ref| <= 4e-5 * max|v|, plus half a
unit of fp16 (2^-11 of the value, 2^-25 below its normal range) where the
output is fp16. Accumulated weights: 4e-5 per query head of the group. Beam
scores: a log probability of size x is formed in fp32 from a sum of V terms:
4e-6 * (1 + |score|). Everything that is moved or chosen is compared exactly.
"""
import numpy as np
import pytest
import torch

import decode_reference as ref
import wgx
from wgx import _lib

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.fixture
def dec():
    import wgx.decode
    wgx.decode.device_error(0, clear=True)
    yield wgx.decode
    wgx.decode.device_error(0, clear=True)


def host(t):
    return t.detach().cpu().numpy()


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


class Cache:
    """A paged cache with scattered pages; table entries nobody uses are
    garbage, unused slots hold NaN and infinities."""

    def __init__(self, lengths, H, D, page, dtype, order="head", room=0, seed=0, layers=0, extra=0,
                 width=None):
        rng = np.random.default_rng(seed)
        self.rng, self.page, self.dtype = rng, page, dtype
        lengths = np.asarray(lengths, np.int32)
        counts = [-(-(int(n) + room) // page) for n in lengths]
        self.width = width or max(1, max(counts)) + 1
        pages = sum(counts) + 3 + extra
        ids = rng.permutation(pages).astype(np.int32)
        self.table = np.full((len(lengths), self.width), -77, np.int32)
        at = 0
        for b, c in enumerate(counts):
            self.table[b, :c] = ids[at:at + c]
            at += c
        self.free = ids[at:]
        lead = (layers,) if layers else ()
        npdt = np.float16 if dtype == F16 else np.float32
        self.k = rng.standard_normal(lead + (pages, H, page, D)).astype(npdt)
        self.v = rng.standard_normal(lead + (pages, H, page, D)).astype(npdt)
        if not layers:
            for b, n in enumerate(lengths):
                for s in range(int(n), counts[b] * page):
                    p, r = self.table[b, s // page], s % page
                    self.k[p, :, r] = [np.nan, np.inf, -np.inf][s % 3]
                    self.v[p, :, r] = [np.inf, np.nan, -np.inf][s % 3]
            for p in self.free:
                self.k[p] = np.nan
                self.v[p] = np.nan
        self.lengths = lengths
        self.order = order
        self.dk, self.dv = self.pool(self.k), self.pool(self.v)
        self.dtable, self.dlengths = dev(self.table), dev(lengths)

    def pool(self, a):
        if self.order == "slot":  # [pages, page_size, heads, D] memory
            return dev(np.moveaxis(a, -2, -3)).transpose(-2, -3)
        if self.order == "padded":  # rows 3 elements apart from each other: nothing aligned
            big = torch.full(a.shape[:-1] + (a.shape[-1] + 3,), float("nan"), dtype=self.dtype, device="cuda")
            view = big[..., 1:1 + a.shape[-1]]
            view.copy_(dev(a))
            return view
        return dev(a)


def attention_close(out, want, vmax, half):
    out = out.astype(np.float64)
    tol = 4e-5 * vmax + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if half else 0)
    assert np.isfinite(out).all()
    bad = np.abs(out - want) - tol
    assert (bad <= 0).all(), f"off by {np.abs(out - want).max()} (excess {bad.max()})"


def check_attention(dec, c, Hq, window=0, mask=None, weights=False, scale=None, seed=1):
    rng = np.random.default_rng(seed)
    B, (_, H, _, D) = len(c.lengths), c.k.shape
    npdt = np.float16 if c.dtype == F16 else np.float32
    q = rng.standard_normal((B, Hq, D)).astype(npdt)
    slots = c.width * c.page
    w = rng.random((B, H, slots)).astype(np.float32) if weights else None
    sc = D ** -0.5 if scale is None else scale
    want, wwant = ref.paged_attention(q, c.k, c.v, c.table, c.lengths, sc, window, mask, w)
    dw = dev(w) if weights else None
    wo = torch.full_like(dw, -5.0) if weights else None
    out = dec.paged_attention(dev(q), c.dk, c.dv, c.dtable, c.dlengths, scale=scale, window=window,
                              mask=None if mask is None else dev(mask), weights=dw, weights_out=wo)
    vmax = np.abs(np.where(np.isfinite(c.v), c.v, 0)).max()
    attention_close(host(out), want, vmax, c.dtype == F16)
    if weights:
        got = host(wo)
        for b, n in enumerate(c.lengths):
            np.testing.assert_allclose(got[b, :, :n], wwant[b, :, :n], rtol=1e-6,
                                       atol=4e-5 * (Hq // H))
            assert (got[b, :, n:] == -5.0).all()  # not written
    assert dec.device_error(0) == 0
    return out


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [1, 8, 20, 64, 72, 80, 128, 130, 192, 256])
def test_attention_head_sizes(dec, dtype, D):
    check_attention(dec, Cache([37, 1, 0, 160, 16], 2, D, 16, dtype, seed=D), 6)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("H,G", [(1, 1), (3, 1), (2, 3), (2, 8), (1, 9), (2, 16), (1, 17), (1, 40), (1, 128)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_groups(dec, dtype, H, G, D):
    check_attention(dec, Cache([130, 5, 64], H, D, 32, dtype, seed=G), H * G, weights=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("page", [1, 3, 7, 8, 16, 24, 128])
@pytest.mark.parametrize("order", ["head", "slot", "padded"])
def test_attention_pages_and_strides(dec, dtype, page, order):
    check_attention(dec, Cache([1, 15, 16, 17, 0, 129, 255], 2, 64, page, dtype, order, seed=page), 4,
                    weights=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("n", [0, 1, 2, 7, 8, 9, 63, 64, 65, 300, 4097, 20001])
def test_attention_lengths(dec, dtype, n):
    """One sequence: split over the cache's length from the shortest to
    thousands of slots."""
    check_attention(dec, Cache([n], 2, 64, 16, dtype, seed=n), 4, weights=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("width", [4, 14, 30, 60, 400])
@pytest.mark.parametrize("D,G", [(64, 2), (128, 4), (256, 3), (128, 12), (64, 20)])
def test_attention_table_widths(dec, dtype, width, D, G):
    """The same sequences under tables of more and more pages: how a row's work
    is divided (a block, a cluster of blocks, shares of the whole grid) goes by
    what the table can name, the result does not."""
    check_attention(dec, Cache([64, 0, 1, 33, 50], 2, D, 16, dtype, width=width), 2 * G, weights=True)
    check_attention(dec, Cache([64, 7], 2, D, 16, dtype, width=width), 2 * G, window=20)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_attention_ragged_batch(dec, dtype):
    rng = np.random.default_rng(3)
    lengths = rng.integers(0, 700, 150)
    lengths[[0, 17, 149]] = 0
    check_attention(dec, Cache(lengths, 3, 64, 16, dtype), 6, weights=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 5000])
def test_attention_window(dec, dtype, window):
    check_attention(dec, Cache([0, 1, 16, 90, 333, 1025], 2, 80, 16, dtype), 4, window=window, weights=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("kind", ["random", "left", "none", "alternate", "short"])
def test_attention_mask(dec, dtype, kind):
    """Masks, one that leaves a sequence nothing and one shorter than the
    cache; masked slots hold NaN and infinities."""
    lengths = [40, 0, 17, 260, 1]
    c = Cache(lengths, 2, 64, 16, dtype)
    n = c.width * c.page
    rng = np.random.default_rng(5)
    mask = {"random": rng.random((5, n)) < 0.5, "left": np.arange(n)[None] >= np.array([[3], [0], [17], [255], [0]]),
            "none": np.zeros((5, n), bool), "alternate": np.tile(np.arange(n) % 2 == 1, (5, 1)),
            "short": np.ones((5, 33), bool)}[kind].copy()
    if kind == "random":
        mask[3] = False
    for b, m in enumerate(lengths):
        for s in range(m):
            if s >= mask.shape[1] or not mask[b, s]:
                p, r = c.table[b, s // 16], s % 16
                c.k[p, :, r] = np.nan if s % 2 else np.inf
                c.v[p, :, r] = np.inf if s % 2 else np.nan
    c.dk, c.dv = c.pool(c.k), c.pool(c.v)
    check_attention(dec, c, 6, mask=mask, weights=True)
    check_attention(dec, c, 6, mask=mask.astype(np.uint8) * 3, window=30)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("window", [1, 8, 17, 64, 200])
@pytest.mark.parametrize("lengths", [[40, 700, 16], [3000]])
def test_attention_window_over_a_long_cache(dec, dtype, window, lengths):
    """The window's slots only, whatever the table can name; weights in place:
    the slots in front of the window stay as they are."""
    c = Cache(lengths, 2, 64, 16, dtype)
    check_attention(dec, c, 4, window=window)
    check_attention(dec, c, 4, window=window, weights=True)
    rng = np.random.default_rng(1)
    q = rng.standard_normal((len(lengths), 4, 64)).astype(np.float16 if dtype == F16 else np.float32)
    w = rng.random((len(lengths), 2, c.width * 16)).astype(np.float32)
    dw = dev(w)
    dec.paged_attention(dev(q), c.dk, c.dv, c.dtable, c.dlengths, window=window, weights=dw, weights_out=dw)
    _, want = ref.paged_attention(q, c.k, c.v, c.table, c.lengths, 0.125, window, None, w)
    got = host(dw)
    for b, n in enumerate(lengths):
        first = max(0, n - window)
        np.testing.assert_array_equal(got[b, :, :first], w[b, :, :first])
        np.testing.assert_allclose(got[b, :, first:n], want[b, :, first:n], rtol=1e-6, atol=8e-5)
        np.testing.assert_array_equal(got[b, :, n:], w[b, :, n:])


def test_attention_extreme_scores(dec):
    """Scores far apart (one slot takes all) and a scale of zero (all equal)."""
    for dtype in (F16, F32):
        c = Cache([100, 37], 2, 64, 16, dtype)
        q = np.random.default_rng(0).standard_normal((2, 4, 64)).astype(np.float16 if dtype == F16 else np.float32)
        for scale in (0.0, 30.0, -30.0):
            # exp of a score s is off by |s| * 2^-23: relative, on top of the
            # products' error, for |s| up to about 30 * 8 * 3
            want, _ = ref.paged_attention(q, c.k, c.v, c.table, c.lengths, scale)
            out = host(dec.paged_attention(dev(q), c.dk, c.dv, c.dtable, c.dlengths, scale=scale))
            tol = 2.0 ** -11 * np.abs(want) + (1e-4 if scale == 0 else 2e-2)
            assert (np.abs(out - want) <= tol).all()
        # one K/V row that dwarfs the others
        huge = c.dk.clone()
        p, r = int(c.table[0, 2]), 3
        huge[p, 0, r] = dev(q[0, 0]).to(dtype) * 60
        out = host(dec.paged_attention(dev(q), huge, c.dv, c.dtable, c.dlengths))
        np.testing.assert_allclose(out[0, 0], c.v[p, 0, r], rtol=2e-3, atol=1e-4)


def test_attention_beyond_32_bit_offsets(dec):
    """Pages more than 2^32 elements into the pool."""
    H, page, D = 8, 16, 128
    pages = (1 << 32) // (H * page * D) + 40
    pool = torch.empty(pages, H, page, D, dtype=F16, device="cuda")
    c = Cache([200, 77], H, D, page, F16)
    far = np.arange(pages - c.k.shape[0], pages, dtype=np.int64)
    pool[dev(far)] = c.dk
    vpool = torch.empty(pages, H, page, D, dtype=F16, device="cuda")
    vpool[dev(far)] = c.dv
    used = c.table >= 0
    table = np.where(used, far[np.where(used, c.table, 0)], -1).astype(np.int32)
    q = np.random.default_rng(0).standard_normal((2, 16, D)).astype(np.float16)
    want, _ = ref.paged_attention(q, c.k, c.v, c.table, c.lengths, D ** -0.5)
    out = dec.paged_attention(dev(q), pool, vpool, dev(table), c.dlengths)
    attention_close(host(out), want, 6.0, True)
    new = torch.randn(2, 1, H, D, device="cuda").half()
    dec.kv_append(new, new, pool, vpool, dev(table), c.dlengths, c.dlengths)
    for b, n in enumerate([200, 77]):
        assert (pool[int(table[b, n // page]), :, n % page] == new[b, 0]).all()


def test_attention_strided_query_and_output(dec):
    c = Cache([50, 120], 2, 64, 16, F16)
    rng = np.random.default_rng(2)
    big = dev(rng.standard_normal((2, 3, 4, 64)).astype(np.float16))
    out = torch.zeros(2, 4, 3, 64, dtype=F16, device="cuda")
    dec.paged_attention(big[:, 1], c.dk, c.dv, c.dtable, c.dlengths, out[:, :, 1])
    want, _ = ref.paged_attention(host(big[:, 1]), c.k, c.v, c.table, c.lengths, 0.125)
    attention_close(host(out[:, :, 1]), want, 6.0, True)
    assert (out[:, :, 0] == 0).all() and (out[:, :, 2] == 0).all()


def test_attention_is_deterministic_and_accumulates_in_place(dec):
    c = Cache([3000, 11], 2, 128, 16, F16)
    q = dev(np.random.default_rng(2).standard_normal((2, 8, 128)).astype(np.float16))
    w = torch.zeros(2, 2, c.width * 16, device="cuda")
    first = dec.paged_attention(q, c.dk, c.dv, c.dtable, c.dlengths, weights=w, weights_out=w).clone()
    once = w.clone()
    for _ in range(3):
        again = dec.paged_attention(q, c.dk, c.dv, c.dtable, c.dlengths, weights=w, weights_out=w)
        assert torch.equal(first, again)
    np.testing.assert_allclose(host(w), 4 * host(once), rtol=1e-5)
    # a K/V head's weights of one step sum to its group
    np.testing.assert_allclose(host(once).sum(axis=2), 4.0, rtol=1e-5)


def test_calls_follow_the_current_stream(dec):
    """A call on a side stream is ordered with that stream's work: the cache
    it reads is written there just before, behind a long queue."""
    c = Cache([500, 300], 4, 128, 16, F16)
    q = dev(np.random.default_rng(2).standard_normal((2, 8, 128)).astype(np.float16))
    want = dec.paged_attention(q, c.dk, c.dv, c.dtable, c.dlengths).clone()
    kz, vz = torch.zeros_like(c.dk), torch.zeros_like(c.dv)
    x = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(4):
            x = x @ x * 1e-3
        kz.copy_(c.dk)
        vz.copy_(c.dv)
        out = dec.paged_attention(q, kz, vz, c.dtable, c.dlengths)
    side.synchronize()
    assert torch.equal(out, want)


def test_bad_pages_and_lengths_are_left_out_and_noted(dec):
    """Device data outside the cache is never followed: a bad page's slots are
    left out, a length is held within the table's slots."""
    c = Cache([40, 64], 2, 64, 16, F16)
    q = dev(np.random.default_rng(2).standard_normal((2, 4, 64)).astype(np.float16))
    for bad in (-1, c.k.shape[0], 2 ** 31 - 1):
        table = c.table.copy()
        table[1, 2] = bad
        out = dec.paged_attention(q, c.dk, c.dv, dev(table), c.dlengths)
        mask = np.ones((2, c.width * 16), bool)
        mask[1, 32:48] = False
        want, _ = ref.paged_attention(host(q), c.k, c.v, c.table, c.lengths, 0.125, mask=mask)
        attention_close(host(out), want, 6.0, True)
        assert dec.device_error(0) == 32 and dec.device_error(0) == 0
    out = dec.paged_attention(q, c.dk, c.dv, dev(np.abs(c.table) % c.k.shape[0]),
                              dev(np.array([-3, 10 ** 6], np.int32)))
    assert (out[0] == 0).all()
    assert dec.device_error(0) == 32


# --------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("T", [1, 3, 50])
@pytest.mark.parametrize("D,order", [(64, "head"), (20, "head"), (80, "slot"), (64, "padded")])
def test_append(dec, dtype, T, D, order):
    lengths = [0, 7, 16, 33]
    c = Cache(lengths, 3, D, 16, dtype, order, room=T)
    npdt = np.float16 if dtype == F16 else np.float32
    rng = np.random.default_rng(T)
    k, v = (rng.standard_normal((4, T, 3, D)).astype(npdt) for _ in range(2))
    k0, v0 = host(c.dk).copy(), host(c.dv).copy()
    slots = c.width * 16
    w = torch.ones(4, 3, slots, device="cuda")
    pos = torch.full((4, 3, slots), -1, dtype=torch.int32, device="cuda")
    seen = np.array([0, 9, 40, 33], np.int32)
    ds, dl = dev(seen), c.dlengths.clone()
    dec.kv_append(dev(k), dev(v), c.dk, c.dv, c.dtable, dl, dl, seen=ds, seen_out=ds, positions=pos, weights=w)
    for b, n in enumerate(lengths):
        for t in range(T):
            for h in range(3):
                ref.slot_row(k0, c.table, b, h, n + t)[:] = k[b, t, h]
                ref.slot_row(v0, c.table, b, h, n + t)[:] = v[b, t, h]
        assert (host(w)[b, :, n:n + T] == 0).all() and (host(w)[b, :, :n] == 1).all()
        assert (host(w)[b, :, n + T:] == 1).all()
        assert (host(pos)[b, :, n:n + T] == seen[b] + np.arange(T)).all()
        assert (host(pos)[b, :, :n] == -1).all() and (host(pos)[b, :, n + T:] == -1).all()
    np.testing.assert_array_equal(host(c.dk), k0)  # NaN of unused slots included
    np.testing.assert_array_equal(host(c.dv), v0)
    assert (host(dl) == np.array(lengths) + T).all() and (host(ds) == seen + T).all()
    assert dec.device_error(0) == 0


def test_append_strided_rows_and_many_tokens(dec):
    """K and V as slices of one projection; enough tokens for many blocks."""
    T, H, D = 700, 4, 64
    c = Cache([5, 0], H, D, 32, F16, room=T)
    qkv = torch.randn(2, T, 3 * H, D, device="cuda").half()
    lo = torch.empty_like(c.dlengths)
    dec.kv_append(qkv[:, :, H:2 * H], qkv[:, :, 2 * H:], c.dk, c.dv, c.dtable, c.dlengths, lo)
    assert host(lo).tolist() == [5 + T, T] and host(c.dlengths).tolist() == [5, 0]
    for b, n in enumerate([5, 0]):
        for t in (0, 1, 333, T - 1):
            p, r = int(c.table[b, (n + t) // 32]), (n + t) % 32
            assert (c.dk[p, :, r] == qkv[b, t, H:2 * H]).all() and (c.dv[p, :, r] == qkv[b, t, 2 * H:]).all()


def test_append_without_room_changes_nothing(dec):
    for T in (1, 400):  # one block a sequence, and several
        c = Cache([16, 3], 2, 64, 16, F16, width=1, extra=4)
        k0 = host(c.dk).copy()
        new = torch.ones(2, T, 2, 64, device="cuda").half()
        lo = c.dlengths.clone()
        dec.kv_append(new, new, c.dk, c.dv, c.dtable, lo, lo)
        assert host(lo).tolist() == [16, 4 if T == 1 else 3]
        if T == 1:
            k0[c.table[1, 0], :, 3] = 1
        np.testing.assert_array_equal(host(c.dk), k0)
        assert dec.device_error(0) == 32


# ---------------------------------------------------------------------- evict
def evict_case(dec, lengths, H, D, page, budget, recent, sinks, dtype=F16, order="head", weights=None,
               in_place=False, seed=0, seen=None):
    rng = np.random.default_rng(seed)
    c = Cache(lengths, H, D, page, dtype, order, seed=seed)
    B, slots = len(lengths), c.width * page
    w = rng.random((B, H, slots)).astype(np.float32) ** 3 if weights is None else weights(rng, (B, H, slots))
    seen = np.array([n + n // 4 for n in lengths], np.int32) if seen is None else seen
    pos = np.full((B, H, slots), -1, np.int32)
    for b, n in enumerate(lengths):
        for h in range(H):
            pos[b, h, :n] = rng.permutation(int(seen[b]))[:n]
    dw, dp, dl = dev(w), dev(pos), c.dlengths
    if in_place:
        wo, po, lo = dw, dp, dl
    else:
        wo, po, lo = torch.full_like(dw, -9.0), torch.full_like(dp, -9), torch.empty_like(dl)
    dec.cache_evict(c.dk, c.dv, c.dtable, dl, lo, dw, wo, dp, po, dev(seen), budget=budget, recent=recent,
                    sinks=sinks)
    k, v = c.k, c.v
    lwant = ref.cache_evict(k, v, c.table, c.lengths, w, pos, seen, budget, recent, sinks)
    assert (host(lo) == lwant).all()
    np.testing.assert_array_equal(host(c.dk), k)
    np.testing.assert_array_equal(host(c.dv), v)
    gw, gp = host(wo), host(po)
    for b, n in enumerate(lwant):
        np.testing.assert_array_equal(gw[b, :, :n], w[b, :, :n])
        np.testing.assert_array_equal(gp[b, :, :n], pos[b, :, :n])
        if not in_place:
            assert (gp[b, :, n:] == -9).all()
    assert dec.device_error(0) == 0
    return gp, lwant, seen


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,D,order", [(F16, 64, "head"), (F32, 80, "slot"), (F16, 20, "head"),
                                            (F32, 33, "padded"), (F16, 256, "slot")])
def test_evict_rows(dec, dtype, D, order, in_place):
    evict_case(dec, [0, 1, 50, 51, 90, 333], 3, D, 16, 50, 10, 4, dtype, order, in_place=in_place)


@pytest.mark.parametrize("budget,recent,sinks", [(1, 0, 0), (1, 1, 0), (2, 0, 2), (64, 64, 0), (64, 0, 0),
                                                 (100, 60, 40), (999, 3, 1), (1000, 0, 0), (1200, 5, 5)])
def test_evict_budgets(dec, budget, recent, sinks):
    gp, lo, seen = evict_case(dec, [1000, 63, 64, 65], 2, 64, 32, budget, recent, sinks)
    for b in range(4):  # nobody lost a protected token that the cache held
        for h in range(2):
            kept = set(gp[b, h, :lo[b]].tolist())
            assert len(kept) == lo[b]


@pytest.mark.parametrize("kind", ["equal", "few", "nan", "inf", "negative", "zeros", "tiny"])
def test_evict_ties_and_special_weights(dec, kind):
    def make(rng, shape):
        if kind == "equal":
            return np.full(shape, 0.25, np.float32)
        if kind == "few":
            return rng.integers(0, 3, shape).astype(np.float32)
        if kind == "zeros":  # -0 and +0 tie
            return np.where(rng.random(shape) < 0.5, 0.0, -0.0).astype(np.float32)
        if kind == "tiny":  # neighbours in the last place
            return (np.float32(1) + rng.integers(0, 5, shape).astype(np.float32) * np.float32(2 ** -23))
        w = rng.standard_normal(shape).astype(np.float32)
        if kind == "negative":
            return w - 1
        w[rng.random(shape) < 0.3] = np.nan if kind == "nan" else np.inf
        if kind == "inf":
            w[rng.random(shape) < 0.2] = -np.inf
        return w
    evict_case(dec, [300, 777, 100], 2, 64, 16, 120, 16, 2, weights=make)
    evict_case(dec, [5000], 1, 64, 16, 1300, 0, 0, weights=make)  # a cluster of CTAs


@pytest.mark.parametrize("n,budget", [(2049, 2048), (9000, 100), (20000, 5001), (20000, 19999), (40000, 13000)])
def test_evict_long(dec, n, budget):
    """Sequences spread over the CTAs of a cluster; the budget's place inside
    any of them."""
    evict_case(dec, [n], 1, 8, 64, budget, 50, 4)


# ----------------------------------------------------------------------- beam
def beam_case(dec, logits, scores, finished, eos=2, dtype=None):
    B, W, V = logits.shape
    x = logits if torch.is_tensor(logits) else dev(logits)
    outs = [torch.full((B, W), -1.0, device="cuda"), torch.full((B, W), -1, dtype=torch.int32, device="cuda"),
            torch.full((B, W), -1, dtype=torch.int32, device="cuda"),
            torch.zeros(B, W, dtype=torch.bool, device="cuda")]
    dec.beam_search_step(x, dev(scores), dev(finished), *outs, eos=eos)
    so, pa, to, fo = ref.beam_search_step(host(x), scores, finished, eos)
    got = [host(t) for t in outs]
    np.testing.assert_array_equal(got[1], pa)
    np.testing.assert_array_equal(got[2], to)
    np.testing.assert_array_equal(got[3], fo)
    fin = np.isfinite(so)
    np.testing.assert_array_equal(np.isfinite(got[0]), fin)
    assert (np.abs(got[0][fin] - so[fin]) <= 4e-6 * (1 + np.abs(so[fin]))).all()
    return got


def beam_inputs(B, W, V, np_dtype, seed=0, done=0.15):
    rng = np.random.default_rng(seed)
    return ((rng.standard_normal((B, W, V)) * 3).astype(np_dtype),
            (-rng.random((B, W)) * 4 - 3).astype(np.float32), rng.random((B, W)) < done)


@pytest.mark.parametrize("np_dtype", [np.float16, np.float32])
@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (1, 1, 50257), (3, 2, 2), (2, 4, 3), (1, 5, 8191), (2, 3, 8192),
                                   (1, 4, 8193), (5, 4, 1000), (2, 8, 33333), (1, 16, 20001), (1, 32, 9001),
                                   (40, 2, 517), (1, 32, 7)])
def test_beam_sizes(dec, np_dtype, B, W, V):
    beam_case(dec, *beam_inputs(B, W, V, np_dtype, seed=V))


@pytest.mark.parametrize("np_dtype", [np.float16, np.float32])
@pytest.mark.parametrize("kind", ["equal", "equal_rows", "two_values", "ascending", "descending", "ninf",
                                  "all_ninf", "nan", "pinf", "all_done", "one_open", "ninf_scores"])
def test_beam_ties_and_special_values(dec, np_dtype, kind):
    B, W, V = 2, 4, 9999
    x, s, f = beam_inputs(B, W, V, np_dtype, seed=1)
    rng = np.random.default_rng(9)
    if kind == "equal":  # every logit of a beam: the lowest tokens
        x[:] = 1.0
    elif kind == "equal_rows":  # the first step: all beams alike
        x[:] = x[:, :1]
        s[:] = -1.0
        f[:] = False
    elif kind == "two_values":
        x = rng.integers(0, 2, x.shape).astype(np_dtype)
    elif kind in ("ascending", "descending"):
        r = np.linspace(-8, 8, V)
        x[:] = (r if kind == "ascending" else r[::-1]).astype(np_dtype)
        s = -np.arange(B * W, dtype=np.float32).reshape(B, W)
    elif kind == "ninf":  # all but a few tokens forbidden
        keep = rng.random(x.shape) < 0.001
        x = np.where(keep, x, -np.inf).astype(np_dtype)
    elif kind == "all_ninf":
        x[0] = -np.inf
        x[1, 1] = -np.inf
    elif kind == "nan":
        x[rng.random(x.shape) < 0.3] = np.nan
        x[0, 2] = np.nan
    elif kind == "pinf":
        x[0, 1, 77] = np.inf
    elif kind == "all_done":
        f[:] = True
    elif kind == "one_open":
        f[:] = True
        f[:, 2] = False
    elif kind == "ninf_scores":  # the first step again: only beam 0 counts
        s[:, 1:] = -np.inf
    beam_case(dec, x, s, f)


def test_beam_strided_logits(dec):
    """Rows of a padded vocabulary, at odd starts."""
    for dtype in (F16, F32):
        big = (torch.randn(3, 4, 1, 5013, device="cuda") * 3).to(dtype)
        s = -np.random.default_rng(0).random((3, 4)).astype(np.float32)
        beam_case(dec, big[:, :, 0, 3:5004], s, np.zeros((3, 4), bool))


@pytest.mark.parametrize("dtype,D,layers", [(F16, 64, 1), (F16, 64, 3), (F32, 80, 2), (F16, 20, 2)])
@pytest.mark.parametrize("length", [0, 1, 15, 16, 37, 48])
def test_beam_state(dec, dtype, D, layers, length):
    """Children share their parents' full pages; the used part of a partly
    filled last page is copied in every layer."""
    B, W, V = 2, 3, 501
    n = B * W
    lengths = [length] * W + [max(0, length - 2)] * W
    c = Cache(lengths, 2, D, 16, dtype, layers=layers, extra=n)
    x, s, f = beam_inputs(B, W, V, np.float16, seed=length)
    spare = c.free[:n].copy()
    table = np.where(c.table < 0, 0, c.table)
    outs = [torch.empty(B, W, device="cuda"), torch.empty(B, W, dtype=torch.int32, device="cuda"),
            torch.empty(B, W, dtype=torch.int32, device="cuda"), torch.empty(B, W, dtype=torch.uint8, device="cuda")]
    to, lo = torch.empty(n, c.width, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    k4, v4 = (c.dk[0], c.dv[0]) if layers == 1 else (c.dk, c.dv)
    dec.beam_search_step(dev(x), dev(s), dev(f), *outs, eos=2, k_cache=k4, v_cache=v4, page_table=dev(table),
                         lengths=c.dlengths, spare=dev(spare), page_table_out=to, lengths_out=lo)
    so, pa, tok, fo = ref.beam_search_step(x, s, f, 2)
    np.testing.assert_array_equal(host(outs[1]), pa)
    np.testing.assert_array_equal(host(outs[2]), tok)
    np.testing.assert_array_equal(host(outs[3]) != 0, fo)
    twant, lwant = ref.reorder(c.k, c.v, table, c.lengths, spare, pa, W)
    np.testing.assert_array_equal(host(to), twant)
    np.testing.assert_array_equal(host(lo), lwant)
    np.testing.assert_array_equal(host(c.dk), c.k)
    np.testing.assert_array_equal(host(c.dv), c.v)
    assert dec.device_error(0) == 0


def test_beam_bad_pages_are_not_followed(dec):
    c = Cache([5, 5], 1, 64, 16, F16, layers=1, extra=2)
    x, s, f = beam_inputs(1, 2, 100, np.float16)
    k0 = host(c.dk).copy()
    outs = [torch.empty(1, 2, device="cuda"), torch.empty(1, 2, dtype=torch.int32, device="cuda"),
            torch.empty(1, 2, dtype=torch.int32, device="cuda"), torch.empty(1, 2, dtype=torch.bool, device="cuda")]
    dec.beam_search_step(dev(x), dev(s), dev(f), *outs, eos=2, k_cache=c.dk, v_cache=c.dv, page_table=c.dtable,
                         lengths=c.dlengths, spare=dev(np.array([-1, 10 ** 6], np.int32)),
                         page_table_out=torch.empty_like(c.dtable), lengths_out=torch.empty_like(c.dlengths))
    assert dec.device_error(0) == 32
    np.testing.assert_array_equal(host(c.dk), k0)


# -------------------------------------------------------------- recorded form
def T(ctx, a):
    names = {"float16": "float16", "float32": "float32", "int32": "int32", "bool": "bool", "uint8": "uint8"}
    a = np.ascontiguousarray(a)
    return ctx.tensor(names[a.dtype.name], list(a.shape)).setData(a)


def test_recorded_steps_replay_over_a_growing_cache(ctx):
    """kv_append and paged_attention recorded once; every submit is one more
    token, its length counted on the device."""
    B, H, G, D, page, steps = 2, 2, 3, 64, 16, 20
    c = Cache([14, 0], H, D, page, F16, room=steps)
    rng = np.random.default_rng(0)
    k, v, q = ctx.tensor("float16", [B, 1, H, D]), ctx.tensor("float16", [B, 1, H, D]), ctx.tensor("float16", [B, H * G, D])
    kc, vc, table, length = T(ctx, c.k), T(ctx, c.v), T(ctx, np.where(c.table < 0, 0, c.table)), T(ctx, c.lengths)
    slots = c.width * page
    w, pos, seen = T(ctx, np.zeros((B, H, slots), np.float32)), T(ctx, np.zeros((B, H, slots), np.int32)), T(ctx, c.lengths)
    out = ctx.tensor("float16", [B, H * G, D])
    ctx.recordShader(wgx.shaders.kvAppend, [k, v, table, length, pos, seen, w, kc, vc, seen, length])
    ctx.recordShader(wgx.shaders.pagedAttention, [q, kc, vc, table, length, None, None, 0, w, w, out])
    total = np.zeros((B, H, slots))
    n = c.lengths.copy()
    for _ in range(steps):
        hk, hv = (rng.standard_normal((B, 1, H, D)).astype(np.float16) for _ in range(2))
        hq = rng.standard_normal((B, H * G, D)).astype(np.float16)
        k.setData(hk), v.setData(hv), q.setData(hq)
        ctx.submit()
        ctx.sync()
        for b in range(B):
            for h in range(H):
                ref.slot_row(c.k, c.table, b, h, n[b])[:] = hk[b, 0, h]
                ref.slot_row(c.v, c.table, b, h, n[b])[:] = hv[b, 0, h]
        n += 1
        want, total = ref.paged_attention(hq, c.k, c.v, c.table, n, D ** -0.5, weights=total)
        attention_close(out.numpy(), want, 6.0, True)
    assert (length.numpy() == n).all() and (seen.numpy() == n).all()
    np.testing.assert_allclose(w.numpy(), total, atol=4e-5 * G * steps)
    for b in range(B):
        new = np.arange(c.lengths[b], n[b])
        assert (pos.numpy()[b][:, new] == new).all()
    assert ctx.stats()["commands"] == 2


def test_recorded_evict_and_beam(ctx):
    c = Cache([90, 30], 2, 64, 16, F16)
    slots = c.width * 16
    rng = np.random.default_rng(1)
    w = rng.random((2, 2, slots)).astype(np.float32)
    pos = np.stack([[rng.permutation(slots)] * 2 for _ in range(2)]).astype(np.int32)
    seen = np.array([slots, slots], np.int32)
    kc, vc, table, length = T(ctx, c.k), T(ctx, c.v), T(ctx, c.table), T(ctx, c.lengths)
    dw, dp, ds = T(ctx, w), T(ctx, pos), T(ctx, seen)
    ctx.recordShader(wgx.shaders.cacheEvict, [table, length, ds, dw, dp, 40, 8, 2, kc, vc, dw, dp, length])
    x, s, f = beam_inputs(1, 2, 1000, np.float16)
    spare = T(ctx, c.free[:2])
    so, pa, to = ctx.tensor("float32", [1, 2]), ctx.tensor("int32", [1, 2]), ctx.tensor("int32", [1, 2])
    fo, tout, lout = ctx.tensor("bool", [1, 2]), ctx.tensor("int32", list(c.table.shape)), ctx.tensor("int32", [2])
    ctx.recordShader(wgx.shaders.beamSearchStep, [T(ctx, x), T(ctx, s), T(ctx, f), 2, length, table, spare, kc, vc,
                                                 so, pa, to, fo, tout, lout])
    ctx.submit()
    ctx.sync()
    lwant = ref.cache_evict(c.k, c.v, c.table, c.lengths, w, pos, seen, 40, 8, 2)
    bs, bp, bt, bf = ref.beam_search_step(x, s, f, 2)
    twant, l2 = ref.reorder(c.k[None], c.v[None], c.table, lwant, c.free[:2], bp, 2)
    assert (length.numpy() == lwant).all() and (lout.numpy() == l2).all()
    np.testing.assert_array_equal(pa.numpy(), bp)
    np.testing.assert_array_equal(to.numpy(), bt)
    np.testing.assert_array_equal(tout.numpy(), twant)
    np.testing.assert_array_equal(kc.numpy(), c.k)
    np.testing.assert_array_equal(vc.numpy(), c.v)
    np.testing.assert_array_equal(fo.numpy(), bf)


def test_recorded_in_a_program(ctx):
    """The operators as a Program's chain: the cache is an input that stays in
    place from submit to submit."""
    B, H, D, page = 1, 2, 64, 16
    c = Cache([3], H, D, page, F16, room=4)
    shapes = [("float16", [B, 1, H, D]), ("float16", [B, 1, H, D]), ("float16", [B, H, D]),
              ("float16", list(c.k.shape)), ("float16", list(c.v.shape)), ("int32", list(c.table.shape)),
              ("int32", [B]), ("int32", [B]), ("float16", [B, H, D])]
    prog = {
        "version": "1",
        "chain": [{"name": "wgx.kv_append.default", "args": [0, 1, 5, 6, 9, 9, 9, 3, 4, 9, 7]},
                  {"name": "wgx.paged_attention.default", "args": [2, 3, 4, 5, 7, 9, 9, 9, 9, 9, 8]}],
        "values": [{"type": "tensor", "shape": s, "dtype": dt, "memObjId": i}
                   for i, (dt, s) in enumerate(shapes)] + [{"type": "null"}],
        "inputIds": [0, 1, 2, 3, 4, 5, 6], "outputIds": [7, 8],
        "memoryPlan": {"pools": [{"id": i, "size": int(np.prod(s)) * (2 if dt == "float16" else 4)}
                                 for i, (dt, s) in enumerate(shapes)]},
    }
    rng = np.random.default_rng(0)
    kc, vc, table = T(ctx, c.k), T(ctx, c.v), T(ctx, np.where(c.table < 0, 0, c.table))
    length, lout, out = T(ctx, c.lengths), ctx.tensor("int32", [B]), ctx.tensor("float16", [B, H, D])
    hk, hv = (rng.standard_normal((B, 1, H, D)).astype(np.float16) for _ in range(2))
    hq = rng.standard_normal((B, H, D)).astype(np.float16)
    ctx.recordProgram(prog, b"", [T(ctx, hk), T(ctx, hv), T(ctx, hq), kc, vc, table, length, lout, out])
    ctx.submit()
    ctx.sync()
    for h in range(H):
        ref.slot_row(c.k, c.table, 0, h, 3)[:] = hk[0, 0, h]
        ref.slot_row(c.v, c.table, 0, h, 3)[:] = hv[0, 0, h]
    want, _ = ref.paged_attention(hq, c.k, c.v, c.table, c.lengths + 1, D ** -0.5)
    attention_close(out.numpy(), want, 6.0, True)
    assert lout.numpy().tolist() == [4]
    np.testing.assert_array_equal(kc.numpy(), c.k)  # the caller's cache itself


# ------------------------------------------------------------------- refusals
def test_refusals(dec):
    c = Cache([20, 10], 2, 64, 16, F16)
    q = torch.zeros(2, 4, 64, dtype=F16, device="cuda")
    ok = dict(q=q, k_cache=c.dk, v_cache=c.dv, page_table=c.dtable, lengths=c.dlengths)

    def attention(match, **kw):
        with pytest.raises(wgx.WgxError, match=match):
            dec.paged_attention(**{**ok, **kw})
    attention("multiple of the K/V heads", q=torch.zeros(2, 3, 64, dtype=F16, device="cuda"))
    attention("matching float32 or float16", q=q.float())
    attention("matching float32 or float16", v_cache=c.dv.float())
    attention("matching float32 or float16", k_cache=c.dk.double())
    attention("q must be", q=q[:1])
    attention("v_cache shape", v_cache=c.dv[:1])
    attention("int32", page_table=c.dtable.long())
    attention("lengths", lengths=c.dlengths.long())
    attention("lengths", lengths=c.dlengths[:1])
    attention("window", window=-1)
    attention("NaN", scale=float("nan"))
    attention("come together", weights=torch.zeros(2, 2, 100, device="cuda"))
    attention("cover every slot", weights=torch.zeros(2, 2, 8, device="cuda"),
              weights_out=torch.zeros(2, 2, 8, device="cuda"))
    attention("mask", mask=torch.ones(1, 20, dtype=torch.bool, device="cuda"))
    attention("bool or uint8", mask=torch.ones(2, 20, device="cuda"))
    attention("unit last stride", k_cache=c.dk.transpose(2, 3).contiguous().transpose(2, 3))
    attention("scratch of", workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    attention("workspace", workspace=torch.empty(16, device="cuda"))
    attention("CUDA device", k_cache=c.dk.cpu())
    attention("cache's device", q=q.cpu())
    attention("head size", q=torch.zeros(2, 4, 257, dtype=F16, device="cuda"),
              k_cache=torch.zeros(4, 2, 16, 257, dtype=F16, device="cuda"),
              v_cache=torch.zeros(4, 2, 16, 257, dtype=F16, device="cuda"))
    attention("128 query heads", q=torch.zeros(2, 258, 64, dtype=F16, device="cuda"))

    k = torch.zeros(2, 1, 2, 64, dtype=F16, device="cuda")
    with pytest.raises(wgx.WgxError, match="k and v must be"):
        dec.kv_append(k, k[:, :, :1], c.dk, c.dv, c.dtable, c.dlengths, c.dlengths)
    with pytest.raises(wgx.WgxError, match="at least one token"):
        dec.kv_append(k[:, :0], k[:, :0], c.dk, c.dv, c.dtable, c.dlengths, c.dlengths)
    with pytest.raises(wgx.WgxError, match="come together"):
        dec.kv_append(k, k, c.dk, c.dv, c.dtable, c.dlengths, c.dlengths, seen=c.dlengths)
    with pytest.raises(wgx.WgxError, match="positions need seen"):
        dec.kv_append(k, k, c.dk, c.dv, c.dtable, c.dlengths, c.dlengths,
                      positions=torch.zeros(2, 2, 100, dtype=torch.int32, device="cuda"))

    slots = c.width * 16
    w, p = torch.zeros(2, 2, slots, device="cuda"), torch.zeros(2, 2, slots, dtype=torch.int32, device="cuda")

    def evict(match, **kw):
        with pytest.raises(wgx.WgxError, match=match):
            dec.cache_evict(c.dk, c.dv, c.dtable, c.dlengths, c.dlengths, kw.pop("w", w), kw.pop("wo", w), p, p,
                            c.dlengths, **{**dict(budget=8), **kw})
    evict("budget must be positive", budget=0)
    evict("recent \\+ sinks", recent=7, sinks=2)
    evict("recent \\+ sinks", recent=-1)
    evict("weights_out", wo=w[:, :, :8])
    evict("weights must be", w=w.double())

    x, s = torch.zeros(1, 2, 9, device="cuda"), torch.zeros(1, 2, device="cuda")
    f = torch.zeros(1, 2, dtype=torch.bool, device="cuda")
    i = torch.zeros(1, 2, dtype=torch.int32, device="cuda")

    def step(match, x=x, s=s, so=s.clone(), **kw):
        with pytest.raises(wgx.WgxError, match=match):
            dec.beam_search_step(x, s, f, so, i, i.clone(), f.clone(), eos=0, **kw)
    step("overlap", so=s)
    step("logits", x=x.double())
    step("logits", x=x[0])
    step("scores", s=s[:, :1])
    many = [torch.zeros(1, 33, dtype=d, device="cuda")
            for d in (F32, torch.bool, F32, torch.int32, torch.int32, torch.bool)]
    with pytest.raises(wgx.WgxError, match="beams must be"):
        dec.beam_search_step(torch.zeros(1, 33, 9, device="cuda"), *many, eos=0)
    step("come together", k_cache=c.dk)
    step("overlap", k_cache=c.dk, v_cache=c.dv, page_table=c.dtable, lengths=c.dlengths,
         spare=c.dlengths.clone(), page_table_out=c.dtable, lengths_out=torch.empty_like(c.dlengths))
    assert dec.device_error(0) == 0


def test_refusals_of_the_recorders(ctx):
    t = lambda dt, *s: ctx.tensor(dt, list(s))  # noqa: E731
    kc, vc, table, ln = t("float16", 4, 2, 16, 64), t("float16", 4, 2, 16, 64), t("int32", 2, 2), t("int32", 2)
    q, out = t("float16", 2, 4, 64), t("float16", 2, 4, 64)
    with pytest.raises(wgx.WgxError, match="expected 11 args"):
        ctx.recordShader(wgx.shaders.pagedAttention, [q, kc, vc, table, ln])
    with pytest.raises(wgx.WgxError, match="out shape"):
        ctx.recordShader(wgx.shaders.pagedAttention, [q, kc, vc, table, ln, None, None, None, None, None,
                                                     t("float16", 2, 4, 32)])
    with pytest.raises(wgx.WgxError, match="q has dtype float32"):
        ctx.recordShader(wgx.shaders.pagedAttention, [t("float32", 2, 4, 64), kc, vc, table, ln, None, None, None,
                                                     None, None, out])
    with pytest.raises(wgx.WgxError, match="must be an integer"):
        ctx.recordShader(wgx.shaders.pagedAttention, [q, kc, vc, table, ln, None, None, 1.5, None, None, out])
    with pytest.raises(wgx.WgxError, match="page_table must be a Tensor"):
        ctx.recordShader(wgx.shaders.pagedAttention, [q, kc, vc, None, ln, None, None, None, None, None, out])
    with pytest.raises(wgx.WgxError, match="expected 15 args"):
        ctx.recordShader(wgx.shaders.beamSearchStep, [q])
    with pytest.raises(wgx.WgxError, match="expected 13 args"):
        ctx.recordShader(wgx.shaders.cacheEvict, [q])
    with pytest.raises(wgx.WgxError, match="k shape"):
        ctx.recordShader(wgx.shaders.kvAppend, [q, q, table, ln, None, None, None, kc, vc, None, ln])
    assert ctx.stats()["commands"] == 0


def test_sync_reports_a_bad_page(ctx):
    kc, vc = T(ctx, np.zeros((2, 1, 16, 64), np.float16)), T(ctx, np.zeros((2, 1, 16, 64), np.float16))
    q, out = T(ctx, np.zeros((1, 1, 64), np.float16)), ctx.tensor("float16", [1, 1, 64])
    ctx.recordShader(wgx.shaders.pagedAttention, [q, kc, vc, T(ctx, np.array([[9]], np.int32)),
                                                 T(ctx, np.array([5], np.int32)), None, None, None, None, None, out])
    ctx.submit()
    with pytest.raises(wgx.WgxError, match="page id or length") as e:
        ctx.sync()
    assert e.value.code == _lib.WGX_ERR_DEVICE
    ctx.sync()  # cleared: the context stays usable
    assert (out.numpy() == 0).all()
