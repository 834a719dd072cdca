"""Measured cases of the text-decoding operators: kv_append, paged_attention,
cache_evict and beam_search_step (wgx.decode).

``run`` computes an operator either in its plain form (elementary torch
operations in 32 bits, rounded once at the end) or, where ``own`` is true,
through the calls a user makes. ``exact`` restates the formulas in 64 bits.

Conventions: a paged cache holds K and V as [pages, kv_heads, page_size,
head_dim]; slot s of sequence b lies in page page_table[b][s // page_size], row
s % page_size; lengths[b] slots are in use.
"""
import functools
import math
import os
import sys

import torch

own = False

HALF, SINGLE = "float16", "float32"


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one sequence's new token: the call between every two layers, latency only
        append("append_token_b1", B=1, T=1, Hkv=8, D=128, page=16, lo=700, hi=700),
        # prompts of eight sequences written at once
        append("append_prompt_b8", B=8, T=2048, Hkv=8, D=128, page=16, lo=0, hi=37),
        # the first words of one short answer: latency only
        attend("attend_b1_short", B=1, Hq=8, Hkv=8, D=64, page=16, lo=77, hi=77),
        # one long document: few rows, so the cache's length has to be split
        attend("attend_b1_long", B=1, Hq=32, Hkv=8, D=128, page=64, lo=131071, hi=131071),
        # a serving batch of ragged lengths whose weights feed the eviction
        attend("attend_b64_weights", B=64, Hq=32, Hkv=8, D=128, page=16, lo=17, hi=8192, weights=True),
        # single precision, a head size that is no power of two, left-padded
        # prompts and one sequence whose mask leaves nothing; slot-major pages
        attend("attend_fp32_masked", B=12, Hq=10, Hkv=5, D=80, page=24, lo=129, hi=2001, dtype=SINGLE,
               pad=53, order="slot"),
        # one KV head for sixteen query heads, wide heads, a sliding window
        attend("attend_window_g16", B=48, Hq=16, Hkv=1, D=256, page=32, lo=1000, hi=30000, window=4096),
        # generation under a fixed budget: a few slots go every few steps
        evict("evict_step_b16", B=16, Hkv=8, D=128, page=16, lo=1040, hi=1056, budget=1024, recent=128, sinks=4),
        # after long prompts: most of the cache goes
        evict("evict_prompt_b8", B=8, Hkv=8, D=128, page=16, lo=9000, hi=16384, budget=2048, recent=256, sinks=4),
        # greedy choice (one beam) over an odd vocabulary; the cache stays where it is
        beam("greedy_b32", B=32, W=1, V=50257, layers=0),
        # one sentence with four beams: latency, and a few tail pages
        beam("beam_b1_w4", B=1, W=4, V=32000, layers=4, Hkv=8, D=64, page=16, length=123),
        # a batch of eight-beam searches over a large vocabulary and a deep model
        beam("beam_b16_w8", B=16, W=8, V=131072, layers=24, Hkv=8, D=128, page=16, length=265, dtype=SINGLE),
    ]


def append(name, B, T, Hkv, D, page, lo, hi, dtype=HALF, order="head"):
    return {"op": "append", "name": name, "B": B, "T": T, "Hkv": Hkv, "D": D, "page": page, "lo": lo, "hi": hi,
            "dtype": dtype, "order": order}


def attend(name, B, Hq, Hkv, D, page, lo, hi, dtype=HALF, order="head", window=0, pad=0, weights=False):
    return {"op": "attend", "name": name, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "lo": lo, "hi": hi,
            "dtype": dtype, "order": order, "window": window, "pad": pad, "weights": weights}


def evict(name, B, Hkv, D, page, lo, hi, budget, recent, sinks, dtype=HALF, order="head"):
    return {"op": "evict", "name": name, "B": B, "Hkv": Hkv, "D": D, "page": page, "lo": lo, "hi": hi,
            "budget": budget, "recent": recent, "sinks": sinks, "dtype": dtype, "order": order}


def beam(name, B, W, V, layers, Hkv=1, D=8, page=8, length=0, dtype=HALF, cache_dtype=HALF):
    return {"op": "beam", "name": name, "B": B, "W": W, "V": V, "layers": layers, "Hkv": Hkv, "D": D, "page": page,
            "length": length, "dtype": dtype, "cache_dtype": cache_dtype}


def draw(rng):
    """One more case of the same ranges (log-uniform sizes, odd ones too)."""
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(("append", "attend", "attend", "attend", "evict", "evict", "beam", "beam"))
    dtype = rng.choice((HALF, HALF, HALF, SINGLE))
    order = rng.choice(("head", "slot"))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128))
    D = rng.choice((64, 64, 80, 96, 128, 128, 128, 192, 256))
    if op == "append":
        B, Hkv, T = size(1, 64), size(1, 16), rng.choice((1, 1, size(2, 2048)))
        T = max(1, min(T, (1 << 25) // (B * Hkv * D)))
        lo = size(1, 4000) - 1
        c = append("", B, T, Hkv, D, page, lo, lo + size(1, 500), dtype, order)
    elif op == "attend":
        B, Hkv, group = size(1, 128), size(1, 16), rng.choice((1, 2, 3, 4, 6, 8, 16))
        hi = size(1, 131072)
        most = (1 << 29) // (B * Hkv * D * (4 if dtype == SINGLE else 2))  # at most the largest listed cache
        hi = max(1, min(hi, most))
        lo = rng.choice((hi, hi // 2, 0))
        window = rng.choice((0, 0, 0, size(1, hi)))
        pad = rng.choice((0, 0, size(1, max(1, lo))))
        c = attend("", B, group * Hkv, Hkv, D, page, lo, hi, dtype, order, window, pad, rng.random() < 0.4)
    elif op == "evict":
        B, Hkv = size(1, 32), size(1, 16)
        hi = max(16, min(size(64, 32768), (1 << 27) // (B * Hkv * D)))
        budget = max(4, min(hi - 1, int(hi * rng.uniform(0.1, 0.98))))
        sinks = rng.choice((0, min(4, budget // 2)))
        c = evict("", B, Hkv, D, page, max(1, int(hi * rng.uniform(0.3, 1.0))), hi, budget,
                  rng.randrange(0, budget - sinks + 1), sinks, dtype, order)
    else:
        W = rng.choice((1, 2, 3, 4, 5, 8, 10, 16))
        V = size(1000, 200000) | 1
        B = max(1, min(size(1, 32), (1 << 24) // (W * V)))
        Hkv, length = size(1, 8), size(1, 600)
        layer = B * W * (length // 2 + 2 * page) * Hkv * D * 4  # bytes of one layer's cache
        layers = min(rng.choice((0, 1, size(2, 24))), (1 << 29) // layer)
        c = beam("", B, W, V, layers, Hkv, D, page, length, dtype, rng.choice((HALF, HALF, SINGLE)))
    del c["name"]
    return c


# -------------------------------------------------------------------- inputs
def lengths_of(case):
    """The sequences' lengths, spread evenly from lo to hi in a mixed order:
    the same for every seed, so that the work is known."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [lo + ((hi - lo) * ((b * 7 + 3) % B)) // max(1, B - 1) if B > 1 else hi for b in range(B)]


def pads_of(case):
    """Slots at the front of each sequence that its mask leaves out; the second
    sequence's mask leaves nothing."""
    L = lengths_of(case)
    return [L[b] if b == 1 else min(L[b] - 1, (case["pad"] * b) % (case["pad"] + 7)) for b in range(case["B"])]


def span_of(case):
    """Live slots of each sequence."""
    L = lengths_of(case)
    W = case["window"]
    first = [max(0, n - W) if W else 0 for n in L]
    if case["pad"]:
        first = [max(f, p) for f, p in zip(first, pads_of(case))]
    return [n - f for n, f in zip(L, first)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = getattr(torch, case["dtype"])
    return globals()["prepare_" + case["op"]](case, g, dt)


def paged(case, g, dt, capacities, layers=0):
    """K and V pools of randomly scattered pages, and their page table."""
    B, Hkv, D, page = case["B"], case["Hkv"], case["D"], case["page"]
    counts = [-(-n // page) for n in capacities]
    total, width = sum(counts) + 1, max(1, max(counts))
    lead = (layers,) if layers else ()
    if case.get("order") == "slot":
        pools = [torch.randn(lead + (total, page, Hkv, D), generator=g, device="cuda", dtype=dt).transpose(-3, -2)
                 for _ in range(2)]
    else:
        pools = [torch.randn(lead + (total, Hkv, page, D), generator=g, device="cuda", dtype=dt) for _ in range(2)]
    ids = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32)
    table = torch.zeros(B, width, device="cuda", dtype=torch.int32)
    filled = torch.arange(width, device="cuda")[None, :] < ints(counts)[:, None]
    table[filled] = ids[: sum(counts)]
    return pools[0], pools[1], table


def ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def prepare_append(case, g, dt):
    B, T = case["B"], case["T"]
    L = lengths_of(case)
    k_cache, v_cache, table = paged(case, g, dt, [n + T for n in L])
    k, v = (torch.randn(B, T, case["Hkv"], case["D"], generator=g, device="cuda", dtype=dt) for _ in range(2))
    return {"op": "append", "k": k, "v": v, "k_cache": k_cache, "v_cache": v_cache, "table": table,
            "lengths": ints(L), "lengths_out": torch.empty(B, device="cuda", dtype=torch.int32)}


def prepare_attend(case, g, dt):
    B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
    L = lengths_of(case)
    k_cache, v_cache, table = paged(case, g, dt, L)
    slots = table.shape[1] * case["page"]
    s = {"op": "attend", "k_cache": k_cache, "v_cache": v_cache, "table": table, "lengths": ints(L),
         "q": torch.randn(B, Hq, D, generator=g, device="cuda", dtype=dt), "window": case["window"],
         "scale": 1.0 / math.sqrt(D), "out": torch.empty(B, Hq, D, device="cuda", dtype=dt),
         "mask": None, "weights": None, "weights_out": None}
    if case["pad"]:
        s["mask"] = torch.arange(slots, device="cuda")[None, :] >= ints(pads_of(case))[:, None]
    if case["weights"]:
        # sums of earlier steps' probabilities
        s["weights"] = torch.rand(B, Hkv, slots, generator=g, device="cuda").square() * 3
        s["weights_out"] = torch.zeros(B, Hkv, slots, device="cuda")
    return s


def prepare_evict(case, g, dt):
    B, Hkv = case["B"], case["Hkv"]
    L = lengths_of(case)
    k_cache, v_cache, table = paged(case, g, dt, L)
    slots = table.shape[1] * case["page"]
    weights = torch.rand(B, Hkv, slots, generator=g, device="cuda").pow(4) * 5
    # tokens seen so far: an eighth of them went in earlier evictions, another
    # set for each head; survivors stand in a mixed order
    seen = [n + n // 8 for n in L]
    key = torch.rand(B, Hkv, max(seen), generator=g, device="cuda")
    key.masked_fill_(torch.arange(max(seen), device="cuda") >= ints(seen)[:, None, None], 2.0)
    order = key.argsort(dim=-1).to(torch.int32)
    positions = torch.full((B, Hkv, slots), -1, device="cuda", dtype=torch.int32)
    n = min(slots, max(seen))
    positions[..., :n] = order[..., :n]
    return {"op": "evict", "k_cache": k_cache, "v_cache": v_cache, "table": table, "lengths": ints(L),
            "weights": weights, "positions": positions, "seen": ints(seen), "budget": case["budget"],
            "recent": case["recent"], "sinks": case["sinks"], "lengths_out": torch.empty_like(ints(L)),
            "weights_out": torch.zeros_like(weights), "positions_out": torch.full_like(positions, -1)}


def prepare_beam(case, g, dt):
    B, W, V, layers, cache_dt = case["B"], case["W"], case["V"], case["layers"], getattr(torch, case["cache_dtype"])
    # a peaked distribution over a broad one
    logits = torch.randn(B, W, V, generator=g, device="cuda") * 2
    logits += torch.randn(B, W, V, generator=g, device="cuda").pow(3).clamp(-6, 6)
    scores = -torch.rand(B, W, generator=g, device="cuda") * 3 - 8
    finished = torch.rand(B, W, generator=g, device="cuda") < 0.1
    s = {"op": "beam", "logits": logits.to(dt), "scores": scores.sort(dim=-1, descending=True).values,
         "finished": finished, "eos": 2, "k_cache": None,
         "scores_out": torch.empty(B, W, device="cuda"),
         "parents": torch.empty(B, W, device="cuda", dtype=torch.int32),
         "tokens": torch.empty(B, W, device="cuda", dtype=torch.int32),
         "finished_out": torch.empty(B, W, device="cuda", dtype=torch.bool)}
    if layers:
        # the beams of a sequence share the pages of its prompt (half of the
        # length); each has pages of its own for the rest, and a spare one
        page, n = case["page"], case["length"]
        width = -(-n // page)
        shared = n // 2 // page
        total = B * shared + B * W * (width - shared) + B * W
        shape = (layers, total, case["Hkv"], page, case["D"])
        s["k_cache"], s["v_cache"] = (torch.randn(shape, generator=g, device="cuda", dtype=cache_dt) for _ in range(2))
        ids = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32)
        a, b = B * shared, B * shared + B * W * (width - shared)
        s["table"] = torch.cat([ids[:a].view(B, 1, shared).expand(B, W, shared),
                                ids[a:b].view(B, W, width - shared)], dim=2).reshape(B * W, width).contiguous()
        s["spare"] = ids[b:].clone()
        s["lengths"] = ints([n] * (B * W))
        s["table_out"] = torch.empty_like(s["table"])
        s["lengths_out"] = torch.empty_like(s["lengths"])
    return s


# ----------------------------------------------------------------- operators
def run(state):
    return globals()[("own_" if own else "plain_") + state["op"]](state)


@functools.lru_cache(None)
def decode():
    """wgx.decode: the package's folder is no valid module name, so it is put
    on the path as the repository's own programs do."""
    path = os.path.join(os.getcwd(), "wgpu-executorch_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import wgx.decode
    return wgx.decode


def own_append(s):
    decode().kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["lengths_out"])
    return [s["k_cache"], s["v_cache"], s["lengths_out"]]


def own_attend(s):
    decode().paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["out"],
                             scale=s["scale"], window=s["window"], mask=s["mask"], weights=s["weights"],
                             weights_out=s["weights_out"])
    return [s["out"], s["weights_out"]]


def own_evict(s):
    decode().cache_evict(s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["lengths_out"], s["weights"],
                         s["weights_out"], s["positions"], s["positions_out"], s["seen"], budget=s["budget"],
                         recent=s["recent"], sinks=s["sinks"])
    return [s["k_cache"], s["v_cache"], s["lengths_out"], s["weights_out"], s["positions_out"]]


def own_beam(s):
    cache = {}
    if s["k_cache"] is not None:
        cache = {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "page_table": s["table"],
                 "lengths": s["lengths"], "spare": s["spare"], "page_table_out": s["table_out"],
                 "lengths_out": s["lengths_out"]}
    decode().beam_search_step(s["logits"], s["scores"], s["finished"], s["scores_out"], s["parents"], s["tokens"],
                              s["finished_out"], eos=s["eos"], **cache)
    return beam_outputs(s)


def beam_outputs(s):
    out = [s["scores_out"], s["parents"], s["tokens"], s["finished_out"]]
    return out + [s["table_out"], s["lengths_out"], s["k_cache"], s["v_cache"]] if s["k_cache"] is not None else out


def slot_rows(table, slots, page):
    """(page id, row) of each slot: table [..., width], slots [..., n]."""
    return table.gather(-1, (slots // page).to(torch.int64)).to(torch.int64), (slots % page).to(torch.int64)


def plain_append(s):
    T, page = s["k"].shape[1], s["k_cache"].shape[-2]
    slots = s["lengths"][:, None] + torch.arange(T, device="cuda")
    ids, rows = slot_rows(s["table"], slots, page)
    s["k_cache"][ids, :, rows] = s["k"]
    s["v_cache"][ids, :, rows] = s["v"]
    torch.add(s["lengths"], T, out=s["lengths_out"])
    return [s["k_cache"], s["v_cache"], s["lengths_out"]]


def gathered(cache, table):
    """[B, kv_heads, slots, head_dim] in 32 bits."""
    x = cache[table.to(torch.int64)]  # [B, width, kv_heads, page, D]
    B, width, Hkv, page, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, width * page, D).float()


def live_slots(s, n):
    at, L = torch.arange(n, device="cuda"), s["lengths"][:, None]
    live = at < L
    if s["window"]:
        live &= at >= L - s["window"]
    if s["mask"] is not None:
        live &= s["mask"]
    return live


def plain_attend(s):
    B, Hq, D = s["q"].shape
    K = gathered(s["k_cache"], s["table"])
    Hkv, n = K.shape[1], K.shape[2]
    live = live_slots(s, n)[:, None, None, :]
    score = s["q"].float().view(B, Hkv, Hq // Hkv, D) @ K.transpose(2, 3) * s["scale"]
    del K
    score = score.masked_fill(~live, -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(dim=-1, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    V = gathered(s["v_cache"], s["table"]).masked_fill_(~live_slots(s, n)[:, None, :, None], 0.0)
    s["out"].copy_((p @ V).view(B, Hq, D))
    if s["weights"] is not None:
        used = torch.arange(n, device="cuda") < s["lengths"][:, None, None]
        s["weights_out"].copy_(torch.where(used, s["weights"] + p.sum(dim=2), s["weights_out"]))
    return [s["out"], s["weights_out"]]


def plain_evict(s):
    B, Hkv, n = s["weights"].shape
    page, C, L = s["k_cache"].shape[-2], s["budget"], s["lengths"][:, None, None]
    at = torch.arange(n, device="cuda").expand(B, Hkv, n)
    used = at < L
    kept_all = L <= C
    safe = (s["positions"] >= (s["seen"] - s["recent"])[:, None, None]) | (s["positions"] < s["sinks"])
    w = torch.where(s["weights"].isnan(), -math.inf, s["weights"])
    w = torch.where(safe, math.inf, w)
    order = w.masked_fill(~used, -math.inf).argsort(dim=-1, descending=True, stable=True)
    # the slots' places in the order; used slots before unused ones, protected before others
    group = (~used).to(torch.int8) * 2 + (~safe).to(torch.int8)
    order = order.gather(-1, group.gather(-1, order).argsort(dim=-1, stable=True))
    rank = torch.empty_like(order).scatter_(-1, order, at)
    keep = used & ((rank < C) | kept_all)
    hole = used & ~keep & (at < C)
    mover = keep & (at >= C) & ~kept_all
    # holes and movers, in slot order, side by side
    m = int(max(1, min(C, n - C)))
    holes = torch.argsort((~hole).to(torch.int8), dim=-1, stable=True)[..., :m]
    movers = torch.argsort((~mover).to(torch.int8), dim=-1, stable=True)[..., :m]
    valid = torch.arange(m, device="cuda") < mover.sum(dim=-1, keepdim=True)
    b, h, j = valid.nonzero(as_tuple=True)
    dst, src = holes[b, h, j], movers[b, h, j]
    table = s["table"].to(torch.int64)
    to, fro = table[b, dst // page], table[b, src // page]
    s["k_cache"][to, h, dst % page] = s["k_cache"][fro, h, src % page]
    s["v_cache"][to, h, dst % page] = s["v_cache"][fro, h, src % page]
    stays = keep & ((at < C) | kept_all)
    s["weights_out"].copy_(torch.where(stays, s["weights"], s["weights_out"]))
    s["positions_out"].copy_(torch.where(stays, s["positions"], s["positions_out"]))
    s["weights_out"][b, h, dst] = s["weights"][b, h, src]
    s["positions_out"][b, h, dst] = s["positions"][b, h, src]
    torch.clamp(s["lengths"], max=C, out=s["lengths_out"])
    return [s["k_cache"], s["v_cache"], s["lengths_out"], s["weights_out"], s["positions_out"]]


def plain_beam(s):
    B, W, V = s["logits"].shape
    x = s["logits"].float()
    top = x.amax(dim=-1, keepdim=True)
    log_sum = torch.log(torch.exp(x - top).sum(dim=-1, keepdim=True))
    k = min(W, V)
    # equal logits: the lower token first (a stable sort)
    best, token = x.sort(dim=-1, descending=True, stable=True)
    best, token = best[..., :k], token[..., :k]
    total = s["scores"][..., None] + ((best - top) - log_sum)
    done, first = s["finished"][..., None], torch.arange(k, device="cuda") == 0
    total = torch.where(done, torch.where(first, s["scores"][..., None], -math.inf), total)
    token = torch.where(done, s["eos"], token)
    total, at = total.reshape(B, W * k).sort(dim=-1, descending=True, stable=True)
    at = at[:, :W]
    s["scores_out"].copy_(total[:, :W])
    parent = at // k
    s["parents"].copy_(parent)
    s["tokens"].copy_(token.reshape(B, W * k).gather(-1, at))
    s["finished_out"].copy_(s["finished"].gather(-1, parent) | (s["tokens"] == s["eos"]))
    if s["k_cache"] is not None:
        page = s["k_cache"].shape[-2]
        source = (torch.arange(B, device="cuda")[:, None] * W + parent).reshape(-1)
        length = s["lengths"][source]
        full, tail = (length // page).to(torch.int64), length % page
        width = s["table"].shape[1]
        copied = (torch.arange(width, device="cuda") == full[:, None]) & (tail > 0)[:, None]
        s["table_out"].copy_(torch.where(copied, s["spare"][:, None], s["table"][source]))
        s["lengths_out"].copy_(length)
        old = s["table"][source, full.clamp(max=width - 1)].to(torch.int64)
        new = s["spare"].to(torch.int64)
        row = (torch.arange(page, device="cuda")[None, :] < tail[:, None])[None, :, None, :, None]
        s["k_cache"][:, new] = torch.where(row, s["k_cache"][:, old], s["k_cache"][:, new])
        s["v_cache"][:, new] = torch.where(row, s["v_cache"][:, old], s["v_cache"][:, new])
    return beam_outputs(s)


# ---------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == SINGLE else 2
    if case["op"] == "append":
        rows = case["B"] * case["T"] * case["Hkv"] * 2
        return {"bytes": 2 * rows * case["D"] * e + 12 * case["B"], "flops": 0}
    if case["op"] == "attend":
        live = sum(span_of(case))
        row = case["D"] * e
        moved = live * case["Hkv"] * 2 * row + 2 * case["B"] * case["Hq"] * row
        if case["weights"]:
            moved += 8 * case["Hkv"] * sum(lengths_of(case))
        return {"bytes": moved, "flops": 4 * live * case["Hq"] * case["D"]}
    if case["op"] == "evict":
        C, moved = case["budget"], 0
        for n in lengths_of(case):
            kept = min(n, C)
            # weights and positions in and out; of C survivors of n slots about
            # C (n - C) / n stand behind the budget and move
            moved += case["Hkv"] * (8 * n + 8 * kept)
            if n > C:
                moved += case["Hkv"] * 4 * case["D"] * e * (C * (n - C) // n)
        return {"bytes": moved, "flops": 0}
    rows = case["B"] * case["W"]
    moved = rows * case["V"] * e + rows * 22
    if case["layers"]:
        tail = case["length"] % case["page"]
        moved += rows * (8 * -(-case["length"] // case["page"]) + 12)
        moved += rows * case["layers"] * case["Hkv"] * 4 * tail * case["D"] * (4 if case["cache_dtype"] == SINGLE else 2)
    return {"bytes": moved, "flops": 4 * rows * case["V"]}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """The computed outputs in 64 bits: attention's result and weights, the
    beams' scores. Appending and evicting only move values."""
    if case["op"] == "attend":
        return exact_attend(case, prepare(case, seed))
    if case["op"] == "beam":
        return exact_beam(prepare(case, seed))
    return None


def exact_attend(case, s):
    B, Hq, D = s["q"].shape
    Hkv, page = s["k_cache"].shape[1], s["k_cache"].shape[2]
    out = torch.zeros(B, Hq, D, device="cuda", dtype=torch.float64)
    weights = s["weights_out"].double() if s["weights"] is not None else None
    pads = pads_of(case) if case["pad"] else [0] * B
    for b, n in enumerate(lengths_of(case)):
        first = max(pads[b], n - s["window"] if s["window"] else 0, 0)
        if weights is not None:
            weights[b, :, :n] = s["weights"][b, :, :n].double()
        if first >= n:
            continue
        at = torch.arange(first, n, device="cuda")
        ids = s["table"][b].long()[at // page]
        for h in range(Hkv):
            k = s["k_cache"][ids, h, at % page].double()
            v = s["v_cache"][ids, h, at % page].double()
            heads = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            p = torch.softmax(torch.einsum("gd,nd->gn", s["q"][b, heads].double(), k) * s["scale"], dim=-1)
            out[b, heads] = torch.einsum("gn,nd->gd", p, v)
            if weights is not None:
                weights[b, h, first:n] += p.sum(dim=0)
    return [out, weights]


def exact_beam(s):
    x = s["logits"].double()
    total = s["scores"].double()[..., None] + torch.log_softmax(x, dim=-1)
    total[s["finished"]] = -math.inf
    best = torch.cat([total.flatten(1), s["scores"].double().masked_fill(~s["finished"], -math.inf)], dim=1)
    out = [best.topk(s["scores"].shape[1], dim=1).values, None, None, None]
    return out + [None] * 4 if s["k_cache"] is not None else out
