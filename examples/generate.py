"""Text generation with a small random decoder: the decoding operators
together, as a serving loop uses them.

    python examples/generate.py --beams 4 --steps 48        # beam search
    python examples/generate.py --budget 32 --steps 200     # greedy, evicting cache

Every step appends the new token's K and V rows (kv_append), attends over the
paged cache (paged_attention, which also accumulates each slot's attention
weight when the cache is bounded), shrinks the cache when it is over its budget
(cache_evict) and chooses the next tokens (beam_search_step, which reorders the
page tables). The projections are the engine's mm. Nothing in the loop waits for
the device. The weights are random: the text means nothing.
"""
import argparse
import ctypes
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wgpu-executorch_b200"))

from wgx import _lib  # noqa: E402
from wgx import decode  # noqa: E402

PAGE = 16
EOS = 0


class Decoder:
    """Embedding, `layers` blocks of attention and a two-layer ReLU network,
    each behind a norm and added to its input, and an output projection."""

    def __init__(self, vocab=1000, width=256, layers=3, heads=8, kv_heads=2, head_dim=64, positions=512,
                 dtype=torch.float16, seed=0):
        g = torch.Generator().manual_seed(seed)

        def matrix(rows, cols, gain=1.0):
            return (torch.randn(rows, cols, generator=g) * gain * rows ** -0.5).cuda().to(dtype)
        self.layers, self.heads, self.kv_heads, self.head_dim, self.dtype = layers, heads, kv_heads, head_dim, dtype
        self.embed = torch.randn(vocab, width, generator=g).cuda().to(dtype)
        self.place = torch.randn(positions, width, generator=g).cuda().to(dtype)
        self.blocks = [{"q": matrix(width, heads * head_dim), "k": matrix(width, kv_heads * head_dim),
                        "v": matrix(width, kv_heads * head_dim), "o": matrix(heads * head_dim, width),
                        "up": matrix(width, 2 * width), "down": matrix(2 * width, width)} for _ in range(layers)]
        self.out = matrix(width, vocab, 3.0)


def mm(a, b):
    """a @ b on the current stream by the engine's matrix product."""
    m, k = a.shape
    n = b.shape[1]
    code = 1 if a.dtype == torch.float16 else 0
    out = torch.empty(m, n, dtype=a.dtype, device="cuda")
    need = ctypes.c_uint64()
    _lib.check(_lib.lib.wgx_mm_scratch_bytes(m, n, k, code, ctypes.byref(need)))
    scratch = torch.empty(max(1, need.value), dtype=torch.uint8, device="cuda")
    _lib.check(_lib.lib.wgx_mm(a.data_ptr(), b.data_ptr(), out.data_ptr(), m, n, k, code, scratch.data_ptr(),
                               need.value, torch.cuda.current_stream().cuda_stream))
    return out


def norm(x):
    y = x.float()
    return (y * torch.rsqrt(y.square().mean(dim=-1, keepdim=True) + 1e-6)).to(x.dtype)


class Cache:
    """K and V of all layers in one pool of pages; page tables, lengths and the
    bookkeeping of evictions on the device. All sequences are equally long."""

    def __init__(self, model, sequences, slots, evict):
        n, width = sequences, -(-slots // PAGE)
        pages = n * (width + 1)
        shape = (model.layers, pages, model.kv_heads, PAGE, model.head_dim)
        self.k, self.v = (torch.empty(shape, dtype=model.dtype, device="cuda") for _ in range(2))
        ids = torch.arange(pages, dtype=torch.int32, device="cuda").view(n, width + 1)
        self.fresh = ids[:, :width]                  # page `c` of each sequence's own
        self.spare = ids[:, width].contiguous()      # where a child's last page is copied to
        self.table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
        self.table_out = torch.empty_like(self.table)
        self.lengths, self.next_lengths = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))
        self.columns, self.length = 0, 0             # page columns in use, slots in use (host)
        self.weights = self.positions = None
        if evict:
            self.weights = torch.zeros(model.layers, n, model.kv_heads, width * PAGE, device="cuda")
            self.positions = torch.zeros(model.layers, n, model.kv_heads, width * PAGE, dtype=torch.int32, device="cuda")
            self.seen, self.next_seen = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(2))

    def make_room(self):
        """A page for the next token where the last one is full."""
        if self.length == self.columns * PAGE:
            self.table[:, self.columns] = self.fresh[:, self.columns]
            self.columns += 1


def forward(model, cache, tokens, step):
    """Logits of the next token; the tokens' rows enter the cache."""
    n = tokens.shape[0]
    x = model.embed[tokens.long()] + model.place[step]
    cache.make_room()
    for i, w in enumerate(model.blocks):
        y = norm(x)
        q = mm(y, w["q"]).view(n, model.heads, model.head_dim)
        k, v = (mm(y, w[s]).view(n, 1, model.kv_heads, model.head_dim) for s in "kv")
        held = {} if cache.weights is None else {"weights": cache.weights[i], "positions": cache.positions[i],
                                                 "seen": cache.seen, "seen_out": cache.next_seen}
        decode.kv_append(k, v, cache.k[i], cache.v[i], cache.table, cache.lengths, cache.next_lengths, **held)
        weights = None if cache.weights is None else cache.weights[i]
        y = decode.paged_attention(q, cache.k[i], cache.v[i], cache.table, cache.next_lengths, weights=weights,
                                   weights_out=weights)
        x = x + mm(y.view(n, -1), w["o"])
        x = x + mm(torch.relu(mm(norm(x), w["up"])), w["down"])
    cache.lengths, cache.next_lengths = cache.next_lengths, cache.lengths
    if cache.weights is not None:
        cache.seen, cache.next_seen = cache.next_seen, cache.seen
    cache.length += 1
    return mm(norm(x), model.out)


def shrink(model, cache, budget, recent):
    """Back to `budget` slots in every layer and head."""
    for i in range(model.layers):
        w, p = cache.weights[i], cache.positions[i]
        decode.cache_evict(cache.k[i], cache.v[i], cache.table, cache.lengths, cache.next_lengths, w, w, p, p,
                           cache.seen, budget=budget, recent=recent, sinks=2)
    cache.lengths, cache.next_lengths = cache.next_lengths, cache.lengths
    cache.length = min(cache.length, budget)


def generate(model, start, beams=1, steps=32, budget=0):
    """The `beams` best continuations of each start token: (tokens [batch,
    beams, steps], scores [batch, beams]). budget > 0 (one beam only: beams
    share pages, and a shared page must not be evicted from): at most that many
    slots per head, a sixteenth more before the next eviction."""
    batch, n = len(start), len(start) * beams
    slack = max(1, budget // 16)
    if budget and (beams > 1 or budget < 8):
        raise ValueError("a budget is for one beam, and at least 8 slots")
    cache = Cache(model, n, min(steps, budget + slack) if budget else steps, budget > 0)
    tokens = torch.tensor(start, dtype=torch.int32, device="cuda").repeat_interleave(beams)
    # only the first beam counts at first: the others are copies of it
    scores = torch.full((batch, beams), -float("inf"), device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros(batch, beams, dtype=torch.bool, device="cuda")
    chosen, parents = [], []
    for step in range(steps):
        logits = forward(model, cache, tokens, step).view(batch, beams, -1)
        new_scores, done = torch.empty_like(scores), torch.empty_like(finished)
        new, parent = (torch.empty(batch, beams, dtype=torch.int32, device="cuda") for _ in range(2))
        state = {}
        if beams > 1:
            state = {"k_cache": cache.k, "v_cache": cache.v, "page_table": cache.table, "lengths": cache.lengths,
                     "spare": cache.spare, "page_table_out": cache.table_out, "lengths_out": cache.next_lengths}
        decode.beam_search_step(logits, scores, finished, new_scores, parent, new, done, eos=EOS, **state)
        if beams > 1:
            if cache.length % PAGE:
                # the last pages were copied: the old ones are free for the next step
                cache.spare = cache.table[:, cache.length // PAGE].contiguous()
            cache.table, cache.table_out = cache.table_out, cache.table
            cache.lengths, cache.next_lengths = cache.next_lengths, cache.lengths
        if budget and cache.length >= budget + slack:
            shrink(model, cache, budget, recent=budget // 2)
        scores, finished, tokens = new_scores, done, new.view(-1)
        chosen.append(new)
        parents.append(parent)
    # follow the parents back from the last step
    at = torch.arange(beams, device="cuda").expand(batch, beams)
    out = []
    for new, parent in zip(reversed(chosen), reversed(parents)):
        out.append(new.gather(1, at))
        at = parent.gather(1, at).long()
    return torch.stack(out[::-1], dim=-1), scores


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=2)
    ap.add_argument("--beams", type=int, default=1)
    ap.add_argument("--steps", type=int, default=48)
    ap.add_argument("--budget", type=int, default=0)
    a = ap.parse_args()
    tokens, scores = generate(Decoder(), list(range(1, a.batch + 1)), a.beams, a.steps, a.budget)
    for b in range(a.batch):
        for w in range(a.beams):
            print("%d.%d  %8.3f  %s" % (b, w, scores[b, w], " ".join(map(str, tokens[b, w].tolist()))))


if __name__ == "__main__":
    main()
