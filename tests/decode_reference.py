"""Plain statements of the text-decoding operators (include/wgx.h) in numpy,
64-bit, slot by slot: what the GPU tests compare with."""
import numpy as np


def slot_row(cache, table, b, h, s):
    """View of the cache row of slot s ([pages, kv_heads, page_size, D])."""
    size = cache.shape[2]
    return cache[table[b, s // size], h, s % size]


def gather(cache, table, b, h, n):
    size = cache.shape[2]
    s = np.arange(n)
    return cache[table[b, s // size], h, s % size]


def paged_attention(q, k_cache, v_cache, table, lengths, scale, window=0, mask=None, weights=None):
    """(out, weights_out) in float64."""
    B, Hq, D = q.shape
    H = k_cache.shape[1]
    G = Hq // H
    out = np.zeros((B, Hq, D))
    wout = None if weights is None else weights.astype(np.float64)
    for b in range(B):
        n = int(lengths[b])
        live = np.ones(n, bool)
        if window:
            live[:max(0, n - window)] = False
        if mask is not None:
            m = np.zeros(n, bool)
            w = min(n, mask.shape[1])
            m[:w] = mask[b, :w] != 0
            live &= m
        at = np.nonzero(live)[0]
        if at.size == 0:
            continue
        for h in range(H):
            k = gather(k_cache, table, b, h, n)[at].astype(np.float64)
            v = gather(v_cache, table, b, h, n)[at].astype(np.float64)
            s = q[b, h * G:(h + 1) * G].astype(np.float64) @ k.T * scale
            p = np.exp(s - s.max(axis=1, keepdims=True))
            p /= p.sum(axis=1, keepdims=True)
            out[b, h * G:(h + 1) * G] = p @ v
            if wout is not None:
                wout[b, h, at] += p.sum(axis=0)
    return out, wout


def evict_plan(weights, positions, n, seen, budget, recent, sinks):
    """One head: (slots that stay in place, [(destination, source)])."""
    w = weights[:n].astype(np.float64)
    w = np.where(np.isnan(w), -np.inf, w)
    nan = np.isnan(weights[:n])
    safe = (positions[:n] >= seen - recent) | (positions[:n] < sinks)
    # protected first, then by weight (NaN behind -infinity), then by slot
    order = sorted(range(n), key=lambda i: (not safe[i], nan[i] and not safe[i], 0.0 if safe[i] else -w[i], i))
    keep = np.zeros(n, bool)
    keep[order[:budget]] = True
    holes = [i for i in range(budget) if not keep[i]]
    movers = [i for i in range(budget, n) if keep[i]]
    assert len(holes) == len(movers)
    return [i for i in range(budget) if keep[i]], list(zip(holes, movers))


def cache_evict(k_cache, v_cache, table, lengths, weights, positions, seen, budget, recent, sinks):
    """Evicts in place; returns lengths_out."""
    B, H = weights.shape[:2]
    for b in range(B):
        n = int(lengths[b])
        if n <= budget:
            continue
        for h in range(H):
            _, moves = evict_plan(weights[b, h], positions[b, h], n, seen[b], budget, recent, sinks)
            for dst, src in moves:
                for c in (k_cache, v_cache):
                    slot_row(c, table, b, h, dst)[:] = slot_row(c, table, b, h, src)
                weights[b, h, dst] = weights[b, h, src]
                positions[b, h, dst] = positions[b, h, src]
    return np.minimum(lengths, budget).astype(np.int32)


def beam_search_step(logits, scores, finished, eos):
    """(scores, parents, tokens, finished) of the new beams."""
    B, W, V = logits.shape
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    so = np.zeros((B, W))
    pa = np.zeros((B, W), np.int32)
    to = np.zeros((B, W), np.int32)
    for b in range(B):
        props = []  # (-total, beam, -logit, token)
        for w in range(W):
            sc = float(scores[b, w])
            if finished[b, w]:
                props.append((-sc, w, 0.0, eos))
                continue
            with np.errstate(invalid="ignore", divide="ignore"):
                m = x[b, w].max()
                lse = m + np.log(np.exp(x[b, w] - m).sum()) if np.isfinite(m) else m
                best = np.argsort(-x[b, w], kind="stable")[:W]
                for t in best:
                    total = sc + (x[b, w, t] - lse)
                    total = -np.inf if np.isnan(total) else total
                    props.append((-total, w, -x[b, w, t], int(t)))
        props.sort()
        for r in range(W):
            so[b, r], pa[b, r], to[b, r] = -props[r][0], props[r][1], props[r][3]
    fo = np.take_along_axis(finished.astype(bool), pa.astype(np.int64), axis=1) | (to == eos)
    return so, pa, to, fo


def reorder(k_cache, v_cache, table, lengths, spare, parents, beams):
    """The children's page tables and lengths; copies tails in place
    ([layers, pages, kv_heads, page_size, D])."""
    n, size = table.shape[0], k_cache.shape[3]
    out, lout = table.copy(), lengths.copy()
    for c in range(n):
        p = c // beams * beams + int(parents.reshape(-1)[c])
        out[c] = table[p]
        lout[c] = lengths[p]
        full, tail = divmod(int(lengths[p]), size)
        if tail:
            old = table[p, full]
            out[c, full] = spare[c]
            for x in (k_cache, v_cache):
                x[:, spare[c], :, :tail] = x[:, old, :, :tail]
    return out, lout
