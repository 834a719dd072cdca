"""The example decoder (examples/generate.py): the decoding operators together,
against a plain 64-bit decoder that recomputes every sequence from its start.

The scores are sums of up to 40 log probabilities of a three-layer fp32 model:
activations of size about one with relative errors of 1e-6 a layer, so 1e-3 in
all is far outside what rounding can do and far below a wrong token's effect."""
import importlib.util
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "generate.py")


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("generate_example", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


class Plain:
    """The same model in numpy, 64 bits, without a cache."""

    def __init__(self, m):
        f = lambda t: t.double().cpu().numpy()  # noqa: E731
        self.m, self.embed, self.place, self.out = m, f(m.embed), f(m.place), f(m.out)
        self.blocks = [{k: f(v) for k, v in b.items()} for b in m.blocks]

    @staticmethod
    def norm(x):
        return x / np.sqrt((x ** 2).mean(axis=-1, keepdims=True) + 1e-6)

    def log_probs(self, tokens):
        """Of the token after `tokens`."""
        m, n = self.m, len(tokens)
        x = self.embed[tokens] + self.place[:n]
        mask = np.tril(np.ones((n, n), bool))
        for w in self.blocks:
            y = self.norm(x)
            q = (y @ w["q"]).reshape(n, m.heads, m.head_dim)
            k, v = ((y @ w[s]).reshape(n, m.kv_heads, m.head_dim) for s in "kv")
            att = np.empty_like(q)
            for h in range(m.heads):
                g = h // (m.heads // m.kv_heads)
                s = np.where(mask, q[:, h] @ k[:, g].T * m.head_dim ** -0.5, -np.inf)
                p = np.exp(s - s.max(axis=1, keepdims=True))
                att[:, h] = p / p.sum(axis=1, keepdims=True) @ v[:, g]
            x = x + att.reshape(n, -1) @ w["o"]
            x = x + np.maximum(self.norm(x) @ w["up"], 0) @ w["down"]
        z = self.norm(x[-1]) @ self.out
        return z - (z.max() + np.log(np.exp(z - z.max()).sum()))

    def beam_search(self, start, beams, steps, eos):
        live = [(0.0, [start], False)]
        for _ in range(steps):
            props = []
            for w, (score, seq, done) in enumerate(live):
                if done:
                    props.append((score, w, eos))
                else:
                    lp = self.log_probs(seq)
                    props += [(score + lp[t], w, int(t)) for t in np.argsort(-lp)[:beams]]
            props.sort(key=lambda p: -p[0])
            live = [(s, live[w][1] + [t], live[w][2] or t == eos) for s, w, t in props[:beams]]
        return live


@pytest.mark.parametrize("beams", [1, 3])
def test_beam_search_matches_a_plain_decoder(ex, beams):
    steps = 37  # over two page boundaries
    model = ex.Decoder(vocab=211, width=64, layers=3, heads=4, kv_heads=2, head_dim=32, dtype=torch.float32, seed=3)
    tokens, scores = ex.generate(model, [5, 17], beams, steps)
    plain = Plain(model)
    for b, start in enumerate([5, 17]):
        want = plain.beam_search(start, beams, steps, ex.EOS)
        for w, (score, seq, _) in enumerate(want):
            assert tokens[b, w].tolist() == seq[1:]
            assert abs(float(scores[b, w]) - score) <= 1e-3
    assert ex.decode.device_error(0) == 0


def test_a_budget_that_is_not_reached_changes_nothing(ex):
    model = ex.Decoder(vocab=211, width=64, heads=4, kv_heads=2, head_dim=32, dtype=torch.float32, seed=4)
    free = ex.generate(model, [1, 2, 3], 1, 40)
    held = ex.generate(model, [1, 2, 3], 1, 40, budget=64)
    assert torch.equal(free[0], held[0]) and torch.allclose(free[1], held[1], atol=1e-3)


def test_generation_with_an_evicting_cache(ex, monkeypatch):
    """The cache stays within its budget and slack, keeps the first and the
    most recent tokens, and the text goes on."""
    model = ex.Decoder(vocab=211, width=64, heads=4, kv_heads=2, head_dim=32, dtype=torch.float16, seed=5)
    seen = []
    shrink = ex.shrink

    def spy(m, cache, budget, recent):
        assert int(cache.lengths.max()) == budget + budget // 16
        shrink(m, cache, budget, recent)
        assert (cache.lengths == budget).all()
        last = int(cache.seen[0])
        for kept in cache.positions[..., :budget].reshape(-1, budget).tolist():
            assert {0, 1} <= set(kept) and set(range(last - recent, last)) <= set(kept)
            assert len(set(kept)) == budget
        seen.append(last)
    monkeypatch.setattr(ex, "shrink", spy)
    tokens, scores = ex.generate(model, [1, 2], 1, 150, budget=32)
    assert tokens.shape == (2, 1, 150) and torch.isfinite(scores).all() and len(seen) >= 50
    assert ex.decode.device_error(0) == 0
