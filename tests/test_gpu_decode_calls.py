"""What the decoding operators' calls say beside their results: the launch counts
of recorded commands."""
import numpy as np
import pytest

import wgx
from test_gpu_decode import F16, T, Cache

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
