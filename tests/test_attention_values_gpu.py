"""mxs_prefix_attention where values are infinite or NaN at positions that are
seen: a value counts times its weight, so one of weight 0 that is infinite gives
NaN, whether the position is seen by all of a call's tokens or by the later ones
only."""
import math

import pytest

from test_attention_gpu import inputs, run, sampler, say, torch_mod  # noqa: F401

pytestmark = pytest.mark.gpu

SHAPES = [(1, 2, 1, 4, 2, 64, 50, 30), (1, 2, 5, 4, 2, 64, 50, 30), (1, 1, 6, 4, 1, 80, 30, 90), (2, 1, 33, 2, 2, 128, 9, 40),
          (1, 2, 20, 8, 2, 128, 20, 200), (1, 2, 5, 6, 1, 256, 40, 37), (1, 1, 24, 16, 2, 136, 0, 70)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("scale", [None, -0.2])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_no_numbers(torch_mod, sampler, shape, scale, bad):  # noqa: F811
    torch = torch_mod
    say(f"values {shape} {scale} {bad}")
    x = inputs(torch, *shape, seed=21)
    R, N, D, KV = shape[0] * shape[1], shape[7], shape[5], shape[4]
    x["q"][..., 1] = 1.5
    no = -math.inf if scale is None else math.inf   # (a score of -inf)
    v, k = x["values"], x["keys"]
    for j in (N - 1, N - 3, N - shape[2], 2):       # seen by the last token, by the later ones, by all
        k[0, 0, j, 1] = no
        v[0, 0, j, j % D] = bad                     # weight 0
    v[R - 1, KV - 1, N - 2, 5] = bad                # weight above 0
    v[R - 1, KV - 1, N - 3, 7], v[R - 1, KV - 1, N - 2, 7] = math.inf, -math.inf
    v[R - 1, KV - 1, N - 4, D - 1] = bad
    got = run(torch, sampler, x, weights=True, **({} if scale is None else dict(scale=scale)))
    assert bool(got["out"][0, -1, 0, (N - 1) % D].isnan())
