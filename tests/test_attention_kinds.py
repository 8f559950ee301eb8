"""Which kernels of mxs_prefix_attention the GPU tests launch, by its plan and
without a GPU: every kind that some size reaches, and long loops in each."""
import random

import pytest

from test_attention_gpu import RAGGED, SHAPES
from test_attention_plan import plan, verify  # noqa: F401
from test_attention_steady_gpu import KINDS, MANY_PARTS, STEADY

TILE = 64


def cut(a, b):
    return -(-a // b)


def kinds(p):
    return {("tile", p["dp"], p["rb"], p["wq"], bool(p["small"])), ("join", p["dp"], p["slots"] > 16)}


def test_every_reachable_kind_is_tested(plan):  # noqa: F811
    rng = random.Random(3)
    log = lambda hi: int(2 ** rng.uniform(0, hi))
    reachable = set()
    for _ in range(20000):
        KV = log(6)
        reachable |= kinds(verify(plan, log(6), log(6), log(rng.choice([0, 3, 7])), KV * log(rng.choice([0, 3, 6])), KV, 8 * rng.randint(1, 32),
                                  rng.choice([0, log(10), log(16)]), rng.choice([0, log(8), log(12)])))
    ran = set()
    for shape in SHAPES + [s for s, _, _ in RAGGED] + STEADY + MANY_PARTS + KINDS:
        ran |= kinds(verify(plan, *[v or 0 for v in shape]))
    assert not reachable - ran, reachable - ran


def test_blocks_of_sixteen_have_small_suffixes(plan):  # noqa: F811
    """A block of 16 queries holds all that share a prefix, so all that share a
    suffix: the kernel for larger suffixes is not compiled for it."""
    rng = random.Random(4)
    for _ in range(20000):
        p = verify(plan, rng.randint(1, 40), rng.randint(1, 20), rng.randint(1, 20), rng.choice([1, 2, 4, 16, 40]), 1,
                   8 * rng.randint(1, 32), rng.randint(0, 5000), rng.randint(0, 5000))
        assert p["small"] or (p["rb"], p["wq"]) != (1, 1)


@pytest.mark.parametrize("shape", STEADY, ids=str)
def test_steady_shapes_have_many_tiles_a_part(plan, shape):  # noqa: F811
    G, W, T, H, KV, D, P, N = shape
    p = verify(plan, *shape)
    assert (p["ng"], p["wb"], p["nt"]) == (G, W, T)
    assert cut(cut(P, TILE), p["sp"]) >= 6 and cut(cut(N, TILE), p["ss"]) >= 4
    tiles = max(1, min(64, (G * KV * cut(P, 32) + G * W * KV * cut(N, 32)) // 2048))   # (attention_launch)
    assert tiles >= 2
    assert P % (tiles * 32)   # (a last chunk that is not full)


def test_steady_shapes_take_every_block(plan):  # noqa: F811
    seen = {(p["dp"], p["rb"], p["wq"], bool(p["small"])) for p in (verify(plan, *s) for s in STEADY)}
    assert len(seen) == 21


@pytest.mark.parametrize("shape", MANY_PARTS, ids=str)
def test_many_parts(plan, shape):  # noqa: F811
    assert verify(plan, *shape)["slots"] > 3 * 64
