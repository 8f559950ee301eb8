"""mxs_prefix_attention with many tiles a part, where the tile loop, its ring of
tiles in LDS and the rescaling of sums that are not empty are in their steady
state; weights of several tiles a wave; joins of more parts than a wave has
lanes.  (test_attention_kinds.py holds that these shapes are split so.)

Tolerances are those that test_attention_gpu.py derives, but for the roundings of
an accumulated weight: the weights kernel adds 64 queries' weights at a time
(16 where there are no more, 32 where dim is above 128) to the entry in memory, so
that the entry of a cache head with m queries is rounded ceil(m / 64) (or
ceil(m / 32)) times, each by half a step, 2^-24 of a sum that is at most the last."""
import pytest

from test_attention_gpu import inputs, near, oracle, sampler, say, torch_mod  # noqa: F401

pytestmark = pytest.mark.gpu

# beams, tokens, query heads a cache head: of every block of queries, small suffixes and others
QUERIES = [(2, 1, 4), (5, 1, 4), (1, 6, 4), (6, 1, 8), (2, 5, 5), (9, 1, 8), (2, 6, 8)]


def shape_of(D, W, T, per):
    return (16 if D <= 128 else 8, W, T, 8 * per, 8, D, 1800 + W, 400 + T)


STEADY = [shape_of(D, *q) for D in (64, 80, 128, 256) for q in QUERIES] + [shape_of(40, 2, 6, 8), shape_of(136, 5, 1, 4)]
# more than 64 parts a query
MANY_PARTS = [(1, W, T, per, 1, D, 12900, 700) for D in (64, 128, 256) for W, T, per in ((1, 1, 1), (3, 1, 8), (1, 6, 8))]
# every kind of join and block that the shapes above and test_attention_gpu's leave out
KINDS = [(1, 1, 6, 8, 2, D, 1000, 60) for D in (64, 128, 256)] + [(1, 2, 1, 4, 1, 256, 1100, 30)]


def run(torch, s, x):
    """A call with everything, its outputs against the definition."""
    G, KV, P, D = x["prefix_keys"].shape
    R, T, H, _ = x["q"].shape
    g = torch.Generator(device="cuda").manual_seed(99)
    pw, w = (torch.rand(n, generator=g, device="cuda") for n in ((G, KV, P), (R, KV, x["keys"].shape[2])))
    pw0, w0, lse = pw.clone(), w.clone(), torch.full((R, T, H), 7.0, device="cuda")
    out = s.prefix_attention(x["q"], x["prefix_keys"], x["prefix_values"], x["keys"], x["values"], lse=lse, prefix_weight=pw,
                             weight=w)
    s.sync()
    o = oracle(torch, x)
    near(torch, out, o["out"], o["tout"], "out")
    near(torch, lse, o["lse"], o["tlse"], "lse")
    at_once, per = 64 if D <= 128 else 32, H // KV
    for name, got, old, add, tol, m in (("prefix_weight", pw, pw0, "pw", "tpw", R // G * T * per), ("weight", w, w0, "w", "tw", T * per)):
        want = old.double() + o[add]
        near(torch, got, want, o[tol] + want.abs() * 2.0 ** -24 * -(-m // at_once), name)


@pytest.mark.parametrize("shape", STEADY + MANY_PARTS + KINDS, ids=str)
def test_many_tiles(torch_mod, sampler, shape):  # noqa: F811
    say(f"steady {shape}")
    run(torch_mod, sampler, inputs(torch_mod, *shape, seed=sum(shape)))


@pytest.mark.parametrize("rise", [7.0, -7.0, 100.0, -100.0])
@pytest.mark.parametrize("shape", [s for s in STEADY if s[5] in (64, 128, 256)], ids=str)
def test_the_maximum_grows_within_a_part(torch_mod, sampler, shape, rise):  # noqa: F811
    """Scores that rise or fall by `rise` a tile: at 7 what came before still
    counts (a thousandth of the next tile's), at 100 it must vanish."""
    torch = torch_mod
    say(f"rising {shape} {rise}")
    x = inputs(torch, *shape, seed=6)
    D = shape[5]
    x["q"][..., 0] = 16.0
    for keys in (x["prefix_keys"], x["keys"]):
        step = rise * D ** 0.5 / (16.0 * 64.0)
        keys[..., 0] = (step * torch.arange(keys.shape[2], device="cuda")).to(torch.bfloat16)
    run(torch, sampler, x)


@pytest.mark.parametrize("shape", [s for s in STEADY if s[2] > 1 and s[5] != 40], ids=str)
def test_values_that_are_no_numbers_in_long_suffixes(torch_mod, sampler, shape):  # noqa: F811
    torch = torch_mod
    say(f"long suffixes {shape}")
    x = inputs(torch, *shape, seed=9)
    N, T, D = shape[7], shape[2], shape[5]
    x["values"][0, 0, N - 1, 3] = float("inf")
    x["values"][1, 1, N - T + 1, D - 1] = float("nan")
    x["values"][2, 2, 70, 0] = -float("inf")
    run(torch, sampler, x)
