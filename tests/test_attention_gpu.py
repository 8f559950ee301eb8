"""GPU tests of mxs_prefix_attention against the definition in 64 bits.

Errors, to first order.  A score's D products of bf16 values are exact in f32
and summed in any order: D 2^-24 sum |q k| |scale|; scaling it, taking a
maximum from it and the change of base are 4 more roundings of values up to
|s| + |max|; the exponential itself is within 2^-22.  Together the exponent of
each weight is off by at most e = D 2^-24 max sum |q k| |scale| + 8 2^-24 max
|s| + 2^-22 absolute, a weight by e relative; lse by e and the sum's own n 2^-24,
a normalised weight by twice that.  A weight's product with its value takes a
rounding to bf16 (half a step, 2^-8), the sum over n positions n 2^-24, the
output another 2^-8 of itself.  Accumulated weights: one addition for each
query, of the sum's size.  A weight below 2^-126 may vanish."""
import math
import sys

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_mod():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.fixture(scope="module")
def sampler(torch_mod):
    from metallix_amd import Sampler

    s = Sampler(max_rows=8, max_vocab=1024)
    yield s
    s.close()


def say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def inputs(torch, G, W, T, H, KV, D, P, N, seed=0, plens=None, lens=None, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    bf = torch.bfloat16
    x = dict(q=(spread * r(G * W, T, H, D)).to(bf), prefix_keys=r(G, KV, P, D).to(bf), prefix_values=r(G, KV, P, D).to(bf))
    if N is not None:
        x["keys"], x["values"] = r(G * W, KV, N, D).to(bf), r(G * W, KV, N, D).to(bf)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    if plens is not None:
        x["prefix_lengths"] = i32(plens)
    if lens is not None:
        x["lengths"] = i32(lens)
    return x


def oracle(torch, x, scale=None):
    """out, lse, the two weights' additions and their tolerances, all f64."""
    f = torch.float64
    q = x["q"]
    R, T, H, D = q.shape
    G, KV, P, _ = x["prefix_keys"].shape
    W, per = R // G, H // KV
    N = x["keys"].shape[2] if "keys" in x else 0
    scale = D ** -0.5 if scale is None else scale
    clamp = lambda v, m: max(0, min(int(v), m))
    plen = [P] * G if x.get("prefix_lengths") is None else [clamp(v, P) for v in x["prefix_lengths"].tolist()]
    slen = [N] * R if x.get("lengths") is None else [clamp(v, N) for v in x["lengths"].tolist()]
    z = lambda *s: torch.zeros(s, dtype=f, device="cuda")
    out, lse, tout, tlse = z(R, T, H, D), z(R, T, H), z(R, T, H, D), z(R, T, H)
    pw, w, tpw, tw = z(G, KV, P), z(R, KV, N), z(G, KV, P), z(R, KV, N)
    for r in range(R):
        g = r // W
        for k in range(KV):
            ka, va = x["prefix_keys"][g, k, : plen[g]].to(f), x["prefix_values"][g, k, : plen[g]].to(f)
            if N:
                ka = torch.cat([ka, x["keys"][r, k, : slen[r]].to(f)])
                va = torch.cat([va, x["values"][r, k, : slen[r]].to(f)])
            hs = slice(k * per, (k + 1) * per)
            for t in range(T):
                n = plen[g] + max(0, slen[r] - T + t + 1) if N else plen[g]
                kt, vt = ka[:n], va[:n]
                qt = q[r, t, hs].to(f)
                s = (qt @ kt.t()) * scale
                if n == 0:
                    lse[r, t, hs] = -math.inf
                    continue
                top = s.amax(1, keepdim=True)
                base = torch.where(top == -math.inf, 0.0, top)
                p = torch.exp(s - base)
                tot = p.sum(1, keepdim=True)
                share = torch.where(tot == 0, 0.0, p / tot)
                e = D * 2.0 ** -24 * (qt.abs() @ kt.abs().t()).nan_to_num(0, 0, 0).amax(1) * abs(scale)
                e = e + 8 * 2.0 ** -24 * s.abs().nan_to_num(0, 0, 0).amax(1) + 2.0 ** -22
                rel = 2 * e + n * 2.0 ** -24
                mag = share @ vt.abs()
                out[r, t, hs] = share @ vt
                lse[r, t, hs] = (base + torch.log(tot))[:, 0]
                tout[r, t, hs] = (rel[:, None] + 2.0 ** -8 + n * 2.0 ** -24) * mag * 1.01 + out[r, t, hs].abs() * 2.0 ** -8 + n * 2.0 ** -126
                tlse[r, t, hs] = rel + lse[r, t, hs].abs() * 2.0 ** -23
                add = share.sum(0)
                tadd = (share * rel[:, None]).sum(0) + per * 2.0 ** -126
                m = min(n, plen[g])
                pw[g, k, :m] += add[:m]
                tpw[g, k, :m] += tadd[:m]
                if n > m:
                    w[r, k, : n - m] += add[m:]
                    tw[r, k, : n - m] += tadd[m:]
    queries = W * T * per
    return dict(out=out, lse=lse, tout=tout, tlse=tlse, pw=pw, w=w, tpw=tpw + pw * queries * 2.0 ** -24,
                tw=tw + w * T * per * 2.0 ** -24)


def near(torch, got, want, tol, what):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities"
    fine = ~(inf | want.isnan())
    d, tol = (got - want)[fine].abs(), tol[fine]
    if d.numel():
        worst = (d / tol.clamp(min=1e-300)).max()
        assert bool((d <= tol).all()), f"{what}: off by {float(worst):.3g} tolerances"


def run(torch, s, x, weights=False, **kw):
    """One call over the inputs, its outputs checked; returns them."""
    G, KV, P, _ = x["prefix_keys"].shape
    R, T, H, D = x["q"].shape
    lse = torch.full((R, T, H), 7.0, device="cuda")
    kw = dict(kw, lse=lse, **{k: x[k] for k in ("prefix_lengths", "lengths") if k in x})
    before = {}
    if weights:
        g = torch.Generator(device="cuda").manual_seed(99)
        kw["prefix_weight"] = torch.rand((G, KV, P), generator=g, device="cuda")
        if "keys" in x:
            kw["weight"] = torch.rand((R, KV, x["keys"].shape[2]), generator=g, device="cuda")
        before = {k: kw[k].clone() for k in ("prefix_weight", "weight") if k in kw}
    out = s.prefix_attention(x["q"], x["prefix_keys"], x["prefix_values"], x.get("keys"), x.get("values"), **kw)
    s.sync()
    o = oracle(torch, x, kw.get("scale"))
    near(torch, out, o["out"], o["tout"], "out")
    near(torch, lse, o["lse"], o["tlse"], "lse")
    for name, add, tol in (("prefix_weight", "pw", "tpw"), ("weight", "w", "tw")):
        if name in before and before[name].numel():
            want = before[name].double() + o[add]
            near(torch, kw[name], want, o[tol] + want.abs() * 2.0 ** -24, name)
            unseen = o[add] == 0
            assert torch.equal(kw[name][unseen], before[name][unseen]) or name == "weight" and not unseen.any()
    return dict(out=out, lse=lse, **{k: kw[k] for k in before})


# groups, beams, tokens, heads, kv heads, dim, prefix, suffix (None: no suffix cache)
SHAPES = [
    (1, 1, 1, 1, 1, 8, 1, None), (1, 1, 1, 1, 1, 64, 0, 1), (1, 1, 1, 2, 1, 128, 1, 1), (2, 3, 1, 4, 2, 64, 31, 5),
    (1, 4, 1, 8, 2, 128, 33, 17), (3, 2, 1, 6, 3, 80, 64, 64), (2, 2, 1, 10, 2, 96, 65, 1), (1, 5, 1, 3, 1, 40, 127, 33),
    (1, 16, 1, 8, 8, 128, 128, 32), (1, 17, 1, 4, 4, 64, 129, 40), (2, 16, 1, 8, 4, 128, 500, 31),
    (1, 33, 1, 6, 6, 128, 300, 9), (1, 16, 1, 16, 4, 64, 257, 65), (1, 13, 1, 10, 2, 128, 1000, 70),
    (1, 32, 1, 16, 4, 128, 700, 20), (1, 40, 1, 14, 2, 64, 513, 3), (1, 64, 1, 16, 2, 128, 260, 12),
    (1, 64, 1, 20, 2, 80, 200, 33), (1, 4, 1, 4, 2, 256, 300, 40), (2, 20, 1, 8, 2, 256, 190, 10), (1, 9, 1, 4, 1, 192, 100, 66),
    (1, 3, 1, 2, 2, 136, 77, 8), (1, 2, 1, 2, 1, 72, 50, 50), (1, 2, 2, 2, 1, 64, 40, 2), (2, 3, 6, 6, 2, 80, 99, 30),
    (1, 4, 8, 8, 1, 128, 210, 70), (1, 2, 33, 4, 1, 64, 70, 90), (1, 1, 65, 5, 1, 128, 10, 65), (4, 1, 130, 2, 2, 64, 0, 130),
    (1, 1, 1, 4, 1, 128, 4000, None), (5, 1, 3, 3, 3, 64, 200, 100), (1, 6, 1, 8, 2, 256, 100, 12), (1, 7, 5, 4, 1, 256, 130, 40),
    (2, 2, 3, 12, 2, 160, 70, 20), (1, 2, 9, 4, 2, 64, 75, 33),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("weights", [False, True])
def test_shapes(torch_mod, sampler, shape, weights):
    say(f"shape {shape} weights {weights}")
    run(torch_mod, sampler, inputs(torch_mod, *shape, seed=sum(v or 0 for v in shape)), weights)


RAGGED = [
    # zero, one, past the capacity, negative; tokens past the suffix's length
    ((4, 2, 1, 4, 2, 64, 70, 9), [0, 70, 1, 100], [0, 9, 1, 0, 5, -3, 12, 0]),
    ((3, 2, 4, 4, 2, 128, 130, 40), [0, 64, 129], [0, 2, 3, 4, 33, 40]),
    ((2, 3, 5, 2, 1, 80, 33, 7), [-1, 0], [0, 1, 4, 5, 7, 6]),
    ((2, 16, 1, 8, 2, 64, 300, 50), [300, 1], list(range(0, 32))),
    ((8, 1, 1, 8, 8, 128, 1111, None), [1, 2, 31, 32, 33, 1111, 640, 0], None),
    ((2, 40, 1, 8, 1, 128, 400, 33), [0, 399], [i % 34 for i in range(80)]),
]


@pytest.mark.parametrize("shape,plens,lens", RAGGED, ids=str)
@pytest.mark.parametrize("weights", [False, True])
def test_lengths(torch_mod, sampler, shape, plens, lens, weights):
    """Also: what lies past the lengths, and past what a token sees, is NaN or infinite."""
    torch = torch_mod
    say(f"lengths {shape} {plens} {lens} {weights}")
    x = inputs(torch, *shape, seed=5, plens=plens, lens=lens)
    for g, n in enumerate(plens):
        for t, bad in ((x["prefix_keys"], math.nan), (x["prefix_values"], math.inf)):
            t[g, :, max(0, n):] = bad
    if lens is not None:
        for r, n in enumerate(lens):
            x["keys"][r, :, max(0, n):] = -math.inf
            x["values"][r, :, max(0, n):] = math.nan
    run(torch, sampler, x, weights)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_later_tokens_stay_out(torch_mod, sampler, bad, D):
    """A value or key that is no number at a suffix position reaches only the
    tokens that see it."""
    torch = torch_mod
    say(f"later tokens {bad} {D}")
    x = inputs(torch, 1, 2, 5, 6, 2, D, 40, 37, seed=3)
    x["values"][0, 0, 34, 3] = bad      # seen by tokens 2.. of row 0
    x["values"][1, 1, 36] = bad         # by token 4 of row 1
    if bad != -math.inf:
        x["keys"][1, 0, 35] = bad       # by tokens 3..
    got = run(torch, sampler, x, weights=True)
    assert bool(got["out"][0, :2].isfinite().all()) and not bool(got["out"][0, 2:, :3, 3].isfinite().any())


@pytest.mark.parametrize("shape", [(1, 2, 1, 4, 2, 64, 50, 8), (1, 20, 1, 4, 1, 128, 200, 8), (1, 4, 3, 2, 1, 80, 33, 8)], ids=str)
def test_scores_of_minus_infinity(torch_mod, sampler, shape):
    """Keys of -inf where the queries are positive: such positions weigh
    nothing; a query that sees only such gets out 0 and lse -inf."""
    torch = torch_mod
    say(f"minus infinity {shape}")
    x = inputs(torch, *shape, seed=8)
    G, W, T = shape[:3]
    x["q"][..., 1] = 1.5
    x["prefix_keys"][0, 0, ::3, 1] = -math.inf
    x["keys"][0, :, 1:3, 1] = -math.inf
    run(torch, sampler, x, weights=True)
    x["prefix_keys"][0, 0, :, 1] = -math.inf
    x["keys"][0, 0, :, 1] = -math.inf
    got = run(torch, sampler, x, weights=True)
    per = shape[3] // shape[4]
    assert bool((got["lse"][0, :, :per] == -math.inf).all()) and bool((got["out"][0, :, :per] == 0).all())
    assert bool(got["out"][1:].isfinite().all())


def test_scores_that_are_no_numbers(torch_mod, sampler):
    torch = torch_mod
    x = inputs(torch, 2, 3, 1, 4, 2, 128, 100, 9, seed=9)
    x["q"][1, 0, 2, 7] = math.nan            # one query
    x["prefix_keys"][1, 0, 64, 0] = math.nan  # every query of group 1's first cache head
    x["keys"][2, 1, 4, 3] = math.inf
    x["q"][2, 0, 2:, 3] = 2.0                 # scores of +inf
    got = run(torch, sampler, x, weights=True)
    nan = got["lse"].isnan()[:, 0]
    assert nan.tolist() == [[False] * 4, [False, False, True, False], [False, False, True, True]] + [[True, True, False, False]] * 3


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 20.0])
@pytest.mark.parametrize("shape", [(1, 3, 1, 8, 2, 64, 200, 30), (1, 48, 1, 8, 2, 128, 333, 30)], ids=str)
def test_scales(torch_mod, sampler, scale, shape):
    """Flat, turned over, and so steep that nearly all weight is on one position."""
    say(f"scale {scale} {shape}")
    run(torch_mod, sampler, inputs(torch_mod, *shape, seed=4), weights=True, scale=scale)


def test_the_maximum_grows(torch_mod, sampler):
    """Scores that rise, or fall, by hundreds from position to position."""
    torch = torch_mod
    for sign in (1.0, -1.0):
        for shape in ((1, 2, 1, 4, 1, 64, 300, 40), (1, 80, 1, 4, 1, 128, 300, 40)):
            x = inputs(torch, *shape, seed=6)
            x["q"][..., 0] = 30.0
            x["prefix_keys"][0, 0, :, 0] = sign * torch.arange(300, device="cuda").to(torch.bfloat16) * 4
            x["keys"][:, 0, :, 0] = sign * torch.arange(40, device="cuda").to(torch.bfloat16) * 40
            run(torch, sampler, x, weights=True)


def guarded(torch, shape, dtype, fill):
    """A tensor of `shape` inside a larger one that is `fill` around it."""
    pad = [n + 2 for n in shape[:-1]] + [shape[-1] + 16]
    whole = torch.full(pad, fill, dtype=dtype, device="cuda")
    part = whole
    for d, n in enumerate(shape[:-1]):
        part = part.narrow(d, 1, n)
    return whole, part.narrow(-1, 8, shape[-1])


@pytest.mark.parametrize("shape", [(2, 3, 2, 6, 2, 80, 70, 20), (1, 24, 1, 12, 3, 128, 140, 20), (1, 2, 1, 4, 4, 256, 40, 40)], ids=str)
def test_layouts(torch_mod, sampler, shape):
    """Padded and permuted caches, queries inside a wider projection and an
    output inside a larger tensor whose other elements stay."""
    torch = torch_mod
    say(f"layouts {shape}")
    G, W, T, H, KV, D, P, N = shape
    x = inputs(torch, *shape, seed=7, plens=[P - 3 * g for g in range(G)], lens=[N - r % 4 for r in range(G * W)])
    plain = run(torch, sampler, x, weights=True)
    fused = torch.full((G * W, T, H + 2 * KV, D + 8), math.nan, dtype=torch.bfloat16, device="cuda")
    y = dict(x, q=fused[:, :, KV:KV + H, :D])
    y["q"].copy_(x["q"])
    # [positions, heads, dim] in memory, keys and values in one tensor
    both = torch.full((2, G, P + 3, KV, D), math.inf, dtype=torch.bfloat16, device="cuda")
    for i, n in enumerate(("prefix_keys", "prefix_values")):
        y[n] = both[i, :, :P].transpose(1, 2)
        y[n].copy_(x[n])
    for n in ("keys", "values"):
        _, y[n] = guarded(torch, x[n].shape, torch.bfloat16, math.nan)
        y[n].copy_(x[n])
    whole, out = guarded(torch, x["q"].shape, torch.bfloat16, 3.0)
    marked = whole.clone()
    got = run(torch, sampler, y, weights=True, out=out)
    for n in plain:
        assert torch.equal(got[n], plain[n]), n
    out.fill_(3.0)
    assert torch.equal(whole, marked)


def test_three_dimensions_and_no_extras(torch_mod, sampler):
    torch = torch_mod
    x = inputs(torch, 2, 2, 1, 4, 2, 64, 50, 10, seed=1)
    want = run(torch, sampler, x)["out"]
    got = sampler.prefix_attention(x["q"][:, 0], x["prefix_keys"], x["prefix_values"], x["keys"], x["values"])
    sampler.sync()
    assert got.shape == (4, 4, 64) and torch.equal(got, want[:, 0])


def test_broadcast_inputs(torch_mod, sampler):
    """Strides of 0: one query for all rows, one cache for all groups."""
    torch = torch_mod
    x = inputs(torch, 3, 2, 1, 4, 2, 64, 50, 10, seed=2)
    x["q"] = x["q"][:1].expand(6, 1, 4, 64)
    for n in ("prefix_keys", "prefix_values"):
        x[n] = x[n][:1].expand(3, 2, 50, 64)
    run(torch, sampler, x, weights=True)


def test_many_queries(torch_mod, sampler):
    """More queries than the scratch holds at once."""
    torch = torch_mod
    for shape in ((2, 6, 40, 256, 8, 128, 20, 50), (1, 1, 300, 512, 4, 64, 9, 310), (3, 50, 2, 192, 2, 256, 5, 4)):
        say(f"many {shape}")
        run(torch, sampler, inputs(torch, *shape, seed=11), weights=True)


def test_equal_calls_give_equal_bits(torch_mod, sampler):
    torch = torch_mod
    for shape in ((2, 4, 1, 32, 8, 128, 3000, 100), (1, 64, 1, 32, 4, 64, 2000, 60)):
        x = inputs(torch, *shape, seed=13)
        one = [run_only(torch, sampler, x) for _ in range(3)]
        for other in one[1:]:
            assert all(torch.equal(a, b) for a, b in zip(one[0], other))


def run_only(torch, s, x):
    G, KV, P, _ = x["prefix_keys"].shape
    pw = torch.zeros((G, KV, P), device="cuda")
    w = torch.zeros(x["keys"].shape[:3], device="cuda")
    lse = torch.zeros(x["q"].shape[:3], device="cuda")
    out = s.prefix_attention(x["q"], x["prefix_keys"], x["prefix_values"], x["keys"], x["values"], lse=lse,
                             prefix_weight=pw, weight=w)
    s.sync()
    return out, lse, pw, w


def test_nothing_to_see(torch_mod, sampler):
    """No position at all: caches of none, with and without a suffix's."""
    torch = torch_mod
    for N in (None, 0):
        got = run(torch, sampler, inputs(torch, 2, 3, 2, 4, 2, 64, 0, N))
        assert bool((got["out"] == 0).all()) and bool((got["lse"] == -math.inf).all())


def test_calls_in_a_row(torch_mod, sampler):
    """Calls of different kinds that nothing waits between share the context's
    scratch in turn."""
    torch = torch_mod
    shapes = [(1, 4, 1, 8, 4, 128, 700, 30), (2, 40, 1, 8, 2, 64, 300, 20), (1, 3, 4, 6, 2, 200, 150, 40)]
    xs = [inputs(torch, *shape, seed=50 + i) for i, shape in enumerate(shapes)]
    want = [run_only(torch, sampler, x) for x in xs]
    w = torch.rand((1, 1, 2, 40000), device="cuda")
    cache = torch.randn((1, 2, 40000, 8), device="cuda")
    alone = sampler.cache_evict([cache.clone()], None, w, 500)
    sampler.sync()
    args = [(x, torch.zeros_like(a[1]), torch.zeros_like(a[2]), torch.zeros_like(a[3])) for x, a in zip(xs, want)]
    outs = []
    for i in range(6):
        x, lse, pw, ww = args[i % 3]
        pw.zero_(), ww.zero_()
        outs.append(sampler.prefix_attention(x["q"], x["prefix_keys"], x["prefix_values"], x["keys"], x["values"], lse=lse,
                                             prefix_weight=pw, weight=ww))
        gone = sampler.cache_evict([cache.clone()], None, w, 500)
    sampler.sync()
    assert torch.equal(gone.weight, alone.weight) and torch.equal(gone.index, alone.index)
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % 3][0])
    for (x, lse, pw, ww), a in zip(args, want):
        assert torch.equal(lse, a[1]) and torch.equal(pw, a[2]) and torch.equal(ww, a[3])


def test_nothing_to_do(torch_mod, sampler):
    torch = torch_mod
    x = inputs(torch, 2, 2, 1, 4, 2, 64, 50, 10)
    e = sampler.prefix_attention(x["q"][:0], x["prefix_keys"], x["prefix_values"], x["keys"][:0], x["values"][:0])
    assert e.shape == (0, 1, 4, 64)
    e = sampler.prefix_attention(x["q"][:, :0], x["prefix_keys"], x["prefix_values"], x["keys"], x["values"])
    sampler.sync()
    assert e.shape == (4, 0, 4, 64)


def test_refused_calls_write_nothing(torch_mod, sampler):
    torch = torch_mod
    from metallix_amd import SamplerError

    x = inputs(torch, 2, 2, 1, 4, 2, 64, 50, 10)
    lse = torch.full((4, 1, 4), 5.0, device="cuda")
    with pytest.raises(SamplerError, match="overlaps"):
        sampler.prefix_attention(x["q"], x["prefix_keys"], x["prefix_values"], out=x["q"], lse=lse)
    with pytest.raises(SamplerError, match="scale"):
        sampler.prefix_attention(x["q"], x["prefix_keys"], x["prefix_values"], scale=math.nan, lse=lse)
    with pytest.raises(ValueError):
        sampler.prefix_attention(x["q"].cpu(), x["prefix_keys"], x["prefix_values"], lse=lse)
    torch.cuda.synchronize()
    assert bool((lse == 5.0).all())


def test_a_stream_of_its_own(torch_mod):
    """Calls go to the sampler's stream, whatever the current one."""
    torch = torch_mod
    from metallix_amd import Sampler

    side = torch.cuda.Stream()
    s = Sampler(max_rows=8, max_vocab=1024, stream=side)
    try:
        x = inputs(torch, 1, 4, 1, 8, 4, 128, 900, 20, seed=21)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = run(torch, s, x, weights=False)["out"]
            y = {k: torch.zeros_like(v) for k, v in x.items()}
            for _ in range(50):   # (the copies are still queued on that stream when the call is made)
                for k, v in x.items():
                    y[k].copy_(v)
        got = s.prefix_attention(y["q"], y["prefix_keys"], y["prefix_values"], y["keys"], y["values"])
        s.sync()
        assert torch.equal(got, want)
    finally:
        s.close()


@pytest.mark.parametrize("shape", [(2, 4, 1, 8, 4, 128, 600, 50), (1, 48, 1, 8, 2, 64, 300, 20)], ids=str)
def test_captured_and_replayed(torch_mod, shape):
    """Replays see the queries, caches and lengths as they then are, between
    eager calls on the same context."""
    torch = torch_mod
    from metallix_amd import Sampler

    say(f"captured {shape}")
    side = torch.cuda.Stream()
    s = Sampler(max_rows=8, max_vocab=1024, stream=side)
    try:
        G, W, T, H, KV, D, P, N = shape
        x = inputs(torch, *shape, seed=31, plens=[P] * G, lens=[N] * (G * W))
        lse = torch.zeros((G * W, T, H), device="cuda")
        pw, w = torch.zeros((G, KV, P), device="cuda"), torch.zeros((G * W, KV, N), device="cuda")
        torch.cuda.synchronize()
        call = s.prefix_attention_launcher(x["q"], x["prefix_keys"], x["prefix_values"], x["keys"], x["values"], lse=lse,
                                           prefix_weight=pw, weight=w, prefix_lengths=x["prefix_lengths"], lengths=x["lengths"])
        call()
        s.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
        for i in range(4):
            y = inputs(torch, *shape, seed=40 + i, plens=[P - 7 * i - g for g in range(G)], lens=[N - i for _ in range(G * W)])
            for k in x:
                x[k].copy_(y[k])
            pw.zero_(), w.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in (call.out, lse, pw, w)]
            pw.zero_(), w.zero_()
            torch.cuda.synchronize()
            call()
            s.sync()
            assert all(torch.equal(a, b) for a, b in zip(got, (call.out, lse, pw, w)))
            o = oracle(torch, x)
            near(torch, got[0], o["out"], o["tout"], "out")
            near(torch, got[2], o["pw"], o["tpw"], "prefix_weight")
    finally:
        s.close()


def test_offsets_past_32_bits(torch_mod, sampler):
    """Caches of more than 2^32 bytes: a suffix's rows 2^31 elements apart,
    positions in the middle of a wide row."""
    torch = torch_mod
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    x = inputs(torch, 1, 3, 1, 4, 2, 64, 3000, 40, seed=17)
    wide = torch.empty(((3 << 31) + (1 << 20),), dtype=torch.bfloat16, device="cuda")
    y = dict(x)
    for i, n in enumerate(("keys", "values")):
        y[n] = wide.as_strided((3, 2, 40, 64), ((1 << 31) + (1 << 16), 64, 1 << 14, 1), i * (1 << 17))
        y[n].copy_(x[n])
    for i, n in enumerate(("prefix_keys", "prefix_values")):   # positions 2^20 elements apart
        y[n] = wide.as_strided((1, 2, 3000, 64), (0, 64, 1 << 20, 1), (1 << 18) + 4096 + 128 * i)
        y[n].copy_(x[n])
    run(torch, sampler, y, weights=True)
    del wide, y
    torch.cuda.empty_cache()
