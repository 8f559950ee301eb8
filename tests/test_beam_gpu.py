"""GPU tests of mxs_beam_select and mxs_beam_reorder (no counterpart in the
reference) against their definitions in 64 bits.

A selection's scores: the device's logarithm of the sum is within 2^-39 of
exact, and a score takes three more roundings of 2^-53 of its magnitude (this
oracle's own three the same); tokens and beams are exact, since the seeded
cases hold no two candidates of different beams nearer than that (asserted),
except where whole rows are equal."""
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NORM_ERR = 2.0 ** -39


@pytest.fixture(scope="module")
def torch_mod():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.fixture(scope="module")
def sampler(torch_mod):
    from metallix_amd import Sampler

    s = Sampler(max_rows=256, max_vocab=262144)
    yield s
    s.close()


def say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def bf16(x):
    """f32 values rounded to bf16 (nearest even; NaN and infinities kept)."""
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isfinite(x), r, x).astype(np.float32)


def oracle(x, score, n, *, ended=None, end_token=None, scale=None, mask=None, tokenizer_vocab=None, legal_norm=False):
    """x f32[G * W, V]; mask bool[G * W, V].  Returns token, beam, score,
    ended, status of each group, by the definition."""
    G, W = score.shape
    V = x.shape[1]
    tok, beam = np.full((G, n), -1), np.full((G, n), -1)
    sc, en, st = np.full((G, n), -np.inf), np.zeros((G, n), bool), np.zeros(G, int)
    for g in range(G):
        c = np.ones(W) if scale is None else scale[g]
        found = []   # (rank, beam, logit, token, score) in order of preference
        bad = np.any(~(score[g] < np.inf)) or np.any(~((c > 0) & (c < np.inf)))
        nonfinite = False
        for b in range(W):
            s = score[g, b]
            if bad or not s > -np.inf:
                continue
            if ended is not None and ended[g, b]:
                found.append((np.array([s * c[b]]), b, np.zeros(1), np.array([end_token]), np.array([s])))
                continue
            l = x[g * W + b].astype(np.float64)
            legal = np.ones(V, bool)
            if mask is not None:
                legal = mask[g * W + b] & (np.arange(V) < (V if tokenizer_vocab is None else tokenizer_vocab))
            counts = legal if legal_norm else np.ones(V, bool)
            if np.any(~(l[counts] < np.inf)):
                nonfinite = True
                continue
            m = l[counts].max() if counts.any() else -np.inf
            if not m > -np.inf:
                continue
            norm = m + float(np.log(np.sum(np.exp((l[counts] - m).astype(np.longdouble)))))
            at = np.nonzero(legal & (l > -np.inf))[0]
            v = s + (l[at] - norm)
            found.append((v * c[b], b, l[at], at, v))
        if bad or nonfinite:
            st[g], sc[g] = (-14 if bad else -6), np.nan
            continue
        if not found or not sum(len(f[0]) for f in found):
            st[g] = -3
            continue
        rank = np.concatenate([f[0] for f in found])
        who = np.concatenate([np.full(len(f[0]), f[1]) for f in found])
        logit = np.concatenate([f[2] for f in found])
        token = np.concatenate([f[3] for f in found])
        val = np.concatenate([f[4] for f in found])
        best = np.lexsort((token, -logit, who, -rank))[: n + 1]
        for i, k in zip(best, best[1:]):   # no two candidates of different beams too near to order
            if who[i] != who[k]:
                gap = rank[i] - rank[k]
                assert gap == 0.0 or gap > 2.5 * (NORM_ERR + abs(val[i]) * 2.0 ** -51) * max(c[who[i]], c[who[k]]), gap
        best = best[:n]
        k = len(best)
        tok[g, :k], beam[g, :k], sc[g, :k] = token[best], who[best], val[best]
        en[g, :k] = token[best] == (end_token if end_token is not None else -2)
    return tok, beam, sc, en, st


def words(mask):
    R, V = mask.shape
    W = (V + 31) // 32
    bits = np.zeros((R, W * 32), np.uint8)
    bits[:, :V] = mask
    return np.packbits(bits, axis=1, bitorder="little").view(np.uint32).view(np.int32).copy()


def dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


def upload(torch, x, dtype="f32", pad=0, poison=np.nan):
    """Logits of row stride ceil4(V) + pad, the padding poisoned."""
    R, V = x.shape
    host = np.full((R, (V + 3) // 4 * 4 + pad), poison, dtype=np.float32)
    host[:, :V] = x
    t = dev(torch, host)
    return (t.to(torch.bfloat16) if dtype == "bf16" else t)[:, :V]


def run(torch, sampler, x, score, n, *, dtype="f32", pad=0, mask=None, **kw):
    dk = dict(kw)
    if dk.get("ended") is not None:
        dk["ended"] = dev(torch, dk["ended"])
    if dk.get("scale") is not None:
        dk["scale"] = dev(torch, dk["scale"])
    if mask is not None:
        dk["mask"] = dev(torch, words(mask))
    r = sampler.beam_select(upload(torch, x, dtype, pad), dev(torch, score), n, **dk)
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in (r.token, r.beam, r.score, r.ended, r.status)]


def same(got, want):
    tok, beam, sc, en, st = got
    wt, wb, ws, we, wst = want
    assert np.array_equal(st, wst), (st, wst)
    assert np.array_equal(beam, wb), np.argwhere(beam != wb)[:5]
    assert np.array_equal(tok, wt), (np.argwhere(tok != wt)[:5], tok[tok != wt][:5], wt[tok != wt][:5])
    assert np.array_equal(en.astype(bool), we)
    fin = np.isfinite(ws)
    assert np.array_equal(np.isnan(sc), np.isnan(ws)) and np.array_equal(np.isneginf(sc), np.isneginf(ws))
    err = np.abs(sc[fin] - ws[fin])
    assert np.all(err <= NORM_ERR + np.abs(ws[fin]) * 2.0 ** -50 + 2.0 ** -48), err.max()


def check(torch, sampler, x, score, n, *, dtype="f32", pad=0, name="", **kw):
    say(f"case {name}: {score.shape} vocab {x.shape[1]} n {n} {dtype}")
    if dtype == "bf16":
        x = bf16(x)
    same(run(torch, sampler, x, score, n, dtype=dtype, pad=pad, **kw), oracle(x, score, n, **kw))


def scores(rng, G, W, first=True):
    s = -rng.uniform(1.0, 60.0, (G, 1)) - np.cumsum(rng.uniform(0.0, 1.5, (G, W)), 1)
    if first and G > 2:
        s[2, 1:] = -np.inf
    return s


def logits(rng, R, V, spread=2.5):
    x = (spread * rng.standard_normal((R, V))).astype(np.float32)
    ids = rng.integers(0, V, (R, 1 + V // 40))
    np.put_along_axis(x, ids, (6.0 + 8.0 * rng.random(ids.shape)).astype(np.float32), 1)
    return x


@pytest.mark.parametrize("G,W,V,n,dtype", [
    (1, 1, 1, 1, "f32"), (1, 1, 2, 4, "f32"), (2, 3, 3, 8, "f32"), (4, 2, 5, 16, "bf16"), (1, 4, 63, 8, "f32"),
    (3, 4, 64, 4, "bf16"), (2, 5, 1023, 10, "f32"), (2, 2, 1025, 4, "f32"), (5, 7, 4099, 14, "bf16"),
    (3, 64, 130, 128, "f32"), (2, 33, 2050, 66, "f32"), (4, 4, 8191, 8, "f32"), (4, 4, 8193, 1, "bf16"),
    (16, 16, 9000, 32, "f32"), (1, 64, 20000, 128, "f32"), (8, 8, 50257, 16, "f32"), (3, 5, 151936, 10, "f32"),
    (1, 4, 262144, 8, "bf16"), (1, 2, 262141, 128, "f32"), (64, 4, 7001, 4, "f32")])
def test_shapes(torch_mod, sampler, G, W, V, n, dtype):
    rng = np.random.default_rng(G * 1000 + W * 10 + V)
    check(torch_mod, sampler, logits(rng, G * W, V), scores(rng, G, W), n, dtype=dtype, pad=4 * (V % 3), name="shapes")


@pytest.mark.parametrize("V", [7, 1000, 33333])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ended_scale_and_masks(torch_mod, sampler, V, dtype):
    G, W, n = 6, 5, 10
    rng = np.random.default_rng(V)
    x, s = logits(rng, G * W, V), scores(rng, G, W)
    ended = rng.random((G, W)) < 0.4
    ended[1] = True                       # a group whose beams have all ended
    scale = ((5.0 + rng.integers(1, 40, (G, W))) / 6.0) ** -0.8
    mask = rng.random((G * W, V)) < 0.3
    mask[0:W] = False                     # a group without a legal token
    mask[2 * W] = False                   # a beam without one (its group's only live one: its first step)
    mask[3 * W, : V - 1] = False          # a beam with one
    kw = dict(ended=ended, end_token=min(V - 1, 3))
    t = torch_mod
    check(t, sampler, x, s, n, dtype=dtype, name="ended", **kw)
    check(t, sampler, x, s, n, dtype=dtype, name="scale", scale=scale, **kw)
    for norm in (False, True):
        check(t, sampler, x, s, n, dtype=dtype, name=f"mask {norm}", mask=mask, legal_norm=norm)
        check(t, sampler, x, s, n, dtype=dtype, name=f"all {norm}", mask=mask, legal_norm=norm,
              tokenizer_vocab=V - V // 7, scale=scale, **kw)


def test_values_in_masked_and_dead_places(torch_mod, sampler):
    G, W, V, n = 5, 3, 9001, 6
    rng = np.random.default_rng(5)
    x, s = logits(rng, G * W, V), scores(rng, G, W, first=False)
    mask = rng.random((G * W, V)) < 0.5
    s[0, 1] = -np.inf
    x[1] = np.nan                         # row of a beam that is not there
    ended = np.zeros((G, W), bool)
    ended[1, 2] = True
    x[5] = np.inf                         # row of an ended beam
    kw = dict(ended=ended, end_token=0)
    bad = np.where(mask, x, rng.choice([np.nan, np.inf, -np.inf, -3.4028235e38], x.shape).astype(np.float32))
    check(torch_mod, sampler, bad, s, n, mask=mask, legal_norm=True, name="poisoned masked places", **kw)
    low = np.where(mask, x, np.float32(-3.4028235e38))
    check(torch_mod, sampler, low, s, n, mask=mask, name="lowest value", **kw)
    check(torch_mod, sampler, low, s, n, name="lowest value, no mask", **kw)
    inf = np.where(mask, x, -np.inf).astype(np.float32)
    inf[12] = -np.inf                     # a row of nothing
    check(torch_mod, sampler, inf, s, n, name="-inf logits", **kw)
    inf[12:15] = -np.inf
    check(torch_mod, sampler, inf, s, n, name="a group of nothing", **kw)
    for v, at in ((np.nan, 0), (np.inf, V - 1), (np.nan, 8192), (-np.nan, 4444)):
        y = x.copy()
        y[7, at] = v                      # group 2 fails, the others stand
        got = run(torch_mod, sampler, y, s, n, **kw)
        assert got[4].tolist() == [0, 0, -6, 0, 0]
        same(got, oracle(y, s, n, **kw))
    s2 = s.copy()
    s2[3, 0], s2[4, 1] = np.nan, np.inf
    check(torch_mod, sampler, x, s2, n, name="scores", **kw)
    scale = np.ones((G, W))
    scale[0, 0], scale[1, 1], scale[2, 2], scale[3, 0] = 0.0, -1.0, np.nan, np.inf
    check(torch_mod, sampler, x, s, n, name="scales", scale=scale, **kw)


@pytest.mark.parametrize("V,n", [(100, 16), (8192, 16), (40000, 64), (151936, 128)])
def test_ties_and_orders(torch_mod, sampler, V, n):
    """Equal logits by lower token, equal beams by lower beam; rising and
    falling rows; few distinct values; zeros of both signs."""
    W = 4
    rng = np.random.default_rng(V)
    r = np.arange(V, dtype=np.float32)
    rows = [np.zeros(V), np.full(V, 5.0), r * 1e-3, -r * 1e-3, rng.integers(-2, 3, V), np.where(r % 7 == 0, 4.0, -1.0),
            np.where(r % 2 == 0, 0.0, -0.0), np.where(r % 5 == 0, 1.0, np.where(r % 3 == 0, 0.0, -0.0)),
            np.full(V, -1e30), np.full(V, 3e38), -r * 1e30, np.where(r == V // 2, 700.0, -700.0)]
    x = np.stack(rows).astype(np.float32)
    s = np.tile(np.array([-1.0, -2.5, -4.25, -6.125]), (3, 1))
    check(torch_mod, sampler, x, s, n, name="ties")
    same_rows = np.repeat(logits(rng, 2, V), W, 0)        # beams that are copies of one another
    check(torch_mod, sampler, same_rows, np.full((2, W), -3.5), n, name="equal beams")
    check(torch_mod, sampler, np.zeros((2 * W, V), np.float32), np.full((2, W), -3.5), n, name="all equal", dtype="bf16")


@pytest.mark.parametrize("G,W,V,n,dtype", [(8, 32, 151936, 64, "f32"), (4, 32, 50257, 64, "bf16"), (2, 64, 40000, 128, "f32"),
                                           (3, 1, 9000, 128, "bf16"), (2, 16, 20000, 100, "bf16")])
def test_first_steps_and_many_candidates(torch_mod, sampler, G, W, V, n, dtype):
    """One live beam a group (few chunks hold all candidates), many wanted;
    a group whose beams are nearly level; rows of few distinct values, whose
    ties pass every list's length."""
    rng = np.random.default_rng(V + n)
    x, s = logits(rng, G * W, V), scores(rng, G, W)
    s[0, 1:] = -np.inf
    s[1] = -4.0 - 1e-3 * np.arange(W)
    x[(G - 1) * W :] = np.round(x[(G - 1) * W :])
    check(torch_mod, sampler, x, s, n, dtype=dtype, name="many")


@pytest.mark.parametrize("top", [-3e38, -1e4, -750.0, -90.0, 0.0, 90.0, 800.0, 1e5, 3e38])
def test_ranges_of_logits(torch_mod, sampler, top):
    G, W, V, n = 2, 3, 20011, 6
    rng = np.random.default_rng(int(abs(top)) % 1000)
    with np.errstate(over="ignore"):
        x = (top - np.abs(logits(rng, G * W, V))).astype(np.float32)
    x[1, 15000] = x[1].max() + np.float32(1.0 if abs(top) < 1e6 else 0.0)   # a late maximum
    x[2, :8192] = -3.4028235e38
    x[3] -= np.float32(abs(top)) * np.float32(0.01) * rng.integers(0, 2, V).astype(np.float32)
    x = np.clip(x, -3.4028235e38, 3.4028235e38)
    check(torch_mod, sampler, x, scores(rng, G, W), n, name=f"top {top}")


def test_rising_rows(torch_mod, sampler):
    """Every token larger than all before it, so that a running threshold
    never rejects one, over several tiles; and jumps past e^700 midway."""
    G, W, V, n = 2, 2, 100003, 16
    rng = np.random.default_rng(9)
    x = np.sort(logits(rng, G * W, V), 1)
    x[1] = np.linspace(-2000.0, 2000.0, V)
    x[2, V // 2:] += 1500.0
    x[3] = x[3, ::-1]
    check(torch_mod, sampler, x, scores(rng, G, W, first=False), n, name="rising")


def test_outputs_in_place_of_inputs(torch_mod, sampler):
    torch = torch_mod
    G, W, V = 6, 4, 5000
    rng = np.random.default_rng(17)
    x, s = logits(rng, G * W, V), scores(rng, G, W)
    ended = rng.random((G, W)) < 0.3
    from metallix_amd import BeamResult

    sc, en = dev(torch, s), dev(torch, ended)
    e = lambda: torch.empty((G, W), dtype=torch.int32, device="cuda")
    out = BeamResult(token=e(), beam=e(), score=sc, ended=en, status=torch.empty(G, dtype=torch.int32, device="cuda"))
    sampler.beam_select(upload(torch, x), sc, W, ended=en, end_token=2, out=out)
    torch.cuda.synchronize()
    same([t.cpu().numpy() for t in (out.token, out.beam, sc, en, out.status)], oracle(x, s, W, ended=ended, end_token=2))


def test_captured_and_replayed(torch_mod):
    """A captured selection and move, replayed over new inputs with eager
    calls of another shape on the same context in between."""
    torch = torch_mod
    from metallix_amd import Sampler

    G, W, V, n = 3, 4, 30011, 4
    rng = np.random.default_rng(23)
    stream = torch.cuda.Stream()
    s = Sampler(max_rows=64, max_vocab=32768, stream=stream)
    try:
        with torch.cuda.stream(stream):
            lg = upload(torch, logits(rng, G * W, V))
            sc = dev(torch, scores(rng, G, W))
            state = torch.zeros((G * W, 5, 33), device="cuda")
            call = s.beam_launcher(lg, sc, n)
            move = s.reorder_launcher([state], call.out.beam)
            other, osc = upload(torch, logits(rng, 10, 9999), "bf16"), dev(torch, scores(rng, 2, 5))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call(lg)
            move()
        for i in range(4):
            x, ss = logits(rng, G * W, V), scores(rng, G, W, first=i % 2 == 0)
            st = rng.standard_normal((G * W, 5, 33)).astype(np.float32)
            with torch.cuda.stream(stream):
                lg.copy_(dev(torch, x))
                sc.copy_(dev(torch, ss))
                state.copy_(dev(torch, st))
                s.beam_select(other, osc, 10)
                graph.replay()
            torch.cuda.synchronize()
            o = call.out
            want = oracle(x, ss, n)
            same([t.cpu().numpy() for t in (o.token, o.beam, o.score, o.ended, o.status)], want)
            rows = (want[1] + np.arange(G)[:, None] * W).ravel()
            assert np.array_equal(state.cpu().numpy(), st[rows])
            assert move.status.cpu().tolist() == [0] * G
    finally:
        s.close()


def test_two_contexts_on_two_streams(torch_mod):
    torch = torch_mod
    from metallix_amd import Sampler

    rng = np.random.default_rng(29)
    jobs = []
    for i in range(2):
        st = torch.cuda.Stream()
        x, sc = logits(rng, 32, 50257), scores(rng, 8, 4)
        jobs.append((Sampler(max_rows=32, max_vocab=50304, stream=st), st, x, sc, upload(torch, x), dev(torch, sc), []))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, st, x, sc, lg, dsc, outs in jobs:
            outs.append(s.beam_select(lg, dsc, 8))
    torch.cuda.synchronize()
    for s, st, x, sc, lg, dsc, outs in jobs:
        want = oracle(x, sc, 8)
        for o in (outs[0], outs[7], outs[-1]):
            same([t.cpu().numpy() for t in (o.token, o.beam, o.score, o.ended, o.status)], want)
        first = outs[0].score.cpu().numpy()
        assert all(np.array_equal(o.score.cpu().numpy(), first) for o in outs)   # the same call gives the same bits
        s.close()


def test_refused_on_the_device(torch_mod, sampler):
    from metallix_amd import SamplerError

    torch = torch_mod
    lg, sc = torch.zeros((8, 100), device="cuda"), torch.zeros((2, 4), dtype=torch.float64, device="cuda")
    for kw in (dict(n=0), dict(n=129), dict(n=4, end_token=100), dict(n=4, legal_norm=True)):
        with pytest.raises(SamplerError, match="mxs_beam_select"):
            sampler.beam_select(lg, sc, **kw)
    with pytest.raises(SamplerError, match="max_rows"):
        sampler.beam_select(torch.zeros((260, 8), device="cuda"), torch.zeros((65, 4), dtype=torch.float64, device="cuda"), 4)
    with pytest.raises(ValueError):
        sampler.beam_select(lg, sc.cpu(), 4)
    with pytest.raises(ValueError):
        sampler.beam_reorder([lg.cpu()], torch.zeros((2, 4), dtype=torch.int32, device="cuda"))
    with pytest.raises(SamplerError, match="overlap"):
        sampler.beam_reorder([lg[:1].expand(8, 100)], torch.zeros((2, 4), dtype=torch.int32, device="cuda"))
    assert sampler.beam_select(lg[:0], sc[:0], 4).token.shape == (0, 4)


# ---------------------------------------------------------------------------
# The move of the states

PARENTS = {
    "stay": lambda rng, W: np.arange(W),
    "swap": lambda rng, W: np.arange(W) ^ 1 if W % 2 == 0 else np.roll(np.arange(W), 1),
    "cycle": lambda rng, W: np.roll(np.arange(W), 1),
    "back": lambda rng, W: np.roll(np.arange(W), -1),
    "one": lambda rng, W: np.full(W, W - 1),
    "first": lambda rng, W: np.zeros(W, int),
    "any": lambda rng, W: rng.integers(0, W, W),
    "holes": lambda rng, W: np.where(rng.random(W) < 0.4, -1, rng.integers(0, W, W)),
}


def moved(a, parent, lengths=None, dim=None):
    """a [G * W, ...] numpy: the state after the move."""
    G, W = parent.shape
    out = a.copy()
    for g in range(G):
        for b in range(W):
            p = parent[g, b]
            if p < 0:
                continue
            if lengths is None or dim is None:
                out[g * W + b] = a[g * W + p]
            else:
                at = (slice(None),) * (dim - 1) + (slice(0, max(0, int(lengths[g]))),)
                out[g * W + b][at] = a[g * W + p][at]
    return out


def fill(torch, rng, shape, dtype):
    size = torch.empty((), dtype=dtype).element_size()
    raw = rng.integers(0, 256, (*shape[:-1], shape[-1] * size), dtype=np.uint8)
    return dev(torch, raw).view(dtype)


def dtype_u8():
    import torch

    return torch.uint8


def bits(t):
    """A tensor's bytes, numpy, last dimension widened."""
    return t.contiguous().view(dtype_u8()).cpu().numpy()


@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 8, 9, 16, 31, 33, 64])
@pytest.mark.parametrize("kind", sorted(PARENTS))
def test_moves(torch_mod, sampler, W, kind):
    torch = torch_mod
    rng = np.random.default_rng(W * 100 + len(kind))
    G = 3
    parent = np.stack([PARENTS[kind](rng, W) for _ in range(G)])
    shapes = [((G * W, 3, 40), torch.float32), ((G * W, 7), torch.uint8), ((G * W, 2, 9, 33), torch.bfloat16),
              ((G * W,), torch.float64), ((G * W, 1001), torch.bfloat16)]
    say(f"case moves {kind} W {W}")
    states = [fill(torch, rng, s, d) for s, d in shapes]
    before = [bits(t) for t in states]
    st = sampler.beam_reorder(states, dev(torch, parent.astype(np.int32)))
    torch.cuda.synchronize()
    assert st.cpu().tolist() == [0] * G
    for t, b in zip(states, before):
        if t.dim() == 1:
            b = b.reshape(G * W, -1)
        assert np.array_equal(bits(t).reshape(b.shape), moved(b, parent)), (kind, W, t.shape)


@pytest.mark.parametrize("heads,P,dim,dtype,W", [(8, 48, 128, "bfloat16", 4), (3, 17, 65, "bfloat16", 5),
                                                 (1, 1, 1, "uint8", 2), (2, 300, 80, "float32", 16),
                                                 (5, 33, 7, "uint8", 3), (2, 9, 130, "bfloat16", 40)])
def test_moves_of_the_positions_in_use(torch_mod, sampler, heads, P, dim, dtype, W):
    torch = torch_mod
    rng = np.random.default_rng(heads * P + dim)
    G = 6
    parent = rng.integers(-1, W, (G, W))
    lengths = np.array([0, 1, P, P // 2, -3, P + 9])      # none, one, all, half; below and past the ends
    for order in ("heads", "positions", "time"):
        shape = (G * W, heads, P, dim) if order == "heads" else (G * W, P, heads, dim)
        t = fill(torch, rng, shape, getattr(torch, dtype))
        d = 2 if order == "heads" else 1
        if order == "time":                                # memory [heads][rows][positions][dim], rows within heads
            t = t.permute(2, 0, 1, 3).contiguous().permute(1, 0, 2, 3)
            d = 2
        a = bits(t)
        say(f"case lengths {order} {tuple(t.shape)} {dtype}")
        sampler.beam_reorder([t], dev(torch, parent.astype(np.int32)), lengths=dev(torch, lengths.astype(np.int32)),
                             length_dim=d)
        torch.cuda.synchronize()
        assert np.array_equal(bits(t), moved(a, parent, lengths, d)), order


def test_many_states_at_once_and_odd_addresses(torch_mod, sampler):
    """More states than one launch takes, some with lengths and some without,
    inside larger buffers whose other bytes stay, at odd addresses."""
    torch = torch_mod
    rng = np.random.default_rng(41)
    G, W, P = 2, 4, 11
    parent, lengths = rng.integers(0, W, (G, W + 3)), np.array([3, P])
    bufs, states, dims, want = [], [], [], []
    for i in range(150):
        n = int(rng.integers(1, 90))
        off = int(rng.integers(0, 40))
        buf = fill(torch, rng, (G * W * P * n + 80,), torch.uint8)
        t = buf[off : off + G * W * P * n].view(G * W, P, n)
        d = 1 if i % 3 else None
        b = buf.cpu().numpy()
        b[off : off + G * W * P * n] = moved(b[off : off + G * W * P * n].reshape(G * W, P, n).copy(), parent[:, :W],
                                             lengths if d else None, d).ravel()
        bufs.append(buf), states.append(t), dims.append(d), want.append(b)
    say("case many states")
    pt = dev(torch, parent.astype(np.int32))
    st = sampler.beam_reorder(states, pt, beams=W, lengths=dev(torch, lengths.astype(np.int32)), length_dim=dims)
    torch.cuda.synchronize()
    assert st.cpu().tolist() == [0, 0]
    for i, (b, w) in enumerate(zip(bufs, want)):
        assert np.array_equal(b.cpu().numpy(), w), i


def test_parents_outside_the_group(torch_mod, sampler):
    torch = torch_mod
    rng = np.random.default_rng(43)
    G, W = 5, 4
    parent = rng.integers(0, W, (G, W))
    parent[1, 2], parent[3, 0], parent[4, 3] = W, -2, 2 ** 31 - 1
    states = [fill(torch, rng, (G * W, 100), torch.float32) for _ in range(70)]
    before = [bits(t) for t in states]
    say("case parents outside")
    st = sampler.beam_reorder(states, dev(torch, parent.astype(np.int32)))
    torch.cuda.synchronize()
    assert st.cpu().tolist() == [0, -16, 0, -16, -16]
    good = parent.copy()
    good[[1, 3, 4]] = -1
    for t, b in zip(states, before):
        assert np.array_equal(bits(t), moved(b, good))


def test_a_move_past_32_bits(torch_mod, sampler):
    """One state of 6 GB whose rows lie past 2^32 bytes from its start."""
    torch = torch_mod
    rows, n = 6, 1 << 30
    t = torch.zeros((rows, n), dtype=torch.uint8, device="cuda")
    at = torch.tensor([0, 1, 12345677, n // 2 + 3, n - 17, n - 1], device="cuda")
    for r in range(rows):
        t[r, at] = torch.arange(6, dtype=torch.uint8, device="cuda") + 10 * (r + 1)
    say("case 6 GB")
    parent = torch.tensor([[5, 5, 0, 1, 4, 3]], dtype=torch.int32, device="cuda")
    sampler.beam_reorder([t], parent)
    torch.cuda.synchronize()
    assert (t[:, at] - torch.arange(6, dtype=torch.uint8, device="cuda")).cpu()[:, 0].tolist() == [60, 60, 10, 20, 50, 40]
    assert all(len(set(r)) == 1 for r in (t[:, at] - torch.arange(6, dtype=torch.uint8, device="cuda")).cpu().tolist())
    assert [int(t[r].count_nonzero()) for r in range(rows)] == [6] * rows


@pytest.mark.parametrize("n", [1, 2, 5, 10, 31, 64, 100, 128])
@pytest.mark.parametrize("blocks", [(2,), (0, 3), (1, 2, 3), (0, 1, 2, 3)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_legal_tokens_in_some_blocks_only(torch_mod, sampler, n, blocks, dtype):
    """Legal tokens in some of the 256-token blocks of every 1024, whole,
    sparse or in runs, so that only some waves hold candidates; the vocabulary
    ends inside a block."""
    G, W, V = 3, 2, 3 * 4096 + 300
    rng = np.random.default_rng(n + 7 * len(blocks))
    x, s = logits(rng, G * W, V), scores(rng, G, W)
    at = np.arange(V)
    mask = np.broadcast_to(np.isin(at // 256 % 4, blocks), (G * W, V)).copy()
    mask[1] &= rng.random(V) < 0.02       # sparse
    mask[2] &= at // 40 % 7 == 0          # runs
    mask[3] &= at % 1024 < 300            # the first two blocks at most
    mask[5] &= at >= 3 * 4096             # the last tile, which the row's end cuts
    check(torch_mod, sampler, x, s, n, dtype=dtype, name=f"blocks {blocks}", mask=mask, legal_norm=n % 2 == 0)


@pytest.mark.parametrize("W,n", [(1, 64), (1, 100), (2, 32), (6, 7), (20, 24), (64, 128)])
@pytest.mark.parametrize("centre", [-1.0, 0.0, 0.5, 2.0, 4.0])
def test_ranks_on_both_sides_of_a_power_of_two(torch_mod, sampler, W, n, centre):
    """Groups whose listed candidates' ranks straddle 0 and the powers of two
    (cumulative scores may have any sign), many of them close together."""
    G, V = 2, 20000
    rng = np.random.default_rng(W + n)
    x = (0.3 * rng.standard_normal((G * W, V))).astype(np.float32)
    ids = rng.integers(0, V, (G * W, 400))
    np.put_along_axis(x, ids, (9.0 + 0.4 * rng.standard_normal(ids.shape)).astype(np.float32), 1)
    # candidates near -ln(400): their scores near `centre`
    s = centre + np.log(400.0) + np.cumsum(rng.uniform(0.0, 0.2, (G, W)), 1)
    check(torch_mod, sampler, x, s, n, name=f"centre {centre}")
