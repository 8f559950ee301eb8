"""GPU tests of mxs_cache_evict against a direct statement of its rule: all
results are moved values, so they are equal."""
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


def rule(weight, index, n, first, recent):
    """Where each of the n slots takes its content from, for one row in use."""
    L = len(weight)
    if L <= n:
        return list(range(L))
    newest = max(index)
    kept_anyway = [p < first or p > newest - recent for p in index]
    key = lambda i: (not kept_anyway[i], 0.0 if kept_anyway[i] else math.inf if math.isnan(weight[i]) else -weight[i],
                     not kept_anyway[i] and math.isnan(weight[i]), i)
    kept = set(sorted(range(L), key=key)[:n])
    late = iter(sorted(i for i in kept if i >= n))
    return [i if i in kept else next(late) for i in range(n)]


def inputs(torch, L, S, H, C, D, seed=0, dtype=None, ties=8.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = dtype or torch.bfloat16
    cache = lambda: [torch.randn((S, H, C, D), generator=g, device="cuda").to(dt) for _ in range(L)]
    w = torch.exp(2.0 * torch.randn((L, S, H, C), generator=g, device="cuda"))
    if ties:
        w = torch.round(w * ties) / ties
    index = torch.argsort(torch.rand((L, S, H, C), generator=g, device="cuda"), -1).to(torch.int32)
    return cache(), cache(), w, index


def check(torch, s, keys, values, w, index, lengths, n, first=0, recent=0, **kw):
    L, S, H, C = w.shape
    k0, v0 = [t.clone() for t in keys], None if values is None else [t.clone() for t in values]
    w0, i0 = w.clone(), None if index is None else index.clone()
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = s.cache_evict(keys, values, w, n, index=index, lengths=lens, keep_first=first, keep_recent=recent, **kw)
    s.sync()
    assert torch.equal(w.view(torch.int32), w0.view(torch.int32)) and (index is None or torch.equal(index, i0))
    used = [C] * S if lengths is None else [max(0, min(v, C)) for v in lengths]
    assert out.lengths.tolist() == [min(u, n) for u in used]
    wl = w.cpu().tolist()
    il = [[[list(range(C))] * H] * S] * L if index is None else index.cpu().tolist()
    source = torch.arange(C, device="cuda").expand(L, S, H, C).clone()
    for l in range(L):
        for g in range(S):
            for h in range(H):
                src = rule(wl[l][g][h][: used[g]], il[l][g][h][: used[g]], n, first, recent)
                source[l, g, h, : len(src)] = torch.tensor(src, dtype=torch.long)
    full = torch.arange(C, dtype=torch.int32, device="cuda").expand(L, S, H, C) if index is None else index
    inside = torch.arange(C, device="cuda") < torch.tensor([min(u, n) for u in used], device="cuda")[None, :, None, None]
    want_w = torch.where(inside, torch.gather(w, 3, source), 0.0)
    assert torch.equal(out.weight.view(torch.int32), want_w.view(torch.int32)), "weight"
    assert torch.equal(out.index, torch.where(inside, torch.gather(full, 3, source), -1)), "index"
    for now, before in ((keys, k0), (values, v0)):
        if now is None:
            continue
        for l in range(L):
            want = torch.gather(before[l], 2, torch.where(inside, source, torch.arange(C, device="cuda"))[l][..., None].expand_as(before[l]))
            assert torch.equal(now[l].contiguous().view(torch.uint8), want.contiguous().view(torch.uint8)), f"layer {l}"
    return out


CASES = [
    # layers, segments, heads, capacity, dim, budget, first, recent, lengths, with an index
    (1, 1, 1, 1, 8, 1, 0, 0, None, False), (1, 1, 1, 2, 8, 1, 0, 0, None, False), (1, 1, 2, 2, 8, 1, 0, 1, None, True),
    (2, 3, 2, 64, 16, 63, 1, 5, None, True), (2, 3, 2, 65, 40, 64, 4, 16, [65, 64, 0], True),
    (3, 2, 1, 200, 64, 100, 4, 30, [200, 101], False), (1, 4, 3, 130, 80, 1, 0, 0, [130, 2, 1, 0], True),
    (1, 4, 3, 130, 80, 1, 1, 0, [130, 2, 1, -5], True), (1, 4, 3, 130, 80, 1, 0, 1, [130, 2, 1, 500], True),
    (1, 1, 2, 1025, 128, 1024, 4, 256, None, True), (2, 1, 2, 3000, 24, 700, 4, 128, [2999], True),
    (1, 2, 1, 5000, 8, 4999, 0, 0, None, False), (1, 2, 1, 5000, 8, 2500, 100, 2400, None, True),
    (1, 1, 1, 20000, 16, 64, 2, 8, None, True), (70, 1, 1, 40, 8, 17, 1, 3, None, True), (1, 1, 3, 40000, 8, 30000, 4, 1000, [39999], True),
    (20, 2, 8, 90, 32, 40, 4, 20, [90, 77], True),
]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_cases(torch_mod, sampler, case):
    torch = torch_mod
    say(f"evict {case}")
    L, S, H, C, D, n, first, recent, lengths, indexed = case
    keys, values, w, index = inputs(torch, L, S, H, C, D, seed=C)
    check(torch, sampler, keys, values, w, index if indexed else None, lengths, n, first, recent)


def test_equal_weights(torch_mod, sampler):
    """All equal: the lowest slots stay, and nothing moves."""
    torch = torch_mod
    for fill in (0.0, 1.5, math.inf, -math.inf, math.nan):
        keys, values, w, index = inputs(torch, 1, 1, 2, 300, 16)
        w.fill_(fill)
        before = keys[0].clone()
        check(torch, sampler, keys, values, w, None, None, 120)
        assert torch.equal(keys[0], before)
        check(torch, sampler, keys, values, w, index, None, 120, 3, 50)


def test_weights_of_every_kind(torch_mod, sampler):
    """NaN behind everything, infinities, zeros of both signs (equal), negative
    and subnormal ones."""
    torch = torch_mod
    keys, values, w, index = inputs(torch, 2, 2, 2, 500, 16, seed=3)
    kinds = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, -3.0, 3.4e38, 1.0], device="cuda")
    pick = torch.randint(10, w.shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    w.copy_(kinds[pick])
    for n in (1, 49, 50, 51, 120, 250, 400, 449, 499):
        check(torch, sampler, [k.clone() for k in keys], [v.clone() for v in values], w, index, None, n, min(2, n - 1), min(9, n // 2))


def test_one_at_a_time(torch_mod, sampler):
    """A full cache that takes a position and loses one, again and again, as a
    generation does: the weights and positions of one eviction go into the next."""
    torch = torch_mod
    L, S, H, C, D, n = 2, 2, 3, 41, 16, 40
    keys, values, w, index = inputs(torch, L, S, H, C, D, seed=9)
    index = torch.arange(C, dtype=torch.int32, device="cuda").expand(L, S, H, C).contiguous()
    g = torch.Generator(device="cuda").manual_seed(1)
    for step in range(60):
        out = check(torch, sampler, keys, values, w, index, None, n, 4, 8)
        w, index = out.weight, out.index
        assert int(index[..., :n].min()) == 0 and bool((index[..., n:] == -1).all())
        live = index[..., :n].sort(-1).values
        assert bool((live[..., 1:] != live[..., :-1]).all()) and bool((live[..., :4] == torch.arange(4, device="cuda")).all())
        assert bool((live[..., -8:] == torch.arange(C + step - 8, C + step, device="cuda")).all())
        w[..., :n] += torch.rand((L, S, H, n), generator=g, device="cuda")
        w[..., n] = torch.rand((L, S, H), generator=g, device="cuda")
        index[..., n] = C + step
        for t in keys + values:
            t[:, :, n] = step


@pytest.mark.parametrize("D,dtype", [(1, "uint8"), (7, "uint8"), (130, "bfloat16"), (65, "bfloat16"), (33, "float32"), (3, "float64")])
def test_types_and_alignments(torch_mod, sampler, D, dtype):
    """Positions of any number of bytes at any alignment; neighbours stay."""
    torch = torch_mod
    dt = getattr(torch, dtype)
    L, S, H, C = 2, 2, 3, 70
    g = torch.Generator(device="cuda").manual_seed(D)
    whole = torch.randint(0, 200, (2, L, S, H, C, D + 3), generator=g, device="cuda").to(dt)
    before = whole.clone()
    caches = whole[..., 1:1 + D]
    _, _, w, index = inputs(torch, L, S, H, C, 8, seed=2)
    check(torch, sampler, list(caches[0]), list(caches[1]), w, index, [70, 55], 30, 2, 6)
    assert torch.equal(whole[..., 0], before[..., 0]) and torch.equal(whole[..., 1 + D:], before[..., 1 + D:])


def test_layouts(torch_mod, sampler):
    """[positions, heads, dim] in memory; keys alone; the outputs given."""
    torch = torch_mod
    from metallix_amd import EvictResult

    keys, values, w, index = inputs(torch, 2, 2, 3, 90, 32, seed=4)
    turned = lambda ts: [t.transpose(1, 2).contiguous().transpose(1, 2) for t in ts]
    check(torch, sampler, turned(keys), turned(values), w, index, [90, 80], 33, 1, 5)
    check(torch, sampler, keys, None, w, index, [90, 80], 33, 1, 5)
    keys, values, w, index = inputs(torch, 2, 2, 3, 90, 32, seed=4)
    out = EvictResult(torch.full_like(w, 9.0), torch.full_like(index, 9), torch.zeros(2, dtype=torch.int32, device="cuda"))
    got = check(torch, sampler, keys, values, w, index, None, 90, out=out)   # nothing to evict
    assert got is out and torch.equal(out.weight, w) and torch.equal(out.index, index)


def test_long_caches(torch_mod, sampler):
    """The most slots; a tensor of more than 2^32 bytes."""
    torch = torch_mod
    C = 1 << 20
    g = torch.Generator(device="cuda").manual_seed(7)
    w = torch.rand((1, 1, 1, C), generator=g, device="cuda")
    x = torch.randint(0, 1 << 30, (1, 1, C, 2), generator=g, device="cuda", dtype=torch.int32)
    for n in (5, C // 3, C - 1):
        say(f"long {n}")
        check(torch, sampler, [x.clone()], None, w, None, None, n, 4, 1)
    big = torch.empty((2, 2, 9000, 8, 16384), dtype=torch.bfloat16, device="cuda")[:, 0, :, 3].unsqueeze(1)   # 4.7 GB, wide strides
    big.copy_(torch.randint(0, 200, big.shape, generator=g, device="cuda"))
    check(torch, sampler, [big], None, torch.rand((1, 2, 1, 9000), generator=g, device="cuda"), None, [9000, 8500], 8000, 4, 100)


@pytest.mark.parametrize("ties", [0.0, 4.0, 0.02])
def test_long_rows_of_few_caches(torch_mod, sampler, ties):
    """Rows that several workgroups share: some within the budget, distinct
    weights, many equal ones, and nearly all equal."""
    torch = torch_mod
    for L, S, H, C, lengths, n, first, recent in ((1, 3, 1, 50001, [50001, 900, 33000], 1000, 4, 300), (2, 1, 2, 40000, None, 39000, 0, 0),
                                                  (1, 2, 1, 100000, [99999, 65537], 65536, 0, 64)):
        say(f"long rows {C} {ties}")
        keys, values, w, index = inputs(torch, L, S, H, C, 8, seed=6, ties=ties)
        check(torch, sampler, keys, values, w, index, lengths, n, first, recent)
        check(torch, sampler, keys, None, w, None, lengths, n, first, recent)


def test_nothing_to_do_and_refusals(torch_mod, sampler):
    torch = torch_mod
    from metallix_amd import SamplerError

    keys, values, w, index = inputs(torch, 1, 2, 2, 30, 16)
    before = keys[0].clone()
    for bad, word in ((dict(budget=0), "budget"), (dict(budget=5, keep_first=6), "keep_first")):
        with pytest.raises(SamplerError, match=word):
            sampler.cache_evict(keys, values, w, **bad)
    with pytest.raises(SamplerError, match="overlap"):
        sampler.cache_evict([keys[0][:, :1].expand(2, 2, 30, 16)], None, w, 5)
    with pytest.raises(ValueError):
        sampler.cache_evict(keys, values, w.cpu(), 5)
    e = sampler.cache_evict([], [], w[:0], 5)
    sampler.sync()
    assert e.weight.shape == (0, 2, 2, 30) and torch.equal(keys[0], before)


@pytest.mark.parametrize("C,n", [(200, 80), (50000, 3000)])
def test_captured_and_replayed(torch_mod, C, n):
    torch = torch_mod
    from metallix_amd import Sampler

    side = torch.cuda.Stream()
    s = Sampler(max_rows=8, max_vocab=1024, stream=side)
    try:
        keys, values, w, index = inputs(torch, 3, 2, 2, C, 16, seed=1)
        lens = torch.tensor([C, C - 50], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        call = s.cache_evict_launcher(keys, values, w, n, index=index, lengths=lens, keep_first=2, keep_recent=10)
        call()
        s.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
        for i in range(4):
            k, v, w1, i1 = inputs(torch, 3, 2, 2, C, 16, seed=20 + i)
            n1 = torch.tensor([C - 50 * i, C - 10], dtype=torch.int32, device="cuda")
            for a, b in zip(keys + values + [w, index, lens], k + v + [w1, i1, n1]):
                a.copy_(b)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = check(torch, s, k, v, w1, i1, n1.tolist(), n, 2, 10)
            assert torch.equal(call.out.weight, want.weight) and torch.equal(call.out.index, want.index)
            assert all(torch.equal(a, b) for a, b in zip(keys + values, k + v))
    finally:
        s.close()
