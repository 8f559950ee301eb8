"""BeamSearch.attention at steps of a search, its calls captured, its own caches
evicted, its sequences ended, against the definition."""
import pytest

from test_attention_gpu import near, oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_mod():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


G, W, H, KV, D, P, N, V = 2, 3, 4, 2, 64, 50, 12, 300


def setup(torch, stream=None, seed=1, **kw):
    """A search of N tokens, logits, the arguments of its attention."""
    from metallix_amd import BeamSearch, Sampler

    s = Sampler(max_rows=G * W, max_vocab=V, **({} if stream is None else dict(stream=stream)))
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *d: torch.randn(d, generator=g, device="cuda")
    bf = lambda *d: r(*d).to(torch.bfloat16)
    x = dict(q=bf(G * W, H, D), prefix_keys=bf(G, KV, P, D), prefix_values=bf(G, KV, P, D), keys=bf(G * W, KV, N, D),
             values=bf(G * W, KV, N, D))
    torch.cuda.synchronize()
    return s, BeamSearch(s, G, W, N, **kw), (lambda: 3.0 * r(G * W, V)), x


def call(search, x, **kw):
    return search.attention(x["q"], x["prefix_keys"], x["prefix_values"], x["keys"], x["values"], **kw)


def definition(torch, x, lengths, **kw):
    return oracle(torch, dict(x, q=x["q"][:, None], lengths=lengths, **kw))


def test_a_captured_call_says_nothing_about_eager_ones(torch_mod):
    """A step's first attention is captured; an eager one that comes before the
    replay, and replays after later steps, read the positions of their own step."""
    torch = torch_mod
    side = torch.cuda.Stream()
    s, search, logits, x = setup(torch, stream=side)
    try:
        with torch.cuda.stream(side):
            for _ in range(3):
                search.step(logits())
                call(search, x)
            search.step(logits())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = call(search, x)
        for i in range(4):
            steps = search.steps
            out = call(search, x)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for what, got, n in (("eager", out, steps), ("replayed", captured, 4)):
                o = definition(torch, x, torch.full((G * W,), n))
                near(torch, got[:, None], o["out"], o["tout"], f"{what} after {steps} steps")
            with torch.cuda.stream(side):
                search.step(logits())
    finally:
        s.close()


def test_own_caches_that_are_evicted(torch_mod):
    """The search goes on over own caches that are held to a budget: their
    lengths come from the eviction, and a new position goes behind what is left."""
    torch = torch_mod
    s, search, logits, x = setup(torch)
    rows, budget = G * W, 4
    try:
        keys, values = x["keys"][:, :, :budget + 2].clone(), x["values"][:, :, :budget + 2].clone()
        C = budget + 2
        w = torch.zeros((1, rows, KV, C), device="cuda")
        index = torch.arange(C, dtype=torch.int32, device="cuda").expand(1, rows, KV, C).contiguous()
        n = torch.zeros((rows, 1), dtype=torch.int32, device="cuda")
        for step in range(N):
            search.step(logits(), [keys, values, w[0], index[0], n])
            at = n.long().view(rows, 1, 1).expand(rows, KV, 1)
            keys.scatter_(2, at[..., None].expand(-1, -1, -1, D), x["keys"][:, :, step:step + 1])
            values.scatter_(2, at[..., None].expand(-1, -1, -1, D), x["values"][:, :, step:step + 1])
            index[0].scatter_(2, at, step)
            n += 1
            w0 = w.clone()
            out = call(search, dict(x, keys=keys, values=values), weight=w[0], lengths=n.view(-1))
            s.sync()
            y = dict(x, keys=keys, values=values)
            o = definition(torch, y, n.view(-1))
            near(torch, out[:, None], o["out"], o["tout"], f"step {step}: out")
            near(torch, w[0], w0[0].double() + o["w"], o["tw"] + (w0[0] + 1).double() * 2.0 ** -23, f"step {step}: weight")
            assert n.view(-1).tolist() == [min(step + 1, budget + 1)] * rows
            e = s.cache_evict([keys], [values], w, budget, index=index, lengths=n.view(-1), keep_recent=2)
            w, index, n = e.weight, e.index, e.lengths.view(-1, 1)
    finally:
        s.close()


def test_ended_and_empty_beams_add_no_weights(torch_mod):
    """Of a group, one sequence that has ended, one beam without a sequence, whose
    query is NaN, and one that goes on: the weights are the last one's."""
    torch = torch_mod
    end = 7
    s, search, _, x = setup(torch, end_token=end)
    try:
        logits = torch.full((G * W, V), -float("inf"), device="cuda")
        logits[0, [end, 3]] = torch.tensor([1.0, 0.5], device="cuda")          # group 0: two sequences, one of them ended
        logits[W, [end, 4, 5]] = torch.tensor([0.1, 1.0, 0.5], device="cuda")  # group 1: three
        search.step(logits)
        live = [False, True, False, True, True, False]
        assert ((search.score > -float("inf")) & ~search.ended).view(-1).tolist() == live
        x["q"][2] = float("nan")
        pw, w = torch.rand((G, KV, P), device="cuda"), torch.rand((G * W, KV, N), device="cuda")
        pw0, w0 = pw.clone(), w.clone()
        lse = torch.empty((G * W, H), device="cuda")
        out = call(search, x, prefix_weight=pw, weight=w, lse=lse)
        s.sync()
        o = definition(torch, x, torch.ones(G * W))
        near(torch, out[:, None], o["out"], o["tout"], "out")      # every row's
        near(torch, lse[:, None], o["lse"], o["tlse"], "lse")
        add, tol = torch.zeros_like(o["pw"]), torch.zeros_like(o["pw"])
        for r in range(G * W):
            g = r // W
            if not live[r]:
                assert torch.equal(w[r], w0[r])
                continue
            y = {k: v[g:g + 1] if k.startswith("prefix") else v[r:r + 1] for k, v in x.items()}
            one = definition(torch, y, torch.ones(1))
            add[g] += one["pw"][0]
            tol[g] += one["tpw"][0]
            near(torch, w[r], w0[r].double() + one["w"][0], one["tw"][0] + (w0[r] + 1).double() * 2.0 ** -23, f"weight {r}")
        near(torch, pw, pw0.double() + add, tol + (pw0 + 1).double() * 2.0 ** -22, "prefix_weight")
    finally:
        s.close()


@pytest.mark.parametrize("shape", [(2, 3, 1, 8, 2, 64, 200, 20), (1, 20, 3, 4, 1, 128, 300, 30), (2, 2, 2, 6, 1, 256, 70, 40)], ids=str)
def test_rows_that_do_not_count(torch_mod, shape):
    """Sampler.prefix_attention with `counted`: the weights of the rows that
    count, bit for bit what these add where they are all there is to add."""
    torch = torch_mod
    from metallix_amd import Sampler
    from test_attention_gpu import inputs

    G, W, T, H, KV, D, P, N = shape
    x = inputs(torch, *shape, seed=3, lens=[N - r % 5 for r in range(G * W)])
    counted = torch.tensor([r % 3 != 1 for r in range(G * W)], device="cuda")
    s = Sampler(max_rows=8, max_vocab=1024)
    try:
        def go(x, **kw):
            pw, w = torch.zeros((G, KV, P), device="cuda"), torch.zeros((G * W, KV, N), device="cuda")
            out = s.prefix_attention(x["q"], x["prefix_keys"], x["prefix_values"], x["keys"], x["values"], lengths=x["lengths"],
                                     prefix_weight=pw, weight=w, **kw)
            s.sync()
            return out, pw, w

        every, some, as_bytes = go(x), go(x, counted=counted), go(x, counted=counted.to(torch.uint8) * 5)
        assert torch.equal(some[0], every[0]) and all(torch.equal(a, b) for a, b in zip(some, as_bytes))
        assert torch.equal(some[2][counted], every[2][counted]) and not bool(some[2][~counted].any())
        o = oracle(torch, x)
        pw = torch.zeros_like(o["pw"])
        for r in counted.nonzero().view(-1).tolist():
            y = {k: v[r // W:r // W + 1] if k.startswith("prefix") else v[r:r + 1] for k, v in x.items()}
            pw[r // W] += oracle(torch, y)["pw"][0]
        near(torch, some[1], pw, o["tpw"], "prefix_weight")
        poisoned = dict(x, q=x["q"].clone())
        poisoned["q"][~counted] = float("nan")
        got = go(poisoned, counted=counted)
        assert torch.equal(got[1], some[1]) and torch.equal(got[2], some[2])
        assert not bool(go(x, counted=torch.zeros_like(counted))[1].any())
        assert all(torch.equal(a, b) for a, b in zip(go(x, counted=torch.ones_like(counted)), every))
    finally:
        s.close()
