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
