"""The cache operators together, as a search uses them: a small decoder whose
sequences attend to their prompt's shared cache and to their own, with the
weights accumulating; the own caches and weights move with the beams; the
prompt's cache is brought down to a budget on the way.  Every attention is
checked against the definition over the caches as they then are."""
import pytest

from test_attention_gpu import near, oracle
from test_evict_gpu import rule

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_mod():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.mark.parametrize("G,W,H,KV,D,P,end", [(2, 3, 4, 2, 64, 50, None), (3, 5, 6, 1, 80, 90, 7), (1, 16, 8, 2, 128, 200, 7)])
def test_search_with_attention(torch_mod, G, W, H, KV, D, P, end):
    torch = torch_mod
    from metallix_amd import BeamSearch, Sampler

    V, T, E, n = 500, 7, 64, 24
    rows, per = G * W, H // KV
    s = Sampler(max_rows=rows, max_vocab=V)
    g = torch.Generator(device="cuda").manual_seed(G)
    r = lambda *d: torch.randn(d, generator=g, device="cuda")
    bf = lambda *d: r(*d).to(torch.bfloat16)
    embed, wq, wk, wv = bf(V, E), bf(H * D, E), bf(KV * D, E), bf(KV * D, E)
    head = (r(V, H * D) * (H * D) ** -0.5 * 3).to(torch.bfloat16)
    pk, pv = bf(G, KV, P, D), bf(G, KV, P, D)
    plen = torch.tensor([P - 3 * i for i in range(G)], dtype=torch.int32, device="cuda")
    index = torch.arange(P, dtype=torch.int32, device="cuda").expand(1, G, KV, P).contiguous()
    pw = torch.zeros((G, KV, P), device="cuda")
    keys, values = (torch.zeros((rows, KV, T, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    w = torch.zeros((rows, KV, T), device="cuda")
    search = BeamSearch(s, G, W, T, end_token=end)
    with pytest.raises(ValueError, match="first step"):
        search.attention(bf(rows, H, D), pk, pv, keys, values)
    tok = search.step(r(rows, V) * 3.0, [keys, values, w])
    for t in range(1, T):
        h = embed[tok.clamp(min=0).long()]
        q = s.linear(h, wq).view(rows, H, D)
        keys[:, :, t - 1] = s.linear(h, wk).view(rows, KV, D)
        values[:, :, t - 1] = s.linear(h, wv).view(rows, KV, D)
        pw0, w0 = pw.clone(), w.clone()
        lse = torch.empty((rows, H), device="cuda")
        out = search.attention(q, pk, pv, keys, values, prefix_lengths=plen, prefix_weight=pw, weight=w, lse=lse, scale=0.02)
        x = dict(q=q[:, None], prefix_keys=pk, prefix_values=pv, keys=keys, values=values, prefix_lengths=plen,
                 lengths=torch.full((rows,), t, device="cuda"))
        o = oracle(torch, x, 0.02)
        s.sync()
        near(torch, out[:, None], o["out"], o["tout"], f"step {t}: out")
        near(torch, lse[:, None], o["lse"], o["tlse"], f"step {t}: lse")
        near(torch, pw, pw0.double() + o["pw"], o["tpw"] + (pw0 + 1).double() * 2.0 ** -23, f"step {t}: prefix_weight")
        near(torch, w, w0.double() + o["w"], o["tw"] + (w0 + 1).double() * 2.0 ** -23, f"step {t}: weight")
        if t in (2, 4):   # the prompt's cache down to n, then to n - 5
            budget = n if t == 2 else n - 5
            k0, i0, used = pk.clone(), index.clone(), plen.tolist()
            e = s.cache_evict([pk], [pv], pw[None], budget, index=index, lengths=plen, keep_first=2, keep_recent=4)
            s.sync()
            for a in range(G):
                for k in range(KV):
                    src = rule(pw[a, k].tolist()[: used[a]], index[0, a, k].tolist()[: used[a]], budget, 2, 4)
                    assert e.index[0, a, k].tolist() == [int(i0[0, a, k, i]) for i in src] + [-1] * (P - len(src))
                    assert torch.equal(pk[a, k, : len(src)], k0[a, k, src])
            pw, index, plen = e.weight[0].contiguous(), e.index, e.lengths
        logits = s.linear(out.view(rows, H * D), head, out_dtype=torch.float32)
        before = [v.clone() for v in (keys, values, w)]
        tok = search.step(logits, [keys, values, w])
        s.sync()
        parent = (search.picked.beam.long() + torch.arange(G, device="cuda")[:, None] * W).view(-1)
        there = search.picked.beam.view(-1) >= 0
        for now, old in zip((keys, values, w), before):
            assert torch.equal(now[there], old[parent[there]])
    assert search.status() == [0] * G
    for bad in (dict(q=q[:1]), dict(keys=keys[:, :, :1]), dict(lengths=plen)):
        kw = dict(dict(q=q, keys=keys), **bad)
        with pytest.raises(ValueError):
            search.attention(kw.pop("q"), pk, pv, kw.pop("keys"), values, **kw)
    s.close()
