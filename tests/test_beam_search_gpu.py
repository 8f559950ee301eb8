"""The beam operators together, as a search uses them: a small recurrent
model whose block (mxs_linear_bf16 with bias, silu and residual) and biased
output projection give the logits of all beams, the selection, and the move of
the hidden states and of a cache that grows by one position a step."""
import numpy as np
import pytest

from test_beam_gpu import oracle, same

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_mod():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


class Toy:
    def __init__(self, torch, s, H, V, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *n: torch.randn(n, generator=g, device="cuda")
        bf = torch.bfloat16
        self.s = s
        self.embed = r(V, H).to(bf)
        self.w, self.b = (r(H, H) * H ** -0.5).to(bf), r(H).to(bf)
        self.head, self.hb = (r(V, H) * 2.5 * H ** -0.5).to(bf), r(V)

    def __call__(self, torch, h, tok):
        """New hidden states and the logits after `tok`."""
        x = h + self.embed[tok.clamp(min=0).long()]
        h = self.s.linear(x, self.w, self.b, activation="silu", residual=x)
        h = (h.float() / (1.0 + h.float().abs().amax(1, keepdim=True))).to(torch.bfloat16)
        return h, self.s.linear(h, self.head, self.hb, out_dtype=torch.float32)


@pytest.mark.parametrize("G,W,V,penalty", [(1, 4, 500, 0.0), (5, 3, 2003, 0.8), (24, 4, 999, 0.0)])
def test_search(torch_mod, G, W, V, penalty):
    torch = torch_mod
    from metallix_amd import BeamSearch, Sampler

    H, T, END = 64, 9, 7
    s = Sampler(max_rows=G * W, max_vocab=V)
    toy = Toy(torch, s, H, V, G)
    toy.hb[END] += 4.0                    # some beams end
    search = BeamSearch(s, G, W, T, end_token=END, length_penalty=penalty)
    rows = G * W
    h = torch.zeros((rows, H), dtype=torch.bfloat16, device="cuda")
    cache = torch.zeros((rows, 2, T, H // 2), dtype=torch.bfloat16, device="cuda")
    tok = torch.arange(rows, device="cuda") // W % V
    start = tok.clone()
    length = np.zeros((G, W), int)
    for t in range(T):
        h, lg = toy(torch, h, tok)
        cache[:, :, t] = h.view(rows, 2, H // 2)
        score, ended = search.score.cpu().numpy(), search.ended.cpu().numpy()
        n = np.where(ended, length, t + 1)
        scale = ((5.0 + n) / 6.0) ** -penalty if penalty else None
        vp = (V + 3) // 4 * 4
        lgp = torch.zeros((rows, vp), device="cuda")
        lgp[:, :V] = lg
        lengths = torch.full((G,), t + 1, dtype=torch.int32, device="cuda")
        tok = search.step(lgp[:, :V], [h, cache], lengths=lengths, length_dim=[None, 2])
        torch.cuda.synchronize()
        want = oracle(lg.cpu().numpy(), score, W, ended=ended, end_token=END, scale=scale)
        p = search.picked
        same([a.cpu().numpy() for a in (p.token, p.beam, p.score, p.ended, p.status)], want)
        length = np.take_along_axis(n, want[1], 1)
        assert search.moved.cpu().tolist() == [0] * G
    assert not search.done() or bool(search.ended.all())
    res = search.result()
    assert any(hyp.ended for g in res for hyp in g)
    # every hypothesis again, fed its own tokens row by row: the same scores and the same cached states
    h2 = torch.zeros_like(h)
    cur = start.clone()
    hist = search.tokens.cpu().numpy()
    total = np.zeros(rows)
    alive = np.ones(rows, bool)
    for t in range(T):
        h2, lg = toy(torch, h2, cur)
        lp = torch.log_softmax(lg.double(), 1).cpu().numpy()
        got = cache[:, :, t].reshape(rows, H)
        live = torch.from_numpy(alive).to("cuda")
        assert torch.equal(got[live], h2[live]), t
        total += np.where(alive, lp[np.arange(rows), hist[:, t]], 0.0)
        alive &= hist[:, t] != END
        cur = torch.from_numpy(hist[:, t].copy()).to("cuda")
    for g in range(G):
        assert len(res[g]) == W
        for b, hyp in enumerate(res[g]):
            r = g * W + b
            assert abs(hyp.score - total[r]) <= T * (2.0 ** -38 + 64 * 2.0 ** -50)
            k = hyp.tokens.index(END) + 1 if END in hyp.tokens else T
            assert hyp.tokens == hist[r, :k].tolist() and hyp.ended == (END in hyp.tokens)
            assert hist[r, k:].tolist() == [END] * (T - k)
    with pytest.raises(ValueError):
        search.step(lgp[:, :V])
    s.close()


def test_a_refused_step_leaves_the_search_as_it_was(torch_mod):
    """States or logits that do not fit raise before anything moves: the step
    with the right ones gives what a search without the mistakes gives."""
    torch = torch_mod
    from metallix_amd import BeamSearch, Sampler

    G, W, V, T = 2, 3, 40, 4
    s = Sampler(max_rows=G * W, max_vocab=V)
    g = torch.Generator(device="cuda").manual_seed(5)
    steps = [torch.randn((G * W, V), generator=g, device="cuda") for _ in range(T)]
    found = []
    for mistakes in (False, True):
        search = BeamSearch(s, G, W, T, end_token=3, length_penalty=0.5)
        state = torch.arange(G * W * 5, dtype=torch.float32, device="cuda").view(G * W, 5).clone()
        for lg in steps:
            if mistakes:
                for bad in (dict(states=[state[:-1]]), dict(states=[state, state]), dict(states=[state.cpu()]),
                            dict(states=[state], length_dim=[1, 1]), dict(states=[state], mask=state),
                            dict(states=[state], lengths=torch.zeros(G, device="cuda"))):
                    with pytest.raises(ValueError):
                        search.step(lg, **bad)
                with pytest.raises(ValueError):
                    search.step(lg[:-1], [state])
            search.step(lg, [state])
        found.append((search.result(), state.cpu()))
        with pytest.raises(ValueError):
            search.step(steps[0], [state])
    assert found[0][0] == found[1][0] and torch.equal(found[0][1], found[1][1])
    s.close()
