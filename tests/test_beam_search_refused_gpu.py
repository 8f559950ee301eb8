"""A step that a search refuses leaves its scores, flags, tokens, lengths, states
and result as they were, whichever check refuses it: compared right after the
refusal, with no accepted step in between."""
import pytest

pytestmark = pytest.mark.gpu

G, W, V, T, END = 2, 3, 40, 5, 3


@pytest.fixture(scope="module")
def torch_mod():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


class Run:
    """A search some steps on, with one state."""

    def __init__(self, torch, steps, **kw):
        from metallix_amd import BeamSearch, Sampler

        self.torch = torch
        self.s = Sampler(max_rows=G * W, max_vocab=V)
        self.search = BeamSearch(self.s, G, W, T, **kw)
        self.g = torch.Generator(device="cuda").manual_seed(17)
        self.state = torch.arange(G * W * 5, dtype=torch.float32, device="cuda").view(G * W, 5).clone()
        for _ in range(steps):
            lg = self.logits()
            lg[:, END] += 3.0
            self.search.step(lg, [self.state])

    def logits(self, stride=V):
        lg = self.torch.zeros((G * W, stride), device="cuda")[:, :V]
        lg.copy_(self.torch.randn((G * W, V), generator=self.g, device="cuda"))
        return lg

    def seen(self):
        c = self.search
        self.s.sync()
        p = c.picked
        return (c.result(), c.steps, c.done(), *(t.cpu().tolist() for t in
                (c.score, c.ended, c.length, c.tokens, p.token, p.beam, p.status, self.state)))

    def refuses(self, error, match, logits, states=None, **kw):
        before = self.seen()
        with pytest.raises(error, match=match):
            self.search.step(logits, [self.state] if states is None else states, **kw)
        assert self.seen() == before


@pytest.fixture(params=[(0, {}), (1, {}), (2, dict(end_token=END)), (3, dict(end_token=END, length_penalty=0.7))],
                ids=["first", "second", "ended", "penalty"])
def run(torch_mod, request):
    r = Run(torch_mod, request.param[0], **request.param[1])
    yield r
    r.s.close()


def test_logits_that_the_selection_refuses(run):
    from metallix_amd import SamplerError

    torch = run.torch
    run.refuses(SamplerError, "multiple of 4", run.logits(V + 2))
    run.refuses(SamplerError, "aligned", torch.zeros((G * W, V + 4), device="cuda")[:, 1 : V + 1])
    run.refuses(SamplerError, "legal_norm", run.logits(), legal_norm=True)
    run.refuses(SamplerError, "max_vocab", torch.zeros((G * W, V + 4), device="cuda"))
    run.refuses(ValueError, "logits", run.logits()[:-1])
    run.refuses(ValueError, "mask", run.logits(), mask=run.state)
    run.refuses(ValueError, "vocab", run.logits(), vocab=V + 1)
