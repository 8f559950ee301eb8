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


def test_states_that_the_move_refuses(run):
    """Layouts that only the move's own checks look at: they are refused before
    the selection has written over the scores."""
    from metallix_amd import SamplerError

    torch = run.torch
    rows = G * W
    z = lambda *n: torch.zeros(n, device="cuda")
    run.refuses(SamplerError, "overlap", run.logits(), [run.state, z(1, 4).expand(rows, 4)])
    run.refuses(SamplerError, "overlap", run.logits(), [z(rows + 3).unfold(0, 4, 1), run.state])
    run.refuses(SamplerError, "overlap", run.logits(), [z(rows, 1, 4).expand(rows, 3, 4)], length_dim=2)
    run.refuses(SamplerError, "overlap", run.logits(), [run.state] * 1 + [z(rows, 9).unfold(1, 4, 1)])
    run.refuses(ValueError, "rows", run.logits(), [run.state[:-1]])
    run.refuses(ValueError, "lengths", run.logits(), lengths=z(G))


def test_a_move_is_refused_where_it_is_described(torch_mod):
    """The launcher refuses what its calls would, before the first of them."""
    from metallix_amd import Sampler, SamplerError

    torch = torch_mod
    s = Sampler(max_rows=G * W, max_vocab=V)
    parent = torch.zeros((G, W), dtype=torch.int32, device="cuda")
    with pytest.raises(SamplerError, match="overlap"):
        s.reorder_launcher([torch.zeros((1, 4), device="cuda").expand(G * W, 4)], parent)
    with pytest.raises(SamplerError, match="one state"):
        s.reorder_launcher([], parent)
    with pytest.raises(SamplerError, match="65535"):
        s.reorder_launcher([torch.zeros((1 << 16, 1), device="cuda")], torch.zeros((1 << 16, 1), dtype=torch.int32, device="cuda"))
    s.close()


def test_rules_that_are_the_searchs_own(run):
    """An end token, ended beams or a scale given to one step would disagree
    with the search's flags and lengths."""
    torch = run.torch
    run.refuses(ValueError, "end_token", run.logits(), end_token=1)
    run.refuses(ValueError, "ended", run.logits(), ended=torch.zeros((G, W), dtype=torch.bool, device="cuda"))
    if run.search.length_penalty:
        run.refuses(ValueError, "scale", run.logits(), scale=torch.ones((G, W), dtype=torch.float64, device="cuda"))
