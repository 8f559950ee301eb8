"""What a search gives back: its steps' tokens and its groups' outcomes."""
import pytest

pytestmark = pytest.mark.gpu

G, W, V, T, END = 3, 4, 60, 6, 5


@pytest.fixture(scope="module")
def torch_mod():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.fixture
def sampler(torch_mod):
    from metallix_amd import Sampler

    s = Sampler(max_rows=G * W, max_vocab=V)
    yield s
    s.close()


def logits(torch, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return 3.0 * torch.randn((G * W, V), generator=g, device="cuda")


def test_a_steps_tokens_stay_what_they_were(torch_mod, sampler):
    """A caller may keep the tensors that the steps return."""
    from metallix_amd import BeamSearch

    torch = torch_mod
    search = BeamSearch(sampler, G, W, T)
    kept, then = [], []
    for t in range(T):
        kept.append(search.step(logits(torch, t)))
        torch.cuda.synchronize()
        then.append(kept[-1].cpu())
        assert torch.equal(search.picked.token.view(-1).cpu(), then[-1])
    assert len({tuple(t.tolist()) for t in then}) == T   # the steps' tokens differ
    for k, w in zip(kept, then):
        assert torch.equal(k.cpu(), w)


@pytest.mark.parametrize("at", [0, 2, T - 1])
def test_what_stopped_a_group_is_kept(torch_mod, sampler, at):
    """A group whose logits hold a NaN at one step, and one left without a
    legal token, say so at the end; the third gives what it gives alone."""
    from metallix_amd import BeamSearch

    torch = torch_mod
    alone = BeamSearch(sampler, G, W, T, end_token=END)
    search = BeamSearch(sampler, G, W, T, end_token=END)
    mask = torch.full((G * W, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
    none = mask.clone()
    none[2 * W :] = 0
    for t in range(T):
        lg = logits(torch, 50 + t)
        lg[:, END] = -30.0                     # (no beam ends)
        alone.step(lg, mask=mask)
        if t == at:
            lg = lg.clone()
            lg[0, 7] = float("nan")
        search.step(lg, mask=none if t == at else mask)
        assert search.status() == ([0, 0, 0] if t < at else [-6, 0, -3]), t
    assert alone.status() == [0, 0, 0]
    want, got = alone.result(), search.result()
    assert got == [[], want[1], []] and len(want[1]) == W
    assert alone.done() is False


def test_a_search_on_a_stream_of_its_own(torch_mod):
    """What reads back waits for the steps, whatever stream is current."""
    from metallix_amd import BeamSearch, Sampler

    torch = torch_mod
    lgs = [logits(torch, 90 + t) for t in range(T)]
    lgs[3][W + 1, 9] = float("inf")            # group 1 stops
    torch.cuda.synchronize()
    found = []
    for stream in (None, torch.cuda.Stream()):
        s = Sampler(max_rows=G * W, max_vocab=V, stream=stream)
        search = BeamSearch(s, G, W, T, end_token=END, length_penalty=0.3)
        kept = [search.step(lg) for lg in lgs]
        found.append((search.status(), search.done(), search.result(), [k.cpu().tolist() for k in kept]))
        s.close()
    assert found[0] == found[1] and found[0][0] == [0, -6, 0]
