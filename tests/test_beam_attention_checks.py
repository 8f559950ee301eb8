"""What BeamSearch.attention hands to the sampler and what it refuses, without a
GPU: a search whose sampler only writes down what it is asked for."""
import contextlib
import types

import pytest
import torch

from metallix_amd import BeamSearch

BF, I32 = torch.bfloat16, torch.int32
G, W, H, KV, D, P, N = 2, 3, 4, 2, 16, 20, 6


class Recorder:
    """Stands in for a Sampler: notes each prefix_attention call."""

    def __init__(self):
        cuda = types.SimpleNamespace(stream=lambda s: contextlib.nullcontext(), is_current_stream_capturing=lambda: False)
        t = {n: getattr(torch, n) for n in ("full", "zeros", "empty", "arange", "int32", "bool", "float64")}
        self.torch = types.SimpleNamespace(cuda=cuda, device=lambda *a: torch.device("cpu"), **t)
        self.stream, self.device, self.calls = None, 0, []

    def prefix_attention(self, q, *caches, **kw):
        self.calls.append((q, caches, kw))
        return q


def search(steps=2, max_new=5):
    s = BeamSearch(Recorder(), G, W, max_new)
    s.steps = steps
    s.score.zero_()
    return s


def args(groups=G):
    return (torch.zeros(G * W, H, D, dtype=BF), torch.zeros(groups, KV, P, D, dtype=BF), torch.zeros(groups, KV, P, D, dtype=BF),
            torch.zeros(G * W, KV, N, D, dtype=BF), torch.zeros(G * W, KV, N, D, dtype=BF))


@pytest.mark.parametrize("groups", [0, 1, 3, G * W])
def test_prompts_of_another_number_of_groups_are_refused(groups):
    """(one prompt, or one for each sequence, would be read by the wrong groups without an error)"""
    s = search()
    with pytest.raises(ValueError, match="prefix_keys"):
        s.attention(*args(groups))
    q, pk, _, k, v = args()
    with pytest.raises(ValueError, match="prefix_values"):
        s.attention(q, pk, torch.zeros(groups, KV, P, D, dtype=BF), k, v)
    assert not s.sampler.calls
    s.attention(*args())
    assert len(s.sampler.calls) == 1


@pytest.mark.parametrize("i", range(5))
@pytest.mark.parametrize("bad", [None, torch.zeros((), dtype=BF), torch.zeros(0, KV, P, D, dtype=BF)], ids=["none", "scalar", "empty"])
def test_arguments_that_are_missing_or_have_no_rows(i, bad):
    a = list(args())
    a[i] = bad
    s = search()
    with pytest.raises(ValueError, match=("q", "prefix_keys", "prefix_values", "keys", "values")[i]):
        s.attention(*a)
    assert not s.sampler.calls


def test_each_step_has_lengths_of_its_own():
    """A call that is captured, and so runs later or again, keeps its step's lengths."""
    s = search(steps=0, max_new=4)
    s.sampler.calls.clear()
    for s.steps in (1, 2, 2, 4):
        s.attention(*args())
    for (_, _, kw), n in zip(s.sampler.calls, (1, 2, 2, 4)):
        assert kw["lengths"].tolist() == [n] * (G * W) and kw["lengths"].dtype == I32 and kw["lengths"].is_contiguous()


def test_own_lengths():
    """Own caches that were evicted hold fewer positions than there were steps."""
    s = search(steps=5)
    q, pk, pv, k, v = args()
    own = torch.tensor([4] * (G * W), dtype=I32)
    s.attention(q, pk, pv, k[:, :, :4], v[:, :, :4], lengths=own)
    assert s.sampler.calls[-1][2]["lengths"] is own
    with pytest.raises(ValueError, match="5 positions"):
        s.attention(q, pk, pv, k[:, :, :4], v[:, :, :4])


def test_only_live_sequences_count():
    """Rows whose sequence has ended, or that hold none, add no weights."""
    s = search(steps=3)
    s.ended[0, 1] = True
    s.score[1, 2], s.score[1, 0] = float("-inf"), float("nan")
    w, pw = torch.zeros(G * W, KV, N), torch.zeros(G, KV, P)
    s.attention(*args())
    assert s.sampler.calls[-1][2].get("counted") is None   # (no weights: nothing to count)
    for kw in (dict(weight=w), dict(prefix_weight=pw), dict(weight=w, prefix_weight=pw)):
        s.attention(*args(), **kw)
        assert s.sampler.calls[-1][2]["counted"].tolist() == [True, False, True, False, True, False]
    first = s.sampler.calls[-1][2]["counted"]
    s.steps, s.ended[0, 0] = 4, True
    s.attention(*args(), weight=w)
    assert s.sampler.calls[-1][2]["counted"].tolist() == [False, False, True, False, True, False]
    assert first.tolist() == [True, False, True, False, True, False]
    # captured: looked at when it is replayed, so worked out in the graph, each time
    s.sampler.torch.cuda.is_current_stream_capturing = lambda: True
    s.attention(*args(), weight=w)
    s.attention(*args(), weight=w)
    a, b = (c[2]["counted"] for c in s.sampler.calls[-2:])
    assert a.tolist() == b.tolist() and a.data_ptr() != b.data_ptr()
    every = torch.ones(G * W, dtype=torch.bool)
    s.attention(*args(), weight=w, counted=every)
    assert s.sampler.calls[-1][2]["counted"] is every
