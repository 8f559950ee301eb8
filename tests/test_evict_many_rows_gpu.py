"""mxs_cache_evict over many long rows at once (all layers of a long document),
where each row has a workgroup of its own: against the rule, which a stable sort
states.  All results are moved values, so they are equal."""
import pytest

from test_evict_gpu import inputs, rule, sampler, say, torch_mod  # noqa: F401

pytestmark = pytest.mark.gpu


def source_of(torch, w, index, lengths, n, first, recent):
    """Where each slot takes its content from and whether it is in use
    afterwards, both of w's shape (no NaN among the weights)."""
    C = w.shape[3]
    slot = torch.arange(C, device="cuda")
    length = lengths.long()[None, :, None, None].clamp(0, C)
    used = (slot < length).expand_as(w)
    newest = torch.where(used, index, -1).amax(-1, keepdim=True)
    anyway = (index < first) | (index > newest - recent)
    key = torch.where(used, torch.where(anyway, float("inf"), w.double()), -float("inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(used).scatter_(-1, order[..., :n], True) & used
    kept = torch.where(length <= n, used, kept)
    source = slot.expand_as(w).clone()
    for r in range(w[..., 0].numel()):
        k = kept.view(-1, C)[r]
        free, late = (~k[:n]).nonzero().view(-1), n + k[n:].nonzero().view(-1)
        source.view(-1, C)[r, free[: len(late)]] = late
    return source, (slot < length.clamp(max=n)).expand_as(w)


def test_the_sorted_rule_is_the_rule(torch_mod):  # noqa: F811
    torch = torch_mod
    _, _, w, index = inputs(torch, 2, 3, 2, 40, 1, seed=4)
    lengths = torch.tensor([40, 25, 9], device="cuda")
    source, _ = source_of(torch, w, index, lengths, 17, 3, 5)
    for l in range(2):
        for s, used in enumerate(lengths.tolist()):
            for h in range(2):
                want = rule(w[l, s, h, :used].tolist(), index[l, s, h, :used].tolist(), 17, 3, 5)
                assert source[l, s, h, : len(want)].tolist() == want


@pytest.mark.parametrize("ties", [0.0, 4.0, 0.02], ids=["distinct", "ties", "nearly-equal"])
@pytest.mark.parametrize("L,S,H,C,lengths,n,first,recent", [
    (9, 2, 8, 40000, [40000, 39990], 9000, 4, 600), (43, 3, 1, 33000, [33000, 500, 32790], 32000, 0, 0),
    (66, 1, 4, 32769, [32769], 32768, 4, 256), (17, 1, 8, 70001, [69999], 3, 1, 1)])
@pytest.mark.parametrize("indexed", [False, True])
def test_many_long_rows(torch_mod, sampler, ties, L, S, H, C, lengths, n, first, recent, indexed):  # noqa: F811
    torch = torch_mod
    assert L * S * H > 128 and C > 32768
    say(f"many long rows {L} {S} {H} {C} {n} {ties} {indexed}")
    keys, values, w, index = inputs(torch, L, S, H, C, 8, seed=C, ties=ties)
    if not indexed:
        index = torch.arange(C, dtype=torch.int32, device="cuda").expand(L, S, H, C).contiguous()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    source, inside = source_of(torch, w, index, lens, n, first, recent)
    k0, v0 = [t.clone() for t in keys], [t.clone() for t in values]
    out = sampler.cache_evict(keys, values, w, n, index=index if indexed else None, lengths=lens, keep_first=first, keep_recent=recent)
    sampler.sync()
    assert out.lengths.tolist() == [min(v, n) for v in lengths]
    assert torch.equal(out.weight, torch.where(inside, w.gather(3, source), 0.0))
    assert torch.equal(out.index, torch.where(inside, index.gather(3, source), -1))
    slot = torch.arange(C, device="cuda")
    for l in range(L):
        at = torch.where(inside[l], source[l], slot)[..., None]
        for now, before in ((keys[l], k0[l]), (values[l], v0[l])):
            assert torch.equal(now.view(torch.int16), before.gather(2, at.expand_as(before)).view(torch.int16)), f"layer {l}"
