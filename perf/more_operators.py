"""The work of sequences that share a prompt, and of a cache that is kept within a budget, as measurable cases.

Each case is one pass through one operator, over inputs made on the GPU from a
seed:

  attend   one layer's attention of groups of sequences (beams, choices,
           drafts): every query over its group's shared prefix and its own
           suffix, where asked for with the weight that each position got
           added to its accumulated one
  evict    caches brought down to a budget of positions: the newest, the first
           and those with the largest accumulated weights stay, and what stays
           behind the budget moves into the slots that became free

`run` computes a case in plain torch operations, or, where `own` is true,
through the package's entry points.  `exact` restates attention in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

MOST_FLOPS = 4 * 8 * 512 * 32768 * 128      # of a drawn attention
MOST_SCORES = 8 * 512 * 32768               # query rows times positions
MOST_CACHE = 2 * 8 * 131072 * 128 * 2       # bytes of keys and values
MOST_EVICT = 2 * 28 * 8 * 8192 * 128 * 2    # bytes of keys and values of a drawn eviction


def listed():
    return [
        # One interactive request decoded with 4 beams early in its answer: latency.
        dict(name="attend_one", kind="attend", groups=1, beams=4, tokens=1, heads=16, kv=8, dim=128, prefix=512,
             suffix=48, weights=False),
        # A serving batch of 8 requests of 4 beams, prompts of different lengths up to 4096 tokens.
        dict(name="attend_serve", kind="attend", groups=8, beams=4, tokens=1, heads=32, kv=8, dim=128, prefix=4096,
             suffix=128, weights=False),
        # Drafts of 6 tokens scored for 5 requests of 3 sequences; odd sizes.
        dict(name="attend_drafts", kind="attend", groups=5, beams=3, tokens=6, heads=15, kv=5, dim=80, prefix=1999,
             suffix=77, weights=False),
        # A long document, 4 answers sampled at once: the stream of its cache.
        dict(name="attend_long", kind="attend", groups=1, beams=4, tokens=1, heads=32, kv=8, dim=128, prefix=131072,
             suffix=256, weights=False),
        # The largest: 64 sequences on one prompt, 512 queries for each head of the cache.
        dict(name="attend_many", kind="attend", groups=1, beams=64, tokens=1, heads=64, kv=8, dim=128, prefix=32768,
             suffix=200, weights=False),
        # The serving batch while weights accumulate for a later eviction.
        dict(name="weigh_serve", kind="attend", groups=8, beams=4, tokens=1, heads=32, kv=8, dim=128, prefix=4096,
             suffix=128, weights=True),
        # 16 sequences on a prompt of 16384 tokens, heads of 64, weights accumulating.
        dict(name="weigh_many", kind="attend", groups=1, beams=16, tokens=1, heads=32, kv=8, dim=64, prefix=16384,
             suffix=64, weights=True),
        # A full cache after each token of one request, 28 layers: one position goes.  Latency.
        dict(name="evict_token", kind="evict", layers=28, segments=1, heads=8, capacity=1040, length=1025, budget=1024,
             dim=128, first=4, recent=256, again=True),
        # After the prompt: 8192 positions of 28 layers to 2048.
        dict(name="evict_prompt", kind="evict", layers=28, segments=1, heads=8, capacity=8192, length=8192, budget=2048,
             dim=128, first=4, recent=512, again=False),
        # A batch of 7 caches of different lengths, some within the budget; odd sizes.
        dict(name="evict_batch", kind="evict", layers=5, segments=7, heads=3, capacity=2500, length=2411, budget=1333,
             dim=80, first=1, recent=77, again=True),
        # A long document's caches, two layers at a time: 131072 positions to 16384.
        dict(name="evict_long", kind="evict", layers=2, segments=1, heads=8, capacity=131072, length=131072,
             budget=16384, dim=128, first=4, recent=1024, again=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dim = rng.choice([40, 64, 80, 96, 128, 128, 128, 192, 256])
    if rng.random() < 0.65:
        groups, beams, kv = _log_int(rng, 1, 16), _log_int(rng, 1, 64), rng.choice([1, 2, 3, 4, 8, 8, 16])
        tokens, per = rng.choice([1, 1, 1, 1, rng.randint(2, 8)]), rng.randint(1, 8)
        most = min(MOST_FLOPS // (4 * dim), MOST_SCORES) // (groups * kv * beams * tokens * per)
        most = min(most, MOST_CACHE // (4 * groups * kv * dim))
        suffix = rng.choice([0, tokens + _log_int(rng, 1, 500), tokens + _log_int(rng, 1, 100)])
        suffix = min(suffix, most // 2, MOST_CACHE // (8 * groups * beams * kv * dim))
        prefix = max(1, min(_log_int(rng, 1, 131072), most - suffix * beams))
        return dict(kind="attend", groups=groups, beams=beams, tokens=tokens, heads=kv * per, kv=kv, dim=dim,
                    prefix=prefix, suffix=suffix, weights=rng.random() < 0.4)
    layers, segments, heads = _log_int(rng, 1, 28), _log_int(rng, 1, 8), rng.randint(1, 8)
    length = max(8, min(_log_int(rng, 8, 131072), MOST_EVICT // (4 * layers * segments * heads * dim) - 8))
    budget = rng.choice([length - 1, rng.randint(1, length - 1), _log_int(rng, 1, length - 1)])
    first = rng.randint(0, min(4, budget // 2))
    return dict(kind="evict", layers=layers, segments=segments, heads=heads, capacity=length + rng.choice([0, 1, 7]),
                length=length, budget=budget, dim=dim, first=first, recent=rng.randint(0, budget // 2),
                again=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# Inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 2654435761 + 12345) % (1 << 62))
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _uniform(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _falling(most, count):
    """`count` lengths that fall from `most` towards half of it."""
    return most - torch.arange(count, device="cuda") * most // (2 * count)


def _prepare_attend(case, seed):
    """Caches [segments, kv heads, positions, dim] in bf16.  The queries of a
    head share a direction that the prefix's first key has too, which so takes
    a large share of most rows' weight, as first tokens do.  Prefixes fall from
    their full length to half of it, suffixes to their last tokens."""
    g = _gen(seed)
    G, W, T, H, KV, D = (case[k] for k in ("groups", "beams", "tokens", "heads", "kv", "dim"))
    P, N, bf = case["prefix"], case["suffix"], torch.bfloat16
    common = _normal(g, KV, D)
    q = 1.3 * _normal(g, G * W, T, KV, H // KV, D) + 0.6 * common[:, None]
    keys, values = torch.empty((2, G, KV, P, D), dtype=bf, device="cuda").unbind(0)
    keys.copy_(_normal(g, G, KV, P, D))
    keys[:, :, 0] = (common * 1.2).to(bf)
    values.copy_(_normal(g, G, KV, P, D))
    s = dict(case=case, q=q.view(G * W, T, H, D).to(bf), prefix_keys=keys, prefix_values=values,
             prefix_lengths=_falling(P, G)[torch.argsort(_uniform(g, G))].to(torch.int32))
    if N:
        s["keys"], s["values"] = _normal(g, G * W, KV, N, D).to(bf), _normal(g, G * W, KV, N, D).to(bf)
        s["lengths"] = torch.clamp(_falling(N, G * W), min=min(T, N))[torch.argsort(_uniform(g, G * W))].to(torch.int32)
    if case["weights"]:   # what earlier steps have added
        s["prefix_weight"] = torch.exp(2.0 * _normal(g, G, KV, P))
        if N:
            s["weight"] = torch.exp(_normal(g, G * W, KV, N))
    return s


def _prepare_evict(case, seed):
    """Accumulated weights over some orders of magnitude, rounded so that the
    small ones are often equal; after earlier evictions the positions lie in no
    order."""
    g = _gen(seed)
    L, S, H, C, D = (case[k] for k in ("layers", "segments", "heads", "capacity", "dim"))
    cache = torch.empty((2, L, S, H, C, D), dtype=torch.bfloat16, device="cuda")
    for part in cache.view(2 * L, S, H, C, D):
        part.copy_(_normal(g, S, H, C, D))
    weight = torch.round(torch.exp(2.5 * _normal(g, L, S, H, C)) * 64.0) / 64.0
    index = torch.arange(C, dtype=torch.int32, device="cuda").expand(L, S, H, C).contiguous()
    if case["again"]:
        index = torch.argsort(_uniform(g, L, S, H, C), -1).to(torch.int32)
    lengths = _falling(case["length"], S)[torch.argsort(_uniform(g, S))].to(torch.int32)
    return dict(case=case, keys=cache[0], values=cache[1], weight=weight, index=index, lengths=lengths)


def prepare(case, seed):
    return {"attend": _prepare_attend, "evict": _prepare_evict}[case["kind"]](case, seed)


# ---------------------------------------------------------------------------
# The plain forms

def _scores(q, keys, seen):
    """q [B, M, D] over keys [B, P, D], -inf where not seen ([B, M, P])."""
    x = torch.matmul(q, keys.transpose(1, 2)) * q.shape[-1] ** -0.5
    return x.masked_fill(~seen, -math.inf)


def _plain_attend(s):
    case = s["case"]
    G, W, T, H, KV, D = (case[k] for k in ("groups", "beams", "tokens", "heads", "kv", "dim"))
    P, N, per = case["prefix"], case["suffix"], H // KV
    q = s["q"].float().view(G, W, T, KV, per, D)
    at = torch.arange(P, device="cuda")
    seen = (at < s["prefix_lengths"][:, None]).repeat_interleave(KV, 0)[:, None]
    qp = q.permute(0, 3, 1, 2, 4, 5).reshape(G * KV, W * T * per, D)
    x = _scores(qp, s["prefix_keys"].float().view(G * KV, P, D), seen)
    # [G * KV, W * T * per] and [G * W * KV, T * per] and back
    own_rows = lambda v: v.view(G, KV, W, T * per, -1).transpose(1, 2).reshape(G * W * KV, T * per, -1)
    all_rows = lambda v: v.view(G, W, KV, T * per, -1).transpose(1, 2).reshape(G * KV, W * T * per, -1)
    top = x.amax(2, keepdim=True)
    if N:
        # token t of the T newest sees the suffix up to itself
        last = s["lengths"][:, None] - T + torch.arange(T, device="cuda") + 1
        seen = (torch.arange(N, device="cuda") < last[:, :, None]).repeat_interleave(per, 1).repeat_interleave(KV, 0)
        y = _scores(own_rows(qp), s["keys"].float().view(G * W * KV, N, D), seen)
        top = torch.maximum(top, all_rows(y.amax(2, keepdim=True)))
    top = top.clamp_(min=-1e30)   # (a row that sees nothing)
    x = torch.exp(x - top)
    total = x.sum(2, keepdim=True)
    out = torch.matmul(x, s["prefix_values"].float().view(G * KV, P, D))
    if N:
        y = torch.exp(y - own_rows(top))
        total = total + all_rows(y.sum(2, keepdim=True))
        out = out + all_rows(torch.matmul(y, s["values"].float().view(G * W * KV, N, D)))
    share = 1.0 / torch.where(total > 0, total, 1.0)
    rows = lambda v: v.view(G, KV, W, T, per, -1).permute(0, 2, 3, 1, 4, 5).reshape(G * W, T, H, -1)
    res = dict(out=rows(out * share).to(torch.bfloat16), lse=rows(top + torch.log(total))[..., 0])
    if case["weights"]:
        s["prefix_weight"] += torch.matmul(share.transpose(1, 2), x).view(G, KV, P)
        res["prefix_weight"] = s["prefix_weight"]
        if N:
            s["weight"] += torch.matmul(own_rows(share).transpose(1, 2), y).view(G * W, KV, N)
            res["weight"] = s["weight"]
    return res


def _plain_evict(s):
    case = s["case"]
    L, S, H, C, D, n = (case[k] for k in ("layers", "segments", "heads", "capacity", "dim", "budget"))
    weight, index = s["weight"].view(-1, C), s["index"].view(-1, C)
    length = s["lengths"][None, :, None].expand(L, S, H).reshape(-1, 1)
    slot = torch.arange(C, device="cuda")
    used = slot < length
    newest = torch.where(used, index, -1).amax(1, keepdim=True)
    kept_anyway = (index < case["first"]) | (index > newest - case["recent"])
    key = torch.where(kept_anyway, math.inf, weight.double())
    order = torch.sort(torch.where(used, key, -math.inf), dim=1, descending=True, stable=True).indices
    kept = torch.zeros_like(used).scatter_(1, order[:, :n], True) & used
    room = torch.clamp(length, max=n)
    free, late = ~kept & (slot < room), kept & (slot >= n)
    # the j-th free slot takes what the j-th late one holds
    table = torch.zeros((weight.shape[0], n + 1), dtype=torch.int64, device="cuda")
    table.scatter_(1, torch.where(late, torch.cumsum(late, 1) - 1, n), slot.expand_as(late))
    table[:, n] = 0
    source = torch.where(free, table.gather(1, (torch.cumsum(free, 1) - 1).clamp(0, n)), slot)[:, :n]
    inside = used[:, :n]
    moved = lambda v, none: torch.cat([torch.where(inside, v.gather(1, source), none),
                                       torch.full_like(v[:, n:], none)], 1).view(L, S, H, C)
    rows = source[:, :, None].expand(-1, -1, D)
    keys, values = s["keys"].view(-1, C, D), s["values"].view(-1, C, D)
    keys[:, :n] = keys.gather(1, rows)
    values[:, :n] = values.gather(1, rows)
    return dict(keys=s["keys"], values=s["values"], weight=moved(weight, 0.0), index=moved(index, -1),
                lengths=torch.clamp(s["lengths"], max=n))


# ---------------------------------------------------------------------------
# The framework's calls

_handle = []


def _sampler():
    """The program's one sampler context, made at its first call."""
    if not _handle:
        from metallix_amd import Sampler

        _handle.append(Sampler(max_rows=64, max_vocab=4096))
    return _handle[0]


def _own_attend(s):
    call = s.get("call")
    if call is None:
        c = s["case"]
        s["lse"] = torch.empty((c["groups"] * c["beams"], c["tokens"], c["heads"]), device="cuda")
        call = s["call"] = _sampler().prefix_attention_launcher(
            s["q"], s["prefix_keys"], s["prefix_values"], s.get("keys"), s.get("values"),
            prefix_lengths=s["prefix_lengths"], lengths=s.get("lengths"), lse=s["lse"],
            prefix_weight=s.get("prefix_weight"), weight=s.get("weight"))
    call()
    res = dict(out=call.out, lse=s["lse"])
    res.update({k: s[k] for k in ("prefix_weight", "weight") if k in s})
    return res


def _own_evict(s):
    call = s.get("call")
    if call is None:
        c = s["case"]
        call = s["call"] = _sampler().cache_evict_launcher(
            list(s["keys"]), list(s["values"]), s["weight"], c["budget"], index=s["index"], lengths=s["lengths"],
            keep_first=c["first"], keep_recent=c["recent"])
    call()
    o = call.out
    return dict(keys=s["keys"], values=s["values"], weight=o.weight, index=o.index, lengths=o.lengths)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attend": _own_attend, "evict": _own_evict}[kind](state)
    return {"attend": _plain_attend, "evict": _plain_evict}[kind](state)


# ---------------------------------------------------------------------------

def _sum_falling(most, count):
    return sum(most - i * most // (2 * count) for i in range(count))


def work(case):
    if case["kind"] == "attend":
        G, W, T, H, KV, D = (case[k] for k in ("groups", "beams", "tokens", "heads", "kv", "dim"))
        prefix = _sum_falling(case["prefix"], G)                       # positions used, of all groups
        suffix = _sum_falling(case["suffix"], G * W) if case["suffix"] else 0
        small = G * W * T * H * (4 * D + 4) + (8 * KV * (prefix + suffix) if case["weights"] else 0)
        return {"bytes": 4 * KV * D * (prefix + suffix) + small, "flops": 4 * D * T * H * (W * prefix + suffix)}
    L, S, H, C, D, n = (case[k] for k in ("layers", "segments", "heads", "capacity", "dim", "budget"))
    moved, read = 0.0, 0
    for i in range(S):
        length = case["length"] - i * case["length"] // (2 * S)
        read += length
        if length > n:
            # the newest lie last (or anywhere, after earlier evictions); of the others each stays with the same chance
            others = max(1, length - case["first"] - case["recent"])
            stay = max(0, n - case["first"] - case["recent"]) / others
            late = length - n
            new = case["recent"] * (late / length if case["again"] else 1.0)
            moved += min(late, new) + stay * max(0.0, late - new)
    return {"bytes": L * H * (8 * read + 8 * S * C + 8 * D * moved), "flops": 0}


def exact(case, seed):
    """What run returns, from the definition in 64 bits, one head of the cache
    at a time.  An eviction's moved values are not computed numbers."""
    if case["kind"] == "evict":
        return None
    s = prepare(case, seed)
    G, W, T, H, KV, D = (case[k] for k in ("groups", "beams", "tokens", "heads", "kv", "dim"))
    P, N, per, f = case["prefix"], case["suffix"], H // KV, torch.float64
    out = torch.zeros((G * W, T, H, D), dtype=f, device="cuda")
    lse = torch.zeros((G * W, T, H), dtype=f, device="cuda")
    prefix_weight = s["prefix_weight"].to(f) if case["weights"] else None
    weight = s["weight"].to(f) if case["weights"] and N else None
    for g in range(G):
        used = int(s["prefix_lengths"][g])
        for h in range(KV):
            heads = slice(h * per, (h + 1) * per)
            pk, pv = s["prefix_keys"][g, h, :used].to(f), s["prefix_values"][g, h, :used].to(f)
            shared = torch.matmul(s["q"][g * W:(g + 1) * W, :, heads].to(f).reshape(-1, D), pk.t()) / math.sqrt(D)
            shared = shared.view(W, T * per, used)
            for b in range(W):
                r = g * W + b
                q = s["q"][r, :, heads].to(f)   # [T, per, D]
                x, v = shared[b].view(T, per, used), pv
                if N:
                    n = int(s["lengths"][r])
                    y = torch.matmul(q, s["keys"][r, h, :n].to(f).t()) / math.sqrt(D)
                    ahead = torch.arange(n, device="cuda")[None, None] > (n - T + torch.arange(T, device="cuda"))[:, None, None]
                    x, v = torch.cat([x, y.masked_fill(ahead, -math.inf)], 2), torch.cat([pv, s["values"][r, h, :n].to(f)])
                share = torch.softmax(x, 2)
                out[r, :, heads] = torch.matmul(share, v)
                lse[r, :, heads] = torch.logsumexp(x, 2)
                if case["weights"]:
                    total = share.sum((0, 1))
                    prefix_weight[g, h, :used] += total[:used]
                    if N:
                        weight[r, h, :n] += total[used:]
    res = dict(out=out, lse=lse)
    if case["weights"]:
        res["prefix_weight"] = prefix_weight
        if N:
            res["weight"] = weight
    return res
