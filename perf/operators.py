"""The work of a beam search, and of the matrix products around it, as measurable cases.

Each case is one pass through one operator, over inputs made on the GPU from a
seed:

  select   one step's selection: every live beam's log-softmax, the n best of
           all (beam, token) candidates of a group by cumulative score
  reorder  the beams' states (key-value caches, recurrent states) moved to
           their children, in place
  linear   a bf16 matrix product with bias, activation and residual in its
           epilogue

`run` computes a case in plain torch operations, or, where `own` is true,
through the package's entry points.  `exact` restates them in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

VOCAB = 151936
LARGE_VOCAB = 262144
MOST_LOGITS = 256 * LARGE_VOCAB * 4       # bytes of logits a drawn selection takes at most
MOST_STATE = 56 * 32 * 8 * 520 * 128 * 2  # bytes of states
MOST_FLOPS = 2 * 8192 * 4096 * 14336
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def listed():
    return [
        # One interactive request decoded with 4 beams: latency.  Twice as many candidates as beams, so that
        # those that end leave enough.
        dict(name="select_one", kind="select", groups=1, beams=4, vocab=50257, dtype="f32", n=8, ended=False,
             mask=False, legal_norm=False, scale=False),
        # A serving batch of 16 requests with 4 beams each; ended beams stay in the race, scores divided by a
        # power of the length.
        dict(name="select_serve", kind="select", groups=16, beams=4, vocab=VOCAB, dtype="f32", n=4, ended=True,
             mask=False, legal_norm=False, scale=True),
        # Constrained decoding under grammar masks, bf16 logits, a ragged number of beams, probabilities over
        # the legal tokens.
        dict(name="select_grammar", kind="select", groups=7, beams=5, vocab=VOCAB, dtype="bf16", n=10, ended=False,
             mask=True, legal_norm=True, scale=False),
        # The largest batch: 16 requests of 16 beams over 262144 tokens.
        dict(name="select_wide", kind="select", groups=16, beams=16, vocab=LARGE_VOCAB, dtype="f32", n=32, ended=False,
             mask=False, legal_norm=False, scale=False),
        # The caches of that one request, early in its answer: 28 layers' keys and values.
        dict(name="reorder_one", kind="reorder", states=56, groups=1, beams=4, heads=8, positions=48, dim=128,
             dtype="bf16", lengths=True),
        # The caches of 8 requests of 4 beams, of different lengths up to 520 positions.
        dict(name="reorder_serve", kind="reorder", states=56, groups=8, beams=4, heads=8, positions=520, dim=128,
             dtype="bf16", lengths=True),
        # Recurrent states (f32, one matrix a head, no length) of 16 requests of 16 beams.
        dict(name="reorder_wide", kind="reorder", states=2, groups=16, beams=16, heads=16, positions=128, dim=128,
             dtype="f32", lengths=False),
        # A drafter's residual block for one token: x + silu(W x + b).
        dict(name="linear_one", kind="linear", rows=1, k=1024, n=1024, act="silu", bias="bf16", residual=True, out="bf16"),
        # The output projection of 32 requests of 4 beams, with a bias, to f32 logits.
        dict(name="linear_head", kind="linear", rows=128, k=1024, n=VOCAB, act="none", bias="f32", residual=False,
             out="f32"),
        # An odd batch and odd widths.
        dict(name="linear_ragged", kind="linear", rows=333, k=1000, n=2050, act="gelu", bias="f32", residual=True,
             out="bf16"),
        # A residual block over a prompt of 2048 tokens.
        dict(name="linear_prompt", kind="linear", rows=2048, k=4096, n=4096, act="gelu_tanh", bias="bf16",
             residual=True, out="bf16"),
        # The widening product of a feed-forward block over 8192 prompt tokens.
        dict(name="linear_large", kind="linear", rows=8192, k=4096, n=14336, act="relu", bias="bf16", residual=False,
             out="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["select", "select", "reorder", "linear", "linear"])
    if kind == "select":
        vocab = rng.choice([VOCAB, _log_int(rng, 1000, LARGE_VOCAB), _log_int(rng, 20000, LARGE_VOCAB)])
        beams = _log_int(rng, 1, 32)
        groups = min(_log_int(rng, 1, 64), max(1, min(256, MOST_LOGITS // (4 * vocab)) // beams))
        mask = rng.random() < 0.3
        return dict(kind=kind, groups=groups, beams=beams, vocab=vocab, dtype=rng.choice(["f32", "bf16"]),
                    n=rng.choice([1, beams, beams, 2 * beams, 2 * beams]), ended=rng.random() < 0.4, mask=mask,
                    legal_norm=mask and rng.random() < 0.5, scale=rng.random() < 0.4)
    if kind == "reorder":
        states, groups, beams = rng.randint(1, 56), _log_int(rng, 1, 16), rng.randint(2, 16)
        heads, dim = rng.randint(1, 16), rng.choice([40, 64, 80, 128, 130])
        dtype = rng.choice(["bf16", "f32"])
        most = MOST_STATE // (states * groups * beams * heads * dim * (2 if dtype == "bf16" else 4))
        positions = max(1, min(_log_int(rng, 1, 2000), most))
        return dict(kind=kind, states=states, groups=groups, beams=beams, heads=heads, positions=positions, dim=dim,
                    dtype=dtype, lengths=rng.random() < 0.7)
    rows, k, n = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192), _log_int(rng, 16, 32768)
    n = max(16, min(n, MOST_FLOPS // (2 * rows * k)))
    return dict(kind=kind, rows=rows, k=k, n=n, act=rng.choice(ACTIVATIONS), bias=rng.choice(["none", "bf16", "f32"]),
                residual=rng.random() < 0.5, out=rng.choice(["bf16", "bf16", "f32"]))


# ---------------------------------------------------------------------------
# Inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 2654435761 + 12345) % (1 << 62))
    return g


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device="cuda", dtype=torch.float64)


def _padded(rows, cols, unit, dtype):
    """A [rows, cols] view of rows whose stride is cols rounded up to `unit`."""
    return torch.zeros((rows, -(-cols // unit) * unit), dtype=dtype, device="cuda")[:, :cols]


def _prepare_select(case, seed):
    """Logits as N(0, 2.5^2) with a head that falls with its rank, as a
    language model gives them; cumulative scores some nats apart; every fifth
    group at its first step, with one live beam; a quarter of the beams ended
    where the case has ended ones; masks of token runs, some rows with few
    legal tokens and one row with none."""
    g = _gen(seed)
    G, W, V = case["groups"], case["beams"], case["vocab"]
    x = _padded(G * W, V, 4, torch.float32)
    x.copy_(2.5 * torch.randn((G * W, V), generator=g, device="cuda"))
    H = min(2048, V // 2)
    fall = (1.2 + 2.8 * _rand(g, G * W, 1)).float() * torch.log(torch.arange(1, H + 1, device="cuda").float())
    ids = torch.randint(V, (G * W, H), generator=g, device="cuda")
    x.scatter_reduce_(1, ids, 18.0 - fall + 0.3 * torch.randn((G * W, H), generator=g, device="cuda"), "amax")
    if case["dtype"] == "bf16":
        b = _padded(G * W, V, 4, torch.bfloat16)
        b.copy_(x)
        x = b
    score = -(5.0 + 60.0 * _rand(g, G, 1)) - torch.cumsum(1.5 * _rand(g, G, W), 1)
    score[4::5] = -math.inf
    score[4::5, 0] = 0.0
    s = dict(case=case, logits=x, score=score)
    if case["ended"]:
        s["ended"] = (_rand(g, G, W) < 0.25) & (score > -math.inf)
    if case["scale"]:
        length = torch.randint(4, 60, (G, W), generator=g, device="cuda").double()
        s["scale"] = ((5.0 + length) / 6.0) ** -0.8
    if case["mask"]:
        runs = max(4, V // 2000)
        start = torch.randint(V, (G * W, runs), generator=g, device="cuda")
        stop = (start + torch.randint(1, 65, (G * W, runs), generator=g, device="cuda")).clamp_(max=V)
        edge = torch.zeros((G * W, V + 1), dtype=torch.int32, device="cuda")
        edge.scatter_add_(1, start, torch.ones_like(start, dtype=torch.int32))
        edge.scatter_add_(1, stop, -torch.ones_like(stop, dtype=torch.int32))
        legal = torch.cumsum(edge, 1)[:, :V] > 0
        legal[3::8] &= torch.arange(V, device="cuda") % 512 == 0
        legal[G * W // 2] = False
        bits = torch.zeros((G * W, (V + 31) // 32 * 32), dtype=torch.int64, device="cuda")
        bits[:, :V] = legal
        w = (bits.view(G * W, -1, 32) << torch.arange(32, device="cuda")).sum(2)
        s["mask"] = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
    return s


def _prepare_reorder(case, seed):
    """States [states, groups * beams, heads, positions, dim]; the surviving
    half of a group's beams, in any order, have two children each; the
    groups' lengths fall from the full number of positions to half of it."""
    g = _gen(seed)
    S, G, W = case["states"], case["groups"], case["beams"]
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    shape = (S, G * W, case["heads"], case["positions"], case["dim"])
    st = torch.empty(shape, dtype=dt, device="cuda")
    for i in range(S):
        st[i] = torch.randn(shape[1:], generator=g, device="cuda", dtype=torch.float32)
    order = torch.argsort(_rand(g, G, W), 1)
    child = torch.arange(W, device="cuda") * ((W + 1) // 2) // W
    s = dict(case=case, state=st, parent=order[:, child].to(torch.int32).contiguous())
    if case["lengths"]:
        which = torch.argsort(_rand(g, G))
        s["lengths"] = _lengths(case).to("cuda")[which].contiguous()
    return s


def _lengths(case):
    P, G = case["positions"], case["groups"]
    return (P - torch.arange(G) * P // (2 * G)).to(torch.int32)


def _prepare_linear(case, seed):
    g = _gen(seed)
    R, K, N = case["rows"], case["k"], case["n"]
    x, w = _padded(R, K, 8, torch.bfloat16), _padded(N, K, 8, torch.bfloat16)
    x.copy_(torch.randn((R, K), generator=g, device="cuda"))
    w.copy_(torch.randn((N, K), generator=g, device="cuda") * K ** -0.5)
    s = dict(case=case, x=x, weight=w)
    if case["bias"] != "none":
        b = torch.randn(N, generator=g, device="cuda")
        s["bias"] = b.to(torch.bfloat16) if case["bias"] == "bf16" else b
    dt = torch.bfloat16 if case["out"] == "bf16" else torch.float32
    if case["residual"]:
        s["residual"] = torch.randn((R, N), generator=g, device="cuda").to(dt)
    return s


def prepare(case, seed):
    return {"select": _prepare_select, "reorder": _prepare_reorder, "linear": _prepare_linear}[case["kind"]](case, seed)


# ---------------------------------------------------------------------------
# The plain forms

END = 2   # the end token


def _legal(s, V):
    words = s["mask"].to(torch.int64) & 0xFFFFFFFF
    bits = (words[:, :, None] >> torch.arange(32, device="cuda")) & 1
    return bits.reshape(words.shape[0], -1)[:, :V].bool()


def _best(rank, n):
    """The n largest of each row, equal ones by lower index.  topk leaves the
    order of equal values open, so it takes 64 more (more than share one
    value), which are put in index order and sorted stably."""
    _, at = torch.topk(rank, min(rank.shape[1], n + 64), dim=1)
    at = at.sort(1).values
    by = torch.sort(torch.gather(rank, 1, at), dim=1, descending=True, stable=True).indices
    return torch.gather(at, 1, by)[:, :n]


def _plain_select(s):
    case = s["case"]
    G, W, V, n = case["groups"], case["beams"], case["vocab"], case["n"]
    x = s["logits"].double()
    legal = _legal(s, V) if case["mask"] else None
    if case["legal_norm"]:
        x = x.masked_fill(~legal, -math.inf)
    top = x.amax(1, keepdim=True).clamp_(min=-1e300)   # (a row without a legal token: no candidates)
    norm = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    score = s["score"].view(G * W, 1)
    cand = torch.where(x > -math.inf, score + (x - norm), -math.inf)
    if legal is not None:
        cand = cand.masked_fill(~legal, -math.inf)
    if case["ended"]:
        ended = s["ended"].view(G * W)
        cand[ended] = -math.inf
        cand[:, END] = torch.where(ended, score[:, 0], cand[:, END])
    rank = cand * s["scale"].view(G * W, 1) if case["scale"] else cand
    at = _best(rank.view(G, W * V), n)
    got = torch.gather(cand.view(G, W * V), 1, at)
    there = got > -math.inf
    beam, token = at // V, at % V
    ends = token == END   # an ended beam's own candidate carries that token too
    pad = n - at.shape[1]
    out = dict(token=torch.where(there, token, -1).to(torch.int32), beam=torch.where(there, beam, -1).to(torch.int32),
               score=got, ended=there & ends)
    if pad > 0:
        fill = dict(token=-1, beam=-1, score=-math.inf, ended=False)
        out = {k: torch.nn.functional.pad(v, (0, pad), value=fill[k]) for k, v in out.items()}
    return out


def _plain_reorder(s):
    case, st = s["case"], s["state"]
    S, G, W = case["states"], case["groups"], case["beams"]
    rows = (s["parent"].long() + torch.arange(G, device="cuda")[:, None] * W).view(-1)
    new = st[:, rows]
    if case["lengths"]:
        keep = torch.arange(case["positions"], device="cuda") < s["lengths"][:, None]
        keep = keep.repeat_interleave(W, 0)[None, :, None, :, None]
        new = torch.where(keep, new, st)
    st.copy_(new)
    return st


def _activate(y, act):
    if act == "relu":
        return torch.clamp(y, min=0.0)
    if act == "silu":
        return y / (1.0 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _plain_linear(s):
    y = s["x"].float() @ s["weight"].float().t()
    if "bias" in s:
        y = y + s["bias"].float()
    y = _activate(y, s["case"]["act"])
    if "residual" in s:
        y = y + s["residual"].float()
    return y.to(torch.bfloat16 if s["case"]["out"] == "bf16" else torch.float32)


# ---------------------------------------------------------------------------
# The framework's calls

_handle = []


def _sampler():
    """The program's one sampler context, made at its first call."""
    if not _handle:
        from metallix_amd import Sampler

        _handle.append(Sampler(max_rows=256, max_vocab=LARGE_VOCAB))
    return _handle[0]


def _own_select(s):
    call = s.get("call")
    if call is None:
        c = s["case"]
        call = s["call"] = _sampler().beam_launcher(s["logits"], s["score"], c["n"], ended=s.get("ended"), end_token=END,
                                                    scale=s.get("scale"), mask=s.get("mask"), legal_norm=c["legal_norm"])
    call(s["logits"])
    o = call.out
    return dict(token=o.token, beam=o.beam, score=o.score, ended=o.ended)


def _own_reorder(s):
    call = s.get("call")
    if call is None:
        call = s["call"] = _sampler().reorder_launcher(list(s["state"]), s["parent"], lengths=s.get("lengths"),
                                                       length_dim=2)
    call()
    return s["state"]


def _own_linear(s):
    call = s.get("call")
    if call is None:
        c = s["case"]
        call = s["call"] = _sampler().linear_launcher(s["x"], s["weight"], s.get("bias"), activation=c["act"],
                                                      residual=s.get("residual"),
                                                      out_dtype=torch.bfloat16 if c["out"] == "bf16" else torch.float32)
    call(s["x"])
    return call.out


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"select": _own_select, "reorder": _own_reorder, "linear": _own_linear}[kind](state)
    return {"select": _plain_select, "reorder": _plain_reorder, "linear": _plain_linear}[kind](state)


# ---------------------------------------------------------------------------

def work(case):
    if case["kind"] == "select":
        G, W, V, n = case["groups"], case["beams"], case["vocab"], case["n"]
        # the rows of live beams: the first steps' groups have one, and a quarter may have ended
        first = (G + 0) // 5
        live = ((G - first) * W + first) * (0.75 if case["ended"] else 1.0)
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": live * (V * size + (V / 8 if case["mask"] else 0)) + G * n * 17 + G * W * 8, "flops": live * V * 2}
    if case["kind"] == "reorder":
        G, W = case["groups"], case["beams"]
        size = case["states"] * case["heads"] * case["dim"] * (2 if case["dtype"] == "bf16" else 4)
        positions = float(_lengths(case).sum()) if case["lengths"] else case["positions"] * G
        # each surviving parent's state is read and each moved child's written; one child a group stays in place on average
        return {"bytes": size * positions * ((W + 1) // 2 + W - 1), "flops": 0}
    R, K, N = case["rows"], case["k"], case["n"]
    out = 2 if case["out"] == "bf16" else 4
    bias = {"none": 0, "bf16": 2, "f32": 4}[case["bias"]] * N
    return {"bytes": 2 * K * (R + N) + R * N * out * (2 if case["residual"] else 1) + bias, "flops": 2 * R * K * N}


def exact(case, seed):
    """What run returns, from the definitions in 64 bits.  A selection's whole
    numbers and a reordering's moved values are not computed numbers."""
    s = prepare(case, seed)
    if case["kind"] == "reorder":
        return None
    if case["kind"] == "linear":
        y = torch.matmul(s["x"].double(), s["weight"].double().t())
        if "bias" in s:
            y += s["bias"].double()
        F = torch.nn.functional
        y = {"none": lambda v: v, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
             "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[case["act"]](y)
        return y + s["residual"].double() if "residual" in s else y
    G, W, V, n = case["groups"], case["beams"], case["vocab"], case["n"]
    out = torch.full((G, n), -math.inf, dtype=torch.float64, device="cuda")
    for g in range(G):
        found, ranks = [], []
        for b in range(W):
            r = g * W + b
            if float(s["score"][g, b]) == -math.inf:
                continue
            c = s["scale"][g, b] if case["scale"] else 1.0
            if case["ended"] and bool(s["ended"][g, b]):
                found.append(s["score"][g, b][None])
            else:
                x = s["logits"][r].double()
                legal = None
                if case["mask"]:
                    at = torch.arange(V, device="cuda")
                    legal = (s["mask"][r][at // 32].long() >> (at % 32)) & 1 != 0
                if case["legal_norm"]:
                    x = x[legal]
                lp = x - torch.logsumexp(x, 0) if x.numel() else x
                if case["mask"] and not case["legal_norm"]:
                    lp = lp[legal]
                found.append(s["score"][g, b] + lp.sort(descending=True).values[:n])
            ranks.append(found[-1] * c)
        if found:
            v, order = torch.cat(ranks).sort(descending=True, stable=True)
            v = torch.cat(found)[order][:n]
            out[g, : v.numel()] = v
    return dict(token=None, beam=None, score=out, ended=None)
