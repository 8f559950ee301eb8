"""GPU tests of mxs_beam_select where a row's logits are large and its maximum
comes late.  The oracle's norms are long doubles."""
import numpy as np
import pytest

from test_beam_gpu import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_mod():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.fixture(scope="module")
def sampler(torch_mod):
    from metallix_amd import Sampler

    s = Sampler(max_rows=256, max_vocab=262144)
    yield s
    s.close()


@pytest.mark.parametrize("base", [2.0 ** k for k in range(10, 40)] + [-(2.0 ** k) for k in range(10, 40, 3)])
def test_maxima_that_come_late(torch_mod, sampler, base):
    """Each row rises by steps between its tiles, by the smallest f32 step that
    is at least 1, 300, 600 or 1000, so that a later maximum lies just below,
    at and above the point where the weights' unit moves; the last step's
    tokens are the row's best."""
    W, V = 64, 100003                       # 25 tiles in chunks of 4
    x = np.empty((W, V), np.float32)
    steps = [1.0, 300.0, 600.0, 1000.0]
    for b in range(W):
        v = np.float32(base * (1.0 + 0.001 * (b // 4)))
        for t in range(25):
            x[b, t * 4096 : (t + 1) * 4096] = v
            if t % 8 != 7:
                ulp = np.spacing(np.abs(v))
                v = np.float32(v + max(ulp, np.float32(np.ceil(steps[b % 4] / ulp) * ulp)))
    score = np.full((1, W), -np.inf)
    for b in (0, 1, 2, 3, 21, 42, 63):      # one live beam at a time: its own scores
        s = score.copy()
        s[0, b] = -2.0
        tok, beam, sc, _, st = run(torch_mod, sampler, x, s, 8)
        l = x[b].astype(np.longdouble)
        norm = l.max() + np.log(np.sum(np.exp(l - l.max())))
        assert st.tolist() == [0], (base, b)
        assert beam.tolist() == [[b] * 8]
        at = np.nonzero(x[b] == x[b].max())[0][:8]
        assert tok.tolist() == [at.tolist()]
        want = -2.0 + (l.max() - norm)
        # the logarithm of the sum within 2^-39, and its own and the score's roundings
        assert np.all(np.abs(sc - float(want)) <= 2.0 ** -39 + 2.0 ** -52 * abs(float(norm)) + 2.0 ** -50), (base, b, sc, want)


@pytest.mark.parametrize("size", [1.0, 300.0, 900.0, 2.0 ** 12, 2.0 ** 14, 1e5, 3e6, 2.0 ** 30])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_logarithms_stated_bound(torch_mod, sampler, size, sign, dtype):
    """Scores of single beams against norms in long double: the logarithm N
    within 2^-39 + 2^-52 |N|; l - N and the score add their own roundings,
    2^-53 of their sizes each, and the long doubles 2^-60."""
    G, W, V, n = 6, 1, 30011, 5
    rng = np.random.default_rng(int(size) % 9973)
    x = (sign * size + rng.standard_normal((G, V)) * 2.5).astype(np.float32)
    x[1] = (sign * size * (1.0 + 0.5 * rng.random(V))).astype(np.float32)
    x[2, :20000] -= np.float32(50.0)
    if dtype == "bf16":
        b = x.view(np.uint32)
        x = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    score = -rng.uniform(0.0, 3.0, (G, W))
    tok, beam, sc, _, st = run(torch_mod, sampler, x, score, n, dtype=dtype)
    assert st.tolist() == [0] * G
    for g in range(G):
        l = x[g].astype(np.longdouble)
        norm = l.max() + np.log(np.sum(np.exp(l - l.max())))
        at = np.lexsort((np.arange(V), -x[g]))[:n]
        assert tok[g].tolist() == at.tolist()
        lp = l[at] - norm
        want = score[g, 0] + lp
        err = 2.0 ** -39 + 2.0 ** -52 * abs(norm) + 2.0 ** -53 * (np.abs(lp) + np.abs(want)) + 2.0 ** -60 * abs(norm)
        assert np.all(np.abs(sc[g].astype(np.longdouble) - want) <= err), (g, sc[g], want, norm)


@pytest.mark.parametrize("score,scale", [([-0.0, 0.0, -0.0, 0.0], None), ([0.0, -0.0, 0.0, -0.0], None),
                                         ([-1e-200, 0.0, -1e-200, 0.0], [1e-200, 1.0, 1e-200, 1.0])])
def test_ranks_of_either_zero_are_equal(torch_mod, sampler, score, scale):
    """Ended beams whose rank is 0 of either sign (certain, or a product that
    underflows) are equal: the lower beam first.  (Live ones are not: their
    scores are off by up to 2^-39.)"""
    W, V = 4, 50
    x = np.zeros((W, V), np.float32)
    kw = {} if scale is None else dict(scale=np.array([scale]))
    tok, beam, sc, en, st = run(torch_mod, sampler, x, np.array([score]), W, ended=np.ones((1, W), bool), end_token=7, **kw)
    assert st.tolist() == [0] and beam.tolist() == [[0, 1, 2, 3]]
    assert tok.tolist() == [[7] * W] and en.all()
    assert sc[0].tolist() == score
