"""Products whose results go on to the framework's other calls, at widths that
are no multiple of anything."""
import pytest

from test_linear_gpu import inputs, verify

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

    s = Sampler(max_rows=160, max_vocab=50257)
    yield s
    s.close()


@pytest.mark.parametrize("G,W,K,V", [(1, 4, 64, 50257), (2, 3, 40, 1001), (40, 4, 72, 2050), (1, 1, 8, 7), (3, 2, 16, 64)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_logits_to_a_selection(torch_mod, sampler, G, W, K, V, out):
    torch = torch_mod
    x, w, b, _, dt = inputs(torch, G * W, K, V, V + K, "f32", False, out)
    lg = sampler.linear(x, w, b, out_dtype=dt)
    score = torch.zeros((G, W), dtype=torch.float64, device="cuda")
    r = sampler.beam_select(lg, score, W)
    torch.cuda.synchronize()
    assert lg.shape == (G * W, V) and lg.dtype == dt
    verify(torch, lg, x, w, b, None, "none")
    padded = torch.zeros((G * W, V + (-V) % 4), dtype=dt, device="cuda")[:, :V]
    padded.copy_(lg)
    want = sampler.beam_select(padded, score, W)
    torch.cuda.synchronize()
    for f in ("token", "beam", "score", "status"):
        assert torch.equal(getattr(r, f), getattr(want, f)), f
    assert r.status.cpu().tolist() == [0] * G


@pytest.mark.parametrize("R,K,N1,N2", [(1, 24, 7, 5), (5, 40, 333, 130), (70, 64, 2050, 65), (300, 1000, 1030, 257)])
def test_a_product_of_a_product(torch_mod, sampler, R, K, N1, N2):
    torch = torch_mod
    x, w, b, _, _ = inputs(torch, R, K, N1, R + N1, "f32", False, "bf16")
    y = sampler.linear(x, w, b, activation="silu")
    w2 = torch.zeros((N2, N1 + (-N1) % 8), dtype=torch.bfloat16, device="cuda")[:, :N1]
    w2.copy_(inputs(torch, 1, N1, N2, N2, "none", False, "bf16")[1])
    z = sampler.linear(y, w2, out_dtype=torch.float32)
    torch.cuda.synchronize()
    verify(torch, y, x, w, b, None, "silu")
    verify(torch, z, y, w2, None, None, "none")
