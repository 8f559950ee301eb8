"""The epilogue's activations alone: a product of zeros leaves act(bias), so any
f32 argument is exact, and f32 results show the activation's own error: within
2^-20 of the value's size plus 2^-30, as the header has it, and the output's
2^-24."""
import pytest

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

    s = Sampler(max_rows=8, max_vocab=1024)
    yield s
    s.close()


def f64(torch, y, act):
    """The formulas in f64, the small side of the normal integral by erfc."""
    y = y.double()
    if act == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return 0.5 * y * torch.erfc(-y * 0.5 ** 0.5)
    return y * torch.sigmoid(1.5957691216057308 * (y + 0.044715 * y ** 3))


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("rows", [1, 200])      # the kernel of few rows, and tiles
def test_every_size_of_argument(torch_mod, sampler, act, rows):
    torch = torch_mod
    g = torch.Generator(device="cuda").manual_seed(3)
    e = torch.linspace(-126.0, 126.0, 4096, dtype=torch.float64, device="cuda")
    wide = torch.exp2(e) * (1.0 + torch.rand(4096, generator=g, device="cuda", dtype=torch.float64))
    near = torch.linspace(-20.0, 20.0, 65536, dtype=torch.float64, device="cuda")
    far = torch.linspace(-120.0, 120.0, 8192, dtype=torch.float64, device="cuda")
    y = torch.cat([wide, -wide, near, far, torch.tensor([0.0, -0.0], device="cuda")]).float()
    x = torch.zeros((rows, 8), dtype=torch.bfloat16, device="cuda")
    w = torch.zeros((y.numel(), 8), dtype=torch.bfloat16, device="cuda")
    got = sampler.linear(x, w, y, activation=act, out_dtype=torch.float32)
    torch.cuda.synchronize()
    want = y.double() if act == "none" else f64(torch, y, act)
    err = want.abs() * (0.0 if act in ("none", "relu") else 2.0 ** -20 + 2.0 ** -24)
    err = err + (0.0 if act in ("none", "relu") else 2.0 ** -30)
    off = (got.double() - want).abs()
    assert bool((off <= err).all()), (y[(off > err).any(0)][:5], float((off - err).max()))


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_arguments_that_are_not_finite(torch_mod, sampler, act):
    torch = torch_mod
    inf, nan = float("inf"), float("nan")
    y = torch.tensor([inf, -inf, nan, 1.0], device="cuda")
    x = torch.zeros((1, 8), dtype=torch.bfloat16, device="cuda")
    w = torch.zeros((4, 8), dtype=torch.bfloat16, device="cuda")
    got = sampler.linear(x, w, y, activation=act, out_dtype=torch.float32)[0].cpu()
    torch.cuda.synchronize()
    assert got[0] == inf and got[2].isnan() and got[3].isfinite()
    assert got[1] == (-inf if act == "none" else 0.0) if act in ("none", "relu") else got[1].isnan()
