"""GPU tests of mxs_linear_bf16 with long sums, at sizes that take each of its
kernels (tests/test_linear_choice.py holds the sizes to that), against the
definition in 64 bits.

Where K is long, a bound on the sums' rounding is wider than a single product,
so a product left out or taken twice would pass it.  Small whole numbers leave
none: every product and partial sum below 2^24 is exact in f32, and the results
have to be equal."""
import pytest

from test_linear_gpu import inputs, padded, say, verify

pytestmark = pytest.mark.gpu

# rows, k and features that leave the last tiles unfilled, and whole ones
LONG = [(250, 1290, 2500), (200, 4104, 3333), (129, 1300, 5001), (256, 1280, 4096), (68, 3074, 3181), (220, 2915, 1599),
        (40, 14344, 200), (164, 3467, 1075), (33, 8200, 1023), (148, 2954, 7861), (757, 1940, 5114), (1857, 3332, 1884),
        (1005, 2146, 7233), (997, 1668, 8390), (2367, 1803, 3777), (3, 8200, 300), (16, 4092, 1000)]
# one of each kernel of long sums
FEW = [(250, 1290, 2500), (68, 3074, 3181), (164, 3467, 1075), (757, 1940, 5114), (1005, 2146, 7233), (997, 1668, 8390)]


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


def whole(torch, R, K, N, seed):
    """x, weight and bias of whole numbers in -8..8, none of them 0: partial
    sums stay below 64 * 14344 + 8 < 2^24."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*n):
        v = torch.randint(1, 9, n, generator=g, device="cuda").float()
        return torch.where(torch.randint(0, 2, n, generator=g, device="cuda") == 1, v, -v)

    return r(R, K).to(torch.bfloat16), r(N, K).to(torch.bfloat16), r(N)


@pytest.mark.parametrize("R,K,N", LONG)
def test_whole_numbers_are_exact(torch_mod, sampler, R, K, N):
    torch = torch_mod
    say(f"case whole numbers R {R} K {K} N {N}")
    x, w, b = whole(torch, R, K, N, R + K)
    x, w = padded(torch, x, R % 2), padded(torch, w, R % 3)
    got = sampler.linear(x, w, b, out_dtype=torch.float32)
    relu = sampler.linear(x, w, b, activation="relu", residual=got, out_dtype=torch.float32)
    torch.cuda.synchronize()
    want = x.double() @ w.double().t().contiguous() + b.double()
    assert torch.equal(got.double(), want)
    assert torch.equal(relu.double(), want.clamp(min=0.0) + want)


@pytest.mark.parametrize("R,K,N", LONG)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_long_sums(torch_mod, sampler, R, K, N, act):
    torch = torch_mod
    i = len(act) + R
    for out in ("bf16", "f32"):
        say(f"case long R {R} K {K} N {N} {act} {out}")
        x, w, b, res, dt = inputs(torch, R, K, N, i + N, ["none", "bf16", "f32"][i % 3], i % 2 == 0, out, 2.0)
        x, w = padded(torch, x, i % 2), padded(torch, w, i % 2)
        got = sampler.linear(x, w, b, activation=act, residual=res, out_dtype=dt)
        torch.cuda.synchronize()
        verify(torch, got, x, w, b, res, act)
        i += 1


@pytest.mark.parametrize("R,K,N", FEW)
def test_strides_and_in_place(torch_mod, sampler, R, K, N):
    torch = torch_mod
    for dt, name in ((torch.bfloat16, "bf16"), (torch.float32, "f32")):
        for off, stride in ((0, N + 8 - N % 8), (1, N + 2), (3, N)):
            x, w, b, res, _ = inputs(torch, R, K, N, off + R, "bf16", True, name)
            x, w = padded(torch, x, 1), padded(torch, w, 0)
            big = torch.full((R * stride + 8,), 7.5, dtype=dt, device="cuda")
            out = big[off : off + R * stride].view(R, stride)[:, :N]
            out.copy_(res)
            say(f"case long strides R {R} K {K} N {N} {name} off {off} stride {stride}, in place")
            sampler.linear(x, w, b, activation="relu", residual=out, out=out)
            torch.cuda.synchronize()
            verify(torch, out, x, w, b, res, "relu")
            keep = torch.ones_like(big, dtype=torch.bool)
            keep[off : off + R * stride].view(R, stride)[:, :N] = False
            assert bool((big[keep] == 7.5).all())


@pytest.mark.parametrize("R,K,N", FEW)
def test_not_finite_and_repeated(torch_mod, sampler, R, K, N):
    """A NaN or infinity, at either end of the sum, stays in its row or
    feature; equal calls give equal bits."""
    torch = torch_mod
    x, w, b, _, _ = inputs(torch, R, K, N, R, "f32", False, "f32")
    x, w = padded(torch, x, 1), padded(torch, w, 2)
    base = sampler.linear(x, w, b, out_dtype=torch.float32)
    again = sampler.linear(x, w, b, out_dtype=torch.float32)
    for ka, kb in ((K - 1, 0), (0, K - 1), (K // 2, K // 3)):
        x2, w2 = x.clone(), w.clone()
        x2[R - 1, ka] = float("nan")
        w2[N - 1, kb] = float("inf")
        x2, w2 = padded(torch, x2, 1), padded(torch, w2, 2)
        got = sampler.linear(x2, w2, b, out_dtype=torch.float32)
        torch.cuda.synchronize()
        assert bool(got[R - 1].isnan().all()) and bool((~got[: R - 1, N - 1].isfinite()).all())
        assert torch.equal(got[: R - 1, : N - 1], base[: R - 1, : N - 1])
    assert torch.equal(base, again)


def test_captured_and_replayed(torch_mod):
    torch = torch_mod
    from metallix_amd import Sampler

    stream = torch.cuda.Stream()
    s = Sampler(max_rows=8, max_vocab=1024, stream=stream)
    try:
        for R, K, N in FEW:
            say(f"case long captured R {R} K {K} N {N}")
            x, w, b, res, _ = inputs(torch, R, K, N, R, "bf16", True, "bf16")
            x, w = padded(torch, x, 1), padded(torch, w, 1)
            torch.cuda.synchronize()
            call = s.linear_launcher(x, w, b, activation="gelu", residual=res)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                call(x)
            for i in range(3):
                new = inputs(torch, R, K, N, R + i + 1, "none", False, "bf16")[0]
                torch.cuda.synchronize()
                with torch.cuda.stream(stream):
                    x.copy_(new)
                    s.linear(x, w)
                    graph.replay()
                torch.cuda.synchronize()
                verify(torch, call.out, x, w, b, res, "gelu")
    finally:
        s.close()
