"""GPU tests of mxs_linear_bf16 against the definition in 64 bits.

The sum of K products of bf16 values (exact in f32) in f32 is off by at most
K 2^-24 sum |x w| (any order), the bias adds one rounding.  The activations
grow an error by at most 1.13 (their steepest slope) and are themselves within
2^-20 of the value's magnitude (an f32 exponential and a division); residual
and output add a rounding each, the output's by its type: bf16 2^-8 relative,
f32 2^-24."""
import math
import sys

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


def say(msg):
    print(msg, flush=True)
    sys.stdout.flush()


def padded(torch, t, pad, poison=float("nan")):
    """t as a view of rows whose stride is padded, the padding poisoned."""
    R, K = t.shape
    b = torch.full((R, -(-K // 8) * 8 + 8 * pad), poison, dtype=t.dtype, device=t.device)
    b[:, :K] = t
    return b[:, :K]


def act64(torch, y, act):
    F = torch.nn.functional
    return {"none": lambda v: v, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
            "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[act](y)


def inputs(torch, R, K, N, seed, bias, residual, out, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    x, w = r(R, K).to(torch.bfloat16), (r(N, K) * spread * K ** -0.5).to(torch.bfloat16)
    dt = torch.bfloat16 if out == "bf16" else torch.float32
    b = None if bias == "none" else r(N).to(torch.bfloat16 if bias == "bf16" else torch.float32)
    return x, w, b, (r(R, N).to(dt) if residual else None), dt


def verify(torch, got, x, w, b, res, act):
    # 64-bit products on the host's terms: float64 matmul of 2-d operands
    x64, w64 = x.double(), w.double().t().contiguous()
    y = x64 @ w64
    mag = x64.abs() @ w64.abs()
    K = x.shape[1]
    err = mag * (K * 2.0 ** -24)
    if b is not None:
        y = y + b.double()
        err = err + y.abs() * 2.0 ** -23
    a = act64(torch, y, act)
    if act != "none":
        err = 1.13 * err + a.abs() * 2.0 ** -20 + 2.0 ** -30
    if res is not None:
        a = a + res.double()
        err = err + a.abs() * 2.0 ** -23
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    err = err * (1 + half) + a.abs() * half + 1e-37
    off = (got.double() - a).abs()
    assert bool((off <= err).all()), (float((off / err).max()), int((off > err).sum()))


def check(torch, sampler, R, K, N, *, act="none", bias="none", residual=False, out="bf16", pad=0, spread=1.0, seed=0):
    say(f"case linear R {R} K {K} N {N} {act} bias {bias} residual {residual} out {out} pad {pad}")
    x, w, b, res, dt = inputs(torch, R, K, N, 1000 * R + K + N + seed, bias, residual, out, spread)
    x, w = (padded(torch, t, pad) if pad or K % 8 else t for t in (x, w))
    got = sampler.linear(x, w, b, activation=act, residual=res, out_dtype=dt)
    torch.cuda.synchronize()
    verify(torch, got, x, w, b, res, act)


SHAPES = [(1, 1, 1), (1, 8, 1), (2, 7, 3), (1, 32, 16), (3, 33, 17), (1, 1024, 1024), (1, 1000, 2050), (4, 4096, 63),
          (5, 63, 1027), (8, 129, 4099), (16, 512, 512), (17, 1000, 255), (32, 2048, 100), (33, 64, 2048),
          (63, 96, 65), (64, 1024, 4096), (65, 1024, 1000), (100, 31, 129), (127, 520, 257), (128, 1024, 8200),
          (129, 4096, 127), (200, 100, 1), (255, 8, 300), (256, 256, 256), (257, 72, 513), (333, 1000, 2050),
          (512, 640, 1024), (700, 2056, 130), (1024, 128, 1025), (1500, 1032, 777), (2048, 512, 640)]


@pytest.mark.parametrize("R,K,N", SHAPES)
def test_shapes(torch_mod, sampler, R, K, N):
    acts = ["none", "relu", "silu", "gelu", "gelu_tanh"]
    i = R + K + N
    check(torch_mod, sampler, R, K, N, act=acts[i % 5], bias=["none", "bf16", "f32"][i % 3], residual=i % 2 == 0,
          out=["bf16", "f32"][(i // 2) % 2], pad=i % 3)
    check(torch_mod, sampler, R, K, N, out="f32")


@pytest.mark.parametrize("R,K,N", [(1, 256, 512), (20, 264, 130), (300, 136, 390)])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_epilogues(torch_mod, sampler, R, K, N, act, out):
    for bias in ("none", "bf16", "f32"):
        for residual in (False, True):
            check(torch_mod, sampler, R, K, N, act=act, bias=bias, residual=residual, out=out, spread=4.0)


@pytest.mark.parametrize("R", [1, 40, 300])
def test_strides_and_untouched_memory(torch_mod, sampler, R):
    """Outputs and residuals in wider rows at element alignment: what lies
    beside them stays."""
    torch = torch_mod
    K, N = 72, 133
    for dt, name in ((torch.bfloat16, "bf16"), (torch.float32, "f32")):
        for off, stride in ((0, 136), (1, 140), (2, 133 + 2), (3, 137)):
            x, w, b, res, _ = inputs(torch, R, K, N, off + R, "f32", True, name)
            big = torch.full((R * stride + 8,), 7.5, dtype=dt, device="cuda")
            out = big[off : off + R * stride].view(R, stride)[:, :N]
            rbig = torch.zeros((R, N + 3), dtype=dt, device="cuda")
            rv = rbig[:, 1 : N + 1]
            rv.copy_(res)
            say(f"case strides R {R} {name} off {off} stride {stride}")
            sampler.linear(x, w, b, activation="silu", residual=rv, out=out)
            torch.cuda.synchronize()
            verify(torch, out, x, w, b, res, "silu")
            keep = torch.ones_like(big, dtype=torch.bool)
            keep[off : off + R * stride].view(R, stride)[:, :N] = False
            assert bool((big[keep] == 7.5).all())


@pytest.mark.parametrize("R,K,N", [(1, 128, 128), (70, 128, 128), (513, 128, 128)])
def test_residual_in_place(torch_mod, sampler, R, K, N):
    torch = torch_mod
    x, w, b, res, _ = inputs(torch, R, K, N, R, "bf16", True, "bf16")
    out = res.clone()
    assert sampler.linear(x, w, b, activation="silu", residual=out, out=out) is out
    torch.cuda.synchronize()
    verify(torch, out, x, w, b, res, "silu")


@pytest.mark.parametrize("R", [2, 70, 400])
def test_values_that_are_not_finite(torch_mod, sampler, R):
    """A NaN or infinity stays in its row (x) or its feature (weight)."""
    torch = torch_mod
    K, N = 136, 200
    x, w, b, _, _ = inputs(torch, R, K, N, R, "f32", False, "f32")
    base = sampler.linear(x, w, b, out_dtype=torch.float32)
    x2, w2 = x.clone(), w.clone()
    x2[R - 1, K - 1] = float("nan")
    w2[N - 1, 0] = float("inf")
    got = sampler.linear(x2, w2, b, out_dtype=torch.float32)
    relu = sampler.linear(x2, w2, b, activation="relu", out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert bool(got[R - 1].isnan().all()) and bool(relu[R - 1].isnan().all())
    assert bool((~got[: R - 1, N - 1].isfinite()).all())
    assert torch.equal(got[: R - 1, : N - 1], base[: R - 1, : N - 1])   # elsewhere the same bits


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "relu"])
def test_large_arguments(torch_mod, sampler, act):
    torch = torch_mod
    x = torch.zeros((4, 8), dtype=torch.bfloat16, device="cuda")
    x[:, 0] = torch.tensor([1.0, -1.0, 64.0, -64.0])
    w = torch.zeros((64, 8), dtype=torch.bfloat16, device="cuda")
    w[:, 0] = torch.logspace(-3, 3.5, 64, device="cuda")
    got = sampler.linear(x, w, activation=act, out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert bool(got.isfinite().all())
    verify(torch, got, x, w, None, None, act)


def test_captured_and_replayed(torch_mod):
    torch = torch_mod
    from metallix_amd import Sampler

    stream = torch.cuda.Stream()
    s = Sampler(max_rows=8, max_vocab=1024, stream=stream)
    try:
        for R, K, N in ((2, 256, 300), (150, 520, 260), (600, 256, 512)):
            x, w, b, res, _ = inputs(torch, R, K, N, R, "bf16", True, "bf16")
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


def test_no_rows_and_refusals(torch_mod, sampler):
    from metallix_amd import SamplerError

    torch = torch_mod
    bf = torch.bfloat16
    z = lambda *s: torch.zeros(s, dtype=bf, device="cuda")
    assert sampler.linear(z(0, 16), z(4, 16)).shape == (0, 4)
    with pytest.raises(SamplerError, match="multiples of 8"):
        sampler.linear(z(4, 12), z(4, 12))
    with pytest.raises(SamplerError, match="aligned"):
        sampler.linear(z(4, 24)[:, 4:20], z(4, 16))
    big = z(8, 16)
    with pytest.raises(SamplerError, match="overlaps"):
        sampler.linear(big[:4], z(16, 16), out=big[2:6])
    with pytest.raises(ValueError):
        sampler.linear(z(4, 16), z(4, 16).cpu())
    with pytest.raises(ValueError):
        sampler.linear(z(4, 16), z(4, 16), activation="swish")


# Sizes whose tiles are 128 x 128, 128 x 256 (features x rows) and 256 x 256,
# and those summed in parts, each with a last tile that rows, features and k
# leave unfilled.
LARGER = [(2999, 31, 1025), (2900, 328, 1100), (257, 72, 12001), (300, 1000, 12003), (1031, 392, 7799),
          (2999, 200, 4099), (4100, 1032, 2056), (700, 2056, 130), (33, 8200, 1023), (65, 1350, 130), (130, 1300, 2050), (40, 14344, 200),
          (20, 11272, 1025)]


@pytest.mark.parametrize("R,K,N", LARGER)
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_larger_tiles(torch_mod, sampler, R, K, N, act):
    i = len(act) + R
    for out in ("bf16", "f32"):
        check(torch_mod, sampler, R, K, N, act=act, bias=["none", "bf16", "f32"][i % 3], residual=i % 2 == 0, out=out,
              pad=i % 2, spread=2.0, seed=i)
        i += 1


@pytest.mark.parametrize("R,K,N", [(2999, 72, 1025), (257, 72, 12001), (1031, 392, 7799), (700, 2056, 130)])
def test_larger_tiles_strides_and_in_place(torch_mod, sampler, R, K, N):
    torch = torch_mod
    for dt, name in ((torch.bfloat16, "bf16"), (torch.float32, "f32")):
        for off, stride in ((0, N + 8 - N % 8), (1, N + 2), (3, N)):
            x, w, b, res, _ = inputs(torch, R, K, N, off + R, "bf16", True, name)
            big = torch.full((R * stride + 8,), 7.5, dtype=dt, device="cuda")
            out = big[off : off + R * stride].view(R, stride)[:, :N]
            out.copy_(res)
            say(f"case strides R {R} K {K} N {N} {name} off {off} stride {stride}, in place")
            sampler.linear(x, w, b, activation="relu", residual=out, out=out)
            torch.cuda.synchronize()
            verify(torch, out, x, w, b, res, "relu")
            keep = torch.ones_like(big, dtype=torch.bool)
            keep[off : off + R * stride].view(R, stride)[:, :N] = False
            assert bool((big[keep] == 7.5).all())


@pytest.mark.parametrize("R,K,N", [(2999, 72, 1025), (257, 72, 12001), (1031, 392, 7799), (700, 2056, 130)])
def test_larger_tiles_not_finite_and_repeated(torch_mod, sampler, R, K, N):
    """A NaN or infinity stays in its row or feature; equal calls give equal
    bits."""
    torch = torch_mod
    x, w, b, _, _ = inputs(torch, R, K, N, R, "f32", False, "f32")
    x, w = padded(torch, x, 1), padded(torch, w, 2)
    base = sampler.linear(x, w, b, out_dtype=torch.float32)
    again = sampler.linear(x, w, b, out_dtype=torch.float32)
    x2, w2 = x.clone(), w.clone()
    x2[R - 1, K - 1] = float("nan")
    w2[N - 1, 0] = float("inf")
    got = sampler.linear(x2, w2, b, out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert torch.equal(base, again)
    assert bool(got[R - 1].isnan().all()) and bool((~got[: R - 1, N - 1].isfinite()).all())
    assert torch.equal(got[: R - 1, : N - 1], base[: R - 1, : N - 1])


def test_largest_tiles_captured_and_replayed(torch_mod):
    torch = torch_mod
    from metallix_amd import Sampler

    stream = torch.cuda.Stream()
    s = Sampler(max_rows=8, max_vocab=1024, stream=stream)
    try:
        for R, K, N in ((2999, 200, 4099), (300, 1000, 12003), (700, 2056, 130)):
            x, w, b, res, _ = inputs(torch, R, K, N, R, "bf16", True, "bf16")
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
