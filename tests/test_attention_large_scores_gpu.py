"""mxs_prefix_attention where scores are so large that a unit in the last place of
the largest is a large part of the exponential's range, up to the 2^30 that the
header allows: all weight is on the largest score.

Tolerances: the largest score's exponential is 2^d with |d| up to half a last place of
the reference, which its sum holds too; it is rounded to bf16 once (2^-8) and the
output once more.  lse: scale, product, reference and its return to base e are a
rounding each, 2^-24 of it."""
import pytest

from test_attention_gpu import inputs, sampler, say, torch_mod  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 20, 2.0 ** 27, 2.0 ** 29])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("shape", [(1, 2, 1, 4, 2, 64, 300, 20), (1, 40, 2, 4, 1, 128, 450, 20), (2, 3, 1, 4, 2, 256, 130, 20),
                                   (16, 5, 1, 32, 8, 128, 1800, 100)], ids=str)
def test_large_scores(torch_mod, sampler, size, sign, shape):  # noqa: F811
    """Scores of one product each, so that they are exact; from the largest on
    they fall by size / 128 and more, at the least size by 32."""
    torch = torch_mod
    say(f"large scores {size} {sign} {shape}")
    G, W, T, H, KV, D, P, N = shape
    x = inputs(torch, *shape, seed=3)
    x["q"].zero_()
    x["q"][..., 3] = 1.37 * size ** 0.5
    g = torch.Generator(device="cuda").manual_seed(1)
    for keys in (x["prefix_keys"], x["keys"]):
        mult = torch.randint(100, 128, keys.shape[:3], generator=g, device="cuda")
        keys[..., 3] = (sign * mult * size ** 0.5 / 64).to(torch.bfloat16)
    x["prefix_keys"][:, :, 7, 3] = sign * (140 if sign > 0 else 90) * size ** 0.5 / 64
    lse = torch.empty((G * W, T, H), device="cuda")
    out = sampler.prefix_attention(x["q"], x["prefix_keys"], x["prefix_values"], x["keys"], x["values"], scale=0.3, lse=lse)
    sampler.sync()
    v = x["prefix_values"][:, :, 7].double().repeat_interleave(W, 0).repeat_interleave(H // KV, 1)[:, None].expand(G * W, T, H, D)
    assert bool(((out.double() - v).abs() <= v.abs() * (2.0 ** -7 + 2.0 ** -15)).all())
    score = float(x["q"][0, 0, 0, 3].double() * x["prefix_keys"][0, 0, 7, 3].double()) * 0.3
    assert size > abs(score) / 2 and bool(((lse.double() - score).abs() <= abs(score) * 2.0 ** -22).all())
