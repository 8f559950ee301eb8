"""mxs_prefix_attention at a scale of 0 and next to it, with products as large as
f32 holds: every score is (next to) 0, all positions weigh the same."""
import pytest

from test_attention_gpu import inputs, run, sampler, say, torch_mod  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [0.0, -0.0, 2.0 ** -149, -2.0 ** -140, 2.0 ** -130])
@pytest.mark.parametrize("shape", [(1, 2, 1, 4, 2, 64, 100, 20), (1, 40, 2, 4, 1, 128, 150, 20), (2, 3, 1, 4, 2, 256, 70, 20)], ids=str)
def test_large_products(torch_mod, sampler, scale, shape):  # noqa: F811
    torch = torch_mod
    say(f"large products {scale} {shape}")
    x = inputs(torch, *shape, seed=12)
    x["q"][..., 2] = 2.0 ** 63
    for keys in (x["prefix_keys"], x["keys"]):
        keys[..., 2] = (2.0 ** 61 * (torch.arange(keys.shape[2], device="cuda") % 3 - 1)).to(torch.bfloat16)   # products of +-2^124
    run(torch, sampler, x, weights=True, scale=scale)
