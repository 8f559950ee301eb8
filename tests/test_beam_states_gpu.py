"""Moves of states whose dimensions lie in memory in another order than their
own."""
import numpy as np
import pytest

from test_beam_gpu import bits, dev, fill, moved

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_mod():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    return torch


@pytest.mark.parametrize("order,dim", [((0, 2, 1, 3), 2), ((0, 2, 1, 3), None), ((0, 3, 2, 1), 2), ((0, 2, 3, 1), 1),
                                       ((0, 3, 1, 2), None), ((0, 2, 3, 1), 3)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32", "uint8"])
def test_moves_of_views(torch_mod, order, dim, dtype):
    torch = torch_mod
    from metallix_amd import Sampler

    rng = np.random.default_rng(sum(order[2:]) + (dim or 0))
    G, W, shape = 3, 4, (12, 11, 3, 10)
    parent, lengths = rng.integers(-1, W, (G, W)), np.array([0, 3, 50])
    s = Sampler(max_rows=8, max_vocab=64)
    t = fill(torch, rng, shape, getattr(torch, dtype)).permute(*order)
    a = bits(t)
    kw = {} if dim is None else dict(lengths=dev(torch, lengths.astype(np.int32)), length_dim=dim)
    size = t.element_size()
    print(f"case views {order} {dim} {dtype}", flush=True)
    s.beam_reorder([t], dev(torch, parent.astype(np.int32)), **kw)
    torch.cuda.synchronize()
    # (bits widens the last dimension to bytes; where that is the positions', their bytes)
    want = moved(a, parent, lengths * (size if dim == 3 else 1), dim) if dim else moved(a, parent)
    assert np.array_equal(bits(t), want)
    s.close()
