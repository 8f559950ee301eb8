"""A prebuilt call holds the tensors whose addresses it passes, also where the
caller's list of them, or result object, changes or goes away.  No GPU: the
entry points only note that they were called."""
import gc
import types
import weakref

import pytest
import torch

from metallix_amd.sampler import EvictResult, Sampler

BF, I32 = torch.bfloat16, torch.int32


def stub():
    lib = types.SimpleNamespace(**{n: (lambda *a: 0) for n in ("mxs_cache_evict", "mxs_beam_reorder", "mxs_beam_reorder_check")})
    return types.SimpleNamespace(torch=torch, lib=lib, ctx=None, _device=lambda: torch.device("cpu"), _check=lambda rc, what: None)


def caches():
    return [torch.zeros(3, 2, 10, 16, dtype=BF) for _ in range(2)]


def gone(refs):
    gc.collect()
    return [r() is None for r in refs]


@pytest.mark.parametrize("how", ["list", "iterator"])
def test_evict(how):
    keys, values = caches(), caches()
    out = EvictResult(torch.zeros(2, 3, 2, 10), torch.zeros(2, 3, 2, 10, dtype=I32), torch.zeros(3, dtype=I32))
    refs = [weakref.ref(t) for t in keys + values + [out.weight, out.index, out.lengths]]
    f = Sampler.cache_evict_launcher(stub(), iter(keys) if how == "iterator" else keys, iter(values) if how == "iterator" else values,
                                     torch.zeros(2, 3, 2, 10), 5, out=out)
    keys.clear(), values.clear()
    out.weight = out.index = out.lengths = None
    assert not any(gone(refs))
    f()
    del f
    assert all(gone(refs))


def test_reorder():
    states = [torch.zeros(6, 4), torch.zeros(6, 5)]
    refs = [weakref.ref(t) for t in states]
    f = Sampler.reorder_launcher(stub(), states, torch.zeros(2, 3, dtype=I32), status=torch.zeros(2, dtype=I32))
    states.clear()
    assert not any(gone(refs))
    f()
    del f
    assert all(gone(refs))
