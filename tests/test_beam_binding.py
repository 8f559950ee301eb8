"""What the Python binding of the beam entry points refuses and how it reads
its tensors, without a GPU."""
import pytest
import torch

from metallix_amd import sampler as S

CPU = torch.device("cpu")


def result(G, n, **kw):
    e = lambda dt: torch.zeros((G, n), dtype=dt)
    r = S.BeamResult(token=e(torch.int32), beam=e(torch.int32), score=e(torch.float64), ended=e(torch.bool),
                     status=torch.zeros(G, dtype=torch.int32))
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def test_outputs_of_a_selection():
    G, n = 3, 5
    r = result(G, n)
    o = S.beam_out_struct(torch, CPU, r, G, n)
    assert (o.token, o.beam, o.score) == (r.token.data_ptr(), r.beam.data_ptr(), r.score.data_ptr())
    assert (o.ended, o.status) == (r.ended.data_ptr(), r.status.data_ptr())
    assert S.beam_out_struct(torch, CPU, result(G, n, ended=None), G, n).ended is None
    wide = lambda dt: torch.zeros((G, 2 * n), dtype=dt)[:, :n]
    for kw in (dict(token=wide(torch.int32)), dict(beam=wide(torch.int32)), dict(score=wide(torch.float64)),
               dict(ended=wide(torch.bool)), dict(score=torch.zeros((G, n))), dict(status=torch.zeros(G)),
               dict(status=torch.zeros(G + 1, dtype=torch.int32)), dict(status=torch.zeros((G, 1), dtype=torch.int32))):
        with pytest.raises(ValueError):
            S.beam_out_struct(torch, CPU, result(G, n, **kw), G, n)


def test_a_status_with_gaps_is_refused():
    """The status goes to consecutive entries: a column of a table would get
    its neighbours' too."""
    table = torch.zeros((4, 3), dtype=torch.int32)
    with pytest.raises(ValueError, match="status must be contiguous"):
        S.beam_out_struct(torch, CPU, result(4, 2, status=table[:, 0]), 4, 2)
    t, parent = torch.zeros(8, 3), torch.zeros((4, 2), dtype=torch.int32)
    assert S.reorder_struct(torch, CPU, [t], parent, table[1:2, 0].expand(4).clone()).groups == 4
    with pytest.raises(ValueError, match="status must be contiguous"):
        S.reorder_struct(torch, CPU, [t], parent, table[:, 0])
