"""What the Python binding of the beam entry points refuses and how it reads
its tensors, without a GPU."""
import itertools

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


def pieces(t, rows, length_dim, L):
    """The elements (as offsets in the storage) that a move of t takes in each
    row, from its description and from its index."""
    m = S.state_struct(t, rows, length_dim)
    es, base = t.element_size(), (t.data_ptr() - t.untyped_storage().data_ptr()) // t.element_size()
    used = min(m.segment_bytes, L * m.position_bytes) if length_dim is not None else m.segment_bytes
    assert used % es == 0 and m.data == t.data_ptr()
    told = [sorted(base + (r * m.row_stride + s * m.segment_stride) // es + i for s in range(m.segments)
                   for i in range(used // es)) for r in range(rows)]
    flat = torch.arange(t.untyped_storage().nbytes() // es).as_strided(t.shape, t.stride(), t.storage_offset())
    if length_dim is not None:
        flat = flat.narrow(length_dim, 0, min(L, t.shape[length_dim]))
    return told, [sorted(flat[r].reshape(-1).tolist()) for r in range(rows)]


@pytest.mark.parametrize("shape", [(4, 5, 3, 2), (4, 1, 3, 6), (4, 5, 1, 2), (4, 5, 3, 1), (4, 1, 1, 3), (1, 5, 3, 2)])
def test_states_in_any_order_of_their_dimensions(shape):
    """Dense rows move whole in any order of their dimensions, as a cache
    [rows, positions, heads, dim] seen as [rows, heads, positions, dim]."""
    for order in itertools.permutations(range(1, 4)):
        t = torch.zeros(shape, dtype=torch.bfloat16).permute(0, *order)
        m = S.state_struct(t, shape[0])
        assert m.segments * m.segment_bytes == t[0].numel() * 2
        told, want = pieces(t, shape[0], None, 0)
        assert told == want, order
        for d in range(1, 4):
            for L in (0, 1, 2, 9):
                told, want = pieces(t, shape[0], d, L)
                assert told == want, (order, d, L)


def test_positions_in_any_order_of_the_dimensions():
    t = torch.zeros((4, 7, 3, 8))                        # [rows, positions, heads, dim]
    m = S.state_struct(t.transpose(1, 2), 4, 2)          # ... seen as [rows, heads, positions, dim]
    assert (m.segments, m.segment_bytes, m.position_bytes, m.row_stride) == (1, 7 * 96, 96, 7 * 96)
    m = S.state_struct(t.permute(0, 2, 3, 1), 4, 2)      # [rows, heads, dim, positions], the dim's first entries
    assert (m.segments, m.segment_bytes, m.position_bytes, m.segment_stride) == (21, 32, 4, 32)
    h = torch.zeros((4, 3, 7, 8))                        # [rows, heads, positions, dim]
    for view, d in ((h, 2), (h.transpose(1, 2), 1), (h.permute(0, 3, 2, 1), 2), (h.permute(0, 2, 3, 1), 1)):
        m = S.state_struct(view, 4, d)
        assert (m.segments, m.segment_bytes, m.position_bytes, m.segment_stride) == (3, 224, 32, 224)
        for L in (0, 3, 7):
            told, want = pieces(view, 4, d, L)
            assert told == want
    c = torch.zeros((3, 4, 7, 8)).permute(1, 2, 0, 3)    # memory [heads][rows][positions][dim]
    for L in (0, 3, 7):
        told, want = pieces(c, 4, 1, L)
        assert told == want
    for bad, d in ((torch.zeros((4, 5, 6, 7))[:, ::2, ::2], None), (torch.zeros((4, 5, 6))[:, :, ::2].transpose(1, 2), 2),
                   (torch.zeros((4, 5, 6, 7))[:, :, :4].transpose(1, 3), 1)):
        with pytest.raises(ValueError):
            S.state_struct(bad, 4, d)


def test_numbers_that_32_bits_do_not_hold():
    """ctypes keeps the low 32 bits: 2^32 + 4 candidates, rows or pieces would
    be 4."""
    big = (1 << 32) + 4
    meta, bf = torch.device("meta"), torch.bfloat16
    z = lambda *n, dt=torch.float32: torch.zeros(n, dtype=dt, device="meta")
    lg, sc = torch.zeros(8, 100), torch.zeros(2, 4, dtype=torch.float64)
    f = lambda n=4, **kw: S.beam_struct(torch, CPU, lg, sc, n, **kw)
    mask = torch.zeros(8, 4, dtype=torch.int32)
    assert f(mask=mask, tokenizer_vocab=(1 << 32) - 1).tokenizer_vocab == (1 << 32) - 1
    for kw in (dict(n=big), dict(n=-1), dict(end_token=big), dict(end_token=(1 << 32) - 1), dict(mask=mask, tokenizer_vocab=big),
               dict(mask=mask, tokenizer_vocab=-1)):
        with pytest.raises(ValueError):
            f(**kw)
    with pytest.raises(ValueError, match="groups"):
        S.beam_struct(torch, meta, z(big, 4), z(big, 1, dt=torch.float64), 1)
    for R, K, N in ((big, 8, 8), (8, big, 8), (8, 8, big)):
        with pytest.raises(ValueError, match="2.32"):
            S.linear_struct(torch, meta, z(R, K, dt=bf), z(N, K, dt=bf), None, None, z(R, N, dt=bf), None)
    with pytest.raises(ValueError, match="pieces"):
        S.state_struct(z(2, 1 << 31, 4, 8)[:, :, :, :4], 2)
    parent, status = z(2, big, dt=torch.int32), z(2, dt=torch.int32)
    with pytest.raises(ValueError, match="row stride"):
        S.reorder_struct(torch, meta, [z(8, 4)], parent, status, beams=4)
