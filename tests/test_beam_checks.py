"""What the beam and linear entry points refuse, without a GPU: the checks of
the C ABI (mxs_checks.h, built with the host compiler) and those of the Python
binding."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from metallix_amd import sampler as S

HERE = Path(__file__).resolve().parent
CPU = torch.device("cpu")


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    so = tmp_path_factory.mktemp("checks") / "checks.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", str(HERE / "beam_checks.cpp"), "-o", str(so)],
                   check=True)
    lib = ctypes.CDLL(str(so))
    for f in (lib.check_beam, lib.check_reorder, lib.check_linear):
        f.restype = ctypes.c_char_p
    return lib


def beam(**kw):
    b = S.MxsBeam()
    b.logits, b.dtype, b.groups, b.beams, b.vocab, b.row_stride = 0x100000, 0, 3, 4, 1000, 1000
    b.score, b.n, b.end_token = 0x2000, 4, -1
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def beam_out(**kw):
    o = S.MxsBeamOut()
    o.token, o.beam, o.score, o.status = 0x3000, 0x4000, 0x5000, 0x6000
    for k, v in kw.items():
        setattr(o, k, v)
    return o


BEAM_BAD = [
    (dict(logits=None), {}, "required"), (dict(score=None), {}, "required"), ({}, dict(token=None), "required"),
    ({}, dict(status=None), "required"), (dict(dtype=2), {}, "dtype"), (dict(beams=0), {}, "beams"),
    (dict(beams=65, groups=1), {}, "beams"), (dict(n=0), {}, "n must"), (dict(n=129), {}, "n must"),
    (dict(vocab=0), {}, "vocab"), (dict(groups=300), {}, "max_rows"), (dict(vocab=300000, row_stride=300000), {}, "max_vocab"),
    (dict(groups=1 << 30, beams=4), {}, "max_rows"), (dict(row_stride=996), {}, "row_stride"),
    (dict(row_stride=1002), {}, "row_stride"), (dict(logits=0x1008), {}, "aligned"),
    (dict(logits=0x1004, dtype=1), {}, "aligned"), (dict(end_token=1000), {}, "end_token"),
    (dict(end_token=-2), {}, "end_token"), (dict(ended=0x7000), {}, "end_token"),
    (dict(mask_words=0x8000, mask_stride=31), {}, "mask_stride"), (dict(legal_norm=1), {}, "mask_words"),
    (dict(row_stride=1 << 62), {}, "range"), (dict(mask_words=0x8000, mask_stride=1 << 62), {}, "range"),
    ({}, dict(score=0x2008), "overlaps"), ({}, dict(score=0x1ff8), "overlaps"), (dict(scale=0x5058), {}, "overlaps"),
    (dict(ended=0x7000, end_token=2), dict(ended=0x7001), "overlaps"), ({}, dict(token=0x100000 + 47996), "overlaps"),
    (dict(mask_words=0x8000, mask_stride=32), dict(status=0x85fc), "overlaps"), ({}, dict(beam=0x302c), "outputs"),
    ({}, dict(status=0x5000), "outputs"), ({}, dict(ended=0x6004), "outputs"),
    (dict(n=8), dict(score=0x2000), "n == beams"), (dict(n=3, ended=0x7000, end_token=2), dict(ended=0x7000), "n == beams"),
]


@pytest.mark.parametrize("b,o,word", BEAM_BAD)
def test_beam_select_refuses(checks, b, o, word):
    msg = checks.check_beam(ctypes.byref(beam(**b)), ctypes.byref(beam_out(**o)), 1000, 262144)
    assert msg and word in msg.decode(), msg


@pytest.mark.parametrize("b,o", [({}, {}), (dict(groups=0, logits=None), {}), (dict(logits=0x100008, dtype=1), {}),
                                 ({}, dict(score=0x2000)), (dict(ended=0x7000, end_token=0), dict(ended=0x7000)),
                                 (dict(mask_words=0x8000, mask_stride=32, legal_norm=1), {}),
                                 (dict(mask_words=0x8000, mask_stride=32), dict(status=0x8600)),
                                 ({}, dict(beam=0x3030)), ({}, dict(token=0x100000 + 48000))])
def test_beam_select_accepts(checks, b, o):
    assert checks.check_beam(ctypes.byref(beam(**b)), ctypes.byref(beam_out(**o)), 1000, 262144) is None


def state(**kw):
    s = S.MxsState()
    s.data, s.row_stride, s.segment_stride, s.segment_bytes, s.position_bytes, s.segments = 0x1000, 4096, 512, 512, 64, 8
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def reorder(states, **kw):
    r = S.MxsReorder()
    arr = (S.MxsState * max(1, len(states)))(*states)
    r.states, r.count = ctypes.cast(arr, ctypes.POINTER(S.MxsState)), len(states)
    r.groups, r.beams, r.parent_stride, r.parent, r.status = 2, 4, 4, 0x2000, 0x3000
    for k, v in kw.items():
        setattr(r, k, v)
    r.keep = arr
    return r


REORDER_BAD = [
    (dict(), dict(parent=None), "required"), (dict(), dict(status=None), "required"), (dict(), dict(count=0), "one state"),
    (dict(), dict(beams=0), "beams"), (dict(), dict(beams=65, parent_stride=65), "beams"),
    (dict(), dict(groups=65536), "groups"), (dict(), dict(parent_stride=3), "parent_stride"),
    (dict(data=None), {}, "null"), (dict(segments=0), {}, "positive"), (dict(segment_bytes=0), {}, "positive"),
    (dict(segment_bytes=1 << 36, row_stride=1 << 40, segment_stride=1 << 36), {}, "32 GiB"),
    (dict(position_bytes=513), {}, "position_bytes"), (dict(row_stride=0), {}, "overlap"),
    (dict(row_stride=4095), {}, "overlap"), (dict(segment_stride=511), {}, "overlap"),
    (dict(segment_stride=0), {}, "overlap"), (dict(row_stride=512, segment_stride=4095), {}, "overlap"),
    (dict(row_stride=1 << 50), {}, "range"),
    # products that wrap 64 bits: segments that would come back to the row's start, positions to no bytes
    (dict(segments=(1 << 17) + 1, segment_stride=1 << 47, row_stride=4096), {}, "range"),
    (dict(segment_bytes=1 << 34, position_bytes=1 << 34, segments=1, segment_stride=1 << 34, row_stride=1 << 34), {}, "4 GiB"),
]


@pytest.mark.parametrize("s,r,word", REORDER_BAD)
def test_beam_reorder_refuses(checks, s, r, word):
    msg = checks.check_reorder(ctypes.byref(reorder([state(), state(**s)], **r)))
    assert msg and word in msg.decode(), msg


@pytest.mark.parametrize("s", [{}, dict(row_stride=512, segment_stride=4096), dict(segments=1, segment_stride=0),
                               dict(position_bytes=0), dict(segments=1, segment_stride=1 << 60),
                               dict(segment_bytes=1 << 32, position_bytes=(1 << 32) - 1, segments=1, row_stride=1 << 32)])
def test_beam_reorder_accepts(checks, s):
    assert checks.check_reorder(ctypes.byref(reorder([state(**s)]))) is None


def linear(**kw):
    a = S.MxsLinear()
    a.x, a.x_stride, a.weight, a.weight_stride, a.out, a.out_stride = 0x10000, 64, 0x20000, 64, 0x40000, 32
    a.rows, a.in_features, a.out_features, a.out_dtype = 16, 64, 32, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


LINEAR_BAD = [
    (dict(x=None), "required"), (dict(weight=None), "required"), (dict(out=None), "required"),
    (dict(in_features=0), "positive"), (dict(out_features=0), "positive"), (dict(act=5), "act"), (dict(act=-1), "act"),
    (dict(out_dtype=2), "out_dtype"), (dict(bias=0x50000, bias_dtype=7), "bias_dtype"), (dict(x_stride=60), "x_stride"),
    (dict(x_stride=68), "x_stride"), (dict(weight_stride=56), "weight_stride"), (dict(out_stride=31), "out_stride"),
    (dict(residual=0x60000, residual_stride=31), "residual_stride"), (dict(x=0x10008), "aligned"),
    (dict(weight=0x20008), "aligned"), (dict(out=0x40001), "aligned"), (dict(out=0x40002, out_dtype=0), "aligned"),
    (dict(out=0x10010), "overlaps"), (dict(out=0x20ff0), "overlaps"), (dict(bias=0x40010, bias_dtype=1), "overlaps"),
    (dict(residual=0x40002, residual_stride=32), "residual"), (dict(residual=0x40000, residual_stride=48), "residual"),
    (dict(rows=1 << 31), "2^30"), (dict(rows=1 << 30, x_stride=64, in_features=64, out_features=64, out_stride=64), "2^35"),
    (dict(rows=1 << 18, out_features=1 << 17, out_stride=1 << 17), "2^35"), (dict(x_stride=1 << 41), "range"),
]


@pytest.mark.parametrize("a,word", LINEAR_BAD)
def test_linear_refuses(checks, a, word):
    msg = checks.check_linear(ctypes.byref(linear(**a)))
    assert msg and word in msg.decode(), msg


@pytest.mark.parametrize("a", [{}, dict(rows=0, x=None), dict(residual=0x40000, residual_stride=32),
                               dict(in_features=57), dict(out_features=31), dict(bias=0x40400, bias_dtype=0),
                               dict(rows=(1 << 29) - 64, out_stride=32, out=1 << 44, x=1 << 45)])
def test_linear_accepts(checks, a):
    assert checks.check_linear(ctypes.byref(linear(**a))) is None


# ---- the binding's checks

def test_beam_struct_refuses():
    lg, sc = torch.zeros(8, 100), torch.zeros(2, 4, dtype=torch.float64)
    f = lambda logits=lg, score=sc, n=4, **kw: S.beam_struct(torch, CPU, logits, score, n, **kw)
    b = f(ended=torch.zeros(2, 4, dtype=torch.bool), end_token=3, scale=torch.ones_like(sc))
    assert (b.groups, b.beams, b.vocab, b.row_stride, b.end_token) == (2, 4, 100, 100, 3)
    bad = [dict(score=sc.float()), dict(score=sc[0]), dict(logits=lg[:7]), dict(logits=lg.half()), dict(vocab=101),
           dict(logits=torch.zeros(100, 8).t()), dict(score=torch.zeros(4, 2, dtype=torch.float64).t()),
           dict(ended=torch.zeros(2, 3, dtype=torch.bool)), dict(ended=torch.zeros(2, 4)),
           dict(scale=torch.ones(2, 4)), dict(mask=torch.zeros(8, 3, dtype=torch.int32)),
           dict(mask=torch.zeros(7, 4, dtype=torch.int32)), dict(mask=torch.zeros(8, 4))]
    for kw in bad:
        with pytest.raises(ValueError):
            f(**kw)
    with pytest.raises(ValueError):
        S.beam_struct(torch, torch.device("meta"), lg, sc, 4)


def test_state_struct_layouts():
    t = torch.zeros(6, 5, 7, 3, dtype=torch.float32)
    m = S.state_struct(t, 6)
    assert (m.segments, m.segment_bytes, m.row_stride, m.position_bytes) == (1, 420, 420, 0)
    m = S.state_struct(t, 6, 2)
    assert (m.segments, m.segment_bytes, m.segment_stride, m.position_bytes) == (5, 84, 84, 12)
    m = S.state_struct(t.permute(1, 0, 2, 3)[:4], 4)          # [segments][rows]
    assert (m.segments, m.row_stride, m.segment_stride, m.segment_bytes) == (6, 84, 420, 84)
    m = S.state_struct(t[:, :, 1:4], 6)
    assert (m.segments, m.segment_bytes, m.segment_stride, m.row_stride) == (5, 36, 84, 420)
    m = S.state_struct(torch.zeros(6), 6)
    assert (m.segments, m.segment_bytes, m.row_stride) == (1, 4, 4)
    m = S.state_struct(t[:, ::2], 6, 2)                       # evenly spaced pieces
    assert (m.segments, m.segment_stride, m.segment_bytes) == (3, 168, 84)
    for bad, d in ((t[:5], None), (t[:, :, :, ::2], 2), (t, 0), (t, 4), (t[:, :0], None), (t[:, :, :4], 3)):
        with pytest.raises(ValueError):
            S.state_struct(bad, 6, d)


def test_reorder_struct_refuses():
    t, p, st = torch.zeros(8, 3), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    f = lambda states=(t,), parent=p, **kw: S.reorder_struct(torch, CPU, list(states), parent, st, **kw)
    assert (f().groups, f().beams, f().count) == (2, 4, 1)
    assert f(states=[t[:4]], beams=2).parent_stride == 4
    for kw in (dict(parent=p.long()), dict(parent=p[0]), dict(beams=5), dict(beams=0), dict(states=[t[:7]]),
               dict(states=[t, t]), dict(states=[t, torch.zeros(8, 2), t[:, :2]]),
               dict(lengths=torch.zeros(3, dtype=torch.int32)), dict(lengths=torch.zeros(2)),
               dict(length_dim=[1, 1]), dict(length_dim=2), dict(parent=torch.zeros(4, 2, dtype=torch.int32).t())):
        with pytest.raises(ValueError):
            f(**kw)


def test_linear_struct_refuses():
    bf = torch.bfloat16
    x, w, o = torch.zeros(4, 16, dtype=bf), torch.zeros(10, 16, dtype=bf), torch.zeros(4, 10, dtype=bf)
    f = lambda x=x, w=w, bias=None, res=None, out=o, act=None: S.linear_struct(torch, CPU, x, w, bias, res, out, act)
    assert (f().rows, f().in_features, f().out_features) == (4, 16, 10)
    for kw in (dict(x=x.float()), dict(w=w[:, :15]), dict(out=o[:3]), dict(out=o.half()), dict(bias=torch.zeros(9)),
               dict(bias=torch.zeros(10, dtype=torch.float64)), dict(res=o.float()), dict(res=o[:, :9]), dict(act="tanh"),
               dict(x=torch.zeros(16, 4, dtype=bf).t()), dict(bias=torch.zeros(20)[::2])):
        with pytest.raises(ValueError):
            f(**kw)
