"""What the attention and eviction entry points refuse, without a GPU: the
checks of the C ABI (mxs_attention_checks.h, built with the host compiler) and
those of the Python binding."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from metallix_amd import sampler as S

HERE = Path(__file__).resolve().parent
CPU = torch.device("cpu")
BF = torch.bfloat16


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    so = tmp_path_factory.mktemp("checks") / "checks.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
                    str(HERE / "attention_checks.cpp"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    for f in (lib.check_attention, lib.check_evict):
        f.restype = ctypes.c_char_p
    return lib


def attention(**kw):
    """2 groups of 3 rows, 2 tokens, 8 heads over 4, dim 64; prefix 100, suffix 10; all dense."""
    a = S.MxsAttention()
    a.groups, a.beams, a.tokens, a.heads, a.kv_heads, a.dim, a.prefix, a.suffix, a.scale = 2, 3, 2, 8, 4, 64, 100, 10, 0.125
    a.q, a.q_row, a.q_token, a.q_head = 0x100000, 1024, 512, 64                          # 12288 bytes
    a.out, a.out_row, a.out_token, a.out_head = 0x110000, 1024, 512, 64
    a.prefix_keys, a.prefix_values = 0x200000, 0x300000                                  # 102400 bytes each
    a.prefix_group, a.prefix_head, a.prefix_position = 25600, 6400, 64
    a.keys, a.values, a.row, a.head, a.position = 0x400000, 0x500000, 2560, 640, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


ATTENTION_BAD = [
    (dict(q=None), "required"), (dict(out=None), "required"), (dict(heads=0), "multiple of kv_heads"),
    (dict(kv_heads=0), "multiple of kv_heads"), (dict(kv_heads=3), "multiple of kv_heads"),
    (dict(heads=8192), "4096"), (dict(dim=0), "dim"), (dict(dim=60), "dim"), (dict(dim=264), "dim"),
    (dict(prefix=(1 << 30) + 1), "2^30"), (dict(suffix=(1 << 30) + 1), "2^30"),
    (dict(groups=1 << 16, beams=1 << 16), "2^31"), (dict(tokens=1 << 29), "2^31"),
    (dict(prefix_keys=None), "prefix needs"), (dict(prefix_values=None), "prefix needs"),
    (dict(keys=None), "suffix needs"), (dict(values=None), "suffix needs"),
    (dict(prefix=0, prefix_weight=0x600000), "needs a prefix"), (dict(suffix=0, weight=0x600000), "needs a suffix"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=-2.5e38), "scale"),
    (dict(q_row=1028), "multiples of 8"), (dict(out_token=516), "multiples of 8"), (dict(prefix_group=25601), "multiples of 8"),
    (dict(position=65), "multiples of 8"), (dict(q_head=1 << 41), "range"), (dict(prefix_head=1 << 41), "range"),
    (dict(prefix_position=1 << 22), "2^22"), (dict(position=1 << 22), "2^22"),
    (dict(groups=1 << 15, beams=1, tokens=1, q_row=1 << 36), "range"), (dict(groups=1 << 15, beams=1, tokens=1, row=1 << 36), "range"),
    (dict(q=0x100008), "aligned"), (dict(out=0x110008), "aligned"), (dict(prefix_keys=0x200008), "aligned"),
    (dict(values=0x500002), "aligned"), (dict(lse=0x600002), "aligned"), (dict(lengths=0x600001), "aligned"),
    (dict(out_head=56), "rows overlap"), (dict(out_token=0), "rows overlap"), (dict(out_row=1016), "rows overlap"),
    (dict(out=0x100000), "overlaps an input"), (dict(out=0x102ff0), "overlaps an input"),
    (dict(out=0x200000 + 102384), "overlaps an input"), (dict(out=0x300000), "overlaps an input"),
    (dict(out=0x400000), "overlaps an input"), (dict(out=0x500000 + 30704), "overlaps an input"),
    (dict(lse=0x100010), "overlaps an input"), (dict(prefix_lengths=0x600000, lse=0x600004), "overlaps an input"),
    (dict(lengths=0x600000, prefix_weight=0x600014), "overlaps an input"),
    (dict(lse=0x110000), "outputs overlap"), (dict(prefix_weight=0x600000, weight=0x600000), "outputs overlap"),
    (dict(lse=0x600000, weight=0x60017c), "outputs overlap"),
]


@pytest.mark.parametrize("a,word", ATTENTION_BAD)
def test_attention_refuses(checks, a, word):
    msg = checks.check_attention(ctypes.byref(attention(**a)))
    assert msg and word in msg.decode(), msg


@pytest.mark.parametrize("a", [
    {}, dict(groups=0, q=None), dict(tokens=0, q=None), dict(beams=0), dict(prefix=0, prefix_keys=None, prefix_values=None),
    dict(prefix=0, prefix_keys=0x1, prefix_position=3), dict(suffix=0, keys=None, values=None, position=1 << 30),
    dict(out=0x103000), dict(out=0x200000 + 102400), dict(lse=0x600000, weight=0x600180, prefix_weight=0x600f00),
    dict(q_row=0, q_token=0, q_head=0), dict(prefix_group=0, row=0),                       # inputs may share memory
    dict(prefix_values=0x200000), dict(out_token=64, out_row=128, out_head=768),           # any order of the dimensions
    dict(groups=1, beams=1, out_row=0), dict(scale=0.0), dict(scale=-1.0)])
def test_attention_accepts(checks, a):
    assert checks.check_attention(ctypes.byref(attention(**a))) is None


def evict(count=2, caches=None, **kw):
    """2 layers of 3 segments x 4 heads, 100 slots of 128 bytes; all dense."""
    e = S.MxsEvict()
    arr = (S.MxsCache * count)()
    for i in range(count):
        arr[i].keys, arr[i].values = 0x100000 * (2 * i + 1), 0x100000 * (2 * i + 2)
    if caches is not None:
        arr[caches].keys = None
    e.caches, e.layers, e.segments, e.heads, e.capacity = ctypes.cast(arr, ctypes.POINTER(S.MxsCache)), count, 3, 4, 100
    e.segment_stride, e.head_stride, e.position_stride, e.position_bytes = 51200, 12800, 128, 128
    e.budget, e.keep_first, e.keep_recent = 50, 4, 10
    e.weight, e.weight_out = 0x10000, 0x20000   # 9600 bytes
    for k, v in kw.items():
        setattr(e, k, v)
    e.hold = arr
    return e


EVICT_BAD = [
    (dict(weight=None), "required"), (dict(weight_out=None), "required"), (dict(capacity=0), "capacity"),
    (dict(capacity=(1 << 20) + 1), "capacity"), (dict(segments=1 << 20), "2^21"), (dict(segments=1 << 24, heads=1 << 12), "2^21"),
    (dict(budget=0, keep_first=0, keep_recent=0), "budget"), (dict(keep_first=51), "at most budget"),
    (dict(keep_recent=47), "at most budget"), (dict(keep_first=1 << 31, keep_recent=1 << 31), "at most budget"),
    (dict(position_bytes=0), "position_bytes"), (dict(position_bytes=65537), "position_bytes"),
    (dict(segment_stride=1 << 47), "range"), (dict(head_stride=1 << 47), "range"), (dict(position_stride=1 << 28), "range"),
    (dict(position_stride=127), "positions overlap"), (dict(head_stride=12799), "positions overlap"),
    (dict(segment_stride=51199), "positions overlap"), (dict(position_stride=0), "positions overlap"),
    (dict(weight=0x10002), "aligned"), (dict(index=0x30001), "aligned"), (dict(lengths_out=0x30002), "aligned"),
    (dict(caches=1), "null"), (dict(weight_out=0x10000), "overlaps an input"), (dict(weight_out=0x1257c), "overlaps an input"),
    (dict(index=0x30000, index_out=0x30000), "overlaps an input"), (dict(lengths=0x30000, lengths_out=0x30000), "overlaps an input"),
    (dict(index_out=0x20000), "outputs overlap"), (dict(lengths_out=0x2257c), "outputs overlap"),
]


@pytest.mark.parametrize("e,word", EVICT_BAD)
def test_evict_refuses(checks, e, word):
    msg = checks.check_evict(ctypes.byref(evict(**e)))
    assert msg and word in msg.decode(), msg


@pytest.mark.parametrize("e", [
    {}, dict(layers=0, weight=None), dict(segments=0), dict(heads=0), dict(budget=1000), dict(keep_first=40),
    dict(weight_out=0x12580), dict(segment_stride=128, head_stride=384, position_stride=1536),   # any order
    dict(segments=1, segment_stride=0), dict(lengths=0x30000, lengths_out=0x3000c), dict(index_out=0x22580)])
def test_evict_accepts(checks, e):
    assert checks.check_evict(ctypes.byref(evict(**e))) is None


# ---------------------------------------------------------------------------
# The binding

def call(q=None, pk=None, pv=None, k=None, v=None, out=None, **kw):
    q = torch.zeros(6, 2, 8, 64, dtype=BF) if q is None else q
    pk = torch.zeros(2, 4, 100, 64, dtype=BF) if pk is None else pk
    pv = torch.zeros(2, 4, 100, 64, dtype=BF) if pv is None else pv
    k = torch.zeros(6, 4, 10, 64, dtype=BF) if k is None else k
    v = torch.zeros(6, 4, 10, 64, dtype=BF) if v is None else v
    out = torch.zeros(q.shape, dtype=BF) if out is None else out
    return S.attention_struct(torch, CPU, q, pk, pv, k, v, out, **kw)


def test_attention_struct_strides():
    fused = torch.zeros(6, 2, 8 + 8, 64, dtype=BF)
    cache = torch.zeros(2, 4, 120, 64, dtype=BF)[:, :, :100]
    mine = torch.zeros(6, 10, 2, 4, 64, dtype=BF).permute(2, 0, 3, 1, 4)   # [2, rows, heads, positions, dim]
    a = call(q=fused[:, :, :8], pk=cache, pv=cache, k=mine[0], v=mine[1])
    assert (a.groups, a.beams, a.tokens, a.heads, a.kv_heads, a.dim, a.prefix, a.suffix) == (2, 3, 2, 8, 4, 64, 100, 10)
    assert (a.q_row, a.q_token, a.q_head) == (2 * 16 * 64, 16 * 64, 64)
    assert (a.prefix_group, a.prefix_head, a.prefix_position) == (4 * 120 * 64, 120 * 64, 64)
    assert (a.row, a.head, a.position) == (10 * 512, 64, 512)
    assert a.scale == 0.125 and a.keys == mine.data_ptr() and a.values == mine.data_ptr() + 512
    a = call(q=torch.zeros(6, 8, 64, dtype=BF), scale=0.5)
    assert a.tokens == 1 and a.scale == 0.5 and a.q_token == 0
    a = S.attention_struct(torch, CPU, torch.zeros(6, 8, 64, dtype=BF), torch.zeros(2, 4, 0, 64, dtype=BF),
                           torch.zeros(2, 4, 0, 64, dtype=BF), None, None, torch.zeros(6, 8, 64, dtype=BF))
    assert a.prefix == a.suffix == 0 and not a.keys and not a.prefix_keys


I32, F32 = torch.int32, torch.float32
CALL_BAD = [
    (dict(q=torch.zeros(6, 64, dtype=BF)), "shape"), (dict(q=torch.zeros(6, 2, 8, 64)), "bfloat16"),
    (dict(q=torch.zeros(5, 2, 8, 64, dtype=BF), k=torch.zeros(5, 4, 10, 64, dtype=BF), v=torch.zeros(5, 4, 10, 64, dtype=BF)), "same number"),
    (dict(out=torch.zeros(6, 2, 8, 32, dtype=BF)), "out"), (dict(out=torch.zeros(6, 2, 8, 64)), "out"),
    (dict(q=torch.zeros(6, 2, 8, 128, dtype=BF)[..., ::2]), "consecutive"), (dict(pk=torch.zeros(2, 4, 100, 32, dtype=BF)), "prefix_keys"),
    (dict(pk=torch.zeros(2, 4, 100, dtype=BF)), "prefix_keys"), (dict(pv=torch.zeros(2, 4, 99, 64, dtype=BF)), "same"),
    (dict(pv=torch.zeros(2, 4, 120, 64, dtype=BF)[:, :, :100]), "same"), (dict(k=torch.zeros(6, 2, 10, 64, dtype=BF)), "keys"),
    (dict(k=torch.zeros(5, 4, 10, 64, dtype=BF)), "keys"), (dict(v=torch.zeros(6, 4, 10, 64)), "values"),
    (dict(prefix_lengths=torch.zeros(3, dtype=I32)), "prefix_lengths"), (dict(lengths=torch.zeros(2, dtype=I32)), "lengths"),
    (dict(lengths=torch.zeros(6, dtype=torch.int64)), "lengths"), (dict(lse=torch.zeros(6, 2, 8, dtype=BF)), "lse"),
    (dict(lse=torch.zeros(6, 2, 9)[..., :8]), "lse"), (dict(prefix_weight=torch.zeros(2, 4, 99)), "prefix_weight"),
    (dict(weight=torch.zeros(6, 4, 11)), "weight"), (dict(weight=torch.zeros(6, 4, 20)[..., ::2]), "contiguous"),
]


@pytest.mark.parametrize("kw,word", CALL_BAD)
def test_attention_struct_refuses(kw, word):
    with pytest.raises(ValueError, match=word):
        call(**kw)


def test_attention_struct_needs_pairs():
    q = torch.zeros(6, 8, 64, dtype=BF)
    pk, k = torch.zeros(2, 4, 100, 64, dtype=BF), torch.zeros(6, 4, 10, 64, dtype=BF)
    for args, kw in (((None, pk, k, k), {}), ((pk, pk, k, None), {}), ((None, None, k, k), {}),
                     ((pk, pk, None, None), dict(lengths=torch.zeros(6, dtype=I32))),
                     ((pk, pk, None, None), dict(weight=torch.zeros(6, 4, 10)))):
        with pytest.raises(ValueError):
            S.attention_struct(torch, CPU, q, *args, q.clone(), **kw)


def ecall(keys=None, values=None, weight=None, budget=5, out=None, **kw):
    keys = [torch.zeros(3, 2, 10, 16, dtype=BF) for _ in range(2)] if keys is None else keys
    values = [torch.zeros(3, 2, 10, 16, dtype=BF) for _ in range(2)] if values is None else values
    weight = torch.zeros(2, 3, 2, 10) if weight is None else weight
    out = S.EvictResult(torch.zeros(2, 3, 2, 10), torch.zeros(2, 3, 2, 10, dtype=I32), torch.zeros(3, dtype=I32)) if out is None else out
    return S.evict_struct(torch, CPU, keys, values, weight, budget, out, **kw)


def test_evict_struct():
    both = torch.zeros(2, 2, 3, 10, 2, 16, dtype=BF).transpose(3, 4)   # [2, layers, segments, heads, positions, dim]
    e = ecall(keys=list(both[0]), values=list(both[1]), keep_first=1, keep_recent=2)
    assert (e.layers, e.segments, e.heads, e.capacity, e.budget, e.keep_first, e.keep_recent) == (2, 3, 2, 10, 5, 1, 2)
    assert (e.segment_stride, e.head_stride, e.position_stride, e.position_bytes) == (10 * 64, 32, 64, 32)
    assert e.caches[1].keys == both[0, 1].data_ptr() and e.caches[0].values == both[1, 0].data_ptr()
    e = S.evict_struct(torch, CPU, list(both[0]), None, torch.zeros(2, 3, 2, 10), 5,
                       S.EvictResult(torch.zeros(2, 3, 2, 10), None, None))
    assert not e.caches[0].values and not e.index_out and not e.lengths_out


SAME = torch.zeros(3, 2, 10, 16, dtype=BF)


@pytest.mark.parametrize("kw,word", [
    (dict(keys=[SAME]), "each of the 2"), (dict(keys=[SAME, SAME]), "twice"), (dict(weight=torch.zeros(3, 2, 10)), "weight"),
    (dict(weight=torch.zeros(2, 3, 2, 20)[..., ::2]), "contiguous"), (dict(keys=[SAME, torch.zeros(3, 2, 10, 8, dtype=BF)]), "a cache"),
    (dict(keys=[SAME, torch.zeros(3, 2, 10, 16)]), "a cache"), (dict(keys=[SAME, torch.zeros(3, 2, 12, 16, dtype=BF)[:, :, :10]]), "strides"),
    (dict(keys=[SAME, torch.zeros(3, 2, 10, 32, dtype=BF)[..., ::2]]), "consecutive"), (dict(index=torch.zeros(2, 3, 2, 10)), "index"),
    (dict(lengths=torch.zeros(2, dtype=I32)), "lengths"), (dict(budget=1 << 32), "budget"), (dict(budget=-1), "budget"),
    (dict(keep_recent=-1), "keep_recent")])
def test_evict_struct_refuses(kw, word):
    with pytest.raises(ValueError, match=word):
        ecall(**kw)
