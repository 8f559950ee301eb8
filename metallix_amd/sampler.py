"""ctypes binding of libmx_sampler.so (include/mx_sampler.h).

`Sampler` mirrors the reference's device-pick plugin: one handle owns the
kernels and scratch (mlx_kernels::MetalKernel, crates/metal/mlx-kernels/src/
lib.rs:203-215); `sample` queues a batched pick on the stream like
Qwen3TokenPicks::start_with (crates/models/qwen/src/forward/picks.rs:279-381)
and returns device tensors the caller reads back after synchronising, the
Qwen3TokenPicks::wait step (picks.rs:390-401).  Per-row statuses mirror
engine::sampling::SamplingError (crates/core/engine/src/sampling.rs:19-43).
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from pathlib import Path
from typing import Optional, Sequence

LIB_PATH = Path(__file__).resolve().parent / "_build" / "libmx_sampler.so"

MXS_F32 = 0
MXS_BF16 = 1

ROW_STATUS = {
    0: "ok",
    1: "uncertified",
    -1: "EmptyLogits",
    -2: "MaskLengthMismatch",
    -3: "EmptySupport",
    -4: "InvalidTemperature",
    -5: "InvalidUniform",
    -6: "NonFiniteLogit",
    -7: "VocabularyTooLarge",
    -8: "InvalidTopP",
    -9: "InvalidMinP",
    -10: "InvalidPenalty",
    -11: "InvalidHistory",
    -12: "InvalidBias",
    -13: "TokenOutOfRange",
    -14: "Probabilities",
    -15: "UnsupportedRule",   # mxs_finish_tiles: a rule other than greedy or top-k
    -16: "InvalidParent",     # mxs_beam_reorder: a parent outside the group
}

_vp = ctypes.c_void_p


class MxsBatch(ctypes.Structure):
    _fields_ = [
        ("logits", _vp), ("dtype", ctypes.c_int32), ("rows", ctypes.c_uint32),
        ("vocab", ctypes.c_uint32), ("row_stride", ctypes.c_uint64),
        ("temperature", _vp), ("top_k", _vp), ("top_p", _vp), ("min_p", _vp),
        ("repetition", _vp), ("presence", _vp), ("frequency", _vp), ("uniform", _vp),
        ("history_offsets", _vp), ("history_ids", _vp),
        ("bias_offsets", _vp), ("bias_ids", _vp), ("bias_values", _vp),
        ("mask_words", _vp), ("mask_stride", ctypes.c_uint64),
        ("tokenizer_vocab", ctypes.c_uint32), ("reserved", ctypes.c_uint32),
    ]


class MxsOut(ctypes.Structure):
    _fields_ = [
        ("token", _vp), ("sampling_logprob", _vp), ("status", _vp),
        ("kept_count", _vp), ("adjusted", _vp), ("kept_bits", _vp),
    ]


class MxsRace(ctypes.Structure):
    _fields_ = [("seed", _vp), ("choice", _vp), ("position", _vp)]


class MxsReceipts(ctypes.Structure):
    _fields_ = [
        ("top", _vp), ("n", ctypes.c_uint32), ("reserved", ctypes.c_uint32),
        ("ids", _vp), ("logprobs", _vp), ("token_logprob", _vp), ("status", _vp),
    ]


class MxsBeam(ctypes.Structure):
    _fields_ = [
        ("logits", _vp), ("dtype", ctypes.c_int32), ("groups", ctypes.c_uint32), ("beams", ctypes.c_uint32),
        ("vocab", ctypes.c_uint32), ("row_stride", ctypes.c_uint64),
        ("score", _vp), ("ended", _vp), ("scale", _vp),
        ("mask_words", _vp), ("mask_stride", ctypes.c_uint64), ("tokenizer_vocab", ctypes.c_uint32),
        ("legal_norm", ctypes.c_uint32), ("n", ctypes.c_uint32), ("end_token", ctypes.c_int32),
    ]


class MxsBeamOut(ctypes.Structure):
    _fields_ = [("token", _vp), ("beam", _vp), ("score", _vp), ("ended", _vp), ("status", _vp)]


class MxsState(ctypes.Structure):
    _fields_ = [
        ("data", _vp), ("row_stride", ctypes.c_uint64), ("segment_stride", ctypes.c_uint64),
        ("segment_bytes", ctypes.c_uint64), ("position_bytes", ctypes.c_uint64),
        ("segments", ctypes.c_uint32), ("reserved", ctypes.c_uint32),
    ]


class MxsReorder(ctypes.Structure):
    _fields_ = [
        ("states", ctypes.POINTER(MxsState)), ("count", ctypes.c_uint32), ("groups", ctypes.c_uint32),
        ("beams", ctypes.c_uint32), ("parent_stride", ctypes.c_uint32), ("parent", _vp), ("lengths", _vp),
        ("status", _vp),
    ]


class MxsLinear(ctypes.Structure):
    _fields_ = [
        ("x", _vp), ("x_stride", ctypes.c_uint64), ("weight", _vp), ("weight_stride", ctypes.c_uint64),
        ("bias", _vp), ("residual", _vp), ("residual_stride", ctypes.c_uint64), ("out", _vp),
        ("out_stride", ctypes.c_uint64), ("rows", ctypes.c_uint32), ("in_features", ctypes.c_uint32),
        ("out_features", ctypes.c_uint32), ("act", ctypes.c_int32), ("out_dtype", ctypes.c_int32),
        ("bias_dtype", ctypes.c_int32),
    ]


class MxsAttention(ctypes.Structure):
    _fields_ = [
        ("q", _vp), ("q_row", ctypes.c_uint64), ("q_token", ctypes.c_uint64), ("q_head", ctypes.c_uint64),
        ("prefix_keys", _vp), ("prefix_values", _vp), ("prefix_group", ctypes.c_uint64),
        ("prefix_head", ctypes.c_uint64), ("prefix_position", ctypes.c_uint64), ("prefix_lengths", _vp),
        ("keys", _vp), ("values", _vp), ("row", ctypes.c_uint64), ("head", ctypes.c_uint64),
        ("position", ctypes.c_uint64), ("lengths", _vp),
        ("out", _vp), ("out_row", ctypes.c_uint64), ("out_token", ctypes.c_uint64), ("out_head", ctypes.c_uint64),
        ("lse", _vp), ("prefix_weight", _vp), ("weight", _vp),
        ("groups", ctypes.c_uint32), ("beams", ctypes.c_uint32), ("tokens", ctypes.c_uint32),
        ("heads", ctypes.c_uint32), ("kv_heads", ctypes.c_uint32), ("dim", ctypes.c_uint32),
        ("prefix", ctypes.c_uint32), ("suffix", ctypes.c_uint32), ("scale", ctypes.c_float),
        ("reserved", ctypes.c_uint32),
    ]


class MxsCache(ctypes.Structure):
    _fields_ = [("keys", _vp), ("values", _vp)]


class MxsEvict(ctypes.Structure):
    _fields_ = [
        ("caches", ctypes.POINTER(MxsCache)), ("layers", ctypes.c_uint32), ("segments", ctypes.c_uint32),
        ("heads", ctypes.c_uint32), ("capacity", ctypes.c_uint32), ("segment_stride", ctypes.c_uint64),
        ("head_stride", ctypes.c_uint64), ("position_stride", ctypes.c_uint64), ("position_bytes", ctypes.c_uint32),
        ("budget", ctypes.c_uint32), ("keep_first", ctypes.c_uint32), ("keep_recent", ctypes.c_uint32),
        ("weight", _vp), ("index", _vp), ("lengths", _vp), ("weight_out", _vp), ("index_out", _vp),
        ("lengths_out", _vp),
    ]


# Exported symbols and their prototypes, as declared in include/mx_sampler.h.
PROTOTYPES = {
    "mxs_abi_version": (ctypes.c_int, []),
    "mxs_status_string": (ctypes.c_char_p, [ctypes.c_int32]),
    "mxs_create": (ctypes.c_int, [ctypes.c_int, _vp, ctypes.c_uint32, ctypes.c_uint32, ctypes.POINTER(_vp)]),
    "mxs_destroy": (ctypes.c_int, [_vp]),
    "mxs_set_stream": (ctypes.c_int, [_vp, _vp]),
    "mxs_sample": (ctypes.c_int, [_vp, ctypes.POINTER(MxsBatch), ctypes.POINTER(MxsOut)]),
    "mxs_sample_race": (ctypes.c_int, [_vp, ctypes.POINTER(MxsBatch), ctypes.POINTER(MxsRace),
                                       ctypes.POINTER(MxsOut)]),
    "mxs_logsoftmax_topn": (ctypes.c_int, [_vp, _vp, ctypes.c_int32, ctypes.c_uint32, ctypes.c_uint32,
                                           ctypes.c_uint64, ctypes.c_uint32, _vp, _vp, _vp, _vp, _vp]),
    "mxs_logsoftmax_topn_noalloc": (ctypes.c_int, [_vp, _vp, ctypes.c_int32, ctypes.c_uint32, ctypes.c_uint32,
                                                   ctypes.c_uint64, ctypes.c_uint32, _vp, _vp, _vp, _vp, _vp]),
    "mxs_spec_verify": (ctypes.c_int, [_vp, _vp, _vp, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint32,
                                       _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "mxs_step": (ctypes.c_int, [_vp, ctypes.POINTER(MxsBatch), ctypes.POINTER(MxsRace), ctypes.POINTER(MxsOut),
                                ctypes.POINTER(MxsReceipts)]),
    "mxs_mask_host": (ctypes.c_int, [_vp, ctypes.c_uint32, ctypes.POINTER(_vp), ctypes.POINTER(ctypes.c_uint64)]),
    "mxs_mask_upload": (ctypes.c_int, [_vp, ctypes.c_uint32, ctypes.c_uint32, ctypes.POINTER(_vp)]),
    "mxs_sync": (ctypes.c_int, [_vp]),
    "mxs_export_candidates": (ctypes.c_int, [_vp, ctypes.c_uint32, ctypes.c_uint32, _vp, _vp, _vp]),
    "mxs_lmhead_bf16": (ctypes.c_int, [_vp, _vp, _vp, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint32, _vp,
                                       ctypes.c_uint64, _vp]),
    "mxs_finish_tiles": (ctypes.c_int, [_vp, ctypes.POINTER(MxsBatch), _vp, ctypes.POINTER(MxsOut)]),
    "mxs_beam_select": (ctypes.c_int, [_vp, ctypes.POINTER(MxsBeam), ctypes.POINTER(MxsBeamOut)]),
    "mxs_beam_reorder": (ctypes.c_int, [_vp, ctypes.POINTER(MxsReorder)]),
    "mxs_beam_reorder_check": (ctypes.c_int, [_vp, ctypes.POINTER(MxsReorder)]),
    "mxs_linear_bf16": (ctypes.c_int, [_vp, ctypes.POINTER(MxsLinear)]),
    "mxs_prefix_attention": (ctypes.c_int, [_vp, ctypes.POINTER(MxsAttention)]),
    "mxs_prefix_attention_counted": (ctypes.c_int, [_vp, ctypes.POINTER(MxsAttention), _vp]),
    "mxs_cache_evict": (ctypes.c_int, [_vp, ctypes.POINTER(MxsEvict)]),
    "mxs_debug_set_timing": (ctypes.c_int, [_vp, _vp]),
    "mxs_debug_floor": (ctypes.c_int, [_vp, _vp, ctypes.c_int32, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint32,
                                       ctypes.c_uint32, _vp, _vp]),
    "mxs_debug_set_paths": (ctypes.c_int, [_vp, _vp]),
    "mxs_last_error": (ctypes.c_char_p, [_vp]),
}

_LIB = None


class SamplerError(RuntimeError):
    pass


ABI_VERSION = 2                 # MXS_ABI_VERSION of include/mx_sampler.h
RECEIPT_NONE = 0xFFFFFFFF       # MXS_RECEIPT_NONE: a receipt_top entry for "no receipt"
TILE_TOKENS = 256               # MXS_TILE_TOKENS: vocabulary entries per epilogue-statistics tile
TILE_STAT_BYTES = 8             # MXS_TILE_STAT_BYTES: bytes per (row, tile)


BEAM_MAX = 64                   # MXS_BEAM_MAX: beams per group
BEAM_N_MAX = 128                # MXS_BEAM_N_MAX: candidates per group
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}   # MXS_ACT_*


def load_library(path: Optional[Path] = None):
    """Loads the built library; raises when it is missing (no fallback)."""
    global _LIB
    if _LIB is not None and path is None:
        return _LIB
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise SamplerError(f"{p} is not built: run `python -m metallix_amd.build` (hipcc, gfx950)")
    lib = ctypes.CDLL(str(p))
    for name, (res, args) in PROTOTYPES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if lib.mxs_abi_version() != ABI_VERSION:
        raise SamplerError(f"{p} implements ABI {lib.mxs_abi_version()}, these bindings ABI {ABI_VERSION}: rebuild")
    if path is None:
        _LIB = lib
    return lib


def with_suppression(rows: int, suppress_ids, bias_offsets=None, bias_ids=None, bias_values=None, *,
                     vocab: Optional[int] = None):
    """Host-side CSR for the sampler's bias stage with the checkpoint's
    suppressed tokens merged in (ChatFormat::suppress,
    crates/core/chat-format/src/lib.rs:761-780): every row gets a -inf entry
    for each id of `suppress_ids` (ids are per checkpoint, the same for every
    row), which the sampler turns into an adjusted logit of f32::MIN.  A
    suppressed id keeps no bias of its own.  An id at or past `vocab` (the
    logit row's length) is skipped, as the reference's `logits.get_mut`
    returns None for it (:771-778); without `vocab` every id is kept, and the
    sampler reports one past the row as an invalid bias entry.  Returns
    numpy (offsets u32[rows + 1], ids u32, values f32), ids strictly
    increasing within a row."""
    import numpy as np

    sup = np.unique(np.asarray(suppress_ids, dtype=np.int64))
    if vocab is not None:
        sup = sup[(sup >= 0) & (sup < int(vocab))]
    sup = sup.astype(np.uint32)
    offs, ids, vals = [0], [], []
    for r in range(rows):
        if bias_offsets is not None:
            b0, b1 = int(bias_offsets[r]), int(bias_offsets[r + 1])
            bi = np.asarray(bias_ids[b0:b1], dtype=np.uint32)
            bv = np.asarray(bias_values[b0:b1], dtype=np.float32)
            keep = ~np.isin(bi, sup)
            bi, bv = bi[keep], bv[keep]
        else:
            bi, bv = np.zeros(0, np.uint32), np.zeros(0, np.float32)
        ri = np.concatenate([bi, sup])
        rv = np.concatenate([bv, np.full(sup.size, -np.inf, dtype=np.float32)])
        order = np.argsort(ri, kind="stable")
        ids.append(ri[order])
        vals.append(rv[order])
        offs.append(offs[-1] + ri.size)
    return (np.asarray(offs, dtype=np.uint32), np.concatenate(ids).astype(np.uint32),
            np.concatenate(vals).astype(np.float32))


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _need(t, name: str, device, dtypes, shape) -> None:
    """Raises ValueError unless `t` is a tensor on `device` of one of the
    dtypes and of the shape (None: any size)."""
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, not {t.device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, not {t.dtype}")
    if t.dim() != len(shape) or any(want is not None and got != want for got, want in zip(t.shape, shape)):
        raise ValueError(f"{name} must have the shape {list(shape)}, not {list(t.shape)}")


def _dense(t, name: str) -> None:
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _u32(v, name: str) -> int:
    """v as the ABI's 32-bit count; ctypes would keep its low bits only."""
    v = int(v)
    if not 0 <= v < 1 << 32:
        raise ValueError(f"{name} must be in 0..2^32 - 1, not {v}")
    return v


def _float_code(torch, dtype) -> int:
    return MXS_BF16 if dtype == torch.bfloat16 else MXS_F32


def beam_struct(torch, device, logits, score, n: int, *, ended=None, end_token: Optional[int] = None, scale=None,
                mask=None, tokenizer_vocab: Optional[int] = None, legal_norm: bool = False,
                vocab: Optional[int] = None) -> MxsBeam:
    """The mxs_beam of a call, its tensors checked against `device` and each
    other (ValueError)."""
    _need(score, "score", device, (torch.float64,), (None, None))
    groups, beams = score.shape
    V = logits.shape[-1] if vocab is None else int(vocab)
    _need(logits, "logits", device, (torch.float32, torch.bfloat16), (groups * beams, None))
    if not 0 < V <= logits.shape[1] or logits.stride(1) != 1:
        raise ValueError("logits rows must hold `vocab` consecutive elements")
    _dense(score, "score")
    if ended is not None:
        _need(ended, "ended", device, (torch.bool, torch.uint8), (groups, beams))
        _dense(ended, "ended")
    if scale is not None:
        _need(scale, "scale", device, (torch.float64,), (groups, beams))
        _dense(scale, "scale")
    b = MxsBeam()
    b.logits, b.dtype = logits.data_ptr(), _float_code(torch, logits.dtype)
    b.groups, b.beams, b.vocab = _u32(groups, "groups"), _u32(beams, "beams"), _u32(V, "vocab")
    # (a single row's stride says nothing: any multiple of 4 that holds it)
    b.row_stride = logits.stride(0) if groups * beams > 1 else (V + 3) // 4 * 4
    b.score, b.ended, b.scale = score.data_ptr(), _ptr(ended), _ptr(scale)
    if mask is not None:
        if not isinstance(mask, DeviceWords):
            _need(mask, "mask", device, (torch.int32,), (groups * beams, None))
            if mask.shape[1] < (V + 31) // 32 or mask.stride(1) != 1:
                raise ValueError("mask rows must hold ceil(vocab / 32) consecutive words")
        elif mask.rows < groups * beams:
            raise ValueError("mask holds fewer rows than the batch")
        b.mask_words = mask.data_ptr()
        b.mask_stride = mask.stride(0) if groups * beams > 1 else (V + 31) // 32
        b.tokenizer_vocab = V if tokenizer_vocab is None else _u32(tokenizer_vocab, "tokenizer_vocab")
    b.legal_norm = 1 if legal_norm else 0
    b.n = _u32(n, "n")
    b.end_token = -1 if end_token is None else int(end_token)
    if end_token is not None and b.end_token != int(end_token):
        raise ValueError(f"end_token must be a token of the vocabulary, not {end_token}")
    return b


def beam_out_struct(torch, device, out, groups: int, n: int) -> MxsBeamOut:
    """The mxs_beam_out of a call's outputs, checked against `device` and the
    sizes (ValueError)."""
    for name, dts in (("token", (torch.int32,)), ("beam", (torch.int32,)), ("score", (torch.float64,)),
                      ("ended", (torch.bool, torch.uint8))):
        t = getattr(out, name)
        if t is not None or name != "ended":
            _need(t, f"out.{name}", device, dts, (groups, n))
            _dense(t, f"out.{name}")
    _need(out.status, "out.status", device, (torch.int32,), (groups,))
    _dense(out.status, "out.status")
    o = MxsBeamOut()
    o.token, o.beam, o.score = out.token.data_ptr(), out.beam.data_ptr(), out.score.data_ptr()
    o.ended, o.status = _ptr(out.ended), out.status.data_ptr()
    return o


def state_struct(t, rows: int, length_dim: Optional[int] = None) -> MxsState:
    """The mxs_state of a tensor whose dimension 0 is the rows: the pieces of
    a row from `length_dim` on (or the longest run of dimensions that lie
    consecutively in memory), one per index of the dimensions before, which
    must be evenly spaced; the dimensions are taken in the order of their
    strides.  ValueError for any other layout."""
    if t.dim() < 1 or t.shape[0] != rows:
        raise ValueError(f"a state must have {rows} rows, not {list(t.shape)}")
    size, stride = list(t.shape), list(t.stride())
    if 0 in size:
        raise ValueError("a state must not be empty")
    es, nd = t.element_size(), t.dim()
    if length_dim is not None and not 1 <= length_dim < nd:
        raise ValueError(f"length_dim must be in 1..{nd - 1}")

    if not t.is_contiguous():
        # Largest stride first, as [rows, positions, heads, dim] seen as [rows,
        # heads, positions, dim] lies in memory; a dimension of one index goes
        # with the one after it.  (Stride 0, rows on top of one another, is
        # refused later.)
        by = stride + [1]
        for d in range(nd - 1, 0, -1):
            if size[d] == 1:
                by[d] = by[d + 1]
        if all(by[1:nd]):
            order = [0, *sorted(range(1, nd), key=lambda d: -by[d])]
            size, stride = [size[d] for d in order], [stride[d] for d in order]
            length_dim = None if length_dim is None else order.index(length_dim)

    def run(d):   # elements of dimensions d.. when they are consecutive, else 0
        n = 1
        for i in range(nd - 1, d - 1, -1):
            if size[i] != 1 and stride[i] != n:
                return 0
            n *= size[i]
        return n

    if length_dim is None:
        first = nd
        while first > 1 and run(first - 1):
            first -= 1
    else:
        first = length_dim
        if not run(first):
            raise ValueError("a state's elements from length_dim on must be consecutive")
    outer = [(n, s) for n, s in zip(size[1:first], stride[1:first]) if n != 1]
    for (_, s), (n1, s1) in zip(outer, outer[1:]):
        if s != n1 * s1:
            raise ValueError("a state's dimensions before its pieces must be evenly spaced")
    m = MxsState()
    m.data = t.data_ptr()
    m.segment_bytes = run(first) * es
    m.segments = _u32(math.prod(n for n, _ in outer), "a state's pieces")
    m.segment_stride = outer[-1][1] * es if outer else m.segment_bytes
    m.row_stride = stride[0] * es if rows > 1 else m.segments * m.segment_stride
    m.position_bytes = 0 if length_dim is None else run(first) * es // size[first]
    return m


def reorder_struct(torch, device, states, parent, status, *, beams: Optional[int] = None, lengths=None,
                   length_dim=None) -> MxsReorder:
    """The mxs_reorder of a call, its tensors checked against `device` and
    each other (ValueError)."""
    _need(parent, "parent", device, (torch.int32,), (None, None))
    groups = parent.shape[0]
    W = parent.shape[1] if beams is None else int(beams)
    if not 0 < W <= parent.shape[1] or (parent.shape[1] > 1 and parent.stride(1) != 1):
        raise ValueError("parent rows must hold `beams` consecutive entries")
    _need(status, "status", device, (torch.int32,), (groups,))
    _dense(status, "status")
    if lengths is not None:
        _need(lengths, "lengths", device, (torch.int32,), (groups,))
        _dense(lengths, "lengths")
    dims = list(length_dim) if isinstance(length_dim, (list, tuple)) else [length_dim] * len(states)
    if len(dims) != len(states):
        raise ValueError("length_dim must be one dimension or one per state")
    at = [t.data_ptr() for t in states]
    if len(set(at)) != len(at):
        raise ValueError("a state is given twice: its rows would move twice at once")
    arr = (MxsState * max(1, len(states)))()
    last = None   # a cache's layers share one layout
    for i, (t, d, p) in enumerate(zip(states, dims, at)):
        if t.device != device:
            raise ValueError(f"states must be on {device}, not {t.device}")
        like = (t.shape, t.stride(), t.dtype, d)
        if like != last:
            m, last = state_struct(t, groups * W, d), like
        m.data = p
        arr[i] = m
    r = MxsReorder()
    r.states, r.count = ctypes.cast(arr, ctypes.POINTER(MxsState)), len(states)
    r.groups, r.beams = _u32(groups, "groups"), W
    r.parent = parent.data_ptr()
    r.parent_stride = _u32(parent.stride(0) if groups > 1 else parent.shape[1], "parent's row stride")
    r.lengths, r.status = _ptr(lengths), status.data_ptr()
    r.keep = arr
    return r


def linear_struct(torch, device, x, weight, bias, residual, out, activation) -> MxsLinear:
    """The mxs_linear of a call, its tensors checked against `device` and each
    other (ValueError)."""
    _need(x, "x", device, (torch.bfloat16,), (None, None))
    R, K = x.shape
    _need(weight, "weight", device, (torch.bfloat16,), (None, K))
    N = weight.shape[0]
    _need(out, "out", device, (torch.bfloat16, torch.float32), (R, N))
    if bias is not None:
        _need(bias, "bias", device, (torch.bfloat16, torch.float32), (N,))
        _dense(bias, "bias")
    if residual is not None:
        _need(residual, "residual", device, (out.dtype,), (R, N))
    for t, name in ((x, "x"), (weight, "weight"), (out, "out"), (residual, "residual")):
        if t is not None and t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"{name} rows must be consecutive elements")
    act = ACTIVATIONS.get("none" if activation is None else activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}")
    # a single row's stride says nothing
    rows_of = lambda t, unit: t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // unit) * unit
    a = MxsLinear()
    a.x, a.x_stride = x.data_ptr(), rows_of(x, 8)
    a.weight, a.weight_stride = weight.data_ptr(), rows_of(weight, 8)
    a.bias, a.residual = _ptr(bias), _ptr(residual)
    a.residual_stride = rows_of(residual, 1) if residual is not None else 0
    a.out, a.out_stride = out.data_ptr(), rows_of(out, 1)
    a.rows, a.in_features, a.out_features = _u32(R, "rows"), _u32(K, "in_features"), _u32(N, "out_features")
    a.act = act
    a.out_dtype = _float_code(torch, out.dtype)
    a.bias_dtype = _float_code(torch, bias.dtype) if bias is not None else MXS_F32
    return a


def _cache_pair(torch, device, keys, values, names, shape, dtypes):
    """Strides of dimensions 0 to 2 of two like caches of 4 dimensions, the last
    of them consecutive; a dimension of one index has stride 0."""
    for t, name in ((keys, names[0]), (values, names[1])):
        _need(t, name, device, dtypes, shape)
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise ValueError(f"{name}: a position's elements must be consecutive")
    st = lambda t: [s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3])]
    if values.shape != keys.shape or values.dtype != keys.dtype or st(values) != st(keys):
        raise ValueError(f"{names[0]} and {names[1]} must have the same type, shape and strides")
    return st(keys)


def attention_struct(torch, device, q, prefix_keys, prefix_values, keys, values, out, *, prefix_lengths=None,
                     lengths=None, scale=None, lse=None, prefix_weight=None, weight=None, counted=None) -> MxsAttention:
    """The mxs_attention of a call (and, as its attribute, the address of
    `counted`), its tensors checked against `device` and each other (ValueError)."""
    bf = (torch.bfloat16,)
    if q.dim() not in (3, 4):
        raise ValueError(f"q must have the shape [rows, (tokens,) heads, dim], not {list(q.shape)}")
    _need(q, "q", device, bf, (None,) * q.dim())
    _need(out, "out", device, bf, tuple(q.shape))
    if lse is not None:
        _need(lse, "lse", device, (torch.float32,), tuple(q.shape[:-1]))
        _dense(lse, "lse")
    if q.dim() == 3:
        q, out = q.unsqueeze(1), out.unsqueeze(1)
    rows, tokens, heads, dim = q.shape
    for t, name in ((q, "q"), (out, "out")):
        if dim > 1 and t.stride(3) != 1:
            raise ValueError(f"{name}: a head's elements must be consecutive")
    if (prefix_keys is None) != (prefix_values is None) or (keys is None) != (values is None):
        raise ValueError("keys and values come together")
    if prefix_keys is None:
        raise ValueError("a prefix is required (of no positions, where there is none)")
    if prefix_keys.dim() != 4:
        raise ValueError(f"prefix_keys must have the shape [groups, kv_heads, positions, dim], not {list(prefix_keys.shape)}")
    groups, kv, P, _ = prefix_keys.shape
    a = MxsAttention()
    a.prefix_group, a.prefix_head, a.prefix_position = _cache_pair(
        torch, device, prefix_keys, prefix_values, ("prefix_keys", "prefix_values"), (None, None, None, dim), bf)
    if rows and (groups == 0 or rows % groups):
        raise ValueError(f"q's {rows} rows must be the same number for each of the {groups} groups")
    N = 0
    if keys is not None:
        a.row, a.head, a.position = _cache_pair(torch, device, keys, values, ("keys", "values"), (rows, kv, None, dim), bf)
        N = keys.shape[2]
        if N:
            a.keys, a.values = keys.data_ptr(), values.data_ptr()
    elif lengths is not None or weight is not None:
        raise ValueError("lengths and weight need keys and values")
    for t, name, shape, dt in ((prefix_lengths, "prefix_lengths", (groups,), torch.int32),
                               (lengths, "lengths", (rows,), torch.int32),
                               (prefix_weight, "prefix_weight", (groups, kv, P), torch.float32),
                               (weight, "weight", (rows, kv, N), torch.float32)):
        if t is not None:
            _need(t, name, device, (dt,), shape)
            _dense(t, name)
    if counted is not None:
        _need(counted, "counted", device, (torch.bool, torch.uint8), (rows,))
        _dense(counted, "counted")
    a.counted = _ptr(counted)
    st = lambda t: [s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3])]
    a.q, (a.q_row, a.q_token, a.q_head) = q.data_ptr(), st(q)
    a.out, (a.out_row, a.out_token, a.out_head) = out.data_ptr(), st(out)
    if P:
        a.prefix_keys, a.prefix_values = prefix_keys.data_ptr(), prefix_values.data_ptr()
        a.prefix_weight = _ptr(prefix_weight)
    if N:
        a.weight = _ptr(weight)
    a.prefix_lengths, a.lengths, a.lse = _ptr(prefix_lengths), _ptr(lengths), _ptr(lse)
    a.groups, a.beams = _u32(groups, "groups"), _u32(rows // groups if groups else 0, "beams")
    a.tokens, a.heads, a.kv_heads, a.dim = _u32(tokens, "tokens"), _u32(heads, "heads"), _u32(kv, "kv_heads"), _u32(dim, "dim")
    a.prefix, a.suffix = _u32(P, "prefix"), _u32(N, "suffix")
    a.scale = float(scale) if scale is not None else dim ** -0.5 if dim else 0.0   # (dim 0 is refused by the call)
    return a


def evict_struct(torch, device, keys, values, weight, budget, out, *, index=None, lengths=None, keep_first: int = 0,
                 keep_recent: int = 0) -> MxsEvict:
    """The mxs_evict of a call, its tensors checked against `device` and each
    other (ValueError)."""
    keys, values = list(keys), None if values is None else list(values)
    _need(weight, "weight", device, (torch.float32,), (None,) * 4)
    L, S, H, C = weight.shape
    if len(keys) != L or (values is not None and len(values) != L):
        raise ValueError(f"keys and values must hold one cache for each of the {L} layers")
    for t, name, shape, dt in ((weight, "weight", (L, S, H, C), torch.float32), (index, "index", (L, S, H, C), torch.int32),
                               (lengths, "lengths", (S,), torch.int32), (out.weight, "out.weight", (L, S, H, C), torch.float32),
                               (out.index, "out.index", (L, S, H, C), torch.int32),
                               (out.lengths, "out.lengths", (S,), torch.int32)):
        if t is not None:
            _need(t, name, device, (dt,), shape)
            _dense(t, name)
    every = keys + (values or [])
    if len({t.data_ptr() for t in every}) != len(every) and 0 not in weight.shape:
        raise ValueError("a cache is given twice: its positions would move twice at once")
    e = MxsEvict()
    arr = (MxsCache * max(1, L))()
    st = None
    for i, t in enumerate(every):
        _need(t, "a cache", device, (every[0].dtype,), (S, H, C, every[0].shape[3] if every[0].dim() == 4 else None))
        mine = [s if n > 1 else 0 for n, s in zip(t.shape, t.stride())]
        if t.shape[3] > 1 and t.stride(3) != 1:
            raise ValueError("a cache's elements of a position must be consecutive")
        if st is None:
            st = mine
        if mine != st:
            raise ValueError("the caches must have the same strides")
        if i < L:
            arr[i].keys = t.data_ptr()
        else:
            arr[i - L].values = t.data_ptr()
    es = every[0].element_size() if every else 1
    e.caches, e.layers, e.segments, e.heads = ctypes.cast(arr, ctypes.POINTER(MxsCache)), L, S, H
    e.capacity = _u32(C, "capacity")
    if every:
        e.segment_stride, e.head_stride, e.position_stride = (s * es for s in st[:3])
        e.position_bytes = _u32(every[0].shape[3] * es, "position_bytes")
    e.budget, e.keep_first, e.keep_recent = _u32(budget, "budget"), _u32(keep_first, "keep_first"), _u32(keep_recent, "keep_recent")
    e.weight, e.index, e.lengths = weight.data_ptr(), _ptr(index), _ptr(lengths)
    e.weight_out, e.index_out, e.lengths_out = out.weight.data_ptr(), _ptr(out.index), _ptr(out.lengths)
    e.keep = arr
    return e


class DeviceWords:
    """A staging slot's device mask words, as `Sampler.sample(mask=...)`
    takes them (a data pointer and a row stride in words)."""

    def __init__(self, ptr: int, stride: int, rows: int):
        self.ptr, self.stride_words, self.rows = ptr, stride, rows

    def data_ptr(self) -> int:
        return self.ptr

    def stride(self, dim: int) -> int:
        assert dim == 0
        return self.stride_words


@dataclass
class ReceiptResult:
    """Device tensors of one step's receipts (mxs_receipts)."""
    ids: "object"
    logprobs: "object"
    token_logprob: "object"
    status: "object"


@dataclass
class BeamResult:
    """Device tensors of one selection (mxs_beam_out), [groups, n] and, the
    status, [groups]."""
    token: "object"
    beam: "object"
    score: "object"
    ended: "object"
    status: "object"


@dataclass
class EvictResult:
    """Device tensors of one eviction (mxs_evict): the slots' weights and
    positions, [layers, segments, heads, capacity], and the new lengths,
    [segments]."""
    weight: "object"
    index: "object"
    lengths: "object"


@dataclass
class SampleResult:
    token: "object"
    sampling_logprob: "object"
    status: "object"
    kept_count: "object"
    adjusted: "object" = None
    kept_bits: "object" = None


class Sampler:
    """One sampler context on one GPU and stream (not thread-safe)."""

    def __init__(self, max_rows: int, max_vocab: int, device: int = 0, stream=None):
        import torch

        if not torch.cuda.is_available():
            raise SamplerError("no GPU visible: the HIP sampler has no CPU path")
        self.torch = torch
        self.lib = load_library()
        self.device = device
        self.stream = stream if stream is not None else torch.cuda.current_stream(device)
        ctx = _vp()
        rc = self.lib.mxs_create(device, _vp(self.stream.cuda_stream), max_rows, max_vocab, ctypes.byref(ctx))
        if rc != 0:
            raise SamplerError(f"mxs_create failed: {rc}")
        self.ctx = ctx
        self.max_rows = max_rows
        self.max_vocab = max_vocab

    def close(self):
        if getattr(self, "ctx", None):
            self.lib.mxs_destroy(self.ctx)
            self.ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc: int, what: str):
        if rc != 0:
            msg = self.lib.mxs_last_error(self.ctx)
            raise SamplerError(f"{what} failed ({rc}): {msg.decode() if msg else ''}")

    def sample(self, logits, temperature, *, top_k=None, top_p=None, min_p=None, repetition=None,
               presence=None, frequency=None, uniform=None, history=None, bias=None, mask=None,
               tokenizer_vocab=None, debug: bool = False, out: Optional[SampleResult] = None,
               vocab: Optional[int] = None, race=None) -> SampleResult:
        """Queues one batched pick.  All tensor arguments live on the GPU.

        history: (offsets u32[rows+1], ids u32) CSR; bias: (offsets, ids, values f32);
        mask: u32[rows, mask_stride].
        race: (seed u64 as int64[rows], choice u32[rows] or None, position u32[rows])
        selects race-v2 (Qwen3Selection::Race, picks.rs:40-66) instead of the
        inverse-CDF draw; `uniform` is then unused.
        """
        b, o, r, out = self._structs(logits, temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                                     repetition=repetition, presence=presence, frequency=frequency, uniform=uniform,
                                     history=history, bias=bias, mask=mask, tokenizer_vocab=tokenizer_vocab,
                                     debug=debug, out=out, vocab=vocab, race=race)
        if r is not None:
            self._check(self.lib.mxs_sample_race(self.ctx, ctypes.byref(b), ctypes.byref(r), ctypes.byref(o)),
                        "mxs_sample_race")
            self._keep = (b, o, r)
            return out
        self._check(self.lib.mxs_sample(self.ctx, ctypes.byref(b), ctypes.byref(o)), "mxs_sample")
        self._keep = (b, o)
        return out

    def lmhead(self, hidden, weight, *, stats: bool = False, logits=None):
        """Queues the bf16 lm_head GEMM (mxs_lmhead_bf16): hidden bf16[rows,
        hidden_dim], weight bf16[vocab, hidden_dim] on the device; returns
        (logits f32[rows, vocab], tile statistics u8[rows, ceil(vocab/256)
        * TILE_STAT_BYTES] or None).  With stats the epilogue also writes the statistics
        finish_tiles reads."""
        torch = self.torch
        rows, K = hidden.shape
        V = weight.shape[0]
        dev = hidden.device
        with torch.cuda.stream(self.stream):
            if logits is None:
                logits = torch.empty((rows, V), dtype=torch.float32, device=dev)
            st = (torch.empty((rows, -(-V // TILE_TOKENS) * TILE_STAT_BYTES), dtype=torch.uint8, device=dev)
                  if stats else None)
        self._check(self.lib.mxs_lmhead_bf16(self.ctx, hidden.data_ptr(), weight.data_ptr(), rows, K, V,
                                             logits.data_ptr(), logits.stride(0), _ptr(st)), "mxs_lmhead_bf16")
        return logits, st

    def finish_tiles(self, logits, tile_stats, temperature, *, top_k=None, top_p=None, min_p=None, uniform=None,
                     debug: bool = False, out: Optional[SampleResult] = None) -> SampleResult:
        """Queues the finish-only pick (mxs_finish_tiles) over the lm_head's
        logits and tile statistics: greedy and top-k rows, as `sample`
        picks them (no penalties, bias or mask)."""
        rows, V = logits.shape
        need = rows * -(-V // TILE_TOKENS) * TILE_STAT_BYTES
        if tile_stats.device != logits.device or tile_stats.numel() * tile_stats.element_size() < need:
            raise ValueError(f"tile_stats must hold {need} bytes on the logits' device")
        b, o, _, out = self._structs(logits, temperature, top_k=top_k, top_p=top_p, min_p=min_p, uniform=uniform,
                                     debug=debug, out=out)
        o.adjusted = None
        out.adjusted = None
        self._check(self.lib.mxs_finish_tiles(self.ctx, ctypes.byref(b), tile_stats.data_ptr(), ctypes.byref(o)),
                    "mxs_finish_tiles")
        self._keep = (b, o)
        return out

    def lmhead_launcher(self, hidden, weight, logits, tile_stats=None):
        """Pre-built lmhead for repeated calls into the same logits (and tile
        statistics): returns f() that re-issues mxs_lmhead_bf16."""
        rows, K = hidden.shape
        V = weight.shape[0]
        fn = self.lib.mxs_lmhead_bf16
        args = (self.ctx, hidden.data_ptr(), weight.data_ptr(), rows, K, V, logits.data_ptr(), logits.stride(0),
                _ptr(tile_stats))

        def launch():
            rc = fn(*args)
            if rc != 0:
                self._check(rc, "mxs_lmhead_bf16")

        return launch

    def finish_launcher(self, logits, tile_stats, temperature, **rule):
        """Pre-built finish_tiles for repeated calls over the same logits and
        tile statistics with the same rules and outputs: returns f() that
        re-issues mxs_finish_tiles (f.out holds the outputs)."""
        out = self.finish_tiles(logits, tile_stats, temperature, **rule)
        b, o = self._keep
        bp, op, sp = ctypes.byref(b), ctypes.byref(o), tile_stats.data_ptr()
        fn, ctx = self.lib.mxs_finish_tiles, self.ctx

        def launch():
            rc = fn(ctx, bp, sp, op)
            if rc != 0:
                self._check(rc, "mxs_finish_tiles")

        launch.out = out
        launch.keep = (b, o)
        return launch

    def step(self, logits, temperature, *, receipt_top=None, n: int = 28, race=None, **kw):
        """Queues one engine step (mxs_step): every row's pick as `sample`
        does, then the receipts over the suppressed logits (the bias
        entries of -inf) of the rows whose receipt_top entry (u32[rows] on
        the device; None: every row) is not RECEIPT_NONE, with n IDs per
        row (an entry of 0 still gets the picked token's log probability).
        Returns (SampleResult, ReceiptResult) of device tensors."""
        torch = self.torch
        b, o, r, out = self._structs(logits, temperature, race=race, **kw)
        rows, dev = logits.shape[0], logits.device
        with torch.cuda.stream(self.stream):   # the fills run before the step on its stream
            rec = ReceiptResult(
                ids=torch.full((rows, n), -1, dtype=torch.int32, device=dev),
                logprobs=torch.full((rows, n), float("nan"), dtype=torch.float64, device=dev),
                token_logprob=torch.full((rows,), float("nan"), dtype=torch.float64, device=dev),
                status=torch.zeros(rows, dtype=torch.int32, device=dev),
            )
        R = MxsReceipts()
        R.top = _ptr(receipt_top)
        R.n = n
        R.ids, R.logprobs = rec.ids.data_ptr(), rec.logprobs.data_ptr()
        R.token_logprob, R.status = rec.token_logprob.data_ptr(), rec.status.data_ptr()
        rp = ctypes.byref(r) if r is not None else None
        self._check(self.lib.mxs_step(self.ctx, ctypes.byref(b), rp, ctypes.byref(o), ctypes.byref(R)), "mxs_step")
        self._keep = (b, o, r, R)
        return out, rec

    def step_launcher(self, logits, *, receipt_top=None, n: int = 28, **kw):
        """Pre-built mxs_step for repeated steps with the same rules and
        outputs: returns f(logits) that only swaps the logits pointer (its
        .out and .receipts hold the device outputs)."""
        out, rec = self.step(logits, receipt_top=receipt_top, n=n, **kw)
        b, o, r, R = self._keep
        bp, op, Rp = ctypes.byref(b), ctypes.byref(o), ctypes.byref(R)
        rp = ctypes.byref(r) if r is not None else None
        ctx, fs = self.ctx, self.lib.mxs_step

        def launch(t):
            b.logits = t.data_ptr()
            rc = fs(ctx, bp, rp, op, Rp)
            if rc != 0:
                self._check(rc, "mxs_step")

        launch.out, launch.receipts = out, rec
        return launch

    def _structs(self, logits, temperature, *, top_k=None, top_p=None, min_p=None, repetition=None,
                 presence=None, frequency=None, uniform=None, history=None, bias=None, mask=None,
                 tokenizer_vocab=None, debug: bool = False, out: Optional[SampleResult] = None,
                 vocab: Optional[int] = None, race=None):
        torch = self.torch
        rows = logits.shape[0]
        V = vocab if vocab is not None else logits.shape[1]
        dev = logits.device
        if out is None:
            out = SampleResult(
                token=torch.empty(rows, dtype=torch.int32, device=dev),
                sampling_logprob=torch.empty(rows, dtype=torch.float64, device=dev),
                status=torch.empty(rows, dtype=torch.int32, device=dev),
                kept_count=torch.empty(rows, dtype=torch.int32, device=dev),
            )
            if debug:
                out.adjusted = torch.empty((rows, V), dtype=torch.float32, device=dev)
                out.kept_bits = torch.empty((rows, (V + 31) // 32), dtype=torch.int32, device=dev)
        b = MxsBatch()
        b.logits = logits.data_ptr()
        b.dtype = MXS_BF16 if logits.dtype == torch.bfloat16 else MXS_F32
        b.rows = rows
        b.vocab = V
        b.row_stride = logits.stride(0)
        b.temperature = _ptr(temperature)
        b.top_k = _ptr(top_k)
        b.top_p = _ptr(top_p)
        b.min_p = _ptr(min_p)
        b.repetition = _ptr(repetition)
        b.presence = _ptr(presence)
        b.frequency = _ptr(frequency)
        b.uniform = _ptr(uniform)
        if history is not None:
            b.history_offsets, b.history_ids = _ptr(history[0]), _ptr(history[1])
        if bias is not None:
            b.bias_offsets, b.bias_ids, b.bias_values = _ptr(bias[0]), _ptr(bias[1]), _ptr(bias[2])
        if mask is not None:
            b.mask_words = mask.data_ptr()
            b.mask_stride = mask.stride(0)
            b.tokenizer_vocab = V if tokenizer_vocab is None else tokenizer_vocab
        o = MxsOut()
        o.token = out.token.data_ptr()
        o.sampling_logprob = _ptr(out.sampling_logprob)
        o.status = out.status.data_ptr()
        o.kept_count = _ptr(out.kept_count)
        o.adjusted = _ptr(out.adjusted)
        o.kept_bits = _ptr(out.kept_bits)
        r = None
        if race is not None:
            r = MxsRace()
            r.seed, r.choice, r.position = _ptr(race[0]), _ptr(race[1]), _ptr(race[2])
        return b, o, r, out

    def launcher(self, logits, **kw):
        """Pre-built launch for repeated picks with the same parameters and
        outputs: returns f(logits) that only swaps the logits pointer."""
        out = self.sample(logits, **kw)
        keep = self._keep
        b, o = keep[:2]
        bp, op = ctypes.byref(b), ctypes.byref(o)
        ctx = self.ctx
        if len(keep) == 3:   # race-v2
            rp, fr = ctypes.byref(keep[2]), self.lib.mxs_sample_race
            fn, what = (lambda: fr(ctx, bp, rp, op)), "mxs_sample_race"
        else:
            fs = self.lib.mxs_sample
            fn, what = (lambda: fs(ctx, bp, op)), "mxs_sample"

        def launch(t):
            b.logits = t.data_ptr()
            rc = fn()
            if rc != 0:
                self._check(rc, what)

        launch.out = out
        return launch

    def verify_point_mass(self, logits, draft, temperature, uniform, *, stop_ids=(), **rule):
        """Point-mass speculative verification on device picks (A9): the
        walk of accept_and_roll_back (crates/core/engine/src/speculative.rs:
        318-347, as accept_verified exposes it for device picks) over S
        sequences of K + 1 scored positions.  `logits` [S * (K + 1), V] on
        the device, sequence-major; `draft` host ints [S, K]; `temperature`,
        `uniform` and the other rule tensors of `sample` are per row (row i
        of a sequence carries uniform_ahead(i), crates/app/cli/src/
        qwen_forward.rs:283-292).  Every row is picked in one mxs_sample
        call; on the host each sequence keeps picks in order until one
        leaves the draft, is a stop token, or is the bonus row.  Returns, per
        sequence, dict(emitted, accepted, stopped, status): status is 0, or
        the first non-zero row status among the settled rows (1: the host
        settles that row, as TokenPicker does, chat_turn.rs:348-358)."""
        import numpy as np

        draft = np.asarray(draft)
        S, K = draft.shape
        assert logits.shape[0] == S * (K + 1), "logits rows must be S * (K + 1)"
        out = self.sample(logits, temperature, uniform=uniform, **rule)
        self.sync()
        tok = out.token.cpu().numpy().reshape(S, K + 1)
        st = out.status.cpu().numpy().reshape(S, K + 1)
        stops = set(int(t) for t in stop_ids)
        res = []
        for s_ in range(S):
            emitted, accepted, stopped, status = [], 0, False, 0
            for i in range(K + 1):
                if status == 0 and st[s_, i] != 0:
                    status = int(st[s_, i])
                t = int(tok[s_, i])
                emitted.append(t)
                matches = i < K and int(draft[s_, i]) == t
                accepted += int(matches)
                if t in stops:
                    stopped = True
                    break
                if not matches:
                    break
            res.append(dict(emitted=emitted, accepted=accepted, stopped=stopped, status=status))
        return res

    def logsoftmax_topn(self, logits, n: int, *, vocab: Optional[int] = None):
        """Queues the T=1 log-softmax of every row with its n most likely IDs
        (token_logprob, crates/app/cli/src/chat_turn.rs:506-563).  Returns
        device tensors (ids i32[rows, n], logprobs f64[rows, n], maximum
        f64[rows], log_normalizer f64[rows], status i32[rows])."""
        torch = self.torch
        rows = logits.shape[0]
        V = vocab if vocab is not None else logits.shape[1]
        dev = logits.device
        ids = torch.empty((rows, max(n, 1)), dtype=torch.int32, device=dev)
        lps = torch.empty((rows, max(n, 1)), dtype=torch.float64, device=dev)
        mx = torch.empty(rows, dtype=torch.float64, device=dev)
        ln = torch.empty(rows, dtype=torch.float64, device=dev)
        st = torch.empty(rows, dtype=torch.int32, device=dev)
        dtype = MXS_BF16 if logits.dtype == torch.bfloat16 else MXS_F32
        rc = self.lib.mxs_logsoftmax_topn(self.ctx, logits.data_ptr(), dtype, rows, V, logits.stride(0), n,
                                          ids.data_ptr(), lps.data_ptr(), mx.data_ptr(), ln.data_ptr(),
                                          st.data_ptr())
        self._check(rc, "mxs_logsoftmax_topn")
        return ids[:, :n], lps[:, :n], mx, ln, st

    def spec_verify(self, target, draft, draft_tokens, temperature, accept_uniform, resample_uniform,
                    bonus_uniform):
        """Queues speculative verification (accept_or_resample position by
        position, crates/core/engine/src/speculative.rs:369-444; the bonus
        draw past an accepted draft).  target f32[rows, K+1, V], draft
        f32[rows, K, V], draft_tokens i32[rows, K], temperature f64[rows],
        accept/resample f64[rows, K], bonus f64[rows].  Returns device tensors
        (out_tokens i32[rows, K+1], count, accepted, status i32[rows])."""
        torch = self.torch
        rows, k1, V = target.shape
        K = k1 - 1
        dev = target.device
        out = torch.empty((rows, k1), dtype=torch.int32, device=dev)
        cnt = torch.empty(rows, dtype=torch.int32, device=dev)
        acc = torch.empty(rows, dtype=torch.int32, device=dev)
        st = torch.empty(rows, dtype=torch.int32, device=dev)
        rc = self.lib.mxs_spec_verify(self.ctx, target.data_ptr(), _ptr(draft) if K else None, rows, K, V,
                                      _ptr(draft_tokens) if K else None, temperature.data_ptr(),
                                      _ptr(accept_uniform) if K else None, _ptr(resample_uniform) if K else None,
                                      bonus_uniform.data_ptr(), out.data_ptr(), cnt.data_ptr(), acc.data_ptr(),
                                      st.data_ptr())
        self._check(rc, "mxs_spec_verify")
        return out, cnt, acc, st

    def export_candidates(self, rows: int, width: int):
        """Queues mxs_export_candidates for the first `rows` rows of the last
        pick on this context: returns device tensors (count i32[rows], ids
        i32[rows, width], logits f32[rows, width]); count -1 marks a row with
        no candidate list, otherwise the first count entries are the row's
        candidates (its top `width` when it had more) in token-ID order."""
        torch = self.torch
        dev = torch.device("cuda", self.device)
        count = torch.empty(rows, dtype=torch.int32, device=dev)
        ids = torch.empty((rows, width), dtype=torch.int32, device=dev)
        logits = torch.empty((rows, width), dtype=torch.float32, device=dev)
        self._check(self.lib.mxs_export_candidates(self.ctx, rows, width, count.data_ptr(), ids.data_ptr(),
                                                   logits.data_ptr()), "mxs_export_candidates")
        return count, ids, logits

    def spec_launcher(self, target, draft, draft_tokens, temperature, accept_uniform, resample_uniform,
                      bonus_uniform):
        """Pre-built spec_verify for repeated calls with the same per-row
        inputs and outputs: returns f(target, draft) that only swaps the two
        logits pointers (f.out holds spec_verify's output tensors)."""
        out = self.spec_verify(target, draft, draft_tokens, temperature, accept_uniform, resample_uniform,
                               bonus_uniform)
        rows, k1, V = target.shape
        K = k1 - 1
        fn, ctx = self.lib.mxs_spec_verify, self.ctx
        rest = (_ptr(draft_tokens) if K else None, temperature.data_ptr(),
                _ptr(accept_uniform) if K else None, _ptr(resample_uniform) if K else None,
                bonus_uniform.data_ptr(), *(t.data_ptr() for t in out))

        def launch(tgt, drf):
            rc = fn(ctx, tgt.data_ptr(), drf.data_ptr() if K else None, rows, K, V, *rest)
            if rc != 0:
                self._check(rc, "mxs_spec_verify")

        launch.out = out
        return launch

    def _device(self):
        return self.torch.device("cuda", self.device)

    def beam_select(self, logits, score, n: int, *, out: Optional[BeamResult] = None, **kw) -> BeamResult:
        """Queues one beam-search selection (mxs_beam_select): logits
        [groups * beams, >= vocab] f32 or bf16, score f64[groups, beams]; the
        n best (beam, token) candidates of each group, best first.  ended:
        bool[groups, beams] (with end_token); scale: f64[groups, beams], the
        length penalty that orders the candidates; mask: allowed-token words
        as `sample` takes them, with legal_norm for probabilities over the
        legal tokens."""
        return self.beam_launcher(logits, score, n, out=out, **kw).out

    def beam_launcher(self, logits, score, n: int, *, out: Optional[BeamResult] = None, **kw):
        """Pre-built beam_select for repeated selections with the same
        outputs (the first of them queued here): returns f(logits) that only
        swaps the logits pointer (f.out holds the outputs).  `out` may hold
        the input's own score and ended tensors when n == beams."""
        torch, dev = self.torch, self._device()
        b = beam_struct(torch, dev, logits, score, n, **kw)
        groups = score.shape[0]
        if out is None:
            with torch.cuda.stream(self.stream):
                e = lambda dt: torch.empty((groups, n), dtype=dt, device=dev)
                out = BeamResult(token=e(torch.int32), beam=e(torch.int32), score=e(torch.float64),
                                 ended=e(torch.bool), status=torch.empty(groups, dtype=torch.int32, device=dev))
        o = beam_out_struct(torch, dev, out, groups, n)
        fn, ctx, bp, op = self.lib.mxs_beam_select, self.ctx, ctypes.byref(b), ctypes.byref(o)

        def launch(t):
            b.logits = t.data_ptr()
            rc = fn(ctx, bp, op)
            if rc != 0:
                self._check(rc, "mxs_beam_select")

        launch(logits)
        launch.out, launch.keep = out, (b, o, score, kw)
        return launch

    def beam_reorder(self, states, parent, *, status=None, **kw):
        """Queues the move of the beams' states to their children
        (mxs_beam_reorder), in place: row g * beams + b of every tensor of
        `states` becomes what row g * beams + parent[g, b] was (-1: stays).
        parent: int32[groups, >= beams] (its first `beams` columns; default
        all).  lengths: int32[groups], the positions in use along each
        state's length_dim (one dimension, or one per state, None for states
        that move whole).  The states must not share memory with one another,
        parent, lengths or the status.  Returns the status, int32[groups]."""
        f = self.reorder_launcher(states, parent, status=status, **kw)
        f()
        return f.status

    def reorder_launcher(self, states, parent, *, status=None, **kw):
        """Pre-built beam_reorder for repeated moves of the same states:
        returns f() that re-issues mxs_beam_reorder with what parent and
        lengths then hold (f.status holds the status).  What the call would
        refuse is refused here."""
        torch, dev = self.torch, self._device()
        if status is None:
            with torch.cuda.stream(self.stream):
                status = torch.empty(parent.shape[0], dtype=torch.int32, device=dev)
        r = reorder_struct(torch, dev, states, parent, status, **kw)
        fn, ctx, rp = self.lib.mxs_beam_reorder, self.ctx, ctypes.byref(r)
        self._check(self.lib.mxs_beam_reorder_check(ctx, rp), "mxs_beam_reorder")

        def launch():
            rc = fn(ctx, rp)
            if rc != 0:
                self._check(rc, "mxs_beam_reorder")

        launch.status, launch.keep = status, (r, list(states), parent, kw)
        return launch

    def linear(self, x, weight, bias=None, *, activation=None, residual=None, out=None, out_dtype=None):
        """Queues out = act(x @ weight.T + bias) + residual (mxs_linear_bf16):
        x bf16[rows, in_features], weight bf16[out_features, in_features],
        row strides multiples of 8; bias f32 or bf16; activation none, relu,
        silu, gelu or gelu_tanh; residual of out's type (bf16 by default; it
        may be out itself).  Returns out; where none is given, a tensor whose
        row stride is out_features rounded up to a multiple of 8, as
        beam_select and another linear take it."""
        return self.linear_launcher(x, weight, bias, activation=activation, residual=residual, out=out,
                                    out_dtype=out_dtype).out

    def linear_launcher(self, x, weight, bias=None, *, activation=None, residual=None, out=None, out_dtype=None):
        """Pre-built linear for repeated products into the same output (the
        first of them queued here): returns f(x) that only swaps x's pointer
        (f.out holds the output)."""
        torch, dev = self.torch, self._device()
        if out is None:
            with torch.cuda.stream(self.stream):
                N = weight.shape[0]   # (rows start where beam_select and another product take them)
                out = torch.empty((x.shape[0], -(-N // 8) * 8), dtype=out_dtype or torch.bfloat16, device=dev)[:, :N]
        elif out_dtype is not None and out.dtype != out_dtype:
            raise ValueError(f"out must be {out_dtype}, not {out.dtype}")
        a = linear_struct(torch, dev, x, weight, bias, residual, out, activation)
        fn, ctx, ap = self.lib.mxs_linear_bf16, self.ctx, ctypes.byref(a)

        def launch(t):
            a.x = t.data_ptr()
            rc = fn(ctx, ap)
            if rc != 0:
                self._check(rc, "mxs_linear_bf16")

        launch(x)
        launch.out, launch.keep = out, (a, weight, bias, residual)
        return launch

    def prefix_attention(self, q, prefix_keys, prefix_values, keys=None, values=None, *, out=None, **kw):
        """Queues one layer's attention of sequences that share a prefix
        (mxs_prefix_attention): q bf16[groups * beams, (tokens,) heads, dim],
        the newest tokens of every sequence, over the first prefix_lengths[g]
        positions of its group's prefix_keys and prefix_values [groups,
        kv_heads, positions, dim] and, causally, the first lengths[r] of its
        own keys and values [groups * beams, kv_heads, positions, dim], the
        queries' own positions last (lengths int32 on the device; default
        all).  scale: dim ** -0.5 by default.  lse: f32, q's shape without
        dim, gets the logarithms of the sums.  prefix_weight f32[groups,
        kv_heads, positions] and weight f32[groups * beams, kv_heads,
        positions] get the weights of every position added, those of all rows'
        queries or, with counted (bool or uint8[groups * beams] on the device),
        of the rows whose entry is not 0.  Returns out, bf16 of q's shape."""
        f = self.prefix_attention_launcher(q, prefix_keys, prefix_values, keys, values, out=out, **kw)
        f()
        return f.out

    def prefix_attention_launcher(self, q, prefix_keys, prefix_values, keys=None, values=None, *, out=None, **kw):
        """Pre-built prefix_attention for repeated calls over the same
        tensors: returns f() that queues it with what they then hold (f.out
        holds the output).  Nothing is queued here."""
        torch, dev = self.torch, self._device()
        if out is None:
            with torch.cuda.stream(self.stream):
                out = torch.empty(q.shape, dtype=torch.bfloat16, device=dev)
        a = attention_struct(torch, dev, q, prefix_keys, prefix_values, keys, values, out, **kw)
        fn, ctx, ap, counted = self.lib.mxs_prefix_attention_counted, self.ctx, ctypes.byref(a), a.counted

        def launch():
            rc = fn(ctx, ap, counted)
            if rc != 0:
                self._check(rc, "mxs_prefix_attention")

        launch.out, launch.keep = out, (a, q, prefix_keys, prefix_values, keys, values, kw)
        return launch

    def cache_evict(self, keys, values, weight, budget: int, *, out: Optional[EvictResult] = None, **kw) -> EvictResult:
        """Queues the eviction of caches down to `budget` positions
        (mxs_cache_evict): keys and values, a tensor [segments, heads,
        capacity, dim] for each layer (values None: the layers have one array
        each), of which the first lengths[s] slots are in use (int32[segments];
        default all); weight f32[layers, segments, heads, capacity], their
        accumulated weights; index int32, the same shape, the slots' positions
        (default: in order).  The keep_first first positions, the keep_recent
        newest and the largest weights stay.  The caches change in place;
        returns the slots' new weights and positions and the new lengths, as
        the next eviction takes them."""
        f = self.cache_evict_launcher(keys, values, weight, budget, out=out, **kw)
        f()
        return f.out

    def cache_evict_launcher(self, keys, values, weight, budget: int, *, out: Optional[EvictResult] = None, **kw):
        """Pre-built cache_evict for repeated calls over the same tensors:
        returns f() that queues it with what they then hold (f.out holds the
        outputs).  Nothing is queued here."""
        torch, dev = self.torch, self._device()
        keys, values = list(keys), None if values is None else list(values)   # (the caller's may change)
        if out is None:
            with torch.cuda.stream(self.stream):
                e = lambda shape, dt: torch.empty(shape, dtype=dt, device=dev)
                out = EvictResult(weight=e(weight.shape, torch.float32), index=e(weight.shape, torch.int32),
                                  lengths=e(weight.shape[1:2], torch.int32))
        m = evict_struct(torch, dev, keys, values, weight, budget, out, **kw)
        fn, ctx, mp = self.lib.mxs_cache_evict, self.ctx, ctypes.byref(m)

        def launch():
            rc = fn(ctx, mp)
            if rc != 0:
                self._check(rc, "mxs_cache_evict")

        launch.out, launch.keep = out, (m, keys, values, weight, (out.weight, out.index, out.lengths), kw)
        return launch

    def mask_host(self, slot: int):
        """The pinned host words of staging slot `slot` as a numpy u32 array
        [max_rows, stride] (mxs_mask_host: returns once the slot's previous
        upload has read them, so the caller may overwrite them)."""
        import numpy as np

        ptr, stride = _vp(), ctypes.c_uint64()
        self._check(self.lib.mxs_mask_host(self.ctx, slot, ctypes.byref(ptr), ctypes.byref(stride)), "mxs_mask_host")
        self._mask_stride = stride.value
        n = self.max_rows * stride.value
        buf = (ctypes.c_uint32 * n).from_address(ptr.value)
        return np.frombuffer(buf, dtype=np.uint32).reshape(self.max_rows, stride.value)

    def mask_upload(self, slot: int, rows: int) -> DeviceWords:
        """Queues the upload of the slot's first `rows` rows (mxs_mask_upload);
        returns the device words for `sample(mask=...)`."""
        ptr = _vp()
        self._check(self.lib.mxs_mask_upload(self.ctx, slot, rows, ctypes.byref(ptr)), "mxs_mask_upload")
        return DeviceWords(ptr.value, self._mask_stride, rows)

    def sync(self):
        self._check(self.lib.mxs_sync(self.ctx), "mxs_sync")
