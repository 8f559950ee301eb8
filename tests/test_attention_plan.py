"""How mxs_prefix_attention splits its work (mxs_attention_plan.h), without a
GPU: every split fits the scratch and a launch, covers all positions, and every
kind of kernel is reached by sizes that the GPU tests run."""
import ctypes
import random
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
SCRATCH = 64 << 20


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    so = tmp_path_factory.mktemp("plan") / "plan.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", str(HERE / "attention_plan.cpp"),
                    "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.bytes.restype = ctypes.c_uint64
    lib.bytes.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint32]

    def f(*sizes):
        out = (ctypes.c_uint32 * 10)()
        lib.plan((ctypes.c_uint32 * 8)(*sizes), out)
        return dict(zip(("dp", "rb", "wq", "small", "sp", "ss", "slots", "ng", "wb", "nt"), out))

    f.bytes = lib.bytes
    return f


def verify(plan, G, W, T, H, KV, D, P, N):
    p = plan(G, W, T, H, KV, D, P, N)
    assert D <= p["dp"] and p["dp"] in (64, 128, 256)
    assert (p["rb"], p["wq"]) in ({(1, 1), (1, 2), (1, 4), (1, 8)} if p["dp"] == 256 else {(1, 1), (2, 1), (2, 2), (2, 4)})
    assert 1 <= p["ng"] <= G and 1 <= p["wb"] <= W and 1 <= p["nt"] <= T
    assert p["wb"] == W or p["ng"] == 1
    assert p["nt"] == T or p["wb"] == 1
    queries = p["ng"] * p["wb"] * p["nt"] * H
    assert plan.bytes(queries, p["slots"], p["dp"]) <= SCRATCH
    assert p["slots"] == p["sp"] + p["ss"]
    assert (p["sp"] >= 1) == (P > 0) and (p["ss"] >= 1) == (N > 0)
    assert p["sp"] <= -(-P // 64) and p["ss"] <= -(-N // 64)
    per = H // KV
    if p["small"]:
        assert p["nt"] * per <= 16
    rows = 16 * p["rb"] * p["wq"]
    ms = p["nt"] * per
    jobs = p["ng"] * KV * -(-p["wb"] * ms // rows) * p["sp"]
    jobs += p["ng"] * p["wb"] * KV * (1 if p["small"] else -(-ms // rows)) * p["ss"]
    assert jobs < 1 << 23   # (512 threads at most: a launch holds below 2^32)
    return p


def test_random_sizes(plan):
    rng = random.Random(1)
    log = lambda hi: int(2 ** rng.uniform(0, hi))
    for _ in range(20000):
        KV = log(6)
        verify(plan, log(9), log(9), log(rng.choice([0, 3, 9])), KV * log(rng.choice([0, 3, 6])), KV, 8 * rng.randint(1, 32),
               rng.choice([0, log(10), log(20), log(30)]), rng.choice([0, log(8), log(20)]))


def test_extremes(plan):
    for sizes in [(1, 1, 1, 1, 1, 8, 1, 0), (1, 1, 1, 1, 1, 8, 0, 0), (1, 1, 1, 4096, 1, 256, 1 << 30, 1 << 30),
                  (1, 1, 1 << 19, 4096, 4096, 64, 1 << 30, 1 << 30), (1 << 30, 1, 1, 1, 1, 8, 1, 1), (1, 1 << 30, 1, 1, 1, 256, 1, 1)]:
        verify(plan, *sizes)


def test_every_kind_is_tested(plan):
    from test_attention_gpu import RAGGED, SHAPES

    seen = {(p["dp"], p["rb"], p["wq"], p["small"]) for p in
            (verify(plan, *[v or 0 for v in shape]) for shape in SHAPES + [s for s, _, _ in RAGGED])}
    wants = {(dp, rb, wq) for dp in (64, 128) for rb, wq in ((1, 1), (2, 1), (2, 2), (2, 4))} | {(256, 1, wq) for wq in (1, 2, 4, 8)}
    missing = wants - {k[:3] for k in seen}
    assert not missing, missing
    assert {k[3] for k in seen} == {0, 1}
