"""The sizes of the GPU tests of mxs_linear_bf16 reach every kernel that its
sizes choose from (mxs_linear_choice.h, built with the host compiler), so that
a moved threshold cannot leave one untested."""
import ctypes
import subprocess
from pathlib import Path

import pytest

import test_linear_gpu as short
import test_linear_long_gpu as long_

HERE = Path(__file__).resolve().parent
KERNELS = ["rows", "split", "split_long", "64", "64_long", "128", "128_256", "256"]
TILE = {"split": (64, 64), "split_long": (64, 64), "64": (64, 64), "64_long": (64, 64), "128": (128, 128),
        "128_256": (128, 256), "256": (256, 256)}           # features, rows
ACTS = range(5)


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    so = tmp_path_factory.mktemp("choice") / "choice.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", str(HERE / "linear_choice.cpp"), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))

    def f(R, K, N, act=0):
        parts, span = ctypes.c_uint32(), ctypes.c_uint32()
        return KERNELS[lib.choose(R, K, N, act, ctypes.byref(parts), ctypes.byref(span))], parts.value, span.value

    return f


def reached(choose, shapes, act):
    out = {}
    for s in shapes:
        out.setdefault(choose(*s, act)[0], []).append(s)
    return out


@pytest.mark.parametrize("act", ACTS)
def test_long_sums_reach_every_kernel(choose, act):
    got = reached(choose, long_.LONG, act)
    assert set(got) == set(KERNELS)
    for k, (bo, br) in TILE.items():      # each with unfilled last tiles of rows, features and k, and over 17 steps
        assert any(R % br and N % bo and K % 64 and K > 17 * 64 for R, K, N in got[k]), k


@pytest.mark.parametrize("act", ACTS)
def test_the_few_reach_every_tile(choose, act):
    """Those of the tests in place, not finite, repeated and captured."""
    assert {choose(*s, act)[0] for s in long_.FEW} == {"64_long", "split_long", "split", "128", "128_256", "256"}


@pytest.mark.parametrize("act", ACTS)
def test_short_sums_reach_the_others(choose, act):
    assert set(reached(choose, short.SHAPES + short.LARGER, act)) >= {"rows", "split", "split_long", "64", "128", "256"}


def test_split_sums_hold_their_scratch(choose):
    """At most 288 parts of 64 x 64, each of whole steps, none of them empty."""
    for R in (1, 5, 16, 17, 63, 64, 65, 130, 500, 1100, 4000):
        for K in (64, 1279, 1280, 1281, 2000, 4096, 8191, 14336, 60000, 1 << 22):
            for N in (1, 64, 65, 200, 1023, 4096, 9000):
                kernel, parts, span = choose(R, K, N)
                if not kernel.startswith("split"):
                    assert (parts, span) == (0, 0)
                    continue
                assert 2 <= parts <= 8 and -(-R // 64) * -(-N // 64) * parts <= 288
                assert span % 64 == 0 and (parts - 1) * span < K <= parts * span
