"""Which rows' weights count (mxs_prefix_attention_counted): what its checks and
the Python binding's refuse, without a GPU."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from test_attention_checks import attention, call

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    so = tmp_path_factory.mktemp("counted") / "counted.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", str(HERE / "attention_counted.cpp"),
                    "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.check.restype = ctypes.c_char_p
    return lambda a, counted: lib.check(ctypes.byref(attention(**a)), ctypes.c_void_p(counted))


@pytest.mark.parametrize("a,counted,word", [
    (dict(out=0x110000), 0x110000, "overlaps an input"), (dict(lse=0x600000), 0x60017f, "overlaps an input"),
    (dict(weight=0x600000), 0x5ffffb, "overlaps an input"), (dict(prefix_weight=0x600000), 0x600c7f, "overlaps an input"),
    (dict(q=None), 0x700000, "required")])
def test_refused(check, a, counted, word):
    msg = check(a, counted)
    assert msg and word in msg.decode(), msg


def test_accepted(check):
    for a, counted in (({}, None), ({}, 0x700001), (dict(lse=0x600000), 0x600180), (dict(weight=0x600000), 0x5ffffa),
                       (dict(lengths=0x700000), 0x700000)):   # (6 rows; inputs may share memory)
        assert check(a, counted) is None


def test_binding():
    ok = torch.ones(6, dtype=torch.bool)
    assert call(counted=ok).counted == ok.data_ptr() and call().counted is None
    assert call(counted=ok.to(torch.uint8)).reserved == 0
    for bad in (torch.ones(2, dtype=torch.bool), torch.ones(6, 1, dtype=torch.bool), torch.ones(6), torch.ones(6, dtype=torch.int32),
                torch.ones(12, dtype=torch.bool)[::2], torch.ones(6, dtype=torch.bool, device="meta")):
        with pytest.raises(ValueError, match="counted"):
            call(counted=bad)
