"""Calls that the binding passes on to the entry point's own checks, without a GPU."""
import ctypes

import torch

from test_attention_checks import call, checks  # noqa: F401

BF = torch.bfloat16


def test_heads_without_elements(checks):  # noqa: F811
    z = lambda *s: torch.zeros(*s, 0, dtype=BF)
    a = call(q=z(6, 2, 8), pk=z(2, 4, 100), pv=z(2, 4, 100), k=z(6, 4, 10), v=z(6, 4, 10))
    a.q = a.out = 0x1000   # (an empty tensor has no address)
    assert b"dim" in checks.check_attention(ctypes.byref(a))
