"""Softmax scales that are nothing, or infinite, in the 32 bits in which the kernels multiply by them are refused; nothing runs."""
import struct

import pytest

from dispec_b200.ops import library as L
from test_beams_checks_cpu import attention as shared
from test_tree_checks_cpu import F32, I32, I64, described


def tree(scale):
    t = [described(F32, (2, 32)), described(F32, (2, 2, 4, 8)), described(F32, (2, 2, 4, 8)), described(I32, (1, 8)), described(I32, (1,)),
         described(I32, (2,)), described(I32, (2,)), described(I64, (2, 1)), described(F32, (2, 32)), described(I32, (0,))]
    with pytest.raises(L.KernelError) as refused:
        L.check(L.core().dsp_tree_attention(b"".join(t), struct.pack("4qd", 4, 0, 148, 0, scale), None))
    return str(refused.value)


@pytest.mark.parametrize("attention", [lambda s: shared(scale=s), tree], ids=["shared", "tree"])
def test_scales_beyond_32_bits(attention):
    for scale in (1e-60, 1e-46, 2.9e38, 3e38, 1e300, float("inf"), float("nan"), 0.0, -1.0, -1e-60):
        assert "scale" in attention(scale)
    for scale in (1e-44, 1e-38, 1.0, 2.3e38):  # (what is wrong then is the scratch)
        assert "scratch" in attention(scale)
