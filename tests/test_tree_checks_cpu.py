"""What the C entry points of the operators on drafted trees refuse, asked with descriptions of tensors alone: nothing runs."""
import struct

import pytest

from dispec_b200.ops import library as L

DESC = struct.Struct("Q4i5q5q")
OPTIONS = struct.Struct("4qd")  # max_nodes, window, sms, tensor_cores, scale
F32, BF16, I32, I64 = 0, 1, 2, 3


def described(dtype, size, stride=None, contiguous=None, data=1 << 20, device=0):
    full = [1] * len(size)
    for i in range(len(size) - 2, -1, -1):
        full[i] = full[i + 1] * size[i + 1]
    stride = full if stride is None else list(stride)
    pad = lambda v: list(v) + [0] * (5 - len(v))
    dense = stride == full if contiguous is None else contiguous
    return DESC.pack(data, dtype, device, len(size), int(dense), *pad(size), *pad(stride))


NONE = DESC.pack(0, -1, -1, -1, 0, *[0] * 10)


def attention(T, scratch=0, max_nodes=4, table=(1, 8), page=4, **change):
    """Arguments of a call whose only flaw, unless ``change`` brings another, is a scratch without room."""
    t = dict(q=described(F32, (T, 32)), k=described(F32, (2, 2, page, 8)), v=described(F32, (2, 2, page, 8)),
             table=described(I32, table), ctx=described(I32, table[:1]), start=described(I32, (table[0] + 1,)), depth=described(I32, (T,)),
             visible=described(I64, (T, 1)), out=described(F32, (T, 32)), scratch=described(I32, (scratch,)))
    t.update(change)
    names = ("q", "k", "v", "table", "ctx", "start", "depth", "visible", "out", "scratch")
    with pytest.raises(L.KernelError) as refused:
        L.check(L.core().dsp_tree_attention(b"".join(t[n] for n in names), OPTIONS.pack(max_nodes, 0, 148, 0, 1.0), None))
    return str(refused.value)


@pytest.mark.parametrize("T", [1, 2, 9])
def test_columns_that_are_not_neighbours_are_refused(T):
    assert "scratch" in attention(T)
    strided = described(F32, (T, 32), (64, 2))
    assert "neighbours" in attention(T, q=strided)
    assert "neighbouring columns" in attention(T, out=strided)
    wide = described(F32, (T, 32), (64, 1), contiguous=T == 1)
    assert "scratch" in attention(T, q=wide, out=wide)


def test_more_key_tiles_than_are_counted_are_refused():
    assert "scratch" in attention(1 << 16, table=(1 << 10, 1 << 16), page=4)
    assert "too many" in attention(1 << 20, table=(1 << 16, 1 << 18), page=4)
    assert "too many" in attention(0x7fffffff)
