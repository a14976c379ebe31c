"""What C code is told of tensors."""
import struct

import pytest
import torch

from dispec_b200.ops import library as L

DESC = struct.Struct("Q4i5q5q")


def test_descriptors():
    a = torch.zeros(3, 4, 5, dtype=torch.bfloat16).transpose(0, 1)
    b = torch.zeros((), dtype=torch.int64)
    got = L.describe()(a, None, b, torch.zeros(2, dtype=torch.float64))
    assert len(got) == 4 * DESC.size
    rows = [DESC.unpack_from(got, i * DESC.size) for i in range(4)]
    assert rows[0][:5] == (a.data_ptr(), 1, -1, 3, 0) and rows[0][5:8] == (4, 3, 5) and rows[0][10:13] == (5, 20, 1)
    assert rows[1][0] == 0 and rows[1][3] == -1
    assert rows[2][1:5] == (3, -1, 0, 1)
    assert rows[3][1] == -1
    assert [DESC.unpack(L.describe()(torch.zeros(1, dtype=t)))[1] for t in (torch.float32, torch.bfloat16, torch.int32, torch.int64)] == [0, 1, 2, 3]


def test_what_is_no_tensor_is_refused():
    with pytest.raises(TypeError):
        L.describe()(torch.zeros(1), 3)
    assert L.describe()() == b""
