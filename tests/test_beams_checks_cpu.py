"""What the C entry points of the operators on beams refuse, asked with descriptions of tensors alone: nothing runs."""
import struct

import pytest

from dispec_b200.ops import library as L
from test_tree_checks_cpu import BF16, F32, I32, I64, NONE, described

OPTIONS = struct.Struct("4qd")  # window, sms, the tensor-core kernels, scale


def refused(call):
    with pytest.raises(L.KernelError) as error:
        L.check(call())
    return str(error.value)


def attention(R=3, scratch=0, table=None, scale=1.0, window=0, groups=1, page=4, dim=8, **change):
    """Arguments of a call whose only flaw, unless ``change`` brings another, is a scratch without room."""
    t = dict(q=described(F32, (R, 4 * dim)), k=described(F32, (2, 2, page, dim)), v=described(F32, (2, 2, page, dim)),
             table=described(I32, table or (R, 8)), ctx=described(I32, (R,)), start=described(I32, (groups + 1,)),
             prefix=described(I32, (groups,)), out=described(F32, (R, 4 * dim)), scratch=described(I32, (scratch,)))
    t.update(change)
    names = ("q", "k", "v", "table", "ctx", "start", "prefix", "out", "scratch")
    return refused(lambda: L.core().dsp_shared_attention(b"".join(t[n] for n in names), OPTIONS.pack(window, 148, 0, 0, scale), None))


@pytest.mark.parametrize("R", [1, 2, 9])
def test_columns_that_are_not_neighbours_are_refused(R):
    assert "scratch" in attention(R)
    strided = described(F32, (R, 32), (64, 2))
    assert "neighbours" in attention(R, q=strided)
    assert "neighbouring columns" in attention(R, out=strided)
    wide = described(F32, (R, 32), (64, 1), contiguous=R == 1)
    assert "scratch" in attention(R, q=wide, out=wide)


def test_attention_types_sizes_and_options_are_refused():
    assert "float32 and bfloat16" in attention(q=described(I32, (3, 32)))
    assert "alike" in attention(k=described(BF16, (2, 2, 4, 8)))
    assert "alike" in attention(v=described(F32, (2, 2, 8, 8)))
    assert "alike" in attention(v=described(F32, (2, 2, 4, 8), device=1))
    assert "columns" in attention(dim=12)
    assert "columns" in attention(dim=264)
    assert "columns" in attention(q=described(F32, (3, 24)))
    assert "scale" in attention(scale=0.0) and "scale" in attention(scale=float("nan")) and "scale" in attention(scale=float("inf"))
    assert "window" in attention(window=-1) and "window" in attention(window=1 << 31)
    assert "groups" in attention(groups=1025)
    assert "scratch" in attention(groups=1024)
    assert "int32" in attention(ctx=described(I32, (2,))) and "int32" in attention(start=described(I32, (3,)))
    assert "int32" in attention(prefix=described(I64, (1,)))
    assert "page_table" in attention(table=(2, 8)) and "page_table" in attention(table=(3, 8, 1))
    assert "like the queries" in attention(out=described(BF16, (3, 32)))
    assert "two rows in one place" in attention(out=described(F32, (3, 32), (0, 1), contiguous=0))
    assert "two rows in one place" in attention(out=described(F32, (3, 32), (16, 1), contiguous=0))
    assert "scratch" in attention(q=described(F32, (3, 32), (0, 1), contiguous=0))
    assert "16 bytes" in attention(q=described(F32, (3, 32), data=(1 << 20) + 4))
    assert "16 bytes" in attention(q=described(F32, (3, 32), (33, 1), contiguous=0))


def test_more_key_tiles_than_are_counted_are_refused():
    assert "scratch" in attention(1 << 16, table=(1 << 16, 1 << 10))
    assert "too many" in attention(1 << 20, table=(1 << 20, 1 << 18))
    assert "too many" in attention(0x7fffffff)


def test_a_device_that_is_not_the_current_one_is_refused():
    assert "current device" in attention(scratch=1 << 24)  # (here there is none)


def select(R=3, V=100, n=4, groups=2, scratch=0, **change):
    t = dict(logits=described(F32, (R, V)), scores=described(F32, (R,)), start=described(I32, (groups + 1,)),
             parent=described(I32, (groups, n)), token=described(I32, (groups, n)), score=described(F32, (groups, n)),
             scratch=described(F32, (scratch,)))
    t.update(change)
    names = ("logits", "scores", "start", "parent", "token", "score", "scratch")
    return refused(lambda: L.core().dsp_beam_select(b"".join(t[n] for n in names), None))


def test_select_refusals():
    assert "current device" in select()
    assert "CUDA" in select(logits=described(F32, (3, 100), device=-1))
    assert "float32 or bfloat16" in select(logits=described(I32, (3, 100)))
    assert "side by side" in select(logits=described(F32, (3, 100), (1, 3)))
    assert "side by side" in select(1, logits=described(F32, (1, 100), (200, 2)))
    assert "aligned" in select(logits=described(F32, (3, 100), data=(1 << 20) + 2))
    assert "count" in select(n=257) and "count" in select(n=0)
    assert "65535" in select(65536) and "65535" in select(V=0)
    assert "scores" in select(scores=described(BF16, (3,))) and "scores" in select(scores=NONE)
    assert "group_start" in select(start=described(I64, (3,))) and "group_start" in select(start=described(I32, (0,)))
    assert "results" in select(token=described(I32, (2, 5)))


def reorder(pools, n=2, src=None, dst=None):
    return refused(lambda: L.core().dsp_reorder_slots((src or described(I32, (n,))) + (dst or described(I32, (n,))) + b"".join(pools),
                                                      len(pools), None))


def test_reorder_refusals():
    good = described(BF16, (2, 8, 4, 16))
    assert "current device" in reorder([good])
    assert "1 to 64" in reorder([]) and "1 to 64" in reorder([good] * 65)
    assert "same memory" in reorder([good, good])
    assert "three to five" in reorder([described(BF16, (2, 8))]) and "three to five" in reorder([described(-1, (2, 8, 4))])
    assert "three to five" in reorder([described(BF16, (2, 8, 4), (64, 8, 2))]) and "three to five" in reorder([described(BF16, (2, 8, 4), device=1)])
    assert "slots" in reorder([good, described(BF16, (2, 9, 4, 16), data=1 << 22)])
    behind = described(BF16, (2, 8, 4, 16), data=(1 << 20) + 2 * 8 * 4 * 16 * 2)
    inside = described(BF16, (2, 8, 4, 16), data=(1 << 20) + 8 * 4 * 16 * 2)
    assert "current device" in reorder([good, behind]) and "current device" in reorder([behind, good])
    assert "same memory" in reorder([good, inside]) and "same memory" in reorder([inside, behind])
    assert "one length" in reorder([good], src=described(I32, (3,))) and "one length" in reorder([good], dst=described(I64, (2,)))
    assert "8192" in reorder([good], n=8193)
