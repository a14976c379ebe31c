"""Several continuations of one prompt: attention of sequences that share their beginning, the choice of the best
continuations of every group of beams, and caches and states that follow the choice.

Sequences of a step are rows of one flat batch, those of group g in rows ``group_start[g] .. group_start[g + 1] - 1``."""
from __future__ import annotations

import struct
from dataclasses import dataclass

import torch

from dispec_b200.ops import library as L
from dispec_b200.ops import tuning

_ATTENTION = struct.Struct("4qd")
_PIECE = 8192  # logits of a piece of a row (csrc/beam_select.cu)


# The tensor-core kernels are built for these head sizes and pages, and bfloat16; everything else takes the 32-bit kernel.
TENSOR_CORE_DIMS, TENSOR_CORE_PAGES = (32, 64, 128), (8, 16, 32, 64)
ON_FMA_UNITS = "32 bits for tensor cores"  # that kernel, where single tokens have one on the tensor cores


def on_tensor_cores(dim: int, page_size: int, dtype: torch.dtype) -> bool:
    return dtype is torch.bfloat16 and dim in TENSOR_CORE_DIMS and page_size in TENSOR_CORE_PAGES


def takes_heads(dim: int) -> bool:
    """Heads of which there is a kernel at all."""
    return dim % 8 == 0 and 8 <= dim <= 256


def _refuse(what: str, message: str):
    raise L.KernelError(f"{what}: {message}")


_describe = None


def _load_describe():
    global _describe
    _describe = L.describe()
    return _describe


_tensor_core_calls: dict = {}  # head size -> addresses of the tensor-core kernels' entry points


def _tensor_core_call(dim: int) -> tuple:
    calls = _tensor_core_calls.get(dim)
    if calls is None:
        lib = L.shared_attention_library(dim)
        # (heads of 32 have no kernel for many rows)
        calls = tuple(L.address_of(lib, f"dsp_shared_attention_{rows}_d{dim}") if rows == "few" or dim >= 64 else 0
                      for rows in ("few", "many"))
        _tensor_core_calls[dim] = calls
    return calls


def shared_prefix_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, page_table: torch.Tensor,
                            ctx_len: torch.Tensor, group_start: torch.Tensor, prefix_len: torch.Tensor, *, scale: float,
                            window: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Single tokens of sequences in groups: the keys and values of a group's shared beginning are read once for all of them.

    ``q`` [R, H * D], bfloat16 or float32 (rows may be those of a wider matrix), already turned by their positions: the
    newest token of each sequence, whose key and value are stored.  ``k_pool``, ``v_pool`` [pages, KVH, page_size, D] of the
    same type, H a multiple of KVH; ``page_table`` int32 [R, pages of a sequence]; ``ctx_len`` int32 [R]: stored tokens, the
    newest among them.  ``group_start`` int32 [groups + 1]: the sequences of each group; ``prefix_len`` int32 [groups]: so many
    first tokens are the same for all of a group's sequences, and are read through the pages of its first one (any number;
    it need not fill pages).  Head h of row r of group g, n = ctx_len[r]:

        sum_j w_j v_j / sum_j w_j,   w_j = exp(scale * q . k_j),   max(0, n - window) <= j < n  (window 0: all j < n)

    zero where there is none.  Pages that no row of the group sees may be gone from the tables.

    Scores, maxima, sums and the joining of parts are in 32 bits, and the result [R, H * D] is rounded once.  In bfloat16 with heads
    of 32, 64 or 128 and pages of 8 to 64 tokens (tensor cores) the weights are rounded to bfloat16 as well, for their product
    with the values, though not in their sum; in heads of 128, where many rows share keys, a quarter of them come from a
    polynomial that is 1.1e-4 off.  The result is then 2.1e-3 to 2.3e-3 off, 1.7e-3 of it by its own rounding.  Everything else is
    computed on FMA units.

    Rows of no group are left as they are; a group whose sequences are not all among the R, or that does not begin behind the
    groups before it, is recorded as a device error and left out.  At most 1,024 groups.  ``scale`` is positive and finite in 32
    bits.  Nothing is read back."""
    what = "shared_prefix_attention"
    if not q.is_cuda:
        _refuse(what, "CUDA tensors only (there is no CPU path)")
    if q.dim() != 2 or k_pool.dim() != 4 or page_table.dim() != 2:
        _refuse(what, "q [R, H * D], two pools [pages, heads, page_size, D] and a page_table [R, pages of a sequence] expected")
    if out is None:
        out = q.new_empty(q.shape)
    dev = q.get_device()
    (rows, columns), (_, kv_heads, page, dim) = q.shape, k_pool.shape
    sms = tuning._sm_count.get(dev) or tuning.sm_count(dev)
    tensor_cores = on_tensor_cores(dim, page, q.dtype)
    # scratch of this call alone (calls on several streams do not meet in it): two partial results for each row, and for each
    # kernel two of a tile of rows for each CTA and what the merge has to know of every item (csrc/shared_schedule.cuh)
    share, groups = columns // max(1, kv_heads * dim), prefix_len.numel()
    tile, ctas = (64, 2 * sms) if tensor_cores else (32, sms * (1 if dim > 128 else 2))
    items = (rows * share // tile + groups + 1 + rows * -(-share // tile)) * kv_heads + 1
    rest = ctas * tile * (dim + 2) + items
    # (the rule by which the kernel for many rows is taken as well: csrc/shared_attn.cu)
    many = tensor_cores and dim >= 64 and rows * share > 64 * groups and (
        -(-rows * share // 64) * kv_heads * (page_table.shape[1] * page // 64 + 1) > 12 * sms)
    if many:
        rest += sms * 256 * (dim + 2) + (rows * share // 256 + groups + 1) * kv_heads + 1
    scratch = prefix_len.new_empty(2 * (rows * kv_heads * share * (dim + 2) + rest))
    tensors = (_describe or _load_describe())(q, k_pool, v_pool, page_table, ctx_len, group_start, prefix_len, out, scratch)
    few_call, many_call = _tensor_core_call(dim) if tensor_cores else (0, 0)
    L.check(L.core().dsp_shared_attention(tensors, _ATTENTION.pack(window, sms, few_call, many_call, scale), L.stream_handle()),
            launches=3 if many else 2)
    return out


@dataclass
class Selected:
    parent: torch.Tensor  # int32 [groups, count]: row of the beam that is continued, -1 where there are no more
    token: torch.Tensor   # int32 [groups, count]: by this token, -1
    score: torch.Tensor   # float32 [groups, count]: the continuation's score, descending, -inf


def beam_select(logits: torch.Tensor, scores: torch.Tensor, group_start: torch.Tensor, *, count: int) -> Selected:
    """The ``count`` best continuations of every group of beams, over all its beams and the vocabulary.

    ``logits`` [R, V], float32 or bfloat16: behind every beam; ``scores`` float32 [R]: its sum of log-probabilities so far;
    ``group_start`` int32 [groups + 1]: the beams of each group.  A continuation of row r by token v scores
    ``scores[r] + log_softmax(logits[r])[v]``; the best come first, ties to the lowest row, then the lowest token.  Scores are
    compared in 64 bits; of a row, the logarithm of its sum of exponentials is rounded to 32.

    NaN counts as -inf, and what is -inf is never chosen; where the largest logits of a row are infinite they share its mass;
    a beam whose score is not finite has no continuations.  A group whose rows are not all among the R is recorded as a device
    error and has none.  ``count`` is at most 256."""
    what = "beam_select"
    if not logits.is_cuda:
        _refuse(what, "CUDA tensors only (there is no CPU path)")
    if logits.dim() != 2 or group_start.dim() != 1 or not 1 <= count <= 256:
        _refuse(what, f"logits [R, V], group_start [groups + 1] and a count {count} of 1 to 256 expected")
    (rows, vocab), groups = logits.shape, max(0, group_start.shape[0] - 1)
    parent, token = group_start.new_empty((groups, count)), group_start.new_empty((groups, count))
    score = scores.new_empty((groups, count))
    # scratch of this call alone: what the CTAs leave of their parts of rows, and of every piece (csrc/beam_select.cu)
    dev = logits.get_device()
    pieces = -(-vocab // _PIECE)
    parts = rows + min(rows * pieces, 3 * (tuning._sm_count.get(dev) or tuning.sm_count(dev)))
    scratch = scores.new_empty(parts * (2 * count + 1) + 2 * rows * (8 * pieces + 1))
    tensors = (_describe or _load_describe())(logits, scores, group_start, parent, token, score, scratch)
    L.check(L.core().dsp_beam_select(tensors, L.stream_handle()), launches=2)
    return Selected(parent, token, score)


def reorder_slots(pools: list, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Slots of caches or states follow a choice, in place: ``pool[:, dst[i]] = pool[:, src[i]]`` for all i and every pool, as
    though all were read before any is written (a slot may be read by several and written by another).

    ``pools``: up to 64 contiguous tensors [layers, slots, ...] of three to five dimensions, float32, bfloat16, int32 or int64,
    with the same number of slots and no memory in common, with each other or with ``src`` and ``dst``;
    ``src``, ``dst`` int32 [n], n up to 8,192, ``dst`` ascending: what does not ascend, or names a slot that is not there, is
    left from there on and recorded as a device error."""
    what = "reorder_slots"
    if not pools or not pools[0].is_cuda:
        _refuse(what, "CUDA tensors only (there is no CPU path)" if pools else "no pools")
    tensors = (_describe or _load_describe())(src, dst, *pools)
    L.check(L.core().dsp_reorder_slots(tensors, len(pools), L.stream_handle()))
