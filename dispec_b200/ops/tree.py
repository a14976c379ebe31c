"""Drafted trees over the paged cache: attention of their nodes, their verification against the target's
distribution, and the accepted branch put into line in the cache.

A step checks one tree of drafted tokens per request.  Node 0, the root, is the token that the step before
drew; every other node is a draft of the token behind its parent, whose number is smaller.  The nodes of
all trees are rows of one flat batch, tree s in rows ``node_start[s] .. node_start[s + 1] - 1``, and node i
keeps its key and value at place ``ctx_len[s] + i`` of its request's cache until ``keep_path`` moves those
of the accepted branch."""
from __future__ import annotations

import struct
from dataclasses import dataclass

import torch

from dispec_b200.ops import library as L
from dispec_b200.ops import tuning

_ATTENTION = struct.Struct("4qd")
_VERIFY = struct.Struct("q")


def _refuse(what: str, message: str):
    raise L.KernelError(f"{what}: {message}")


# A call is made once a layer, and its checks are part of what it costs: tensors are described to the C entry points as they
# are (types, devices, sizes, strides), which refuse what they cannot take.
_tensor_core_calls: dict = {}  # (device, head size) -> address of the tensor-core kernel's entry point


def _tensor_core_call(device: int, dim: int) -> int:
    call = _tensor_core_calls.get((device, dim))
    if call is None:
        call = L.address_of(L.tree_attention_library(dim), f"dsp_tree_attention_tcgen05_d{dim}")
        _tensor_core_calls[(device, dim)] = call
    return call


def tree_attention(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, page_table: torch.Tensor,
                   ctx_len: torch.Tensor, node_start: torch.Tensor, visible: torch.Tensor,
                   depth: torch.Tensor | None = None, *, max_nodes: int, scale: float, window: int = 0,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Every node's queries over its request's stored keys and the nodes of its own tree that it sees.

    ``q`` [T, H * D], bfloat16 or float32 (rows may be those of a wider matrix), already turned by their
    positions; ``k_pool``, ``v_pool`` [pages, KVH, page_size, D] of the same type, H a multiple of KVH;
    ``page_table`` int32 [S, pages of a request].  ``ctx_len`` int32 [S]: stored tokens in front of each
    tree; ``node_start`` int32 [S + 1].  ``visible`` int64 [T, words]: bit j % 64 of word j // 64 says that
    the row sees node j of its tree (``ancestors`` gives node and ancestors).  Row of node i, head h:

        sum_j w_j v_j / sum_j w_j,   w_j = exp(scale * q . k_j)

    over the keys it sees, zero where there is none.  ``window`` W > 0: a node at depth d (``depth`` int32
    [T], the root at 0) is at position ctx_len + d and sees positions above ctx_len + d - W only; pages that
    no node sees may be gone from the table.  ``max_nodes``: no tree has more nodes, as far as the host knows.
    32-bit sums and softmax; the result [T, H * D] is rounded once.  Rows of no tree are left as they are; a tree whose rows are not
    all among the T is recorded as a device error and left out.  Nothing is read back."""
    what = "tree_attention"
    if not q.is_cuda:
        _refuse(what, "CUDA tensors only (there is no CPU path)")
    if out is None:
        out = q.new_empty(q.shape)
    dev, dim = q.get_device(), k_pool.shape[-1] if k_pool.dim() else 0
    sms = tuning._sm_count.get(dev) or tuning.sm_count(dev)
    # the tensor-core kernel is built for these head sizes
    tensor_cores = _tensor_core_call(dev, dim) if q.dtype is torch.bfloat16 and dim in (64, 128) else 0
    # scratch of this call alone (calls on several streams do not meet in it): two partial results of 128 rows for
    # each CTA, or of 32 rows where there are two CTAs an SM, and what the merge has to know of it
    scratch = node_start.new_empty(sms * (2 * (128 if tensor_cores else 64) * (dim + 2) + 16))
    tensors = (_describe or _load_describe())(q, k_pool, v_pool, page_table, ctx_len, node_start, depth, visible, out, scratch)
    L.check(L.core().dsp_tree_attention(tensors, _ATTENTION.pack(max_nodes, window, sms, tensor_cores, scale),
                                        L.stream_handle()), launches=2)
    return out


_describe = None


def _load_describe():
    global _describe
    _describe = L.describe()
    return _describe


def ancestors(parents: list) -> tuple[list, list]:
    """(visible, depth) of a tree given by its nodes' parents (-1: the root): the words of every node's bits for
    ``tree_attention``'s ``visible``, node and ancestors set, and its depth.  On the host."""
    words = max(1, -(-len(parents) // 64))
    bits, depth = [], []
    for i, p in enumerate(parents):
        if not -1 <= p < i or (p < 0) != (i == 0):
            raise ValueError(f"node {i} has parent {p}: the root comes first, every other node behind its parent")
        bits.append((bits[p] if i else 0) | 1 << i)
        depth.append(depth[p] + 1 if i else 0)
    low = (1 << 64) - 1
    signed = lambda w: w - (1 << 64) if w >> 63 else w
    return [[signed(b >> (64 * k) & low) for k in range(words)] for b in bits], depth


@dataclass
class Verified:
    count: torch.Tensor  # int32 [S]: accepted nodes, the root among them
    path: torch.Tensor   # int32 [S, max_nodes]: those nodes, root first, -1 behind them
    token: torch.Tensor  # int32 [S]: the token drawn behind the last of them


def verify_tree(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, node_start: torch.Tensor,
                temperature: torch.Tensor, uniforms: torch.Tensor, draws: torch.Tensor,
                draft_probs: torch.Tensor | None = None, *, max_nodes: int) -> Verified:
    """Accepts drafts so that the accepted tokens and the one drawn behind them are distributed as tokens that the
    target samples one by one.

    ``logits`` [T, V], float32 or bfloat16: the target's, behind each node.  ``tokens``, ``parents`` int32 [T] (parents
    are numbers inside the tree, the root's -1; siblings are tried in the order of their numbers).  ``temperature``
    float32 [S], 0 or less: the largest logit, ties to the lowest index.  ``uniforms`` float32 [T] in [0, 1): a node's
    test; ``draws`` float32 [S] in [0, 1): the token drawn at the end, by the inverse of the cumulative distribution in
    vocabulary order.  ``draft_probs`` float32 [T, V]: row i is the distribution that the children of node i were drawn
    from, each on its own; None: drafts are certain (looked up, or a draft model's likeliest).

    Distributions are held in whole numbers (the likeliest token's mass is 2^40), so that no decision depends on the
    order of a sum.  A token id outside the vocabulary is recorded as a device error and never accepted.  A tree without nodes
    gives count 0 and token -1, and so does one whose rows are not all among the T, which is recorded as a device error;
    nodes beyond ``max_nodes`` are not tried."""
    what = "verify_tree"
    if not logits.is_cuda:
        _refuse(what, "CUDA tensors only (there is no CPU path)")
    S = temperature.shape[0]
    count, path, token = tokens.new_empty(S), tokens.new_empty((S, max_nodes if max_nodes > 0 else 0)), tokens.new_empty(S)
    tensors = (_describe or _load_describe())(logits, draft_probs, tokens, parents, node_start, temperature, uniforms, draws,
                                              path, count, token)
    L.check(L.core().dsp_tree_verify(tensors, _VERIFY.pack(max_nodes), L.stream_handle()))
    return Verified(count, path, token)


def keep_path(pools: list, page_table: torch.Tensor, ctx_len: torch.Tensor, path: torch.Tensor, count: torch.Tensor) -> None:
    """Moves what the cache keeps of the accepted nodes into line, in place: of tree s, place ``ctx_len[s] + j`` gets the
    rows of node ``path[s, j]`` for j < ``count[s]``.

    ``pools``: up to eight contiguous tensors [layers, pages, heads, page_size, width] of rows of whole 16-byte pieces,
    all with the pages of ``page_table`` [S, pages of a request]; ``path`` int32 [S, n] ascends within a tree, as
    ``verify_tree`` gives it (one that does not is left from there on and recorded as a device error)."""
    what = "keep_path"
    if not pools or not pools[0].is_cuda:
        _refuse(what, "CUDA tensors only (there is no CPU path)" if pools else "no pools")
    tensors = (_describe or _load_describe())(page_table, ctx_len, path, count, *pools)
    L.check(L.core().dsp_tree_keep(tensors, len(pools), L.stream_handle()))
