"""Drafted trees over the paged cache: attention of their nodes, their verification against the target's
distribution, and the accepted branch put into line in the cache.

A step checks one tree of drafted tokens per request.  Node 0, the root, is the token that the step before
drew; every other node is a draft of the token behind its parent, whose number is smaller.  The nodes of
all trees are rows of one flat batch, tree s in rows ``node_start[s] .. node_start[s + 1] - 1``, and node i
keeps its key and value at place ``ctx_len[s] + i`` of its request's cache until ``keep_path`` moves those
of the accepted branch."""
from __future__ import annotations

import ctypes
import struct
from dataclasses import dataclass

import torch

from dispec_b200.ops import library as L
from dispec_b200.ops import tuning
from dispec_b200.ops.attention import _TCGEN05_ERRORS, _device_error_address

MAX_HEAD_DIM = 256
TENSOR_CORE_ROWS, FMA_ROWS = 128, 32  # rows of a tile of the two attention kernels
MAX_POOLS = 8
MAX_VOCAB = 3 << 17  # of a verified tree: a row is shared by at most 16 CTAs
MAX_TREE = 1024  # nodes of a tree that is verified
_ATTENTION = struct.Struct("10q13qd")
_VERIFY = struct.Struct("11q6q")
_KEEP = struct.Struct("4q6q40q")


def _refuse(what: str, message: str):
    raise L.KernelError(f"{what}: {message}")


# A call is made once a layer: the checks below cost a few microseconds of the host together, which is what a call on a small
# batch takes on the device.
def _is(t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: int) -> bool:
    return t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous()


def _ints(what: str, name: str, t: torch.Tensor, shape: tuple, device: int) -> None:
    if not _is(t, torch.int32, shape, device):
        _refuse(what, f"{name} must be contiguous int32 {list(shape)} on cuda:{device}, not {t.dtype} {list(t.shape)} on {t.device}")


def _table(what: str, table: torch.Tensor, seqs: int, device: int) -> None:
    if table.dtype is not torch.int32 or table.get_device() != device or table.dim() != 2 or table.shape[0] < seqs \
            or table.stride(1) != 1:
        _refuse(what, f"page_table must be int32 [{seqs}, pages] on cuda:{device} with neighbouring pages side by side")


_tensor_core_calls: dict = {}  # (device, head size) -> entry point, address of the merge, address of the error word


def _tensor_core_call(device: int, dim: int):
    call = _tensor_core_calls.get((device, dim))
    if call is None:
        call = (getattr(L.tree_attention_library(dim), f"dsp_tree_attention_tcgen05_d{dim}"),
                ctypes.c_void_p(L.address_of(L.core(), "dsp_tree_combine")), ctypes.c_void_p(_device_error_address(device)))
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
    32-bit sums and softmax; the result [T, H * D] is rounded once.  Nothing is read back."""
    what = "tree_attention"
    if not q.is_cuda:
        _refuse(what, "CUDA tensors only (there is no CPU path)")
    if q.dim() != 2 or k_pool.dim() != 4 or k_pool.shape != v_pool.shape:
        _refuse(what, f"q [T, H * D] and two pools [pages, heads, page_size, D] expected, got {list(q.shape)}, "
                      f"{list(k_pool.shape)} and {list(v_pool.shape)}")
    T, S, dev = q.shape[0], ctx_len.shape[0], q.get_device()
    num_pages, kv_heads, page_size, dim = k_pool.shape
    columns, dtype = q.shape[1], q.dtype
    code = L.dtype_code(dtype)
    if k_pool.dtype is not dtype or v_pool.dtype is not dtype or k_pool.get_device() != dev or v_pool.get_device() != dev:
        _refuse(what, f"q ({dtype}) and the pools ({k_pool.dtype}, {v_pool.dtype}) must be of one type on one device")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()) or (T > 1 and q.stride(1) != 1):
        _refuse(what, "the pools must be contiguous and the columns of q neighbours")
    heads = columns // dim if dim else 0
    if dim % 8 or not 8 <= dim <= MAX_HEAD_DIM or heads * dim != columns or heads == 0 or heads % kv_heads:
        _refuse(what, f"{columns} query columns on {kv_heads} heads of {dim} (a multiple of 8 up to {MAX_HEAD_DIM})")
    words = visible.shape[1] if visible.dim() == 2 else 0
    if not _is(visible, torch.int64, (T, words), dev) or 64 * words < max_nodes:
        _refuse(what, f"visible must be contiguous int64 [{T}, words] with a bit for each of {max_nodes} nodes")
    if not scale > 0.0 or window < 0 or max_nodes < 1:
        _refuse(what, f"scale {scale} must be positive, window {window} not negative, max_nodes {max_nodes} at least 1")
    _ints(what, "ctx_len", ctx_len, (S,), dev)
    _ints(what, "node_start", node_start, (S + 1,), dev)
    _table(what, page_table, S, dev)
    if depth is not None:
        _ints(what, "depth", depth, (T,), dev)
    elif window:
        _refuse(what, "a window needs the depths of the nodes")
    if out is None:
        out = q.new_empty((T, columns))
    elif out.shape != (T, columns) or out.dtype is not dtype or out.get_device() != dev or (T > 1 and out.stride(1) != 1):
        _refuse(what, f"out must be {dtype} [{T}, {columns}] with neighbouring columns")
    if T == 0 or S == 0:
        return out
    ctas = tuning._sm_count.get(dev) or tuning.sm_count(dev)
    # the tensor-core kernel is built for these head and page sizes; bfloat16 in others and float32 take the 32-bit kernel
    tensor_cores = code == L.BF16 and dim in (64, 128) and page_size in (8, 16, 32, 64) and num_pages > 0
    rows = TENSOR_CORE_ROWS if tensor_cores else FMA_ROWS
    # a multiple of the row tiles that trees have: then those of one head read its keys at the same time
    row_tiles = -(-max_nodes * (heads // kv_heads) // rows)
    if row_tiles < ctas:
        ctas -= ctas % row_tiles
    # scratch of this call alone (calls on several streams do not meet in it): two partial results for each CTA, and what
    # the merge has to know of it
    scratch = node_start.new_empty(2 * ctas * rows * (dim + 2) + 8 * ctas)
    args = _ATTENTION.pack(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(), ctx_len.data_ptr(), node_start.data_ptr(),
        0 if depth is None else depth.data_ptr(), visible.data_ptr(), out.data_ptr(), scratch.data_ptr(), q.stride(0),
        out.stride(0), page_table.stride(0), words, S, heads, kv_heads, dim, page_size, num_pages, window, code, ctas, scale)
    if tensor_cores:
        kernel, combine, error_word = _tensor_core_call(dev, dim)
        rc = kernel(args, combine, error_word, L.stream_handle())
        L.LaunchCounter.n += 2
        if rc != 0:
            _refuse(what, _TCGEN05_ERRORS.get(rc, str(rc)))
    else:
        L.check(L.core().dsp_tree_attention(args, L.stream_handle()), launches=2)
    return out


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
    gives count 0 and token -1; nodes beyond ``max_nodes`` are not tried."""
    what = "verify_tree"
    if not logits.is_cuda:
        _refuse(what, "CUDA tensors only (there is no CPU path)")
    if logits.dim() != 2 or logits.stride(1) != 1 or not 1 <= logits.shape[1] <= MAX_VOCAB:
        _refuse(what, f"logits must be [T, V] with neighbouring columns and V up to {MAX_VOCAB}, not {list(logits.shape)}")
    (T, V), S, dev = logits.shape, temperature.shape[0], logits.get_device()
    code = L.dtype_code(logits.dtype)
    _ints(what, "tokens", tokens, (T,), dev)
    _ints(what, "parents", parents, (T,), dev)
    _ints(what, "node_start", node_start, (S + 1,), dev)
    if not (_is(temperature, torch.float32, (S,), dev) and _is(uniforms, torch.float32, (T,), dev)
            and _is(draws, torch.float32, (S,), dev)):
        _refuse(what, f"temperature [{S}], uniforms [{T}] and draws [{S}] must be contiguous float32 on cuda:{dev}")
    if draft_probs is not None and (draft_probs.dtype is not torch.float32 or draft_probs.get_device() != dev
                                    or draft_probs.shape != (T, V) or draft_probs.stride(1) != 1):
        _refuse(what, f"draft_probs must be float32 [{T}, {V}] with neighbouring columns on cuda:{dev}")
    if not 1 <= max_nodes <= MAX_TREE:
        _refuse(what, f"max_nodes {max_nodes} outside 1 .. {MAX_TREE}")
    count, path, token = tokens.new_empty(S), tokens.new_empty((S, max_nodes)), tokens.new_empty(S)
    if S:
        draft, ldq = (0, 0) if draft_probs is None else (draft_probs.data_ptr(), draft_probs.stride(0))
        args = _VERIFY.pack(
            logits.data_ptr(), draft, tokens.data_ptr(), parents.data_ptr(), node_start.data_ptr(), temperature.data_ptr(),
            uniforms.data_ptr(), draws.data_ptr(), path.data_ptr(), count.data_ptr(), token.data_ptr(), logits.stride(0), ldq,
            S, V, max_nodes, code)
        L.check(L.core().dsp_tree_verify(args, L.stream_handle()))
    return Verified(count, path, token)


def keep_path(pools: list, page_table: torch.Tensor, ctx_len: torch.Tensor, path: torch.Tensor, count: torch.Tensor) -> None:
    """Moves what the cache keeps of the accepted nodes into line, in place: of tree s, place ``ctx_len[s] + j`` gets the
    rows of node ``path[s, j]`` for j < ``count[s]``.

    ``pools``: up to eight contiguous tensors [layers, pages, heads, page_size, width] of rows of whole 16-byte pieces,
    all with the pages of ``page_table`` [S, pages of a request]; ``path`` int32 [S, n] ascends within a tree, as
    ``verify_tree`` gives it (one that does not is left from there on and recorded as a device error)."""
    what = "keep_path"
    if not pools or len(pools) > MAX_POOLS:
        _refuse(what, f"{len(pools)} pools (1 to {MAX_POOLS})")
    if not pools[0].is_cuda:
        _refuse(what, "CUDA tensors only (there is no CPU path)")
    dev, S = pools[0].get_device(), ctx_len.shape[0]
    page_size = pools[0].shape[3] if pools[0].dim() == 5 else 0
    flat = []
    for p in pools:
        if p.dim() != 5 or p.shape[3] != page_size or not p.is_contiguous() or p.get_device() != dev:
            _refuse(what, f"a pool must be contiguous [layers, pages, heads, {page_size}, width] on cuda:{dev}, not {list(p.shape)}")
        layers, pages, heads, _, width = p.shape
        address, row = p.data_ptr(), width * p.element_size()
        if row % 16 or address % 16:
            _refuse(what, f"rows of {row} bytes (whole 16-byte pieces are moved)")
        flat += (address, layers, pages, heads, row)
    _ints(what, "ctx_len", ctx_len, (S,), dev)
    _ints(what, "count", count, (S,), dev)
    _table(what, page_table, S, dev)
    if path.dim() != 2:
        _refuse(what, f"path must be [S, n], not {list(path.shape)}")
    _ints(what, "path", path, (S, path.shape[1]), dev)
    if S == 0 or path.shape[1] == 0:
        return
    flat += [0] * (5 * MAX_POOLS - len(flat))
    args = _KEEP.pack(page_table.data_ptr(), ctx_len.data_ptr(), path.data_ptr(), count.data_ptr(), page_table.stride(0),
                      path.stride(0), path.shape[1], page_size, S, len(pools), *flat)
    L.check(L.core().dsp_tree_keep(args, L.stream_handle()))
