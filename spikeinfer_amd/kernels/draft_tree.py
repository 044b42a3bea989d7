"""Trees of drafted tokens: several tokens of a sequence verified in one step.

A step takes, per sequence, its last token (row 0 of its tree) and the drafted tokens
that may follow it, each below another.  The rows of all sequences lie one behind the
other, ``row_starts[n] .. row_starts[n + 1]`` those of sequence ``n``, a parent always
before its children.  Their q/k/v words come from :func:`qkv_rope_lif_pack` with
``kv_packed`` and every slot -1: the cache holds accepted tokens only, drafted keys stay
in the step's buffers until :func:`accept_draft_tree` moves the accepted path's.

    masks, depths = draft_tree_masks(parents, row_starts, max_nodes)
    out = paged_spike_attn_tree(q, k, v, k_cache, v_cache, tables, context_lens, row_starts, masks, ...)
    path, count, after = accept_draft_tree(tokens, parents, targets, row_starts, max_nodes, drafts, layers, ...)

Lengths, starts, parents and masks are device tensors that the kernels read, so a
captured step takes other trees on replay.  The reference decodes one token a step;
these have no counterpart there.
"""
from __future__ import annotations

import functools
import math

import torch

from .. import _lib
from .packing import packed_width
from .spike_attention import _as_int32, _check_packed

MAX_NODES = 1024


def _vector(name: str, t: torch.Tensor, entries: int, dtype: torch.dtype) -> torch.Tensor:
    if t.ndim != 1 or t.numel() < entries:
        raise ValueError(f"{name} must be a vector of {entries} entries, got {tuple(t.shape)}")
    if t.dtype != dtype:
        if dtype != torch.int32 or t.dtype != torch.int64:
            raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
        t = _as_int32(t)
    return t.contiguous()


def _max_nodes(max_nodes: int) -> None:
    if not 0 < max_nodes <= MAX_NODES:
        raise ValueError(f"max_nodes={max_nodes} must be in 1..{MAX_NODES}")


@functools.lru_cache(maxsize=256)
def tree_attn_workspace_bytes(T: int, n_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int,
                              max_nodes: int, block_size: int, max_blocks: int) -> int:
    """Scratch bytes :func:`paged_spike_attn_tree` needs for this shape."""
    return int(_lib.load().spk_tree_attn_workspace_bytes(T, n_seqs, num_q_heads, num_kv_heads, head_dim, max_nodes,
                                                         block_size, max_blocks))


def paged_spike_attn_tree(
    q_packed: torch.Tensor,
    k_words: torch.Tensor,
    v_words: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    row_starts: torch.Tensor,
    masks: torch.Tensor,
    max_nodes: int,
    head_dim: int,
    block_size: int,
    out: torch.Tensor | None = None,
    dtype: torch.dtype = torch.float32,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of drafted tokens: each row sees its sequence's cached context and
    the rows of its own tree that its mask names.

    Args:
        q_packed: ``int32 [T, R, H_q, W]`` query words of the rows.
        k_words, v_words: ``int32 [T, R, H_kv, W]`` the rows' own keys and values.
        k_cache, v_cache: ``int32 [T, H_kv, slots, W]``.
        block_tables: ``int32 [N, max_blocks]``; context_lens ``int32 [N]`` (cached
            tokens, the tree's not among them).
        row_starts: ``int32 [N + 1]``; a tree has at most ``max_nodes`` rows (others
            are left out).
        masks: ``int64 [R, M]``, ``M >= ceil(max_nodes / 64)``: bit ``i % 64`` of word
            ``i / 64`` lets the row see row ``i`` of its tree (:func:`draft_tree_masks`).
        out: optional ``[T, R, H_q, head_dim]``, channels contiguous (needed for graph
            capture); by default a new tensor of ``dtype``, zeros in rows of no sequence.
        workspace: optional ``uint8`` scratch of :func:`tree_attn_workspace_bytes`; calls that
            may run at once need one each.

    A row that sees nothing gets zeros; rows of ``out`` that are no sequence's are left as they
    were.  A sequence's outputs do not depend on the batch.
    """
    native = _lib.native()
    if native is not None:  # the usual form of the arguments, checked and launched in C++
        done = native.tree_attn(q_packed, k_words, v_words, k_cache, v_cache, block_tables, context_lens, row_starts,
                                masks, max_nodes, head_dim, block_size, out, dtype, workspace)
        if done is not None:
            return done
    T, R, n_heads, words = q_packed.shape
    dev = _lib.require_gpu(q_packed, k_words, v_words, k_cache, v_cache, block_tables, context_lens, row_starts, masks,
                           out, workspace)
    for name, t in (("q_packed", q_packed), ("k_words", k_words), ("v_words", v_words), ("k_cache", k_cache),
                    ("v_cache", v_cache)):
        _check_packed(name, t)
    if words != packed_width(head_dim):
        raise ValueError(f"q has {words} words, expected {packed_width(head_dim)}")
    hkv = k_cache.shape[1]
    if k_cache.shape != v_cache.shape or k_cache.stride() != v_cache.stride():
        raise ValueError("k and v caches must have the same shape and strides")
    if k_cache.shape[0] != T or k_cache.shape[3] != words or n_heads % max(hkv, 1):
        raise ValueError(f"cache shape {tuple(k_cache.shape)} does not match q {tuple(q_packed.shape)}")
    if tuple(k_words.shape) != (T, R, hkv, words) or k_words.shape != v_words.shape \
            or k_words.stride() != v_words.stride():
        raise ValueError(f"k_words and v_words must be {(T, R, hkv, words)} with the same strides")
    _max_nodes(max_nodes)
    if block_tables.ndim != 2:
        raise ValueError("block_tables must be [N, max_blocks]")
    block_tables = _as_int32(block_tables)
    n_seqs, max_blocks = block_tables.shape
    context_lens = _vector("context_lens", context_lens, n_seqs, torch.int32)
    row_starts = _vector("row_starts", row_starts, n_seqs + 1, torch.int32)
    if masks.dtype != torch.int64 or masks.ndim != 2 or masks.shape[0] != R or not masks.is_contiguous() \
            or masks.shape[1] * 64 < max_nodes:
        raise ValueError(f"masks must be contiguous int64 [{R}, >= {-(-max_nodes // 64)}]")
    if out is None:
        out = torch.zeros((T, R, n_heads, head_dim), dtype=dtype, device=dev)
    elif tuple(out.shape) != (T, R, n_heads, head_dim) or out.stride(-1) != 1:
        raise ValueError(f"out must be {(T, R, n_heads, head_dim)} with contiguous channels")
    if n_seqs == 0 or R == 0:
        return out
    need = tree_attn_workspace_bytes(T, n_seqs, n_heads, hkv, head_dim, max_nodes, block_size, max_blocks)
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        elif workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous():
            raise ValueError(f"workspace must hold {need} contiguous bytes")
    _lib.check(
        _lib.launch(
            "spk_tree_attn", dev, q_packed.data_ptr(), _lib.strides(q_packed), k_words.data_ptr(), v_words.data_ptr(),
            _lib.strides(k_words), k_cache.data_ptr(), v_cache.data_ptr(), _lib.strides(k_cache), k_cache.shape[2],
            block_tables.data_ptr(), block_tables.stride(0), block_tables.stride(1), context_lens.data_ptr(),
            row_starts.data_ptr(), masks.data_ptr(), masks.shape[1], out.data_ptr(), _lib.dtype_code(out.dtype),
            _lib.strides(out), R, n_seqs, max_nodes, T, n_heads, hkv, head_dim, block_size, max_blocks,
            1.0 / math.sqrt(head_dim), workspace.data_ptr() if need else None, need),
        "paged_spike_attn_tree",
    )
    return out


def draft_tree_masks(parents: torch.Tensor, row_starts: torch.Tensor, max_nodes: int,
                     masks: torch.Tensor | None = None,
                     depths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Masks ``int64 [R, ceil(max_nodes / 64)]`` of every row's ancestors and itself, and
    depths ``int32 [R]`` (0 for a root: row ``r`` stands at position ``context + depth``).

    ``parents int32 [R]`` numbers a row's parent within its tree, below the row itself;
    -1 (or a number that is not below it) has none.  Rows of no sequence are left as
    they were (zeros in new tensors)."""
    dev = _lib.require_gpu(parents, row_starts, masks, depths)
    _max_nodes(max_nodes)
    R, n_seqs = parents.numel(), row_starts.numel() - 1
    if n_seqs < 0:
        raise ValueError("row_starts must be [N + 1]")
    parents = _vector("parents", parents, R, torch.int32)
    row_starts = _vector("row_starts", row_starts, n_seqs + 1, torch.int32)
    words = -(-max_nodes // 64)
    if masks is None:
        masks = torch.zeros((R, words), dtype=torch.int64, device=dev)
    elif tuple(masks.shape[:1]) != (R,) or masks.ndim != 2 or masks.shape[1] < words or masks.dtype != torch.int64 \
            or not masks.is_contiguous():
        raise ValueError(f"masks must be contiguous int64 [{R}, >= {words}]")
    if depths is None:
        depths = torch.zeros(R, dtype=torch.int32, device=dev)
    elif tuple(depths.shape) != (R,) or depths.dtype != torch.int32 or not depths.is_contiguous():
        raise ValueError(f"depths must be contiguous int32 [{R}]")
    _lib.check(_lib.launch("spk_tree_masks", dev, parents.data_ptr(), row_starts.data_ptr(), R, n_seqs, max_nodes,
                           masks.data_ptr(), masks.shape[1], depths.data_ptr()), "draft_tree_masks")
    return masks, depths


def _same_layout(name: str, pairs, dev) -> tuple[torch.Size, tuple[int, ...]]:
    """Shape and strides that the packed tensors of every layer share."""
    for pair in pairs:
        if len(pair) != 2:
            raise ValueError(f"{name}: every layer must be a (k, v) pair, got {len(pair)} tensors")
    first = pairs[0][0]
    _check_packed(name, first)
    for pair in pairs:
        for t in pair:
            if t.shape != first.shape or t.stride() != first.stride() or t.dtype != torch.int32 or t.device != dev:
                raise ValueError(f"{name}: every layer's k and v must be int32 tensors of one shape, layout and device")
    return first.shape, first.stride()


def accept_draft_tree(
    tokens: torch.Tensor,
    parents: torch.Tensor,
    targets: torch.Tensor,
    row_starts: torch.Tensor,
    max_nodes: int,
    drafts: list[tuple[torch.Tensor, torch.Tensor]] = (),
    layers: list[tuple[torch.Tensor, torch.Tensor]] = (),
    block_tables: torch.Tensor | None = None,
    context_lens: torch.Tensor | None = None,
    block_size: int = 0,
    out: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The accepted path of every tree, and its words into the caches.

    From row 0 (accepted already: the sequence's last token) the walk goes to the
    lowest-numbered child whose token is the model's token after the current row, and
    ends where there is none.  With ``targets`` drawn by :func:`sample_tokens` from each
    row's logits the accepted tokens are distributed as tokens decoded one by one.

    Args:
        tokens, targets: ``int64 [R]`` each row's token and the model's token after it.
        parents, row_starts, max_nodes: as :func:`draft_tree_masks`.
        drafts: each layer's ``(k_words, v_words)``, ``int32 [T, R, H_kv, W]``.
        layers: each layer's ``(k_cache, v_cache)``, ``int32 [T, H_kv, slots, W]``; the
            path's words go to positions ``context_lens[n], context_lens[n] + 1, ...`` of
            ``block_tables[n]`` (``int32 [N, max_blocks]``).  A path ends before the first
            row whose position lies past the table or in a block outside the cache, so that
            ``count`` names the rows that are cached.  Without layers nothing moves.
        out: optional ``(path, count, next)`` buffers (for graph capture).

    Returns ``path int32 [N, max_nodes]`` (rows of the tree, -1 behind the path),
    ``count int32 [N]`` (the path's rows, row 0 among them; 0 for a sequence without rows,
    or without a place for row 0) and ``next int64 [N]``, the model's token after the path
    (-1 where ``count`` is 0).
    """
    native = _lib.native()
    if native is not None and layers:
        done = native.accept_tree(tokens, parents, targets, row_starts, max_nodes, drafts, layers, block_tables,
                                  context_lens, block_size, out)
        if done is not None:
            return done
    dev = _lib.require_gpu(tokens, parents, targets, row_starts, block_tables, context_lens, *(out or ()))
    _max_nodes(max_nodes)
    R, n_seqs = tokens.numel(), row_starts.numel() - 1
    if n_seqs < 0:
        raise ValueError("row_starts must be [N + 1]")
    tokens = _vector("tokens", tokens, R, torch.int64)
    targets = _vector("targets", targets, R, torch.int64)
    parents = _vector("parents", parents, R, torch.int32)
    row_starts = _vector("row_starts", row_starts, n_seqs + 1, torch.int32)
    if len(drafts) != len(layers):
        raise ValueError(f"{len(drafts)} layers of drafted words for {len(layers)} caches")
    new, cache, hkv, words, T, slots, max_blocks = (0, 0, 0), (0, 0, 0), 0, 0, 0, 0, 0
    bt, bts = None, (0, 0)
    if layers:
        if block_tables is None or context_lens is None or block_tables.ndim != 2 or block_tables.shape[0] != n_seqs:
            raise ValueError(f"caches need block_tables [{n_seqs}, max_blocks] and context_lens")
        (T, hkv, slots, words), cache = _same_layout("layers", layers, dev)
        shape, new = _same_layout("drafts", drafts, dev)
        if tuple(shape) != (T, R, hkv, words):
            raise ValueError(f"drafts are {tuple(shape)}, expected {(T, R, hkv, words)}")
        block_tables = _as_int32(block_tables)
        context_lens = _vector("context_lens", context_lens, n_seqs, torch.int32)
        max_blocks = block_tables.shape[1]
        bt, bts = block_tables.data_ptr(), block_tables.stride()
    if out is None:
        out = (torch.empty((n_seqs, max_nodes), dtype=torch.int32, device=dev),
               torch.empty(n_seqs, dtype=torch.int32, device=dev),
               torch.empty(n_seqs, dtype=torch.int64, device=dev))
    elif len(out) != 3:
        raise ValueError(f"out must be (path, count, next), got {len(out)} tensors")
    for t, shape, dt in zip(out, ((n_seqs, max_nodes), (n_seqs,), (n_seqs,)), (torch.int32, torch.int32, torch.int64)):
        if tuple(t.shape) != shape or t.dtype != dt or not t.is_contiguous():
            raise ValueError(f"out needs contiguous {dt} {shape}, got {t.dtype} {tuple(t.shape)}")
    i64x3 = _lib.ctypes.c_int64 * 3
    _lib.check(
        _lib.launch(
            "spk_accept_tree", dev, tokens.data_ptr(), parents.data_ptr(), targets.data_ptr(), row_starts.data_ptr(),
            R, n_seqs, max_nodes, *(t.data_ptr() for t in out),
            _lib.pack_pointers(d + c for d, c in zip(map(tuple, drafts), map(tuple, layers))), len(layers),
            i64x3(*new[:3]), i64x3(*cache[:3]), slots, bt, *bts, _lib.ptr(context_lens) if layers else None, T, hkv,
            32 * words, block_size, max_blocks),
        "accept_draft_tree",
    )
    return out
