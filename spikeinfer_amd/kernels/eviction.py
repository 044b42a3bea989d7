"""Keeping a cache within a budget: the attention weight of cached tokens, and the
eviction of those that get least.

    mass = paged_spike_attn_key_mass(q, k_cache, tables, lens, D, bs, out=mass, accumulate=True)   # every step
    keep, lens = evict_cache([(k_cache, v_cache)], mass[None], tables, lens, budget, bs)            # now and then

A cached key carries its rotary position in its bits, so tokens may move to other
slots; after an eviction ``seq_lens`` counts the tokens that stay, and the positions of
new tokens go on from the sequence's own.  The reference keeps every token; these have
no counterpart there.
"""
from __future__ import annotations

import functools
import math

import torch

from .. import _lib
from .draft_tree import _same_layout, _vector
from .packing import packed_width
from .spike_attention import _as_int32, _check_packed


@functools.lru_cache(maxsize=256)
def key_mass_workspace_bytes(T: int, n_seqs: int, num_q_heads: int, num_kv_heads: int, head_dim: int, max_rows: int,
                             block_size: int, max_blocks: int) -> int:
    """Scratch bytes :func:`paged_spike_attn_key_mass` needs for this shape."""
    return int(_lib.load().spk_key_mass_workspace_bytes(T, n_seqs, num_q_heads, num_kv_heads, head_dim, max_rows,
                                                        block_size, max_blocks))


def paged_spike_attn_key_mass(
    q_packed: torch.Tensor,
    k_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    head_dim: int,
    block_size: int,
    row_starts: torch.Tensor | None = None,
    max_rows: int = 1,
    out: torch.Tensor | None = None,
    accumulate: bool = False,
    workspace: torch.Tensor | None = None,
) -> torch.Tensor:
    """The softmax weight of every cached token, summed over timesteps, the query heads
    of its kv head and the sequence's last rows.

    Args:
        q_packed: ``int32 [T, R, H_q, W]``: without ``row_starts`` row ``n`` is sequence
            ``n``'s last token; with ``row_starts int32 [N + 1]`` rows ``row_starts[n] ..
            row_starts[n + 1]`` are its last ones, each seeing the positions up to its own.
            Of more than ``max_rows`` rows the last ``max_rows`` count; rows that
            ``q_packed`` does not have do not.
        k_cache: ``int32 [T, H_kv, slots, W]``; block_tables ``int32 [N, max_blocks]``;
            seq_lens ``int32 [N]`` with the rows' own tokens.
        out: optional ``float32 [N, H_kv, cap]``, entries contiguous; by default a new one
            of ``max_blocks * block_size`` entries.  Entries behind a sequence become 0;
            tokens at ``cap`` and behind are left out.
        accumulate: add to ``out`` instead, and leave the rest of it as it was.
        workspace: optional ``uint8`` scratch of :func:`key_mass_workspace_bytes`; calls that
            may run at once need one each.
    """
    native = _lib.native()
    if native is not None:
        done = native.key_mass(q_packed, k_cache, block_tables, seq_lens, head_dim, block_size, row_starts, max_rows,
                               out, accumulate, workspace)
        if done is not None:
            return done
    T, R, n_heads, words = q_packed.shape
    dev = _lib.require_gpu(q_packed, k_cache, block_tables, seq_lens, row_starts, out, workspace)
    _check_packed("q_packed", q_packed)
    _check_packed("k_cache", k_cache)
    if words != packed_width(head_dim):
        raise ValueError(f"q has {words} words, expected {packed_width(head_dim)}")
    hkv = k_cache.shape[1]
    if k_cache.shape[0] != T or k_cache.shape[3] != words or n_heads % max(hkv, 1):
        raise ValueError(f"cache shape {tuple(k_cache.shape)} does not match q {tuple(q_packed.shape)}")
    if block_tables.ndim != 2:
        raise ValueError("block_tables must be [N, max_blocks]")
    block_tables = _as_int32(block_tables)
    n_seqs, max_blocks = block_tables.shape
    seq_lens = _vector("seq_lens", seq_lens, n_seqs, torch.int32)
    if row_starts is not None:
        row_starts = _vector("row_starts", row_starts, n_seqs + 1, torch.int32)
    elif R < n_seqs:
        raise ValueError(f"q has {R} rows for {n_seqs} sequences")
    else:
        max_rows = 1
    if max_rows <= 0:
        raise ValueError(f"max_rows={max_rows} must be positive")
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs out")
        out = torch.empty((n_seqs, hkv, max_blocks * block_size), dtype=torch.float32, device=dev)
    elif out.ndim != 3 or tuple(out.shape[:2]) != (n_seqs, hkv) or out.dtype != torch.float32 or out.stride(-1) != 1:
        raise ValueError(f"out must be float32 [{n_seqs}, {hkv}, cap] with contiguous entries")
    need = key_mass_workspace_bytes(T, n_seqs, n_heads, hkv, head_dim, max_rows, block_size, max_blocks)
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        elif workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous():
            raise ValueError(f"workspace must hold {need} contiguous bytes")
    _lib.check(
        _lib.launch(
            "spk_key_mass", dev, q_packed.data_ptr(), _lib.strides(q_packed), k_cache.data_ptr(), _lib.strides(k_cache),
            k_cache.shape[2], block_tables.data_ptr(), block_tables.stride(0), block_tables.stride(1),
            seq_lens.data_ptr(), _lib.ptr(row_starts), out.data_ptr(), _lib.strides(out), out.shape[2], int(accumulate),
            R, n_seqs, max_rows, T, n_heads, hkv, head_dim, block_size, max_blocks,
            1.0 / math.sqrt(head_dim), workspace.data_ptr() if need else None, need),
        "paged_spike_attn_key_mass",
    )
    return out


def evict_cache(
    layers: list[tuple[torch.Tensor, torch.Tensor]],
    mass: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    budget: int,
    block_size: int,
    sinks: int = 4,
    recent: int = 32,
    dst_tables: torch.Tensor | None = None,
    mass_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Cuts every sequence of more than ``budget`` tokens to ``budget``, per layer and kv
    head: the first ``sinks`` and the last ``recent`` tokens stay, and of the others those
    of largest mass (equal: the lowest positions; NaN: last).

    Args:
        layers: each layer's ``(k_cache, v_cache)``, ``int32 [T, H_kv, slots, W]``.
        mass: ``float32 [L, N, H_kv, cap]``, entries contiguous; ``cap`` covers the
            sequences (tokens behind it are dropped).
        block_tables: ``int32 [N, max_blocks]``; seq_lens ``int32 [N]``.
        dst_tables: ``int32 [N, blocks]``, where the kept words go; by default the
            sequences' own blocks (which no other sequence may share).  These blocks must
            be none that the call reads, and lie in the cache (words for others are dropped).
        mass_out: where the kept masses go (0 behind them); by default ``mass`` itself, else a
            tensor apart from it.

    Returns ``keep int32 [L, N, H_kv, budget]``, the kept positions in order (-1 behind), and
    ``new_lens int32 [N] = min(seq_lens, budget)``.  The kept tokens stand at positions 0,
    1, ... of the destination; blocks behind them are free.
    """
    native = _lib.native()
    if native is not None:
        done = native.evict(layers, mass, block_tables, seq_lens, budget, block_size, sinks, recent, dst_tables, mass_out)
        if done is not None:
            return done
    dev = _lib.require_gpu(mass, block_tables, seq_lens, dst_tables, mass_out)
    if block_tables.ndim != 2 or (dst_tables is not None and
                                  (dst_tables.ndim != 2 or dst_tables.shape[0] != block_tables.shape[0])):
        raise ValueError("block_tables and dst_tables must be [N, blocks]")
    block_tables = _as_int32(block_tables)
    n_seqs, max_blocks = block_tables.shape
    seq_lens = _vector("seq_lens", seq_lens, n_seqs, torch.int32)
    if not layers:
        raise ValueError("no layers")
    (T, hkv, slots, words), strides = _same_layout("layers", layers, dev)
    for name, t in (("mass", mass), ("mass_out", mass_out)):
        if t is not None and (t.dtype != torch.float32 or t.ndim != 4 or t.stride(-1) != 1 or
                              tuple(t.shape[:3]) != (len(layers), n_seqs, hkv) or t.shape[3] != mass.shape[3]):
            raise ValueError(f"{name} must be float32 [{len(layers)}, {n_seqs}, {hkv}, cap] with contiguous entries")
    if mass_out is None:
        mass_out = mass
    dst, dst_strides, dst_blocks = None, (0, 0), 0
    if dst_tables is not None:
        dst_tables = _as_int32(dst_tables)
        dst, dst_strides, dst_blocks = dst_tables.data_ptr(), dst_tables.stride(), dst_tables.shape[1]
    keep = torch.empty((len(layers), n_seqs, hkv, max(budget, 0)), dtype=torch.int32, device=dev)
    new_lens = torch.empty(n_seqs, dtype=torch.int32, device=dev)
    i64x3 = _lib.ctypes.c_int64 * 3
    _lib.check(
        _lib.launch(
            "spk_evict", dev, _lib.pack_pointers(layers), len(layers), i64x3(*strides[:3]), slots, mass.data_ptr(),
            i64x3(*mass.stride()[:3]), mass_out.data_ptr(), i64x3(*mass_out.stride()[:3]), mass.shape[3],
            block_tables.data_ptr(), block_tables.stride(0), block_tables.stride(1), max_blocks, dst, *dst_strides,
            dst_blocks, seq_lens.data_ptr(), new_lens.data_ptr(), keep.data_ptr(), budget, sinks, recent, T, n_seqs,
            hkv, 32 * words, block_size),
        "evict_cache",
    )
    return keep, new_lens
