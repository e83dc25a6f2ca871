"""Pages of a paged cache shared between sequences: copied, forked, compacted.

Several continuations of one prompt (samples, beams) have the prompt's whole
pages in common; each needs a page of its own only from the one on that it
goes on writing.  ``CachePages`` holds the pools that one page numbering
serves, K and V of every layer and key weights, and moves their pages
together, from block tables on the device and without waiting for it.

No counterpart in the reference, whose pages belong to one sequence each.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from naivllm_amd import _lib


class _Pool(ctypes.Structure):
    """nsv_pool of include/naivspec.h."""

    _fields_ = [("base", ctypes.c_void_p), ("segments", ctypes.c_int32), ("key_bytes", ctypes.c_int32)]


@functools.lru_cache(maxsize=256)
def _fork_bytes(*shape: int) -> int:
    return int(_lib.lib().nsv_fork_pages_workspace_size(*shape))


@functools.lru_cache(maxsize=256)
def _compact_bytes(num_blocks: int) -> int:
    return int(_lib.lib().nsv_compact_pages_workspace_size(num_blocks))


class CachePages:
    """The pools of one page numbering.

    caches: K and V pools (num_blocks, block_size, Hkv, D), of any layers,
    bfloat16 or float32; key_weights: their (num_blocks, Hkv, block_size)
    float32 tables.  All contiguous and apart, on one device, of one num_blocks
    (at most 262,144) and block_size.  The handle keeps the tensors; it holds no
    other state, so several threads, streams and captured graphs may use it."""

    def __init__(self, caches, key_weights=()):
        caches, key_weights = list(caches), list(key_weights)
        if not caches:
            raise ValueError("CachePages needs at least one cache")
        first = caches[0]
        for t in caches:
            if not t.is_cuda:
                raise ValueError("CachePages moves pages on the GPU; a cache is on the CPU")
            if t.dim() != 4 or t.numel() == 0 or not t.is_contiguous():
                raise ValueError("caches must be contiguous (num_blocks, block_size, num_kv_heads, head_dim)")
            _lib.dtype_code(t.dtype)
            if t.device != first.device or t.shape[:2] != first.shape[:2]:
                raise ValueError("caches must share their device, num_blocks and block_size")
        nb, bs = first.shape[:2]
        for t in key_weights:
            if t.dim() != 3 or t.numel() == 0 or not t.is_contiguous() or t.dtype != torch.float32 or t.device != first.device:
                raise ValueError(f"key weights must be contiguous float32 on {first.device}")
            if t.shape[0] != nb or t.shape[2] != bs:
                raise ValueError(f"key weights must be ({nb}, num_kv_heads, {bs}), got {tuple(t.shape)}")
        self.device, self.num_blocks, self.block_size = first.device, nb, bs
        self._tensors = caches + key_weights
        at = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in self._tensors)
        if any(end > start for (_, end), (start, _) in zip(at, at[1:])):
            raise ValueError("pools overlap (their pages are moved at once)")
        pools = [_Pool(t.data_ptr(), 1, t.shape[2] * t.shape[3] * t.element_size()) for t in caches]
        pools += [_Pool(t.data_ptr(), t.shape[1], 4) for t in key_weights]
        self._pools = (_Pool * len(pools))(*pools)
        self._shape = (ctypes.addressof(self._pools), len(pools), nb, bs)

    def _like(self, t: torch.Tensor, shape: tuple, name: str, dtype=torch.int32) -> torch.Tensor:
        if t.dtype is not dtype or t.shape != shape or t.device != self.device:
            raise ValueError(f"{name} must be a {dtype} {shape} tensor on {self.device}, got {t.dtype} {tuple(t.shape)}")
        return t if t.is_contiguous() else t.contiguous()

    def _held(self, held: torch.Tensor | None) -> torch.Tensor | None:
        if held is None:
            return None
        if held.dtype is not torch.bool and held.dtype is not torch.uint8:
            raise ValueError(f"held must be bool or uint8, got {held.dtype}")
        return self._like(held, (self.num_blocks,), "held", held.dtype)

    def _out(self, t: torch.Tensor | None, like: torch.Tensor, name: str) -> torch.Tensor:
        if t is None:
            return torch.empty_like(like)
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        return self._like(t, like.shape, name, like.dtype)

    def copy(self, src: torch.Tensor, dst: torch.Tensor, keys: torch.Tensor | None = None) -> None:
        """Page src[i] to page dst[i] (int32, on the device) in every pool: its
        first keys[i] keys, or the whole page without ``keys``.  No page may be
        the target of two pairs, nor both a target and a source; a pair with an
        id outside the pools is left out."""
        if src.dim() != 1:
            raise ValueError("src must be (pairs,)")
        n = src.shape[0]
        src, dst = self._like(src, (n,), "src"), self._like(dst, (n,), "dst")
        keys = None if keys is None else self._like(keys, (n,), "keys")
        with _lib.on_device(self.device):
            rc = _lib.lib().nsv_copy_pages(*self._shape, src.data_ptr(), dst.data_ptr(), _lib.ptr(keys), n,
                                           _lib.stream_ptr(self.device))
        _lib.check(rc, "copy")

    def fork(self, block_tables: torch.Tensor, context_lens: torch.Tensor, parents: torch.Tensor, *,
             held: torch.Tensor | None = None, out_tables: torch.Tensor | None = None,
             out_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Rows that go on from other rows: row b of the new tables continues
        row parents[b] of the old (-1: the row ends, its pages are free unless
        another row has them).

        block_tables (B, pages) int32, -1 unmapped; context_lens (B,) int64;
        parents (B,) int32; B at most 4,096.  A row shares the pages that its
        parent's keys fill.  The partly filled page and those kept for later
        keys stay with the parent's first child (the lowest row); the later
        children get free pages in their place and a copy of the partly filled
        one's keys.  Free is a page that no new row has and that ``held``
        (num_blocks,), bool or uint8, does not mark; the lowest ids go first,
        row by row.  block_tables must hold every row that has pages: what
        they do not name is free.

        Returns (tables (B, pages), lens (B,), lacking ()): lacking is 0, or
        how many pages were short; then the first row that could not get its
        pages, and every later one that needs any, is empty.  ``out_tables``
        and ``out_lens`` may not overlap the old ones."""
        if block_tables.dim() != 2 or block_tables.shape[1] == 0:
            raise ValueError("block_tables must be (batch, pages)")
        shape = B, width = block_tables.shape
        block_tables = self._like(block_tables, shape, "block_tables")
        context_lens = self._like(context_lens, (B,), "context_lens", torch.int64)
        parents, held = self._like(parents, (B,), "parents"), self._held(held)
        out_tables = self._out(out_tables, block_tables, "out_tables")
        out_lens = self._out(out_lens, context_lens, "out_lens")
        lacking = parents.new_empty(())
        if B == 0:
            return out_tables, out_lens, lacking.zero_()
        h, nbytes = _lib.lib(), _fork_bytes(B, width, self.num_blocks)
        with _lib.on_device(self.device):
            stream = _lib.stream_ptr(self.device)
            scratch = _lib.stream_scratch(self.device, stream)
            with scratch.lock:
                ws = scratch.take(nbytes)
                rc = h.nsv_fork_pages(
                    *self._shape, block_tables.data_ptr(), context_lens.data_ptr(), parents.data_ptr(), _lib.ptr(held), B,
                    width, out_tables.data_ptr(), out_lens.data_ptr(), lacking.data_ptr(), ws.data_ptr(), nbytes, stream)
        _lib.check(rc, "fork")
        return out_tables, out_lens, lacking

    def compact(self, block_tables: torch.Tensor, *, held: torch.Tensor | None = None,
                out_tables: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Moves the pages that block_tables (B, pages) name, and ``held`` does
        not, to the front of the pools: the highest to the lowest free one
        while that lies before it.

        Returns (tables with the new ids, new_ids (num_blocks,) int32, top ()):
        new_ids is where a page in use or held is now (-1 for the others), and
        the first ``top`` pages are all that are in use or held.
        ``out_tables`` may be block_tables itself.  Block tables that are not
        given, a prefix cache's ids and the like follow by new_ids; pages that
        only they name must be held."""
        if block_tables.dim() != 2 or block_tables.shape[1] == 0:
            raise ValueError("block_tables must be (batch, pages)")
        shape = B, width = block_tables.shape
        block_tables = self._like(block_tables, shape, "block_tables")
        held = self._held(held)
        out_tables = self._out(out_tables, block_tables, "out_tables")
        new_ids, top = block_tables.new_empty(self.num_blocks), block_tables.new_empty(())
        h, nbytes = _lib.lib(), _compact_bytes(self.num_blocks)
        with _lib.on_device(self.device):
            stream = _lib.stream_ptr(self.device)
            scratch = _lib.stream_scratch(self.device, stream)
            with scratch.lock:
                ws = scratch.take(nbytes)
                rc = h.nsv_compact_pages(
                    *self._shape, block_tables.data_ptr(), _lib.ptr(held), B, width, out_tables.data_ptr(),
                    new_ids.data_ptr(), top.data_ptr(), ws.data_ptr(), nbytes, stream)
        _lib.check(rc, "compact")
        return out_tables, new_ids, top
