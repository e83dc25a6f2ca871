"""Verify-attention and KV-store operators with the reference's signatures.

Drop-in for ``paged_attention_verify`` and ``store_kvcache`` of
src/myvllm/layers/attention.py (:615-668 and :71-112) and for the verify
branch of ``Attention.forward`` (:689-731).  Both operators launch the
gfx950 kernels of libnaivspec.so on torch's current stream; there is no
PyTorch fallback.
"""

from __future__ import annotations

import ctypes
import functools

import torch
import torch.nn as nn

from naivllm_amd import _lib
from naivllm_amd.utils.context import get_context

_INDEX_DTYPES = {
    "block_tables": torch.int32,
    "context_lens": torch.int64,
    "cu_seqlens_q": torch.int32,
    "positions": torch.int64,
    "slot_mapping": torch.int64,
}


def _as(t: torch.Tensor, name: str) -> torch.Tensor:
    want = _INDEX_DTYPES[name]
    if t.dtype != want:
        t = t.to(want)
    return t if t.is_contiguous() else t.contiguous()


def _check_cache(cache: torch.Tensor, name: str) -> tuple[int, int, int, int]:
    if cache.dim() != 4:
        raise ValueError(f"{name} must be (num_blocks, block_size, num_kv_heads, head_dim), got {tuple(cache.shape)}")
    if not cache.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return tuple(cache.shape)


def verify_attention_workspace_bytes(batch_size: int, num_heads: int, num_kv_heads: int, head_dim: int,
                                     block_size: int, max_num_blocks: int, max_q_len: int,
                                     dtype: torch.dtype, kv_split_tokens: int = 0) -> int:
    return int(_lib.lib().nsv_verify_attention_workspace_size(
        batch_size, num_heads, num_kv_heads, head_dim, block_size, max_num_blocks, max_q_len,
        _lib.dtype_code(dtype), kv_split_tokens))


ATTN_KERNELS = {0: "d-sliced", 1: "key-split", 2: "fp32"}


def verify_attention_plan(batch_size: int, num_heads: int, num_kv_heads: int, head_dim: int, block_size: int,
                          max_num_blocks: int, max_q_len: int, dtype: torch.dtype, kv_split_tokens: int = 0,
                          cus: int = 0) -> tuple[str, int]:
    """(kernel, most key splits of a sequence) that paged_attention_verify runs
    for this shape on a device with ``cus`` compute units (0: the current
    one); a context shorter than the table may be cut into fewer."""
    kind, splits = ctypes.c_int(), ctypes.c_int()
    rc = _lib.lib().nsv_verify_attention_plan(batch_size, num_heads, num_kv_heads, head_dim, block_size,
                                             max_num_blocks, max_q_len, _lib.dtype_code(dtype), kv_split_tokens,
                                             cus, ctypes.addressof(kind), ctypes.addressof(splits))
    _lib.check(rc, "verify_attention_plan")
    return ATTN_KERNELS[kind.value], splits.value


def paged_attention_verify(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    positions: torch.Tensor,
    scale: float,
    num_heads: int,
    num_kv_heads: int,
    head_dim: int,
    block_size: int,
    block_m: int,
    *,
    max_q_len: int | None = None,
    kv_split_tokens: int = 0,
    out: torch.Tensor | None = None,
    allocation_free: bool = False,
    tile_references: bool = False,
) -> torch.Tensor:
    """Verify a chunk of drafted tokens against the paged KV cache.

    Same arguments and result as the reference (layers/attention.py:615-668):
      query (T, H, D); k_cache/v_cache (num_blocks, block_size, Hkv, D);
      block_tables (B, max_num_blocks), -1 padded; context_lens (B,);
      cu_seqlens_q (B+1,); positions (T,), -1 marks an inert pad row;
      block_m >= every per-sequence query length.
    Returns (T, H, D) in query's dtype.  Keyword-only extras: ``max_q_len``
    (a tighter bound than block_m: fewer padded MFMA rows and partials),
    ``kv_split_tokens`` (keys per workgroup split, 0 = automatic), ``out``
    (a preallocated result) and ``allocation_free`` (run through
    nsv_verify_attention_noalloc: the library's fixed per-device scratch
    instead of a workspace, ``out`` required, index tensors already int32 /
    int64 and contiguous, so the call allocates nothing), ``tile_references``
    (an exponent reference per tile of keys, nsv_verify_attention_tile_refs;
    not with allocation_free).  Rows at position
    -1 come back as zeros (the reference leaves them meaningless; nothing
    reads them).
    """
    if query.dim() != 3 or query.shape[1] != num_heads or query.shape[2] != head_dim:
        raise ValueError(f"query must be (T, {num_heads}, {head_dim}), got {tuple(query.shape)}")
    nb, bs, hkv, d = _check_cache(k_cache, "k_cache")
    if tuple(v_cache.shape) != (nb, bs, hkv, d) or not v_cache.is_contiguous():
        raise ValueError("k_cache and v_cache must have the same contiguous shape")
    if bs != block_size or hkv != num_kv_heads or d != head_dim:
        raise ValueError("cache shape disagrees with block_size / num_kv_heads / head_dim")
    if query.dtype != k_cache.dtype or v_cache.dtype != k_cache.dtype:
        raise ValueError("query and caches must share one dtype")
    if not query.is_cuda:
        raise ValueError("paged_attention_verify runs on the GPU; query is on the CPU")
    query = query.contiguous()
    block_tables = _as(block_tables, "block_tables")
    context_lens = _as(context_lens, "context_lens")
    cu_seqlens_q = _as(cu_seqlens_q, "cu_seqlens_q")
    positions = _as(positions, "positions")
    batch_size, max_num_blocks = block_tables.shape
    qlen_bound = int(max_q_len if max_q_len is not None else block_m)
    code = _lib.dtype_code(query.dtype)
    h = _lib.lib()
    if out is not None and (tuple(out.shape) != tuple(query.shape) or out.dtype != query.dtype
                            or out.device != query.device or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous {query.dtype} tensor of shape {tuple(query.shape)} on "
                         f"{query.device}")
    if allocation_free:
        if out is None:
            raise ValueError("allocation_free=True needs a preallocated out")
        if tile_references:
            raise ValueError("allocation_free=True takes no tile_references")
        rc = h.nsv_verify_attention_noalloc(
            out.data_ptr(), query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(),
            context_lens.data_ptr(), cu_seqlens_q.data_ptr(), positions.data_ptr(), float(scale), batch_size,
            query.shape[0], num_heads, num_kv_heads, head_dim, block_size, max_num_blocks, qlen_bound, code,
            kv_split_tokens, _lib.stream_ptr(query.device))
        _lib.check(rc, "paged_attention_verify (allocation-free)")
        return out
    if out is None:
        out = torch.empty_like(query)
    ws_bytes = int(h.nsv_verify_attention_workspace_size(
        batch_size, num_heads, num_kv_heads, head_dim, block_size, max_num_blocks, qlen_bound, code,
        kv_split_tokens))
    stream = _lib.stream_ptr(query.device)
    name = "verify_attention"
    if tile_references and not torch.cuda.is_current_stream_capturing():
        # (prefill steps may run beside another stream's rounds: scratch of
        # their own per stream, of which torch has a fixed pool)
        name = f"verify_attention on stream {stream}"
    ws = _lib.workspace(query.device, ws_bytes, name)
    rc = (h.nsv_verify_attention_tile_refs if tile_references else h.nsv_verify_attention)(
        out.data_ptr(), query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        block_tables.data_ptr(), context_lens.data_ptr(), cu_seqlens_q.data_ptr(), positions.data_ptr(),
        float(scale), batch_size, query.shape[0], num_heads, num_kv_heads, head_dim, block_size,
        max_num_blocks, qlen_bound, code, kv_split_tokens,
        _lib.ptr(ws), ws_bytes, stream)
    _lib.check(rc, "paged_attention_verify")
    return out


def _few_rows(query, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, positions, num_heads: int,
              num_kv_heads: int, head_dim: int, block_size: int, out, what: str) -> tuple:
    """The checks of the few-row operators over a paged cache; returns query,
    the index tensors in the kernels' types, and the output.  What a serving
    loop passes goes through one condition; everything else is told apart,
    converted or refused, in _check_few_rows."""
    dev, kshape = query.get_device(), k_cache.shape
    B, T = context_lens.numel(), positions.numel()
    if not (dev >= 0 and query.shape == (T, num_heads, head_dim) and v_cache.shape == kshape
            and kshape[1:] == (block_size, num_kv_heads, head_dim) and kshape[0] * block_size <= 0x7fffffff
            and query.dtype == k_cache.dtype == v_cache.dtype and query.is_contiguous() and k_cache.is_contiguous()
            and v_cache.is_contiguous() and (query.data_ptr() | k_cache.data_ptr() | v_cache.data_ptr()) % 16 == 0
            and k_cache.get_device() == v_cache.get_device() == block_tables.get_device() == context_lens.get_device()
            == cu_seqlens_q.get_device() == positions.get_device() == dev
            and block_tables.dtype == cu_seqlens_q.dtype == torch.int32 and block_tables.is_contiguous()
            and context_lens.dtype == positions.dtype == torch.int64 and context_lens.is_contiguous()
            and positions.is_contiguous() and cu_seqlens_q.is_contiguous() and block_tables.dim() == 2
            and block_tables.shape[0] == B and context_lens.dim() == cu_seqlens_q.dim() == positions.dim() == 1
            and cu_seqlens_q.numel() == B + 1 and out is None):
        return _check_few_rows(query, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, positions, num_heads,
                               num_kv_heads, head_dim, block_size, out, what)
    return query, block_tables, context_lens, cu_seqlens_q, positions, torch.empty_like(query)


def _check_few_rows(query, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, positions, num_heads: int,
                    num_kv_heads: int, head_dim: int, block_size: int, out, what: str) -> tuple:
    """The checks of the few-row operators over a paged cache; returns the
    index tensors in the kernels' types and the output."""
    if not query.is_cuda:
        raise ValueError(f"{what} runs on the GPU; query is on the CPU")
    if query.dim() != 3 or query.shape[1] != num_heads or query.shape[2] != head_dim:
        raise ValueError(f"query must be (T, {num_heads}, {head_dim}), got {tuple(query.shape)}")
    nb, bs, hkv, d = _check_cache(k_cache, "k_cache")
    if v_cache.shape != k_cache.shape or not v_cache.is_contiguous():
        raise ValueError("k_cache and v_cache must have the same contiguous shape")
    if bs != block_size or hkv != num_kv_heads or d != head_dim:
        raise ValueError("cache shape disagrees with block_size / num_kv_heads / head_dim")
    if query.dtype != k_cache.dtype or v_cache.dtype != k_cache.dtype:
        raise ValueError("query and caches must share one dtype")
    if nb * bs > 0x7fffffff:
        raise ValueError(f"{what} addresses fewer than 2^31 cached keys, got {nb} pages of {bs}")
    if (k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise ValueError("k_cache and v_cache must start on 16 bytes")
    dev = query.device
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables),
                    ("context_lens", context_lens), ("cu_seqlens_q", cu_seqlens_q), ("positions", positions)):
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, query on {dev}")
    if block_tables.dim() != 2:
        raise ValueError(f"block_tables must be (B, max_num_blocks), got {tuple(block_tables.shape)}")
    B, T = block_tables.shape[0], query.shape[0]
    if tuple(context_lens.shape) != (B,) or tuple(cu_seqlens_q.shape) != (B + 1,) or tuple(positions.shape) != (T,):
        raise ValueError(f"context_lens, cu_seqlens_q and positions must have {B}, {B + 1} and {T} entries, got "
                         f"{tuple(context_lens.shape)}, {tuple(cu_seqlens_q.shape)} and {tuple(positions.shape)}")
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {query.dtype} tensor of shape {tuple(query.shape)} on {dev}")
    elif out.data_ptr() % 16:
        raise ValueError("out must start on 16 bytes")
    elif out.numel() and abs(out.data_ptr() - query.data_ptr()) < out.numel() * out.element_size():
        raise ValueError("out must not overlap query")
    return (_aligned(query.contiguous()), _as(block_tables, "block_tables"), _as(context_lens, "context_lens"),
            _as(cu_seqlens_q, "cu_seqlens_q"), _as(positions, "positions"), out)


def _check_key_weights(key_weights: torch.Tensor, k_cache: torch.Tensor) -> None:
    nb, bs, hkv, _ = k_cache.shape
    if (tuple(key_weights.shape) != (nb, hkv, bs) or key_weights.dtype != torch.float32
            or key_weights.device != k_cache.device or not key_weights.is_contiguous()):
        raise ValueError(f"key_weights must be a contiguous fp32 tensor of shape {(nb, hkv, bs)} on {k_cache.device}, got "
                         f"{key_weights.dtype} {tuple(key_weights.shape)} on {key_weights.device}")


@functools.lru_cache(maxsize=512)
def _window_workspace_bytes(*shape: int) -> int:
    return int(_lib.lib().nsv_window_attention_workspace_size(*shape))


@functools.lru_cache(maxsize=512)
def _evict_workspace_bytes(*shape: int) -> int:
    return int(_lib.lib().nsv_evict_workspace_size(*shape))


@functools.lru_cache(maxsize=512)
def _weights_workspace_bytes(*shape: int) -> int:
    return int(_lib.lib().nsv_weights_attention_workspace_size(*shape))


def _int_arg(value, name: str, least: int) -> int:
    """A host integer of at least ``least``, capped where it means no bound
    to the kernels (no table holds 2^30 keys)."""
    try:
        whole = int(value) == value and value >= least
    except (OverflowError, TypeError, ValueError):  # (infinite; no number; NaN)
        whole = False
    if not whole:
        raise ValueError(f"{name} must be an integer of at least {least}, got {value}")
    return min(int(value), 1 << 30)


def paged_attention_window(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    positions: torch.Tensor,
    scale: float,
    num_heads: int,
    num_kv_heads: int,
    head_dim: int,
    block_size: int,
    block_m: int,
    *,
    window: int,
    sinks: int = 0,
    max_q_len: int | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """paged_attention_verify with a sliding window: the row at position p
    sees the keys j <= p with j > p - window or j < sinks (a few first tokens
    that stay visible); bfloat16 and float32, up to 64 rows per sequence.

    Only keys that some row of their sequence sees are read, so the pages
    between the sinks and the windows may be given to other sequences (their
    entries any value, -1 included), and what they hold (NaN, say) reaches no
    result; a key that one row sees and another does not must be finite.  A row
    that sees no key, and a row at position -1, comes back as zeros; rows behind
    the last sequence (cu_seqlens_q[-1]) are not written.  Scratch
    and arrival counters are the stream's own (a captured call's scratch its
    graph's): calls on several streams, and captured ones, share nothing.
    No counterpart in the reference, whose attention sees every key."""
    window, sinks = _int_arg(window, "window", 1), _int_arg(sinks, "sinks", 0)
    query, block_tables, context_lens, cu_seqlens_q, positions, out = _few_rows(
        query, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, positions, num_heads, num_kv_heads, head_dim,
        block_size, out, "paged_attention_window")
    B, max_blocks = block_tables.shape
    shape = (num_heads, num_kv_heads, head_dim, block_size, max_blocks, int(block_m if max_q_len is None else max_q_len),
             _lib.dtype_code(query.dtype), window, sinks)
    dev = query.device
    with _lib.on_device(dev):
        stream = _lib.stream_ptr(dev)
        scratch = _lib.stream_scratch(dev, stream)
        with scratch.lock:
            ws = scratch.take(_window_workspace_bytes(B, *shape))
            rc = _lib.lib().nsv_window_attention(
                out.data_ptr(), query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(),
                context_lens.data_ptr(), cu_seqlens_q.data_ptr(), positions.data_ptr(), scale, B, query.shape[0], *shape,
                _lib.ptr(scratch.counters), ws.data_ptr(), ws.numel(), stream)
    _lib.check(rc, "paged_attention_window")
    return out


def paged_attention_weights(
    query: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    key_weights: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    positions: torch.Tensor,
    scale: float,
    num_heads: int,
    num_kv_heads: int,
    head_dim: int,
    block_size: int,
    block_m: int,
    *,
    max_q_len: int | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """paged_attention_verify that also keeps score of the keys:
    ``key_weights`` (num_blocks, num_kv_heads, block_size) fp32, paged as the
    cache is, holds for every (key, kv head) the attention weights that the
    key got, summed over rows and over the query heads of its kv head.

    A call adds its rows' weights to the keys before the position of the
    sequence's first row; those from there on are new, and their places are
    set (so nothing has to be cleared when a page is handed out).  Rows at
    position -1 see nothing and add nothing.  Places of keys past the last
    row, and of unmapped pages, keep what they hold.  evict_kvcache reads the
    table; prefill_key_weights adds a prompt's rows.  bfloat16 and float32, up
    to 64 rows per sequence.  A page that several sequences of a call share
    gets the sum of theirs, in no fixed order, on top of nothing where the key
    is new to one of them.  Scratch as paged_attention_window's.  No
    counterpart in the reference."""
    query, block_tables, context_lens, cu_seqlens_q, positions, out = _few_rows(
        query, k_cache, v_cache, block_tables, context_lens, cu_seqlens_q, positions, num_heads, num_kv_heads, head_dim,
        block_size, out, "paged_attention_weights")
    _check_key_weights(key_weights, k_cache)
    B, max_blocks = block_tables.shape
    shape = (num_heads, num_kv_heads, head_dim, block_size, max_blocks, int(block_m if max_q_len is None else max_q_len),
             _lib.dtype_code(query.dtype))
    dev = query.device
    with _lib.on_device(dev):
        stream = _lib.stream_ptr(dev)
        scratch = _lib.stream_scratch(dev, stream)
        with scratch.lock:
            ws = scratch.take(_weights_workspace_bytes(B, *shape))
            rc = _lib.lib().nsv_weights_attention(
                out.data_ptr(), query.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), key_weights.data_ptr(),
                block_tables.data_ptr(), context_lens.data_ptr(), cu_seqlens_q.data_ptr(), positions.data_ptr(), scale, B,
                query.shape[0], *shape, ws.data_ptr(), ws.numel(), stream)
    _lib.check(rc, "paged_attention_weights")
    return out


def store_kvcache(
    key: torch.Tensor,
    value: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    block_size: int,
) -> None:
    """Scatter (T, Hkv, D) key/value rows into the paged caches at
    ``slot_mapping`` (slot -1 = skip), as layers/attention.py:71-112."""
    num_tokens, num_kv_heads, head_dim = key.shape
    key = key.contiguous()
    value = value.contiguous()
    if k_cache.shape != v_cache.shape:
        raise ValueError("K and V cache shapes must match")
    if slot_mapping.numel() != num_tokens:
        raise ValueError("Slot mapping size must match number of tokens")
    nb, bs, hkv, d = _check_cache(k_cache, "k_cache")
    if not v_cache.is_contiguous():
        raise ValueError("v_cache must be contiguous")
    if (bs, hkv, d) != (block_size, num_kv_heads, head_dim):
        raise ValueError("cache shape disagrees with key shape / block_size")
    if key.dtype != k_cache.dtype or value.dtype != v_cache.dtype:
        raise ValueError("key/value and caches must share one dtype")
    slot_mapping = _as(slot_mapping, "slot_mapping")
    rc = _lib.lib().nsv_store_kv(
        key.data_ptr(), value.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(),
        num_tokens, num_kv_heads, head_dim, block_size, _lib.dtype_code(key.dtype),
        _lib.stream_ptr(key.device))
    _lib.check(rc, "store_kvcache")


def _prefill_lengths(seqlens_q, seqlens_k) -> tuple[list[int], list[int]]:
    """The lengths as lists of ints, checked."""
    seqlens_q, seqlens_k = [int(x) for x in seqlens_q], [int(x) for x in seqlens_k]
    if len(seqlens_q) != len(seqlens_k):
        raise ValueError("seqlens_q and seqlens_k differ in length")
    for i, (ql, kl) in enumerate(zip(seqlens_q, seqlens_k)):
        if not 0 < ql <= kl:
            raise ValueError(f"prefill sequence {i}: {ql} query rows over {kl} keys")
    return seqlens_q, seqlens_k


def _host_list(build, seqlens_q, seqlens_k, words_of, pinned: bool, what: str) -> tuple[torch.Tensor, list[int]]:
    """A native work list of the sequences in a host tensor: build(seqlens_q,
    seqlens_k, n, its address, its words, counts) fills it, and says
    (words_of(counts)) how many words it has.  Returns (the words, counts)."""
    seqlens_q, seqlens_k = _prefill_lengths(seqlens_q, seqlens_k)
    n = len(seqlens_q)
    q, k, counts = (ctypes.c_int64 * n)(*seqlens_q), (ctypes.c_int64 * n)(*seqlens_k), (ctypes.c_int32 * 4)()
    words = 4096
    while True:
        buf = torch.empty(words, dtype=torch.int32, pin_memory=pinned)
        rc = build(q, k, n, buf.data_ptr(), words, counts)
        need = words_of(counts)
        if rc == 0 or need <= words:
            break
        words = need
    _lib.check(rc, what)
    return buf[:need], list(counts)


def _prefill_work(seqlens_q, seqlens_k, num_heads: int, num_kv_heads: int, block_size: int | None, cus: int,
                  window: int, sinks: int, pinned: bool) -> tuple[torch.Tensor, list[int]]:
    """nsv_prefill_window_tiles into a host tensor; returns (its words,
    [tiles, merges, tile_rows, slots])."""
    def build(q, k, n, at, words, counts):
        return _lib.lib().nsv_prefill_window_tiles(q, k, n, num_heads, num_kv_heads, block_size or 0, cus, window, sinks,
                                                   at, words, counts)

    return _host_list(build, seqlens_q, seqlens_k, lambda c: 8 * c[0] + 4 * c[1], pinned, "prefill_tiles")


def prefill_tiles(seqlens_q, seqlens_k, num_heads: int, num_kv_heads: int, block_size: int | None, cus: int):
    """The prefill kernel's work list for sequences of seqlens_q new rows
    ending seqlens_k keys each (nsv_prefill_tiles); block_size None: K/V are
    the sequences' keys back to back.  Host only.
    Returns (tiles [n, 8] int32, merges [m, 4] int32, tile_rows, slots)."""
    work, (nt, nm, rows, slots) = _prefill_work(seqlens_q, seqlens_k, num_heads, num_kv_heads, block_size, cus, 0, 0, False)
    return work[:8 * nt].view(nt, 8).numpy(), work[8 * nt:].view(nm, 4).numpy(), rows, slots


class _StepList:
    """A prefill step's metadata on the device, in one transfer (``work``).

    The transfer is enqueued on the stream that is current here and not waited
    for; a call on another stream waits for it on the device (use_on)."""

    def _send(self, work: torch.Tensor, device, ahead: bool) -> None:
        self.work = work.to(device, non_blocking=ahead)
        stream = torch.cuda.current_stream(device)
        self.stream = stream.cuda_stream
        self.ready = torch.cuda.Event() if ahead else None  # the transfer is done
        if ahead:
            self.ready.record(stream)

    def use_on(self, stream) -> None:
        """Order work enqueued on ``stream`` after the transfer, and keep the
        list's memory until that work is done.  A capture on another stream
        can hold no wait for an event from outside it, and needs none:
        torch.cuda.graph waits for the device before it begins, and whoever
        replays the graph keeps the plan."""
        if stream.cuda_stream == self.stream or torch.cuda.is_current_stream_capturing():
            return
        if self.ready is not None:
            stream.wait_event(self.ready)
        self.work.record_stream(stream)

    def use_here(self, device: torch.device) -> int:
        """use_on the device's current stream; returns its handle."""
        stream = _lib.stream_ptr(device)
        if stream != self.stream:
            self.use_on(torch.cuda.current_stream(device))
        return stream


def _send_ahead() -> bool:
    """As _lib.upload: a step's transfer is not waited for, except inside a
    capture, which refuses the wait."""
    return not torch.cuda.is_current_stream_capturing()


class PrefillPlan(_StepList):
    """The prefill kernel's work list of one step on the device.  window and
    sinks: every row sees its last ``window`` keys and its sequence's first
    ``sinks`` (window 0: all keys up to it)."""

    def __init__(self, seqlens_q, seqlens_k, num_heads: int, num_kv_heads: int, block_size: int | None, device,
                 window: int = 0, sinks: int = 0):
        self.window, self.sinks = _int_arg(window, "window", 0), _int_arg(sinks, "sinks", 0)
        cus = torch.cuda.get_device_properties(device).multi_processor_count
        ahead = _send_ahead()
        work, (self.ntiles, self.nmerges, self.tile_rows, self.slots) = _prefill_work(
            seqlens_q, seqlens_k, num_heads, num_kv_heads, block_size, cus, self.window, self.sinks, ahead)
        self.num_heads, self.num_kv_heads, self.block_size = num_heads, num_kv_heads, block_size
        self.sequences, self.rows, self.keys = len(seqlens_q), int(sum(seqlens_q)), int(sum(seqlens_k))
        self._send(work, device, ahead)


class KeyWeightsPlan(_StepList):
    """The work list of prefill_key_weights of one step on the device."""

    def __init__(self, seqlens_q, seqlens_k, num_heads: int, num_kv_heads: int, block_size: int, device):
        cus = torch.cuda.get_device_properties(device).multi_processor_count
        ahead = _send_ahead()

        def build(q, k, n, at, words, counts):
            return _lib.lib().nsv_key_weights_units(q, k, n, num_heads, num_kv_heads, cus, at, words, counts)

        work, (self.nunits, self.nsums, _, _) = _host_list(build, seqlens_q, seqlens_k, lambda c: 8 * c[0] + 6 * c[1],
                                                           ahead, "key_weights_units")
        self.num_heads, self.num_kv_heads, self.block_size = num_heads, num_kv_heads, block_size
        self.sequences, self.rows, self.longest = len(seqlens_q), int(sum(seqlens_q)), int(max(seqlens_k, default=0))
        self._send(work, device, ahead)


class PrefillRows(_StepList):
    """The verify kernel's metadata of a prefill step of a few rows per
    sequence (verify_serves_prefill) on the device: context_lens, positions
    and cu_seqlens_q, one entry per sequence or row."""

    def __init__(self, seqlens_q, seqlens_k, device):
        ql, kl = _prefill_lengths(seqlens_q, seqlens_k)
        n, rows, ahead = len(ql), sum(ql), _send_ahead()
        work = torch.empty(n + rows + n // 2 + 1, dtype=torch.int64, pin_memory=ahead)
        work[:n] = torch.tensor(kl, dtype=torch.int64)
        work[n:n + rows] = torch.cat([torch.arange(k - q, k) for q, k in zip(ql, kl)])
        work[n + rows:].view(torch.int32)[:n + 1] = torch.tensor([0] + ql).cumsum(0)
        self.sequences, self.rows, self.max_q_len = n, rows, max(ql)
        self._send(work, device, ahead)
        self.context_lens, self.positions = self.work[:n], self.work[n:n + rows]
        self.cu_seqlens_q = self.work[n + rows:].view(torch.int32)[:n + 1]


class _WeightTurns(_StepList):
    """The calls of an fp32 prefill step with key weights, in one transfer:
    causal blocks of up to ``q_block`` rows, a sequence's in turns of their own
    (two in one call would add to the same places), every sequence's by the
    block's first position, so that a prefix that one of them computes is set
    before the others that have it behind them add to it.  ``turns``: (rows, or
    the first and last + 1 of neighbours; block tables, context_lens,
    cu_seqlens_q, positions)."""

    def __init__(self, seqlens_q, seqlens_k, block_tables: torch.Tensor, q_block: int, device):
        ql, kl = _prefill_lengths(seqlens_q, seqlens_k)
        if block_tables.shape[0] < len(ql):
            raise ValueError(f"{len(ql)} sequences but {block_tables.shape[0]} block-table rows")
        tables = block_tables.to("cpu", torch.int32)  # (waits, once per step)
        blocks: dict[int, list[tuple[int, int, int, int]]] = {}  # turn -> (sequence, first row, rows, first position)
        row0 = 0
        for b, (n, end) in enumerate(zip(ql, kl)):
            for r in range(0, n, q_block):
                first = end - n + r
                blocks.setdefault(first // q_block, []).append((b, row0 + r, min(q_block, n - r), first))
            row0 += n
        words: list[torch.Tensor] = []  # int64: per turn rows, lens, positions, then cu and the tables in halves of words
        cuts, at = [], 0
        for _, turn in sorted(blocks.items()):
            rows = torch.cat([torch.arange(r, r + n) for _, r, n, _ in turn])
            lens = torch.tensor([p + n for _, _, n, p in turn])
            positions = torch.cat([torch.arange(p, p + n) for _, _, n, p in turn])
            half = torch.cat([torch.tensor([0] + [n for _, _, n, _ in turn]).cumsum(0).to(torch.int32),
                              tables[[b for b, *_ in turn]].flatten()])
            half = torch.cat([half, half.new_zeros(half.numel() % 2)]).view(torch.int64)
            words += [rows, lens, positions, half]
            cuts.append((at, rows.numel(), len(turn), (int(rows[0]), int(rows[-1]) + 1) if len(turn) == 1 else None))
            at += 2 * rows.numel() + lens.numel() + half.numel()
        ahead = _send_ahead()
        work = torch.cat(words)
        self._send(work.pin_memory() if ahead else work, device, ahead)
        self.rows, self.turns = row0, []
        for at, n, count, whole in cuts:
            rows, lens, positions = self.work[at:at + n], self.work[at + n:at + n + count], self.work[at + n + count:at + 2 * n + count]
            half = self.work[at + 2 * n + count:].view(torch.int32)
            self.turns.append((whole or rows, half[count + 1:count + 1 + count * tables.shape[1]].view(count, -1), lens,
                               half[:count + 1], positions))


def verify_serves_prefill(seqlens_q, seqlens_k, num_heads: int, num_kv_heads: int, block_size: int,
                          max_num_blocks: int) -> bool:
    """Whether a paged bf16 prefill step runs on the verify kernel, one block
    of rows per sequence, and not on the prefill kernel.

    The prefill kernel's waves hold 32 rows of one query head and a workgroup
    two heads of a kv head, so a short suffix behind a long prefix leaves most
    of its waves without rows and a group of 4 or more heads reads its K/V
    twice or more; the verify kernel packs the group's rows.  MI355X,
    graph-replayed, prefill -> verify kernel, us per layer: 16/8 heads, one
    sequence of 9 rows behind 1,024 keys 14.7 -> 8.8, behind 16,384 47 -> 28,
    eight of 24 behind 4,096 61 -> 30; 32/8 heads, eight of 4 behind 4,096 98 ->
    26, of 12 99 -> 31.  The lines: up to 48 packed rows (the key-split kernel's
    three row tiles) wherever that kernel takes the table and 8 pairs or more
    are there, beyond one row tile (2 pairs and 16 rows of 3 heads: 17 -> 22);
    where it does not take the table (24,000 keys in pages of one or 16 tokens)
    groups of more than two heads only (32/8 heads 524 -> 342, 16/8 274 -> 336).
    Up to 64 packed rows (the verify kernel's most) groups of more than two
    heads with 1,536 keys or more: 32/8 heads, eight of 16 rows behind 4,096
    keys 101 -> 77, behind 1,024 24 -> 27; 16/8 heads, of 32 63 -> 77."""
    group, pairs, longest = num_heads // num_kv_heads, len(seqlens_q) * num_kv_heads, max(seqlens_k, default=0)
    rows = group * max(seqlens_q, default=0)
    if rows < 1 or rows > 64 or max_num_blocks * block_size >= 1 << 22:
        return False
    key_split = block_size >= 16 and max_num_blocks <= 1024
    if rows <= 48:
        return (pairs >= 8 or rows <= 16) and (key_split or group > 2)
    return pairs >= 8 and key_split and group > 2 and longest >= 1536


def few_rows_serve_prefill(seqlens_q, num_heads: int, num_kv_heads: int) -> bool:
    """Whether a paged bf16 prefill step with a window, or with key weights,
    runs on the few-row kernels (paged_attention_window / _weights), one block
    of rows per sequence, and not on the prefill kernels: up to 48 packed rows
    (query heads of a kv head x rows).  MI355X, graph-replayed, prefill kernels
    -> few-row ones, us per layer: a window of 1,024 behind 4,096 keys, 16/8
    heads, one sequence of 9 rows 15.7 -> 11.5, eight 18.2 -> 16.2, of 32 21.7 ->
    24.0 (64 packed rows: the prefill kernels), 32/8 heads, eight of 9 23.8 ->
    19.8, of 16 25.2 -> 23.8; behind 256 keys 15.3 -> 14.1, of 16 15.8 -> 16.9.
    Key weights of the same: 29.6 -> 17.7, 87.6 -> 47.1, 90.3 -> 66.5, 135.7 ->
    55.4; behind 256 keys 23.4 -> 21.8, of 16 23.9 -> 29.8."""
    return 1 <= num_heads // num_kv_heads * max(seqlens_q, default=0) <= 48


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t on 16 bytes, as the loads of the prefill kernel that go straight to
    LDS need it: a view at an odd offset is copied (what torch allocates is
    aligned)."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def prefill_attention(query: torch.Tensor, k: torch.Tensor, v: torch.Tensor, plan: PrefillPlan, scale: float,
                      head_dim: int, block_tables: torch.Tensor | None = None, *,
                      stats: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of a prefill step's rows (bf16): query [rows, H, D];
    k, v the step's own [keys, Hkv, D], or with block_tables the paged caches
    [num_blocks, block_size, Hkv, D] (layers/attention.py:123-363).  With a
    window in the plan every row sees that many keys and the first ``sinks``
    (no reference counterpart), and keys that no row sees are not read.
    ``stats``: an fp32 [rows, H, 2] that takes the rows' softmax statistics,
    for prefill_key_weights (a plan with a window is refused then)."""
    H, Hkv = plan.num_heads, plan.num_kv_heads
    if not query.is_cuda:
        raise ValueError("prefill_attention runs on the GPU; query is on the CPU")
    if query.dtype != torch.bfloat16 or k.dtype != query.dtype or v.dtype != query.dtype:
        raise ValueError("query, k and v must be bfloat16")
    _check_devices(query, plan, k=k, v=v, block_tables=block_tables)
    if query.dim() != 3 or tuple(query.shape[1:]) != (H, head_dim) or query.shape[0] < plan.rows:
        raise ValueError(f"query must be (at least {plan.rows}, {H}, {head_dim}), got {tuple(query.shape)}")
    max_blocks = 0
    if block_tables is None:
        if tuple(k.shape) != tuple(v.shape) or tuple(k.shape[1:]) != (Hkv, head_dim) or k.shape[0] < plan.keys:
            raise ValueError(f"k and v must be (at least {plan.keys}, {Hkv}, {head_dim}), got {tuple(k.shape)}")
        k, v = k.contiguous(), v.contiguous()
    else:
        nb, bs, hkv, d = _check_cache(k, "k_cache")
        if tuple(v.shape) != (nb, bs, hkv, d) or not v.is_contiguous():
            raise ValueError("k_cache and v_cache must have the same contiguous shape")
        if (bs, hkv, d) != (plan.block_size, Hkv, head_dim):
            raise ValueError("cache shape disagrees with block_size / num_kv_heads / head_dim")
        block_tables = _as(block_tables, "block_tables")
        if block_tables.shape[0] < plan.sequences:
            raise ValueError(f"{plan.sequences} sequences but {block_tables.shape[0]} block-table rows")
        max_blocks = block_tables.shape[1]
    query = query.contiguous()
    if (query.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
        query, k, v = _aligned(query), _aligned(k), _aligned(v)
    if stats is not None:
        if plan.window:
            raise ValueError("stats are of attention without a window")
        _check_stats(stats, plan.rows, H, query.device)
    out = torch.empty_like(query)
    # (the plan's list is the only memory that calls on several streams or
    # threads share, and they only read it)
    with _lib.on_device(query.device):
        stream = plan.use_here(query.device)
        part = torch.empty(plan.slots * H * plan.tile_rows * (head_dim + 2), dtype=torch.float32,
                           device=query.device) if plan.slots else None
        tiles = plan.work.data_ptr()
        rc = _lib.lib().nsv_prefill_window_attention(
            out.data_ptr(), query.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.ptr(block_tables), tiles, plan.ntiles,
            plan.tile_rows, tiles + plan.ntiles * 32, plan.nmerges, float(scale), H, Hkv, head_dim,
            plan.block_size or 1, max_blocks, plan.window, plan.sinks, _lib.ptr(stats), _lib.ptr(part), stream)
    _lib.check(rc, "prefill_attention")
    return out


def _check_devices(query: torch.Tensor, plan: _StepList, **others: torch.Tensor | None) -> None:
    dev = query.get_device()
    for name, t in (*others.items(), ("the plan", plan.work)):
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name} is on {t.device}, query on {query.device}")


def _check_stats(stats: torch.Tensor, rows: int, num_heads: int, device) -> None:
    if (stats.dim() != 3 or stats.shape[0] < rows or tuple(stats.shape[1:]) != (num_heads, 2)
            or stats.dtype != torch.float32 or stats.device != device or not stats.is_contiguous()):
        raise ValueError(f"stats must be a contiguous fp32 tensor of (at least {rows}, {num_heads}, 2) on {device}, got "
                         f"{stats.dtype} {tuple(stats.shape)} on {stats.device}")


def prefill_key_weights(query: torch.Tensor, k_cache: torch.Tensor, key_weights: torch.Tensor, plan: KeyWeightsPlan,
                        stats: torch.Tensor, scale: float, head_dim: int, block_tables: torch.Tensor) -> None:
    """Adds the attention weights of a prefill step's rows (bf16) to the paged
    ``key_weights`` (num_blocks, num_kv_heads, block_size) fp32: for every
    (key, kv head) the weights it gets from the rows at or behind it, summed
    over them and over the kv head's query heads.  ``query`` and ``scale`` are
    those of the step's prefill_attention call over the same paged K, which
    left ``stats``.  The places of the step's own keys are set, those of keys
    before its first row added to.  A page that several sequences of the step
    share (a prefix that one computes and another has behind it) gets the sum
    of theirs, in no fixed order.  No counterpart in the reference."""
    H, Hkv = plan.num_heads, plan.num_kv_heads
    if not query.is_cuda:
        raise ValueError("prefill_key_weights runs on the GPU; query is on the CPU")
    if query.dtype != torch.bfloat16 or k_cache.dtype != torch.bfloat16:
        raise ValueError("query and k_cache must be bfloat16")
    if query.dim() != 3 or tuple(query.shape[1:]) != (H, head_dim) or query.shape[0] < plan.rows:
        raise ValueError(f"query must be (at least {plan.rows}, {H}, {head_dim}), got {tuple(query.shape)}")
    if _check_cache(k_cache, "k_cache")[1:] != (plan.block_size, Hkv, head_dim):
        raise ValueError("cache shape disagrees with block_size / num_kv_heads / head_dim")
    _check_devices(query, plan, k_cache=k_cache, block_tables=block_tables)
    if k_cache.data_ptr() % 16:
        raise ValueError("k_cache must start on 16 bytes")
    _check_key_weights(key_weights, k_cache)
    _check_stats(stats, plan.rows, H, query.device)
    block_tables = _as(block_tables, "block_tables")
    if block_tables.dim() != 2 or block_tables.shape[0] < plan.sequences:
        raise ValueError(f"{plan.sequences} sequences but block tables of {tuple(block_tables.shape)}")
    if block_tables.shape[1] * plan.block_size < plan.longest:
        raise ValueError(f"block tables of {block_tables.shape[1]} pages for sequences of up to {plan.longest} keys")
    query = _aligned(query.contiguous())
    with _lib.on_device(query.device):
        stream = plan.use_here(query.device)
        part = torch.empty(plan.nunits * Hkv * 256, dtype=torch.float32, device=query.device)
        units = plan.work.data_ptr()
        rc = _lib.lib().nsv_prefill_key_weights(
            query.data_ptr(), k_cache.data_ptr(), key_weights.data_ptr(), stats.data_ptr(), block_tables.data_ptr(), units,
            plan.nunits, units + plan.nunits * 32, plan.nsums, float(scale), H, Hkv, head_dim, plan.block_size,
            block_tables.shape[1], part.data_ptr(), stream)
    _lib.check(rc, "prefill_key_weights")


def _evict_tables(block_tables: torch.Tensor, out_block_tables: torch.Tensor | None) -> tuple:
    """The two tables in the kernel's type, the second None where it is the
    first one itself (an eviction in place)."""
    tables = _as(block_tables, "block_tables")
    if out_block_tables is None or out_block_tables is block_tables:
        return tables, None
    out = _as(out_block_tables, "block_tables")
    return tables, None if out.data_ptr() == tables.data_ptr() and out.shape == tables.shape else out


def evict_kvcache(k_cache: torch.Tensor, v_cache: torch.Tensor, key_weights: torch.Tensor, block_tables: torch.Tensor,
                  context_lens: torch.Tensor, budget: int, *, sinks: int = 0, recent: int = 0,
                  out_block_tables: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cuts every sequence's cache to at most ``budget`` keys by the weights
    that paged_attention_weights and prefill_key_weights left.

    For each (sequence, kv head) with more keys than that, the first ``sinks``
    and the last ``recent`` stay, and of the rest those with the most weight
    (of equal ones the lower position; NaN counts as -inf).  Their rows of
    ``k_cache``, ``v_cache`` (num_blocks, block_size, Hkv, D; bfloat16 or
    float32) and ``key_weights`` (num_blocks, Hkv, block_size) move, in the
    order of their positions, to the first places of the sequence's table, or
    of its row of ``out_block_tables`` (which also gets the sequences that are
    short enough; pages of the old table that the new one does not hold keep
    what they hold, so it is the form for pages that other sequences share).
    Every page of the context must be mapped.  A sequence's new row may hold
    pages of its context at the same places (a copy of the table, its first
    columns), but none of a context's pages at another place or of another
    sequence.  What rows go to is rewritten: a prefix cache must not serve
    those pages by their old tokens.  In place, few sequences of many kept rows
    go by way of scratch as large as those rows of K and V.

    Returns (lens (B,) int64: min(length, budget); kept (B, Hkv, budget)
    int32: the positions that stay, ascending, -1 behind the last).  Keys hold
    their rotary embedding, so later queries keep their true positions for
    that, and use their places in the cache (lens, lens + 1, ..) as the
    ``positions`` and context lengths of the attention.  No counterpart in the
    reference."""
    if not k_cache.is_cuda:
        raise ValueError("evict_kvcache runs on the GPU; k_cache is on the CPU")
    nb, bs, hkv, d = _check_cache(k_cache, "k_cache")
    if v_cache.shape != k_cache.shape or not v_cache.is_contiguous() or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must have the same contiguous shape and dtype")
    _check_key_weights(key_weights, k_cache)
    dev, out_tables = k_cache.device, block_tables if out_block_tables is None else out_block_tables
    if not v_cache.device == context_lens.device == block_tables.device == out_tables.device == dev:
        raise ValueError(f"the caches, the block tables and context_lens must be on {dev}")
    if block_tables.dim() != 2 or out_tables.dim() != 2 or out_tables.shape[0] != block_tables.shape[0]:
        raise ValueError("block_tables and out_block_tables must be (B, pages)")
    B, max_blocks = block_tables.shape
    if tuple(context_lens.shape) != (B,):
        raise ValueError(f"context_lens must have {B} entries, got {tuple(context_lens.shape)}")
    budget, sinks, recent = _int_arg(budget, "budget", 1), _int_arg(sinks, "sinks", 0), _int_arg(recent, "recent", 0)
    if sinks + recent > budget:
        raise ValueError(f"{sinks} sinks and {recent} recent keys exceed the budget of {budget}")
    if out_block_tables is not None and out_block_tables.shape[1] * bs < min(budget, max_blocks * bs):
        raise ValueError(f"out_block_tables of {out_block_tables.shape[1]} pages do not hold {budget} keys")
    if nb * bs > 0x7fffffff:
        raise ValueError(f"evict_kvcache addresses fewer than 2^31 cached keys, got {nb} pages of {bs}")
    block_tables, out_block_tables = _evict_tables(block_tables, out_block_tables)
    context_lens = _as(context_lens, "context_lens")
    lens = torch.empty(B, dtype=torch.int64, device=dev)
    kept = torch.empty((B, hkv, budget), dtype=torch.int32, device=dev)
    code = _lib.dtype_code(k_cache.dtype)
    with _lib.on_device(dev):
        stream = _lib.stream_ptr(dev)
        ws_bytes = _evict_workspace_bytes(B, hkv, d, bs, max_blocks, int(out_block_tables is not None), code, budget)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None  # (too large to keep)
        rc = _lib.lib().nsv_evict_kv(
            k_cache.data_ptr(), v_cache.data_ptr(), key_weights.data_ptr(), block_tables.data_ptr(),
            context_lens.data_ptr(), _lib.ptr(out_block_tables), lens.data_ptr(), kept.data_ptr(), B, hkv, d, bs,
            max_blocks, 0 if out_block_tables is None else out_block_tables.shape[1], code, budget, sinks, recent,
            _lib.ptr(ws), ws_bytes, stream)
    _lib.check(rc, "evict_kvcache")
    return lens, kept


_prefill_plan: tuple = (None, None)  # (the Context it was built for, its tensors)


def _prefill_rows(ctx, num_heads: int, num_kv_heads: int, device) -> tuple:
    """Verify-kernel metadata of an fp32 prefill step, built once per Context.

    Sequence i has seqlens_q[i] new rows at positions seqlens_k[i] -
    seqlens_q[i] .. seqlens_k[i] - 1.  Its rows are cut into causal blocks of
    q_block = 64 // G rows (G query heads per kv head: the kernel holds up to
    64 query rows per (sequence, kv head)); each block is one entry of the
    kernel's batch with context = the block's last position + 1, so every
    row attends exactly keys 0 .. its position.  Block-table row of block j:
    the sequence's row of context.block_tables (paged prefill) or, without
    block tables, the sequence's keys in the step's own contiguous K/V read
    as one-token pages (cu_seqlens_k[i] + p for position p).
    Returns (block_tables, context_lens, cu_seqlens_q, positions, q_block)."""
    import numpy as np

    global _prefill_plan
    if _prefill_plan[0] is ctx:
        return _prefill_plan[1]
    if ctx.seqlens_q is None or ctx.seqlens_k is None:
        raise ValueError("a prefill step needs context.seqlens_q and context.seqlens_k")
    q_block = max(1, 64 // (num_heads // num_kv_heads))
    paged = ctx.block_tables is not None
    tables = ctx.block_tables.cpu().numpy() if paged else None
    width = tables.shape[1] if paged else max(ctx.seqlens_k)
    bt, lens, cu, pos = [], [], [0], []
    k_start = 0
    for i, (ql, kl) in enumerate(zip(ctx.seqlens_q, ctx.seqlens_k)):
        if not 0 < ql <= kl:
            raise ValueError(f"prefill sequence {i}: {ql} query rows over {kl} keys")
        if paged:
            row = tables[i].astype(np.int32)
        else:
            row = np.full(width, -1, dtype=np.int32)
            row[:kl] = np.arange(k_start, k_start + kl, dtype=np.int32)
        for b0 in range(kl - ql, kl, q_block):
            b1 = min(kl, b0 + q_block)
            bt.append(row)
            lens.append(b1)
            cu.append(cu[-1] + (b1 - b0))
        pos.append(np.arange(kl - ql, kl, dtype=np.int64))
        k_start += kl
    t = lambda x, dt: torch.from_numpy(np.ascontiguousarray(x, dtype=dt)).to(device)  # noqa: E731
    out = (t(np.stack(bt), np.int32), t(lens, np.int64), t(cu, np.int32), t(np.concatenate(pos), np.int64), q_block)
    _prefill_plan = (ctx, out)
    return out


class Attention(nn.Module):
    """Attention layer of the reference (layers/attention.py:670-767):
    writes this step's K/V into the paged cache at context.slot_mapping,
    then attends from the query rows the global Context describes:
      * verify (context.is_verify): a chunk of drafted tokens per sequence
        with a causal mask from absolute positions (:704-731);
      * prefill (context.is_prefill, :733-757): every new prompt row of each
        sequence, causally over its keys.  With context.block_tables (a
        prompt behind a cached prefix) the keys come from the paged cache,
        the step's own K/V already stored in it, as the reference's
        paged_attention_prefill (:328-363); without, from the step's
        contiguous K/V, as its varlen flash path (:257-325).  bf16 runs on
        the prefill kernel (``prefill_attention``), paged steps of a few rows
        per sequence on the verify kernel (``verify_serves_prefill``), fp32 on
        the verify kernel over causal blocks of rows (``_prefill_rows``);
      * decode (neither flag): one query row per sequence attending its
        whole context (:759-767), served by the same verify kernel with
        each row at position context_lens - 1.

    A layer over a bounded cache (no reference counterpart):
      * ``window`` > 0: every row sees its last ``window`` keys and its
        sequence's first ``sinks`` only, in all three kinds of steps;
      * ``key_weights`` set to an fp32 (num_blocks, num_kv_heads, block_size)
        table beside the caches: every step adds its rows' attention weights
        to their keys' places (a prefill step needs block tables then), for
        evict_kvcache to cut the cache by."""

    def __init__(self, num_heads: int, head_dim: int, scale: float = 1.0, num_kv_heads: int | None = None,
                 block_size: int = 16, window: int = 0, sinks: int = 0):
        super().__init__()
        self.window, self.sinks = _int_arg(window, "window", 0), _int_arg(sinks, "sinks", 0)
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads if num_kv_heads is not None else num_heads
        self.block_size = block_size
        self.k_cache = self.v_cache = torch.tensor([])
        self.key_weights: torch.Tensor | None = None

    def _few(self, q, tables, context_lens, cu_seqlens_q, positions, scale: float, max_q_len: int,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """A few rows per sequence over the paged cache: with the layer's
        window, with its key weights, or as the verify round does."""
        shape = (tables, context_lens, cu_seqlens_q, positions, scale, self.num_heads, self.num_kv_heads, self.head_dim,
                 self.block_size, max(16, 1 << (max_q_len - 1).bit_length()))
        if self.window:
            return paged_attention_window(q, self.k_cache, self.v_cache, *shape, window=self.window, sinks=self.sinks,
                                          max_q_len=max_q_len, out=out)
        if self.key_weights is not None:
            return paged_attention_weights(q, self.k_cache, self.v_cache, self.key_weights, *shape, max_q_len=max_q_len,
                                           out=out)
        return paged_attention_verify(q, self.k_cache, self.v_cache, *shape, max_q_len=max_q_len, out=out)

    def _prefill_f32_weights(self, context, q, scale: float) -> torch.Tensor:
        """An fp32 prefill step with key weights: causal blocks of rows in
        several calls (_WeightTurns, built by the step's first layer)."""
        if context.seqlens_q is None or context.seqlens_k is None:
            raise ValueError("a prefill step needs context.seqlens_q and context.seqlens_k")
        q_block = max(1, 64 // (self.num_heads // self.num_kv_heads))
        plans, key = context.__dict__.setdefault("prefill_plans", {}), ("turns", q_block, q.device)
        plan = plans.get(key)
        if plan is None:
            plan = plans[key] = _WeightTurns(context.seqlens_q, context.seqlens_k, context.block_tables, q_block, q.device)
        if q.shape[0] < plan.rows:
            raise ValueError(f"query must have at least {plan.rows} rows, got {q.shape[0]}")
        plan.use_on(torch.cuda.current_stream(q.device))
        out = torch.empty_like(q, memory_format=torch.contiguous_format)  # (rows past the step's: unwritten)
        for rows, *meta in plan.turns:
            if isinstance(rows, tuple):
                at = slice(*rows)
                self._few(q[at], *meta, scale, q_block, out[at])
            else:
                out.index_copy_(0, rows, self._few(q.index_select(0, rows), *meta, scale, q_block))
        return out

    def _prefill_bf16(self, context, q, k, v, scale: float) -> torch.Tensor:
        """The prefill branch on the prefill kernel, or on the verify kernel
        for a few rows per sequence; the step's work list is built by its
        first layer and kept with the step's Context."""
        paged = context.block_tables is not None
        if context.seqlens_q is None or context.seqlens_k is None:
            raise ValueError("a prefill step needs context.seqlens_q and context.seqlens_k")
        bs = self.block_size if paged else None
        key = (self.num_heads, self.num_kv_heads, bs, q.device)
        plans = context.__dict__.setdefault("prefill_plans", {})
        if self.window or self.key_weights is not None:
            few = paged and few_rows_serve_prefill(context.seqlens_q, self.num_heads, self.num_kv_heads)
        else:
            few = paged and verify_serves_prefill(context.seqlens_q, context.seqlens_k, self.num_heads, self.num_kv_heads,
                                                  bs, context.block_tables.shape[1])
        if few:
            return self._prefill_few(context, plans, q, scale)
        if self.window:
            key += (self.window, self.sinks)
        plan = plans.get(key)
        if plan is None:
            plan = plans[key] = PrefillPlan(context.seqlens_q, context.seqlens_k, self.num_heads, self.num_kv_heads,
                                            bs, q.device, self.window, self.sinks)
        if paged and self.key_weights is not None:
            adder = plans.get((*key, "weights"))
            if adder is None:
                adder = plans[(*key, "weights")] = KeyWeightsPlan(context.seqlens_q, context.seqlens_k, self.num_heads,
                                                                  self.num_kv_heads, bs, q.device)
            tables = context.block_tables.to(q.device)
            stats = torch.empty((plan.rows, self.num_heads, 2), dtype=torch.float32, device=q.device)
            out = prefill_attention(q, self.k_cache, self.v_cache, plan, scale, self.head_dim, tables, stats=stats)
            prefill_key_weights(q, self.k_cache, self.key_weights, adder, stats, scale, self.head_dim, tables)
            return out
        if paged:
            return prefill_attention(q, self.k_cache, self.v_cache, plan, scale, self.head_dim,
                                     context.block_tables.to(q.device))
        return prefill_attention(q, k.reshape(-1, self.num_kv_heads, self.head_dim),
                                 v.reshape(-1, self.num_kv_heads, self.head_dim), plan, scale, self.head_dim)

    def _prefill_few(self, context, plans: dict, q, scale: float) -> torch.Tensor:
        """A paged prefill step of a few rows per sequence as one verify call."""
        rows = plans.get(q.device)
        if rows is None:
            rows = plans[q.device] = PrefillRows(context.seqlens_q, context.seqlens_k, q.device)
        if q.shape[0] < rows.rows:
            raise ValueError(f"query must have at least {rows.rows} rows, got {q.shape[0]}")
        tables = context.block_tables.to(q.device)
        if tables.shape[0] < rows.sequences:
            raise ValueError(f"{rows.sequences} sequences but {tables.shape[0]} block-table rows")
        rows.use_on(torch.cuda.current_stream(q.device))
        if self.window or self.key_weights is not None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)  # (rows past the step's: unwritten)
            self._few(q[:rows.rows], tables[:rows.sequences], rows.context_lens, rows.cu_seqlens_q, rows.positions, scale,
                      rows.max_q_len, out[:rows.rows])
            return out
        return paged_attention_verify(
            q, self.k_cache, self.v_cache, tables[:rows.sequences], rows.context_lens, rows.cu_seqlens_q, rows.positions,
            scale, self.num_heads, self.num_kv_heads, self.head_dim, self.block_size, 64, max_q_len=rows.max_q_len,
            tile_references=True)

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        context = get_context()
        k_cache, v_cache = self.k_cache, self.v_cache
        if self.key_weights is not None:
            if self.window:
                raise ValueError("a layer has a window or key weights, not both")
            if context.block_tables is None:
                raise ValueError("a layer with key weights needs context.block_tables: the weights are paged")
        if k_cache.numel() > 0 and v_cache.numel() > 0 and context.slot_mapping is not None:
            store_kvcache(k.reshape(-1, self.num_kv_heads, self.head_dim),
                          v.reshape(-1, self.num_kv_heads, self.head_dim),
                          k_cache, v_cache, context.slot_mapping, self.block_size)
        scale = self.scale / (self.head_dim ** 0.5)
        q = q.reshape(-1, self.num_heads, self.head_dim)
        if context.is_prefill and not context.is_verify:
            if context.cu_seqlens_q is None:
                raise ValueError("cu_seqlens_q must be provided for varlen attention")
            if q.dtype == torch.bfloat16:
                o = self._prefill_bf16(context, q, k, v, scale)
                return o.reshape(o.shape[0], self.num_heads * self.head_dim)
            if self.key_weights is not None:
                o = self._prefill_f32_weights(context, q, scale)
                return o.reshape(o.shape[0], self.num_heads * self.head_dim)
            bt, lens, cu, positions, q_block = _prefill_rows(context, self.num_heads, self.num_kv_heads, q.device)
            if context.block_tables is not None:
                kc, vc, bs = k_cache, v_cache, self.block_size
            else:  # the step's own keys, one token per page
                kc = k.reshape(-1, 1, self.num_kv_heads, self.head_dim).contiguous()
                vc = v.reshape(-1, 1, self.num_kv_heads, self.head_dim).contiguous()
                bs = 1
            shape = (bt, lens, cu, positions, scale, self.num_heads, self.num_kv_heads, self.head_dim, bs, max(16, q_block))
            if self.window:
                rows, o = positions.numel(), torch.empty_like(q, memory_format=torch.contiguous_format)
                paged_attention_window(q[:rows], kc, vc, *shape, window=self.window, sinks=self.sinks, max_q_len=q_block,
                                       out=o[:rows])
            else:
                o = paged_attention_verify(q, kc, vc, *shape, max_q_len=q_block)
            return o.reshape(o.shape[0], self.num_heads * self.head_dim)
        if context.is_verify:
            max_q_len = max(context.seqlens_q)
            cu, positions = context.cu_seqlens_q, context.positions
        else:
            # decode: row b is the newest token of sequence b
            max_q_len = 1
            cu = torch.arange(0, q.shape[0] + 1, dtype=torch.int32, device=q.device)
            positions = context.context_lens.to(torch.int64) - 1
        o = self._few(q, context.block_tables, context.context_lens, cu, positions, scale, max_q_len)
        return o.reshape(o.shape[0], self.num_heads * self.head_dim)
