"""A chunk of new tokens per sequence over the device-resident state (`SparseMLACache`).

The reference extends its state one token at a time (oracle/v4_fast.py:82-122) or builds it from
position 0 (oracle/v4_prefill.py). These ops take the step between: several new tokens of each
sequence on top of what the cache holds, for a prompt taken in chunks, a further turn of a
conversation, or drafted tokens that are checked at once. The order of a layer's chunk is

  positions, rows = chunk_rows(cache, cu_seqlens, start, total)   where the tokens are
  norm_rope into the pool at `rows`                               their kv rows, staged
  compressor_chunk(...)                                           the compressed rows they complete
  o = chunk_attention(cache, q, sink, cu_seqlens, start)          window + compressed rows of each token
  chunk_commit(cache, cu_seqlens, start, total)                   the staged rows into the window rings

`DecodeBlock.extend` runs it. Sequence b has the tokens [cu_seqlens[b], cu_seqlens[b+1]) of the batch,
the first of them at position start[b] of cache slot seqs[b] (default b). Rows of the batch behind
cu_seqlens[-1] belong to no sequence (a padded batch).
"""
import ctypes

import torch

from . import _lib as L
from .norm_rope import rope_freqs


def _index_tensor(name, t, pool, n):
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or (t.dtype != torch.int32 and t.dtype != torch.int64):
        raise TypeError(f"{name} must be a 1-d int32 tensor")
    if t.get_device() != pool.get_device():
        L.require_cuda(t)
        raise ValueError(f"{name} is on {t.device}, the cache on {pool.device}")
    if n is not None and t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} values, the chunk has {n} sequences")
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _f32(t):
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def _sequences(cache, cu_seqlens, start, seqs, total):
    """The chunk's sequences as int32 tensors, checked against the cache."""
    pool = cache.kv_pool
    cu = _index_tensor("cu_seqlens", cu_seqlens, pool, None)
    n = cu.numel() - 1
    if n < 0:
        raise ValueError("cu_seqlens holds one value more than there are sequences")
    start = _index_tensor("start", start, pool, n)
    if seqs is not None:
        seqs = _index_tensor("seqs", seqs, pool, n)
    elif n > cache.batch:
        raise ValueError(f"a chunk of {n} sequences, the cache has {cache.batch} slots")
    if total > cache.max_chunk:
        raise ValueError(f"a chunk of {total} tokens, the cache stages {cache.max_chunk} (SparseMLACache(max_chunk=...))")
    return cu, start, seqs


def _chunk(cache, cu_seqlens, start, seqs, total):
    """dsv4_chunk of the cache, and the tensors it points to."""
    cu, start, seqs = _sequences(cache, cu_seqlens, start, seqs, total)
    c = _layout(cache.kv_pool, cache.block_table, cache.win_base, cu, start, seqs, total, cache.comp_base, cache.stage_base,
                cache.window, cache.ratio, cache.page, cache.max_comp)
    return c, (cu, start, seqs)


def _layout(pool, table, win_base, cu, start, seqs, total, comp_base, stage_base, window, ratio, page, max_comp):
    return L.Chunk(cu.data_ptr(), start.data_ptr(), None if seqs is None else seqs.data_ptr(), win_base.data_ptr(),
                   table.data_ptr() if max_comp else None, comp_base, stage_base, pool.shape[0], cu.numel() - 1, total,
                   win_base.numel(), window, ratio, page, table.shape[1], max_comp)


def chunk_rows(cache, cu_seqlens, start, total, seqs=None):
    """(positions int32 [total], rows int64 [total]): the position of each token of the chunk and the
    pool row where its kv row is staged. Positions behind the last sequence are 0."""
    c, keep = _chunk(cache, cu_seqlens, start, seqs, total)
    dev = cache.kv_pool.device
    positions = torch.zeros(total, dtype=torch.int32, device=dev) if c.n == 0 else \
        torch.empty(total, dtype=torch.int32, device=dev)
    rows = torch.empty(total, dtype=torch.int64, device=dev)
    with L.device_of(positions):
        if c.n == 0:
            return positions, torch.arange(cache.stage_base, cache.stage_base + total, device=dev)
        L.check(L.lib().dsv4_chunk_rows(ctypes.byref(c), L.ptr(positions), L.ptr(rows), None, 0, 0, None,
                                        L.stream_of(positions)))
    return positions, rows


def chunk_commit(cache, cu_seqlens, start, total, seqs=None):
    """Move the chunk's rows into the window rings (the last `window` of each sequence), after its
    attention: what the decode steps and the next chunk see. A slot takes one sequence of a call: the second
    one that names it is left out and raises INDEX_OUT_OF_RANGE on the device error word."""
    c, keep = _chunk(cache, cu_seqlens, start, seqs, total)
    with L.device_of(cache.kv_pool):
        L.check(L.lib().dsv4_chunk_commit(ctypes.byref(c), L.ptr(cache.kv_pool), cache.head_dim,
                                          L.stream_of(cache.kv_pool)))


@torch.library.custom_op("dsv4::chunk_attention", mutates_args=(), device_types="cuda")
def _chunk_attention_op(q: torch.Tensor, kv_pool: torch.Tensor, block_table: torch.Tensor, win_base: torch.Tensor,
                        sink: torch.Tensor, cu_seqlens: torch.Tensor, start: torch.Tensor, seqs: torch.Tensor | None,
                        rows: torch.Tensor | None, freqs: torch.Tensor, comp_base: int, stage_base: int, window: int,
                        ratio: int, page: int, max_comp: int, scale: float, out_dtype: torch.dtype,
                        num_splits: int) -> torch.Tensor:
    _check_rows(q, kv_pool)
    return _attention(q, kv_pool, block_table, win_base, sink, cu_seqlens, start, seqs, rows, freqs, comp_base, stage_base,
                      window, ratio, page, max_comp, scale, out_dtype, num_splits)


@_chunk_attention_op.register_fake
def _(q, kv_pool, block_table, win_base, sink, cu_seqlens, start, seqs, rows, freqs, comp_base, stage_base, window, ratio,
      page, max_comp, scale, out_dtype, num_splits):
    _check_rows(q, kv_pool)
    return torch.empty_like(q, dtype=out_dtype, memory_format=torch.contiguous_format)


def _check_rows(q, kv_pool):
    """What the custom op, called by itself, has to hold: the kernels' tiles take 64 heads of 512 bf16 whatever the
    tensors are (`chunk_attention` checks it with the rest)."""
    if q.dim() != 3 or q.shape[1] != 64 or q.shape[2] != 512 or kv_pool.dim() != 2 or kv_pool.shape[1] != 512:
        raise ValueError(f"dsv4::chunk_attention: q [total, 64, 512] over rows of 512, got {tuple(q.shape)} and {tuple(kv_pool.shape)}")
    if q.dtype != torch.bfloat16 or kv_pool.dtype != torch.bfloat16:
        raise TypeError(f"dsv4::chunk_attention: q and the pool are bf16, got {q.dtype} and {kv_pool.dtype}")


def _attention(q, kv_pool, block_table, win_base, sink, cu_seqlens, start, seqs, rows, freqs, comp_base, stage_base, window,
               ratio, page, max_comp, scale, out_dtype, num_splits):
    c = _layout(kv_pool, block_table, win_base, cu_seqlens, start, seqs, q.shape[0], comp_base, stage_base, window, ratio,
                page, max_comp)
    with L.device_of(q):
        # lists differ from token to token, and pages that no box of rows divides have no run to load: those
        # go through an index, token by token
        if rows is None and (page % 8 == 0 or not max_comp) and window <= 1024:
            return _attend(kv_pool, c, q, sink, scale, freqs, out_dtype, num_splits)
        return _attend_listed(kv_pool, c, q, sink, rows, scale, freqs, out_dtype)


def _attend(kv_pool, c, q, sink, scale, freqs, out_dtype, num_splits):
    """All visible rows: dsv4_chunk_attn, which finds them by itself."""
    out = torch.empty_like(q, dtype=out_dtype)
    p = L.ChunkAttnParams(c, q.data_ptr(), kv_pool.data_ptr(), sink.data_ptr(), out.data_ptr(), freqs.data_ptr(),
                          2 * freqs.numel(), L.dtype_code(out), scale, num_splits)
    lib, ref = L.lib(), ctypes.byref(p)
    nbytes = lib.dsv4_chunk_attn_workspace_size(ref)
    if nbytes:
        ws = L.workspace(nbytes, q.device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    L.check(lib.dsv4_chunk_attn(ref, L.stream_of(q)))
    return out


def _attend_listed(kv_pool, c, q, sink, rows, scale, freqs, out_dtype):
    """Every token's list and position (one allocation), and the sparse attention over them."""
    lib, stream = L.lib(), L.stream_of(q)
    total, heads, dim = q.shape
    cols = c.max_comp if rows is None else rows.shape[1]
    t = c.window + cols
    lists = torch.empty(total * (t + 1), dtype=torch.int32, device=q.device)
    idx = lists.data_ptr()
    pos = idx + 4 * total * t
    L.check(lib.dsv4_chunk_rows(ctypes.byref(c), pos, None, idx, t, cols, None if rows is None else rows.data_ptr(), stream))
    out = torch.empty_like(q, dtype=out_dtype)
    p = L.SparseAttnParams(q.data_ptr(), kv_pool.data_ptr(), sink.data_ptr(), idx, out.data_ptr(), total, c.pool_rows, heads,
                           dim, t, L.BF16, L.I32, L.dtype_code(out), scale, freqs.data_ptr(), pos, 2 * freqs.numel())
    ref = ctypes.byref(p)
    nbytes = lib.dsv4_sparse_attn_workspace_size(ref)
    if nbytes:
        ws = L.workspace(nbytes, q.device)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    L.check(lib.dsv4_sparse_attn(ref, stream))
    return out


def chunk_attention(cache, q, sink, cu_seqlens, start, seqs=None, rows=None, scale=None, freqs=None,
                    out_dtype=torch.bfloat16, num_splits=0):
    """Attention of a chunk of new tokens over the cache, their kv rows staged (`chunk_rows`) and their
    compressed rows written (`compressor_chunk`).

    q [total, 64, 512] bf16 after the per-head norm and RoPE (`norm_rope`), sink [64]. The token at
    position p sees the window rows of positions p-window+1 .. p, from the ring before the chunk and from
    the stage in it, and every compressed entry j < (p+1) // ratio (the list of
    oracle/decode_engine.py:110-116), or with `rows` (int32 [total, k] pool rows, -1 for none: the
    indexer's selection) those instead. `num_splits`: over how many CTA pairs the rows of two tokens are split
    (0: automatic; all visible rows only). Returns o [total, 64, 512] after the inverse RoPE; what it holds
    behind the last sequence, and for a sequence that the error word reports (a slot that does not exist, tokens
    outside of q), is not defined. A row that is not finite reaches the tokens that see it and no others (a
    head that scores it -inf weighs it 0 and may leave it out). The custom op `dsv4::chunk_attention`."""
    index = cache.kv_pool.get_device()
    if not L.one_device(index, (q, sink, rows, freqs)):
        L.require_cuda(q, sink, rows, freqs)
        raise ValueError("chunk_attention: q, sink, rows and freqs must be on the cache's device")
    shape = q.shape
    if len(shape) != 3 or shape[2] != 512 or cache.head_dim != 512:
        raise ValueError(f"chunk_attention: q must be [total, 64, 512] over a cache of 512-wide rows, got {tuple(q.shape)} and "
                         f"head_dim {cache.head_dim}")
    if q.dtype != torch.bfloat16:
        raise TypeError(f"chunk_attention: q is the bf16 output of norm_rope, got {q.dtype}")
    if shape[1] != 64 or sink.numel() != 64:
        raise ValueError(f"chunk_attention: 64 heads, got q {tuple(q.shape)} and {sink.numel()} sinks")
    if out_dtype != torch.bfloat16 and out_dtype != torch.float32:
        raise TypeError(f"chunk_attention: out_dtype must be bfloat16 or float32, got {out_dtype}")
    total = shape[0]
    if rows is not None:
        if rows.dim() != 2 or rows.shape[0] != total or rows.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"chunk_attention: rows must be int32 [{total}, k], got {rows.dtype} {tuple(rows.shape)}")
        rows = rows.to(torch.int32).contiguous()
    freqs = rope_freqs(64, q.device) if freqs is None else _f32(freqs)
    if not 0 < freqs.numel() <= 32:
        raise ValueError(f"chunk_attention: 1 to 32 rotation frequencies, got {freqs.numel()}")
    if not 0 <= num_splits <= 64:
        raise ValueError(f"chunk_attention: 0 to 64 splits, got {num_splits}")
    scale = cache.head_dim ** -0.5 if scale is None else float(scale)
    cu, start, seqs = _sequences(cache, cu_seqlens, start, seqs, total)
    if total == 0 or cu.numel() == 1:
        return torch.empty(q.shape, dtype=out_dtype, device=q.device)
    # traced programs see the custom op; an eager call goes straight to its body
    f = _chunk_attention_op if L.through_op(q, cache.kv_pool, sink, cu) else _attention
    return f(q.contiguous(), cache.kv_pool, cache.block_table, cache.win_base, _f32(sink), cu, start, seqs, rows, freqs,
             cache.comp_base, cache.stage_base, cache.window, cache.ratio, cache.page, cache.max_comp, scale, out_dtype,
             int(num_splits))
