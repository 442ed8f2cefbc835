"""Pages of a paged `SparseMLACache`: handing out, giving back, branching and compacting.

The reference copies the whole state of a conversation to branch it (oracle/v4_fast.py:150-159
clone_states). Here a branch shares the full pages of compressed rows and copies only what its tokens
will write to (the last partial page, the window ring, the compressor rings) and the indexer keys,
which are laid out by slot. Tables and counts stay on the device: every call is asynchronous on the
current stream, can be captured in a CUDA graph, and gives the same tables for the same input. What a
call cannot do for one sequence it leaves out for that sequence, and raises the device error word
(`_lib.device_error`): NO_PAGES, or INDEX_OUT_OF_RANGE for a slot that does not exist, a branch of more
tokens than the cache or its source's pages hold, or a branch onto a slot that has pages. A window-only cache (no compressed rows)
has no pages: it is branched by a copy of the window ring, and the other calls leave it as it is.
"""
import ctypes

import torch

from . import _lib as L


def _params(cache):
    if not cache.compressed:   # window rings alone: nothing is paged, a branch is a copy of its ring
        L.require_cuda(cache.kv_pool)
        p = L.Pages(pool=cache.kv_pool.data_ptr(), win_base=cache.win_base.data_ptr(), comp_base=cache.comp_base)
        p.slots, p.page, p.window, p.head_dim, p.ratio = cache.batch, 1, cache.window, cache.head_dim, 1
        return p
    if cache.page_refs is None:
        raise ValueError("SparseMLACache: pages are handed out and shared only in a paged cache (n_pages=...)")
    L.require_cuda(cache.kv_pool)
    img, inv, nmax = cache.key_image
    k, table = cache.k_idx, cache.block_table
    return L.Pages(cache.kv_pool.data_ptr(), cache.win_base.data_ptr(), table.data_ptr(), cache.page_refs.data_ptr(),
                   k.data_ptr(), img.data_ptr(), inv.data_ptr(), nmax.data_ptr(), cache.ring_kv.data_ptr(),
                   cache.ring_score.data_ptr(), cache.ring_k_idx.data_ptr(), cache.ring_s_idx.data_ptr(), cache.comp_base,
                   cache.batch, cache.page_refs.numel(), table.shape[1], cache.page, cache.max_comp, cache.window,
                   cache.head_dim, k.shape[2], cache.ratio)


def _ints(name, cache, *ts):
    """Sequences and token counts (lists, or tensors on the cache's device) as int32 tensors of one length."""
    dev, index, out = cache.block_table.device, cache.block_table.get_device(), []
    n = None
    for t in ts:
        if not isinstance(t, torch.Tensor):
            t = torch.tensor(t, dtype=torch.int32, device=dev)
        elif t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
            if t.dtype not in (torch.int32, torch.int64):
                L.require_cuda(t)
                raise TypeError(f"{name}: sequences and token counts are integers, got {t.dtype}")
            t = t.reshape(-1).to(torch.int32).contiguous()
        if t.get_device() != index:
            L.require_cuda(t)
            raise ValueError(f"{name}: tensors on {t.device}, the cache is on {dev}")
        if n is None:
            n = t.numel()
        elif t.numel() != n:
            raise ValueError(f"{name}: {n} sequences, {t.numel()} of their counts")
        out.append(t)
    return out


def _workspace(p, n, device):
    nbytes = L.lib().dsv4_pages_workspace_size(ctypes.byref(p), n)
    return torch.empty(nbytes, dtype=torch.uint8, device=device), nbytes


def pages_free(cache, seqs):
    """Give back the pages of slots `seqs` (a page shared with another slot stays with that one) and
    empty their table rows. A slot named twice gives its pages back once. The slot's next sequence begins at
    position 0: nothing else of the last one is read from there (window rows and entries are seen by position,
    and the first block has none before it)."""
    p = _params(cache)
    seqs, = _ints("pages_free", cache, seqs)
    with L.device_of(seqs):
        L.check(L.lib().dsv4_pages_free(ctypes.byref(p), seqs.data_ptr(), seqs.numel(), L.stream_of(seqs)))


def pages_reserve(cache, seqs, tokens, add=0):
    """Pages for the compressed rows of `tokens + add` tokens of slots `seqs` (None: slot k for the
    k-th count); pages they have stay. A slot that finds too few free pages gets none, and those behind it
    are served from what it leaves; one named twice gets the pages of the larger count. A count past the
    cache gets all the pages that the slot has entries for, and raises INDEX_OUT_OF_RANGE; one below 0 is none."""
    p = _params(cache)
    if seqs is None:
        tokens, = _ints("pages_reserve", cache, tokens)
        if tokens.numel() > cache.batch:
            raise ValueError(f"pages_reserve: {tokens.numel()} counts, the cache has {cache.batch} slots")
    else:
        seqs, tokens = _ints("pages_reserve", cache, seqs, tokens)
    with L.device_of(tokens):
        ws, nbytes = _workspace(p, tokens.numel(), tokens.device)
        L.check(L.lib().dsv4_pages_reserve(ctypes.byref(p), None if seqs is None else seqs.data_ptr(), tokens.data_ptr(),
                                           int(add), tokens.numel(), ws.data_ptr(), nbytes, L.stream_of(tokens)))


def pages_fork(cache, src, dst, tokens):
    """Make slot dst[k], which has no pages, a branch of slot src[k], which holds tokens[k] tokens (all
    that it holds: the window ring and the compressor rings are those of its latest token). A slot may
    be the source of several branches, but not a branch twice, nor a branch and a source."""
    p = _params(cache)
    if cache.image_stale:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("pages_fork: the cache's key image is stale inside a stream capture; call "
                               "cache.refresh_key_image() before capturing")
        cache.refresh_key_image()
    src, dst, tokens = _ints("pages_fork", cache, src, dst, tokens)
    if src.numel() > cache.batch:
        raise ValueError(f"pages_fork: {src.numel()} branches, the cache has {cache.batch} slots")
    with L.device_of(src):
        ws, nbytes = _workspace(p, src.numel(), src.device)
        L.check(L.lib().dsv4_pages_fork(ctypes.byref(p), src.data_ptr(), dst.data_ptr(), tokens.data_ptr(), src.numel(),
                                        ws.data_ptr(),
                                        nbytes, L.stream_of(src)))


def pages_compact(cache):
    """Move the pages in use to the front of the pool, the first free page taking the first page in use
    behind the new end, and so on; tables and counts follow. Returns their number, int32 [1] on the
    device. Page numbers that a caller keeps beside the table are no longer valid."""
    p = _params(cache)
    n = torch.empty(1, dtype=torch.int32, device=cache.block_table.device)
    with L.device_of(n):
        ws, nbytes = _workspace(p, 0, n.device)
        L.check(L.lib().dsv4_pages_compact(ctypes.byref(p), n.data_ptr(), ws.data_ptr(), nbytes, L.stream_of(n)))
    return n
