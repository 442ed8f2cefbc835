"""The structs of the chunk and page entry points match include/dsv4.h field for field, and the entry
points' checks of arguments, which need no GPU."""
import ctypes
import importlib
import os
import shutil
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = "deepseek-v4-flash-mlx_b200"
L = importlib.import_module(PKG + "._lib")
PAIRS = {"dsv4_chunk": L.Chunk, "dsv4_chunk_attn_params": L.ChunkAttnParams,
         "dsv4_compressor_chunk_params": L.CompressorChunkParams, "dsv4_pages": L.Pages}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a host C compiler")
def test_struct_layouts_match_header():
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "dsv4.h"', "int main(void) {"]
    for cname, py in PAIRS.items():
        lines.append(f'  printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f[0]} %zu\\n", offsetof({cname}, {f[0]}));' for f in py._fields_]
    lines.append("  return 0;\n}")
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        open(src, "w").write("\n".join(lines))
        subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split("\n")
    got = {tuple(ln.split()[:2]): int(ln.split()[2]) for ln in out if ln}
    for cname, py in PAIRS.items():
        assert got[(cname, "sizeof")] == ctypes.sizeof(py), cname
        for f in py._fields_:
            assert got[(cname, f[0])] == getattr(py, f[0]).offset, (cname, f[0])


def _chunk(**kw):
    c = L.Chunk()
    one = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(one) + 15) // 16 * 16
    for name in ("cu_seqlens", "start", "win_base", "block_table"):
        setattr(c, name, at)
    c.comp_base, c.stage_base, c.pool_rows = 128, 128 + 64, 128 + 64 + 8
    c.n, c.total, c.slots, c.window, c.ratio, c.page, c.bt_stride, c.max_comp = 1, 8, 1, 128, 4, 64, 1, 64
    for k, v in kw.items():
        setattr(c, k, v)
    c._keep = one
    return c


@pytest.mark.parametrize("bad", [dict(window=100), dict(pool_rows=199), dict(max_comp=65), dict(cu_seqlens=None),
                                 dict(block_table=None), dict(n=2), dict(total=-1), dict(stage_base=100), dict(ratio=0),
                                 dict(pool_rows=1 << 31)])
def test_chunk_refusals_of_the_c_entry(bad):
    """Each is refused on the host, before any launch."""
    c = _chunk(**bad)
    at = c.start
    assert L.lib().dsv4_chunk_rows(ctypes.byref(c), at, at, None, 0, 0, None, None) == 1
    assert L.lib().dsv4_chunk_commit(ctypes.byref(c), at, 512, None) == 1
    assert L.lib().dsv4_last_error()


def test_chunk_list_refusals_of_the_c_entry():
    c = _chunk()
    at = c.start
    assert L.lib().dsv4_chunk_rows(ctypes.byref(c), at, at, at, 128 + 3, 4, None, None) == 1   # row shorter than its list
    assert L.lib().dsv4_chunk_rows(ctypes.byref(c), at, at, None, 0, 4, at, None) == 1         # a list to nowhere
    assert L.lib().dsv4_chunk_commit(ctypes.byref(c), at + 4, 512, None) == 1                  # misaligned pool
    assert L.lib().dsv4_chunk_commit(ctypes.byref(c), at, 12, None) == 1


def _compressor(**kw):
    p = L.CompressorChunkParams()
    buf = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    for name in ("kv", "score", "ape", "norm_w", "ring_kv", "ring_score", "out", "freqs", "cu_seqlens", "start",
                 "block_table"):
        setattr(p, name, at)
    p.out_rows, p.n, p.total, p.slots, p.bt_stride, p.page, p.max_comp = 64, 1, 4, 1, 1, 64, 64
    p.head_dim, p.ratio, p.rope_dim, p.out_dtype, p.norm_dtype = 512, 4, 64, 1, 0
    for k, v in kw.items():
        setattr(p, k, v)
    p._keep = buf
    return p


@pytest.mark.parametrize("bad,code", [(dict(ratio=9), 1), (dict(ratio=0), 1), (dict(head_dim=511), 1), (dict(head_dim=1026), 1),
                                      (dict(rope_dim=514), 1), (dict(act_quant=2), 1), (dict(n=2), 1), (dict(max_comp=65), 1),
                                      (dict(out=None), 1), (dict(out_dtype=2), 2), (dict(norm_dtype=3), 2),
                                      (dict(key_image=16), 1), (dict(act_quant=3), 1)])
def test_compressor_refusals_of_the_c_entry(bad, code):
    assert L.lib().dsv4_compressor_chunk(ctypes.byref(_compressor(**bad)), None) == code


def _pages(**kw):
    p = L.Pages()
    buf = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    for name in ("pool", "win_base", "block_table", "refs"):
        setattr(p, name, at)
    p.slots, p.n_pages, p.bt_stride, p.page, p.max_comp, p.window, p.head_dim, p.idx_dim, p.ratio = 2, 4, 2, 64, 128, 128, 512, 128, 4
    for k, v in kw.items():
        setattr(p, k, v)
    p._keep = buf
    return p


@pytest.mark.parametrize("bad", [dict(refs=None), dict(max_comp=129), dict(head_dim=12), dict(key_image=16), dict(ring_kv=16),
                                 dict(page=0), dict(pool=24), dict(slots=0)])
def test_pages_refusals_of_the_c_entry(bad):
    p, lib = _pages(**bad), L.lib()
    at = p.win_base
    assert lib.dsv4_pages_free(ctypes.byref(p), at, 1, None) == 1
    assert lib.dsv4_pages_reserve(ctypes.byref(p), at, at, 0, 1, at, 1 << 20, None) == 1
    assert lib.dsv4_pages_fork(ctypes.byref(p), at, at, at, 1, at, 1 << 20, None) == 1
    assert lib.dsv4_pages_compact(ctypes.byref(p), at, at, 1 << 20, None) == 1


def test_pages_workspace_and_counts():
    p, lib = _pages(), L.lib()
    at = p.win_base
    need = lib.dsv4_pages_workspace_size(ctypes.byref(p), 2)
    assert need % 16 == 0 and need >= 2 * 24 + 2 * 9 * 8 + 8 + 8
    assert lib.dsv4_pages_reserve(ctypes.byref(p), at, at, 0, 1, None, 0, None) == 6
    assert lib.dsv4_pages_fork(ctypes.byref(p), at, at, at, 2, at, need - 16, None) == 6
    assert lib.dsv4_pages_compact(ctypes.byref(p), at, None, 0, None) == 6
    assert lib.dsv4_pages_fork(ctypes.byref(p), at, at, at, 3, at, 1 << 20, None) == 1       # more branches than slots
    assert lib.dsv4_pages_free(ctypes.byref(p), None, 1, None) == 1
    assert lib.dsv4_pages_free(ctypes.byref(p), None, 0, None) == 0                           # nothing to do


def test_python_refusals():
    D = importlib.import_module(PKG + ".decode")
    pkg = importlib.import_module(PKG)
    static = D.SparseMLACache(1, 8, device="cpu")
    for call in (lambda: static.free([0]), lambda: static.reserve([0], [4]), lambda: static.fork([0], [0], [4]), static.compact):
        with pytest.raises(ValueError, match="paged"):
            call()
    with pytest.raises(ValueError):
        D.SparseMLACache(1, 8, device="cpu", n_pages=2, page_order=torch.arange(1))
    paged = D.SparseMLACache(2, 100, device="cpu", n_pages=3, max_chunk=5)
    assert paged.kv_pool.shape[0] == 2 * 128 + 3 * 64 + 5 and paged.stage_base == 2 * 128 + 3 * 64
    assert (paged.block_table == -1).all() and paged.block_table.shape == (2, 2) and paged.page_refs.tolist() == [0, 0, 0]
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.free([0])
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.chunk_attention(paged, torch.zeros(1, 64, 512, dtype=torch.bfloat16), torch.zeros(64), torch.tensor([0, 1]),
                            torch.tensor([0]))
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.compressor_chunk((torch.zeros(1, 1024),) * 2, torch.tensor([0, 1]), torch.tensor([0]), None, None, None, None, None, 1)
    st = paged.state_dict()
    assert "page_refs" in st
    with pytest.raises(ValueError, match="paged or staged"):
        D.SparseMLACache(2, 100, device="cpu", max_chunk=5).load_state_dict(st)
    with pytest.raises(ValueError, match="paged or staged"):
        D.SparseMLACache(2, 100, device="cpu", n_pages=3).load_state_dict(st)
    other = D.SparseMLACache(2, 100, device="cpu", n_pages=3, max_chunk=5)
    paged.page_refs[1] = 2
    other.load_state_dict(paged.state_dict())
    assert other.page_refs.tolist() == [0, 2, 0] and paged.clone().page_refs.tolist() == [0, 2, 0]


def _attn(**kw):
    p = L.ChunkAttnParams()
    buf = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    chunk = {k: kw.pop(k) for k in list(kw) if hasattr(p.chunk, k)}
    p.chunk = _chunk(**chunk)
    p.q = p.pool = p.sink = p.out = p.rope_freqs = p.workspace = at
    p.rope_dim, p.out_dtype, p.scale, p.num_splits, p.workspace_bytes = 64, 1, 0.04, 1, 0
    for k, v in kw.items():
        setattr(p, k, at + 4 if v == "misaligned" else v)
    p._keep = buf
    return p


@pytest.mark.parametrize("bad,code", [
    (dict(window=1088), 1), (dict(window=100), 1), (dict(page=36), 1), (dict(page=4), 1), (dict(q=None), 1), (dict(sink=None), 1),
    (dict(out=None), 1), (dict(pool=None), 1), (dict(q="misaligned"), 1), (dict(pool="misaligned"), 1), (dict(out="misaligned"), 1),
    (dict(out_dtype=2), 2), (dict(rope_dim=66), 1), (dict(rope_dim=0), 1), (dict(rope_dim=7), 1), (dict(num_splits=65), 1),
    (dict(num_splits=-1), 1), (dict(num_splits=2), 6), (dict(num_splits=2, workspace=None, workspace_bytes=1 << 40), 6),
    (dict(num_splits=2, workspace="misaligned", workspace_bytes=1 << 40), 6)])
def test_attention_refusals_of_the_c_entry(bad, code):
    """Each is refused on the host, before any launch."""
    assert L.lib().dsv4_chunk_attn(ctypes.byref(_attn(**bad)), None) == code


def test_attention_workspace_and_nothing_to_do():
    lib = L.lib()
    assert lib.dsv4_chunk_attn_workspace_size(ctypes.byref(_attn())) == 0
    total = _attn().chunk.total
    assert lib.dsv4_chunk_attn_workspace_size(ctypes.byref(_attn(num_splits=5))) == total * 5 * (64 * 512 + 128) * 4
    assert lib.dsv4_chunk_attn_workspace_size(ctypes.byref(_attn(num_splits=5, n=0))) == 0
    assert lib.dsv4_chunk_attn(ctypes.byref(_attn(num_splits=5, n=0)), None) == 0
    assert lib.dsv4_chunk_attn(None, None) == 1


def test_pages_of_a_window_only_cache():
    """No table and no counts, only the window rings: nothing to reserve, and no half of a paged cache."""
    none = dict(block_table=None, refs=None, max_comp=0, n_pages=0, bt_stride=0)
    p, lib = _pages(**none), L.lib()
    at = p.win_base
    assert lib.dsv4_pages_reserve(ctypes.byref(p), at, at, 0, 1, at, 1 << 20, None) == 0
    for bad in (dict(n_pages=4), dict(bt_stride=2), dict(pool=None), dict(win_base=None)):
        assert lib.dsv4_pages_reserve(ctypes.byref(_pages(**{**none, **bad})), at, at, 0, 1, at, 1 << 20, None) == 1
    D = importlib.import_module(PKG + ".decode")
    c = D.SparseMLACache(2, 0, device="cpu", n_pages=7)   # a window-only layer of a paged model holds no pages
    assert c.kv_pool.shape[0] == 2 * 128 and c.page_refs is None
    with pytest.raises(RuntimeError, match="CUDA"):
        c.fork([0], [1], [4])


def test_chunk_ops_trace_on_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    importlib.import_module(PKG)
    with FakeTensorMode():
        e = lambda *s, dtype=torch.int32: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        f32, bf16 = torch.float32, torch.bfloat16
        o = torch.ops.dsv4.chunk_attention(e(7, 64, 512, dtype=bf16), e(1000, 512, dtype=bf16), e(2, 3),
                                           e(2, dtype=torch.int64), e(64, dtype=f32), e(3), e(2), None, None, e(32, dtype=f32),
                                           256, 640, 128, 4, 64, 100, 0.04, f32, 0)
        assert o.shape == (7, 64, 512) and o.dtype == f32 and o.device.type == "cuda"
        assert torch.ops.dsv4.compressor_chunk(
            e(7, 1024, dtype=f32), e(7, 1024, dtype=f32), e(3), e(2), None, e(4, 1024, dtype=f32), None,
            e(2, 8, 1024, dtype=f32), e(2, 8, 1024, dtype=f32), e(1000, 512, dtype=bf16), e(2, 3), 64, 256, 100, 512, 4, 64,
            e(32, dtype=f32), 1e-6, None, None, None, 0) is None
