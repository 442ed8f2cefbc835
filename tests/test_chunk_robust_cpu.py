"""What the chunk and page entry points refuse before any launch, and how they trace: on the CPU, with fake tensors
that say they are on a GPU."""
import importlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

PKG = "deepseek-v4-flash-mlx_b200"
F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32


def _e(*shape, dtype=F32, device="cuda"):
    return torch.empty(*shape, dtype=dtype, device=device)


def _mods():
    return importlib.import_module(PKG), importlib.import_module(PKG + ".decode")


@pytest.mark.parametrize("head_dim", [64, 256, 576, 1024])
def test_chunk_attention_takes_rows_of_512(head_dim):
    """The kernel's tiles are 512 wide whatever the tensors: a cache of another width is refused, with q of that width,
    and so is the custom op's call with it."""
    pkg, D = _mods()
    with FakeTensorMode():
        c = D.SparseMLACache(2, 64, head_dim=head_dim, max_chunk=8)
        q, sink, cu, start, freqs = _e(4, 64, head_dim, dtype=BF16), _e(64), _e(2, dtype=I32), _e(1, dtype=I32), _e(32)
        for rows in (None, _e(4, 3, dtype=I32)):
            with pytest.raises(ValueError, match="512"):
                pkg.chunk_attention(c, q, sink, cu, start, rows=rows, freqs=freqs)
            for heads, qd, pd, qt, pt in ((64, head_dim, head_dim, BF16, BF16), (64, 512, head_dim, BF16, BF16), (32, 512, 512, BF16, BF16),
                                          (64, 512, 512, F32, BF16), (64, 512, 512, BF16, F32)):
                with pytest.raises((ValueError, TypeError)):
                    torch.ops.dsv4.chunk_attention(_e(4, heads, qd, dtype=qt), _e(1000, pd, dtype=pt), c.block_table, c.win_base, sink, cu, start,
                                                   None, rows, freqs, 256, 384, 128, 4, 64, 64, 0.04, BF16, 0)


def _attention_args():
    _, D = _mods()
    c = D.SparseMLACache(2, 64, max_chunk=8)
    return c, (_e(7, 64, 512, dtype=BF16), _e(64), _e(3, dtype=I32), _e(2, dtype=I32))


def _compressor_args(c):
    return ((_e(7, 1024), _e(7, 1024)), _e(3, dtype=I32), _e(2, dtype=I32), _e(4, 1024), _e(512), c.ring_kv, c.ring_score, c.kv_pool, 64)


def test_chunk_calls_on_fake_tensors():
    """The public calls, as a mode that holds no data sees them: inside it, and on its tensors outside of it."""
    pkg, _ = _mods()
    mode = FakeTensorMode()
    with mode:
        c, args = _attention_args()
        freqs, comp = _e(32), _compressor_args(c)
        kw = dict(block_table=c.block_table, page=64, out_base=256)
        for rows in (None, _e(7, 5, dtype=I32)):
            o = pkg.chunk_attention(c, *args, rows=rows, freqs=freqs, out_dtype=F32)
            assert o.shape == (7, 64, 512) and o.dtype == F32 and o.is_cuda
        assert pkg.compressor_chunk(*comp, freqs=freqs, **kw) is None
    assert pkg.chunk_attention(c, *args, freqs=freqs).shape == (7, 64, 512)
    assert pkg.compressor_chunk(*comp, freqs=freqs, **kw) is None


def test_chunk_calls_are_one_op_in_a_graph():
    from torch.fx.experimental.proxy_tensor import make_fx
    pkg, _ = _mods()
    with FakeTensorMode():
        c, args = _attention_args()
        freqs, comp = _e(32), _compressor_args(c)

        def f(q, kv):
            pkg.compressor_chunk((kv, comp[0][1]), *comp[1:], freqs=freqs, block_table=c.block_table, page=64, out_base=256)
            return pkg.chunk_attention(c, q, *args[1:], freqs=freqs)

        names = [str(n.target) for n in make_fx(f)(args[0], comp[0][0]).graph.nodes if n.op == "call_function"]
    assert names == ["dsv4.compressor_chunk.default", "dsv4.chunk_attention.default"]


def test_chunk_calls_refuse_tensors_of_another_device():
    pkg, D = _mods()
    with FakeTensorMode():
        c, (q, sink, cu, start) = _attention_args()
        ok = dict(cache=c, q=q, sink=sink, cu_seqlens=cu, start=start, seqs=_e(2, dtype=I32), rows=_e(7, 5, dtype=I32), freqs=_e(32))
        for name in ("q", "sink", "cu_seqlens", "start", "seqs", "rows", "freqs"):
            for device, err in (("cuda:1", ValueError), ("cpu", RuntimeError)):
                with pytest.raises(err):
                    pkg.chunk_attention(**{**ok, name: torch.empty_like(ok[name], device=device)})
        proj, _, _, ape, nw, rk, rs, out, most = _compressor_args(c)
        ok = dict(proj=proj, cu_seqlens=cu, start=start, ape=ape, norm_w=nw, ring_kv=rk, ring_score=rs, out=out, max_comp=most,
                  block_table=c.block_table, page=64, out_base=256, seqs=_e(2, dtype=I32), freqs=_e(32))
        for name in ok:
            for device, err in (("cuda:1", ValueError), ("cpu", RuntimeError)):
                if name == "proj":
                    with pytest.raises(err):
                        pkg.compressor_chunk(**{**ok, name: (proj[0], torch.empty_like(proj[1], device=device))})
                elif isinstance(ok[name], torch.Tensor):
                    with pytest.raises(err):
                        pkg.compressor_chunk(**{**ok, name: torch.empty_like(ok[name], device=device)})
        with pytest.raises(RuntimeError):   # all of them on the CPU
            cpu = {k: torch.empty_like(v, device="cpu") if isinstance(v, torch.Tensor) else v for k, v in ok.items()}
            pkg.compressor_chunk(**{**cpu, "proj": tuple(torch.empty_like(t, device="cpu") for t in proj)})


def test_a_chunk_of_keys_refuses_an_image_that_is_not_the_slots():
    """The image is written by slot and entry without a look at its size."""
    pkg, _ = _mods()
    I = importlib.import_module(PKG + ".indexer")  # noqa: E741
    with FakeTensorMode():
        slots, most = 2, 300
        ring = _e(slots, 8, 256), _e(slots, 8, 256)
        call = lambda image: pkg.compressor_chunk(  # noqa: E731
            (_e(7, 256), _e(7, 256)), _e(3, dtype=I32), _e(2, dtype=I32), _e(4, 256), _e(128), *ring, _e(slots, most, 128), most,
            head_dim=128, freqs=_e(32), key_image=image)
        img, inv, nmax = I.key_image_buffers(slots, most, "cuda")
        assert call((img, inv, nmax)) is None
        small = I.key_image_buffers(slots, 256, "cuda")
        for bad in ((small[0], inv, nmax), (img, small[1], nmax), (img, inv, nmax[:1]), (img.view(torch.int8), inv, nmax),
                    (img, inv.half(), nmax), (img, inv, nmax.double()), (img[::2], inv, nmax), (img, inv)):
            with pytest.raises((ValueError, TypeError)):
                call(bad)
        for k in range(3):
            image = [img, inv, nmax]
            image[k] = torch.empty_like(image[k], device="cuda:1")
            with pytest.raises(ValueError):
                call(tuple(image))


def test_rows_are_filled_into_pages_that_the_slot_holds_alone():
    """A cell without a page is -1: rows put there would land in front of the pages, in the window rings."""
    _, D = _mods()
    c = D.SparseMLACache(3, 100, device="cpu", page=16, n_pages=9)
    rows, keys = torch.ones(20, 512), torch.ones(20, 128)
    for table in ([-1] * 7, [4, -1, -1, -1, -1, -1, -1]):
        c.block_table[1] = torch.tensor(table, dtype=I32)
        with pytest.raises(ValueError, match="page"):
            c.fill_compressed(1, rows, keys)
        assert not c.kv_pool.any() and not c.k_idx.any() and not c.image_stale
    c.block_table[1, :2] = torch.tensor([4, 2], dtype=I32)
    c.page_refs[4], c.page_refs[2] = 2, 1
    with pytest.raises(ValueError, match="page"):
        c.fill_compressed(1, rows, keys)          # another slot reads the first page
    assert not c.kv_pool.any()
    c.fill_compressed(1, rows[:0], keys[:0])
    c.page_refs[4] = 1
    c.fill_compressed(1, rows, keys)
    at = c.comp_base + torch.cat([4 * 16 + torch.arange(16), 2 * 16 + torch.arange(4)])
    assert (c.kv_pool[at] == 1).all() and c.kv_pool.float().sum() == 20 * 512 and c.k_idx.sum() == 20 * 128
    with pytest.raises(ValueError):
        c.fill_compressed(1, torch.ones(101, 512), torch.ones(101, 128))


def test_default_frequencies_are_kept_for_real_calls_only():
    """The table that a call without `freqs` takes is kept between calls; not one without data, nor one for a mode."""
    pkg, _ = _mods()
    N = importlib.import_module(PKG + ".norm_rope")
    real = N.rope_freqs(64, "cpu", base=12345.0)
    with FakeTensorMode():
        c, args = _attention_args()
        assert pkg.chunk_attention(c, *args).shape == (7, 64, 512)
        assert type(N.rope_freqs(64, "cpu", base=12345.0)) is not torch.Tensor
        assert type(N.rope_freqs(32, "cpu", base=12345.0)) is not torch.Tensor
    assert N.rope_freqs(64, "cpu", base=12345.0) is real
    assert type(N.rope_freqs(32, "cpu", base=12345.0)) is torch.Tensor
    assert all(type(t) is torch.Tensor for t in N._freq_cache.values())
