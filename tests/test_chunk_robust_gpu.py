"""Chunks over a used cache: repeated long chunks, slots that begin again, rows that are no rows of the pool, values
that are not finite."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
PKG = "deepseek-v4-flash-mlx_b200"


def _mods():
    return importlib.import_module(PKG), importlib.import_module(PKG + ".decode"), importlib.import_module(PKG + "._lib")


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("d,quant,start", [(512, 0, 3), (512, 1, 0), (512, 0, 1000001), (512, 1, 4000002), (128, 0, 7), (128, 1, 2000003),
                                           (128, 2, 5), (64, 0, 1), (192, 0, 2)])
def test_long_chunks_again_and_again(d, quant, start):
    """A chunk that is streamed, bit for bit as the kernel that takes a row at a time leaves it, every time. (That
    kernel takes projections that are not 16-byte aligned, whatever their number.)"""
    pkg, _, L = _mods()
    g = torch.Generator(device="cuda").manual_seed(d + quant)
    n, page = 30001, 64
    first, most = start // 4, (start + n) // 4 + 1
    pages = (most - 1) // page - first // page + 1
    # only the pages that the chunk writes to are there, in another order than that of their entries
    table = torch.full((1, (most - 1) // page + 1), -1, dtype=torch.int32)
    table[0, first // page:] = torch.randperm(pages, generator=torch.Generator().manual_seed(d)).to(torch.int32)
    table = table.cuda()
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kv, sc, ape, nw = rnd(n, 2 * d), rnd(n, 2 * d), rnd(4, 2 * d), 1 + 0.1 * rnd(d)
    ring, rope = (rnd(1, 8, 2 * d), rnd(1, 8, 2 * d)), 64 if d > 64 else 0
    freqs = 1.0 / (160000.0 ** (torch.arange(0, 64, 2, dtype=torch.float32, device="cuda") / 64))
    off = [torch.empty(n * 2 * d + 2, device="cuda")[2:].view(n, 2 * d).copy_(t) for t in (kv, sc)]
    assert all(t.data_ptr() % 16 == 8 for t in off)

    def run(proj):
        rings = [t.clone() for t in ring]
        out = torch.zeros(pages * page, d, device="cuda", dtype=torch.bfloat16 if d == 512 else torch.float32)
        pkg.compressor_chunk(proj, _i32(0, n), _i32(start), ape, nw, *rings, out, most, block_table=table, page=page, head_dim=d,
                             freqs=freqs, rope_head_dim=rope, act_quant=quant == 1, rotate=quant == 2)
        return out, *rings

    want = run(off)
    for _ in range(20):
        for name, a, b in zip(("rows", "ring_kv", "ring_score"), run((kv, sc)), want):
            assert torch.equal(a, b), name
    assert L.device_error() == 0
