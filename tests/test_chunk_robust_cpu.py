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
