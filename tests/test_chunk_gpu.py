"""Chunks of new tokens over a (paged) cache: attention, compressor, row moves and whole layers, against
plain forms in 64 bits and against one token after the other.

Tolerances. The attention rounds each probability and the output to bf16, each by half a step at most,
a relative 2^-8 (torch.finfo(bf16).eps / 2 = 2^-8); products and sums are fp32. With p_j the exact
normalised weights, the rounded weights w_j = p_j (1 + d_j), |d_j| <= 2^-8, give
|o' - o| <= sum_j p_j |d_j| |v_j| + |o| sum_j p_j |d_j| (the denominator's change, where the sum is of
rounded weights) <= 2^-8 (A + |o|) <= 2^-7 A with A = sum_j p_j |v_j|, and the rounding of the output adds 2^-8 |o| <= 2^-8 A.
So |got - exact| <= 3 * 2^-8 A per element, and before the inverse rotation; the rotation mixes two
elements, whose bounds then add up to sqrt(2) times the larger at most: 3 * 2^-8 * (A_d + A_d').
The fp32 parts (512-term products, exp) stay below 2^-14 of the same scale and are covered by one more 2^-8 A.
"""
import importlib

import numpy as np
import pytest
import torch

from helpers import rel_rms

pytestmark = pytest.mark.gpu
PKG = "deepseek-v4-flash-mlx_b200"
H, D, W, R = 64, 512, 128, 4
EPS = torch.finfo(torch.bfloat16).eps / 2   # 2^-8


def _mods():
    return importlib.import_module(PKG), importlib.import_module(PKG + ".decode"), importlib.import_module(PKG + "._lib")


def _freqs():
    return 1.0 / (160000.0 ** (torch.arange(0, 64, 2, dtype=torch.float32) / 64))


def _case(lens, start, page=64, ratio=4, seed=0, paged=False, seqs=None, slots=None, pad=0, window=W):
    """A cache with random rows, a chunk staged in it and its queries."""
    pkg, Dm, _ = _mods()
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(lens) + pad
    slots = slots or len(lens)
    seqs = seqs or list(range(len(lens)))
    most = max(max((s + n) // ratio for n, s in zip(lens, start)), 1) if ratio else 0
    per = -(-most // page)
    if paged:
        c = Dm.SparseMLACache(slots, most, page=page, ratio=ratio or 4, n_pages=slots * per + 5, max_chunk=total, window=window)
        c.reserve(seqs, [s + n for n, s in zip(lens, start)])
    else:
        order = torch.randperm(slots * per, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        c = Dm.SparseMLACache(slots, most, page=page, ratio=ratio or 4, page_order=order if most else None, max_chunk=total,
                              window=window)
    c.kv_pool.copy_(torch.randn(c.kv_pool.shape, generator=g, device="cuda").to(torch.bfloat16))
    q = torch.randn(total, H, D, generator=g, device="cuda")
    q = (q * torch.rsqrt(q.square().mean(-1, keepdim=True))).to(torch.bfloat16)
    sink = torch.randn(H, generator=g, device="cuda")
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    return c, q, sink, cu, torch.tensor(start, dtype=torch.int32, device="cuda"), torch.tensor(seqs, dtype=torch.int32, device="cuda")


def _rotate64(x, pos, f, sign):
    a = (pos.float()[:, None] * f.to(pos.device)).double()[:, None, :] * sign
    y = x.clone()
    y[..., -64::2] = x[..., -64::2] * a.cos() - x[..., -63::2] * a.sin()
    y[..., -63::2] = x[..., -64::2] * a.sin() + x[..., -63::2] * a.cos()
    return y


def _attention64(c, q, sink, lens, start, seqs, rows=None, scale=D ** -0.5):
    """o and the bound of each element, in 64 bits, token by token."""
    f, pool = _freqs().cuda(), c.kv_pool.double()
    out, tol = [], []
    at = 0
    for n, s, b in zip(lens, start, seqs):
        for i in range(n):
            p = s + i
            r = []
            for w in range(max(0, p - c.window + 1), p + 1):
                r.append(c.stage_base + at + w - s if w >= s else int(c.win_base[b]) + w % c.window)
            r = torch.tensor(r, device="cuda")
            if rows is not None:
                mine = rows[at + i].long()
                r = torch.cat([r, mine[mine >= 0]])
            elif c.compressed:
                e = torch.arange(min((p + 1) // c.ratio, c.max_comp), device="cuda")
                if e.numel():
                    r = torch.cat([r, c.comp_base + c.block_table[b].long()[e // c.page] * c.page + e % c.page])
            kv = pool[r]
            x = torch.cat([q[at + i].double() @ kv.T * scale, sink.double()[:, None]], 1)
            w = torch.softmax(x, -1)[:, :-1]
            o, a = w @ kv, w @ kv.abs()
            a[:, -64:] = a[:, -64:] + a[:, -64:].reshape(H, 32, 2).flip(-1).reshape(H, 64)
            out.append(_rotate64(o[None], torch.tensor([p], device="cuda"), f, -1)[0])
            tol.append(4 * EPS * a)
        at += n
    return torch.stack(out), torch.stack(tol)


def _check(got, want, tol):
    got = got[:want.shape[0]].double()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / tol).max().item()
    assert worst <= 1, worst


# lengths and starts around the ring's and the tiles' borders: empty windows, a window that the chunk
# fills, a ring that has wrapped, one token, more than two windows of tokens, odd and even counts
CASES = [([1], [0]), ([1], [127]), ([2], [3]), ([5], [0]), ([3], [126]), ([7, 1, 2], [300, 0, 1023]), ([64], [64]),
         ([129], [60]), ([130, 1], [511, 4000]), ([300], [0]), ([0, 4, 0, 1], [9, 700, 1, 5000]), ([33, 34], [255, 256])]


@pytest.mark.parametrize("lens,start", CASES)
def test_chunk_attention(lens, start):
    pkg, _, L = _mods()
    c, q, sink, cu, st, _ = _case(lens, start, seed=1)
    o = pkg.chunk_attention(c, q, sink, cu, st, freqs=_freqs().cuda())
    assert o.dtype == torch.bfloat16 and L.device_error() == 0
    want, tol = _attention64(c, q, sink, lens, start, range(len(lens)))
    _check(o, want, tol)


@pytest.mark.parametrize("page", [8, 16, 24, 32, 48, 64, 100, 128, 256])
def test_chunk_attention_page_sizes(page):
    """Pages smaller than, larger than and out of step with the rows taken at a time, handed out by the cache."""
    pkg, _, L = _mods()
    lens, start = [5, 70, 1], [611, 1200, 37]
    c, q, sink, cu, st, _ = _case(lens, start, page=page, seed=2, paged=True)
    o = pkg.chunk_attention(c, q, sink, cu, st, freqs=_freqs().cuda())
    assert L.device_error() == 0
    want, tol = _attention64(c, q, sink, lens, start, range(3))
    _check(o, want, tol)


def test_chunk_attention_window_only_slots_padding_and_types():
    """A cache without compressed rows; sequences in other slots than their order; rows behind the last
    sequence; an fp32 output; strided queries, 64-bit indices; another window."""
    pkg, _, L = _mods()
    f = _freqs().cuda()
    lens, start, seqs = [9, 200, 3], [50, 1000, 0], [4, 0, 2]
    for ratio, window in ((0, 128), (4, 128), (4, 256), (4, 64)):
        c, q, sink, cu, st, sq = _case(lens, start, ratio=ratio, seed=3, seqs=seqs, slots=5, pad=7, window=window)
        wide = torch.empty(q.shape[0], H, 2 * D, dtype=q.dtype, device="cuda")
        wide[..., :D] = q
        o = pkg.chunk_attention(c, wide[..., :D], sink, cu.long(), st.long(), seqs=sq.long(), freqs=f, out_dtype=torch.float32)
        assert o.dtype == torch.float32 and o.shape == q.shape
        want, tol = _attention64(c, q, sink, lens, start, seqs)
        _check(o, want, tol)
        assert L.device_error() == 0


@pytest.mark.parametrize("lens,start,k", [([40], [3000], 64), ([5, 17], [100, 2000], 33), ([2], [9], 16), ([1], [40000], 512)])
def test_chunk_attention_listed(lens, start, k):
    """Given rows instead of all: lists with gaps, empty lists, the first tokens without any entry."""
    pkg, _, L = _mods()
    c, q, sink, cu, st, _ = _case(lens, start, seed=4)
    rng = np.random.default_rng(5)
    rows = np.full((sum(lens), k), -1, np.int32)
    at = 0
    for b, (n, s) in enumerate(zip(lens, start)):
        for i in range(n):
            seen = (s + i + 1) // R
            e = np.sort(rng.choice(seen, min(k, seen), replace=False)) if i % 5 != 4 else np.zeros(0, int)
            put = np.sort(rng.choice(k, len(e), replace=False))
            bt = c.block_table[b].cpu().numpy()
            rows[at + i, put] = c.comp_base + bt[e // c.page] * c.page + e % c.page
        at += n
    rows = torch.from_numpy(rows).cuda()
    o = pkg.chunk_attention(c, q, sink, cu, st, rows=rows, freqs=_freqs().cuda())
    assert L.device_error() == 0
    want, tol = _attention64(c, q, sink, lens, start, range(len(lens)), rows)
    _check(o, want, tol)


def test_chunk_attention_masked_rows_may_hold_anything():
    """NaN and infinities in every row that no token of the chunk sees: ring slots out of the window,
    entries not yet complete, other sequences' stages and pages, rows behind the stage."""
    pkg, _, L = _mods()
    lens, start, seqs = [3, 70], [130, 77], [0, 1]
    c, q, sink, cu, st, _ = _case(lens, start, seed=6, slots=3, pad=60)
    seen = torch.zeros(c.kv_pool.shape[0], dtype=torch.bool, device="cuda")
    at = 0
    for n, s, b in zip(lens, start, seqs):
        seen[c.stage_base + at:c.stage_base + at + n] = True
        w = torch.arange(max(0, s - c.window + 1), s, device="cuda")
        seen[b * c.window + w % c.window] = True
        e = torch.arange((s + n) // R, device="cuda")
        seen[c.comp_base + c.block_table[b].long()[e // c.page] * c.page + e % c.page] = True
        at += n
    want, tol = _attention64(c, q, sink, lens, start, seqs)
    bad = torch.tensor([float("nan"), float("inf"), float("-inf")], device="cuda").to(torch.bfloat16)
    fill = bad[torch.arange(c.kv_pool.shape[0], device="cuda") % 3]
    c.kv_pool[~seen] = fill[~seen][:, None]
    q[sum(lens):] = float("nan")
    o = pkg.chunk_attention(c, q, sink, cu, st, freqs=_freqs().cuda())
    _check(o, want, tol)
    assert L.device_error() == 0


def test_chunk_attention_large_scores_and_sinks():
    """Scores far apart (a running maximum that keeps growing along the list), sinks that swallow all or nothing."""
    pkg, _, _ = _mods()
    lens, start = [6], [2100]
    c, q, sink, cu, st, _ = _case(lens, start, seed=7)
    grow = torch.linspace(0.01, 12, c.kv_pool.shape[0], device="cuda")[:, None]
    c.kv_pool.copy_((c.kv_pool.float() * grow).to(torch.bfloat16))
    sink = torch.linspace(-300, 300, H, device="cuda")
    o = pkg.chunk_attention(c, q, sink, cu, st, freqs=_freqs().cuda())
    want, tol = _attention64(c, q, sink, lens, start, [0])
    # scores up to 12 * 60: their fp32 rounding (512 products) moves a weight by up to 2^-24 * 512 * 720 / sqrt(512) = 2^-10
    _check(o, want, tol * 1.25 + 1e-30)


def test_chunk_attention_graph_streams_and_repeat():
    """Captured and replayed with other inputs; two streams at once; the same call twice, bit for bit."""
    pkg, _, _ = _mods()
    f = _freqs().cuda()
    a = _case([5, 3], [900, 40], seed=8)
    b = _case([5, 3], [900, 40], seed=9)
    args = lambda k: (k[0], k[1], k[2], k[3], k[4])  # noqa: E731
    want_a, want_b = pkg.chunk_attention(*args(a), freqs=f), pkg.chunk_attention(*args(b), freqs=f)
    assert torch.equal(want_a, pkg.chunk_attention(*args(a), freqs=f))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s, k in ((s1, a), (s2, b)):
            with torch.cuda.stream(s):
                outs.append(pkg.chunk_attention(*args(k), freqs=f))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want_a) for x in outs[::2]) and all(torch.equal(x, want_b) for x in outs[1::2])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = pkg.chunk_attention(*args(a), freqs=f)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want_a)
    a[0].kv_pool.copy_(b[0].kv_pool), a[0].block_table.copy_(b[0].block_table), a[1].copy_(b[1]), a[2].copy_(b[2])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want_b)


def test_chunk_attention_refusals():
    pkg, Dm, L = _mods()
    c, q, sink, cu, st, sq = _case([4], [100], seed=10)
    ok = dict(cache=c, q=q, sink=sink, cu_seqlens=cu, start=st)
    for err, kw in ((TypeError, dict(q=q.float())), (ValueError, dict(q=q[:, :32])), (ValueError, dict(q=q[..., :256])),
                    (ValueError, dict(sink=sink[:3])), (TypeError, dict(out_dtype=torch.float16)),
                    (ValueError, dict(start=st.repeat(2))), (TypeError, dict(cu_seqlens=cu.float())),
                    (ValueError, dict(seqs=sq.repeat(2))), (ValueError, dict(cu_seqlens=torch.zeros(3, dtype=torch.int32, device="cuda"),
                                                                            start=st.repeat(2))),
                    (ValueError, dict(rows=torch.zeros(3, 5, dtype=torch.int32, device="cuda"))),
                    (ValueError, dict(rows=torch.zeros(4, 5, device="cuda"))), (RuntimeError, dict(sink=sink.cpu())),
                    (ValueError, dict(q=q.repeat(2, 1, 1)))):
        with pytest.raises(err):
            pkg.chunk_attention(**{**ok, **kw})
    assert pkg.chunk_attention(**{**ok, "q": q[:0], "cu_seqlens": cu * 0}).shape == (0, H, D)
    # an entry whose page the sequence does not have: reported, and the rest of its rows still attended
    p, q, sink, cu, st, _ = _case([4], [1000], seed=11, paged=True)
    p.block_table[0, 2] = -1
    o = pkg.chunk_attention(p, q, sink, cu, st, freqs=_freqs().cuda())
    assert torch.isfinite(o).all() and L.device_error() == 4 and L.device_error() == 0


# ---- the compressor over a chunk ----

def _compress_by_step(pkg, kv, sc, lens, start, seqs, ape, nw, rk, rs, out, rows_of, d, ratio, f, **kw):
    """One compressor_decode_step per token."""
    at = 0
    for n, s, b in zip(lens, start, seqs):
        for i in range(n):
            p = torch.tensor([s + i], dtype=torch.int32, device="cuda")
            r = torch.tensor([rows_of(b, max((s + i + 1) // ratio - 1, 0))], device="cuda")
            pkg.compressor_decode_step(p, kv, kv, ape, nw, rk[b:b + 1], rs[b:b + 1], p, out, r, head_dim=d, ratio=ratio, freqs=f,
                                       proj=(kv[at + i:at + i + 1].contiguous(), sc[at + i:at + i + 1].contiguous()), **kw)
        at += n


@pytest.mark.parametrize("d,ratio,lens,start", [
    (512, 4, [1], [0]), (512, 4, [1], [3]), (512, 4, [4, 4, 4, 4], [0, 1, 2, 3]), (512, 4, [9, 1, 0, 30], [0, 7, 5, 10]),
    (128, 4, [17, 2, 3], [6, 0, 13]), (1024, 4, [21], [2]), (96, 4, [11, 8], [1, 4]), (64, 1, [5, 3], [0, 7]),
    (512, 2, [7, 1], [1, 3]), (128, 3, [10, 2], [4, 0]), (512, 8, [37, 5], [3, 16]), (512, 5, [23], [7])])
@pytest.mark.parametrize("quant", [0, 1, 2])
def test_compressor_chunk_equals_the_steps(d, ratio, lens, start, quant):
    """Rows, rings and key image bit for bit as one decode step per token leaves them (the order of the
    operations in a row is the same)."""
    pkg, Dm, L = _mods()
    if (quant == 2 and d != 128) or (quant == 1 and d % 64):
        pytest.skip("a quantisation of other widths")
    I = importlib.import_module(PKG + ".indexer")
    g = torch.Generator(device="cuda").manual_seed(d + ratio)
    rope = min(64, d - 64 if quant == 1 and d > 64 else d)
    if quant == 1 and d == 64:
        rope = 0
    f = (_freqs() if rope else torch.zeros(1)).cuda()
    slots, page = len(lens) + 2, 16
    seqs = list(range(1, len(lens) + 1))
    most = max((s + n) // ratio for n, s in zip(lens, start)) + 3
    per = -(-most // page)
    table = torch.randperm(slots * per, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(slots, per).cuda()
    total = sum(lens)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kv, sc, ape, nw = rnd(total, 2 * d), rnd(total, 2 * d), rnd(ratio, 2 * d), 1 + 0.1 * rnd(d)
    rk, rs = rnd(slots, 2 * ratio, 2 * d), rnd(slots, 2 * ratio, 2 * d)
    for s, b in zip(start, seqs):
        if s < ratio:
            rk[b], rs[b, :ratio] = 0, float("-inf")
            rs[b, ratio + s:] = float("-inf")
    keys = d == 128 and ratio == 4
    dt = torch.float32 if d == 128 else torch.bfloat16
    out = torch.zeros((3 + slots * per * page, d), dtype=dt, device="cuda")
    image = I.key_image_buffers(slots, most, "cuda") if keys else None
    state = [rk, rs, out, *(image or ())]
    mine, ref = [t.clone() for t in state], [t.clone() for t in state]
    bt = table.cpu()
    if keys:
        rows_of, kw, ckw = (lambda b, e: b * most + e), dict(key_image=(*ref[3:], most)), dict(key_image=mine[3:])
    else:
        rows_of, kw, ckw = (lambda b, e: 3 + int(bt[b, e // page]) * page + e % page), {}, dict(block_table=table, page=page, out_base=3)
    q = dict(act_quant=quant == 1, rotate=quant == 2, rope_head_dim=rope)
    _compress_by_step(pkg, kv, sc, lens, start, seqs, ape, nw, ref[0], ref[1], ref[2], rows_of, d, ratio, f, **kw, **q)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    pkg.compressor_chunk((kv, sc), cu, torch.tensor(start, dtype=torch.int32, device="cuda"), ape, nw, mine[0], mine[1], mine[2],
                         most, seqs=torch.tensor(seqs, dtype=torch.int32, device="cuda"), head_dim=d, ratio=ratio, freqs=f,
                         **ckw, **q)
    assert L.device_error() == 0
    for name, a, b in zip(("ring_kv", "ring_score", "rows", "image", "inv", "norm_max"), mine, ref):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("d,lens,start,quant", [(512, [5000, 3, 0, 40], [3, 8, 1, 5], 0), (512, [2600], [0], 1), (128, [9999, 777], [1, 30], 2),
                                               (128, [12000], [4], 0), (64, [4, 20000], [2, 7], 0)])
def test_compressor_chunk_long(d, lens, start, quant):
    """Chunks long enough to be streamed, bit for bit the same as in pieces of at most 37 tokens, which are
    not; padding behind the last sequence, several sequences, odd starts, a paged table and keys."""
    pkg, _, L = _mods()
    I = importlib.import_module(PKG + ".indexer")
    g = torch.Generator(device="cuda").manual_seed(d)
    f, page = _freqs().cuda(), 16
    most = max((s + n) // 4 for n, s in zip(lens, start)) + 1
    slots, per = len(lens), -(-most // page)
    table = torch.randperm(slots * per, generator=torch.Generator().manual_seed(2)).to(torch.int32).view(slots, per).cuda()
    total = sum(lens) + 9
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kv, sc, ape, nw = rnd(total, 2 * d), rnd(total, 2 * d), rnd(4, 2 * d), 1 + 0.1 * rnd(d)
    keys = d == 128
    out = torch.zeros(slots * per * page if not keys else slots * most, d, device="cuda", dtype=torch.float32 if keys else torch.bfloat16)
    state = [rnd(slots, 8, 2 * d), rnd(slots, 8, 2 * d), out, *(I.key_image_buffers(slots, most, "cuda") if keys else ())]
    a, b = [t.clone() for t in state], [t.clone() for t in state]
    kw = lambda st: dict(key_image=st[3:]) if keys else dict(block_table=table, page=page)  # noqa: E731
    q = dict(act_quant=quant == 1, rotate=quant == 2, rope_head_dim=min(64, d) if d > 64 or not quant else 0)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    pkg.compressor_chunk((kv, sc), i32(np.concatenate([[0], np.cumsum(lens)])), i32(start), ape, nw, a[0], a[1], a[2], most, head_dim=d,
                         freqs=f, **kw(a), **q)
    at = 0
    for slot, (n, s) in enumerate(zip(lens, start)):
        for o in range(0, n, 37):
            m = min(37, n - o)
            pkg.compressor_chunk((kv[at + o:at + o + m], sc[at + o:at + o + m]), i32([0, m]), i32([s + o]), ape, nw, b[0], b[1], b[2], most,
                                 seqs=i32([slot]), head_dim=d, freqs=f, **kw(b), **q)
        at += n
    assert L.device_error() == 0
    for name, x, y in zip(("ring_kv", "ring_score", "rows", "image", "inv", "norm_max"), a, b):
        assert torch.equal(x, y), name


def test_compressor_chunk_against_the_definition():
    """Rows in 64 bits: eight-slot softmax, norm and rotation. fp32 arithmetic: at most 40 roundings of
    2^-24 on values of the row's scale (each output is a normalised weighted mean; the norm divides by the
    rms, 512 terms summed in a tree), plus the rotation's angle, an exact product of fp32 in both."""
    pkg, _, L = _mods()
    g = torch.Generator(device="cuda").manual_seed(3)
    n, s, d = 203, 5, 512
    kv, sc = (torch.randn(n, 2 * d, generator=g, device="cuda") for _ in range(2))
    ape, nw = torch.randn(4, 2 * d, generator=g, device="cuda"), torch.ones(d, device="cuda")
    rk, rs = (torch.randn(1, 8, 2 * d, generator=g, device="cuda") for _ in range(2))
    k = torch.cat([rk[0, :5], kv]).double()                       # positions 0..4 from the ring (block 0, then token 4)
    x = torch.cat([rs[0, :5], sc + ape[(s + torch.arange(n, device="cuda")) % 4]]).double()
    blocks = k.shape[0] // 4
    k, x = k[:blocks * 4].view(blocks, 4, 2, d), x[:blocks * 4].view(blocks, 4, 2, d)
    w = torch.softmax(torch.cat([x[:-1, :, 0], x[1:, :, 1]], 1), 1)
    row = (w * torch.cat([k[:-1, :, 0], k[1:, :, 1]], 1)).sum(1)
    row = row / (row.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    pos = 4 * torch.arange(1, blocks, device="cuda")
    row = _rotate64(row[:, None], pos, _freqs(), 1)[:, 0]
    out = torch.zeros(60, d, device="cuda")
    pkg.compressor_chunk((kv, sc), torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                         torch.tensor([s], dtype=torch.int32, device="cuda"), ape, nw, rk, rs, out, 60, freqs=_freqs().cuda())
    assert L.device_error() == 0
    assert (out[0] == 0).all() and (out[blocks:] == 0).all()
    assert ((out[1:blocks].double() - row).abs() <= 40 * 2.0 ** -24 * row.abs().amax(-1, keepdim=True)).all()


def test_compressor_chunk_errors_and_refusals():
    pkg, _, L = _mods()
    g = torch.Generator(device="cuda").manual_seed(4)
    kv, sc = (torch.randn(12, 1024, generator=g, device="cuda") for _ in range(2))
    ape, nw = torch.zeros(4, 1024, device="cuda"), torch.ones(512, device="cuda")
    ring = lambda: (torch.zeros(2, 8, 1024, device="cuda"), torch.zeros(2, 8, 1024, device="cuda"))  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    # past the end of the cache, a missing page, a page outside of `out`, a slot that does not exist: reported, not stored
    for table, most, seqs in ((i32(0).view(1, 1).repeat(2, 1), 2, None), (i32(-1).view(1, 1).repeat(2, 1), 8, None),
                              (i32(9).view(1, 1).repeat(2, 1), 8, None), (i32(0).view(1, 1).repeat(2, 1), 8, i32(7))):
        out = torch.zeros(16, 512, device="cuda")
        pkg.compressor_chunk((kv, sc), i32(0, 12), i32(0), ape, nw, *ring(), out, most, block_table=table, page=8, seqs=seqs)
        assert L.device_error() == 4
        assert (out[2 if most == 2 else 0:] == 0).all()
    out, r = torch.zeros(16, 512, device="cuda"), ring()
    good = dict(proj=(kv, sc), cu_seqlens=i32(0, 12), start=i32(0), ape=ape, norm_w=nw, ring_kv=r[0], ring_score=r[1], out=out,
                max_comp=8)
    for err, kw in ((ValueError, dict(proj=(kv[:, :512], sc[:, :512]))), (ValueError, dict(proj=(kv.half(), sc.half()))),
                    (ValueError, dict(ring_kv=r[0][:, :4])), (ValueError, dict(ring_score=r[1][:1])), (ValueError, dict(out=out.half())),
                    (ValueError, dict(out=out[:, :256])), (ValueError, dict(start=i32(0, 1))), (TypeError, dict(start=i32(0).long())),
                    (ValueError, dict(max_comp=9)), (ValueError, dict(ape=ape[:2])), (ValueError, dict(norm_w=nw[:9])),
                    (ValueError, dict(block_table=i32(0).view(1, 1), page=8)), (RuntimeError, dict(start=torch.tensor([0], dtype=torch.int32))),
                    (ValueError, dict(freqs=torch.ones(3, device="cuda"))), (ValueError, dict(seqs=i32(0, 1)))):
        with pytest.raises(err):
            pkg.compressor_chunk(**{**good, **kw})


# ---- rows, and whole layers ----

def test_chunk_rows_and_commit():
    pkg, _, L = _mods()
    lens, start, seqs = [300, 2, 0, 64], [10, 127, 3, 500], [1, 0, 4, 2]
    c, q, sink, cu, st, sq = _case(lens, start, seed=12, seqs=seqs, slots=5, pad=3)
    pos, rows = pkg.chunk_rows(c, cu, st, q.shape[0], sq)
    want = np.concatenate([np.arange(s, s + n) for n, s in zip(lens, start)] + [np.zeros(3, int)])
    assert (pos.cpu().numpy() == want).all()
    assert torch.equal(rows, c.stage_base + torch.arange(q.shape[0], device="cuda"))
    ref, at = c.kv_pool.clone(), 0
    for n, s, b in zip(lens, start, seqs):
        for i in range(max(0, n - W), n):
            ref[b * W + (s + i) % W] = ref[c.stage_base + at + i]
        at += n
    pkg.chunk_commit(c, cu, st, q.shape[0], sq)
    assert torch.equal(c.kv_pool, ref) and L.device_error() == 0


def _block(ratio, batch, max_ctx, top_k, **kw):
    Lm, C = importlib.import_module(PKG + ".layer"), importlib.import_module(PKG + ".configs")
    dims = C.LayerDims(ratio=ratio)
    Wt = Lm.make_attention_weights(40 + ratio, dims=dims).to("cuda")
    return Lm.DecodeBlock(Wt, batch, max_ctx, top_k=top_k, dims=dims, **kw), Wt, dims, Lm


# both take the same bf16 roundings at the same places; the projections' sums run in another order (fp32),
# which moves a value across a rounding border here and there: the block bound of the layer tests
BLOCK_REL = 1e-2


@pytest.mark.parametrize("ratio,paged,top_k", [(4, False, 512), (4, True, 512), (4, True, 32), (0, False, 512), (128, False, 512)])
def test_extend_equals_the_steps(ratio, paged, top_k):
    """Chunks and single tokens on two sequences, against single tokens alone: outputs, window rings,
    compressed rows and compressor rings."""
    pkg, _, L = _mods()
    kw = dict(n_pages=24) if paged else {}
    a, Wt, dims, Lm = _block(ratio, 2, 640, top_k, max_chunk=320, page=16, **kw)
    b, _, _, _ = _block(ratio, 2, 640, top_k, page=16, **kw)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(2, 330, 4096, generator=g, device="cuda")
    outs = [[], []]
    o = a.extend(torch.cat([x[0, :150], x[1, :150], x[0, :9]]), [150, 150], [0, 0])       # nine rows of padding
    outs[0].append(o[:150]), outs[1].append(o[150:300])
    o = a.extend(torch.cat([x[1, 150:157], x[0, 150:320]]), [7, 170], [150, 150], seqs=[1, 0])
    outs[1].append(o[:7]), outs[0].append(o[7:])
    o = a.extend(x[1, 157:320], [163], [157], seqs=[1])
    outs[1].append(o)
    o = a.step(x[:, 320], torch.full((2,), 320, dtype=torch.int32, device="cuda"))
    outs[0].append(o[:1]), outs[1].append(o[1:])
    ref = [b.step(x[:, p], torch.full((2,), p, dtype=torch.int32, device="cuda")) for p in range(321)]
    ref = torch.stack(ref, 1)
    assert L.device_error() == 0
    for s in range(2):
        got = torch.cat(outs[s])
        if top_k > 80:
            assert rel_rms(got, ref[s]) <= BLOCK_REL
        else:   # selections from scores an fp32 rounding apart: the tokens before the first selection, and most after
            assert rel_rms(got[:4 * top_k], ref[s][:4 * top_k]) <= BLOCK_REL
            near = ((got - ref[s]).norm(dim=-1) / ref[s].norm(dim=-1)) <= 2 * BLOCK_REL
            assert near.float().mean() >= 0.9
        assert rel_rms(a.cache.kv_pool[s * W:(s + 1) * W].float(), b.cache.kv_pool[s * W:(s + 1) * W].float()) <= BLOCK_REL
        if ratio == 4:
            e = torch.arange(80, device="cuda")
            assert rel_rms(a.cache.kv_pool[a.cache.comp_rows(s, e)].float(), b.cache.kv_pool[b.cache.comp_rows(s, e)].float()) <= BLOCK_REL
            assert rel_rms(a.cache.k_idx[s, :80], b.cache.k_idx[s, :80]) <= BLOCK_REL
            assert rel_rms(a.cache.ring_kv[s], b.cache.ring_kv[s]) <= BLOCK_REL


def test_extend_continues_a_prefill_and_refuses():
    """prefill_layer of a prompt, then a chunk: the rows of the whole prompt's prefill."""
    pkg, _, L = _mods()
    blk, Wt, dims, Lm = _block(4, 1, 640, 512, max_chunk=128, n_pages=5, page=32)
    x = torch.randn(300, 4096, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    whole = Lm.prefill_layer(x, Wt, dims=dims)
    _, aux = Lm.prefill_layer(x[:190], Wt, dims=dims, return_aux=True)
    blk.load_prefill(0, aux)
    o = blk.extend(x[190:300], [110], [190])
    assert L.device_error() == 0 and rel_rms(o, whole[190:]) <= BLOCK_REL
    assert blk.cache.page_refs.sum() == -(-75 // 32)
    for kw in (dict(lengths=[3], start=[300, 1]), dict(lengths=[5], start=[300]), dict(lengths=[-1], start=[300]),
               dict(lengths=[4], start=[-1]), dict(lengths=[1, 1], start=[3, 4], seqs=[0, 0]), dict(lengths=[4], start=[700]),
               dict(lengths=[4], start=[300], seqs=[1])):
        with pytest.raises(ValueError):
            blk.extend(x[:4], **kw)
    with pytest.raises(ValueError, match="max_chunk"):
        blk.extend(x[:200], [200], [300])


# ---- calls at the edges of what the entry points allow ----

@pytest.mark.parametrize("splits", [1, 2, 3, 7, 8, 9, 33, 64])
def test_chunk_attention_any_number_of_splits(splits):
    """More splits than a token has tiles leave some without rows."""
    pkg, _, L = _mods()
    lens, start = [3, 0, 2], [1700, 9, 20]
    c, q, sink, cu, st, _ = _case(lens, start, seed=31)
    want, tol = _attention64(c, q, sink, lens, start, range(3))
    for dtype in (torch.bfloat16, torch.float32):
        _check(pkg.chunk_attention(c, q, sink, cu, st, freqs=_freqs().cuda(), num_splits=splits, out_dtype=dtype), want, tol)
    assert L.device_error() == 0


def test_chunk_attention_many_sequences():
    """More sequences than a warp looks at together, and more pairs of tokens than clusters."""
    pkg, _, L = _mods()
    rng = np.random.default_rng(5)
    lens, start = [int(n) for n in rng.integers(0, 6, 75)], [int(p) for p in rng.integers(0, 400, 75)]
    seqs = [int(b) for b in rng.permutation(80)[:75]]
    c, q, sink, cu, st, sq = _case(lens, start, seed=32, seqs=seqs, slots=80, page=16, paged=True, pad=5)
    o = pkg.chunk_attention(c, q, sink, cu, st, seqs=sq, freqs=_freqs().cuda())
    assert L.device_error() == 0
    want, tol = _attention64(c, q, sink, lens, start, seqs)
    _check(o, want, tol)


@pytest.mark.parametrize("window", [64, 192, 1024, 2048])
def test_chunk_attention_windows(window):
    pkg, _, L = _mods()
    lens, start = [3, 70, 1], [window + 11, 2 * window - 30, window - 1]
    c, q, sink, cu, st, _ = _case(lens, start, seed=33, window=window)
    o = pkg.chunk_attention(c, q, sink, cu, st, freqs=_freqs().cuda())
    assert L.device_error() == 0
    want, tol = _attention64(c, q, sink, lens, start, range(3))
    _check(o, want, tol)


def test_rows_past_32_bit_offsets():
    """Pages and stage behind 4 GB and 2^31 elements of pool: attention both ways, compressor, commit."""
    pkg, Dm, L = _mods()
    n_pages, n, s = 70000, 9, 1001
    c = Dm.SparseMLACache(1, 260, n_pages=n_pages, max_chunk=n)
    g = torch.Generator(device="cuda").manual_seed(34)
    c.block_table.copy_(torch.arange(n_pages - 1, n_pages - 6, -1, dtype=torch.int32)[None])
    assert c.stage_base * 512 > 1 << 31
    hi = c.comp_base + (n_pages - 5) * 64
    c.kv_pool[hi:] = torch.randn(c.kv_pool[hi:].shape, generator=g, device="cuda").to(torch.bfloat16)
    c.kv_pool[:W] = torch.randn(W, D, generator=g, device="cuda").to(torch.bfloat16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cu, st = i32(0, n), i32(s)
    kv, sc = (torch.randn(n, 1024, generator=g, device="cuda") for _ in range(2))
    ape, nw, f = torch.randn(4, 1024, generator=g, device="cuda"), torch.ones(512, device="cuda"), _freqs().cuda()
    low, rings = torch.zeros(260, 512, dtype=torch.bfloat16, device="cuda"), []
    for out, base, table in ((c.kv_pool, c.comp_base, c.block_table), (low, 0, None)):
        rings.append((torch.zeros(1, 8, 1024, device="cuda"), torch.zeros(1, 8, 1024, device="cuda")))
        pkg.compressor_chunk((kv, sc), cu, st, ape, nw, *rings[-1], out, 260, block_table=table, page=64, out_base=base, freqs=f)
    e = torch.arange((s + n) // 4, device="cuda")
    rows = c.comp_rows(0, e)
    new = e[s // 4:]
    assert new.numel() == 2 and torch.equal(c.kv_pool[rows[new]], low[new])
    q = torch.randn(n, H, D, generator=g, device="cuda").to(torch.bfloat16) / 8
    sink = torch.randn(H, generator=g, device="cuda")
    want, tol = _attention64(c, q, sink, [n], [s], [0])
    _check(pkg.chunk_attention(c, q, sink, cu, st, freqs=f), want, tol)
    given = torch.full((n, e.numel()), -1, dtype=torch.int32, device="cuda")
    for i in range(n):
        given[i, :(s + i + 1) // 4] = rows[:(s + i + 1) // 4].to(torch.int32)
    _check(pkg.chunk_attention(c, q, sink, cu, st, rows=given, freqs=f), want, tol)
    pkg.chunk_commit(c, cu, st, n)
    assert torch.equal(c.kv_pool[[(s + i) % W for i in range(n)]], c.kv_pool[c.stage_base:])
    assert L.device_error() == 0


BAD = [dict(start=-1), dict(start=2 ** 31 - 5), dict(start=2 ** 31 - 1), dict(slot=9), dict(slot=-1), dict(end=99)]


@pytest.mark.parametrize("bad", BAD)
def test_sequences_that_are_not_valid_are_reported_and_left_out(bad):
    """The first sequence is a good one: it comes out as if alone, and nothing of the second is written."""
    pkg, _, L = _mods()
    lens, start = [5, 12], [601, 8]
    c, q, sink, cu, st, sq = _case(lens, start, seed=35)
    f, (want, tol) = _freqs().cuda(), _attention64(c, q, sink, lens, start, range(2))
    st[1], sq[1], cu[2] = bad.get("start", 8), bad.get("slot", 1), bad.get("end", 17)
    pos, _ = pkg.chunk_rows(c, cu, st, 17, sq)
    assert L.device_error() == 4
    assert pos.tolist() == list(range(601, 606)) + [0] * 12
    for rows in (None, torch.full((17, 1), -1, dtype=torch.int32, device="cuda")):
        o = pkg.chunk_attention(c, q, sink, cu, st, seqs=sq, rows=rows, freqs=f)
        assert L.device_error() == 4
        if rows is None:
            _check(o[:5], want[:5], tol[:5])
    for total in (17, 4 * 4000):   # few tokens and long chunks take different kernels
        kv = torch.randn(total, 1024, device="cuda")
        ape, nw = torch.zeros(4, 1024, device="cuda"), torch.ones(512, device="cuda")
        rings = [torch.zeros(2, 8, 1024, device="cuda") for _ in range(2)]
        out = torch.zeros(2 * 5000, 512, device="cuda")
        cu2, st2 = cu.clone(), st.clone()
        cu2[2], st2[0] = total + 7 if "end" in bad else total, 1
        pkg.compressor_chunk((kv, kv), cu2, st2, ape, nw, *rings, out, 5000, seqs=sq, freqs=f)
        assert L.device_error() == 4
        assert out[0].any() and not out[1:].any() and not rings[0][1].any() and not rings[1][1].any()
    before = c.kv_pool.clone()
    pkg.chunk_commit(c, cu, st, 17, sq)
    assert L.device_error() == 4
    for i in range(5):
        before[(601 + i) % W] = before[c.stage_base + i]
    assert torch.equal(c.kv_pool, before)


def test_a_slot_named_twice():
    """Reading it twice is a call like any other; the ring takes the first, and the second is reported. Empty
    sequences (a batch padded to a fixed number of them) name what they like."""
    pkg, _, L = _mods()
    lens, start = [3, 2], [300, 300]
    c, q, sink, cu, st, sq = _case(lens, start, seed=36, seqs=[1, 1], slots=2)
    _check(pkg.chunk_attention(c, q, sink, cu, st, seqs=sq, freqs=_freqs().cuda()), *_attention64(c, q, sink, lens, start, [1, 1]))
    assert L.device_error() == 0
    before = c.kv_pool.clone()
    pkg.chunk_commit(c, cu, st, 5, sq)
    assert L.device_error() == 4
    for i in range(3):
        before[W + (300 + i) % W] = before[c.stage_base + i]
    assert torch.equal(c.kv_pool, before)
    kv = torch.randn(5, 1024, device="cuda")
    ape, nw, out = torch.zeros(4, 1024, device="cuda"), torch.ones(512, device="cuda"), torch.zeros(200, 512, device="cuda")
    rings = [torch.zeros(2, 8, 1024, device="cuda") for _ in range(2)]
    pkg.compressor_chunk((kv, kv), cu, st, ape, nw, *rings, out, 100, seqs=sq)
    assert L.device_error() == 4
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cu, st, sq = i32(0, 3, 3, 3, 5), i32(300, 0, 0, 300), i32(1, 1, 0, 0)
    pkg.chunk_commit(c, cu, st, 5, sq)
    pkg.compressor_chunk((kv, kv), cu, st, ape, nw, *rings, out, 100, seqs=sq)
    assert L.device_error() == 0


def test_chunk_ops_compile_as_one_graph():
    """Traced whole (a graph break raises), the compressor writing what the attention then reads: the eager bits."""
    import torch._dynamo
    torch._dynamo.reset()
    pkg, _, L = _mods()
    lens, start = [9, 6], [400, 31]
    c, q, sink, cu, st, _ = _case(lens, start, seed=37, paged=True)
    g = torch.Generator(device="cuda").manual_seed(38)
    kv, sc = (torch.randn(15, 1024, generator=g, device="cuda") for _ in range(2))
    ape, nw, f = torch.randn(4, 1024, generator=g, device="cuda"), torch.ones(512, device="cuda"), _freqs().cuda()

    def run(c, kv, sc, q, sink, cu, st):
        pkg.compressor_chunk((kv, sc), cu, st, ape, nw, c.ring_kv, c.ring_score, c.kv_pool, c.max_comp,
                             block_table=c.block_table, page=c.page, out_base=c.comp_base, freqs=f)
        return pkg.chunk_attention(c, q, sink, cu, st, freqs=f)

    other = c.clone()
    want = run(c, kv, sc, q, sink, cu, st)
    got = torch.compile(run, fullgraph=True, backend="aot_eager")(other, kv, sc, q, sink, cu, st)
    assert torch.equal(got, want) and torch.equal(other.kv_pool, c.kv_pool) and torch.equal(other.ring_kv, c.ring_kv)
    assert L.device_error() == 0


def test_two_graphs_and_an_eager_call_share_nothing():
    """Split attentions have a workspace: two captured graphs replayed on two streams at once, and eager calls
    between, each keep their own."""
    pkg, _, L = _mods()
    lens, start, f = [2], [9000], _freqs().cuda()
    cases = [_case(lens, start, seed=40 + i) for i in range(3)]
    wants = [pkg.chunk_attention(c, q, sink, cu, st, freqs=f) for c, q, sink, cu, st, _ in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c, q, sink, cu, st, _ in cases[:2]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(pkg.chunk_attention(c, q, sink, cu, st, freqs=f))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for gr, sm in zip(graphs, streams):
            with torch.cuda.stream(sm):
                gr.replay()
        c, q, sink, cu, st, _ = cases[2]
        assert torch.equal(pkg.chunk_attention(c, q, sink, cu, st, freqs=f), wants[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1], wants[1])
    assert L.device_error() == 0


def test_extend_by_nothing():
    blk, _, dims, _ = _block(4, 2, 256, 512, n_pages=3, max_chunk=8)
    before = {k: v.clone() for k, v in blk.cache.state_dict().items()}
    for x, lengths, start in ((torch.zeros(0, dims.dim, device="cuda"), [], []), (torch.zeros(3, dims.dim, device="cuda"), [0, 0], [4, 9])):
        assert blk.extend(x, lengths, start).shape == x.shape
    for k, v in blk.cache.state_dict().items():
        assert torch.equal(v, before[k]), k


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("window", [False, True])
def test_listed_rows_that_are_masked_may_hold_anything(dtype, window):
    """The gathered kernel: row 0 of the pool and the rows that no list names hold no numbers, and masked entries
    stand everywhere in the lists."""
    S = importlib.import_module(PKG + ".sparse_attn")
    _, _, L = _mods()
    g = torch.Generator(device="cuda").manual_seed(50)
    n, s, t = 900, 20, 300
    pool = torch.randn(n, D, generator=g, device="cuda").to(torch.bfloat16)
    idx = torch.randint(200, n, (s, t), generator=g, device="cuda")
    idx[torch.rand(s, t, generator=g, device="cuda") < 0.4] = -1
    idx[3], idx[4, :200] = -1, -1
    idx[3, 299] = 777
    named = torch.zeros(n, dtype=torch.bool, device="cuda")
    named[idx[idx >= 0]] = True
    pos = torch.arange(20, 20 + s, dtype=torch.int32, device="cuda")
    if window:
        named[1:129] = True                     # the ring's rows 1 ..
    pool[~named] = torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda").to(torch.bfloat16)[
        torch.arange(int((~named).sum()), device="cuda") % 3][:, None]
    q = torch.randn(s, H, D, generator=g, device="cuda").to(torch.bfloat16) / 4
    sink, f = torch.randn(H, generator=g, device="cuda"), _freqs().cuda()
    out = torch.empty(s, H, D, dtype=torch.bfloat16, device="cuda")
    kw = dict(window=128, win_base=torch.ones(s, dtype=torch.int64, device="cuda")) if window else {}
    S.sparse_attn_into(out, q, pool, sink, idx.to(dtype), D ** -0.5, f, pos, 64, kernel=2, **kw)
    assert L.device_error() == 0
    kv, want, tol = pool.double(), [], []
    for i in range(s):
        r = idx[i][idx[i] >= 0]
        if window:
            r = torch.cat([1 + torch.arange(int(pos[i]) + 1, device="cuda"), r])
        x = torch.cat([q[i].double() @ kv[r].T * D ** -0.5, sink.double()[:, None]], 1)
        w = torch.softmax(x, -1)[:, :-1]
        a = w @ kv[r].abs()
        a[:, -64:] = a[:, -64:] + a[:, -64:].reshape(H, 32, 2).flip(-1).reshape(H, 64)
        want.append(_rotate64((w @ kv[r])[None], pos[i:i + 1], f, -1)[0])
        tol.append(4 * EPS * a)
    _check(out, torch.stack(want), torch.stack(tol))


def test_a_replay_takes_what_its_tensors_then_hold():
    """Lengths, positions, slots and the table are read on the device: one captured chunk serves others that fit."""
    pkg, _, L = _mods()
    c, q, sink, cu, st, sq = _case([5, 3], [900, 40], seed=51, seqs=[1, 0], slots=3, pad=2)
    f = _freqs().cuda()
    pkg.chunk_attention(c, q, sink, cu, st, seqs=sq, freqs=f)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        pos, rows = pkg.chunk_rows(c, cu, st, 10, sq)
        o = pkg.chunk_attention(c, q, sink, cu, st, seqs=sq, freqs=f)
    for lens, start, seqs in (([5, 3], [900, 40], [1, 0]), ([1, 9], [700, 3], [2, 1]), ([0, 4], [5, 0], [0, 2]), ([10, 0], [333, 1], [0, 0])):
        cu.copy_(torch.tensor([0, lens[0], sum(lens)])), st.copy_(torch.tensor(start)), sq.copy_(torch.tensor(seqs))
        gr.replay()
        assert L.device_error() == 0
        assert pos.tolist() == [p + i for n, p in zip(lens, start) for i in range(n)] + [0] * (10 - sum(lens))
        _check(o, *_attention64(c, q, sink, lens, start, seqs))


@pytest.mark.parametrize("quant,act_quant", [(True, False), (False, True), (True, True)])
def test_extend_with_8_bit_weights_and_quantised_rows(quant, act_quant):
    """Chunks above and below the 64 tokens at which the projections change kernels."""
    Lm, C = importlib.import_module(PKG + ".layer"), importlib.import_module(PKG + ".configs")
    _, _, L = _mods()
    dims = C.LayerDims(ratio=4)
    Wt = Lm.make_attention_weights(70, dims=dims, quant=quant).to("cuda")
    a = Lm.DecodeBlock(Wt, 2, 256, dims=dims, act_quant=act_quant, max_chunk=80, n_pages=8)
    b = Lm.DecodeBlock(Wt, 2, 256, dims=dims, act_quant=act_quant)
    x = torch.randn(2, 80, 4096, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    got = [torch.cat([a.extend(x[0, :75], [75], [0]), a.extend(x[0, 75:], [5], [75])]), a.extend(x[1], [80], [0], seqs=[1])]
    ref = torch.stack([b.step(x[:, p], torch.full((2,), p, dtype=torch.int32, device="cuda")) for p in range(80)], 1)
    assert L.device_error() == 0
    for s in range(2):
        # a cached row that an fp32 sum in another order moves across a border of its 4-bit grid moves by a step, 2^-3 of
        # its value (e4m3); the rows are a mean over the list, so few of those show in an output
        assert rel_rms(got[s], ref[s]) <= (2 if act_quant else 1) * BLOCK_REL


def test_a_conversation_with_branches():
    """A prompt in chunks, branches of it that each go their own way while pages move, drafts on a branch that are
    dropped, and the same tokens one at a time on fixed caches."""
    pkg, _, L = _mods()
    a, Wt, dims, Lm = _block(4, 4, 512, 512, max_chunk=200, page=16, n_pages=24)
    c = a.cache
    g = torch.Generator(device="cuda").manual_seed(7)
    prompt, ways, drafts = (torch.randn(n, 4096, generator=g, device="cuda") for n in (190, 90, 6))
    outs = {0: [a.extend(prompt[:101], [101], [0]), a.extend(prompt[101:], [89], [101])]}
    c.fork([0, 0], [2, 3], [190, 190])
    a.extend(drafts, [6], [190], seqs=[3])                   # not taken: the branch is given back
    c.free([3])
    c.fork([2], [3], [190])
    o = a.extend(torch.cat([ways[:33], ways[40:50], ways[60:61]]), [33, 10, 1], [190, 190, 190], seqs=[0, 2, 3])
    outs[0].append(o[:33]), outs.update({2: [o[33:43]], 3: [o[43:]]})
    c.free([0])                                              # the branches keep the shared pages
    live = int(c.compact())
    assert live == int((c.page_refs > 0).sum()) and (c.page_refs[:live] > 0).all()
    o = a.extend(torch.cat([ways[50:60], ways[61:90]]), [10, 29], [200, 191], seqs=[2, 3])
    outs[2].append(o[:10]), outs[3].append(o[10:])
    assert L.device_error() == 0
    for s, own in ((0, ways[:33]), (2, ways[40:60]), (3, ways[60:90])):
        b, _, _, _ = _block(4, 1, 512, 512, page=16)
        x = torch.cat([prompt, own])
        ref = torch.cat([b.step(x[p:p + 1], torch.tensor([p], dtype=torch.int32, device="cuda")) for p in range(x.shape[0])])
        got = torch.cat(outs[s]) if s == 0 else torch.cat([torch.cat(outs[0])[:190], *outs[s]])
        assert rel_rms(got, ref) <= BLOCK_REL, s
        assert rel_rms(got[190:], ref[190:]) <= BLOCK_REL, s


@pytest.mark.parametrize("lens,start", [([151], [9000]), ([301], [4100]), ([2] * 80, [3000] * 80), ([1] * 76, list(range(2900, 2976))),
                                        ([1, 0, 3] * 30, [4000, 7, 3900] * 30), ([40, 1, 120], [6000, 5, 2500])])
def test_chunk_attention_a_little_more_than_a_round(lens, start):
    """A few pairs of tokens more than the clusters take in whole rounds, and fewer in a replay's lengths."""
    pkg, _, L = _mods()
    c, q, sink, cu, st, _ = _case(lens, start, seed=60, page=32)
    want, tol = _attention64(c, q, sink, lens, start, range(len(lens)))
    for dtype in (torch.bfloat16, torch.float32):
        _check(pkg.chunk_attention(c, q, sink, cu, st, freqs=_freqs().cuda(), out_dtype=dtype), want, tol)
    assert L.device_error() == 0
    # lengths that a replay may find: fewer pairs than clusters, or none
    for keep in (5, 0):
        few = torch.clamp(cu, max=keep)
        o = pkg.chunk_attention(c, q, sink, few, st, freqs=_freqs().cuda())
        if keep:
            n = [int(b - a) for a, b in zip(few[:-1], few[1:])]
            _check(o[:keep], *[x[:keep] for x in _attention64(c, q, sink, n, start, range(len(n)))])
    assert L.device_error() == 0
