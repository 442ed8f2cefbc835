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


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("how", ["extend", "step", "both"])
def test_a_slot_begins_again(paged, how):
    """A slot that held another conversation starts from position 0 as a slot of a new cache does, bit for bit:
    outputs, compressed rows, keys and rings."""
    Lm = importlib.import_module(PKG + ".layer")
    _, _, L = _mods()
    Wt = Lm.make_attention_weights(90).to("cuda")
    used, new = (Lm.DecodeBlock(Wt, 2, 512, page=16, max_chunk=160, **(dict(n_pages=40) if paged else {})) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(140, 4096, generator=g, device="cuda")
    used.extend(x, [70, 70], [0, 0])                       # both slots, the second in the middle of a block
    new.extend(x[:70], [70], [0])
    if paged:
        used.cache.free([1])
    y, other = torch.randn(41, 4096, generator=g, device="cuda"), torch.randn(41, 4096, generator=g, device="cuda")
    sizes = {"extend": [2, 1, 30, 8], "step": [1] * 41, "both": [3, 1, 1, 33, 1, 1, 1]}[how]
    at = 0
    for n in sizes:
        outs = []
        for blk in (used, new):
            if n == 1:   # a step takes both slots
                outs.append(blk.step(torch.stack([other[at], y[at]]), _i32(70 + at, at))[1])
            else:
                outs.append(blk.extend(y[at:at + n], [n], [at], seqs=[1]))
        assert torch.equal(*outs), at
        at += n
    assert at == 41 and L.device_error() == 0
    a, b, e = used.cache, new.cache, torch.arange(10, device="cuda")
    assert torch.equal(a.kv_pool[a.comp_rows(1, e)], b.kv_pool[b.comp_rows(1, e)])
    assert torch.equal(a.k_idx[1, :10], b.k_idx[1, :10])
    assert torch.equal(a.key_image[1].view(2, -1)[1, :10], b.key_image[1].view(2, -1)[1, :10])
    for name in ("ring_kv", "ring_score", "ring_k_idx", "ring_s_idx"):
        assert torch.equal(getattr(a, name)[1, :5], getattr(b, name)[1, :5]), name


@pytest.mark.parametrize("ratio,d", [(1, 64), (2, 512), (3, 128), (4, 128), (4, 512), (4, 1024), (8, 512)])
def test_the_first_block_has_none_before_it(ratio, d):
    """The row of block 0 is that of an empty ring, whatever the ring holds of a sequence before: steps and chunks."""
    pkg, _, L = _mods()
    g = torch.Generator(device="cuda").manual_seed(ratio)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    n = 2 * ratio + 1
    kv, sc, ape, nw, freqs = rnd(n, 2 * d), rnd(n, 2 * d), rnd(ratio, 2 * d), 1 + 0.1 * rnd(d), rnd(32)
    empty = (torch.zeros(1, 2 * ratio, 2 * d, device="cuda"), torch.full((1, 2 * ratio, 2 * d), -float("inf"), device="cuda"))
    rope, outs = min(64, d), []
    for ring in (empty, (rnd(1, 2 * ratio, 2 * d), 5 * rnd(1, 2 * ratio, 2 * d))):
        for sizes in ([n], [1] * n, [ratio, ratio + 1], [-n]):
            rk, rs = (t.clone() for t in ring)
            out, at = torch.zeros(3, d, device="cuda"), 0
            if sizes[0] < 0:    # one token at a time
                for p in range(n):
                    pkg.compressor_decode_step(rk, None, None, ape, nw, rk, rs, _i32(p), out, torch.tensor([p // ratio], device="cuda"),
                                               head_dim=d, ratio=ratio, rope_head_dim=rope, freqs=freqs, proj=(kv[p:p + 1], sc[p:p + 1]))
            else:
                for m in sizes:
                    pkg.compressor_chunk((kv[at:at + m], sc[at:at + m]), _i32(0, m), _i32(at), ape, nw, rk, rs, out, 3, head_dim=d,
                                         ratio=ratio, rope_head_dim=rope, freqs=freqs)
                    at += m
            outs.append((out, rk[:, :ratio + 1], rs[:, :ratio + 1]))
    assert L.device_error() == 0 and outs[0][0][:2].any(-1).all()
    for o in outs[1:]:
        for x, y in zip(o, outs[0]):
            assert torch.equal(x, y)


def _plain64(q, kv, sink, lists, pos, freqs, scale=512 ** -0.5):
    """Attention of each query over its list of pool rows in 64 bits, and the bound of each element: probabilities and
    output are rounded to bf16, half a step of 2^-8 each, 3 * 2^-8 of the weighted mean of |kv| with the denominator's
    share, and one more for the sums in 32 bits; the rotation adds up the two of a pair."""
    want, tol, eps = [], [], torch.finfo(torch.bfloat16).eps / 2
    for i, rows in enumerate(lists):
        r = torch.tensor([x for x in rows if x >= 0], device="cuda", dtype=torch.long)
        v = kv[r].double()
        w = torch.softmax(torch.cat([q[i].double() @ v.T * scale, sink.double()[:, None]], 1), -1)[:, :-1]
        o, a = w @ v, w @ v.abs()
        t = (pos[i].float() * freqs).double()
        y, x = o.clone(), o[:, -64:].reshape(-1, 32, 2)
        y[:, -64::2] = x[..., 0] * t.cos() + x[..., 1] * t.sin()
        y[:, -63::2] = x[..., 1] * t.cos() - x[..., 0] * t.sin()
        a[:, -64:] += a[:, -64:].reshape(-1, 32, 2).flip(-1).reshape(-1, 64)
        want.append(y), tol.append(4 * eps * a)
    return torch.stack(want), torch.stack(tol)


@pytest.mark.parametrize("kernel,s", [(0, 3), (0, 20), (1, 3), (1, 20), (2, 3), (2, 20), (2, 200), (3, 3)])
@pytest.mark.parametrize("linear", [False, True])
def test_window_rows_past_the_pool(kernel, s, linear):
    """Rows of the implicit window that are no rows of kv are left out, those past its end reported, by every kernel.
    kv lies inside a larger tensor of NaN, so that a row that is read all the same shows."""
    pkg, _, L = _mods()
    g = torch.Generator(device="cuda").manual_seed(s)
    n, window, off, t = 500, 128, 600, 40
    big = torch.full((off + n + 600, 512), float("nan"), device="cuda", dtype=torch.bfloat16)
    kv = big[off:off + n]
    kv.copy_(torch.randn(n, 512, generator=g, device="cuda"))
    q, sink = torch.randn(s, 64, 512, generator=g, device="cuda").to(torch.bfloat16), torch.randn(64, generator=g, device="cuda")
    freqs = 1.0 / (160000.0 ** (torch.arange(0, 64, 2, dtype=torch.float32, device="cuda") / 64))
    idx = torch.randint(0, n, (s, t), generator=g, device="cuda", dtype=torch.int32)
    # (window base, position): inside; past the end by some rows or all; below 0; the ring not yet full; before position 0
    kinds = [(7, 300, False), (n - 40, 300, True), (n, 300, True), (2 ** 33, 300, True), (-30, 300, False), (-500, 300, False),
             (-2 ** 33, 300, False), (n - 10, 20, True), (n - 10, 9, False), (3, -1, False), (n - 128, 127, False)]
    if linear:
        kinds = [(0, 300, False), (0, n, True), (0, n + 100, True), (0, n + 400, True), (0, 2 ** 30, True), (0, 5, False), (40, n - 41, False),
                 (40, n - 40, True), (-300, 350, False), (-2 ** 33, 350, False), (0, -1, False)]
    for base, p, over in kinds:
        pos = torch.full((s,), p, dtype=torch.int32, device="cuda")
        if linear:
            rows = [base + u for u in range(max(0, p - window + 1), p + 1)]
        else:
            rows = [base + u % window for u in range(max(0, p - window + 1), p + 1)]
        assert any(r >= n for r in rows) == over
        lists = [[r if 0 <= r < n else -1 for r in rows] + idx[i].tolist() for i in range(s)]
        o = pkg.sparse_attn_rope(q, kv, sink, idx, 512 ** -0.5, pos, freqs, win_base=torch.full((s,), base, device="cuda"), window=window,
                                 window_linear=linear, kernel=kernel)
        assert L.device_error() == (4 if over else 0), (base, p)
        want, tol = _plain64(q, kv, sink, lists, pos, freqs)
        assert torch.isfinite(o).all(), (base, p)
        assert ((o.double() - want).abs() <= tol).all(), (base, p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("s,kernel", [(20, 0), (20, 2), (3, 2), (200, 2)])
def test_gathered_attention_into_an_output_at_any_element(dtype, s, kernel):
    """An output that starts at any element of a tensor, and nothing beside it."""
    S = importlib.import_module(PKG + ".sparse_attn")
    _, _, L = _mods()
    g = torch.Generator(device="cuda").manual_seed(s)
    n, t = 700, 300
    kv = torch.randn(n, 512, generator=g, device="cuda").to(torch.bfloat16)
    q, sink = torch.randn(s, 64, 512, generator=g, device="cuda").to(torch.bfloat16), torch.randn(64, generator=g, device="cuda")
    idx = torch.randint(-1, n, (s, t), generator=g, device="cuda", dtype=torch.int32)
    pos = torch.arange(s, dtype=torch.int32, device="cuda")
    freqs = 1.0 / (160000.0 ** (torch.arange(0, 64, 2, dtype=torch.float32, device="cuda") / 64))
    size = s * 64 * 512
    want = S.sparse_attn_into(torch.empty(s, 64, 512, device="cuda", dtype=dtype), q, kv, sink, idx, 512 ** -0.5, freqs, pos, 64,
                              num_splits=1, kernel=2)
    for at in (1, 2, 3, 4):
        all_ = torch.full((size + 8,), 7.0, device="cuda", dtype=dtype)
        out = all_[at:at + size].view(s, 64, 512)
        S.sparse_attn_into(out, q, kv, sink, idx, 512 ** -0.5, freqs, pos, 64, num_splits=1, kernel=kernel)
        assert torch.equal(out, want), at
        assert (all_[:at] == 7).all() and (all_[at + size:] == 7).all()
    assert L.device_error() == 0


def _paged(slots, max_comp, page, n_pages):
    _, Dm, _ = _mods()
    return Dm.SparseMLACache(slots, max_comp, page=page, n_pages=n_pages)


def test_a_reservation_that_cannot_be_met_leaves_the_others_theirs():
    """In the order of the call, each sequence gets its pages if there are as many left; one that finds too few gets
    none, and those behind it are served from what it left."""
    _, _, L = _mods()
    for wants in ([10, 2], [2, 10, 3], [10, 5], [6, 6, 6], [1, 5, 4, 1], [5], [0, 7, 0, 5], [3, 3, 2]):
        c = _paged(len(wants) + 1, 640, 64, 5)
        c.reserve(list(range(len(wants), 0, -1)), [256 * n for n in wants])
        left, table, failed = 5, [[] for _ in range(len(wants) + 1)], False
        for k, n in enumerate(wants):
            if n <= left:
                table[len(wants) - k] = list(range(5 - left, 5 - left + n))
                left -= n
            else:
                failed = True
        assert L.device_error() == (7 if failed else 0), wants
        assert [[int(p) for p in row if p >= 0] for row in c.block_table.tolist()] == table, wants
        assert c.page_refs.tolist() == [1] * (5 - left) + [0] * left, wants
    # over a thousand sequences: the same in every planning batch
    c = _paged(3000, 16, 8, 1500)
    c.reserve(list(range(3000)), [64 if k % 3 == 1 else 32 for k in range(3000)])
    left, at = 1500, []
    for k in range(3000):
        n = 2 if k % 3 == 1 else 1
        at.append(n if n <= left else 0)
        left -= at[-1]
    assert L.device_error() == 7 and left == 0
    assert (c.block_table >= 0).sum(1).tolist() == at and c.page_refs.tolist() == [1] * 1500


def test_a_slot_named_twice_gets_the_pages_of_its_largest_count():
    _, _, L = _mods()
    c = _paged(3, 640, 64, 20)
    c.reserve([0, 1, 0, 2, 0], [4, 256, 1000, 300, 512])
    assert L.device_error() == 0
    assert c.block_table.tolist() == [[0, 1, 2, 3] + [-1] * 6, [4] + [-1] * 9, [5, 6] + [-1] * 8]
    assert c.page_refs.tolist() == [1] * 7 + [0] * 13
    c.reserve([1, 1], [8, 256 * 10], add=0)
    assert (c.block_table[1] >= 0).all() and L.device_error() == 0
    c.free([0, 1, 2])
    # mentions more than a planning batch apart
    big = _paged(1100, 16, 8, 1200)
    big.reserve([7] + list(range(1100)) + [7], [4] + [4] * 1100 + [64])
    assert L.device_error() == 0 and big.block_table[7].tolist() == [0, 1100]


@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("start,n", [(1000, 2), (1002, 2), (1022, 2), (130, 3), (4, 2), (5000, 1), (2047, 64)])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_rows_that_only_one_of_two_tokens_sees(what, start, n, splits):
    """A row that is not finite reaches the tokens that see it and no others: a later draft's row, the entry that a later
    token completes, the ring's row that has left a later token's window; in one dim or in all."""
    pkg, Dm, L = _mods()
    g = torch.Generator(device="cuda").manual_seed(start)
    c = Dm.SparseMLACache(1, (start + n) // 4 + 1, page=16, max_chunk=n)
    c.kv_pool.copy_(torch.randn(c.kv_pool.shape, generator=g, device="cuda"))
    q, sink = torch.randn(n, 64, 512, generator=g, device="cuda").to(torch.bfloat16), torch.randn(64, generator=g, device="cuda")
    call = lambda: pkg.chunk_attention(c, q, sink, _i32(0, n), _i32(start), num_splits=splits)  # noqa: E731
    clean = call()
    assert torch.isfinite(clean).all()
    e = torch.arange((start + n) // 4, device="cuda")
    # (pool row, the first and the last token that see it)
    rows = [(c.stage_base + i, i, n - 1) for i in range(n)]
    rows += [(int(c.comp_rows(0, e[-1])), max(0, 4 * int(e[-1]) + 3 - start), n - 1)]
    if start >= 127:
        rows += [((start - 127) % 128, 0, 0), ((start - 126) % 128, 0, min(1, n - 1))]
    for row, first, last in rows[-5:]:
        for dims in (slice(0, 512), slice(77, 78), slice(300, 301), slice(511, 512)):
            was = c.kv_pool[row].clone()
            c.kv_pool[row, dims] = what
            o = call()
            for i in range(n):
                if first <= i <= last:
                    # every head has it in its score, as NaN or as an infinity; one that scores it -inf weighs it 0 and may
                    # leave it out
                    finite = torch.isfinite(o[i]).all(-1)
                    assert not finite.any() if what != what else not finite.all(), (row, i)
                else:
                    assert torch.equal(o[i], clean[i]), (row, i)
            c.kv_pool[row] = was
    assert torch.equal(call(), clean) and L.device_error() == 0
