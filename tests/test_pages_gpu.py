"""Pages of a paged cache against a plain model on the host: tables, counts and every copied byte are
whole numbers or copies, so everything is compared for equality."""
import importlib
import random

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
PKG = "deepseek-v4-flash-mlx_b200"
W, R = 128, 4
NO_PAGES, OUT_OF_RANGE = 7, 4


def _mods():
    return importlib.import_module(PKG), importlib.import_module(PKG + ".decode"), importlib.import_module(PKG + "._lib")


def _cache(slots, max_comp, page, n_pages, seed=0, fill=True):
    _, Dm, _ = _mods()
    c = Dm.SparseMLACache(slots, max_comp, page=page, n_pages=n_pages, max_chunk=4)
    if fill:
        g = torch.Generator(device="cuda").manual_seed(seed)
        for t in (c.kv_pool, c.k_idx, c.ring_kv, c.ring_score, c.ring_k_idx, c.ring_s_idx, c.key_image[1], c.key_image[2]):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda").to(t.dtype))
        c.key_image[0].copy_(torch.randint(0, 256, c.key_image[0].shape, generator=g, device="cuda", dtype=torch.uint8))
    return c


class Model:
    """The same in lists and numpy arrays."""

    def __init__(self, c):
        self.c = c
        self.table = c.block_table.cpu().numpy().copy()
        self.refs = c.page_refs.cpu().numpy().copy()
        self.st = {k: v.cpu() for k, v in c.state_dict().items() if k not in ("block_table", "page_refs", "meta", "win_base")}
        self.st = {k: v.view(torch.int16).numpy().copy() if v.dtype == torch.bfloat16 else v.numpy().copy() for k, v in self.st.items()}

    def lowest(self, n):
        free = np.flatnonzero(self.refs == 0)
        return free[:n] if len(free) >= n else None

    def free(self, seqs):
        for s in seqs:
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s] = -1

    def reserve(self, seqs, tokens):
        ok, took = True, []
        start = self.refs.copy()
        free = list(np.flatnonzero(start == 0))
        asked = 0
        for s, t in zip(seqs, tokens):
            need = -(-min(t // R, self.c.max_comp) // self.c.page) - int((self.table[s] >= 0).sum())
            if need <= 0:
                continue
            have = int((self.table[s] >= 0).sum())
            if asked + need > len(free):
                ok = False
            else:
                for j in range(need):
                    self.table[s, have + j] = free[asked + j]
                    self.refs[free[asked + j]] = 1
            asked += need
        return ok

    def pages(self):
        return self.st["kv_pool"][self.c.comp_base:self.c.stage_base].reshape(len(self.refs), self.c.page, -1)

    def fork(self, src, dst, tokens):
        free, used = list(np.flatnonzero(self.refs == 0)), 0
        for a, b, t in zip(src, dst, tokens):
            e, page = t // R, self.c.page
            self.table[b, :e // page] = self.table[a, :e // page]
            self.refs[self.table[a, :e // page]] += 1
            if e % page:
                new = free[used]
                used += 1
                self.refs[new], self.table[b, e // page] = 1, new
                self.pages()[new, :e % page] = self.pages()[self.table[a, e // page], :e % page]
            self.st["kv_pool"][b * W:(b + 1) * W] = self.st["kv_pool"][a * W:(a + 1) * W]
            for r in ("ring_kv", "ring_score", "ring_k_idx", "ring_s_idx"):
                self.st[r][b] = self.st[r][a]
            tiles = -(-e // 128)
            self.st["k_idx"][b, :e] = self.st["k_idx"][a, :e]
            img = self.st["key_image.0"].reshape(self.c.batch, -1)
            img[b, :tiles * 65536] = img[a, :tiles * 65536]
            self.st["key_image.1"][b, :tiles * 128] = self.st["key_image.1"][a, :tiles * 128]
            self.st["key_image.2"][b] = self.st["key_image.2"][a]

    def compact(self):
        n = int((self.refs > 0).sum())
        holes = [i for i in range(n) if self.refs[i] == 0]
        movers = [i for i in range(n, len(self.refs)) if self.refs[i] > 0]
        for a, b in zip(movers, holes):
            self.pages()[b] = self.pages()[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.table[self.table == a] = b
        return n

    def check(self):
        c = self.c
        assert (c.block_table.cpu().numpy() == self.table).all()
        assert (c.page_refs.cpu().numpy() == self.refs).all()
        for k, v in c.state_dict().items():
            if k in self.st:
                got = v.cpu()
                got = got.view(torch.int16).numpy() if got.dtype == torch.bfloat16 else got.numpy()
                assert (got == self.st[k]).all(), k


@pytest.mark.parametrize("page,n_pages,slots,max_comp", [(64, 40, 6, 500), (16, 97, 5, 333), (8, 1500, 9, 1024), (100, 7, 3, 250)])
def test_random_life_of_a_pool(page, n_pages, slots, max_comp):
    """Sequences grow, branch, leave and are compacted, in random order; then the empty pool."""
    _, _, L = _mods()
    c = _cache(slots, max_comp, page, n_pages, seed=page)
    m, rng = Model(c), random.Random(page)
    held = [0] * slots
    for _ in range(40):
        op = rng.choice(["reserve", "fork", "free", "compact", "reserve"])
        if op == "reserve":
            seqs = rng.sample(range(slots), rng.randint(1, slots))
            tokens = [min(held[s] + rng.choice([0, 1, 3, 4, 37, 400]), max_comp * R + 3) for s in seqs]
            c.reserve(torch.tensor(seqs, device="cuda"), torch.tensor(tokens, device="cuda"))
            ok = m.reserve(seqs, tokens)
            assert L.device_error() == (0 if ok else NO_PAGES)
            for s, t in zip(seqs, tokens):
                if (m.table[s] >= 0).sum() * page >= t // R:
                    held[s] = max(held[s], t)
        elif op == "fork":
            empty = [s for s in range(slots) if (m.table[s] < 0).all()]
            full = [s for s in range(slots) if s not in empty]
            if not full or not empty:
                continue
            dst = rng.sample(empty, rng.randint(1, len(empty)))
            src = [rng.choice(full) for _ in dst]
            tokens = [held[s] for s in src]
            if len(dst) > (m.refs == 0).sum():
                continue
            c.fork(src, dst, tokens)
            m.fork(src, dst, tokens)
            assert L.device_error() == 0
            for s, t in zip(dst, tokens):
                held[s] = t
        elif op == "free":
            seqs = rng.sample(range(slots), rng.randint(1, 2))
            c.free(seqs + seqs[:1])    # the first one twice
            m.free(seqs)
            for s in seqs:
                held[s] = 0
        else:
            n = c.compact()
            assert n.item() == m.compact()
        m.check()
    c.free(list(range(slots)))
    m.free(range(slots))
    assert c.compact().item() == 0 == m.compact()
    m.check()
    assert (c.page_refs == 0).all()


def test_fork_shares_and_separates():
    """A branch and its source go on apart: what one writes, the other does not see; shared pages go free
    with their last holder."""
    _, _, L = _mods()
    c = _cache(4, 200, 16, 40, seed=1)
    c.reserve([0], [4 * 37])
    c.fork([0, 0], [1, 3], [4 * 37, 4 * 37])
    t = c.block_table.cpu()
    assert t[0, :2].tolist() == t[1, :2].tolist() == t[3, :2].tolist() == [0, 1]
    assert sorted([t[0, 2].item(), t[1, 2].item(), t[3, 2].item()]) == [2, 3, 4] and (t[:, 3:] == -1).all()
    assert c.page_refs[:6].tolist() == [3, 3, 1, 1, 1, 0]
    c.reserve([1], [4 * 49])
    before = c.kv_pool.clone()
    c.kv_pool[c.comp_rows(1, torch.arange(37, 49, device="cuda"))] = 7.0
    for s in (0, 3):
        rows = c.comp_rows(s, torch.arange(37, device="cuda"))
        assert torch.equal(c.kv_pool[rows], before[rows])
    c.free([0])
    c.free([3])
    assert c.page_refs[:6].tolist() == [1, 1, 0, 1, 0, 1] and L.device_error() == 0
    assert torch.equal(c.kv_pool[c.comp_rows(1, torch.arange(37, device="cuda"))], before[c.comp_rows(1, torch.arange(37, device="cuda"))])


def test_what_cannot_be_done_is_reported_and_left_out():
    _, _, L = _mods()
    c = _cache(4, 64, 16, 6, seed=2)
    c.reserve([0, 1], [4 * 33, 4 * 20])             # 3 + 2 of 6 pages
    state = lambda: (c.block_table.clone(), c.page_refs.clone(), c.kv_pool.clone(), c.k_idx.clone())  # noqa: E731
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    was = state()
    for src, dst, tokens, code in (([0], [1], [132], OUT_OF_RANGE), ([0], [0], [132], OUT_OF_RANGE), ([0], [4], [132], OUT_OF_RANGE),
                                   ([-1], [2], [4], OUT_OF_RANGE), ([0], [2], [4 * 65], OUT_OF_RANGE), ([0], [2], [4 * 49], OUT_OF_RANGE),
                                   ([0], [2], [-4], OUT_OF_RANGE), ([2], [3], [4], OUT_OF_RANGE)):
        c.fork(src, dst, tokens)
        assert L.device_error() == code and same(was, state()), (src, dst, tokens)
    c.fork([0, 1], [2, 3], [132, 80])               # one page left for two last pages
    assert L.device_error() == NO_PAGES
    assert c.block_table[2, :3].tolist() == [0, 1, 5] and (c.block_table[3] == -1).all() and c.page_refs.tolist() == [2, 2, 1, 1, 1, 1]
    was = state()
    c.reserve([3], [4])
    assert L.device_error() == NO_PAGES and same(was, state())
    c.reserve([7], [4])
    assert L.device_error() == OUT_OF_RANGE and same(was, state())
    c.free([9, -1])
    assert L.device_error() == OUT_OF_RANGE and same(was, state())
    c.fork([0, 2], [3, 3], [128, 128])              # the same slot twice: the first branch alone
    assert L.device_error() == OUT_OF_RANGE and c.block_table[3].tolist() == [0, 1, -1, -1]
    with pytest.raises(ValueError):
        c.fork([0], [1, 2], [4])
    with pytest.raises(TypeError):
        c.free(torch.zeros(1, device="cuda"))
    with pytest.raises(RuntimeError):
        c.free(torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):
        c.reserve(None, [4] * 5)
    c.free([]), c.reserve([], []), c.fork([], [], [])
    assert L.device_error() == 0


def test_captured_and_two_streams():
    """A beam step (give up the branches, branch again) captured and replayed; two caches on two streams."""
    _, _, L = _mods()
    c = _cache(3, 300, 16, 80, seed=3)
    c.reserve([0], [4 * 77])
    dst, src, tok = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([1, 2], [0, 0], [4 * 77 + 2] * 2))
    c.fork(src, dst, tok)
    m = Model(c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.free(dst)
        c.fork(src, dst, tok)
    c.kv_pool[c.comp_rows(0, torch.arange(64, 77, device="cuda"))] = 3.0
    c.k_idx[0] += 1
    m = Model(c)
    m.free([1, 2])
    m.fork([0, 0], [1, 2], [4 * 77 + 2] * 2)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    m.check()
    a, b = _cache(3, 300, 16, 80, seed=4), _cache(3, 300, 16, 80, seed=5)
    for k in (a, b):
        k.reserve([0], [4 * 290])
    ma, mb = Model(a), Model(b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        for s, k in ((s1, a), (s2, b)):
            with torch.cuda.stream(s):
                k.fork([0, 0], [1, 2], [4 * 290] * 2)
                k.free([1])
                k.compact()
                k.free([2])
    torch.cuda.synchronize()
    for mod in (ma, mb):
        for _ in range(5):
            mod.fork([0, 0], [1, 2], [4 * 290] * 2)
            mod.free([1])
            mod.compact()
            mod.free([2])
        mod.check()
    assert L.device_error() == 0


@pytest.mark.parametrize("n_pages", [1, 1023, 1024, 1025, 70001])
def test_large_pools(n_pages):
    """Compaction and reservation over more pages than a planning block has threads."""
    _, Dm, L = _mods()
    c = Dm.SparseMLACache(1, 64, page=1, n_pages=n_pages, head_dim=8)
    live = np.random.default_rng(n_pages).random(n_pages) < 0.5
    c.page_refs.copy_(torch.from_numpy(live.astype(np.int32)))
    c.kv_pool.copy_(torch.randn(c.kv_pool.shape, device="cuda").to(torch.bfloat16))
    pages = c.kv_pool[c.comp_base:].clone()
    n = int(live.sum())
    holes, movers = np.flatnonzero(~live[:n]), n + np.flatnonzero(live[n:])
    pages[torch.from_numpy(holes).cuda()] = pages[torch.from_numpy(movers).cuda()]
    assert c.compact().item() == n
    assert torch.equal(c.kv_pool[c.comp_base:], pages)
    assert (c.page_refs[:n] == 1).all() and (c.page_refs[n:] == 0).all()
    c.reserve([0], [4 * min(64, n_pages - n)])
    assert L.device_error() == 0
    k = min(64, n_pages - n)
    assert c.block_table[0, :k].tolist() == list(range(n, n + k))


def test_step_on_a_paged_cache():
    """Decode steps of a block over a paged cache equal those over a fixed one; a branch decodes on as its
    source would; without pages left the step reports it and stores no row."""
    Lm, C = importlib.import_module(PKG + ".layer"), importlib.import_module(PKG + ".configs")
    _, _, L = _mods()
    Wt = Lm.make_attention_weights(60).to("cuda")
    fixed, paged = Lm.DecodeBlock(Wt, 2, 256, page=16), Lm.DecodeBlock(Wt, 2, 256, page=16, n_pages=6)
    x = torch.randn(40, 2, 4096, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    pos = lambda p: torch.full((2,), p, dtype=torch.int32, device="cuda")  # noqa: E731
    for p in range(30):
        assert torch.equal(fixed.step(x[p], pos(p)), paged.step(x[p], pos(p)))
    assert L.device_error() == 0
    c = paged.cache
    c.free([1])
    c.fork([0], [1], [30])
    both = paged.step(x[30, :1].expand(2, -1).contiguous(), pos(30))
    assert torch.equal(both[0], both[1])
    assert torch.equal(both[0], fixed.step(x[30, :1].expand(2, -1).contiguous(), pos(30))[0])
    c.page_refs[c.page_refs == 0] = 1    # nothing left
    pool = c.kv_pool[c.comp_base:].clone()
    for p in range(31, 70):
        paged.step(x[p % 40], pos(p))
    assert L.device_error() in (NO_PAGES, OUT_OF_RANGE)
    e = torch.arange(16, 17, device="cuda")
    assert c.block_table[0, 1] == -1 and c.block_table[1, 1] == -1
    other = torch.ones(pool.shape[0], dtype=torch.bool, device="cuda")
    for s in range(2):
        other[c.comp_rows(s, torch.arange(16, device="cuda")) - c.comp_base] = False
    assert torch.equal(c.kv_pool[c.comp_base:][other], pool[other])


def test_branches_of_a_window_only_cache():
    """No pages: a branch is a copy of the window ring; handing out, giving back and compacting do nothing."""
    pkg, Dm, L = _mods()
    c = Dm.SparseMLACache(4, 0, n_pages=3, max_chunk=2)
    c.kv_pool.copy_(torch.randn(c.kv_pool.shape, device="cuda").to(torch.bfloat16))
    want = c.kv_pool.clone()
    c.reserve([0, 1], [1000, 5])
    c.free([3])
    assert c.compact().item() == 0 and torch.equal(c.kv_pool, want)
    c.fork([0, 0], [1, 3], [5000, 7])
    want[W:2 * W] = want[:W]
    want[3 * W:4 * W] = want[:W]
    assert torch.equal(c.kv_pool, want) and L.device_error() == 0
    c.fork([0], [4], [1])
    assert torch.equal(c.kv_pool, want) and L.device_error() == OUT_OF_RANGE


def test_reserve_at_the_ends():
    """More sequences than the planning CTA has threads, a slot named again in the next thousand, counts at the
    end of their type."""
    pkg, Dm, L = _mods()
    c = Dm.SparseMLACache(1100, 8, window=64, page=8, n_pages=1101, idx_dim=128)
    order = list(np.random.default_rng(3).permutation(1100)) + [7, 8]
    c.reserve([int(s) for s in order], [32] * 1102)
    assert L.device_error() == 0
    assert c.block_table[order[:1100], 0].tolist() == list(range(1100))
    assert c.page_refs.tolist() == [1] * 1100 + [0]
    c.free([5])
    c.reserve([5], [2 ** 31 - 1], add=2 ** 31 - 1)   # past the cache: all that it has, and the error word
    assert L.device_error() == OUT_OF_RANGE and int(c.block_table[5, 0]) >= 0
    c.free([5])
    c.reserve([5], [-2 ** 31], add=-2 ** 31)
    c.reserve([5], [-8], add=7)
    assert L.device_error() == 0 and int(c.block_table[5, 0]) == -1


def test_compact_with_a_cell_that_is_not_counted():
    """A table that names a page nobody counted (not one that these calls leave): the cell is emptied."""
    pkg, Dm, L = _mods()
    c = _cache(3, 128, 64, 6)
    c.reserve([0, 1], [512, 256])
    c.free([0])
    c.block_table[2, 0] = 5
    assert c.compact().item() == 1
    assert c.block_table.tolist() == [[-1, -1], [0, -1], [-1, -1]] and c.page_refs.tolist() == [1, 0, 0, 0, 0, 0]
    assert L.device_error() == 0


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("n_keys,page", [(300, 8), (300, 64), (5000, 64), (20000, 8), (20000, 256)])
def test_selection_leaves_out_keys_without_a_page(n_keys, page, rows):
    """Every visible key selected: those on pages that the sequence has, mapped to their rows, and -1 for the
    others (a cache that ran out of pages may hold keys whose rows were never stored)."""
    I = importlib.import_module(PKG + ".indexer")  # noqa: E741
    _, _, L = _mods()
    g = torch.Generator(device="cuda").manual_seed(n_keys + page)
    q, w = torch.randn(1, rows, 64, 128, generator=g, device="cuda"), torch.randn(1, rows, 64, generator=g, device="cuda")
    k = torch.randn(1, n_keys, 128, generator=g, device="cuda")
    pages = -(-n_keys // page)
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table[torch.rand(pages, generator=g, device="cuda") < 0.3] = -1
    pos = torch.full((1, rows), 4 * n_keys, dtype=torch.int32, device="cuda")
    out = torch.empty(1, rows, n_keys, dtype=torch.int32, device="cuda")
    I.indexer_topk_into(out, q, w, k, n_keys, positions=pos, ratio=4, out_offset=1000, block_table=table[None], page=page)
    j = torch.arange(n_keys, device="cuda")
    pg = table[j // page]
    want = torch.where(pg >= 0, 1000 + pg * page + (j % page).to(torch.int32), -1).sort().values.to(torch.int32)
    assert torch.equal(out[0].sort(-1).values, want.expand(rows, -1)) and L.device_error() == 0


def test_forks_of_one_source_at_several_lengths():
    """More branches than a warp looks at together, some of the same rows (read once for all), some shorter, some
    refused."""
    c = _cache(45, 96, 16, 200, seed=9)
    c.reserve([0, 1], [384, 200])
    m = Model(c)
    src = [0 if k % 3 else 1 for k in range(40)]
    tokens = [200 if s == 1 else (384, 100, 131, 64)[k % 4] for k, s in enumerate(src)]
    dst = list(range(2, 42))
    m.fork(src, dst, tokens)
    at = 20                                   # and one onto a slot that has pages, left out alone
    c.fork(src[:at] + [0] + src[at:], dst[:at] + [1] + dst[at:], tokens[:at] + [384] + tokens[at:])
    assert _mods()[2].device_error() == OUT_OF_RANGE
    m.check()


def test_serving_runner_on_a_paged_cache():
    """The captured step hands out its pages at every replay: the runner's outputs are those of a fixed cache."""
    Lm = importlib.import_module(PKG + ".layer")
    _, _, L = _mods()
    Wt = Lm.make_attention_weights(61).to("cuda")
    runs = [Lm.BlockRunner(Lm.DecodeBlock(Wt, 2, 256, page=8, **kw)) for kw in ({}, dict(n_pages=9))]
    x = torch.randn(90, 2, 4096, generator=torch.Generator().manual_seed(2))
    for p in range(90):
        outs = []
        for r in runs:
            hx, hp = r.host_inputs()
            hx.copy_(x[p]), hp.copy_(torch.tensor([p, p + 40], dtype=torch.int32))
            o = r.step_host()
            r.synchronize()
            outs.append(o.clone())
        assert torch.equal(*outs), p
    assert L.device_error() == 0
    t = runs[1].block.cache.block_table
    assert (t >= 0).sum(1).tolist() == [3, 4]   # 22 and 32 entries


def test_hundreds_of_branches():
    c = _cache(300, 40, 16, 700, seed=10)
    c.reserve([0, 1, 2], [160, 100, 64])
    m = Model(c)
    src, dst = [k % 3 for k in range(270)], list(range(20, 290))
    tokens = [(160, 100, 64)[k] for k in src]
    m.fork(src, dst, tokens)
    c.fork(src, dst, tokens)
    assert _mods()[2].device_error() == 0
    m.check()
