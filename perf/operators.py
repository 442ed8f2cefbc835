"""Cases, plain forms and 64-bit values of the operators that extend and manage a paged sparse-MLA cache:

  chunk_attention   attention of a chunk of new tokens per sequence over the cache: each token sees its
                    sliding window (the ring of older rows and the chunk's own rows) and the compressed
                    rows of its paged sequence, all of them or a given list
  compressor_chunk  the KV compressor over a chunk of new tokens, continuing the ring of each sequence
                    and writing the rows it emits through the block table
  fork              a branch of a sequence: full pages shared, the last partial page, the rings and the
                    indexer keys copied
  compact           the pages in use moved to the front of the pool, tables and counts rewritten
"""
import importlib
import math
import random

import torch

own = False

HEADS, DIM, ROPE, WINDOW, RATIO, IDX = 64, 512, 64, 128, 4, 128


def listed():
    return [
        # checking four drafted tokens of each of eight sequences at a short context
        dict(name="attn_verify_8x4_ctx2k", op="chunk_attention", seqs=8, tokens=4, ragged=False, ctx=2048, page=64, top_k=0, ratio=4),
        # one token over every compressed row of a long context
        dict(name="attn_1tok_ctx64k", op="chunk_attention", seqs=1, tokens=1, ragged=False, ctx=65536, page=64, top_k=0, ratio=4),
        # a mixed batch of chunks, down to one token each, small pages
        dict(name="attn_ragged_6_page16", op="chunk_attention", seqs=6, tokens=333, ragged=True, ctx=3001, page=16, top_k=0, ratio=4),
        # a prompt's chunk whose tokens attend to the rows that the indexer listed
        dict(name="attn_listed_1x256_top512", op="chunk_attention", seqs=1, tokens=256, ragged=False, ctx=32768, page=64, top_k=512, ratio=4),
        # a long prompt's chunk: the largest
        dict(name="attn_prefill_1x2048_ctx16k", op="chunk_attention", seqs=1, tokens=2048, ragged=False, ctx=16384, page=64, top_k=0, ratio=4),
        # the compressor behind the drafted tokens, 512-wide rows into pages
        dict(name="comp_verify_8x4", op="compressor_chunk", seqs=8, tokens=4, ragged=False, ctx=2049, page=64, wide=512),
        # the indexer keys' compressor on a mixed batch
        dict(name="comp_keys_ragged_12", op="compressor_chunk", seqs=12, tokens=1501, ragged=True, ctx=7777, page=64, wide=128),
        # the row compressor on a long chunk
        dict(name="comp_rows_2x8192", op="compressor_chunk", seqs=2, tokens=8192, ragged=False, ctx=4095, page=64, wide=512),
        # two branches of a short sequence
        dict(name="fork_1to2_ctx1k", op="fork", sources=1, branches=2, ctx=1003, page=64, spare=32),
        # eight branches of a long one
        dict(name="fork_1to8_ctx64k", op="fork", sources=1, branches=8, ctx=65530, page=64, spare=128),
        # a small pool
        dict(name="compact_96_pages", op="compact", pages=96, page=64, live=0.6),
        # a large pool after most of its sequences have left
        dict(name="compact_8192_pages", op="compact", pages=8192, page=64, live=0.45),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["chunk_attention", "chunk_attention", "compressor_chunk", "fork", "compact"])
    if op == "chunk_attention":
        ratio = rng.choice([4, 4, 4, 0])
        seqs, ctx = _log(rng, 1, 16), _log(rng, 1, 65536)
        top_k = rng.choice([0, 0, 64, 512]) if ratio else 0
        # no more tokens times rows than the largest listed case
        most = min(2048 // seqs, int(2048 * 4096 / (seqs * (ctx / 4 + 300))), 256 if top_k else 2048)
        return dict(op=op, seqs=seqs, tokens=_log(rng, 1, max(1, most)), ragged=rng.random() < 0.5, ctx=ctx,
                    page=rng.choice([16, 64, 64, 128]), top_k=top_k, ratio=ratio)
    if op == "compressor_chunk":
        seqs = _log(rng, 1, 32)
        return dict(op=op, seqs=seqs, tokens=_log(rng, 1, 16384 // seqs), ragged=rng.random() < 0.5, ctx=_log(rng, 1, 16384),
                    page=rng.choice([16, 64]), wide=rng.choice([128, 512]))
    if op == "fork":
        sources = rng.choice([1, 1, 2])
        return dict(op=op, sources=sources, branches=_log(rng, 1, 8 // sources), ctx=_log(rng, 1, 65530),
                    page=rng.choice([16, 64]), spare=rng.randint(16, 128))
    return dict(op=op, pages=_log(rng, 16, 8192), page=rng.choice([16, 64]), live=round(rng.uniform(0.05, 0.95), 3))


# ---- sizes that a case stands for (they go by the case alone) ----

def _lengths(c):
    """The tokens of each sequence's chunk, and how many tokens each has before it."""
    r = random.Random("%s %s %s %s" % (c["op"], c["seqs"], c["tokens"], c["ctx"]))
    n = c["seqs"]
    if not c["ragged"]:
        return [c["tokens"]] * n, [c["ctx"]] * n
    lens = [r.randint(1, c["tokens"]) for _ in range(n)]
    lens[0], lens[-1] = c["tokens"], 1
    return lens, [r.randint(0, c["ctx"]) for _ in range(n)]


def _entries(c, lens, start):
    ratio = c.get("ratio", RATIO)
    return [(s + n) // ratio for n, s in zip(lens, start)] if ratio else [0] * len(lens)


def work(c):
    if c["op"] == "chunk_attention":
        lens, start = _lengths(c)
        pairs = rows = 0
        for n, s in zip(lens, start):
            rows += min(s, WINDOW - 1) + n + ((s + n) // RATIO if c["ratio"] else 0)
            for t in range(s, s + n):
                seen = (t + 1) // RATIO if c["ratio"] else 0
                pairs += min(t + 1, WINDOW) + (min(seen, c["top_k"]) if c["top_k"] else seen)
        if c["top_k"]:  # the listed rows alone are read, each once at the most
            rows = min(rows, pairs)
        lists = sum(lens) * c["top_k"] * 4
        return {"bytes": sum(lens) * HEADS * DIM * 4 + rows * DIM * 2 + lists, "flops": pairs * HEADS * DIM * 4}
    if c["op"] == "compressor_chunk":
        lens, start = _lengths(c)
        w, out = c["wide"], 2 if c["wide"] == 512 else 4
        rows = sum((s + n) // RATIO - s // RATIO for n, s in zip(lens, start))
        ring = 2 * RATIO * 2 * w * 4 * 2
        return {"bytes": sum(lens) * 2 * w * 8 + rows * w * out + 2 * ring * len(lens), "flops": rows * w * 60}
    if c["op"] == "fork":
        e = c["ctx"] // RATIO
        rings = 2 * 2 * RATIO * 2 * (DIM + IDX) * 4
        tiles = -(-e // 128)
        one = (e % c["page"]) * DIM * 2 + WINDOW * DIM * 2 + rings + e * IDX * 4 + tiles * (65536 + 512)
        return {"bytes": (c["sources"] + c["sources"] * c["branches"]) * one, "flops": 0}
    live = _live(c)
    n = sum(live)
    moved = sum(live[n:])
    return {"bytes": 2 * moved * c["page"] * DIM * 2 + 2 * c["pages"] * 8, "flops": 0}


def _live(c):
    r = random.Random("%s %s" % (c["pages"], c["live"]))
    live = [r.random() < c["live"] for _ in range(c["pages"])]
    live[0], live[-1] = False, True
    return live


# ---- inputs ----

def _cache(c, g, batch, entries, n_pages, max_chunk, table=None, refs=None):
    """The decode state of `batch` sequences as tensors: rings of window rows, pages of compressed rows
    in a shuffled order and a chunk's staged rows in one pool, block table, compressor rings, keys."""
    dev, page = "cuda", c["page"]
    per_seq = -(-max(entries, 1) // page) if entries else 0
    comp_base = batch * WINDOW
    st = dict(page=page, entries=entries, batch=batch, comp_base=comp_base, stage=comp_base + n_pages * page)
    st["pool"] = torch.randn(st["stage"] + max_chunk, DIM, generator=g, device=dev).to(torch.bfloat16)
    if table is None and entries:
        table = torch.randperm(n_pages, generator=g, device=dev)[:batch * per_seq].view(batch, per_seq).to(torch.int32)
        refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
        refs[table.long().view(-1)] = 1
    st["table"], st["refs"] = table, refs
    st["freqs"] = 1.0 / (160000.0 ** (torch.arange(0, ROPE, 2, device=dev, dtype=torch.float32) / ROPE))
    return st


def _make_cache(c, st, n_pages, max_chunk):
    """The framework's cache with the values of `st` in it."""
    pkg = importlib.import_module("deepseek-v4-flash-mlx_b200")
    cache = pkg.SparseMLACache(st["batch"], st["entries"], ratio=c.get("ratio", RATIO), page=st["page"], n_pages=n_pages,
                               max_chunk=max_chunk)
    cache.kv_pool.copy_(st["pool"])
    if st["entries"]:
        cache.block_table.copy_(st["table"])
        cache.page_refs.copy_(st["refs"])
    return pkg, cache


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    if c["op"] in ("chunk_attention", "compressor_chunk"):
        lens, start = _lengths(c)
        most, total, batch = max(_entries(c, lens, start)), sum(lens), len(lens)
        per_seq = -(-most // c["page"])
        n_pages = batch * per_seq + 3 if most else 0
        cu = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
        start_t = torch.tensor(start, dtype=torch.int32, device=dev)
    if c["op"] == "chunk_attention":
        st = _cache(c, g, batch, most, n_pages, total)
        st.update(case=c, lens=lens, start=start, cu=cu, start_t=start_t, rows=None)
        # queries as the per-head norm and the rotation leave them: a mean square of one
        q = torch.randn(total, HEADS, DIM, generator=g, device=dev)
        st["q"] = (q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)
        st["sink"] = torch.randn(HEADS, generator=g, device=dev)
        if c["top_k"]:
            # the list of a token: entries that it sees, in ascending order, -1 behind the last
            pos = torch.cat([torch.arange(s, s + n, device=dev) for n, s in zip(lens, start)])
            seq = torch.cat([torch.full((n,), b, device=dev) for b, n in enumerate(lens)])
            score = torch.rand(total, max(most, 1), generator=g, device=dev)
            score = score.masked_fill(torch.arange(max(most, 1), device=dev) >= ((pos + 1) // RATIO)[:, None], -1.0)
            val, e = score.topk(min(c["top_k"], max(most, 1)), dim=-1)
            e = e.masked_fill(val < 0, 1 << 30).sort(-1).values
            e = torch.nn.functional.pad(e, (0, c["top_k"] - e.shape[1]), value=1 << 30)
            none = e >= 1 << 30
            e = e.masked_fill(none, 0)
            rows = st["comp_base"] + st["table"].long()[seq[:, None], e // c["page"]] * c["page"] + e % c["page"] if most else e
            st["rows"] = rows.masked_fill(none, -1).to(torch.int32)
        if own:
            st["pkg"], st["cache"] = _make_cache(c, st, n_pages, total)
        return st
    if c["op"] == "compressor_chunk":
        w, keys = c["wide"], c["wide"] == IDX
        st = _cache(c, g, batch, most, n_pages, 1)
        st.update(case=c, lens=lens, start=start, cu=cu, start_t=start_t, wide=w)
        st["kv"] = torch.randn(total, 2 * w, generator=g, device=dev)
        st["score"] = torch.randn(total, 2 * w, generator=g, device=dev)
        st["ape"] = torch.randn(RATIO, 2 * w, generator=g, device=dev) * 0.1
        st["norm"] = 1 + 0.1 * torch.randn(w, generator=g, device=dev)
        st["ring0"] = (torch.randn(batch, 2 * RATIO, 2 * w, generator=g, device=dev),
                       torch.randn(batch, 2 * RATIO, 2 * w, generator=g, device=dev))
        for b, s in enumerate(start):  # rows of tokens that do not exist are empty
            if s < RATIO:
                st["ring0"][0][b, :RATIO], st["ring0"][1][b, :RATIO] = 0.0, float("-inf")
                st["ring0"][0][b, RATIO + s:], st["ring0"][1][b, RATIO + s:] = 0.0, float("-inf")
        st["ring"] = tuple(t.clone() for t in st["ring0"])
        st["out"] = torch.zeros(batch * max(most, 1), w, device=dev) if keys else st["pool"]
        if own:
            st["pkg"] = importlib.import_module("deepseek-v4-flash-mlx_b200")
        return st
    if c["op"] == "fork":
        e, n_src = c["ctx"] // RATIO, c["sources"]
        page, batch = c["page"], n_src * (1 + c["branches"])
        most = e + 8
        per_seq, held = -(-most // page), -(-e // page)
        n_pages = n_src * held + n_src * c["branches"] + c["spare"]
        table = torch.full((batch, per_seq), -1, dtype=torch.int32, device=dev)
        order = torch.randperm(n_pages, generator=g, device=dev)[:n_src * held].view(n_src, held).to(torch.int32)
        table[:n_src, :held] = order
        refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
        refs[order.long().view(-1)] = 1
        st = _cache(c, g, batch, most, n_pages, 0, table, refs)
        st["case"] = c
        tiles = -(-most // 128)
        st["k_idx"] = torch.randn(batch, most, IDX, generator=g, device=dev)
        st["image"] = torch.randint(0, 256, (batch, tiles * 65536), generator=g, device=dev, dtype=torch.uint8)
        st["inv"] = torch.rand(batch, tiles * 128, generator=g, device=dev) + 0.5
        st["norm_max"] = torch.rand(batch, generator=g, device=dev) + 10
        st["rings"] = [torch.randn(batch, 2 * RATIO, 2 * w, generator=g, device=dev) for w in (DIM, DIM, IDX, IDX)]
        st["src"] = torch.arange(n_src, dtype=torch.int32, device=dev).repeat_interleave(c["branches"])
        st["dst"] = torch.arange(n_src, batch, dtype=torch.int32, device=dev)
        st["tokens"] = torch.full((batch - n_src,), c["ctx"], dtype=torch.int32, device=dev)
        if own:
            _, cache = _make_cache(c, st, n_pages, 0)
            cache.k_idx.copy_(st["k_idx"])
            for t, v in zip(cache.key_image, (st["image"], st["inv"], st["norm_max"])):
                t.copy_(v.view(t.shape))
            for name, v in zip(("ring_kv", "ring_score", "ring_k_idx", "ring_s_idx"), st["rings"]):
                getattr(cache, name).copy_(v)
            st["cache"] = cache
        return st
    live = torch.tensor(_live(c), device=dev)
    n_pages = c["pages"]
    used = live.nonzero().view(-1)
    used = used[torch.randperm(used.numel(), generator=g, device=dev)]
    # sequences of up to 24 pages; the first pages of a sequence may be shared with the next one
    per_seq = 24
    batch = -(-used.numel() // 16)
    table = torch.full((batch, per_seq), -1, dtype=torch.int32, device=dev)
    at = torch.arange(used.numel(), device=dev)
    table[at // 16, at % 16] = used.to(torch.int32)
    shared = torch.rand(batch, generator=g, device=dev) < 0.25
    shared[0] = False
    table[:, 0] = torch.where(shared, table[:, 0].roll(1), table[:, 0])
    held = table[table >= 0].long()
    refs = torch.zeros(n_pages, dtype=torch.int32, device=dev)
    refs.index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    # a page that the sharing left without a holder is held from outside (a pinned prefix)
    refs = torch.where(live & (refs == 0), torch.ones_like(refs), refs)
    st = _cache(c, g, batch, per_seq * c["page"], n_pages, 0, table, refs)
    st["case"], st["table0"], st["refs0"] = c, table.clone(), refs.clone()
    if own:
        _, st["cache"] = _make_cache(c, st, n_pages, 0)
    return st


# ---- the plain forms, and the framework's calls ----

def _rotate(x, pos, freqs, inverse=False):
    """The rotation of the last ROPE dims of x [n, ..., d] at pos [n], pairs interleaved; the angle is the
    float32 product of position and frequency, as the model's tables form it."""
    a = (pos.to(torch.float32)[:, None] * freqs).to(x.dtype)
    a = a.view(a.shape[0], *[1] * (x.dim() - 2), a.shape[1])
    cos, sin = a.cos(), -a.sin() if inverse else a.sin()
    y = x.clone()
    re, im = x[..., -ROPE::2], x[..., -ROPE + 1::2]
    y[..., -ROPE::2], y[..., -ROPE + 1::2] = re * cos - im * sin, re * sin + im * cos
    return y


def _attention(st):
    c, pool, outs = st["case"], st["pool"], []
    dev = pool.device
    for b, (n, s) in enumerate(zip(st["lens"], st["start"])):
        lo = sum(st["lens"][:b])
        pos = torch.arange(s, s + n, device=dev)
        ring = torch.arange(max(0, s - WINDOW), s, device=dev)
        k = torch.cat([b * WINDOW + ring % WINDOW, st["stage"] + lo + torch.arange(n, device=dev)])
        kp = torch.cat([ring, pos])
        seen = (kp[None] <= pos[:, None]) & (kp[None] > pos[:, None] - WINDOW)
        q = st["q"][lo:lo + n].float()
        if c["top_k"]:
            rows = st["rows"][lo:lo + n].long()
            listed_k = pool[rows.clamp(min=0)].float()
            near_k = pool[k].float()
            score = torch.cat([(q.reshape(-1, DIM) @ near_k.T).view(n, HEADS, -1), q @ listed_k.transpose(1, 2)], -1)
            seen = torch.cat([seen, rows >= 0], 1)
        else:
            e = torch.arange((s + n) // RATIO if c["ratio"] else 0, device=dev)
            if e.numel():
                k = torch.cat([k, st["comp_base"] + st["table"][b].long()[e // c["page"]] * c["page"] + e % c["page"]])
                seen = torch.cat([seen, e[None] < ((pos + 1) // RATIO)[:, None]], 1)
            near_k = pool[k].float()
            score = (q.reshape(-1, DIM) @ near_k.T).view(n, HEADS, -1)
        score = (score * DIM ** -0.5).masked_fill_(~seen[:, None], float("-inf"))
        top = score.amax(-1, keepdim=True)
        p = score.sub_(top).exp_()
        den = p.sum(-1, keepdim=True) + (st["sink"].view(1, HEADS, 1) - top).exp()
        m = near_k.shape[0]
        o = (p[..., :m].reshape(n * HEADS, m) @ near_k).view(n, HEADS, DIM)
        if c["top_k"]:
            o = o + p[..., m:] @ listed_k
        outs.append(_rotate(o / den, pos, st["freqs"], inverse=True).to(torch.bfloat16))
    return torch.cat(outs)


def _emitted_rows(st, b, first, count):
    e = first + torch.arange(count, device=st["kv"].device)
    if st["wide"] == IDX:
        return b * st["entries"] + e
    return st["comp_base"] + st["table"][b].long()[e // st["page"]] * st["page"] + e % st["page"]


def _compress(st):
    ring_kv, ring_score, w = *st["ring"], st["wide"]
    for b, (n, s) in enumerate(zip(st["lens"], st["start"])):
        lo = sum(st["lens"][:b])
        pos = torch.arange(s, s + n, device=ring_kv.device)
        kv, score = st["kv"][lo:lo + n], st["score"][lo:lo + n] + st["ape"][pos % RATIO]
        # the tokens from the block before the current one on
        kv = torch.cat([ring_kv[b, :RATIO + s % RATIO], kv])
        score = torch.cat([ring_score[b, :RATIO + s % RATIO], score])
        blocks = kv.shape[0] // RATIO
        kb, sb = kv[:blocks * RATIO].view(blocks, RATIO, 2, w), score[:blocks * RATIO].view(blocks, RATIO, 2, w)
        if blocks > 1:
            k8, s8 = torch.cat([kb[:-1, :, 0], kb[1:, :, 1]], 1), torch.cat([sb[:-1, :, 0], sb[1:, :, 1]], 1)
            p = (s8 - s8.amax(1, keepdim=True)).exp()
            x = (p * k8).sum(1) / p.sum(1)
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * st["norm"]
            x = _rotate(x, (s // RATIO + torch.arange(blocks - 1, device=x.device)) * RATIO, st["freqs"])
            st["out"][_emitted_rows(st, b, s // RATIO, blocks - 1)] = x.to(st["out"].dtype)
            ring_kv[b, :RATIO], ring_score[b, :RATIO] = kv[(blocks - 1) * RATIO:blocks * RATIO], score[(blocks - 1) * RATIO:blocks * RATIO]
        m = min(n, RATIO)
        ring_kv[b, RATIO + pos[-m:] % RATIO], ring_score[b, RATIO + pos[-m:] % RATIO] = kv[-m:], score[-m:]
    return st["out"], ring_kv, ring_score


def _fork(st):
    c, table, refs, page = st["case"], st["table"], st["refs"], st["page"]
    # the branches that are there are given up, then made again
    dst, src = st["dst"].long(), st["src"].long()
    gone = table[dst]
    refs.index_add_(0, gone[gone >= 0].long(), torch.full_like(gone[gone >= 0], -1))
    e = c["ctx"] // RATIO
    full, tail, tiles = e // page, e % page, -(-e // 128)
    table[dst] = -1
    table[dst, :full] = table[src, :full]
    kept = table[dst, :full].reshape(-1).long()
    refs.index_add_(0, kept, torch.ones_like(kept, dtype=torch.int32))
    if tail:
        new = (refs == 0).nonzero().view(-1)[:dst.numel()]
        refs[new] = 1
        row = torch.arange(tail, device=refs.device)
        old = table[src, full].long()
        st["pool"][st["comp_base"] + new[:, None] * page + row] = st["pool"][st["comp_base"] + old[:, None] * page + row]
        table[dst, full] = new.to(torch.int32)
    win = torch.arange(WINDOW, device=refs.device)
    st["pool"][dst[:, None] * WINDOW + win] = st["pool"][src[:, None] * WINDOW + win]
    for r in st["rings"]:
        r[dst] = r[src]
    st["k_idx"][dst, :e] = st["k_idx"][src, :e]
    st["image"][dst, :tiles * 65536] = st["image"][src, :tiles * 65536]
    st["inv"][dst, :tiles * 128] = st["inv"][src, :tiles * 128]
    st["norm_max"][dst] = st["norm_max"][src]
    return [st["pool"], table, refs, st["k_idx"], st["image"], st["inv"], st["norm_max"], *st["rings"]]


def _compact(st):
    refs, page = st["refs0"], st["page"]
    live = refs > 0
    n = live.sum()
    at = torch.arange(refs.numel(), device=refs.device)
    hole, mover = ((at < n) & ~live).nonzero().view(-1), ((at >= n) & live).nonzero().view(-1)
    row = torch.arange(page, device=refs.device)
    st["pool"][st["comp_base"] + hole[:, None] * page + row] = st["pool"][st["comp_base"] + mover[:, None] * page + row]
    to = at.clone()
    to[mover] = hole
    table = torch.where(st["table0"] >= 0, to[st["table0"].clamp(min=0).long()].to(torch.int32), st["table0"])
    refs = refs.clone()
    refs[hole], refs[mover] = refs[mover], torch.zeros_like(refs[mover])
    st["table"], st["refs"] = table, refs
    return [st["pool"], table, refs, n.to(torch.int32).view(1)]


def run(st):
    c = st["case"]
    if c["op"] == "chunk_attention":
        if own:
            return st["pkg"].chunk_attention(st["cache"], st["q"], st["sink"], st["cu"], st["start_t"], rows=st["rows"],
                                             freqs=st["freqs"])
        return _attention(st)
    if c["op"] == "compressor_chunk":
        # each pass starts from the same rings
        for t, v in zip(st["ring"], st["ring0"]):
            t.copy_(v)
        if own:
            keys = c["wide"] == IDX
            st["pkg"].compressor_chunk((st["kv"], st["score"]), st["cu"], st["start_t"], st["ape"], st["norm"], *st["ring"],
                                       st["out"], max_comp=st["entries"], block_table=None if keys else st["table"],
                                       page=st["page"], out_base=0 if keys else st["comp_base"], head_dim=c["wide"],
                                       freqs=st["freqs"])
            return st["out"], *st["ring"]
        return _compress(st)
    if c["op"] == "fork":
        if own:
            cache = st["cache"]
            cache.free(st["dst"])
            cache.fork(st["src"], st["dst"], st["tokens"])
            img, inv, norm_max = cache.key_image
            return [cache.kv_pool, cache.block_table, cache.page_refs, cache.k_idx, img.view(st["image"].shape), inv, norm_max,
                    cache.ring_kv, cache.ring_score, cache.ring_k_idx, cache.ring_s_idx]
        return _fork(st)
    if own:
        # each pass starts from the same tables and counts; the pages that are left behind still hold their rows
        cache = st["cache"]
        cache.block_table.copy_(st["table0"])
        cache.page_refs.copy_(st["refs0"])
        n = cache.compact()
        return [cache.kv_pool, cache.block_table, cache.page_refs, n]
    return _compact(st)


# ---- the same in 64 bits, from the definitions ----

def _exact_attention(st):
    """Token by token: the list of its rows, gathered."""
    c, dev = st["case"], st["pool"].device
    f64 = torch.float64
    outs = []
    for b, (n, s) in enumerate(zip(st["lens"], st["start"])):
        lo = sum(st["lens"][:b])
        ents = (s + n) // RATIO if c["ratio"] and not c["top_k"] else 0
        step = max(1, int(2e8 // ((WINDOW + max(ents, c["top_k"])) * DIM)))
        for a in range(0, n, step):
            t = torch.arange(a, min(n, a + step), device=dev)
            p = s + t
            w = p[:, None] - torch.arange(WINDOW, device=dev)[None]
            row = torch.where(w >= s, st["stage"] + lo + w - s, b * WINDOW + w % WINDOW)
            row = torch.where(w >= 0, row, -1)
            if c["top_k"]:
                row = torch.cat([row, st["rows"][lo + t].long()], 1)
            elif ents:
                e = torch.arange(ents, device=dev)[None].expand(t.numel(), -1)
                r = st["comp_base"] + st["table"][b].long()[e // c["page"]] * c["page"] + e % c["page"]
                row = torch.cat([row, torch.where(e < (p[:, None] + 1) // RATIO, r, -1)], 1)
            kv = st["pool"][row.clamp(min=0)].to(f64)
            x = torch.einsum("thd,tkd->thk", st["q"][lo + t].to(f64), kv) / math.sqrt(DIM)
            x = torch.where((row >= 0)[:, None], x, -math.inf)
            z = torch.cat([x, st["sink"].to(f64).view(1, HEADS, 1).expand(t.numel(), -1, 1)], -1).softmax(-1)[..., :-1]
            outs.append(_turn(torch.einsum("thk,tkd->thd", z, kv), p, st["freqs"], -1))
    return torch.cat(outs)


def _turn(x, pos, freqs, sign):
    """The rotation as a product of complex numbers."""
    angle = (pos.float()[:, None] * freqs).double() * sign
    z = torch.view_as_complex(x[..., -ROPE:].reshape(*x.shape[:-1], ROPE // 2, 2).contiguous())
    turn = torch.polar(torch.ones_like(angle), angle).view(-1, *[1] * (x.dim() - 2), ROPE // 2)
    return torch.cat([x[..., :-ROPE], torch.view_as_real(z * turn).flatten(-2)], -1)


def _exact_compress(st):
    """Row by row from its eight tokens, each found by its position."""
    w, dev = st["wide"], st["kv"].device
    out, rk, rs = st["out"].double(), st["ring0"][0].double(), st["ring0"][1].double()
    new_k, new_s = rk.clone(), rs.clone()
    for b, (n, s) in enumerate(zip(st["lens"], st["start"])):
        lo = sum(st["lens"][:b])

        def token(p):
            """(kv, score with its place's share) of the tokens at positions p, from the chunk or the ring."""
            here, block = p >= s, s // RATIO * RATIO
            i = (lo + p - s).clamp(lo, lo + n - 1)
            place = torch.where(p >= block, RATIO + p % RATIO, p % RATIO)
            k = torch.where(here[..., None], st["kv"][i].double(), rk[b][place])
            v = torch.where(here[..., None], st["score"][i].double() + st["ape"].double()[p % RATIO], rs[b][place])
            return k, v

        g = torch.arange(s // RATIO, (s + n) // RATIO, device=dev)
        if g.numel():
            k0, s0 = token((g[:, None] - 1) * RATIO + torch.arange(RATIO, device=dev))
            k1, s1 = token(g[:, None] * RATIO + torch.arange(RATIO, device=dev))
            z = torch.cat([s0[..., :w], s1[..., w:]], 1).softmax(1)
            x = (z * torch.cat([k0[..., :w], k1[..., w:]], 1)).sum(1)
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * st["norm"].double()
            out[_emitted_rows(st, b, s // RATIO, g.numel())] = _turn(x, g * RATIO, st["freqs"], 1)
            new_k[b, :RATIO], new_s[b, :RATIO] = token(g[-1] * RATIO + torch.arange(RATIO, device=dev))
        last = torch.arange(max(s, s + n - RATIO), s + n, device=dev)
        new_k[b, RATIO + last % RATIO], new_s[b, RATIO + last % RATIO] = token(last)
    return out, new_k, new_s


def exact(c, seed):
    st = prepare(c, seed)
    if c["op"] == "chunk_attention":
        return _exact_attention(st)
    if c["op"] == "compressor_chunk":
        return _exact_compress(st)
    if c["op"] == "fork":
        # where each row of a branch comes from, one index for each part
        src, dst, e, page = st["src"].tolist(), st["dst"].tolist(), c["ctx"] // RATIO, c["page"]
        free = (st["refs"] == 0).nonzero().view(-1).tolist()
        pool, keys, inv, norm_max = st["pool"].double(), st["k_idx"].double(), st["inv"].double(), st["norm_max"].double()
        rings = [r.double() for r in st["rings"]]
        for i, (a, b) in enumerate(zip(src, dst)):
            pool[b * WINDOW:(b + 1) * WINDOW] = pool[a * WINDOW:(a + 1) * WINDOW]
            keys[b, :e], inv[b, :-(-e // 128) * 128], norm_max[b] = keys[a, :e], inv[a, :-(-e // 128) * 128], norm_max[a]
            for r in rings:
                r[b] = r[a]
            if e % page:
                x, y = st["comp_base"] + int(st["table"][a, e // page]) * page, st["comp_base"] + free[i] * page
                pool[y:y + e % page] = pool[x:x + e % page]
        return [pool, None, None, keys, None, inv, norm_max, *rings]
    pool, live = st["pool"].double(), _live(c)
    n, page, base = sum(live), c["page"], st["comp_base"]
    holes = [i for i in range(n) if not live[i]]
    movers = [i for i in range(n, len(live)) if live[i]]
    pages = pool[base:base + len(live) * page].view(len(live), page, DIM)
    pages[holes] = pages[movers]
    return [pool, None, None, None]
