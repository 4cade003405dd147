"""The operators of a server's step over a paged 8-bit cache, as cases to time and compare.

  store    mynah_hip_kv8_store_dev: new keys and values of a ragged batch into an 8-bit cache with a
           scale for each block of positions and head; a block whose new rows are larger than its
           scale allows is scaled anew, old rows included
  attn     mynah_hip_kv8_attention_dev: attention of new tokens (one, a draft's, a prompt's) over
           such a cache
  beam     mynah_hip_pages_fork_dev, then mynah_hip_pages_reserve_dev: sequences continue others,
           sharing their pages, and each gets room for its next tokens in pages of its own
  compact  mynah_hip_pages_compact_dev: the pages in use move to the lowest places of the pool
  logits   mynah_hip_logits_dev: penalties for repeated tokens, biases and grammar masks

With `own` false, run() computes the same in elementary torch operations.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "mynah-slm_amd"))

own = False
GPU = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IDS = {"f32": 0, "f16": 1, "bf16": 30}     # ggml's type ids
FORMATS = {"i8": 0, "e4m3": 1}
MOST = {"i8": 127.0, "e4m3": 448.0}        # the largest code's value
AMAX_MIN = 2.0 ** -100


def _store(seqs, nodes, past, kv_heads, hd, dtype, fmt, block, page=0):
    """page: positions of a cache page, 0 for one run of rows for each sequence. Sequences after
    the first are of any length up to the first's."""
    return {"kind": "store", "seqs": seqs, "nodes": nodes, "past": past, "kv_heads": kv_heads,
            "hd": hd, "dtype": dtype, "format": fmt, "block": block, "page": page}


def _attn(seqs, nodes, past, heads, kv_heads, hd, dtype, fmt, block, page=0, shape="chain"):
    return {**_store(seqs, nodes, past, kv_heads, hd, dtype, fmt, block, page), "kind": "attn",
            "heads": heads, "shape": shape}


def _beam(parents, children, past, new, page, layers, row):
    """row: bytes of a position's keys (and of its values) in one layer."""
    return {"kind": "beam", "parents": parents, "children": children, "past": past, "new": new,
            "page": page, "layers": layers, "row": row}


def _compact(pages, live, page, layers, row):
    return {"kind": "compact", "pages": pages, "live": live, "page": page, "layers": layers,
            "row": row}


def _logits(rows, vocab, dtype, out, history, biases, masks):
    """masks: grammars at work; some rows have none of them."""
    return {"kind": "logits", "rows": rows, "vocab": vocab, "dtype": dtype, "out": out,
            "history": history, "biases": biases, "masks": masks}


def listed():
    return [
        # One decoded token's key and value rows into the last block of a cache.
        {"name": "store_1tok", **_store(1, 1, 513, 8, 128, "f32", "i8", 64)},
        # A prompt of 8190 tokens behind a cached prefix that ends inside a block.
        {"name": "store_prompt", **_store(1, 8190, 1003, 8, 128, "bf16", "e4m3", 64, page=64)},
        # A 0.6B decode step at 513 positions: one token, latency counts.
        {"name": "attn_1tok_f32", **_attn(1, 1, 512, 16, 8, 128, "f32", "i8", 64)},
        # A serving batch's step: 32 ragged sequences, one token each, pages of 64.
        {"name": "attn_batch_bf16", **_attn(32, 1, 16_383, 32, 8, 128, "bf16", "e4m3", 64, page=64)},
        # Eight drafted tokens over one very long context.
        {"name": "attn_long_f16", **_attn(1, 8, 130_001, 32, 8, 128, "f16", "i8", 128, page=256,
                                          shape="tree")},
        # A prompt's chunk of 2048 tokens behind 6144 cached ones.
        {"name": "attn_prompt_bf16", **_attn(1, 2048, 6144, 32, 8, 128, "bf16", "i8", 64, page=64)},
        # Four beams of one request, each continued by two; the last page of each is its own.
        {"name": "beam_4", **_beam(4, 4, 700, 1, 64, 4, 1024)},
        # A batch of 64 requests, a draft of eight tokens for two continuations of each.
        {"name": "beam_64", **_beam(64, 64, 3000, 8, 64, 6, 1024)},
        # A small pool after a few requests have ended.
        {"name": "compact_small", **_compact(96, 60, 16, 4, 1024)},
        # A pool of 640 pages of 64 positions, 400 in use.
        {"name": "compact_640", **_compact(640, 400, 64, 6, 1024)},
        # One row of logits at the full vocabulary, a window of 512 tokens, a grammar.
        {"name": "logits_1row", **_logits(1, 151_936, "f32", "f32", 512, 8, 1)},
        # A batch of 192 rows, long histories, 16 grammars.
        {"name": "logits_192", **_logits(192, 151_936, "bf16", "f32", 4096, 64, 16)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("store", "store", "attn", "attn", "attn", "beam", "compact", "logits"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    fmt = rng.choice(("i8", "e4m3"))
    page = rng.choice((0, 16, 64, 128, 256))
    block = rng.choice([b for b in (16, 32, 64, 128, 256) if b <= (page or 128)])
    hd, kvh = rng.choice((64, 128, 128, 256)), rng.choice((1, 2, 3, 4, 8))
    if kind == "store":
        seqs = rng.choice((1, _log(rng, 1, 64)))
        nodes = min(rng.choice((1, _log(rng, 1, 8190))), 8_000_000 // (seqs * kvh * hd))
        past = _log(rng, 1, min(8000, 16_000_000 // (seqs * kvh * hd)))
        return _store(seqs, max(nodes, 1), past, kvh, hd, dtype, fmt, block, page)
    if kind == "attn":
        group = rng.choice((1, 2, 3, 4, 5, 7, 8, 16))
        seqs, nodes = rng.choice((1, _log(rng, 1, 48))), rng.choice((1, _log(rng, 1, 80), 600))
        if nodes == 600:
            seqs, nodes = rng.randint(1, 4), _log(rng, 81, 2048)
        pairs = (20_000_000_000 if dtype == "f32" else 55_000_000_000) // (seqs * kvh * group * hd)
        past = min(260_000_000 // (seqs * kvh * hd), pairs // nodes - nodes, 131_000)
        past = _log(rng, 1, max(past, 1))
        return _attn(seqs, nodes, past, kvh * group, kvh, hd, dtype, fmt, block, page,
                     "tree" if nodes <= 80 and rng.random() < 0.6 else "chain")
    if kind == "beam":
        parents, page = _log(rng, 1, 48), rng.choice((16, 32, 64, 128))
        row = rng.choice((256, 512, 1024))
        past = min(_log(rng, 1, 4000), 48 * 3000 // parents)
        return _beam(parents, parents * rng.randint(1, 2) if parents < 30 else parents, past,
                     rng.choice((1, _log(rng, 1, 100))), page, rng.randint(1, 6), row)
    if kind == "compact":
        pages = 4 * _log(rng, 4, 150)
        return _compact(pages, rng.randint(1, pages), rng.choice((16, 32, 64)), rng.randint(1, 6),
                        rng.choice((256, 512, 1024)))
    rows = _log(rng, 1, 192)
    vocab = 32 * _log(rng, 10, 4748) - rng.choice((0, 0, 1, 5))
    return _logits(rows, vocab, dtype, rng.choice((dtype, "f32")), rng.choice((0, _log(rng, 1, 4096))),
                   rng.choice((0, _log(rng, 1, min(64, vocab)))), rng.choice((0, 1, rng.randint(1, 16))))


# ── inputs ───────────────────────────────────────────────────────────────────

def _gen(seed, k):
    g = torch.Generator(device=GPU)
    g.manual_seed((int(seed) * 1_000_003 + k) % (1 << 62))
    return g


def _normal(seed, k, *shape):
    return torch.randn(*shape, generator=_gen(seed, k), device=GPU)


def _ints(a, t=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, t)).to(GPU)


def _ancestors(rng, nodes, n):
    """[n][words] int32: bit j of row i where node i is, or descends from, node j."""
    m = np.zeros((n, (nodes + 31) // 32), np.uint32)
    for i in range(n):
        parent = int(rng.integers(-1, i)) if i else -1
        if parent >= 0:
            m[i] = m[parent]
        m[i, i // 32] |= np.uint32(1 << (i % 32))
    return m.view(np.int32)


def _scale_of(amax, fmt):
    """A block's scale for values up to amax: amax / 127, or the least power of two that keeps
    them within 448."""
    amax = amax.clamp_min(AMAX_MIN)
    if fmt == "i8":
        return amax / 127
    m, e = torch.frexp(amax / 448)
    return torch.ldexp(torch.ones_like(amax), torch.where(m > 0.5, e, e - 1))


def _codes(x, inv, fmt):
    """Codes of x times inv, as the type that stands for them."""
    if fmt == "i8":
        return torch.round(x * inv).clamp(-127, 127).to(torch.int8)
    return (x * inv).clamp(-448, 448).to(torch.float8_e4m3fn)


def _cache(case, seed, k, rows):
    """(codes [rows][kv heads][hd], scales [blocks][kv heads]) of a cache in use; blocks differ
    in size."""
    kvh, hd, block, fmt = case["kv_heads"], case["hd"], case["block"], case["format"]
    x = _normal(seed, k, rows // block, block, kvh, hd)
    x *= torch.exp(0.5 * _normal(seed, k + 1, rows // block, 1, kvh, 1))
    s = _scale_of(x.abs().amax((1, 3)), fmt)
    c = _codes(x, (1 / s)[:, None, :, None], fmt)
    return c.reshape(rows, kvh, hd), s.contiguous()


def _prepare_cache(case, seed):
    """What store and attention share: lengths, pages, the cache."""
    rng = np.random.default_rng((int(seed), 77))
    n, page = case["seqs"], case["page"]
    lengths = np.random.default_rng(case["past"])      # the case's own, whatever the seed
    past = np.concatenate([[case["past"]], lengths.integers(0, case["past"] + 1, n - 1)])
    nodes = np.concatenate([[case["nodes"]], lengths.integers(1, case["nodes"] + 1, n - 1)])
    max_kv = case["past"] + case["nodes"]
    s = {"case": case, "n_past": _ints(past), "max_kv": max_kv, "total": int(nodes.sum()),
         "seq_start": _ints(np.concatenate([[0], np.cumsum(nodes)])), "rng": rng, "nodes": nodes}
    if page:
        max_pages = -(-max_kv // page)
        s["pages"] = _ints(rng.permutation(n * max_pages).reshape(n, max_pages))
        rows = n * max_pages * page
    else:
        s["seq_slots"] = -(-max_kv // case["block"]) * case["block"]
        rows = n * s["seq_slots"]
    s["k"], s["ks"] = _cache(case, seed, 1, rows)
    s["v"], s["vs"] = _cache(case, seed, 3, rows)
    return s


def _prepare_store(case, seed):
    s = _prepare_cache(case, seed)
    t, shape = DTYPES[case["dtype"]], (s["total"], case["kv_heads"], case["hd"])
    # Now and then a token is larger than those before it: its block is scaled anew.
    big = torch.exp(0.5 * _normal(seed, 7, s["total"], 1, 1))
    s["kx"] = (_normal(seed, 5, *shape) * big).to(t)
    s["vx"] = (_normal(seed, 6, *shape) * big).to(t)
    return s


def _prepare_attn(case, seed):
    s = _prepare_cache(case, seed)
    # Normalised queries: scores of a few units, some positions far above the rest.
    s["q"] = _normal(seed, 5, s["total"], case["heads"], case["hd"]).to(DTYPES[case["dtype"]])
    s["out"] = torch.empty_like(s["q"])
    if case["shape"] == "tree":
        s["mask"] = _ints(np.concatenate([_ancestors(s["rng"], case["nodes"], int(k))
                                          for k in s["nodes"]]))
    return s


def _parts(case, seed, n_pages):
    """A pool's memory: each layer's keys, values and their scales, as 32-bit words a page."""
    sizes = [case["page"] * case["row"] // 4] * 2 + [case["row"] // 128] * 2
    return [torch.randint(-2 ** 31, 2 ** 31 - 1, (n_pages, w), generator=_gen(seed, 20 + i),
                          device=GPU, dtype=torch.int32)
            for i, w in enumerate(sizes * case["layers"])]


def _prepare_beam(case, seed):
    rng = np.random.default_rng((int(seed), 78))
    w, page, n = case["parents"], case["page"], case["parents"] + case["children"]
    lengths = np.random.default_rng(case["past"])
    past = lengths.integers(1 + case["past"] // 2, case["past"] + 1, w)
    past[0] = case["past"]
    held = -(-past // page)
    more = -(-case["new"] // page) + 1
    max_pages, n_pages = int(held.max()) + more, 4 * (-(-(int(held.sum()) + n * more) // 4) + 1)
    ids = rng.permutation(n_pages)
    table, refs, at = np.full((n, max_pages), -1), np.zeros(n_pages), 0
    for b in range(w):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    refs[ids[:at]] = 1
    s = {"case": case, "pages": _ints(table), "refs": _ints(refs),
         "n_past": _ints(np.concatenate([past, np.zeros(n - w)])),
         "from": _ints(np.concatenate([np.arange(w), np.arange(n - w) % w])),
         "n_new": _ints(np.full(n, case["new"])), "status": _ints([0, 0]),
         "parts": _parts(case, seed, n_pages)}
    return s


def _prepare_compact(case, seed):
    rng = np.random.default_rng((int(seed), 79))
    n_pages, live = case["pages"], case["live"]
    ids = rng.permutation(n_pages)[:live]
    n_seqs = max(1, live // 16)
    max_pages = 4 * (-(-live // n_seqs) // 2 + 1)
    table, refs = np.full((n_seqs, max_pages), -1), np.zeros(n_pages)
    for b in range(n_seqs):
        mine = ids[b::n_seqs]
        table[b, :len(mine)] = mine
        if b % 3 == 2:                       # begins with pages of the sequence before
            table[b, :2] = table[b - 1, :2]
    for p in table[table >= 0]:
        refs[p] += 1
    s = {"case": case, "pages": _ints(table), "refs": _ints(refs), "status": _ints([0, 0]),
         "n_past": _ints((table >= 0).sum(1) * case["page"]), "parts": _parts(case, seed, n_pages)}
    s["pages0"], s["refs0"] = s["pages"].clone(), s["refs"].clone()
    return s


def _prepare_logits(case, seed):
    rng = np.random.default_rng((int(seed), 80))
    n, vocab = case["rows"], case["vocab"]
    s = {"case": case, "x": (3 * _normal(seed, 1, n, vocab)).to(DTYPES[case["dtype"]]),
         "y": torch.empty(n, vocab, device=GPU, dtype=DTYPES[case["out"]])}
    lengths = np.random.default_rng(case["history"] + n)
    if case["history"]:
        size = lengths.integers(1 + case["history"] // 2, case["history"] + 1, n)
        # Text repeats few of its tokens often.
        common = rng.integers(0, vocab, 1 + case["history"] // 4)
        hist = common[(len(common) * rng.random(int(size.sum())) ** 3).astype(np.int64)]
        s["hist"], s["hist_start"] = _ints(hist), _ints(np.concatenate([[0], np.cumsum(size)]), np.int64)
        s["repeat"] = _ints(1 + 0.3 * rng.random(n), np.float32)
        s["freq"] = _ints(0.5 * rng.random(n), np.float32)
        s["presence"] = _ints(0.5 * rng.random(n), np.float32)
    if case["biases"]:
        size = lengths.integers(0, case["biases"] + 1, n)
        size[0] = case["biases"]
        ids = np.concatenate([rng.permutation(vocab)[:k] for k in size])
        s["bias_id"], s["bias_start"] = _ints(ids), _ints(np.concatenate([[0], np.cumsum(size)]), np.int64)
        s["bias"] = _ints(10 * rng.standard_normal(len(ids)), np.float32)
    if case["masks"]:
        words = (vocab + 31) // 32
        s["allowed"] = torch.randint(-2 ** 31, 2 ** 31 - 1, (case["masks"], words), device=GPU,
                                     generator=_gen(seed, 2), dtype=torch.int32)
        of = rng.integers(-1, case["masks"], n)
        of[0] = 0
        s["mask_row"] = _ints(of)
    return s


def prepare(case, seed):
    return {"store": _prepare_store, "attn": _prepare_attn, "beam": _prepare_beam,
            "compact": _prepare_compact, "logits": _prepare_logits}[case["kind"]](case, seed)


# ── the operators in elementary torch operations ─────────────────────────────

def _rows_of(s, seq, pos):
    """Cache rows of positions of sequences."""
    page = s["case"]["page"]
    if page:
        return s["pages"].long()[seq, pos // page] * page + pos % page
    return seq * s["seq_slots"] + pos


def _take(codes, at):
    return codes.view(torch.int8)[at].view(codes.dtype).float()


def _plain_store(s):
    c = s["case"]
    block, fmt, n = c["block"], c["format"], c["seqs"]
    start, past = s["seq_start"].long(), s["n_past"].long()
    row = torch.arange(s["total"], device=GPU)
    seq = torch.searchsorted(start, row, right=True) - 1
    pos = past[seq] + row - start[seq]
    # Every block that a new row falls in, as its cache rows' block.
    blocks, which = torch.unique(_rows_of(s, seq, pos) // block, return_inverse=True)
    first = torch.zeros_like(blocks).scatter_(0, which, pos // block * block)
    owner = torch.zeros_like(blocks).scatter_(0, which, seq)
    old_rows = blocks[:, None] * block + torch.arange(block, device=GPU)
    kept = first[:, None] + torch.arange(block, device=GPU) < past[owner][:, None]
    for codes, scales, x in ((s["k"], s["ks"], s["kx"]), (s["v"], s["vs"], s["vx"])):
        x = x.float()
        amax = torch.zeros(len(blocks), c["kv_heads"], device=GPU)
        amax.scatter_reduce_(0, which[:, None].expand(-1, c["kv_heads"]), x.abs().amax(-1), "amax")
        old = torch.where(kept[:, :1], scales[blocks], 0)
        new = torch.maximum(_scale_of(amax, fmt), old)
        again = _codes(_take(codes, old_rows), (old / new)[:, None, :, None], fmt).view(torch.int8)
        raw = codes.view(torch.int8)
        raw[old_rows[kept]] = again[kept]
        raw[_rows_of(s, seq, pos)] = _codes(x, (1 / new)[which][..., None], fmt).view(torch.int8)
        scales[blocks] = new
    return {"k": s["k"], "ks": s["ks"], "v": s["v"], "vs": s["vs"]}


def _plain_attn(s):
    c = s["case"]
    kvh, hd, n, group = c["kv_heads"], c["hd"], c["nodes"], c["heads"] // c["kv_heads"]
    start, past = s["seq_start"].long(), s["n_past"].long()
    pos = torch.arange(s["max_kv"], device=GPU)
    node = torch.arange(n, device=GPU)
    real = node < (start[1:] - start[:-1]).unsqueeze(1)                       # [seqs][nodes]
    row = torch.where(real, start[:-1].unsqueeze(1) + node, 0)
    length = past + start[1:] - start[:-1]
    there = pos < length.unsqueeze(1)                                         # [seqs][positions]
    at = _rows_of(s, torch.arange(c["seqs"], device=GPU).unsqueeze(1), torch.where(there, pos, 0))
    k = _take(s["k"], at) * s["ks"][at // c["block"]].unsqueeze(-1)
    v = _take(s["v"], at) * s["vs"][at // c["block"]].unsqueeze(-1)
    j = pos - past.unsqueeze(1)                                               # node of a position
    if "mask" in s:
        jc = j.clamp(0, n - 1).unsqueeze(1).expand(-1, n, -1)
        seen = (s["mask"][row].gather(2, jc >> 5) >> (jc & 31)) & 1 == 1
    else:
        seen = j.unsqueeze(1) <= node.unsqueeze(1)
    seen = there.unsqueeze(1) & (seen | (j < 0).unsqueeze(1))
    q = s["q"][row].float().reshape(c["seqs"], n, kvh, group, hd).permute(0, 2, 3, 1, 4)
    q = q.reshape(c["seqs"], kvh, group * n, hd)
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) / math.sqrt(hd)
    score = score.reshape(c["seqs"], kvh, group, n, -1)
    score = score.masked_fill(~seen.unsqueeze(1).unsqueeze(1), -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(c["seqs"], kvh, group * n, -1)
    out = torch.matmul(p, v.permute(0, 2, 1, 3).contiguous())
    out = out.reshape(c["seqs"], kvh, group, n, hd).permute(0, 3, 1, 2, 4)
    return out[real].reshape(-1, c["heads"], hd).to(s["q"].dtype)


def _pool(s):
    return {k: s[k] for k in ("pages", "refs", "n_past", "status")} | {
        f"part{i}": p for i, p in enumerate(s["parts"])}


def _held(table, n_pages):
    """How many entries of the table name each page."""
    flat = table.flatten().long()
    return torch.zeros(n_pages + 1, device=GPU, dtype=torch.int32).index_add_(
        0, torch.where(flat < 0, n_pages, flat), torch.ones_like(flat, dtype=torch.int32))[:n_pages]


def _plain_beam(s):
    page, refs = s["case"]["page"], s["refs"]
    n_pages, source = len(refs), s["from"].long()
    # fork: a row becomes what its source's was
    refs -= _held(s["pages"], n_pages)
    s["pages"].copy_(s["pages"][source])
    s["n_past"].copy_(s["n_past"][source])
    refs += _held(s["pages"], n_pages)
    # reserve: entries of the new positions that name no page, or one that others hold too
    table, past = s["pages"], s["n_past"].long().unsqueeze(1)
    j = torch.arange(table.shape[1], device=GPU)
    new = s["n_new"].long().unsqueeze(1)
    needed = (j >= past // page) & (j < (past + new + page - 1) // page) & (new > 0)
    grows = needed & (table >= 0)
    at = torch.where(grows, table.long(), n_pages).flatten()
    row = torch.arange(len(table), device=GPU).unsqueeze(1).expand_as(table).flatten()
    count = torch.zeros(n_pages + 1, device=GPU, dtype=torch.int32).index_add_(
        0, at, torch.ones_like(at, dtype=torch.int32))
    first = torch.full((n_pages + 1,), len(table), device=GPU).scatter_reduce_(0, at, row, "amin")
    holders = torch.cat([refs, refs.new_ones(1)])
    keeps = (count[at] == holders[at]) & (first[at] == row)
    copied = grows & (holders[at] > 1).reshape(table.shape) & ~keeps.reshape(table.shape)
    wanted = (needed & (table < 0)) | copied
    free = torch.sort(refs != 0, stable=True).indices
    rank = wanted.flatten().cumsum(0).reshape(table.shape) - 1
    missing = wanted.sum() - (refs == 0).sum()
    fits = missing <= 0
    fresh = free[rank.clamp(0, n_pages - 1)].int()
    wanted, copied = wanted & fits, copied & fits
    old, partial = table[copied & (j * page < past)], fresh[copied & (j * page < past)]
    s["status"].copy_(torch.stack([missing.clamp_min(0), torch.zeros_like(missing)]))
    refs.index_add_(0, table[copied].long(), torch.full_like(table[copied], -1))
    table.copy_(torch.where(wanted, fresh, table))
    refs[table[wanted].long()] = 1
    for part in s["parts"]:
        part[partial.long()] = part[old.long()]
    return _pool(s)


def _plain_compact(s):
    s["pages"].copy_(s["pages0"])
    s["refs"].copy_(s["refs0"])
    table, refs = s["pages"], s["refs"]
    used = refs > 0
    live = used.sum()
    ids = torch.arange(len(refs), device=GPU)
    to, source = ids[~used & (ids < live)], ids[used & (ids >= live)]
    new = ids.clone()
    new[source] = to
    table.copy_(torch.where(table >= 0, new[table.long().clamp_min(0)].int(), table))
    refs[to], refs[source] = refs[source], 0
    for part in s["parts"]:
        part[to] = part[source]
    s["status"].copy_(torch.stack([live, live.new_tensor(len(to))]))
    return _pool(s)


def _plain_logits(s):
    c = s["case"]
    n, vocab = c["rows"], c["vocab"]
    x = s["x"].float()
    row = torch.arange(n, device=GPU)
    if "hist" in s:
        of = torch.repeat_interleave(row, s["hist_start"].diff(), output_size=len(s["hist"]))
        count = torch.zeros(n * vocab, device=GPU).index_add_(
            0, of * vocab + s["hist"], torch.ones_like(s["hist"], dtype=torch.float32))
        count = count.reshape(n, vocab)
        rep = s["repeat"].unsqueeze(1)
        y = torch.where(x > 0, x / rep, x * rep)
        y = y - s["freq"].unsqueeze(1) * count - s["presence"].unsqueeze(1)
        x = torch.where(count > 0, y, x)
    if "bias" in s:
        of = torch.repeat_interleave(row, s["bias_start"].diff(), output_size=len(s["bias"]))
        x = x.flatten().index_add(0, of * vocab + s["bias_id"], s["bias"]).reshape(n, vocab)
    if "allowed" in s:
        bit = torch.arange(32, device=GPU, dtype=torch.int32)
        ok = ((s["allowed"].unsqueeze(-1) >> bit) & 1 == 1).flatten(1)[:, :vocab]
        of = s["mask_row"].long().unsqueeze(1)
        x = torch.where((of < 0) | ok[of.squeeze(1).clamp_min(0)], x, -math.inf)
    s["y"].copy_(x)
    return s["y"]


# ── the framework's calls ────────────────────────────────────────────────────

def _kv8(M, s):
    c = s["case"]
    return M.Kv8Cache(
        format=FORMATS[c["format"]], n_kv_heads=c["kv_heads"], head_dim=c["hd"], block=c["block"],
        k=s["k"].data_ptr(), v=s["v"].data_ptr(), slot_stride=c["kv_heads"] * c["hd"],
        n_slots=s["k"].shape[0], k_scale=s["ks"].data_ptr(), v_scale=s["vs"].data_ptr(),
        seq_slots=s.get("seq_slots", 0), pages=s["pages"].data_ptr() if c["page"] else None,
        page_size=c["page"], max_pages=s["pages"].shape[1] if c["page"] else 0)


def _own_store(M, s):
    c = s["case"]
    if "args" not in s:      # a program fills these once and keeps them
        row = c["kv_heads"] * c["hd"]
        s["args"] = M.Kv8Store(
            cache=_kv8(M, s), type=IDS[c["dtype"]], n_seqs=c["seqs"], k=s["kx"].data_ptr(),
            v=s["vx"].data_ptr(), k_stride=row, v_stride=row, n_rows=s["total"],
            seq_start=s["seq_start"].data_ptr(), n_past=s["n_past"].data_ptr(),
            max_nodes=c["nodes"], max_kv=s["max_kv"])
    M.kv8_store_dev(s["args"])
    return {"k": s["k"], "ks": s["ks"], "v": s["v"], "vs": s["vs"]}


def _own_attn(M, s):
    c = s["case"]
    if "args" not in s:      # a program fills these once, with its workspace, and keeps them
        row = c["heads"] * c["hd"]
        s["args"] = M.Kv8Attention(
            cache=_kv8(M, s), type=IDS[c["dtype"]], n_seqs=c["seqs"], n_heads=c["heads"],
            q=s["q"].data_ptr(), q_stride=row, out=s["out"].data_ptr(), out_stride=row,
            n_rows=s["total"], seq_start=s["seq_start"].data_ptr(), n_past=s["n_past"].data_ptr(),
            mask=s["mask"].data_ptr() if "mask" in s else None,
            mask_words=s["mask"].shape[1] if "mask" in s else 0, max_nodes=c["nodes"],
            max_kv=s["max_kv"], scale=1 / math.sqrt(c["hd"]))
        s["ws"] = torch.empty(M.kv8_attention_workspace(s["args"]), device=GPU, dtype=torch.uint8)
    M.kv8_attention_dev(s["args"], s["ws"].data_ptr(), s["ws"].numel())
    return s["out"]


def _own_pool(M, s):
    if "args" not in s:      # a program fills these once, with its workspace, and keeps them
        s["list"] = _ints([[p.data_ptr(), p.shape[1] * 4, p.shape[1] * 4] for p in s["parts"]], np.int64)
        s["args"] = M.PagePool(
            n_pages=len(s["refs"]), n_seqs=s["pages"].shape[0], max_pages=s["pages"].shape[1],
            page_size=s["case"]["page"], n_parts=len(s["parts"]), parts=s["list"].data_ptr(),
            refs=s["refs"].data_ptr(), pages=s["pages"].data_ptr(), n_past=s["n_past"].data_ptr(),
            status=s["status"].data_ptr())
        s["ws"] = torch.empty(M.pages_workspace(s["args"]), device=GPU, dtype=torch.uint8)
        torch.cuda.synchronize()
    return s["args"], s["ws"].data_ptr(), s["ws"].numel()


def _own_beam(M, s):
    pool, ws, size = _own_pool(M, s)
    M.pages_fork_dev(pool, s["from"].data_ptr(), ws, size)
    M.pages_reserve_dev(pool, s["n_new"].data_ptr(), ws, size)
    return _pool(s)


def _own_compact(M, s):
    pool, ws, size = _own_pool(M, s)
    for now, then in (("pages", "pages0"), ("refs", "refs0")):
        M.copy_dev(s[now].data_ptr(), s[then].data_ptr(), 4 * s[now].numel())
    M.pages_compact_dev(pool, ws, size)
    return _pool(s)


def _own_logits(M, s):
    c = s["case"]
    if "args" not in s:      # a program fills these once and keeps them
        at = lambda k: s[k].data_ptr() if k in s else None  # noqa: E731
        s["args"] = M.Logits(
            type=IDS[c["dtype"]], out_type=IDS[c["out"]], n_rows=c["rows"], vocab=c["vocab"],
            x=at("x"), x_stride=c["vocab"], y=at("y"), y_stride=c["vocab"], hist=at("hist"),
            hist_start=at("hist_start"), repeat=at("repeat"), freq=at("freq"),
            presence=at("presence"), bias_id=at("bias_id"), bias=at("bias"),
            bias_start=at("bias_start"), allowed=at("allowed"), mask_row=at("mask_row"),
            mask_words=s["allowed"].shape[1] if "allowed" in s else 0, n_masks=c["masks"])
    M.logits_dev(s["args"])
    return s["y"]


def run(s):
    kind = s["case"]["kind"]
    if own:
        import mynah_amd as M
        return {"store": _own_store, "attn": _own_attn, "beam": _own_beam, "compact": _own_compact,
                "logits": _own_logits}[kind](M, s)
    return {"store": _plain_store, "attn": _plain_attn, "beam": _plain_beam,
            "compact": _plain_compact, "logits": _plain_logits}[kind](s)


# ── what a pass cannot do without ────────────────────────────────────────────

def work(case):
    kind = case["kind"]
    if kind in ("store", "attn"):
        # Sequences after the first are on average half as long, in both.
        size, some = DTYPES[case["dtype"]].itemsize, 1 + (case["seqs"] - 1) / 2
        rows, row = some * case["nodes"], case["kv_heads"] * case["hd"]
        if kind == "store":
            return {"bytes": 2 * rows * row * (size + 1) + 8 * rows * case["kv_heads"] / case["block"],
                    "flops": 4 * rows * row}
        kv = some * (case["past"] + case["nodes"] / 2)
        pairs = (1 + (case["seqs"] - 1) / 4) * case["nodes"] * (case["past"] + case["nodes"] / 2)
        return {"bytes": 2 * kv * (row + 4 * case["kv_heads"] / case["block"])
                + 2 * rows * case["heads"] * case["hd"] * size,
                "flops": 4 * case["hd"] * case["heads"] * pairs}
    if kind in ("beam", "compact"):
        page = case["layers"] * (2 * case["page"] * case["row"] + 8 * (case["row"] // 128))
        if kind == "beam":
            # Every continuation copies one page that is not full.
            moved, table = case["children"] * (1 - 1 / case["page"]), 1 + case["past"] * 0.75 / case["page"]
            entries = table * (case["parents"] + case["children"])
        else:
            moved, entries = case["live"] * (1 - case["live"] / case["pages"]), case["live"]
        return {"bytes": 2 * moved * page + 8 * entries, "flops": 0}
    n, vocab = case["rows"], case["vocab"]
    return {"bytes": n * vocab * (DTYPES[case["dtype"]].itemsize + DTYPES[case["out"]].itemsize)
            + 4 * (n * 0.75 * case["history"] + n * case["biases"] + case["masks"] * vocab / 32),
            "flops": n * vocab}


# ── the same results in 64 bits ──────────────────────────────────────────────

def _exact_store(case, seed):
    """Scales in 64 bits; which codes stand for the values is the format's, in 32 bits."""
    s = _prepare_store(case, seed)
    start, past = s["seq_start"].tolist(), s["n_past"].tolist()
    block, page = case["block"], case["page"]
    out = {"k": None, "v": None}
    for name, x in (("ks", s["kx"]), ("vs", s["vx"])):
        scales = s[name].double()
        amax = x.abs().amax(-1).double().clamp_min(AMAX_MIN)                  # [rows][kv heads]
        for b in range(case["seqs"]):
            n, n0 = start[b + 1] - start[b], past[b]
            for first in range(n0 // block * block, n0 + n, block):
                lo, hi = max(first, n0) - n0, min(first + block, n0 + n) - n0
                top = amax[start[b] + lo:start[b] + hi].amax(0)
                if case["format"] == "i8":
                    new = top / 127
                else:
                    new = torch.exp2(torch.ceil(torch.log2(top / 448)))
                if page:
                    at = (int(s["pages"][b, first // page]) * page + first % page) // block
                else:
                    at = (b * s["seq_slots"] + first) // block
                scales[at] = torch.maximum(new, scales[at]) if first < n0 else new
        out[name] = scales
    return out


def _exact_attn(case, seed):
    s = _prepare_attn(case, seed)
    out = torch.empty(s["q"].shape, device=GPU, dtype=torch.float64)
    start, past = s["seq_start"].tolist(), s["n_past"].tolist()
    group, page = case["heads"] // case["kv_heads"], case["page"]
    for b in range(case["seqs"]):
        n, n0 = start[b + 1] - start[b], past[b]
        if page:
            at = (s["pages"][b].long()[:, None] * page + torch.arange(page, device=GPU)).flatten()
            at = at[:n0 + n]
        else:
            at = torch.arange(b * s["seq_slots"], b * s["seq_slots"] + n0 + n, device=GPU)
        if "mask" in s:
            bits = s["mask"][start[b]:start[b + 1]].cpu().numpy().view(np.uint8)
            see = np.unpackbits(bits, axis=1, bitorder="little")[:, :n].astype(bool)
            hidden = torch.from_numpy(~see).to(GPU)
        else:
            hidden = torch.ones(n, n, device=GPU, dtype=torch.bool).triu(1)
        for g in range(case["kv_heads"]):
            k = _take(s["k"][:, g], at).double() * s["ks"][at // case["block"], g, None].double()
            v = _take(s["v"][:, g], at).double() * s["vs"][at // case["block"], g, None].double()
            kt = k.T.contiguous()
            for h in range(g * group, (g + 1) * group):
                x = s["q"][start[b]:start[b + 1], h].double() @ kt / case["hd"] ** 0.5
                x[:, n0:] = x[:, n0:].masked_fill(hidden, -math.inf)
                out[start[b]:start[b + 1], h] = x.softmax(-1) @ v
    return out


def _exact_pool(s, table, refs, past, status, moves):
    """The pool after the pages of `moves` (from, to) have been copied."""
    source, to = [torch.tensor(m, device=GPU, dtype=torch.long) for m in zip(*moves)] or [None] * 2
    for part in s["parts"]:
        if moves:
            part[to] = part[source]
    return {"pages": _ints(table), "refs": _ints(refs), "n_past": _ints(past),
            "status": _ints(status)} | {f"part{i}": p for i, p in enumerate(s["parts"])}


def _exact_beam(case, seed):
    s = _prepare_beam(case, seed)
    page, n_new = case["page"], s["n_new"].tolist()
    table, past, source = (s[k].tolist() for k in ("pages", "n_past", "from"))
    table, past = [list(table[f]) for f in source], [past[f] for f in source]
    holders = {}
    for b, row in enumerate(table):
        for p in row:
            if p >= 0:
                holders.setdefault(p, []).append(b)
    grows = {}
    spans = [range(n0 // page, -(-(n0 + k) // page) if k else 0) for n0, k in zip(past, n_new)]
    for b, span in enumerate(spans):
        for j in span:
            if table[b][j] >= 0:
                grows.setdefault(table[b][j], []).append(b)
    free = iter([p for p in range(len(s["refs"])) if p not in holders])
    moves = []
    for b, span in enumerate(spans):
        for j in span:
            p = table[b][j]
            if p >= 0 and (len(holders[p]) == 1 or (grows[p] == holders[p] and grows[p][0] == b)):
                continue
            table[b][j] = next(free)
            if p >= 0 and j * page < past[b]:
                moves.append((p, table[b][j]))
    refs = [0] * len(s["refs"])
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return _exact_pool(s, table, refs, past, [0, 0], moves)


def _exact_compact(case, seed):
    s = _prepare_compact(case, seed)
    refs, table = s["refs"].tolist(), s["pages"].tolist()
    live = sum(r > 0 for r in refs)
    to = [p for p in range(live) if refs[p] == 0]
    source = [p for p in range(live, len(refs)) if refs[p] > 0]
    new = dict(zip(source, to))
    table = [[new.get(p, p) for p in row] for row in table]
    for a, b in new.items():
        refs[b], refs[a] = refs[a], 0
    return _exact_pool(s, table, refs, s["n_past"].tolist(), [live, len(to)], list(new.items()))


def _exact_logits(case, seed):
    s = _prepare_logits(case, seed)
    y = s["x"].double()
    for r in range(case["rows"]):
        if "hist" in s:
            a, b = s["hist_start"][r:r + 2].tolist()
            ids, count = s["hist"][a:b].long().unique(return_counts=True)
            x, rep = y[r, ids], s["repeat"][r].double()
            x = torch.where(x > 0, x / rep, x * rep)
            y[r, ids] = x - s["freq"][r].double() * count - s["presence"][r].double()
        if "bias" in s:
            a, b = s["bias_start"][r:r + 2].tolist()
            y[r, s["bias_id"][a:b].long()] += s["bias"][a:b].double()
        if "allowed" in s and int(s["mask_row"][r]) >= 0:
            bits = s["allowed"][int(s["mask_row"][r])].cpu().numpy().view(np.uint8)
            ok = np.unpackbits(bits, bitorder="little")[:case["vocab"]].astype(bool)
            y[r] = torch.where(torch.from_numpy(ok).to(GPU), y[r], -math.inf)
    return y


def exact(case, seed):
    return {"store": _exact_store, "attn": _exact_attn, "beam": _exact_beam,
            "compact": _exact_compact, "logits": _exact_logits}[case["kind"]](case, seed)
