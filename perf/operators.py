"""The operators of one verification step of drafted tokens, as cases to time and compare.

  rope      mynah_hip_rope_dev: rotary positions of [tokens][heads][head_dim] rows, half or
            interleaved pairs, part of the head, frequencies scaled for long contexts
  qk        mynah_hip_qk_norm_rope_dev: a projection's q, k and v rows to the attention: RMSNorm
            of every q and k head, rotation, k and v stored in their cache slots
  tree      mynah_hip_tree_attention_dev: attention of drafted tokens (a tree, or a chain, or one
            token) of a ragged batch over contiguous or paged caches
  fp8       mynah_hip_fp8_matmat_dev: e4m3 weights with a scale per 128 x 128 block times e4m3
            activations with a scale per 128 values
  fp8_quant mynah_hip_fp8_quantize_dev, then the product: a projection of 16- or 32-bit activations

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
LAYOUTS = {"half": 0, "interleaved": 1}
BLOCK, E4M3_MAX, AMAX_MIN = 128, 448.0, 2.0 ** -100


def _rope(tokens, heads, hd, rot, layout, scaling, dtype, far=0):
    """far: the last position, beyond the prompt's own (a long context's tail)."""
    return {"kind": "rope", "tokens": tokens, "heads": heads, "hd": hd, "rot": rot,
            "layout": layout, "scaling": scaling, "dtype": dtype, "far": max(far, tokens)}


def _qk(tokens, heads, kv_heads, hd, layout, scaling, dtype, cache, slots):
    return {"kind": "qk", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "hd": hd,
            "layout": layout, "scaling": scaling, "dtype": dtype, "cache": cache, "slots": slots}


def _tree(seqs, nodes, past, heads, kv_heads, hd, dtype, page=0, shape="tree"):
    """page: positions of a cache page, 0 for one run of rows for each sequence. Sequences after
    the first are of any length up to the first's."""
    return {"kind": "tree", "seqs": seqs, "nodes": nodes, "past": past, "heads": heads,
            "kv_heads": kv_heads, "hd": hd, "dtype": dtype, "page": page, "shape": shape}


def _fp8(rows, cols, tokens, dtype, quantize=False):
    return {"kind": "fp8_quant" if quantize else "fp8", "rows": rows, "cols": cols,
            "tokens": tokens, "dtype": dtype}


def listed():
    return [
        # One decoded token's queries, at a position past the trained context.
        {"name": "rope_1tok", **_rope(1, 32, 128, 128, "half", "yarn", "f32", far=60_000)},
        # A long prompt's queries, half of each head rotated, interleaved pairs.
        {"name": "rope_prompt", **_rope(8192, 32, 128, 64, "interleaved", "linear", "bf16")},
        # The q/k/v rows of one decoded token of a 4B model into the f32 cache.
        {"name": "qk_1tok", **_qk(1, 32, 8, 128, "half", "none", "f32", "f32", 2304)},
        # A prompt chunk of 2047 tokens from f32 projections into a 16-bit cache.
        {"name": "qk_prompt", **_qk(2047, 32, 8, 128, "half", "yarn", "f32", "bf16", 4096)},
        # A 0.6B decode step at 513 positions: one token, latency counts.
        {"name": "tree_1tok_f32", **_tree(1, 1, 512, 16, 8, 128, "f32")},
        # A drafted tree of 24 nodes over the 4B model's 2048-token context, in f32.
        {"name": "tree_24_f32", **_tree(1, 24, 2048, 32, 8, 128, "f32")},
        # A serving batch: 16 ragged sequences, drafted trees, pages of 64 positions.
        {"name": "tree_batch_bf16", **_tree(16, 16, 8191, 32, 8, 128, "bf16", page=64)},
        # A wide tree over one very long context.
        {"name": "tree_long_f16", **_tree(1, 64, 130_001, 32, 8, 128, "f16", page=256)},
        # One token's projection of the 4B feed-forward.
        {"name": "fp8_1tok", **_fp8(9728, 2560, 1, "f32")},
        # A drafted tree's projection, activations quantised on the way.
        {"name": "fp8_quant_37tok", **_fp8(4096, 2560, 37, "bf16", quantize=True)},
        # A prompt's projection at the 1.7B shapes, 512 tokens.
        {"name": "fp8_512tok", **_fp8(6144, 2048, 512, "bf16")},
        # A batch of prompts through the 4B feed-forward.
        {"name": "fp8_8192tok", **_fp8(9728, 2560, 8192, "bf16")},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rope", "qk", "tree", "tree", "tree", "fp8", "fp8", "fp8_quant"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    layout = rng.choice(("half", "interleaved"))
    scaling = rng.choice(("none", "linear", "yarn", "bands"))
    if kind == "rope":
        hd = rng.choice((64, 80, 96, 128, 256))
        heads, rot = rng.randint(1, 40), rng.choice((hd, hd, hd // 2, hd // 16 * 8))
        tokens = min(_log(rng, 1, 9000), 33_000_000 // (heads * hd))
        return _rope(tokens, heads, hd, rot, layout, scaling, dtype,
                     far=rng.choice((0, 0, 40_960, 1_000_000)))
    if kind == "qk":
        hd = rng.choice((64, 80, 96, 128, 256))
        kv_heads, group = rng.randint(1, 8), rng.randint(1, 8)
        tokens = min(_log(rng, 1, 5000), 10_000_000 // (kv_heads * (group + 2) * hd))
        return _qk(tokens, kv_heads * group, kv_heads, hd, layout, scaling, dtype,
                   rng.choice((dtype, dtype, "bf16", "f16")), tokens + _log(rng, 1, 4000))
    if kind == "tree":
        kv_heads, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 5, 7, 8))
        nodes, seqs = rng.choice((1, _log(rng, 1, 80))), rng.choice((1, _log(rng, 1, 32)))
        hd = rng.choice((64, 128, 128, 256))
        most = 60_000_000 // (seqs * kv_heads * hd)
        most = min(most, 400_000_000 // (seqs * kv_heads * group * nodes))
        return _tree(seqs, nodes, _log(rng, 1, max(2, min(40_000, most))), kv_heads * group,
                     kv_heads, hd, dtype, rng.choice((0, 16, 64, 128)),
                     rng.choice(("tree", "tree", "chain")))
    cols = 16 * _log(rng, 8, 608)
    tokens = rng.choice((1, _log(rng, 1, 64), _log(rng, 65, 8192)))
    rows = min(_log(rng, 100, 12_000), 200_000_000_000 // (cols * tokens))
    return _fp8(rows, cols, tokens, dtype, kind == "fp8_quant")


# ── inputs ───────────────────────────────────────────────────────────────────

def _gen(seed, k):
    g = torch.Generator(device=GPU)
    g.manual_seed((int(seed) * 1_000_003 + k) % (1 << 62))
    return g


def _normal(seed, k, *shape):
    return torch.randn(*shape, generator=_gen(seed, k), device=GPU)


# Base, factor, trained context and the turns (or wavelength divisors) that bound the ramp.
THETA, FACTOR, TRAINED = 1e6, 4.0, 32_768
RAMP = {"yarn": (32.0, 1.0), "bands": (4.0, 1.0)}


def _freqs(case, rot):
    """Radians per position of each pair, and what cos and sin are multiplied by."""
    i = np.arange(rot // 2, dtype=np.float64)
    f = THETA ** (-2.0 * i / rot)
    hi, lo = RAMP.get(case["scaling"], (0.0, 0.0))
    if case["scaling"] == "linear":
        return f / FACTOR, 1.0
    if case["scaling"] == "yarn":
        def pair(turns):
            return rot * math.log(TRAINED / (turns * 2 * math.pi)) / (2 * math.log(THETA))
        a, b = max(math.floor(pair(hi)), 0), min(math.ceil(pair(lo)), rot - 1)
        ramp = np.clip((i - a) / max(b - a, 0.001), 0, 1)
        return f / FACTOR * ramp + f * (1 - ramp), 0.1 * math.log(FACTOR) + 1.0
    if case["scaling"] == "bands":
        keep = np.clip((TRAINED * f / (2 * math.pi) - lo) / (hi - lo), 0, 1)
        return f / FACTOR * (1 - keep) + f * keep, 1.0
    return f, 1.0


def _ancestors(case, rng, n):
    """[n][words] int32: bit j of row i where node i is, or descends from, node j."""
    words = (case["nodes"] + 31) // 32
    m = np.zeros((n, words), np.uint32)
    for i in range(n):
        parent = i - 1 if case["shape"] == "chain" else int(rng.integers(-1, i)) if i else -1
        if parent >= 0:
            m[i] = m[parent]
        m[i, i // 32] |= np.uint32(1 << (i % 32))
    return m.view(np.int32)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(GPU)


def _prepare_tree(case, seed):
    rng = np.random.default_rng((int(seed), 77))
    t, hd, kvh = DTYPES[case["dtype"]], case["hd"], case["kv_heads"]
    n, page = case["seqs"], case["page"]
    lengths = np.random.default_rng(case["past"])      # the case's own, whatever the seed
    past = np.concatenate([[case["past"]], lengths.integers(0, case["past"] + 1, n - 1)])
    nodes = np.concatenate([[case["nodes"]], lengths.integers(1, case["nodes"] + 1, n - 1)])
    max_kv = case["past"] + case["nodes"]
    s = {"case": case, "n_past": _ints(past), "max_kv": max_kv, "total": int(nodes.sum()),
         "seq_start": _ints(np.concatenate([[0], np.cumsum(nodes)])),
         "mask": _ints(np.concatenate([_ancestors(case, rng, int(k)) for k in nodes]))}
    if page:
        max_pages = -(-max_kv // page)
        s["pages"] = _ints(rng.permutation(n * max_pages).reshape(n, max_pages))
        rows = n * max_pages * page
    else:
        rows = n * max_kv
    # Normalised keys and queries: scores of a few units, some positions far above the rest.
    s["k"] = _normal(seed, 1, rows, kvh, hd).to(t)
    s["v"] = _normal(seed, 2, rows, kvh, hd).to(t)
    s["q"] = (1.5 * _normal(seed, 3, s["total"], case["heads"], hd)).to(t)
    s["out"] = torch.empty_like(s["q"])
    return s


def _to_e4m3(x):
    return x.to(torch.float8_e4m3fn)


def _quantize(x):
    """(e4m3 values, scales) of x [tokens][cols] in blocks of 128 along cols."""
    tokens, cols = x.shape
    nb = -(-cols // BLOCK)
    b = torch.nn.functional.pad(x, (0, nb * BLOCK - cols)).reshape(tokens, nb, BLOCK)
    amax = b.abs().amax(-1, keepdim=True).clamp_min(AMAX_MIN)
    q = _to_e4m3(b * (E4M3_MAX / amax)).reshape(tokens, -1)[:, :cols].contiguous()
    return q, (amax / E4M3_MAX).squeeze(-1).contiguous()


def prepare(case, seed):
    kind, t = case["kind"], DTYPES[case["dtype"]]
    if kind == "tree":
        return _prepare_tree(case, seed)
    if kind in ("rope", "qk"):
        rot = case.get("rot", case["hd"])
        f, mscale = _freqs(case, rot)
        n, hd = case["tokens"], case["hd"]
        last = case.get("far", case.get("slots"))
        s = {"case": case, "freqs": torch.from_numpy(f).to(GPU), "mscale": mscale,
             "pos": torch.arange(last - n, last, device=GPU, dtype=torch.int32)}
        if kind == "rope":
            s["x"] = _normal(seed, 1, n, case["heads"], hd).to(t)
            s["y"] = torch.empty_like(s["x"])
            return s
        ct, kvh, slots = DTYPES[case["cache"]], case["kv_heads"], case["slots"]
        s["qkv"] = _normal(seed, 1, n, case["heads"] + 2 * kvh, hd).to(t)
        s["qw"] = 1 + 0.1 * _normal(seed, 2, hd)
        s["kw"] = 1 + 0.1 * _normal(seed, 3, hd)
        # A cache in use: the tokens' slots are any free ones.
        s["slots"] = torch.randperm(slots, generator=_gen(seed, 4), device=GPU)[:n].int()
        s["k"] = _normal(seed, 5, slots, kvh, hd).to(ct)
        s["v"] = _normal(seed, 6, slots, kvh, hd).to(ct)
        s["q"] = torch.empty(n, case["heads"], hd, device=GPU, dtype=ct)
        return s
    rows, cols, tokens = case["rows"], case["cols"], case["tokens"]
    nr, nb = -(-rows // BLOCK), -(-cols // BLOCK)
    # Weights whose blocks differ in size, as trained ones do.
    ws = 2.0 ** (2 * torch.rand(nr, nb, generator=_gen(seed, 1), device=GPU) - 1) / 4000
    w = _to_e4m3((_normal(seed, 2, rows, cols) * 90).clamp(-E4M3_MAX, E4M3_MAX))
    x = _normal(seed, 3, tokens, cols)
    x *= torch.exp(0.7 * _normal(seed, 4, cols))        # some channels are larger than others
    s = {"case": case, "w": w, "ws": ws.contiguous(),
         "y": torch.empty(tokens, rows, device=GPU, dtype=t)}
    if kind == "fp8":
        s["xq"], s["xs"] = _quantize(x)
    else:
        s["x"] = x.to(t)
        s["xq"] = torch.empty(tokens, cols, device=GPU, dtype=torch.float8_e4m3fn)
        s["xs"] = torch.empty(tokens, nb, device=GPU)
    return s


# ── the operators in elementary torch operations ─────────────────────────────

def _rotated(x, s, rot):
    """x f32 [tokens][heads][hd] rotated to its positions."""
    a = s["pos"].double().unsqueeze(-1) * s["freqs"]
    cos = (a.cos() * s["mscale"]).float().unsqueeze(1)
    sin = (a.sin() * s["mscale"]).float().unsqueeze(1)
    if s["case"]["layout"] == "half":
        x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
    else:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _normed(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


def _plain_qk(s):
    c, x = s["case"], s["qkv"].float()
    h, kvh, ct = c["heads"], c["kv_heads"], DTYPES[c["cache"]]
    slots = s["slots"].long()
    q = _rotated(_normed(x[:, :h], s["qw"]), s, c["hd"])
    k = _rotated(_normed(x[:, h:h + kvh], s["kw"]), s, c["hd"])
    s["k"][slots] = k.to(ct)
    s["v"][slots] = x[:, h + kvh:].to(ct)
    return {"q": q.to(ct), "k": s["k"], "v": s["v"]}


def _plain_tree(s):
    c = s["case"]
    kvh, hd, n, group = c["kv_heads"], c["hd"], c["nodes"], c["heads"] // c["kv_heads"]
    start, past = s["seq_start"].long(), s["n_past"].long()
    pos = torch.arange(s["max_kv"], device=GPU)
    node = torch.arange(n, device=GPU)
    real = node < (start[1:] - start[:-1]).unsqueeze(1)                       # [seqs][nodes]
    row = torch.where(real, start[:-1].unsqueeze(1) + node, 0)
    if c["page"]:
        at = s["pages"].long()[:, pos // c["page"]] * c["page"] + pos % c["page"]
    else:
        at = torch.arange(c["seqs"], device=GPU).unsqueeze(1) * s["max_kv"] + pos
    length = past + start[1:] - start[:-1]
    at = torch.where(pos < length.unsqueeze(1), at, at[:, :1])
    k, v = s["k"][at].float(), s["v"][at].float()                # [seqs][kv][kv heads][hd]
    j = pos - past.unsqueeze(1)                                   # node of a position
    jc = j.clamp(0, n - 1).unsqueeze(1).expand(-1, n, -1)
    word = s["mask"][row].gather(2, jc >> 5)
    seen = (j < 0).unsqueeze(1) | ((j >= 0) & (j < n)).unsqueeze(1) & (((word >> (jc & 31)) & 1) == 1)
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


def _spread(scales, rows, cols):
    """[rows][cols] of scales given for blocks of 128 columns (and already for each row)."""
    return scales.repeat_interleave(BLOCK, 1)[:rows, :cols]


def _plain_fp8(s):
    c = s["case"]
    rows, cols, tokens = c["rows"], c["cols"], c["tokens"]
    xq, xs = (s["xq"], s["xs"]) if c["kind"] == "fp8" else _quantize(s["x"].float())
    w = s["w"].float() * _spread(s["ws"].repeat_interleave(BLOCK, 0), rows, cols)
    x = xq.float() * _spread(xs, tokens, cols)
    y = torch.matmul(x, w.t()).to(DTYPES[c["dtype"]])
    return {"y": y} if c["kind"] == "fp8" else {"y": y, "xq": xq, "xs": xs}


# ── the framework's calls ────────────────────────────────────────────────────

def _own_rope(M, s):
    c = s["case"]
    h, hd = c["heads"], c["hd"]
    M.rope_dev(IDS[c["dtype"]], LAYOUTS[c["layout"]], s["x"].data_ptr(), h * hd, hd,
               s["y"].data_ptr(), h * hd, hd, c["tokens"], h, hd, c["rot"],
               s["freqs"].data_ptr(), s["mscale"], s["pos"].data_ptr())
    return s["y"]


def _own_qk(M, s):
    c = s["case"]
    if "args" not in s:      # a program fills these once and keeps them
        h, kvh, hd = c["heads"], c["kv_heads"], c["hd"]
        x, size = s["qkv"].data_ptr(), s["qkv"].element_size()
        row = (h + 2 * kvh) * hd
        s["args"] = M.QkNormRope(
            type=IDS[c["dtype"]], out_type=IDS[c["cache"]], layout=LAYOUTS[c["layout"]],
            tokens=c["tokens"], n_heads=h, n_kv_heads=kvh, head_dim=hd, rot_dim=hd,
            q=x, k=x + h * hd * size, v=x + (h + kvh) * hd * size, q_stride=row, k_stride=row,
            v_stride=row, q_norm=s["qw"].data_ptr(), k_norm=s["kw"].data_ptr(), eps=1e-6,
            mscale=s["mscale"], freqs=s["freqs"].data_ptr(), pos=s["pos"].data_ptr(),
            slots=s["slots"].data_ptr(), n_slots=c["slots"], q_out=s["q"].data_ptr(),
            q_out_stride=h * hd, k_cache=s["k"].data_ptr(), v_cache=s["v"].data_ptr(),
            slot_stride=kvh * hd)
    M.qk_norm_rope_dev(s["args"])
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _own_tree(M, s):
    c = s["case"]
    if "args" not in s:      # a program fills these once, with its workspace, and keeps them
        kvh, hd = c["kv_heads"], c["hd"]
        paged = c["page"] > 0
        s["args"] = M.TreeAttention(
            type=IDS[c["dtype"]], n_seqs=c["seqs"], n_heads=c["heads"], n_kv_heads=kvh,
            head_dim=hd, q=s["q"].data_ptr(), q_stride=c["heads"] * hd, out=s["out"].data_ptr(),
            out_stride=c["heads"] * hd, n_rows=s["total"], k_cache=s["k"].data_ptr(),
            v_cache=s["v"].data_ptr(), slot_stride=kvh * hd, n_slots=s["k"].shape[0],
            seq_slots=0 if paged else s["max_kv"], pages=s["pages"].data_ptr() if paged else None,
            page_size=c["page"], max_pages=s["pages"].shape[1] if paged else 0,
            seq_start=s["seq_start"].data_ptr(), n_past=s["n_past"].data_ptr(),
            mask=s["mask"].data_ptr() if c["shape"] == "tree" else None,
            mask_words=s["mask"].shape[1], max_nodes=c["nodes"], max_kv=s["max_kv"],
            scale=1 / math.sqrt(hd))
        s["ws"] = torch.empty(M.tree_attention_workspace(s["args"]), device=GPU, dtype=torch.uint8)
    M.tree_attention_dev(s["args"], s["ws"].data_ptr(), s["ws"].numel())
    return s["out"]


def _own_fp8(M, s):
    c = s["case"]
    rows, cols, tokens, xq, xs = c["rows"], c["cols"], c["tokens"], s["xq"], s["xs"]
    if c["kind"] == "fp8_quant":
        M.fp8_quantize_dev(IDS[c["dtype"]], s["x"].data_ptr(), cols, tokens, cols, xq.data_ptr(),
                           xs.data_ptr())
    M.fp8_matmat_dev(s["w"].data_ptr(), s["ws"].data_ptr(), rows, cols, xq.data_ptr(),
                     xs.data_ptr(), IDS[c["dtype"]], s["y"].data_ptr(), tokens)
    return {"y": s["y"]} if c["kind"] == "fp8" else {"y": s["y"], "xq": xq, "xs": xs}


def run(s):
    kind = s["case"]["kind"]
    if own:
        import mynah_amd as M
        if kind == "rope":
            return _own_rope(M, s)
        if kind == "qk":
            return _own_qk(M, s)
        if kind == "tree":
            return _own_tree(M, s)
        return _own_fp8(M, s)
    if kind == "rope":
        return _rotated(s["x"].float(), s, s["case"]["rot"]).to(s["x"].dtype)
    if kind == "qk":
        return _plain_qk(s)
    if kind == "tree":
        return _plain_tree(s)
    return _plain_fp8(s)


# ── what a pass cannot do without ────────────────────────────────────────────

def work(case):
    kind, size = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind == "rope":
        n = case["tokens"] * case["heads"] * case["hd"]
        return {"bytes": 2 * n * size + 4 * case["tokens"] + 4 * case["rot"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    if kind == "qk":
        qk = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["hd"]
        v = case["tokens"] * case["kv_heads"] * case["hd"]
        return {"bytes": (qk + v) * (size + DTYPES[case["cache"]].itemsize) + 8 * case["tokens"],
                "flops": 7 * qk}
    if kind == "tree":
        # Sequences after the first are on average half as long, in both.
        some = 1 + (case["seqs"] - 1) / 2
        rows, kv = some * case["nodes"], some * (case["past"] + case["nodes"] / 2)
        pairs = (1 + (case["seqs"] - 1) / 4) * case["nodes"] * (case["past"] + case["nodes"] / 2)
        return {"bytes": size * case["hd"] * (2 * rows * case["heads"] + 2 * kv * case["kv_heads"]),
                "flops": 4 * case["hd"] * case["heads"] * pairs}
    rows, cols, tokens = case["rows"], case["cols"], case["tokens"]
    x = tokens * cols * (size if kind == "fp8_quant" else 1)
    return {"bytes": rows * cols + x + tokens * rows * size + rows * cols / 4096
            + (tokens * cols / 32 if kind == "fp8" else 0), "flops": 2 * rows * cols * tokens}


# ── the same results in 64 bits ──────────────────────────────────────────────

def _turn64(x, case, rot, pos):
    f, mscale = _freqs(case, rot)
    a = pos.double()[:, None, None] * torch.from_numpy(f).to(GPU)
    z = torch.polar(torch.full_like(a, mscale), a)
    y = x.clone()
    if case["layout"] == "half":
        r = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * z
        y[..., :rot // 2], y[..., rot // 2:rot] = r.real, r.imag
    else:
        r = torch.complex(x[..., 0:rot:2].contiguous(), x[..., 1:rot:2].contiguous()) * z
        y[..., 0:rot:2], y[..., 1:rot:2] = r.real, r.imag
    return y


def _exact_tree(case, seed):
    s = _prepare_tree(case, seed)
    out = torch.empty(s["q"].shape, device=GPU, dtype=torch.float64)
    start, past, mask = s["seq_start"].tolist(), s["n_past"].tolist(), s["mask"].cpu().numpy()
    group, page = case["heads"] // case["kv_heads"], case["page"]
    for b in range(case["seqs"]):
        n, n0 = start[b + 1] - start[b], past[b]
        if page:
            at = (s["pages"][b].long()[:, None] * page + torch.arange(page, device=GPU)).flatten()
            at = at[:n0 + n]
        else:
            at = torch.arange(b * s["max_kv"], b * s["max_kv"] + n0 + n, device=GPU)
        bits = mask[start[b]:start[b + 1]].view(np.uint32)
        see = np.unpackbits(bits.view(np.uint8), axis=1, bitorder="little")[:, :n].astype(bool)
        hidden = torch.from_numpy(~see).to(GPU)
        for h in range(case["heads"]):
            k, v = s["k"][at, h // group].double(), s["v"][at, h // group].double()
            x = s["q"][start[b]:start[b + 1], h].double() @ k.T.contiguous() / case["hd"] ** 0.5
            x[:, n0:] = x[:, n0:].masked_fill(hidden, -math.inf)
            out[start[b]:start[b + 1], h] = x.softmax(-1) @ v
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "tree":
        return _exact_tree(case, seed)
    s = prepare(case, seed)
    if kind == "rope":
        return _turn64(s["x"].double(), case, case["rot"], s["pos"])
    if kind == "qk":
        h, kvh, x = case["heads"], case["kv_heads"], s["qkv"].double()
        r = (x.square().sum(-1, keepdim=True) / case["hd"] + 1e-6) ** -0.5
        q = _turn64((x * r)[:, :h] * s["qw"].double(), case, case["hd"], s["pos"])
        k = _turn64((x * r)[:, h:h + kvh] * s["kw"].double(), case, case["hd"], s["pos"])
        kc, vc = s["k"].double(), s["v"].double()
        kc[s["slots"].long()], vc[s["slots"].long()] = k, x[:, h + kvh:]
        return {"q": q, "k": kc, "v": vc}
    # Which 8-bit values stand for the activations is the format's, in 32 bits.
    xq, xs = (s["xq"], s["xs"]) if kind == "fp8" else _quantize(s["x"].float())
    y = torch.zeros(case["tokens"], case["rows"], device=GPU, dtype=torch.float64)
    scale = s["ws"].double().repeat_interleave(BLOCK, 0)[:case["rows"]]
    for b in range(xs.shape[1]):
        at = slice(b * BLOCK, min((b + 1) * BLOCK, case["cols"]))
        part = xq[:, at].double() @ s["w"][:, at].double().T.contiguous()
        y += part * xs[:, b:b + 1].double() * scale[:, b]
    if kind == "fp8":
        return {"y": y}
    x = torch.nn.functional.pad(s["x"].double(), (0, -case["cols"] % BLOCK))
    amax = x.reshape(case["tokens"], -1, BLOCK).abs().amax(-1)
    return {"y": y, "xq": None, "xs": amax.clamp_min(AMAX_MIN) / E4M3_MAX}
