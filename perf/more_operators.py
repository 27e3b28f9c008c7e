"""Performance cases of a decoder layer's operators beside its matvecs: norms
around a block, rotary positions of several axes, and attention over the paged
8-bit cache with first tokens that stay visible or a prefix that a batch shares.

A case is a dict of plain values; "kind" names the operator:

  norm    the block's result normalized, gated, scaled and added to the residual
          stream, and that normalized for the next block
  turn    rotary positions of several axes (time, height, width) applied to the
          heads of a row of tokens
  append  new keys and values into the cache at positions of several axes, the
          queries turned with them
  sink    attention of the new tokens' queries over the first tokens of their
          sequence and a sliding window
  shared  attention of a batch whose sequences begin with the same pages

With `own` false, run() computes them from elementary torch operations; with
`own` true, it calls modgrad_amd.norm and modgrad_amd.kvcache. Both work on the
same state; the cache's is

  k       [pages][kv heads][page tokens][head dim]   8-bit values (bytes)
  v       [pages][kv heads][head dim][page tokens]   8-bit values (bytes)
  scales  [pages][kv heads]                          f32, one for k, one for v
  table   [sequences][most pages]                    page of each block of tokens
  length  [sequences]                                tokens with the new ones
  cu      [sequences + 1]                            first new token of each sequence
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

MOST = {"i8": 127.0, "e4m3": 448.0}
EPS = 1e-6
N_POS = 8192  # positions of a rotary table


# ------------------------------------------------------------------- cases --

def listed():
    heads = {"q_heads": 28, "kv_heads": 4, "head_dim": 128}  # of a 7B-class decoder
    wide = {"q_heads": 16, "kv_heads": 8, "head_dim": 256}
    small = {"q_heads": 14, "kv_heads": 2, "head_dim": 64}   # of a 0.5B-class one
    return [
        # one decoded token after a block whose result is normalized too: launch latency
        {"name": "norm_decode_1", "kind": "norm", "rows": 1, "hidden": 3584, "post": True, "gate": "none",
         "h_scale": 1.0, "x_scale": 1.0, "pre": True, "out": "f32"},
        # a served batch: each token's own gate (a conditioned block), the branch scaled down
        {"name": "norm_gated_37", "kind": "norm", "rows": 37, "hidden": 896, "post": False, "gate": "row",
         "h_scale": 1.0, "x_scale": 0.22, "pre": True, "out": "f32"},
        # a long prompt, both norms and a gate for each channel; the result feeds the f16 prefill GEMM
        {"name": "norm_prompt_4096", "kind": "norm", "rows": 4096, "hidden": 3584, "post": True, "gate": "channel",
         "h_scale": 1.0, "x_scale": 0.5, "pre": True, "out": "f16"},
        # a few decoded tokens behind a picture
        {"name": "turn_tokens_7", "kind": "turn", "tokens": 7, "heads": 28, "head_dim": 128,
         "sections": "16,24,24", "order": "blocks", "own": False, "half": True},
        # the patches of a picture of 70 x 70: rows and columns have the same frequencies
        {"name": "turn_patches_4900", "kind": "turn", "tokens": 4900, "heads": 16, "head_dim": 80,
         "sections": "20,20", "order": "blocks", "own": True, "half": True},
        # one token for each of 33 conversations about pictures
        {"name": "append_decode_33", "kind": "append", **heads, "seqs": 33, "new": 1, "past": 2000, "page": 16,
         "format": "i8", "sections": "16,24,24", "order": "blocks", "half": True, "ragged": True},
        # prompts of text and pictures, the axes' pairs in turn
        {"name": "append_pictures_3", "kind": "append", **heads, "seqs": 3, "new": 2500, "past": 700, "page": 64,
         "format": "e4m3", "sections": "24,20,20", "order": "turns", "half": True, "ragged": True},
        # one endless conversation: the middle of its cache has been given back
        {"name": "sink_decode_1", "kind": "sink", **heads, "seqs": 1, "new": 1, "past": 60000, "page": 64,
         "format": "i8", "window": 2048, "sinks": 4, "softcap": 0.0, "out": "f32", "ragged": False},
        # pieces of prompts over a long past, more first tokens than a tile has
        {"name": "sink_pieces_4", "kind": "sink", **wide, "seqs": 4, "new": 250, "past": 9000, "page": 32,
         "format": "e4m3", "window": 1000, "sinks": 100, "softcap": 50.0, "out": "f32", "ragged": True},
        # a few answers to one short instruction
        {"name": "shared_decode_6", "kind": "shared", **small, "seqs": 6, "new": 1, "prefix": 1500, "past": 100,
         "page": 32, "format": "e4m3", "softcap": 0.0, "out": "f32", "ragged": True},
        # a served batch behind one long instruction
        {"name": "shared_decode_64", "kind": "shared", **heads, "seqs": 64, "new": 1, "prefix": 12000, "past": 1500,
         "page": 64, "format": "i8", "softcap": 0.0, "out": "f32", "ragged": True},
        # questions of many tokens about one document; the result feeds the f16 prefill GEMM
        {"name": "shared_questions_8", "kind": "shared", **heads, "seqs": 8, "new": 200, "prefix": 10000, "past": 300,
         "page": 16, "format": "i8", "softcap": 0.0, "out": "f16", "ragged": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _parts(rng, total, n):
    """n whole numbers of 1 and more with this sum, none twice as large as their mean or more."""
    while True:
        cuts = sorted(rng.sample(range(1, total), n - 1))
        p = [b - a for a, b in zip([0] + cuts, cuts + [total])]
        if max(p) * n < 2 * total:
            return ",".join(map(str, p))


def draw(rng):
    kind = rng.choice(["norm", "norm", "turn", "append", "append", "sink", "sink", "sink", "shared", "shared", "shared"])
    if kind == "norm":
        hidden = rng.choice([896, 3584, 4864, _log(rng, 50, 16000)])
        return {"kind": kind, "rows": _log(rng, 1, 2800 * 3584 // hidden), "hidden": hidden,
                "post": rng.random() < 0.6, "gate": rng.choice(["none", "channel", "row"]),
                "h_scale": rng.choice([1.0, 0.75]), "x_scale": rng.choice([1.0, 0.22]), "pre": rng.random() < 0.8,
                "out": rng.choice(["f32", "f16"])}
    if kind == "turn":
        d = rng.choice([64, 72, 80, 96, 128])
        heads, rot, alone = rng.randint(1, 28), rng.choice([d, d, d // 2]), rng.random() < 0.4
        return {"kind": kind, "tokens": _log(rng, 1, 4900 * 16 * 80 // (heads * d)), "heads": heads, "head_dim": d,
                "sections": _parts(rng, rot // 2, rng.randint(2, 4)), "order": rng.choice(["blocks", "turns"]),
                "own": alone, "half": rng.random() < 0.6}
    kv = rng.choice([1, 2, 4, 8])
    d = rng.choice([64, 96, 128, 256])
    case = {"kind": kind, "q_heads": kv * rng.randint(1, 8), "kv_heads": kv, "head_dim": d,
            "page": rng.choice([16, 32, 64, 128]), "format": rng.choice(["i8", "e4m3"]), "ragged": rng.random() < 0.7}
    if kind == "append":
        case["seqs"] = _log(rng, 1, 48)
        most = 4000 * 36 * 128 // (case["seqs"] * (case["q_heads"] + 2 * kv) * d)
        case["new"] = rng.choice([1, _log(rng, 1, max(2, most))])
        case.update(past=_log(rng, 1, 3000), sections=_parts(rng, rng.choice([d, d, d // 2]) // 2, rng.randint(2, 4)),
                    order=rng.choice(["blocks", "turns"]), half=rng.random() < 0.6)
        return case
    case["softcap"] = rng.choice([0.0, 0.0, 30.0])
    case["out"] = rng.choice(["f32", "f32", "f16"])
    case["new"] = rng.choice([1, 1, rng.randint(2, 6), _log(rng, 7, 1500)])
    if kind == "sink":
        case.update(seqs=_log(rng, 1, 32), sinks=_log(rng, 1, 300), window=_log(rng, 20, 5000))
        case["past"] = _log(rng, 1, max(2, min(60000, 2000000 // (case["seqs"] * kv * d // 32))))
    else:
        case.update(seqs=_log(rng, 2, 64), prefix=_log(rng, 60, 20000))
        case["past"] = _log(rng, 1, max(2, min(4000, 2000000 // (case["seqs"] * kv * d // 32))))
    # no more pairs than half of the largest case's
    pairs = 8 * 100 * 10000 * 28 * 128 // 2
    while case["new"] > 1 and (case["seqs"] * case["new"] * case["q_heads"] * d
                               * (case["past"] + case["new"] + case.get("prefix", 0)) > pairs):
        case["new"] = max(1, case["new"] // 2)
    return case


def _shares(n):
    """n shares in (0, 1], the first 1: how ragged lengths are spread."""
    return [1.0] + [((b * 0.6180339887) % 1.0) ** 2 for b in range(1, n)]


def _lengths(case):
    """(new tokens, past tokens behind any prefix) of each sequence: the same for every seed."""
    n = case["seqs"]
    if not case["ragged"]:
        return [case["new"]] * n, [case["past"]] * n
    share = _shares(n)
    return ([max(1, int(case["new"] * s)) for s in share],
            [max(1, int(case["past"] * s)) for s in share[1:] + share[:1]])


def _sections(case):
    return [int(n) for n in case["sections"].split(",")]


def _pairs(case):
    """(axis, column of the rotary table) of each pair that turns."""
    sections, out = _sections(case), []
    if case["order"] == "blocks":
        out = [(a, i) for a, n in enumerate(sections) for i in range(n)]
    else:  # one pair for each axis in turn, until it has its own
        out = [(a, i) for i in range(max(sections)) for a, n in enumerate(sections) if i < n]
    return out if case.get("own") else [(a, p) for p, (a, _) in enumerate(out)]


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _payload(g, fmt, *shape):
    """Bytes of 8-bit values spread as those of quantized normal ones."""
    n = math.prod(shape)
    out = torch.empty(n, dtype=torch.uint8, device="cuda")
    for a in range(0, n, 1 << 26):
        m = min(1 << 26, n - a)
        x = _randn(g, m).mul_(MOST[fmt] / 3).clamp_(-MOST[fmt], MOST[fmt])
        q = x.round_().to(torch.int8) if fmt == "i8" else x.to(torch.float8_e4m3fn)
        out[a:a + m] = q.view(torch.uint8)
    return out.view(shape)


def _page_scales(g, fmt, *shape):
    """Scales that give values near N(0, 1), some pages quieter or louder."""
    return (3 / MOST[fmt]) * torch.exp(0.3 * _randn(g, *shape))


def _cache(case, g):
    """Pages in no order. A prefix's whole pages are in every sequence's list; its last part and what follows are a
    sequence's own. Pages that no new token sees are in no list (sink)."""
    new, past = _lengths(case)
    page, h, d, prefix = case["page"], case["kv_heads"], case["head_dim"], case.get("prefix", 0)
    lens = [prefix + a + b for a, b in zip(new, past)]
    common = prefix // page
    table = np.full((len(lens), max(-(-n // page) for n in lens)), -1, np.int64)
    table[:, :common] = np.arange(common)
    at = common
    for b, n in enumerate(lens):
        slots = np.arange(common, -(-n // page))
        if case["kind"] == "sink":
            seen = n - new[b] - case["window"] + 1
            slots = slots[(slots * page < case["sinks"]) | ((slots + 1) * page > seen)]
        table[b, slots] = at + np.arange(len(slots))
        at += len(slots)
    pages = at + 3
    ids = torch.randperm(pages, generator=g, device="cuda").cpu().numpy()
    table = np.where(table >= 0, ids[table], -1).astype(np.int32)
    return {"k": _payload(g, case["format"], pages, h, page, d), "v": _payload(g, case["format"], pages, h, d, page),
            "k_scale": _page_scales(g, case["format"], pages, h), "v_scale": _page_scales(g, case["format"], pages, h),
            "table": torch.from_numpy(table).cuda(), "length": torch.tensor(lens, dtype=torch.int32, device="cuda"),
            "cu": torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32),
            "tokens": sum(new), "max_new": max(new), "lens": lens, "new": new, "host_table": table}


def _rope_table(n_pos, cols, base=10000.0):
    p = torch.arange(n_pos, device="cuda", dtype=torch.float64)
    a = p[:, None] * base ** (-torch.arange(cols, device="cuda", dtype=torch.float64) / cols)
    return torch.stack([a.cos(), a.sin()], 2).float()


def _positions(n, axes, first, rng):
    """[axes][n]: a run of text, a picture or film of some columns, text again."""
    text = int(rng.integers(0, n // 4 + 1))
    cols = int(rng.integers(1, max(2, int(math.sqrt(n)))))
    grid = (n - text) * 3 // 4 // cols * cols
    t = np.arange(n)
    out = np.empty((axes, n), np.int64)
    out[:] = first + t
    i = np.arange(grid)
    rows = max(1, grid // cols // int(rng.integers(1, 4)))
    parts = [i // (cols * rows), i // cols % rows, i % cols]  # frame, row, column
    for a in range(axes):
        out[a, text:text + grid] = first + text + parts[(a + 3 - min(axes, 3)) % 3]
    after = out[:, text:text + grid].max(initial=first + text - 1) + 1
    out[:, text + grid:] = after + np.arange(n - text - grid)
    return np.minimum(out, N_POS - 1).astype(np.int32)


def prepare(case, seed):
    g, rng = _gen(seed), np.random.default_rng(int(seed))
    kind = case["kind"]
    s = {"case": case}
    if kind == "norm":
        n, d = case["rows"], case["hidden"]
        s["h"] = 3.0 * _randn(g, n, d)
        s["h"][:, ::97] *= 20.0  # some channels of a residual stream are loud
        s["x"] = 0.3 * _randn(g, n, d)
        s["post_w"] = 0.5 + torch.rand(d, device="cuda", generator=g) if case["post"] else None
        s["gate"] = {"none": None, "channel": 0.1 + 0.3 * _randn(g, d), "row": 0.5 + _randn(g, n, d)}[case["gate"]]
        s["norm_w"] = 0.5 + torch.rand(d, device="cuda", generator=g) if case["pre"] else None
        s["h_out"] = torch.empty(n, d, device="cuda")
        s["y"] = None
        if case["pre"]:
            s["y"] = torch.empty(n, d, device="cuda", dtype=torch.float32 if case["out"] == "f32" else torch.float16)
        if own:
            from modgrad_amd.norm import BlockNorm
            s["norm"] = BlockNorm(d, EPS, post_w=s["post_w"], gate=s["gate"] if case["gate"] == "channel" else None,
                                  norm_w=s["norm_w"], h_scale=case["h_scale"], x_scale=case["x_scale"])
        return s
    if kind in ("turn", "append"):
        sections = _sections(case)
        s["axes"] = len(sections)
        s["map"] = _pairs(case)
        s["rope_table"] = _rope_table(N_POS, max(sections) if case.get("own") else sum(sections))
        s["pair_axis"] = torch.tensor([a for a, _ in s["map"]], device="cuda")
        s["pair_col"] = torch.tensor([c for _, c in s["map"]], device="cuda")
        if own:
            from modgrad_amd.kvcache import RopeAxes, RopeTable
            s["rope"] = RopeTable.wrap(s["rope_table"], half=case["half"])
            s["rope_axes"] = RopeAxes(sections, order=case["order"], own=case.get("own", False))
    if kind == "turn":
        s["x"] = _randn(g, case["tokens"], case["heads"], case["head_dim"])
        s["y"] = torch.empty_like(s["x"])
        s["pos"] = torch.from_numpy(_positions(case["tokens"], s["axes"], int(rng.integers(0, 500)), rng)).cuda()
        return s
    s["cache"] = c = _cache(case, g)
    hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "append":
        # one row for each token, [q | k | v] as the fused projection leaves it; some channels of k are loud
        s["qkv"] = _randn(g, c["tokens"], (hq + 2 * h) * d)
        s["qkv"][:, hq * d:(hq + h) * d:37] *= 4.0
        s["q_out"] = torch.empty(c["tokens"], hq * d, device="cuda")
        # positions count a picture's rows or columns, so they fall behind the cache's
        s["pos"] = torch.from_numpy(np.concatenate(
            [_positions(m, s["axes"], (n - m) * 3 // 4, rng) for n, m in zip(c["lens"], c["new"])], 1)).cuda()
        page = case["page"]
        touched = [int(c["host_table"][b, i]) for b, (n, new) in enumerate(zip(c["lens"], c["new"]))
                   for i in range((n - new) // page, (n - 1) // page + 1)]
        s["touched"] = torch.tensor(touched, dtype=torch.int32, device="cuda")
        s["k_out"] = torch.empty(len(touched), h, page, d, device="cuda")
        s["v_out"] = torch.empty(len(touched), h, page, d, device="cuda")
    else:
        s["q"] = 2.0 * _randn(g, c["tokens"], hq * d)
        s["out"] = torch.empty(c["tokens"], hq * d, device="cuda",
                               dtype=torch.float32 if case["out"] == "f32" else torch.float16)
    if own:
        from modgrad_amd.kvcache import KvCache
        s["handle"] = KvCache.wrap(c["k"], c["v"], c["k_scale"], c["v_scale"], c["table"], c["length"],
                                   cu_tokens=c["cu"] if c["max_new"] > 1 else None, fmt=case["format"])
        if kind != "append":
            # whole pages are what the sequences' lists have in common
            s["shared"] = case.get("prefix", 0) // case["page"] * case["page"]
            s["workspace"] = s["handle"].attention_workspace(hq, c["tokens"], c["max_new"], shared=s["shared"])
    return s


# ------------------------------------------------------------ the operators --

def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _own_norm(s):
    case, y = s["case"], s["y"]
    s["norm"].apply(s["h"].data_ptr(), s["x"].data_ptr(), case["rows"], h_out=s["h_out"].data_ptr(),
                    y=0 if y is None else y.data_ptr(), y_f16=case["out"] == "f16",
                    gate=s["gate"].data_ptr() if case["gate"] == "row" else 0)
    return s["h_out"] if y is None else (s["h_out"], y)


def _own_turn(s):
    case, x, y = s["case"], s["x"], s["y"]
    s["rope"].apply(x.data_ptr(), y.data_ptr(), s["pos"].data_ptr(), case["tokens"], case["heads"], case["head_dim"],
                    axes=s["rope_axes"])
    return y


def _own_append(s):
    case, c, qkv = s["case"], s["cache"], s["qkv"]
    hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    row, at = qkv.shape[1], qkv.data_ptr()
    s["handle"].append(at + 4 * hq * d, at + 4 * (hq + h) * d, row, c["tokens"], c["max_new"], rope=s["rope"],
                       q=at, q_stride=row, q_out=s["q_out"].data_ptr(), q_out_stride=hq * d, n_q_heads=hq,
                       axes=s["rope_axes"], pos=s["pos"].data_ptr())
    s["handle"].dequant(s["touched"].data_ptr(), len(s["touched"]), s["k_out"].data_ptr(), s["v_out"].data_ptr())
    return s["q_out"], s["k_out"], s["v_out"]


def _own_attn(s):
    case, c = s["case"], s["cache"]
    d = case["q_heads"] * case["head_dim"]
    s["handle"].attend(s["q"].data_ptr(), d, case["q_heads"], s["out"].data_ptr(), d, c["tokens"], c["max_new"],
                       scale=case["head_dim"] ** -0.5, softcap=case["softcap"], window=case.get("window", 0),
                       sinks=case.get("sinks", 0), shared=s["shared"], out_f16=case["out"] == "f16",
                       workspace=s["workspace"])
    return s["out"]


_own = {"norm": _own_norm, "turn": _own_turn, "append": _own_append, "sink": _own_attn, "shared": _own_attn}


def _plain_norm(s):
    case, z = s["case"], s["x"]
    if case["post"]:
        z = z * torch.rsqrt((z * z).mean(1, keepdim=True) + EPS) * s["post_w"]
    if s["gate"] is not None:
        z = z * s["gate"]
    h = case["h_scale"] * s["h"] + case["x_scale"] * z
    s["h_out"].copy_(h)
    if s["y"] is None:
        return s["h_out"]
    s["y"].copy_(h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["norm_w"])
    return s["h_out"], s["y"]


def _turns(s):
    """(cos, sin) of each token's pairs in 64 bits, [tokens, pairs, 2]."""
    at = s["pos"].long()[s["pair_axis"]].t()
    return s["rope_table"][at, s["pair_col"]].double()


def _rotate(x, cs, half):
    """x [tokens, heads, dim] in 64 bits, cs [tokens, pairs, 2]."""
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    x, rot = x.double(), 2 * cs.shape[1]
    y = x.clone()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., a] = x[..., a] * c - x[..., b] * n
    y[..., b] = x[..., a] * n + x[..., b] * c
    return y


def _plain_turn(s):
    s["y"].copy_(_rotate(s["x"], _turns(s), s["case"]["half"]))
    return s["y"]


def _values(bytes_, fmt):
    return bytes_.view(torch.int8).float() if fmt == "i8" else bytes_.view(torch.float8_e4m3fn).float()


def _quantize(x, fmt):
    """64-bit values in units of their scale -> the 8-bit value's bytes:
    nearest, ties to even, saturating, NaN as 0."""
    x = torch.nan_to_num(x, nan=0.0, posinf=MOST[fmt], neginf=-MOST[fmt]).clamp(-MOST[fmt], MOST[fmt])
    if fmt == "i8":
        return x.round().to(torch.int8).view(torch.uint8)
    e = torch.frexp(x)[1].sub(4).clamp(min=-9)  # the exponent of the last of 3 fraction bits
    step = torch.ldexp(torch.ones_like(x), e)
    return ((x / step).round() * step).float().to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_append(s):
    case, c = s["case"], s["cache"]
    hq, h, d, page, fmt = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["format"]
    q, k, v = s["qkv"].split([hq * d, h * d, h * d], 1)
    t = torch.arange(c["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(c["cu"], t, right=True) - 1
    place = (c["length"][seq] - c["cu"][seq + 1] + t).long()
    pg, off = c["table"][seq, place // page].long(), place % page
    cs = _turns(s)
    s["q_out"].copy_(_rotate(q.view(-1, hq, d), cs, case["half"]).view(-1, hq * d))
    k = _rotate(k.view(-1, h, d), cs, case["half"])
    touched = s["touched"].long()
    n = len(touched)
    index = torch.empty(c["k"].shape[0], dtype=torch.long, device="cuda")
    index[touched] = torch.arange(n, device="cuda")
    at = index[pg]
    first = torch.full((n,), page, device="cuda").scatter_reduce(0, at, off, "amin")
    s["k_out"].copy_(_append_one(c["k"], c["k_scale"], k, fmt, touched, at, off, first))
    # values are held [dim][token]
    s["v_out"].copy_(_append_one(c["v"].transpose(2, 3), c["v_scale"], v.reshape(-1, h, d).double(), fmt, touched, at,
                                 off, first))
    return s["q_out"], s["k_out"], s["v_out"]


def _append_one(bytes_, scale, x, fmt, touched, at, off, first):
    """bytes_ [pages, heads, tokens, dim] (a view), x [new tokens, heads, dim]."""
    n, h, page = len(touched), x.shape[1], bytes_.shape[2]
    size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(2)
    size = torch.zeros(n, h, device="cuda", dtype=torch.float64).scatter_reduce(0, at[:, None].expand(-1, h), size, "amax")
    before = torch.where(first[:, None] > 0, scale[touched], 0.0)
    now = torch.maximum(before, (size / MOST[fmt]).float())
    some = torch.where(now > 0, now, 1.0).double()
    old = bytes_[touched]
    kept = _values(old.contiguous(), fmt).double() * before.double()[..., None, None] / some[..., None, None]
    keep = (torch.arange(page, device="cuda") < first[:, None])[:, None, :, None] & (now > before)[..., None, None]
    old = torch.where(keep, _quantize(kept, fmt), old)
    q = _quantize(x / some[at][..., None], fmt)
    old[at, :, off] = torch.where((now > 0)[at][..., None], q, torch.zeros_like(q))
    bytes_[touched] = old
    scale[touched] = now
    return _values(old, fmt) * now[..., None, None]


def _padded(case, c, q):
    """The queries, padded to the same number for every sequence: their positions [sequence, token] (-1: none), and
    [sequence, kv head, token and head of the group, dim]."""
    b, h, d = case["seqs"], case["kv_heads"], case["head_dim"]
    n = c["cu"][1:] - c["cu"][:-1]
    i = torch.arange(c["max_new"], device="cuda")
    there = i < n[:, None]
    row = torch.where(there, c["cu"][:-1, None] + i, 0)
    pos = torch.where(there, (c["length"] - n)[:, None] + i, -1)
    return pos, q[row].view(b, -1, h, case["q_heads"] // h, d).transpose(1, 2).reshape(b, h, -1, d)


def _tokens(case, c, pages, off):
    """K and V of tokens `off` of pages `pages` (both [.., tokens]) in 32 bits, [.., kv head, token, dim]."""
    fmt, dims = case["format"], pages.dim()
    k = _values(c["k"][pages, :, off], fmt) * c["k_scale"][pages][..., None]
    v = _values(c["v"][pages, :, :, off], fmt) * c["v_scale"][pages][..., None]
    return k.transpose(dims - 1, dims).contiguous(), v.transpose(dims - 1, dims).contiguous()


def _scores(case, x, k):
    w = (x @ k.transpose(-1, -2)) * case["head_dim"] ** -0.5
    return case["softcap"] * torch.tanh(w / case["softcap"]) if case["softcap"] else w


def _softmax(w):
    """exp(w - max), and what it is divided by; w is overwritten."""
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w.sub_(torch.where(torch.isinf(top), 0.0, top)))
    total = w.sum(-1, keepdim=True)
    return w, torch.where(total > 0, total, 1.0)


def _result(s, pos, y):
    case, c = s["case"], s["cache"]
    b, h, d = case["seqs"], case["kv_heads"], case["head_dim"]
    y = y.view(b, h, c["max_new"], -1, d).transpose(1, 2).reshape(b, c["max_new"], -1)
    s["out"].copy_(y[pos >= 0])
    return s["out"]


def _plain_sink(s):
    case, c = s["case"], s["cache"]
    page, group = case["page"], case["q_heads"] // case["kv_heads"]
    pos, x = _padded(case, c, s["q"])
    # of every sequence the first tokens, and from the first new one's window on
    sinks, window = case["sinks"], case["window"]
    lens, new = torch.tensor(c["lens"], device="cuda"), torch.tensor(c["new"], device="cuda")
    lo = (lens - new - window + 1).clamp(min=sinks)
    most = max(max(n - max(n - m - window + 1, sinks) for n, m in zip(c["lens"], c["new"])), 0)
    j = torch.cat([torch.arange(sinks, device="cuda").expand(case["seqs"], -1),
                   lo[:, None] + torch.arange(most, device="cuda")], 1)
    there = j < lens[:, None]
    at = torch.where(there, j, 0)
    pages = torch.gather(c["table"], 1, at // page).long().clamp(min=0)
    k, v = _tokens(case, c, pages, at % page)
    w = _scores(case, x, k)
    sees = there[:, None] & (j[:, None] <= pos[..., None]) \
        & ((j[:, None] < sinks) | (j[:, None] > pos[..., None] - window))
    w = w.masked_fill_(~sees.repeat_interleave(group, 1)[:, None], -math.inf)
    w, total = _softmax(w)
    return _result(s, pos, (w @ v) / total)


def _plain_shared(s):
    case, c = s["case"], s["cache"]
    b, h, d, page = case["seqs"], case["kv_heads"], case["head_dim"], case["page"]
    group, common = case["q_heads"] // h, case["prefix"] // page
    pos, x = _padded(case, c, s["q"])
    t = torch.arange(page, device="cuda")
    # the whole pages that all share, once for all rows
    k0, v0 = _tokens(case, c, c["table"][0, :common].long()[:, None].expand(-1, page).reshape(-1),
                     t.expand(common, -1).reshape(-1))
    w0 = _scores(case, x.transpose(0, 1).reshape(h, -1, d), k0).view(h, b, -1, common * page).transpose(0, 1)
    own_pages = c["table"][:, common:].clamp(min=0).long()
    n = own_pages.shape[1]
    k1, v1 = _tokens(case, c, own_pages[..., None].expand(-1, -1, page).reshape(b, -1), t.expand(b, n, -1).reshape(b, -1))
    w1 = _scores(case, x, k1)
    sees = common * page + torch.arange(n * page, device="cuda") <= pos[..., None]
    w1 = w1.masked_fill_(~sees.repeat_interleave(group, 1)[:, None], -math.inf)
    w, total = _softmax(torch.cat([w0, w1], -1))
    w0, w1 = w.split([common * page, n * page], -1)
    y = (w0.transpose(0, 1).reshape(h, -1, common * page) @ v0).view(h, b, -1, d).transpose(0, 1)
    return _result(s, pos, (y + w1 @ v1) / total)


_plain = {"norm": _plain_norm, "turn": _plain_turn, "append": _plain_append, "sink": _plain_sink,
          "shared": _plain_shared}


# -------------------------------------------------------------------- work --

def work(case):
    kind = case["kind"]
    if kind == "norm":
        n, d = case["rows"], case["hidden"]
        vectors = case["post"] + case["pre"] + (case["gate"] == "channel")
        y = (4 if case["out"] == "f32" else 2) if case["pre"] else 0
        return {"bytes": n * d * (12.0 + y + 4 * (case["gate"] == "row")) + 4.0 * d * vectors,
                "flops": n * d * (2.0 + 4 * case["post"] + 4 * case["pre"] + (case["gate"] != "none"))}
    if kind == "turn":
        n, rot = case["tokens"] * case["heads"], 2 * sum(_sections(case))
        return {"bytes": 8.0 * n * case["head_dim"] + 4.0 * case["tokens"] * (rot + len(_sections(case))),
                "flops": 3.0 * n * rot}
    new, past = _lengths(case)
    hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "append":
        t, page, rot = sum(new), case["page"], 2 * sum(_sections(case))
        pages = sum((n + p - 1) // page - p // page + 1 for n, p in zip(new, past))
        # in: q, k, v, the positions and the table's rows; out: q, the cached bytes, the pages as f32
        return {"bytes": 4.0 * t * ((2 * hq + 2 * h) * d + rot + len(_sections(case))) + 2.0 * t * h * d
                + 2.0 * pages * h * (page * d * 5 + 8),
                "flops": 3.0 * t * (hq + h) * rot + 4.0 * t * h * d}
    out = 4 if case["out"] == "f32" else 2
    prefix, w, sinks = case.get("prefix", 0), case.get("window") or (1 << 60), case.get("sinks", 0)
    # a prefix once; of a sequence the tokens that a new one sees
    seen = prefix + sum(n + min(p, w - 1) + min(sinks, max(0, p - w + 1)) for n, p in zip(new, past))
    pairs = sum(sum(prefix + min(p + i + 1, w) + min(sinks, max(0, p + i + 1 - w)) for i in range(n))
                for n, p in zip(new, past))
    return {"bytes": 2.0 * seen * h * (d + 4.0 / case["page"]) + sum(new) * hq * d * (4.0 + out),
            "flops": 4.0 * pairs * hq * d}


# ------------------------------------------------------------ in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "turn": _exact_turn, "append": _exact_append, "sink": _exact_attn,
            "shared": _exact_attn}[case["kind"]](s)


def _exact_norm(s):
    case = s["case"]
    h, z = (s[n].cpu().numpy().astype(np.float64) for n in ("h", "x"))

    def norm(a, w):
        return a / np.sqrt(np.einsum("nd,nd->n", a, a) / a.shape[1] + EPS)[:, None] * w.cpu().numpy()
    if case["post"]:
        z = norm(z, s["post_w"])
    if s["gate"] is not None:
        z = z * s["gate"].cpu().numpy()
    h = case["h_scale"] * h + case["x_scale"] * z
    return h if s["y"] is None else (h, norm(h, s["norm_w"]))


def _exact_rotate(s, x):
    """x [tokens, heads, dim] turned as complex numbers."""
    half, pos, table = s["case"]["half"], s["pos"].cpu().numpy(), s["rope_table"].cpu().numpy()
    y, n = x.astype(np.float64), len(s["map"])
    for i, (axis, col) in enumerate(s["map"]):
        a, b = (i, n + i) if half else (2 * i, 2 * i + 1)
        cs = table[pos[axis], col].astype(np.float64)
        z = (x[..., a].astype(np.float64) + 1j * x[..., b]) * (cs[:, 0] + 1j * cs[:, 1])[:, None]
        y[..., a], y[..., b] = z.real, z.imag
    return y


def _exact_turn(s):
    return _exact_rotate(s, s["x"].cpu().numpy())


def _grid(fmt):
    """Every finite value of the format, by its byte (NaN where there is none)."""
    b = np.arange(256)
    if fmt == "i8":
        return b.astype(np.uint8).view(np.int8).astype(np.float64)
    e, f = (b >> 3) & 15, b & 7
    x = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    x[(b & 127) == 127] = np.nan
    return np.where(b >= 128, -x, x)


def _exact_round(x, fmt):
    """The format's value nearest to each x, ties to the even byte."""
    if fmt == "i8":
        return np.clip(np.rint(np.nan_to_num(x, nan=0.0)), -127, 127)
    g = _grid(fmt)[:127]  # 0 to 448, growing
    a = np.minimum(np.abs(np.nan_to_num(x, nan=0.0, posinf=448.0, neginf=-448.0)), 448.0)
    hi = np.minimum(np.searchsorted(g, a), 126)
    lo = np.maximum(hi - 1, 0)
    up, down = g[hi] - a, a - g[lo]
    return np.copysign(np.where((up < down) | ((up == down) & (hi % 2 == 0)), g[hi], g[lo]), x)


def _exact_append(s):
    case, c = s["case"], s["cache"]
    hq, h, d, page, fmt = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["format"]
    qkv = s["qkv"].cpu().numpy()
    q = _exact_rotate(s, qkv[:, :hq * d].reshape(-1, hq, d))
    x = {"k": _exact_rotate(s, qkv[:, hq * d:(hq + h) * d].reshape(-1, h, d)),
         "v": qkv[:, (hq + h) * d:].reshape(-1, h, d).astype(np.float64)}
    grid, out = _grid(fmt), {"k": [], "v": []}
    touched = s["touched"].long()
    for name in "kv":
        held = c[name][touched].cpu().numpy()
        held = grid[held if name == "k" else held.transpose(0, 1, 3, 2)]
        scale = c[name + "_scale"][touched].cpu().numpy()
        n = t0 = 0
        for length, m in zip(c["lens"], c["new"]):
            p = length - m
            while p < length:
                a, z = p % page, min(page, p % page + length - p)
                y = x[name][t0:t0 + z - a].transpose(1, 0, 2)
                before = scale[n] if a else np.zeros(h, np.float32)
                now = np.maximum(before, (np.abs(y).max((1, 2)) / MOST[fmt]).astype(np.float32)).astype(np.float64)
                r = held[n].copy()
                for i in range(h):
                    if now[i] > before[i]:
                        r[i, :a] = _exact_round(held[n, i, :a] * float(before[i]) / now[i], fmt)
                    r[i, a:z] = _exact_round(y[i] / now[i], fmt) if now[i] else 0.0
                out[name].append(r * now[:, None, None])
                n, t0, p = n + 1, t0 + z - a, p + z - a
    return q.reshape(-1, hq * d), np.stack(out["k"]), np.stack(out["v"])


def _exact_attn(s):
    """Sequence by sequence over every position, those that a token does not see left out of its softmax."""
    case, c = s["case"], s["cache"]
    hq, h, d, page, fmt = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["format"]
    g, window, sinks = hq // h, case.get("window", 0), case.get("sinks", 0)
    out = torch.empty(c["tokens"], hq, d, dtype=torch.float64, device="cuda")
    grid = torch.from_numpy(_grid(fmt)).cuda()
    q, t0 = s["q"].view(-1, hq, d).double(), 0
    for b, (n, m) in enumerate(zip(c["lens"], c["new"])):
        slots = [i for i in range(-(-n // page)) if c["host_table"][b, i] >= 0]
        ids = torch.tensor(c["host_table"][b, slots], device="cuda").long()
        j = (torch.tensor(slots, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).view(-1)
        for i in range(h):
            k = grid[c["k"][ids, i].long()] * c["k_scale"][ids, i].double()[:, None, None]
            v = grid[c["v"][ids, i].long()].transpose(1, 2) * c["v_scale"][ids, i].double()[:, None, None]
            k, v = k.reshape(-1, d), v.reshape(-1, d)
            for a in range(t0, t0 + m, 512):
                z = min(a + 512, t0 + m)
                p = torch.arange(n - m + a - t0, n - m + z - t0, device="cuda")[:, None]
                w = torch.einsum("tgd,jd->tgj", q[a:z, i * g:(i + 1) * g], k) / math.sqrt(d)
                if case["softcap"]:
                    w = case["softcap"] * torch.tanh(w / case["softcap"])
                hidden = (j > p) | ((j <= p - window) & (j >= sinks)) if window else j > p
                w = torch.softmax(w.masked_fill(hidden[:, None, :], -math.inf), -1)
                out[a:z, i * g:(i + 1) * g] = torch.einsum("tgj,jd->tgd", w, v)
        t0 += m
    return out.view(-1, hq * d)
