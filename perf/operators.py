"""Performance cases of the operators around a paged 8-bit key/value cache, as a
decoder uses them beside this library's matvecs and GEMMs.

A case is a dict of plain values; "kind" names the operator:

  table   cosines and sines of rotary positions, scaled for long contexts
  rope    rotary positions applied to the heads of a row of tokens
  append  new keys and values into the cache (keys rotated, both quantized with
          one scale for each page and head), the queries rotated with them
  attn    attention of the new tokens' queries over the cache

With `own` false, run() computes them from elementary torch operations; with
`own` true, it calls modgrad_amd.kvcache. Both work on the same state:

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


# ------------------------------------------------------------------- cases --

def listed():
    heads = {"q_heads": 28, "kv_heads": 4, "head_dim": 128}  # of a 7B-class decoder
    small = {"q_heads": 14, "kv_heads": 2, "head_dim": 64}   # of a 0.5B-class one
    return [
        # a program's start: the positions of a short context
        {"name": "table_4096", "kind": "table", "n_pos": 4096, "rot": 64, "base": 10000.0, "scaling": "none"},
        # the same for a model stretched to 128 Ki positions
        {"name": "table_131072_scaled", "kind": "table", "n_pos": 131072, "rot": 128, "base": 1000000.0,
         "scaling": "ramp"},
        # one decoded token, the smallest call: launch latency
        {"name": "rope_decode_1", "kind": "rope", "tokens": 1, "heads": 32, "head_dim": 128, "rot": 128,
         "half": True},
        # the queries of a long prompt, half of each head rotated
        {"name": "rope_prompt_4096", "kind": "rope", "tokens": 4096, "heads": 28, "head_dim": 128, "rot": 64,
         "half": False},
        # one token for each of 64 sequences
        {"name": "append_decode_64", "kind": "append", **heads, "seqs": 64, "new": 1, "past": 2000,
         "page": 16, "format": "i8", "rot": 128, "half": True, "ragged": True},
        # a scheduler's mixed step: prompts' pieces of odd lengths
        {"name": "append_pieces_9", "kind": "append", **small, "seqs": 9, "new": 333, "past": 777,
         "page": 32, "format": "e4m3", "rot": 64, "half": True, "ragged": True},
        # a long prompt at once
        {"name": "append_prompt_4096", "kind": "append", **heads, "seqs": 1, "new": 4096, "past": 0,
         "page": 64, "format": "i8", "rot": 128, "half": False, "ragged": False},
        # one sequence decoding in a short context: latency
        {"name": "attn_decode_1", "kind": "attn", **heads, "seqs": 1, "new": 1, "past": 1000, "page": 64,
         "format": "i8", "window": 0, "softcap": 0.0, "out": "f32", "ragged": False},
        # a served batch: lengths from a few tokens to 32 Ki
        {"name": "attn_decode_32", "kind": "attn", **heads, "seqs": 32, "new": 1, "past": 32768, "page": 32,
         "format": "e4m3", "window": 0, "softcap": 0.0, "out": "f32", "ragged": True},
        # one sequence deep in a long document: the work has to be split over its length
        {"name": "attn_decode_long", "kind": "attn", **heads, "seqs": 1, "new": 1, "past": 200000, "page": 128,
         "format": "i8", "window": 0, "softcap": 0.0, "out": "f32", "ragged": False},
        # pieces of prompts over a long past, in a sliding-window layer with bounded scores
        {"name": "attn_pieces_window", "kind": "attn", "q_heads": 16, "kv_heads": 8, "head_dim": 256, "seqs": 4,
         "new": 250, "past": 9000, "page": 32, "format": "e4m3", "window": 4096, "softcap": 50.0, "out": "f32",
         "ragged": True},
        # a long prompt at once; its output feeds the f16 prefill GEMM
        {"name": "attn_prompt_4096", "kind": "attn", **heads, "seqs": 1, "new": 4096, "past": 0, "page": 64,
         "format": "i8", "window": 0, "softcap": 0.0, "out": "f16", "ragged": False},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["table", "rope", "append", "append", "attn", "attn", "attn"])
    if kind == "table":
        return {"kind": kind, "n_pos": _log(rng, 500, 120000), "rot": 2 * rng.randint(8, 64),
                "base": float(rng.choice([10000, 500000, 1000000])),
                "scaling": rng.choice(["none", "linear", "ramp", "factors"])}
    if kind == "rope":
        d = rng.choice([64, 96, 128, 256])
        heads = rng.randint(1, 28)
        return {"kind": kind, "tokens": _log(rng, 1, 4096 * 28 * 128 // (heads * d)), "heads": heads, "head_dim": d,
                "rot": rng.choice([d, d, d // 2, d // 4]), "half": rng.random() < 0.5}
    kv = rng.choice([1, 2, 4, 8])
    d = rng.choice([64, 96, 128, 256])
    case = {"kind": kind, "q_heads": kv * rng.randint(1, 8), "kv_heads": kv, "head_dim": d,
            "page": rng.choice([16, 32, 64, 128]), "format": rng.choice(["i8", "e4m3"]), "ragged": rng.random() < 0.6}
    if kind == "append":
        case["seqs"] = _log(rng, 1, 64)
        most = 4096 * 36 * 128 // (case["seqs"] * (case["q_heads"] + 2 * kv) * d)
        case["new"] = rng.choice([1, _log(rng, 1, max(2, most))])
        case.update(past=_log(rng, 1, 4000), rot=rng.choice([d, d, d // 2]), half=rng.random() < 0.5)
        return case
    case["window"] = rng.choice([0, 0, 0, _log(rng, 50, 5000)])
    case["softcap"] = rng.choice([0.0, 0.0, 30.0])
    case["out"] = rng.choice(["f32", "f32", "f16"])
    case["seqs"] = _log(rng, 1, 32)
    case["new"] = rng.choice([1, 1, rng.randint(2, 6), _log(rng, 7, 2000)])
    # no more cache than a twentieth of the largest case's, and no more pairs than a third
    case["past"] = _log(rng, 1, max(2, min(100000, 4000000 // (case["seqs"] * kv * d // 32))))
    pairs = 4096 * 4096 * 28 * 128 // 6
    while case["seqs"] * case["new"] * (case["past"] + case["new"]) * case["q_heads"] * d > pairs and case["new"] > 1:
        case["new"] = max(1, case["new"] // 2)
    return case


def _shares(n):
    """n shares in (0, 1], the first 1: how ragged lengths are spread."""
    return [1.0] + [((b * 0.6180339887) % 1.0) ** 2 for b in range(1, n)]


def _lengths(case):
    """(new tokens, past tokens) of each sequence: the same for every seed."""
    n = case["seqs"]
    if not case["ragged"]:
        return [case["new"]] * n, [case["past"]] * n
    share = _shares(n)
    return ([max(1, int(case["new"] * s)) for s in share],
            [max(1, int(case["past"] * s)) for s in share[1:] + share[:1]])


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
    new, past = _lengths(case)
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
    lens = [a + b for a, b in zip(new, past)]
    need = [-(-n // page) for n in lens]
    pages, most = sum(need) + 3, max(need)
    ids = torch.randperm(pages, generator=g, device="cuda")[:sum(need)].to(torch.int32).cpu().numpy()
    table = np.full((len(lens), most), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return {"k": _payload(g, case["format"], pages, h, page, d), "v": _payload(g, case["format"], pages, h, d, page),
            "k_scale": _page_scales(g, case["format"], pages, h), "v_scale": _page_scales(g, case["format"], pages, h),
            "table": torch.from_numpy(table).cuda(), "length": torch.tensor(lens, dtype=torch.int32, device="cuda"),
            "cu": torch.tensor([0] + new, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32),
            "tokens": sum(new), "max_new": max(new), "lens": lens, "new": new, "host_table": table}


def _theta(case, lib):
    """Angle of one position for each pair, and the factor of both columns
    (64 bits; `lib` is torch or numpy)."""
    rot, base = case["rot"], case["base"]
    i = lib.arange(rot // 2, dtype=lib.float64)
    theta = base ** (-2.0 * i / rot)
    scaling = case["scaling"]
    if scaling == "linear":
        return theta * 0.25, 1.0
    if scaling == "ramp":
        # high frequencies kept, low ones stretched 4 times, a ramp between
        lo, hi = _ramp(rot, base)
        keep = 1.0 - lib.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return theta * 0.25 * (1.0 - keep) + theta * keep, 1.0 + 0.1 * math.log(4.0)
    return theta, 1.0


def _ramp(rot, base, orig=32768):
    def dim(turns):
        return rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))
    return max(0, math.floor(dim(32.0))), min(rot - 1, math.ceil(dim(1.0)))


def _scaling_args(case):
    return {"none": {}, "factors": {}, "linear": {"freq_scale": 0.25},
            "ramp": {"freq_scale": 0.25, "ext_factor": 1.0, "orig_ctx": 32768}}[case["scaling"]]


def _rope_table(n_pos, rot, first=0, base=10000.0):
    p = torch.arange(first, first + n_pos, device="cuda", dtype=torch.float64)
    a = p[:, None] * base ** (-2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / rot)
    return torch.stack([a.cos(), a.sin()], 2).float()


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "table":
        s["first"] = int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
        s["factors"] = None
        if case["scaling"] == "factors":  # the divisors that some files hold, one for each pair
            s["factors"] = 1.0 + 7.0 * torch.rand(case["rot"] // 2, device="cuda", generator=g)
        s["out"] = torch.empty(case["n_pos"], case["rot"] // 2, 2, device="cuda")
        if own:
            from modgrad_amd.kvcache import RopeScaling
            s["scaling"] = RopeScaling(base=case["base"], factors=s["factors"], **_scaling_args(case))
        return s
    if kind == "rope":
        s["x"] = _randn(g, case["tokens"], case["heads"], case["head_dim"])
        s["y"] = torch.empty_like(s["x"])
        s["table"] = _rope_table(8192, case["rot"])
        s["pos"] = torch.randint(0, 8192 - case["tokens"], (1,), generator=g, device="cuda", dtype=torch.int32) \
            + torch.arange(case["tokens"], device="cuda", dtype=torch.int32)
        if own:
            from modgrad_amd.kvcache import RopeTable
            s["rope"] = RopeTable.wrap(s["table"], half=case["half"])
        return s
    s["cache"] = c = _cache(case, g)
    hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "append":
        # one row for each token, [q | k | v] as the fused projection leaves it; some channels of k are loud
        s["qkv"] = _randn(g, c["tokens"], (hq + 2 * h) * d)
        s["qkv"][:, hq * d:(hq + h) * d:37] *= 4.0
        s["q_out"] = torch.empty(c["tokens"], hq * d, device="cuda")
        s["rope_table"] = _rope_table(c["host_table"].shape[1] * case["page"], case["rot"])
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
        from modgrad_amd.kvcache import KvCache, RopeTable
        s["handle"] = KvCache.wrap(c["k"], c["v"], c["k_scale"], c["v_scale"], c["table"], c["length"],
                                   cu_tokens=c["cu"] if c["max_new"] > 1 else None, fmt=case["format"])
        if kind == "append":
            s["rope"] = RopeTable.wrap(s["rope_table"], half=case["half"])
        else:
            s["workspace"] = s["handle"].attention_workspace(hq, c["tokens"], c["max_new"])
    return s


# ------------------------------------------------------------ the operators --

def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _own_table(s):
    from modgrad_amd.kvcache import kern
    case, out = s["case"], s["out"]
    kern.rope_table(out.data_ptr(), case["n_pos"], s["first"], case["rot"], s["scaling"])
    return out


def _own_rope(s):
    case, x, y = s["case"], s["x"], s["y"]
    d = case["heads"] * case["head_dim"]
    s["rope"].apply(x.data_ptr(), y.data_ptr(), s["pos"].data_ptr(), case["tokens"], case["heads"], case["head_dim"],
                    x_stride=d, y_stride=d)
    return y


def _own_append(s):
    case, c, qkv = s["case"], s["cache"], s["qkv"]
    hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    row, at = qkv.shape[1], qkv.data_ptr()
    s["handle"].append(at + 4 * hq * d, at + 4 * (hq + h) * d, row, c["tokens"], c["max_new"], rope=s["rope"],
                       q=at, q_stride=row, q_out=s["q_out"].data_ptr(), q_out_stride=hq * d, n_q_heads=hq)
    s["handle"].dequant(s["touched"].data_ptr(), len(s["touched"]), s["k_out"].data_ptr(), s["v_out"].data_ptr())
    return s["q_out"], s["k_out"], s["v_out"]


def _own_attn(s):
    case, c = s["case"], s["cache"]
    d = case["q_heads"] * case["head_dim"]
    s["handle"].attend(s["q"].data_ptr(), d, case["q_heads"], s["out"].data_ptr(), d, c["tokens"], c["max_new"],
                       scale=case["head_dim"] ** -0.5, softcap=case["softcap"], window=case["window"],
                       out_f16=case["out"] == "f16", workspace=s["workspace"])
    return s["out"]


_own = {"table": _own_table, "rope": _own_rope, "append": _own_append, "attn": _own_attn}


def _plain_table(s):
    case = s["case"]
    theta, size = _theta(case, torch)
    theta = theta.cuda()
    if s["factors"] is not None:
        theta = theta / s["factors"].double()
    p = torch.arange(s["first"], s["first"] + case["n_pos"], device="cuda", dtype=torch.float64)
    a = p[:, None] * theta
    s["out"][..., 0] = size * a.cos()
    s["out"][..., 1] = size * a.sin()
    return s["out"]


def _rotate(x, cs, rot, half):
    """x [tokens, heads, dim] in 64 bits, cs [tokens, rot/2, 2]."""
    c, n = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    x = x.double()
    y = x.clone()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., a] = x[..., a] * c - x[..., b] * n
    y[..., b] = x[..., a] * n + x[..., b] * c
    return y


def _plain_rope(s):
    case = s["case"]
    s["y"].copy_(_rotate(s["x"], s["table"][s["pos"].long()], case["rot"], case["half"]))
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
    one = torch.ones_like(x)
    step = torch.ldexp(one, e)
    return ((x / step).round() * step).float().to(torch.float8_e4m3fn).view(torch.uint8)


def _places(c, page):
    """Of each new token: its sequence, position, page and place in the page."""
    t = torch.arange(c["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(c["cu"], t, right=True) - 1
    pos = (c["length"][seq] - c["cu"][seq + 1] + t).long()
    return seq, pos, c["table"][seq, pos // page].long(), pos % page


def _plain_append(s):
    case, c = s["case"], s["cache"]
    hq, h, d, page, fmt = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["format"]
    q, k, v = s["qkv"].split([hq * d, h * d, h * d], 1)
    _, pos, pg, off = _places(c, page)
    cs = s["rope_table"][pos]
    s["q_out"].copy_(_rotate(q.view(-1, hq, d), cs, case["rot"], case["half"]).view(-1, hq * d))
    k = _rotate(k.view(-1, h, d), cs, case["rot"], case["half"])
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


def _plain_attn(s):
    case, c, q = s["case"], s["cache"], s["q"]
    hq, h, d, page, fmt = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["format"]
    b, most, g = case["seqs"], c["table"].shape[1], hq // h
    # the queries, padded to the same number for every sequence: [sequence, kv head, token and head of the group, dim]
    i = torch.arange(c["max_new"], device="cuda")
    there = i < (c["cu"][1:] - c["cu"][:-1])[:, None]
    row = torch.where(there, c["cu"][:-1, None] + i, 0)
    pos = torch.where(there, c["length"][:, None] - (c["cu"][1:] - c["cu"][:-1])[:, None] + i, -1)
    x = q[row].view(b, -1, h, g, d).transpose(1, 2).reshape(b, h, -1, d)
    # the cache in 32 bits: [sequence, kv head, position, dim]
    pages = c["table"].clamp(min=0).long()
    k = _values(c["k"][pages], fmt) * c["k_scale"][pages][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(b, h, most * page, d)
    v = _values(c["v"][pages], fmt) * c["v_scale"][pages][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(b, h, most * page, d)
    w = (x @ k.transpose(2, 3)) * d ** -0.5
    if case["softcap"]:
        w = case["softcap"] * torch.tanh(w / case["softcap"])
    j = torch.arange(most * page, device="cuda")
    sees = j <= pos[..., None]
    if case["window"]:
        sees &= j > pos[..., None] - case["window"]
    sees = sees[:, None, :, None, :]
    w = w.view(b, h, -1, g, most * page).masked_fill_(~sees, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w.sub_(torch.where(torch.isinf(top), 0.0, top)))
    total = w.sum(-1, keepdim=True)
    w = w.div_(torch.where(total > 0, total, 1.0)).view(b, h, -1, most * page)
    y = (w @ v).view(b, h, -1, g, d).transpose(1, 2).reshape(b, -1, hq * d)
    s["out"].copy_(y[there])
    return s["out"]


_plain = {"table": _plain_table, "rope": _plain_rope, "append": _plain_append, "attn": _plain_attn}


# -------------------------------------------------------------------- work --

def work(case):
    kind = case["kind"]
    if kind == "table":
        n = case["n_pos"] * case["rot"]
        return {"bytes": 4.0 * n, "flops": 3.0 * n}
    if kind == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 8.0 * n * case["head_dim"] + 4.0 * case["tokens"] * (case["rot"] + 1),
                "flops": 3.0 * n * case["rot"]}
    new, past = _lengths(case)
    hq, h, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if kind == "append":
        t, page = sum(new), case["page"]
        pages = sum((n + p - 1) // page - p // page + 1 for n, p in zip(new, past))
        # in: q, k, v and the table's rows; out: q, the cached bytes, the pages as f32
        return {"bytes": 4.0 * t * ((2 * hq + 2 * h) * d + case["rot"]) + 2.0 * t * h * d
                + 2.0 * pages * h * (page * d * 5 + 8),
                "flops": 3.0 * t * (hq + h) * case["rot"] + 4.0 * t * h * d}
    w = case["window"] or (1 << 60)
    seen = sum(n + min(p, w - 1) for n, p in zip(new, past))
    pairs = sum(sum(min(p + i + 1, w) for i in range(n)) for n, p in zip(new, past))
    out = 4 if case["out"] == "f32" else 2
    return {"bytes": 2.0 * seen * h * (d + 4.0 / case["page"]) + sum(new) * hq * d * (4.0 + out),
            "flops": 4.0 * pairs * hq * d}


# ------------------------------------------------------------ in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return {"table": _exact_table, "rope": _exact_rope, "append": _exact_append, "attn": _exact_attn}[case["kind"]](s)


def _exact_table(s):
    case = s["case"]
    theta, size = _theta(case, np)
    if s["factors"] is not None:
        theta = theta / s["factors"].cpu().numpy().astype(np.float64)
    z = size * np.exp(1j * np.outer(np.arange(s["first"], s["first"] + case["n_pos"], dtype=np.float64), theta))
    return np.stack([z.real, z.imag], 2)


def _exact_turn(x, cs, rot, half):
    """x [tokens, heads, dim] turned as complex numbers."""
    x = x.astype(np.float64)
    z = cs[:, None, :, 0].astype(np.float64) + 1j * cs[:, None, :, 1]
    y = x.copy()
    if half:
        r = (x[..., :rot // 2] + 1j * x[..., rot // 2:rot]) * z
        y[..., :rot // 2], y[..., rot // 2:rot] = r.real, r.imag
    else:
        r = (x[..., 0:rot:2] + 1j * x[..., 1:rot:2]) * z
        y[..., 0:rot:2], y[..., 1:rot:2] = r.real, r.imag
    return y


def _exact_rope(s):
    case = s["case"]
    return _exact_turn(s["x"].cpu().numpy(), s["table"].cpu().numpy()[s["pos"].cpu().numpy()], case["rot"], case["half"])


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
    qkv, turn = s["qkv"].cpu().numpy(), s["rope_table"].cpu().numpy()
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(c["lens"], c["new"])])
    q = _exact_turn(qkv[:, :hq * d].reshape(-1, hq, d), turn[pos], case["rot"], case["half"])
    x = {"k": _exact_turn(qkv[:, hq * d:(hq + h) * d].reshape(-1, h, d), turn[pos], case["rot"], case["half"]),
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
    case, c = s["case"], s["cache"]
    hq, h, d, page, fmt = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["format"]
    g = hq // h
    out = torch.empty(c["tokens"], hq, d, dtype=torch.float64, device="cuda")
    grid = torch.from_numpy(_grid(fmt)).cuda()
    q, t0 = s["q"].view(-1, hq, d).double(), 0
    for b, (n, m) in enumerate(zip(c["lens"], c["new"])):
        first = max(0, n - m - case["window"] + 1) // page if case["window"] else 0
        ids = torch.from_numpy(c["host_table"][b, first:-(-n // page)]).cuda().long()
        for i in range(h):
            k = grid[c["k"][ids, i].long()] * c["k_scale"][ids, i].double()[:, None, None]
            v = grid[c["v"][ids, i].long()].transpose(1, 2) * c["v_scale"][ids, i].double()[:, None, None]
            k, v = k.reshape(-1, d), v.reshape(-1, d)
            j = torch.arange(first * page, first * page + len(k), device="cuda")
            for a in range(t0, t0 + m, 512):
                z = min(a + 512, t0 + m)
                p = torch.arange(n - m + a - t0, n - m + z - t0, device="cuda")[:, None]
                w = torch.einsum("tgd,jd->tgj", q[a:z, i * g:(i + 1) * g], k) / math.sqrt(d)
                if case["softcap"]:
                    w = case["softcap"] * torch.tanh(w / case["softcap"])
                hidden = (j > p) | (j <= p - case["window"]) if case["window"] else j > p
                w = torch.softmax(w.masked_fill(hidden[:, None, :], -math.inf), -1)
                out[a:z, i * g:(i + 1) * g] = torch.einsum("tgj,jd->tgd", w, v)
        t0 += m
    return out.view(-1, hq * d)
