"""What the serving operators over a paged cache are measured on: new rows rotated and
appended to the cache (16-bit, fp8 or 4-bit pages), prompts of different lengths attended
in one packed call, and attention over a cache held in 4 bits, from one token of one user
to batches of long contexts.

`run` makes one pass: with `own`, the calls of puter_amd.Backend; without, the same
operators in elementary torch operations.  `exact` computes them in float64.
"""
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------- the cases --
def listed():
    return [
        # A decode step of 64 users: one new row each from a fused Q/K/V projection, rotated
        # at its own position (Llama-3 frequencies) and stored in 16-bit pages.
        {"name": "append_bf16_64", "kind": "append", "dtype": "bf16", "cache": "same", "group": 0, "batch": 64,
         "new_lo": 1, "new_hi": 1, "past_lo": 512, "past_hi": 8191, "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "half": True, "llama3": True, "fused": True, "shape": 1},
        # One user's token into 4-bit pages, and the page's values read back: what an
        # interactive program waits for at every layer.
        {"name": "append_int4_1", "kind": "append", "dtype": "bf16", "cache": "int4", "group": 64, "batch": 1,
         "new_lo": 1, "new_hi": 1, "past_lo": 1000, "past_hi": 1000, "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "half": True, "llama3": False, "fused": True, "shape": 2},
        # Five prompts stored in 4 bits, small groups, and read back for the next chunk.
        {"name": "append_int4_prompts", "kind": "append", "dtype": "f16", "cache": "int4", "group": 32, "batch": 5,
         "new_lo": 301, "new_hi": 2901, "past_lo": 0, "past_hi": 2000, "heads": 32, "kv": 8, "dim": 128, "page": 32,
         "half": True, "llama3": False, "fused": False, "shape": 3},
        # Prompts into fp8 pages, interleaved pairs.
        {"name": "append_fp8_prompts", "kind": "append", "dtype": "bf16", "cache": "fp8", "group": 0, "batch": 6,
         "new_lo": 500, "new_hi": 4096, "past_lo": 0, "past_hi": 0, "heads": 32, "kv": 8, "dim": 128, "page": 16,
         "half": False, "llama3": False, "fused": True, "shape": 4},
        # A batch of prompts as users send them: a few long ones among short ones.
        {"name": "prompts_bf16_9", "kind": "prompts", "dtype": "bf16", "batch": 9, "lo": 64, "hi": 4096, "past_lo": 0,
         "past_hi": 0, "heads": 32, "kv": 8, "dim": 128, "window": 0, "shape": 5},
        # Many short texts through a small model (an embedding or classification batch).
        {"name": "prompts_f16_48_d64", "kind": "prompts", "dtype": "f16", "batch": 48, "lo": 1, "hi": 200, "past_lo": 0,
         "past_hi": 0, "heads": 16, "kv": 4, "dim": 64, "window": 0, "shape": 6},
        # Two whole documents.
        {"name": "prompts_bf16_2_long", "kind": "prompts", "dtype": "bf16", "batch": 2, "lo": 6001, "hi": 8192,
         "past_lo": 0, "past_hi": 0, "heads": 32, "kv": 8, "dim": 128, "window": 0, "shape": 7},
        # The next chunks of prompts whose beginnings are cached, in f32, a sliding window.
        {"name": "prompts_f32_5_d80", "kind": "prompts", "dtype": "f32", "batch": 5, "lo": 33, "hi": 900, "past_lo": 0,
         "past_hi": 700, "heads": 8, "kv": 8, "dim": 80, "window": 512, "shape": 8},
        # One user's decode step over a short 4-bit context.
        {"name": "int4_decode_1", "kind": "int4", "dtype": "bf16", "batch": 1, "query": 1, "ctx_lo": 777,
         "ctx_hi": 777, "heads": 32, "kv": 8, "dim": 128, "group": 64, "page": 16, "shape": 9},
        # A decode step of 64 users with contexts of very different lengths.
        {"name": "int4_decode_64", "kind": "int4", "dtype": "bf16", "batch": 64, "query": 1, "ctx_lo": 512,
         "ctx_hi": 8192, "heads": 32, "kv": 8, "dim": 128, "group": 128, "page": 16, "shape": 10},
        # Three long documents, few heads, small groups.
        {"name": "int4_decode_3_long", "kind": "int4", "dtype": "bf16", "batch": 3, "query": 1, "ctx_lo": 50001,
         "ctx_hi": 120000, "heads": 16, "kv": 2, "dim": 128, "group": 32, "page": 64, "shape": 11},
        # Five drafted tokens per user attended at once for verification, head dim 64.
        {"name": "int4_verify_16x5", "kind": "int4", "dtype": "f16", "batch": 16, "query": 5, "ctx_lo": 100,
         "ctx_hi": 6000, "heads": 32, "kv": 8, "dim": 64, "group": 64, "page": 24, "shape": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "prompts", "int4"])
    shape = rng.randint(100, 10 ** 6)
    if kind == "append":
        cache = rng.choice(["same", "fp8", "int4", "int4"])
        dim = rng.choice([64, 128, 128, 256] if cache == "int4" else [64, 80, 96, 128, 128, 256])
        kv, per = rng.choice([(8, 4), (8, 1), (4, 7), (2, 8), (1, 8), (5, 3)])
        page = rng.choice([8, 16, 16, 32, 64])
        batch = _log(rng, 1, 200)
        new_hi = rng.choice([1, 1, max(1, min(4096, _log(rng, 2, 8000) // batch))])
        past = rng.choice([0, _log(rng, 1, 120000)])
        return {"kind": kind, "dtype": rng.choice(["bf16", "f16"] if cache == "int4" else ["bf16", "bf16", "f16", "f32"]),
                "cache": cache, "group": rng.choice([g for g in (32, 64, 128) if g <= dim]) if cache == "int4" else 0,
                "batch": batch, "new_lo": max(1, new_hi // rng.randint(1, 9)), "new_hi": new_hi, "past_lo": past // 3,
                "past_hi": past, "heads": kv * per, "kv": kv, "dim": dim, "page": page, "half": rng.random() < 0.7,
                "llama3": rng.random() < 0.4, "fused": rng.random() < 0.6, "shape": shape}
    if kind == "prompts":
        dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
        kv, per = rng.choice([(8, 1), (16, 1), (4, 4), (8, 4), (2, 6), (1, 8)])
        batch = _log(rng, 1, 64)
        hi = min(_log(rng, 2, 4096), int(math.sqrt(4e9 / (batch * kv * per))))
        past = rng.choice([0, 0, _log(rng, 1, 1000)])
        past = min(past, hi)
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "batch": batch,
                "lo": max(1, hi // rng.randint(1, 50)), "hi": hi, "past_lo": past // 2, "past_hi": past,
                "heads": kv * per, "kv": kv, "dim": dim, "window": rng.choice([0, 0, 0, rng.randint(16, 1024)]),
                "shape": shape}
    dim = rng.choice([64, 128, 128, 128, 256])
    kv, per = rng.choice([(8, 4), (8, 1), (4, 7), (2, 8), (1, 16), (5, 3)])
    batch = _log(rng, 1, 64)
    hi = min(_log(rng, 8, 60000), 250000 // batch)
    return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16"]), "batch": batch,
            "query": rng.choice([1, 1, 1, rng.randint(2, 8)]), "ctx_lo": max(8, hi // rng.randint(1, 9)),
            "ctx_hi": max(8, hi), "heads": kv * per, "kv": kv, "dim": dim,
            "group": rng.choice([g for g in (32, 64, 128) if g <= dim]), "page": rng.choice([8, 16, 16, 24, 32, 64]),
            "shape": shape}


def _spread(case, n, lo, hi, salt):
    """n whole numbers spread evenly over lo .. hi, in an order of the case's own."""
    v = [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]
    random.Random(case["shape"] * 7 + salt).shuffle(v)
    return v


def _news(c):
    return _spread(c, c["batch"], c["new_lo"], c["new_hi"], 1), _spread(c, c["batch"], c["past_lo"], c["past_hi"], 2)


def _prompts(c):
    if c["lo"] * 16 < c["hi"]:  # a few long ones among short ones
        r = random.Random(c["shape"] * 7 + 1)
        lens = [_log(r, c["lo"], c["hi"]) for _ in range(c["batch"] - 1)] + [c["hi"]]
    else:
        lens = _spread(c, c["batch"], c["lo"], c["hi"], 1)
    past = _spread(c, c["batch"], c["past_lo"], c["past_hi"], 2)
    return lens, [n + p for n, p in zip(lens, past)]


def _contexts(c):
    return _spread(c, c["batch"], c["ctx_lo"], c["ctx_hi"], 1)


# ------------------------------------------------------------------- inputs --
def _normal(g, shape, dtype, std=1.0):
    return torch.randn(shape, device="cuda", generator=g).mul_(std).to(TORCH[dtype])


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _keys(g, shape, dtype):
    """Keys as models make them: a few dims of each head are much larger than the rest."""
    k = torch.randn(shape, device="cuda", generator=g)
    k *= 1.0 + 4.0 * (torch.rand(shape[-2:], device="cuda", generator=g) > 0.95)
    return k.to(TORCH[dtype])


def _code_pool(g, pages, c):
    """A pool of 4-bit codes and its (scale, offset) pairs."""
    kv, d = c["kv"], c["dim"]
    codes = torch.randint(0, 256, (pages, c["page"], kv, d // 2), device="cuda", generator=g, dtype=torch.uint8)
    shape = (pages, c["page"], kv, d // c["group"])
    scale = 0.2 + 0.2 * torch.rand(shape, device="cuda", generator=g)
    offset = 0.3 * torch.randn(shape, device="cuda", generator=g)
    return codes, torch.stack((scale, offset), -1).half()


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    h, kv, d = c["heads"], c["kv"], c["dim"]
    t = {"case": c}
    if c["kind"] == "prompts":
        lens, keys = _prompts(c)
        std = d ** -0.25  # scores of about one, as after a normalised Q and K
        t["q"] = _normal(g, (sum(lens), h, d), c["dtype"], std)
        t["k"] = _normal(g, (sum(keys), kv, d), c["dtype"], std)
        t["v"] = _normal(g, (sum(keys), kv, d), c["dtype"])
        t["qoff"], t["koff"] = _starts(lens), _starts(keys)
        t["out"] = torch.empty_like(t["q"])
        return t
    page = c["page"]
    if c["kind"] == "int4":
        ctx = _contexts(c)
        counts = [(n + page - 1) // page for n in ctx]
        perm = torch.randperm(sum(counts), generator=host).to(torch.int32)
        table = torch.zeros((len(ctx), max(counts)), dtype=torch.int32)
        at = 0
        for b, n in enumerate(counts):
            table[b, :n] = perm[at:at + n]
            at += n
        t["table"], t["ctx"] = table.cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda")
        t["kcodes"], t["kpar"] = _code_pool(g, sum(counts), c)
        t["vcodes"], t["vpar"] = _code_pool(g, sum(counts), c)
        t["q"] = _normal(g, (c["batch"], c["query"], h, d), c["dtype"])
        t["out"] = torch.empty_like(t["q"])
        return t
    new, past = _news(c)
    # the pages that the new rows touch and two more, in a random order
    first = [p // page for p in past]
    touched = [(p + n - 1) // page - f + 1 for n, p, f in zip(new, past, first)]
    pages, rows = sum(touched) + 2, sum(new)
    perm = torch.randperm(pages, generator=host)
    positions = torch.cat([torch.arange(p, p + n) for n, p in zip(new, past)])
    page_of = torch.cat([torch.arange(p, p + n) // page - f + at for n, p, f, at in
                         zip(new, past, first, [sum(touched[:i]) for i in range(len(touched))])])
    t["positions"] = positions.to(torch.int32).cuda()
    t["ids"] = perm[page_of].to(torch.int32).cuda()
    t["slots"] = (positions % page).to(torch.int32).cuda()
    q, k, v = _normal(g, (rows, h, d), c["dtype"]), _keys(g, (rows, kv, d), c["dtype"]), _normal(g, (rows, kv, d), c["dtype"])
    if c["fused"]:  # one projection's rows: [q | k | v]
        rows3 = torch.cat((q, k, v), 1)
        q, k, v = rows3[:, :h], rows3[:, h:h + kv], rows3[:, h + kv:]
    t["q"], t["k"], t["v"] = q, k, v
    t["qout"] = torch.empty((rows, h, d), device="cuda", dtype=TORCH[c["dtype"]])
    if c["cache"] == "int4":
        t["kpool"], t["kpar"] = _code_pool(g, pages, c)
        t["vpool"], t["vpar"] = _code_pool(g, pages, c)
        t["all"] = torch.arange(pages, dtype=torch.int32, device="cuda")
        t["kvalues"], t["vvalues"] = (torch.empty((pages, page, kv, d), device="cuda", dtype=TORCH[c["dtype"]])
                                      for _ in range(2))
        return t
    shape = (pages, page, kv, d)
    t["kpool"], t["vpool"] = _normal(g, shape, c["dtype"]), _normal(g, shape, c["dtype"])
    t["kpar"] = t["vpar"] = None
    if c["cache"] == "fp8":
        t["kpar"] = torch.rand(kv, device="cuda", generator=g) * 0.01 + 0.05
        t["vpar"] = torch.rand(kv, device="cuda", generator=g) * 0.002 + 0.01
        t["kpool"], t["vpool"] = (t[n].float().to(torch.float8_e4m3fn) for n in ("kpool", "vpool"))
    return t


# -------------------------------------------------------------------- a pass --
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "prompts": _own_prompts, "int4": _own_int4}[kind](state)
    return {"append": _plain_append, "prompts": _plain_prompts, "int4": _plain_int4}[kind](state)


_handle = []


def _backend():
    """The program's one Backend."""
    import puter_amd
    if not _handle:
        _handle.append(puter_amd.Backend())
    return puter_amd, _handle[0]


def _own_append(t):
    p, be = _backend()
    c = t["case"]
    h, kv, d = c["heads"], c["kv"], c["dim"]
    f = {"bf16": p.BF16, "f16": p.F16, "f32": p.F32}[c["dtype"]]
    cache = {"same": f, "fp8": p.F8E4M3, "int4": p.I4}[c["cache"]]
    mode = p.RoPEModeHalf if c["half"] else p.RoPEModeInterleaved
    rope = p.RoPEConfig(500000.0, 0, mode, p.RoPEScalingLlama3, 8.0, 1.0, 4.0, 8192) if c["llama3"] else \
        p.RoPEConfig(BaseFreq=10000.0, Mode=mode)
    pages, rows = t["kpool"].shape[0], t["q"].shape[0]
    be.KVPageAppendRoPE(rope, t["q"], t["k"], t["v"], t["positions"], t["ids"], t["slots"], t["qout"], t["kpool"],
                        t["vpool"], t["kpar"], t["vpar"], rows, h, kv, d, t["q"].stride(0), t["k"].stride(0),
                        t["v"].stride(0), pages, c["page"], c["group"], f, cache)
    if c["cache"] != "int4":
        return t["qout"], t["kpool"], t["vpool"]
    be.KVPageGatherInt4(t["kpool"], t["kpar"], t["all"], t["kvalues"], pages, c["page"], kv, d, c["group"],
                        pages * c["page"], f)
    be.KVPageGatherInt4(t["vpool"], t["vpar"], t["all"], t["vvalues"], pages, c["page"], kv, d, c["group"],
                        pages * c["page"], f)
    return t["qout"], t["kvalues"], t["vvalues"]


def _own_prompts(t):
    p, be = _backend()
    c = t["case"]
    f = {"bf16": p.BF16, "f16": p.F16, "f32": p.F32}[c["dtype"]]
    cfg = p.MultiHeadAttentionConfig(c["heads"], c["dim"], True, c["window"], 0.0, c["kv"])
    be.MultiHeadAttentionPacked(cfg, t["q"], t["k"], t["v"], t["out"], t["qoff"], t["koff"], c["batch"],
                                t["q"].shape[0], t["k"].shape[0], f)
    return t["out"]


def _own_int4(t):
    p, be = _backend()
    c = t["case"]
    h, kv, d = c["heads"], c["kv"], c["dim"]
    f = {"bf16": p.BF16, "f16": p.F16}[c["dtype"]]
    if "workspace" not in t:  # held with the plan, as long as it
        need = be.PagedInt4WorkspaceBytes(c["batch"], c["query"], h, kv, d, c["ctx_hi"])
        t["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    be.PagedInt4Attention(t["q"], t["kcodes"], t["vcodes"], t["kpar"], t["vpar"], t["table"], t["ctx"], c["batch"],
                          c["query"], t["table"].shape[1], c["page"], t["kcodes"].shape[0], h, kv, d, c["group"],
                          c["ctx_hi"], f, t["out"], t["workspace"], t["workspace"].numel())
    return t["out"]


# ----------------------------------------------------------- the plain forms --
def _rotate(x, positions, c):
    """x [rows, heads, dim] in f32, rotated; the angles in 64 bits (positions may be far)."""
    d = c["dim"]
    base = 500000.0 if c["llama3"] else 10000.0
    inv = torch.exp(torch.arange(0, d, 2, device="cuda", dtype=torch.float64) * (-math.log(base) / d))
    if c["llama3"]:  # factor 8, low 1, high 4, trained on 8192
        wave = 2 * math.pi / inv
        mix = (8192.0 / wave - 1.0) / 3.0
        inv = torch.where(wave > 8192.0, inv / 8.0, torch.where(wave < 2048.0, inv, (1 - mix) * inv / 8.0 + mix * inv))
    angle = positions.double()[:, None] * inv
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = (x[..., :d // 2], x[..., d // 2:]) if c["half"] else (x[..., 0::2], x[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.cat((a, b), -1) if c["half"] else torch.stack((a, b), -1).flatten(-2)


def _quantise(x, group):
    """x [rows, kv, dim] as 4-bit codes packed by twos and their (scale, offset) pairs."""
    x = x.unflatten(-1, (-1, group))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).half()
    offset = (0.5 * lo + 0.5 * hi + 0.5 * scale.float()).half()
    inverse = torch.where(scale > 0, 1 / scale.float(), 0.0)
    n = torch.round((x - offset.float()) * inverse).clamp(-8, 7).to(torch.int16).flatten(-2) & 15
    return (n[..., 0::2] | n[..., 1::2] << 4).to(torch.uint8), torch.cat((scale, offset), -1)


def _values(codes, pairs):
    """The f32 values of packed codes [.., dim / 2] with pairs [.., groups, 2]."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    n = (n.to(torch.int8) ^ 8) - 8
    pairs = pairs.float()
    x = n.float().unflatten(-1, (pairs.shape[-2], -1))
    return (x * pairs[..., :1] + pairs[..., 1:]).flatten(-2)


def _plain_append(t):
    c = t["case"]
    q, k, v = _rotate(t["q"].float(), t["positions"], c), _rotate(t["k"].float(), t["positions"], c), t["v"].float()
    t["qout"].copy_(q)
    ids, slots = t["ids"].long(), t["slots"].long()
    if c["cache"] == "int4":
        t["kpool"][ids, slots], t["kpar"][ids, slots] = _quantise(k, c["group"])
        t["vpool"][ids, slots], t["vpar"][ids, slots] = _quantise(v, c["group"])
        t["kvalues"].copy_(_values(t["kpool"], t["kpar"]))
        t["vvalues"].copy_(_values(t["vpool"], t["vpar"]))
        return t["qout"], t["kvalues"], t["vvalues"]
    if c["cache"] == "fp8":
        k, v = ((x / t[s][:, None]).clamp(-448, 448).to(torch.float8_e4m3fn) for x, s in ((k, "kpar"), (v, "vpar")))
        t["kpool"].view(torch.uint8)[ids, slots] = k.view(torch.uint8)
        t["vpool"].view(torch.uint8)[ids, slots] = v.view(torch.uint8)
    else:
        t["kpool"][ids, slots], t["vpool"][ids, slots] = k.to(TORCH[c["dtype"]]), v.to(TORCH[c["dtype"]])
    return t["qout"], t["kpool"], t["vpool"]


def _softmax_product(s, hidden, v):
    """softmax of s where not hidden, times v; rows that see nothing are zero."""
    s.masked_fill_(hidden, -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    return torch.matmul(s, v) / s.sum(-1, keepdim=True).clamp_(min=1e-30)


def _plain_prompts(t):
    c = t["case"]
    h, kv, d = c["heads"], c["kv"], c["dim"]
    lens, keys = _prompts(c)
    b, m, n, g = c["batch"], max(lens), max(keys), h // kv
    qoff, koff = t["qoff"].long(), t["koff"].long()
    qlen, klen = qoff.diff(), koff.diff()
    qi, ki = torch.arange(m, device="cuda"), torch.arange(n, device="cuda")
    at = (qoff[:-1, None] + qi).clamp_(max=t["q"].shape[0] - 1)
    from_ = (koff[:-1, None] + ki).clamp_(max=t["k"].shape[0] - 1)
    q = t["q"].float()[at].view(b, m, kv, g, d).permute(0, 2, 3, 1, 4).reshape(b, kv, g * m, d)
    k = t["k"].float()[from_].permute(0, 2, 3, 1).contiguous()
    v = t["v"].float()[from_].permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(q, k).view(b, kv, g, m, n).mul_(1 / math.sqrt(d))
    row, col = qi[:, None], ki[None]
    hidden = (col > row + (klen - qlen)[:, None, None]) | (col >= klen[:, None, None])
    if c["window"]:
        hidden |= row - col >= c["window"]
    o = _softmax_product(s, hidden[:, None, None], v[:, :, None])
    token = torch.arange(t["q"].shape[0], device="cuda")
    of = (token[:, None] >= qoff[None, 1:]).sum(1)
    t["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(b, m, h, d)[of, token - qoff[of]])
    return t["out"]


def _plain_int4(t):
    c = t["case"]
    h, kv, d, b, m = c["heads"], c["kv"], c["dim"], c["batch"], c["query"]
    table = t["table"].long()
    k = _values(t["kcodes"][table].flatten(1, 2), t["kpar"][table].flatten(1, 2)).permute(0, 2, 3, 1).contiguous()
    v = _values(t["vcodes"][table].flatten(1, 2), t["vpar"][table].flatten(1, 2)).permute(0, 2, 1, 3).contiguous()
    n = k.shape[-1]
    q = t["q"].float().view(b, m, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    s = torch.matmul(q, k).view(b, kv, h // kv, m, n).mul_(1 / math.sqrt(d))
    last = t["ctx"].long()[:, None] - m + torch.arange(m, device="cuda")
    hidden = torch.arange(n, device="cuda") > last[..., None]
    o = _softmax_product(s, hidden[:, None, None], v[:, :, None])
    t["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(b, m, h, d))
    return t["out"]


# ------------------------------------------------------------------ the work --
def _pairs(c):
    """(query, key) pairs that the mask lets through, one head."""
    n = 0
    for m, k in zip(*_prompts(c)):
        q = torch.arange(m, dtype=torch.int64)
        lo = (q - c["window"] + 1).clamp(min=0) if c["window"] else torch.zeros_like(q)
        n += int(((q + k - m + 1).clamp(0, k) - lo).clamp(min=0).sum())
    return n


def work(case):
    c, e = case, SIZE[case["dtype"]]
    h, kv, d = c["heads"], c["kv"], c["dim"]
    if c["kind"] == "prompts":
        lens, keys = _prompts(c)
        return {"bytes": e * d * (2 * h * sum(lens) + 2 * kv * sum(keys)), "flops": 4 * d * h * _pairs(c)}
    if c["kind"] == "int4":
        row = kv * (d // 2 + 4 * (d // c["group"]))
        tokens, q = sum(_contexts(c)), c["batch"] * c["query"] * h * d
        return {"bytes": 2 * tokens * row + 2 * e * q, "flops": 4 * tokens * c["query"] * h * d}
    new, past = _news(c)
    rows, page = sum(new), c["page"]
    row = {"same": e * kv * d, "fp8": kv * d, "int4": kv * (d // 2 + 4 * (d // (c["group"] or d)))}[c["cache"]]
    n = e * rows * (2 * h + 2 * kv) * d + 2 * rows * row + 12 * rows
    if c["cache"] == "int4":  # and every page's values
        pages = sum((p + m - 1) // page - p // page + 1 for m, p in zip(new, past)) + 2
        n += 2 * pages * page * (row + e * kv * d)
    return {"bytes": n, "flops": 3 * rows * (h + kv) * d}


# ------------------------------------------------------------------- float64 --
def exact(case, seed):
    t = prepare(case, seed)
    return {"append": _exact_append, "prompts": _exact_prompts, "int4": _exact_int4}[case["kind"]](case, t)


def _attend(q, k, v, shift, window):
    """q [m, heads, d], k and v [n, kv, d] in float64, head by head."""
    m, h, d = q.shape
    out = torch.zeros_like(q)
    i, j = torch.arange(m, device="cuda")[:, None], torch.arange(k.shape[0], device="cuda")[None]
    seen = j <= i + shift
    if window:
        seen &= i - j < window
    some = seen.any(1, keepdim=True)
    for a in range(h):
        b = a * k.shape[1] // h
        s = (q[:, a].contiguous() @ k[:, b].t().contiguous()) / d ** 0.5
        p = torch.softmax(torch.where(seen | ~some, s, -math.inf), -1)
        out[:, a] = torch.where(some, p @ v[:, b].contiguous(), 0.0)
    return out


def _exact_prompts(c, t):
    out, at, from_ = [], 0, 0
    for m, n in zip(*_prompts(c)):
        k, v = (t[x][from_:from_ + n].double() for x in "kv")
        out.append(_attend(t["q"][at:at + m].double(), k, v, n - m, c["window"]))
        at, from_ = at + m, from_ + n
    return torch.cat(out)


def _decode(codes, pairs):
    """Values of [.., kv, dim / 2] codes: low nibble first, two's complement."""
    low, high = (codes & 0xF).double(), (codes >> 4).double()
    n = torch.stack((low, high), -1).reshape(*codes.shape[:-1], -1)
    n = torch.where(n > 7, n - 16, n)
    g = n.shape[-1] // pairs.shape[-2]
    return n * pairs[..., 0].double().repeat_interleave(g, -1) + pairs[..., 1].double().repeat_interleave(g, -1)


def _exact_int4(c, t):
    out = []
    for b, n in enumerate(_contexts(c)):
        pages = t["table"][b, :-(-n // c["page"])].long()
        k, v = (_decode(t[x + "codes"][pages], t[x + "par"][pages]).flatten(0, 1)[:n] for x in "kv")
        out.append(_attend(t["q"][b].double(), k, v, n - c["query"], 0))
    return torch.stack(out)


def _turned(x, t, c):
    """x [rows, heads, dim] in float64, each pair turned as a complex number."""
    n = c["dim"] // 2
    i = torch.arange(n, device="cuda", dtype=torch.float64)
    freq = (500000.0 if c["llama3"] else 10000.0) ** (-i / n)
    if c["llama3"]:
        turns = 8192.0 * freq / (2 * math.pi)
        share = ((turns - 1.0) / 3.0).clamp(0, 1)
        freq = freq * (share + (1 - share) / 8.0)
    by = torch.polar(torch.ones_like(freq), t["positions"].double()[:, None] * freq)[:, None]
    z = torch.complex(x[..., :n], x[..., n:]) if c["half"] else torch.view_as_complex(x.unflatten(-1, (n, 2)).contiguous())
    z = torch.view_as_real(z * by)
    return z.transpose(-1, -2).flatten(-2) if c["half"] else z.flatten(-2)


def _exact_append(c, t):
    q, k, v = _turned(t["q"].double(), t, c), _turned(t["k"].double(), t, c), t["v"].double()
    ids, slots, new = t["ids"].long(), t["slots"].long(), []
    for x, name in ((k, "k"), (v, "v")):
        if c["cache"] == "int4":
            pool = _decode(t[name + "pool"], t[name + "par"])
            x = x.reshape(*x.shape[:-1], -1, c["group"])
            scale = ((x.max(-1).values - x.min(-1).values) / 15).half().double()
            offset = ((x.max(-1).values + x.min(-1).values + scale) / 2).half().double()
            n = ((x - offset[..., None]) / scale[..., None]).round().clamp(-8, 7)
            x = (n * scale[..., None] + offset[..., None]).flatten(-2)
        else:
            pool = t[name + "pool"].double()
            if c["cache"] == "fp8":
                x = (x / t[name + "par"].double()[:, None]).clamp(-448, 448)
        pool[ids, slots] = x
        new.append(pool)
    return q, new[0], new[1]
