"""GPU: the appending page write with RoPE, the 4-bit cache (gather and attention) and attention
over packed sequences, against plain float64 on the CPU.

Bounds are counted, element by element, from the roundings a call makes: half a step of the
stored format (H = eps / 2, relative), f32 arithmetic (U = 2^-24 an operation) and, in the
attention kernels, P rounded once to 16 bits (H again, relative to sum p |v|).
"""
import math

import numpy as np
import pytest

import puter_amd
from puter_amd import PuterError

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3, I4 = puter_amd.BF16, puter_amd.F16, puter_amd.F32, puter_amd.F8E4M3, puter_amd.I4
T = {BF16: torch.bfloat16, F16: torch.float16, F32: torch.float32}
U = 2.0 ** -24


def H(f):
    return torch.finfo(T[f]).eps / 2


def tiny(f):  # half a step among the format's subnormals
    return {BF16: 0.0, F16: 2.0 ** -25, F32: 0.0}[f]


def randn(seed, shape, f, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(T[f])


def within(got, ref, bound, what=""):
    got, ref = got.double().cpu(), ref.double().cpu()
    over = (got - ref).abs() - bound
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3e} over the bound at {int(over.argmax())}, got {got.flatten()[over.argmax()]}, ref {ref.flatten()[over.argmax()]}"


# ------------------------------------------------------------------- append --
def turned(x, pos, mode, base=10000.0, llama3=None):
    """x [rows, heads, dim] in float64, and sum of the magnitudes that each output adds."""
    d = x.shape[-1]
    inv = base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    if llama3:
        factor, low, high, ctx = llama3
        wave = 2 * math.pi / inv
        s = (ctx / wave - low) / (high - low)
        inv = torch.where(wave > ctx / low, inv / factor, torch.where(wave < ctx / high, inv, (1 - s) * inv / factor + s * inv))
    a = pos.double()[:, None] * inv
    c, s = torch.cos(a)[:, None], torch.sin(a)[:, None]
    e, o = (x[..., :d // 2], x[..., d // 2:]) if mode else (x[..., 0::2], x[..., 1::2])
    r0, r1, m = e * c - o * s, e * s + o * c, e.abs() + o.abs()
    if mode:
        return torch.cat((r0, r1), -1), torch.cat((m, m), -1)
    return torch.stack((r0, r1), -1).flatten(-2), torch.stack((m, m), -1).flatten(-2)


def nibbles(codes):
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(torch.int16)
    return torch.where(n > 7, n - 16, n)


def check_int4(codes, pairs, x, slack, group, what):
    """Codes [.., dim / 2] and pairs [.., groups, 2] of the values x [.., dim] (known to within slack)."""
    n = nibbles(codes).double().unflatten(-1, (-1, group))
    x, slack = x.unflatten(-1, (-1, group)), slack.unflatten(-1, (-1, group))
    scale, offset = pairs[..., 0:1].double(), pairs[..., 1:2].double()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    e = slack.amax(-1, keepdim=True)
    h = 2.0 ** -11
    within(scale, (hi - lo) / 15, h * (hi - lo) / 15 + e + 2.0 ** -25, what + " scale")
    # offset: f16 of the middle plus half the stored scale, f32 roundings of terms below |lo| + |hi|
    mid = (lo + hi) / 2 + scale / 2
    within(offset, mid, h * mid.abs() + e + 4 * U * (lo.abs() + hi.abs()) + 2.0 ** -25, what + " offset")
    # the code: nearest, but for what f32 and the value's own slack move
    want = torch.where(scale > 0, (x - offset) / scale, torch.zeros_like(x)).clamp(-8, 7)
    moved = torch.where(scale > 0, (slack + 4 * U * (x.abs() + offset.abs())) / scale, torch.zeros_like(x))
    within(n, want, 0.5 + moved + 1e-6, what + " codes")


APPENDS = [
    # rows, q heads, kv heads, dim, format, cache, group, mode, page size, fused rows
    (1, 32, 8, 128, BF16, BF16, 0, 1, 16, True),
    (1, 8, 2, 128, BF16, I4, 64, 1, 16, True),
    (5, 7, 1, 64, F16, I4, 64, 1, 3, False),
    (33, 4, 4, 64, BF16, I4, 32, 0, 8, True),
    (130, 8, 2, 256, F16, I4, 128, 1, 32, False),
    (70, 6, 3, 256, BF16, I4, 32, 0, 16, True),
    (40, 4, 2, 128, F32, I4, 128, 1, 16, False),
    (64, 32, 8, 128, BF16, E4M3, 0, 1, 16, True),
    (19, 3, 3, 96, F16, E4M3, 0, 0, 5, False),
    (9, 2, 1, 20, BF16, E4M3, 0, 1, 4, True),
    (77, 5, 5, 80, F32, F32, 0, 1, 7, True),
    (21, 3, 1, 2, F16, F16, 0, 0, 16, False),
    (3, 1, 1, 1022, F32, F32, 0, 1, 2, True),
    (12, 0, 2, 64, BF16, BF16, 0, 1, 4, False),
    (1100, 4, 2, 64, BF16, BF16, 0, 1, 16, True),
    (1500, 2, 2, 128, F16, I4, 32, 1, 64, True),
    (9000, 2, 1, 64, BF16, E4M3, 0, 0, 16, False),
    (4097, 4, 2, 64, BF16, BF16, 0, 1, 16, True),
    (4500, 2, 2, 128, F16, I4, 32, 1, 64, True),
    (6001, 2, 1, 256, BF16, I4, 128, 0, 16, False),
    (4200, 2, 1, 48, F32, F32, 0, 0, 16, False),
    (5000, 1, 1, 36, F32, E4M3, 0, 1, 8, True),
]


def append_state(rows, qh, kvh, dim, f, cache, group, page, fused, seed=0, spare=3):
    pages = -(-rows // page) + spare
    g = torch.Generator().manual_seed(seed + 9)
    slot = torch.randperm(pages * page, generator=g)[:rows]
    s = {"ids": (slot // page).int(), "slots": (slot % page).int(), "pages": pages,
         "pos": torch.randint(0, 131072, (rows,), generator=g, dtype=torch.int32)}
    q, k, v = randn(seed, (rows, qh, dim), f), randn(seed + 1, (rows, kvh, dim), f, 2.0), randn(seed + 2, (rows, kvh, dim), f)
    s["x"] = (q.double(), k.double(), v.double())
    if fused:
        whole = torch.cat((q, k, v), 1).cuda()
        s["dev"] = (whole[:, :qh], whole[:, qh:qh + kvh], whole[:, qh + kvh:])
    else:
        s["dev"] = (q.cuda(), k.cuda(), v.cuda())
    s["qout"] = torch.full((rows, max(qh, 1), dim), 7.0, dtype=T[f], device="cuda")
    if cache == I4:
        s["pools"] = [torch.randint(0, 256, (pages, page, kvh, dim // 2), generator=g, dtype=torch.uint8).cuda() for _ in range(2)]
        s["par"] = [torch.randn((pages, page, kvh, dim // group, 2), generator=g).half().cuda() for _ in range(2)]
    elif cache == E4M3:
        s["pools"] = [torch.randint(0, 120, (pages, page, kvh, dim), generator=g, dtype=torch.uint8).cuda() for _ in range(2)]
        s["par"] = [(torch.rand(kvh, generator=g) * 0.02 + 0.01).cuda() for _ in range(2)]
    else:
        s["pools"] = [randn(seed + 5 + i, (pages, page, kvh, dim), f).cuda() for i in range(2)]
        s["par"] = [None, None]
    return s


def call_append(be, cfg, s, rows, qh, kvh, dim, f, cache, group, page):
    q, k, v = s["dev"]
    be.KVPageAppendRoPE(cfg, q if qh else None, k, v, s["pos"].cuda(), s["ids"].cuda(), s["slots"].cuda(),
                        s["qout"] if qh else None, s["pools"][0], s["pools"][1], s["par"][0], s["par"][1], rows, qh, kvh,
                        dim, q.stride(0) if qh else 0, k.stride(0), v.stride(0), s["pages"], page, group, f, cache)


@pytest.mark.parametrize("rows,qh,kvh,dim,f,cache,group,mode,page,fused", APPENDS)
def test_append(backend, rows, qh, kvh, dim, f, cache, group, mode, page, fused):
    s = append_state(rows, qh, kvh, dim, f, cache, group, page, fused)
    llama3 = (8.0, 1.0, 4.0, 8192) if dim == 128 else None
    cfg = puter_amd.RoPEConfig(500000.0, 3, mode, 1, 8.0, 1.0, 4.0, 8192) if llama3 else \
        puter_amd.RoPEConfig(BaseFreq=10000.0, StartPosition=3, Mode=mode)
    before = [p.clone() for p in s["pools"]], [p.clone() if p is not None else None for p in s["par"]]
    call_append(backend, cfg, s, rows, qh, kvh, dim, f, cache, group, page)
    backend.CheckStatus()
    base = 500000.0 if llama3 else 10000.0
    q, qm = turned(s["x"][0], s["pos"] + 3, mode, base, llama3)
    k, km = turned(s["x"][1], s["pos"] + 3, mode, base, llama3)
    v = s["x"][2]
    # two products and a sum, cos and sin rounded to f32: four roundings of terms up to |x| + |y|
    if qh:
        within(s["qout"], q, H(f) * q.abs() + 5 * U * qm + tiny(f), "query")
    at = (s["ids"].long(), s["slots"].long())
    for i, (x, slack) in enumerate(((k, 5 * U * km), (v, torch.zeros_like(v)))):
        name = "key" if i == 0 else "value"
        pool = s["pools"][i].cpu()
        got = pool[at]
        if cache == I4:
            check_int4(got, s["par"][i].cpu()[at], x, slack, group, name)
        elif cache == E4M3:
            y = x / s["par"][i].double().cpu()[:, None]
            want = y.clamp(-448, 448)
            b = 2.0 ** -4 * want.abs() + 2.0 ** -10 + (slack / s["par"][i].double().cpu()[:, None]) + 2 * U * want.abs()
            within(got.view(torch.float8_e4m3fn).double(), want, b, name)
        else:
            within(got, x, H(f) * x.abs() + slack + tiny(f), name)
        # every other slot is as it was
        keep = torch.ones(pool.shape[:2], dtype=torch.bool)
        keep[at] = False
        assert torch.equal(pool[keep].view(torch.uint8), before[0][i].cpu()[keep].view(torch.uint8))
        if cache == I4:
            assert torch.equal(s["par"][i].cpu()[keep].view(torch.uint8), before[1][i].cpu()[keep].view(torch.uint8))


@pytest.mark.parametrize("f", [BF16, F16, F32])
@pytest.mark.parametrize("mode", [0, 1])
def test_append_is_rope_and_page_write(backend, f, mode):
    """The 16-bit and f32 cache: what RoPE of each row and KVPageWrite leave, to a rounding."""
    rows, qh, kvh, dim, page = 6, 4, 2, 128, 4
    s = append_state(rows, qh, kvh, dim, f, f, 0, page, True, seed=5)
    call_append(backend, puter_amd.RoPEConfig(Mode=mode), s, rows, qh, kvh, dim, f, f, 0, page)
    k, v = s["dev"][1].contiguous(), s["dev"][2].contiguous()
    for r in range(rows):
        backend.RoPE(puter_amd.RoPEConfig(Mode=mode, StartPosition=int(s["pos"][r])), k[r], k[r], 1, kvh, dim, f)
    want = [torch.zeros_like(p) for p in s["pools"]]
    for w, x in zip(want, (k, v)):
        backend.KVPageWrite(w, x, s["ids"].cuda(), s["slots"].cuda(), w, s["pages"], page, kvh * dim, rows, 0, f)
    torch.cuda.synchronize()
    at = (s["ids"].long(), s["slots"].long())
    km = turned(s["x"][1], s["pos"], mode)[1]
    ref = want[0].cpu()[at].double()
    within(s["pools"][0].cpu()[at], ref, 2 * H(f) * ref.abs() + 8 * U * km + 2 * tiny(f), "key")
    assert torch.equal(s["pools"][1].cpu()[at], want[1].cpu()[at])


@pytest.mark.parametrize("f", [BF16, F16, F32])
@pytest.mark.parametrize("rows,dim", [(70, 64), (70, 20), (1500, 64), (4500, 64)])
def test_append_fp8_bytes_are_the_page_write_s(backend, f, rows, dim):
    """Unrotated rows into fp8 pages: byte for byte what KVPageWriteFP8 stores, whatever the scale
    (least, zero, negative, vast, not a number) and the value (ties, infinities, NaN)."""
    scales = torch.tensor([1.0, 0.0078, 3.0, 1e-42, 0.0, 2.0 ** -60, 2.0 ** -61, 1e30, -0.5, math.inf, math.nan, 3e38]).cuda()
    kvh, page = len(scales), 16
    s = append_state(rows, 1, kvh, dim, f, E4M3, 0, page, False, seed=21)
    k = s["dev"][1]
    grid = torch.arange(rows * dim, device="cuda").view(rows, dim)
    tie = ((grid % 127) + 8.5) / 16 * torch.exp2((grid % 23 - 12).float())    # half steps of the format
    for h in range(kvh):
        k[:, h] = (tie * (scales[h] if torch.isfinite(scales[h]) else 1.0)).clamp(-3e38, 3e38).to(T[f])
    k[0, :, :4] = torch.tensor([math.inf, -math.inf, math.nan, 0.0], device="cuda").to(T[f])
    s["par"] = [scales, scales.flip(0).contiguous()]
    want = [p.clone() for p in s["pools"]]
    call_append(backend, None, s, rows, 1, kvh, dim, f, E4M3, 0, page)
    for w, x, p in zip(want, s["dev"][1:], s["par"]):
        backend.KVPageWriteFP8(w, x, s["ids"].cuda(), s["slots"].cuda(), s["pages"], page, kvh, dim, rows, 0, p, f)
    backend.CheckStatus()
    for got, w in zip(s["pools"], want):
        assert torch.equal(got, w)


@pytest.mark.parametrize("rows", [5, 1100, 4400])
@pytest.mark.parametrize("f,dim,mode", [(BF16, 128, 1), (F32, 64, 0), (F16, 36, 0)])
def test_append_turns_queries_in_place(backend, rows, f, dim, mode):
    s = append_state(rows, 4, 2, dim, f, f, 0, 16, False, seed=31)
    own = append_state(rows, 4, 2, dim, f, f, 0, 16, False, seed=31)
    cfg = puter_amd.RoPEConfig(Mode=mode)
    call_append(backend, cfg, s, rows, 4, 2, dim, f, f, 0, 16)
    own["qout"] = own["dev"][0]
    call_append(backend, cfg, own, rows, 4, 2, dim, f, f, 0, 16)
    backend.CheckStatus()
    for a, b in zip([s["qout"]] + s["pools"], [own["qout"]] + own["pools"]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_without_rotation(backend):
    rows, kvh, dim, page = 10, 2, 64, 4
    s = append_state(rows, 3, kvh, dim, BF16, BF16, 0, page, True, seed=8)
    q, k, v = s["dev"]
    backend.KVPageAppendRoPE(None, q, k, v, None, s["ids"].cuda(), s["slots"].cuda(), s["qout"], s["pools"][0], s["pools"][1],
                             None, None, rows, 3, kvh, dim, q.stride(0), k.stride(0), v.stride(0), s["pages"], page, 0, BF16, BF16)
    torch.cuda.synchronize()
    at = (s["ids"].long(), s["slots"].long())
    assert torch.equal(s["qout"], q) and torch.equal(s["pools"][0].cpu()[at], k.cpu()) and torch.equal(s["pools"][1].cpu()[at], v.cpu())


@pytest.mark.parametrize("rows", [3, 40, 700, 2500, 6000])
@pytest.mark.parametrize("cache", [BF16, E4M3, I4])
def test_append_last_row_of_a_slot_wins(backend, rows, cache):
    """Several rows of one slot, near and far apart: the last one's K, V and pair stand."""
    kvh, dim, page, group = 2, 64, 8, 32
    s = append_state(rows, 1, kvh, dim, BF16, cache, group, page, False, seed=3)
    g = torch.Generator().manual_seed(rows)
    s["ids"][:] = torch.randint(0, max(1, s["pages"] // 4), (rows,), generator=g, dtype=torch.int32)
    s["ids"][-1] = s["ids"][0]
    s["slots"][-1] = s["slots"][0]
    cfg = puter_amd.RoPEConfig(Mode=1)
    call_append(backend, cfg, s, rows, 1, kvh, dim, BF16, cache, group, page)
    backend.CheckStatus()
    last = {}
    for r, at in enumerate(zip(s["ids"].tolist(), s["slots"].tolist())):
        last[at] = r
    rows1 = torch.tensor(sorted(last.values()))
    one = append_state(rows, 1, kvh, dim, BF16, cache, group, page, False, seed=3)
    one["dev"] = tuple(x[rows1.cuda()].contiguous() for x in one["dev"])
    for n in ("ids", "slots", "pos"):
        one[n] = s[n][rows1]
    one["qout"] = torch.zeros((len(rows1), 1, dim), dtype=T[BF16], device="cuda")
    call_append(backend, cfg, one, len(rows1), 1, kvh, dim, BF16, cache, group, page)
    torch.cuda.synchronize()
    for a, b in zip(s["pools"] + (s["par"] if cache == I4 else []), one["pools"] + (one["par"] if cache == I4 else [])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("cache", [F16, E4M3, I4])
def test_append_bad_ids_are_flagged_and_skipped(backend, cache):
    rows, kvh, dim, page, group = 9, 2, 64, 4, 32
    s = append_state(rows, 2, kvh, dim, F16, cache, group, page, True, seed=4)
    good = append_state(rows, 2, kvh, dim, F16, cache, group, page, True, seed=4)
    s["ids"][1], s["ids"][4], s["slots"][7], s["slots"][2] = -1, s["pages"], page, -3
    call_append(backend, puter_amd.RoPEConfig(Mode=1), s, rows, 2, kvh, dim, F16, cache, group, page)
    with pytest.raises(PuterError):
        backend.CheckStatus()
    call_append(backend, puter_amd.RoPEConfig(Mode=1), good, rows, 2, kvh, dim, F16, cache, group, page)
    backend.CheckStatus()
    assert torch.equal(s["qout"], good["qout"])   # every query is written
    fresh = append_state(rows, 2, kvh, dim, F16, cache, group, page, True, seed=4)
    skipped = torch.zeros(s["pages"], page, dtype=torch.bool)
    for r in (1, 4, 7, 2):
        skipped[good["ids"][r].long(), good["slots"][r].long()] = True
    for a, b, c in zip(s["pools"], good["pools"], fresh["pools"]):
        a, b, c = (x.cpu().view(torch.uint8) for x in (a, b, c))
        assert torch.equal(a[skipped], c[skipped]) and torch.equal(a[~skipped], b[~skipped])


def test_append_int4_edges(backend):
    """Equal values (scale 0), NaN, infinities, f16's range and its subnormals, one group each."""
    kvh, dim, page, group = 1, 256, 4, 32
    x = torch.zeros(1, 1, dim)
    x[..., 0:32] = 1.5
    x[..., 32:64] = torch.linspace(-3, 4, 32)
    x[..., 40] = float("nan")
    x[..., 64:96] = torch.linspace(-1, 1, 32)
    x[..., 70], x[..., 71] = float("inf"), float("-inf")
    x[..., 96:128] = 3e38 * torch.linspace(-1, 1, 32)
    x[..., 128:160] = torch.linspace(0, 1e-6, 32)
    x[..., 160:192] = torch.linspace(100, 100.5, 32)
    x[..., 192:224] = -torch.linspace(0, 60000, 32)
    codes = [torch.zeros((1, page, kvh, dim // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    pairs = [torch.zeros((1, page, kvh, dim // group, 2), dtype=torch.float16, device="cuda") for _ in range(2)]
    d = x.cuda()
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    backend.KVPageAppendRoPE(None, None, d, d, None, zero, zero, None, codes[0], codes[1], pairs[0], pairs[1], 1, 0, kvh, dim, 0,
                             dim, dim, 1, page, group, F32, I4)
    out = torch.empty((page, kvh, dim), device="cuda")
    backend.KVPageGatherInt4(codes[0], pairs[0], zero, out, 1, page, kvh, dim, group, page, F32)
    backend.CheckStatus()
    got, x = out[0, 0].cpu().double(), x[0, 0].double()
    assert (got[0:32] == 1.5).all()
    assert got[32:64].isnan().all()
    assert torch.isfinite(got[64:]).all()
    assert got[70] > 60000 and got[71] < -60000 and got[127] > 60000
    for lo in (128, 160, 192):
        part, g = x[lo:lo + 32], got[lo:lo + 32]
        step = float(part.max() - part.min()) / 15
        # half a step, the scale's rounding over 8 steps, the offset's
        b = step * (0.5 + 8 * 2.0 ** -11) + 2.0 ** -11 * float(part.abs().max()) + 9 * 2.0 ** -25 + 1e-6 * float(part.abs().max())
        within(g, part, torch.full_like(part, b), f"group at {lo}")
    assert torch.equal(codes[0], codes[1])


@pytest.mark.parametrize("f", [BF16, F16, F32])
@pytest.mark.parametrize("dim,group,kvh,page,rows", [(128, 64, 2, 16, 37), (64, 32, 3, 5, 11), (256, 128, 1, 4, 1)])
def test_gather_int4(backend, f, dim, group, kvh, page, rows):
    g = torch.Generator().manual_seed(dim + rows)
    pages = 9
    codes = torch.randint(0, 256, (pages, page, kvh, dim // 2), generator=g, dtype=torch.uint8)
    pairs = torch.randn((pages, page, kvh, dim // group, 2), generator=g).half()
    table = torch.randint(0, pages, (-(-rows // page),), generator=g, dtype=torch.int32)
    out = torch.full((rows + 2, kvh, dim), 5.0, dtype=T[f], device="cuda")
    backend.KVPageGatherInt4(codes.cuda(), pairs.cuda(), table.cuda(), out, pages, page, kvh, dim, group, rows, f)
    backend.CheckStatus()
    n = nibbles(codes).double().unflatten(-1, (-1, group))
    values = (n * pairs[..., :1].double() + pairs[..., 1:].double()).flatten(-2)
    want = values[table.long()].flatten(0, 1)[:rows]
    big = (8 * pairs[..., :1].double().abs() + pairs[..., 1:].double().abs()).expand_as(n).flatten(-2)[table.long()].flatten(0, 1)[:rows]
    within(out[:rows], want, H(f) * want.abs() + 2 * U * big + tiny(f))
    assert (out[rows:] == 5.0).all()
    table[0] = pages
    backend.KVPageGatherInt4(codes.cuda(), pairs.cuda(), table.cuda(), out, pages, page, kvh, dim, group, rows, f)
    with pytest.raises(PuterError):
        backend.CheckStatus()
    assert (out[:min(page, rows)] == 0).all()


# --------------------------------------------------------- plain attention --
def attend(q, k, v, shift, causal=True, window=0, alibi=0.0):
    """q [m, h, d], k and v [n, kv, d] in float64: outputs, sum p |v|, the largest sum |q k| / sqrt(d)."""
    m, h, d = q.shape
    n, kv = k.shape[0], k.shape[1]
    out, mag, top = torch.zeros(m, h, d, dtype=torch.float64), torch.zeros(m, h, d, dtype=torch.float64), 0.0
    i, j = torch.arange(m)[:, None], torch.arange(n)[None]
    seen = torch.ones(m, n, dtype=torch.bool)
    if causal:
        seen &= j <= i + shift
    if window:
        seen &= i - j < window
    some = seen.any(1, keepdim=True)
    if n == 0:
        return out, mag, top
    for a in range(h):
        b = a * kv // h
        s = q[:, a] @ k[:, b].T / math.sqrt(d) + alibi * (j - i)
        top = max(top, float((q[:, a].abs() @ k[:, b].abs().T).max()) / math.sqrt(d) + abs(alibi) * max(m, n))
        s = torch.where(seen, s, torch.tensor(-math.inf, dtype=torch.float64))
        p = torch.where(some, torch.softmax(torch.where(some, s, torch.zeros_like(s)), -1), torch.zeros_like(s))
        out[:, a], mag[:, a] = p @ v[:, b], p @ v[:, b].abs()
    return out, mag, top


def attention_bound(f, ref, mag, top, d, n, p_bits):
    """Half a step of the output; P's rounding; scores off by at most d + 4 roundings of `top`
    (twice that relative in p / sum p); n roundings in each of the two sums over keys."""
    rel = 2 * (d + 4) * U * top + 2 * (n + 8) * U + 8 * U
    return H(f) * ref.abs() + (p_bits + rel) * mag * (1 + H(f)) + tiny(f)


# -------------------------------------------------------------------- packed --
def packed_state(lens, keys, h, kv, d, f, seed=0):
    q = randn(seed, (sum(lens), h, d), f)
    k, v = randn(seed + 1, (sum(keys), kv, d), f), randn(seed + 2, (sum(keys), kv, d), f)
    off = [torch.tensor(np.concatenate(([0], np.cumsum(x))), dtype=torch.int32) for x in (lens, keys)]
    return q, k, v, off


def packed_refs(q, k, v, lens, keys, **kw):
    refs, a, b = [], 0, 0
    for m, n in zip(lens, keys):
        refs.append(attend(q[a:a + m].double(), k[b:b + n].double(), v[b:b + n].double(), n - m, **kw))
        a, b = a + m, b + n
    return refs


def call_packed(be, q, k, v, out, qoff, koff, h, kv, d, f, causal=True, window=0, alibi=0.0, total_q=None, total_k=None, batch=None):
    cfg = puter_amd.MultiHeadAttentionConfig(h, d, causal, window, alibi, kv)
    be.MultiHeadAttentionPacked(cfg, q, k, v, out, qoff, koff, len(qoff) - 1 if batch is None else batch,
                                q.shape[0] if total_q is None else total_q, k.shape[0] if total_k is None else total_k, f)


def p_bits(f):
    return 0.0 if f == F32 else H(f)


PACKED = [
    ([1], None, 4, 2, 128, {}),
    ([128, 1, 129, 127], None, 4, 1, 128, {}),
    ([0, 5, 0, 130, 0], None, 8, 8, 64, {}),
    ([300, 17, 64, 65], None, 6, 2, 64, {}),
    ([200, 40], None, 2, 2, 256, {}),
    ([33, 100, 7], None, 4, 4, 96, {}),
    ([70, 150], None, 3, 1, 80, {}),
    ([50, 9], None, 5, 5, 20, {}),           # f32: the matrix cores; 16 bits: no multiple of 8
    ([31, 64], None, 2, 1, 7, {}),
    ([12, 200], [112, 300], 4, 2, 128, {}),   # keys before the first query
    ([150, 20, 3], [40, 0, 3], 4, 4, 64, {}),   # fewer keys than queries: rows that see none
    ([200, 90], None, 4, 2, 128, {"window": 50}),
    ([200, 90], [260, 90], 2, 2, 80, {"window": 64}),
    ([150, 3], None, 4, 4, 64, {"alibi": 0.06}),
    ([150, 40], [150, 77], 2, 2, 128, {"causal": False}),
    ([60, 61], None, 4, 2, 128, {"causal": False, "window": 9, "alibi": -0.1}),
]


@pytest.mark.parametrize("f", [BF16, F16, F32])
@pytest.mark.parametrize("lens,keys,h,kv,d,kw", PACKED)
def test_packed(backend, f, lens, keys, h, kv, d, kw):
    own = keys is None
    keys = lens if own else keys
    q, k, v, off = packed_state(lens, keys, h, kv, d, f, seed=d)
    out = torch.full((q.shape[0] + 3, h, d), 9.0, dtype=T[f], device="cuda")
    call_packed(backend, q.cuda(), k.cuda(), v.cuda(), out, off[0].cuda(), None if own else off[1].cuda(), h, kv, d, f, **kw)
    backend.CheckStatus()
    at = 0
    for m, n, (ref, mag, top) in zip(lens, keys, packed_refs(q, k, v, lens, keys, **kw)):
        within(out[at:at + m], ref, attention_bound(f, ref, mag, top, d, n, p_bits(f)), f"{m} of {n}")
        at += m
    assert (out[at:] == 9.0).all()


@pytest.mark.parametrize("f", [BF16, F32])
def test_packed_many_sequences(backend, f):
    """More sequences than a wave, or four, has lanes, empty ones among them."""
    rng = np.random.default_rng(3)
    for count in (65, 300):
        lens = rng.integers(0, 9, count).tolist()
        lens[count // 2] = 150
        q, k, v, off = packed_state(lens, lens, 2, 1, 64, f, seed=count)
        out = torch.zeros(q.shape, dtype=T[f], device="cuda")
        call_packed(backend, q.cuda(), k.cuda(), v.cuda(), out, off[0].cuda(), None, 2, 1, 64, f)
        refs = packed_refs(q, k, v, lens, lens)
        ref, mag = (torch.cat([r[i] for r in refs]) for i in (0, 1))
        within(out, ref, attention_bound(f, ref, mag, max(r[2] for r in refs), 64, 150, p_bits(f)))


@pytest.mark.parametrize("f,d", [(BF16, 128), (F16, 64), (F32, 64), (BF16, 96), (F32, 20), (BF16, 20)])
def test_packed_hidden_values_have_no_effect(backend, f, d):
    """NaN and infinities in keys and values that a row may not see leave it as it is; those it
    sees reach it."""
    lens = [90, 40]
    q, k, v, off = packed_state(lens, lens, 2, 2, d, f, seed=11)
    clean = torch.zeros(q.shape, dtype=T[f], device="cuda")
    call_packed(backend, q.cuda(), k.cuda(), v.cuda(), clean, off[0].cuda(), None, 2, 2, d, f)
    k2, v2 = k.clone(), v.clone()
    v2[50], v2[51, :, 0], k2[70] = float("nan"), float("inf"), float("nan")
    out = torch.zeros(q.shape, dtype=T[f], device="cuda")
    call_packed(backend, q.cuda(), k2.cuda(), v2.cuda(), out, off[0].cuda(), None, 2, 2, d, f)
    torch.cuda.synchronize()
    out, clean = out.cpu(), clean.cpu()
    # (bit-equal where nothing hidden shares a tile; elsewhere the kernels weigh a row again against
    # its final maximum instead of the running one, other roundings of the same sums: each is
    # within the bound of any attention output)
    ref, mag, top = packed_refs(q, k, v, lens, lens)[0]
    bound = attention_bound(f, ref, mag, top, d, 90, p_bits(f))
    within(out[:50], ref[:50], bound[:50], "rows before the NaN")
    assert torch.equal(out[90:], clean[90:])
    assert out[50:90].isnan().all()
    v2 = v.clone()
    v2[51, :, 0] = float("inf")
    call_packed(backend, q.cuda(), k.cuda(), v2.cuda(), (o := torch.zeros(q.shape, dtype=T[f], device="cuda")), off[0].cuda(), None, 2, 2, d, f)
    torch.cuda.synchronize()
    o = o.cpu()
    within(o[:51], ref[:51], bound[:51], "rows before the infinity")
    assert (o[51:90, :, 0] == float("inf")).all()
    within(o[51:90, :, 1:], ref[51:90, :, 1:], bound[51:90, :, 1:], "other dims")


@pytest.mark.parametrize("f,d", [(BF16, 128), (F32, 64), (F16, 20)])
def test_packed_bad_offsets_are_reported(backend, f, d):
    lens = [30, 40, 20]
    q, k, v, off = packed_state(lens, lens, 2, 1, d, f)
    for bad in ([0, 30, 70, 91], [0, 50, 30, 90], [-5, 30, 70, 90], [0, 2 ** 31 - 1, 70, 90], [0, -2 ** 31, 70, 90]):
        out = torch.zeros(q.shape, dtype=T[f], device="cuda")
        b = torch.tensor(bad, dtype=torch.int32).cuda()
        call_packed(backend, q.cuda(), k.cuda(), v.cuda(), out, b, None, 2, 1, d, f)
        with pytest.raises(PuterError):
            backend.CheckStatus()
        call_packed(backend, q.cuda(), k.cuda(), v.cuda(), out, off[0].cuda(), b, 2, 1, d, f)
        with pytest.raises(PuterError):
            backend.CheckStatus()
    # rows before the first offset and from the last on stay
    out = torch.full(q.shape, 4.0, dtype=T[f], device="cuda")
    call_packed(backend, q.cuda(), k.cuda(), v.cuda(), out, torch.tensor([10, 30, 70], dtype=torch.int32).cuda(), None, 2, 1, d, f)
    backend.CheckStatus()
    assert (out[:10] == 4.0).all() and (out[70:] == 4.0).all()
    ref, mag, top = attend(q[10:30].double(), k[10:30].double(), v[10:30].double(), 0)
    within(out[10:30], ref, attention_bound(f, ref, mag, top, d, 20, p_bits(f)))


def test_packed_rows_past_4_gib(backend):
    """Queries and outputs that pass 2^32 bytes: the last sequence's rows."""
    h, kv, d, f, n, b = 32, 2, 128, BF16, 1000, 530
    q = torch.randn((n * b, h, d), dtype=T[f], device="cuda")
    k, v = (torch.randn((n * b, kv, d), dtype=T[f], device="cuda") for _ in range(2))
    off = torch.arange(b + 1, dtype=torch.int32, device="cuda") * n
    out = torch.zeros_like(q)
    call_packed(backend, q, k, v, out, off, None, h, kv, d, f)
    backend.CheckStatus()
    for at in (0, (b - 1) * n):
        rows = slice(at, at + n)
        ref, mag, top = attend(q[rows].double().cpu(), k[rows].double().cpu(), v[rows].double().cpu(), 0)
        within(out[rows], ref, attention_bound(f, ref, mag, top, d, n, p_bits(f)), at)


def test_packed_unaligned(backend):
    lens, h, kv, d = [40, 70], 2, 2, 64
    q, k, v, off = packed_state(lens, lens, h, kv, d, BF16)
    def shifted(x):
        b = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")
        b[1:] = x.flatten().cuda()
        return b[1:].view(x.shape)
    out = shifted(torch.zeros_like(q))
    call_packed(backend, shifted(q), shifted(k), shifted(v), out, off[0].cuda(), None, h, kv, d, BF16)
    refs = packed_refs(q, k, v, lens, lens)
    ref, mag = (torch.cat([r[i] for r in refs]) for i in (0, 1))
    within(out, ref, attention_bound(BF16, ref, mag, max(r[2] for r in refs), d, 70, p_bits(BF16)))


# ---------------------------------------------------------------------- int4 --
def int4_state(ctx, m, h, kv, d, group, page, f, seed=0, table_extra=1):
    g = torch.Generator().manual_seed(seed + 77)
    counts = [-(-max(n, 0) // page) for n in ctx]
    pages = sum(counts) + 2
    perm = torch.randperm(pages, generator=g).int()
    table = torch.full((len(ctx), max(counts) + table_extra), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = perm[at:at + n]
        at += n
    s = {"table": table, "ctx": torch.tensor(ctx, dtype=torch.int32), "pages": pages, "q": randn(seed, (len(ctx), m, h, d), f)}
    for x in "kv":
        s[x + "c"] = torch.randint(0, 256, (pages, page, kv, d // 2), generator=g, dtype=torch.uint8)
        p = torch.rand((pages, page, kv, d // group, 2), generator=g) * 0.3
        p[..., 1] -= 0.15
        s[x + "p"] = p.half()
    return s


def call_int4(be, s, m, h, kv, d, group, page, f, max_context=None, out=None, ws=None, max_pages=None):
    b = len(s["ctx"])
    dev = {n: s[n].cuda() for n in ("q", "kc", "vc", "kp", "vp", "table", "ctx")}
    maxc = max(1, int(s["ctx"].max())) if max_context is None else max_context
    need = be.PagedInt4WorkspaceBytes(b, m, h, kv, d, maxc)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda") if ws is None else ws
    out = torch.full((b, m, h, d), 3.0, dtype=T[f], device="cuda") if out is None else out
    be.PagedInt4Attention(dev["q"], dev["kc"], dev["vc"], dev["kp"], dev["vp"], dev["table"], dev["ctx"], b, m,
                          s["table"].shape[1], page, s["pages"], h, kv, d, group, maxc, f, out, ws, need)
    torch.cuda.synchronize()
    return out


def int4_values(codes, pairs):
    n = nibbles(codes).double().unflatten(-1, (pairs.shape[-2], -1))
    return (n * pairs[..., :1].double() + pairs[..., 1:].double()).flatten(-2)


def check_int4_attention(out, s, m, page, f, d, max_context=None, bad_pages=()):
    for b, n in enumerate(s["ctx"].tolist()):
        n = max(0, n if max_context is None else min(n, max_context))
        ids = s["table"][b, :-(-n // page)].long()
        keep = torch.ones(n, dtype=torch.bool)
        for i in bad_pages:
            if i < len(ids):
                keep[i * page:(i + 1) * page] = False
                ids[i] = 0
        k, v = (int4_values(s[x + "c"][ids], s[x + "p"][ids]).flatten(0, 1)[:n] for x in "kv")
        part = s["vp"][ids].clone()
        part[..., 1] = 0
        codes = int4_values(s["vc"][ids], part).flatten(0, 1)[:n]   # the values without their offsets
        for i in range(m):   # each query with the keys it sees
            mine = keep & (torch.arange(n) <= n - m + i)
            ref, mag, top = attend(s["q"][b, i:i + 1].double(), k[mine], v[mine], 0, causal=False)
            # the code products and the offset sums cancel: terms up to 24 steps beside the value's 8 and offset
            bound = attention_bound(f, ref, 6 * mag + 1e-3 * mag.max(), 6 * top, d, max(n, 1), 2.0 ** -16)
            # P is scaled by the token's scale and rounded once to bf16 for bf16 outputs, half a step, before
            # it meets the code: off by at most H sum p |scale n| (the offsets meet p itself)
            if f == BF16:
                bound += H(f) * (1 + H(f)) * attend(s["q"][b, i:i + 1].double(), k[mine], codes[mine], 0, causal=False)[1]
            within(out[b, i:i + 1], ref, bound, f"sequence {b}, query {i}")


def test_4_bit_pools_past_4_gib(backend):
    """Append, gather and attention on a page whose codes lie past 2^32 bytes of the pool."""
    h, kv, d, group, page, n, f = 4, 2, 128, 64, 16, 40, BF16
    pages = (1 << 32) // (page * kv * d // 2) + 8
    pools = [torch.empty((pages, page, kv, d // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    par = [torch.empty((pages, page, kv, d // group, 2), dtype=torch.float16, device="cuda") for _ in range(2)]
    table = torch.tensor([[pages - 1, pages - 3, pages - 2]], dtype=torch.int32)
    q, k, v = (randn(60 + i, (n, x, d), f).cuda() for i, x in enumerate((h, kv, kv)))
    t = torch.arange(n, dtype=torch.int32)
    backend.KVPageAppendRoPE(None, None, k, v, None, table[0][(t // page).long()].cuda(), (t % page).cuda(), None, pools[0], pools[1],
                             par[0], par[1], n, 0, kv, d, 0, kv * d, kv * d, pages, page, group, f, I4)
    last = slice(pages - 4, pages)
    s = {"table": table - (pages - 4), "ctx": torch.tensor([n], dtype=torch.int32), "q": q.cpu()[-1:].unsqueeze(1)}
    for x, c, p in zip("kv", pools, par):
        s[x + "c"], s[x + "p"] = c[last].cpu(), p[last].cpu()
        out = torch.empty((n, kv, d), dtype=T[f], device="cuda")
        backend.KVPageGatherInt4(c, p, table.cuda(), out, pages, page, kv, d, group, n, f)
        ids = s["table"][0].long()
        val = int4_values(s[x + "c"][ids], s[x + "p"][ids]).flatten(0, 1)[:n]
        within(out, val, H(f) * val.abs() + 2 * U * (val.abs() + 16), "gather")   # a product and a sum, terms below 16
    for i, x in enumerate((k, v)):
        check_int4(s["kv"[i] + "c"][ids].flatten(0, 1)[:n], s["kv"[i] + "p"][ids].flatten(0, 1)[:n], x.double().cpu(),
                   torch.zeros(x.shape, dtype=torch.float64), group, "kv"[i])
    need = backend.PagedInt4WorkspaceBytes(1, 1, h, kv, d, n)
    ws, o = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.zeros((1, 1, h, d), dtype=T[f], device="cuda")
    backend.PagedInt4Attention(q[-1:], pools[0], pools[1], par[0], par[1], table.cuda(), s["ctx"].cuda(), 1, 1, 3, page, pages, h, kv, d,
                               group, n, f, o, ws, need)
    backend.CheckStatus()
    check_int4_attention(o, s, 1, page, f, d)


INT4 = [
    # contexts, queries, heads, kv heads, dim, group, page
    ([1], 1, 1, 1, 64, 64, 1),
    ([1, 2, 16, 17], 1, 4, 1, 128, 64, 16),
    ([63, 64, 65, 255, 256, 257], 1, 8, 2, 128, 128, 16),
    ([0, 40, 0], 1, 4, 4, 128, 32, 16),
    ([500, 3], 1, 16, 1, 128, 32, 64),
    ([90, 333], 1, 6, 3, 64, 32, 24),
    ([90, 333], 1, 5, 5, 256, 128, 8),
    ([77, 130], 1, 14, 2, 256, 32, 5),
    ([1000, 601], 1, 8, 8, 64, 64, 32),
    ([300, 41], 5, 8, 2, 64, 64, 24),
    ([130, 4, 2], 4, 8, 1, 128, 64, 16),   # more queries than tokens in one
    ([200], 17, 4, 2, 128, 32, 16),
    ([90], 90, 2, 1, 64, 32, 16),          # a whole prompt
    ([150, 70], 3, 40, 2, 128, 128, 7),    # 20 heads to a kv head
    ([4100, 900], 1, 4, 2, 128, 64, 16),
    ([2500], 2, 32, 1, 256, 64, 128),
]


@pytest.mark.parametrize("f", [BF16, F16])
@pytest.mark.parametrize("ctx,m,h,kv,d,group,page", INT4)
def test_int4_attention(backend, f, ctx, m, h, kv, d, group, page):
    s = int4_state(ctx, m, h, kv, d, group, page, f, seed=d + m)
    out = call_int4(backend, s, m, h, kv, d, group, page, f)
    check_int4_attention(out, s, m, page, f, d)


@pytest.mark.parametrize("f", [BF16, F16])
def test_int4_many_sequences(backend, f):
    rng = np.random.default_rng(5)
    ctx = rng.integers(0, 120, 300).tolist()
    s = int4_state(ctx, 1, 2, 1, 64, 32, 16, f)
    check_int4_attention(call_int4(backend, s, 1, 2, 1, 64, 32, 16, f), s, 1, 16, f, 64)


def test_int4_contexts_past_the_bound_are_cut(backend):
    s = int4_state([700, 90], 1, 4, 2, 128, 64, 16, BF16)
    out = call_int4(backend, s, 1, 4, 2, 128, 64, 16, BF16, max_context=333)
    check_int4_attention(out, s, 1, 16, BF16, 128, max_context=333)
    s["ctx"][1] = -7
    out = call_int4(backend, s, 1, 4, 2, 128, 64, 16, BF16, max_context=333)
    assert (out[1] == 0).all()


def test_int4_bad_pages_are_hidden(backend):
    for page in (16, 6):
        s = int4_state([200, 64], 2, 4, 2, 128, 32, page, BF16)
        s["table"][:, 1], s["table"][0, 4] = s["pages"], -9
        out = call_int4(backend, s, 2, 4, 2, 128, 32, page, BF16)
        s["ctx"] = s["ctx"][:1]
        check_int4_attention(out, s, 2, page, BF16, 128, bad_pages=(1, 4))
    s = int4_state([50], 1, 2, 1, 64, 64, 16, F16)
    s["table"][:] = -1
    assert (call_int4(backend, s, 1, 2, 1, 64, 64, 16, F16) == 0).all()


@pytest.mark.parametrize("d,group,page,m", [(128, 64, 16, 1), (64, 32, 5, 1), (128, 32, 16, 3), (256, 128, 64, 1)])
def test_int4_hidden_pairs_have_no_effect(backend, d, group, page, m):
    """NaN and infinite scales and offsets behind the context, and in tokens that a query may not see."""
    ctx = [70, 33]
    s = int4_state(ctx, m, 4, 2, d, group, page, BF16, seed=2)
    clean = call_int4(backend, s, m, 4, 2, d, group, page, BF16).cpu()
    for b, n in enumerate(ctx):
        for t in range(n, -(-n // page) * page):
            for x in "kv":
                s[x + "p"][s["table"][b, t // page].long(), t % page] = float("nan")
    spare = sorted(set(range(s["pages"])) - set(s["table"].flatten().tolist()))
    for x in "kv":
        s[x + "p"][spare] = float("inf")
    assert torch.equal(call_int4(backend, s, m, 4, 2, d, group, page, BF16).cpu(), clean)
    # the last token's pair: only the last query sees it
    for x in "kv":
        s[x + "p"][s["table"][0, 69 // page].long(), 69 % page] = float("nan")
    out = call_int4(backend, s, m, 4, 2, d, group, page, BF16).cpu()
    assert torch.equal(out[0, :m - 1], clean[0, :m - 1]) and out[0, m - 1].isnan().all() and torch.equal(out[1], clean[1])


def test_int4_outputs_repeat(backend):
    s = int4_state([3000, 900, 1], 1, 8, 2, 128, 64, 16, BF16)
    one = call_int4(backend, s, 1, 8, 2, 128, 64, 16, BF16)
    for _ in range(3):
        assert torch.equal(call_int4(backend, s, 1, 8, 2, 128, 64, 16, BF16), one)


# ---------------------------------------------------------------- together --
@pytest.mark.parametrize("f", [BF16, F16])
@pytest.mark.parametrize("group", [32, 128])
def test_a_prompt_then_tokens_over_a_4_bit_cache(backend, f, group):
    """Prompts of three lengths: appended to 4-bit pages and attended packed; then tokens one at a
    time through append and attention, against float64 over the values that the pages hold."""
    h, kv, d, page = 4, 2, 128, 16
    lens = [37, 5, 80]
    steps = 3
    pages_of = [-(-(n + steps) // page) for n in lens]
    pages = sum(pages_of)
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int()
    table = torch.zeros((3, max(pages_of)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages_of):
        table[b, :n] = perm[at:at + n]
        at += n
    codes = [torch.zeros((pages, page, kv, d // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    pairs = [torch.zeros((pages, page, kv, d // group, 2), dtype=torch.float16, device="cuda") for _ in range(2)]
    cfg = puter_amd.RoPEConfig(Mode=1)

    def append(rows, seqs, pos, seed):
        x = randn(seed, (rows, h + 2 * kv, d), f).cuda()
        qout = torch.empty((rows, h, d), dtype=T[f], device="cuda")
        seqs, pos = torch.tensor(seqs), torch.tensor(pos)
        ids = table[seqs, pos // page].cuda()
        backend.KVPageAppendRoPE(cfg, x[:, :h], x[:, h:h + kv], x[:, h + kv:], pos.int().cuda(), ids, (pos % page).int().cuda(),
                                 qout, codes[0], codes[1], pairs[0], pairs[1], rows, h, kv, d, x.stride(0), x.stride(0), x.stride(0),
                                 pages, page, group, f, I4)
        return x, qout

    def values(b, n):
        ids = table[b, :-(-n // page)].long()
        return [int4_values(codes[i].cpu()[ids], pairs[i].cpu()[ids]).flatten(0, 1)[:n] for i in range(2)]

    total = sum(lens)
    seqs = [b for b, n in enumerate(lens) for _ in range(n)]
    pos = [i for n in lens for i in range(n)]
    x, q = append(total, seqs, pos, 3)
    off = torch.tensor(np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32).cuda()
    # the prompts attend to what the pages hold: gathered back as values, 16-bit
    k, v = (torch.empty((total, kv, d), dtype=T[f], device="cuda") for _ in range(2))
    rows = 0
    for b, n in enumerate(lens):
        for i, dst in enumerate((k, v)):
            backend.KVPageGatherInt4(codes[i], pairs[i], table[b].cuda(), dst[rows:], pages, page, kv, d, group, n, f)
        rows += n
    out = torch.empty((total, h, d), dtype=T[f], device="cuda")
    call_packed(backend, q, k, v, out, off, None, h, kv, d, f)
    backend.CheckStatus()
    rows = 0
    for b, n in enumerate(lens):
        ref, mag, top = attend(q[rows:rows + n].cpu().double(), k[rows:rows + n].cpu().double(), v[rows:rows + n].cpu().double(), 0)
        within(out[rows:rows + n], ref, attention_bound(f, ref, mag, top, d, n, p_bits(f)), f"prompt {b}")
        want = values(b, n)
        for got, w in zip((k, v), want):
            within(got[rows:rows + n], w, H(f) * w.abs() + 4 * U * w.abs().max() + tiny(f), f"values {b}")
        rows += n
    ws = torch.empty(backend.PagedInt4WorkspaceBytes(3, 1, h, kv, d, 100), dtype=torch.uint8, device="cuda")
    for step in range(steps):
        ctx = [n + step + 1 for n in lens]
        x, q = append(3, [0, 1, 2], [c - 1 for c in ctx], 50 + step)
        o = torch.empty((3, 1, h, d), dtype=T[f], device="cuda")
        backend.PagedInt4Attention(q, codes[0], codes[1], pairs[0], pairs[1], table.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(),
                                   3, 1, table.shape[1], page, pages, h, kv, d, group, min(100, table.shape[1] * page), f, o, ws, ws.numel())
        backend.CheckStatus()
        s = {"ctx": torch.tensor(ctx), "table": table, "q": q.cpu().view(3, 1, h, d), "kc": codes[0].cpu(), "vc": codes[1].cpu(),
             "kp": pairs[0].cpu(), "vp": pairs[1].cpu()}
        check_int4_attention(o, s, 1, page, f, d)


def test_decode_step_in_a_graph(backend, no_collection):
    """Append and 4-bit attention captured on a stream of their own and replayed with other
    positions, slots and lengths, eager calls between the replays."""
    h, kv, d, page, group, b, f = 8, 2, 128, 16, 64, 4, BF16
    pages, maxc = 40, 160
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).int().view(b, 10).cuda()
    codes = [torch.randint(0, 256, (pages, page, kv, d // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
    pairs = [(torch.rand((pages, page, kv, d // group, 2), device="cuda") * 0.2 + 0.1).half() for _ in range(2)]
    x = torch.zeros((b, h + 2 * kv, d), dtype=T[f], device="cuda")
    pos, ids, slots, ctx = (torch.zeros(b, dtype=torch.int32, device="cuda") for _ in range(4))
    q, o = torch.empty((b, h, d), dtype=T[f], device="cuda"), torch.empty((b, h, d), dtype=T[f], device="cuda")
    ws = torch.empty(backend.PagedInt4WorkspaceBytes(b, 1, h, kv, d, maxc), dtype=torch.uint8, device="cuda")

    def step():
        backend.KVPageAppendRoPE(puter_amd.RoPEConfig(Mode=1), x, x[:, h:], x[:, h + kv:], pos, ids, slots, q, codes[0], codes[1],
                                 pairs[0], pairs[1], b, h, kv, d, x.stride(0), x.stride(0), x.stride(0), pages, page, group, f, I4)
        backend.PagedInt4Attention(q, codes[0], codes[1], pairs[0], pairs[1], table, ctx, b, 1, 10, page, pages, h, kv, d, group, maxc,
                                   f, o, ws, ws.numel())

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        lens = torch.randint(1, maxc, (b,), generator=g, dtype=torch.int32)
        x.copy_(randn(seed, (b, h + 2 * kv, d), f).cuda())
        pos.copy_((lens - 1).cuda())
        ctx.copy_(lens.cuda())
        ids.copy_(table[torch.arange(b), ((lens - 1) // page).long()])
        slots.copy_(((lens - 1) % page).cuda())

    side = torch.cuda.Stream()
    inputs(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    start = [t.clone() for t in codes + pairs]
    for seed in range(1, 5):
        inputs(seed)
        for t, c in zip(codes + pairs, start):
            t.copy_(c)
        torch.cuda.synchronize()
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in [o, q] + codes + pairs]
        for t, c in zip(codes + pairs, start):
            t.copy_(c)
        o.zero_()
        q.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip([o, q] + codes + pairs, want))
    backend.CheckStatus()


def test_packed_in_a_graph(backend, no_collection):
    """Captured once, replayed with other lengths of the same total."""
    h, kv, d, f = 4, 2, 128, BF16
    q, k, v = (randn(i, (300, n, d), f).cuda() for i, n in enumerate((h, kv, kv)))
    off = torch.tensor([0, 100, 200, 300], dtype=torch.int32).cuda()
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call_packed(backend, q, k, v, out, off, None, h, kv, d, f)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call_packed(backend, q, k, v, out, off, None, h, kv, d, f)
    for lens in ([100, 100, 100], [1, 298, 1], [0, 0, 300], [129, 128, 43]):
        off.copy_(torch.tensor(np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32))
        call_packed(backend, q, k, v, out, off, None, h, kv, d, f)
        torch.cuda.synchronize()
        want = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), lens
        refs = packed_refs(q.cpu(), k.cpu(), v.cpu(), lens, lens)
        ref, mag = (torch.cat([r[i] for r in refs]) for i in (0, 1))
        within(out, ref, attention_bound(f, ref, mag, max(r[2] for r in refs), d, 300, p_bits(f)))


def test_packed_f32_split_and_in_a_graph(backend, no_collection):
    """f32's key splits (eager calls on streams of their own, one after another on one scratch) and the
    unsplit kernel (in a graph): each within the bound, eager calls equal to each other."""
    h, kv, d, f = 4, 2, 64, F32
    q, k, v = (randn(70 + i, (700, n, d), f).cuda() for i, n in enumerate((h, kv, kv)))
    off = torch.tensor([0, 100, 200, 700], dtype=torch.int32).cuda()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.zeros_like(q) for _ in streams]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    replayed = torch.zeros_like(q)
    with torch.cuda.graph(graph, stream=streams[0]):
        call_packed(backend, q, k, v, replayed, off, None, h, kv, d, f)
    for lens in ([100, 100, 500], [1, 698, 1], [0, 0, 700], [129, 128, 300]):
        off.copy_(torch.tensor(np.concatenate(([0], np.cumsum(lens))), dtype=torch.int32))
        for t in outs + [replayed]:
            t.fill_(8.0)
        torch.cuda.synchronize()
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                call_packed(backend, q, k, v, o, off, None, h, kv, d, f)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        n = sum(lens)
        refs = packed_refs(q.cpu()[:n], k.cpu()[:n], v.cpu()[:n], lens, lens)
        ref, mag = (torch.cat([r[i] for r in refs]) for i in (0, 1))
        bound = attention_bound(f, ref, mag, max(r[2] for r in refs), d, 700, p_bits(f))
        for o in outs[:1] + [replayed]:
            within(o[:n], ref, bound, lens)
            assert (o[n:] == 8.0).all()
        assert all(torch.equal(o, outs[0]) for o in outs)


def test_two_streams_at_once(backend):
    """Two calls of each operator in flight on different streams, each with its own buffers."""
    s = [int4_state([900, 70], 1, 8, 2, 128, 64, 16, BF16, seed=i) for i in (1, 2)]
    want = [call_int4(backend, x, 1, 8, 2, 128, 64, 16, BF16) for x in s]
    dev = [{n: x[n].cuda() for n in ("q", "kc", "vc", "kp", "vp", "table", "ctx")} for x in s]
    need = backend.PagedInt4WorkspaceBytes(2, 1, 8, 2, 128, 900)
    ws, outs = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in s], [torch.zeros_like(w) for w in want]
    p = [packed_state([200, 50], [200, 50], 4, 2, 128, BF16, seed=i) for i in (3, 4)]
    pd = [(q.cuda(), k.cuda(), v.cuda(), off[0].cuda()) for q, k, v, off in p]
    po = [torch.zeros_like(x[0]) for x in pd]
    pw = []
    for q, k, v, off in pd:
        o = torch.zeros_like(q)
        call_packed(backend, q, k, v, o, off, None, 4, 2, 128, BF16)
        pw.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in s]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                x = dev[i]
                backend.PagedInt4Attention(x["q"], x["kc"], x["vc"], x["kp"], x["vp"], x["table"], x["ctx"], 2, 1, x["table"].shape[1], 16,
                                           s[i]["pages"], 8, 2, 128, 64, 900, BF16, outs[i], ws[i], need)
                q, k, v, off = pd[i]
                call_packed(backend, q, k, v, po[i], off, None, 4, 2, 128, BF16)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs + po, want + pw))
