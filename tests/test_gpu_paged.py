"""Paged key-value caches on the GPU against the float64 oracle (oracle/paged.py).

Tolerances.  Copies are exact.  Of attention, with a[k] = scale * sum_i |q_i k_i| and mag = sum_k p[k] |v[k]|:
products of 16-bit values are exact in float32, so a score is off by at most (D + 4) 2^-24 a (D roundings of the sum, those of
the scale, of the maximum's difference and of the exponent), and exp2 by 2^-22; a weight therefore by a factor within
d = 2 max_k (D + 4) 2^-24 a[k] + 2^-21 (its own and the sum's).  Weights enter the 16-bit product as two 16-bit parts: 2^-17 more
for bfloat16, for float16 2^-21 and at most 2^-25 for each key where parts are subnormal (the sum of weights is at least
1).  Adding n terms in float32 costs n 2^-24.  So |o - ref| <= (d + 2^-17 + n 2^-24) mag + n 2^-25 max |v| (float16), and the
output's rounding, half a step: eps / 2 |ref| (and 2^-25 where float16 is subnormal).
Accumulated weights: G (d + n 2^-24) of the added weight, and 2^-23 of the sum."""
import math

import pytest
import torch

from conftest import load_mod
from oracle import paged as oracle

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
BITS = {1: torch.uint8, 2: torch.int16, 4: torch.int32}


def bits(x):
    return x.contiguous().view(BITS[x.element_size()])


def same(a, b, what=""):
    assert a.shape == b.shape and a.dtype == b.dtype
    assert torch.equal(bits(a.cpu()), bits(b.cpu())), what


def pool(g, shape, dtype, layout, fill):
    """A pool on the CPU; `fill`: what lies where nothing has been written."""
    P, H, S, D = shape
    x = torch.randn(shape, generator=g)
    if dtype == "fp8":
        x = (x * 60).clamp(-448, 448)
    x = x.to(DT[dtype])
    if layout == "nhd":
        x = x.transpose(1, 2).contiguous().transpose(1, 2)
    return x


def on_gpu(x, dev):
    """x on the GPU with its strides."""
    if x.dim() == 4 and not x.is_contiguous():
        return x.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    return x.to(dev)


def make(seed, dtype, cache, D, Hq, Hkv, page, layout, lens, extra=0, nan=True):
    """Pages in no order; what no sequence's tokens cover is NaN."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    width = max(1, -(-max(lens) // page)) + extra
    used = [-(-n // page) for n in lens]
    P = sum(used) + 3
    order = torch.randperm(P, generator=g).tolist()
    table = torch.full((B, width), -1, dtype=torch.int32)
    kp, vp = (pool(g, (P, Hkv, page, D), cache, layout, nan) for _ in range(2))
    held = torch.zeros(P, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        for i in range(used[b]):
            table[b, i] = order[at]
            held[order[at], :min(page, n - i * page)] = True
            at += 1
    if nan:
        for x in (kp, vp):
            bits_ = x.view(BITS[x.element_size()]) if x.is_contiguous() else x.transpose(1, 2).view(BITS[x.element_size()]).transpose(1, 2)
            code = {1: 0x7f, 2: 0x7fff, 4: 0x7fffffff}[x.element_size()]
            bits_[(~held)[:, None, :].expand(P, Hkv, page)] = code
    q = torch.randn(B, Hq, D, generator=g).to(DT[dtype]) * 1.5
    sinks = torch.randn(Hq, generator=g)
    return dict(g=g, table=table, lens=torch.tensor(lens, dtype=torch.int32), kp=kp, vp=vp, q=q, sinks=sinks,
                descale=(0.013, 0.021) if cache == "fp8" else (1.0, 1.0), order=order, used=sum(used))


def check_attention(o, c, ref, mag, dtype, D, n, scale, window=None, sink=0):
    B, Hq = c["q"].shape[:2]
    H, S = c["kp"].shape[1:3]
    eps = torch.finfo(DT[dtype]).eps
    for b in range(B):
        pos = [k for k in range(int(c["lens"][b])) if window is None or int(c["lens"][b]) - 1 - k < window or k < sink]
        k, ok = oracle.gather(c["kp"], c["table"], b, pos)
        v, _ = oracle.gather(c["vp"], c["table"], b, pos)
        k, v = k[ok] * c["descale"][0], v[ok] * c["descale"][1]
        for h in range(Hq):
            kh, vh = k[:, h // (Hq // H)], v[:, h // (Hq // H)]
            m = len(kh)
            a = abs(scale) * float((kh.abs() @ c["q"][b, h].double().abs()).max()) if m else 0.0
            d = 2 * (D + 4) * 2.0 ** -24 * a + 2.0 ** -21
            tol = (d + 2.0 ** -17 + m * 2.0 ** -24) * mag[b, h] + eps / 2 * ref[b, h].abs()
            if dtype == "fp16":
                tol = tol + m * 2.0 ** -25 * (float(vh.abs().max()) if m else 0.0) + 2.0 ** -25
            err = (o[b, h].double().cpu() - ref[b, h]).abs()
            assert bool((err <= tol).all()), (b, h, m, float(err.max()), float((err - tol).max()))


ATTEND = [
    # dtype, cache, D, Hq, Hkv, page, layout, lens, window, sink, learned
    ("bf16", "bf16", 64, 8, 1, 16, "hnd", (1, 31, 32, 33, 127, 129, 0, 500), None, 0, True),
    ("bf16", "bf16", 64, 16, 2, 16, "nhd", (513, 1, 1200, 0, 640, 128), None, 0, True),
    ("bf16", "bf16", 64, 8, 2, 7, "hnd", (5, 7, 8, 700, 1033), None, 0, False),
    ("bf16", "bf16", 64, 8, 1, 16, "hnd", (900, 127, 128, 129, 1, 300), 128, 0, True),
    ("bf16", "bf16", 64, 8, 1, 64, "nhd", (900, 133, 3, 131, 132, 300), 128, 4, False),
    ("bf16", "bf16", 64, 8, 1, 16, "hnd", (900, 1500, 3, 0, 700), 600, 33, True),
    ("bf16", "bf16", 64, 8, 1, 16, "hnd", (900, 4, 3, 0), 0, 5, False),
    ("bf16", "bf16", 128, 8, 2, 32, "nhd", (1, 64, 999, 0, 555), None, 0, False),
    ("bf16", "bf16", 32, 6, 2, 16, "hnd", (70, 1, 800), None, 0, True),
    ("bf16", "bf16", 16, 5, 1, 16, "nhd", (70, 1, 800), 100, 2, False),
    ("bf16", "bf16", 64, 33, 1, 16, "hnd", (70, 1, 800), None, 0, True),
    ("bf16", "bf16", 64, 64, 1, 16, "nhd", (1100, 1, 0, 700), None, 0, True),
    ("bf16", "bf16", 128, 40, 1, 16, "hnd", (1100, 5), None, 0, False),
    ("fp16", "fp8", 128, 34, 1, 16, "hnd", (1030, 5), None, 0, True),
    ("bf16", "bf16", 64, 8, 2, 16, "hnd", (1025, 2000, 31, 0, 1500), None, 0, False),
    ("bf16", "bf16", 128, 4, 2, 16, "nhd", (1500, 2, 1024), 1200, 7, True),
    ("fp16", "fp16", 64, 8, 8, 16, "hnd", (70, 1, 800, 129), None, 0, False),
    ("fp16", "fp16", 16, 4, 1, 1, "hnd", (70, 1, 600), None, 0, False),
    ("fp16", "fp16", 128, 20, 1, 256, "hnd", (300, 1, 600), None, 0, True),
    ("bf16", "fp8", 64, 8, 1, 16, "hnd", (70, 1, 800, 0), None, 0, True),
    ("fp16", "fp8", 64, 8, 2, 16, "nhd", (70, 129, 300), 64, 4, False),
    ("bf16", "fp8", 128, 8, 2, 24, "hnd", (70, 33, 777), None, 0, False),
    ("fp16", "fp8", 128, 4, 1, 16, "nhd", (700, 33), None, 0, True),
    ("fp32", "fp32", 16, 4, 4, 16, "hnd", (70, 1, 700, 0), 256, 4, False),
    ("fp32", "fp32", 32, 4, 1, 16, "nhd", (70, 1, 700, 0), None, 0, True),
    ("fp32", "fp32", 64, 8, 1, 16, "hnd", (70, 33, 700), None, 0, False),
    ("fp32", "fp32", 128, 18, 1, 20, "hnd", (70, 32, 700), None, 0, True),
]


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(str(x) for x in c[:7]) + f"-W{c[8]}-S{c[9]}")
@pytest.mark.parametrize("sums", [False, True])
def test_attention(fa, gpu, case, sums):
    dtype, cache, D, Hq, Hkv, page, layout, lens, W, S, learned = case
    c = make(ATTEND.index(case), dtype, cache, D, Hq, Hkv, page, layout, lens)
    print(case, sums, flush=True)
    w0 = torch.rand(len(lens), Hkv, c["table"].shape[1] * page, generator=c["g"]) if sums else None
    sinks = c["sinks"] if learned else None
    ref, mag, ref_sums = oracle.attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], W, S, sinks, descale=c["descale"], sums=w0)
    w = w0.to(gpu) if sums else None
    o = fa.paged_attention(c["q"].to(gpu), on_gpu(c["kp"], gpu), on_gpu(c["vp"], gpu), c["table"].to(gpu), c["lens"].to(gpu), W, S,
                           None if sinks is None else sinks.to(gpu), descale=c["descale"], weight_sums=w)
    assert o.dtype == DT[dtype] and o.shape == c["q"].shape
    check_attention(o, c, ref, mag, dtype, D, max(lens), 1 / math.sqrt(D), W, S)
    if sums:
        G = Hq // Hkv
        a = max(float(x) for x in (c["q"].double().abs().sum(-1).max(),)) * 8 * (1 if cache != "fp8" else 448 * c["descale"][0])
        d = 2 * (D + 4) * 2.0 ** -24 * a / math.sqrt(D) + 2.0 ** -21
        add = ref_sums - w0.double()
        tol = (d + max(lens) * 2.0 ** -24) * add + 2.0 ** -23 * ref_sums.abs()
        err = (w.double().cpu() - ref_sums).abs()
        assert bool((err <= tol).all()), float((err - tol).max())
        assert torch.equal(w.cpu()[add == 0], w0[add == 0])  # keys that nobody sees keep their sums


@pytest.mark.parametrize("B,Hq,Hkv,D,cache,W", [(520, 4, 2, 64, "bf16", 128), (600, 2, 2, 16, "fp16", 33), (513, 2, 2, 64, "fp8", 40),
                                                (140, 4, 2, 64, "bf16", 150), (90, 3, 3, 128, "bf16", None), (64, 2, 2, 64, "bf16", None),
                                                (70, 2, 2, 64, "bf16", None), (70, 4, 4, 128, "fp8", None)])
def test_many_short_sequences(fa, gpu, B, Hq, Hkv, D, cache, W):
    """Batches large enough for a wave, or a workgroup of four, a sequence."""
    dtype = "fp16" if cache == "fp16" else "bf16"
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 260, (B,), generator=g).tolist()
    c = make(B, dtype, cache, D, Hq, Hkv, 16, "hnd", lens, extra={64: 100, 70: 150}.get(B, 0))
    ref, mag, _ = oracle.attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], W, 3 if W else 0, c["sinks"], descale=c["descale"])
    o = fa.paged_attention(c["q"].to(gpu), c["kp"].to(gpu), c["vp"].to(gpu), c["table"].to(gpu), c["lens"].to(gpu), W, 3 if W else 0,
                           c["sinks"].to(gpu), descale=c["descale"])
    check_attention(o, c, ref, mag, dtype, D, 260, 1 / math.sqrt(D), W, 3 if W else 0)


@pytest.mark.parametrize("lens", [[300001, 70000, 140000], [610001, 200000]])
def test_large_cache(fa, gpu, lens):
    """260 and 415 MB of K and V, so that loads are marked as read once and more workgroups used, in two layouts, with weights."""
    B, Hq, Hkv, D, page = len(lens), 16, 2, 64, 64
    g = torch.Generator(device=gpu).manual_seed(5)
    used = [-(-n // page) for n in lens]
    P = sum(used)
    order = torch.randperm(P, generator=g, device=gpu).to(torch.int32)
    table = torch.full((B, max(used)), -1, dtype=torch.int32, device=gpu)
    for b in range(B):
        table[b, :used[b]] = order[sum(used[:b]):sum(used[:b + 1])]
    q = torch.randn(B, Hq, D, generator=g, device=gpu).to(torch.bfloat16) * 2
    tl = torch.tensor(lens, dtype=torch.int32, device=gpu)
    for layout in ("hnd", "nhd"):
        shape = (P, Hkv, page, D) if layout == "hnd" else (P, page, Hkv, D)
        kp, vp = (torch.randn(shape, generator=g, device=gpu).to(torch.bfloat16) for _ in range(2))
        if layout == "nhd":
            kp, vp = kp.transpose(1, 2), vp.transpose(1, 2)
        sums = torch.zeros(B, Hkv, max(used) * page, device=gpu)
        o = fa.paged_attention(q, kp, vp, table, tl, weight_sums=sums)
        for b, n in enumerate(lens):
            at = table[b, :used[b]].long()
            for h in range(Hkv):
                k, v = (x[at, h].reshape(-1, D)[:n].double() for x in (kp, vp))
                p = torch.softmax(q[b, 8 * h:8 * h + 8].double() @ k.t() / 8, -1)
                ref, mag = p @ v, p @ v.abs()
                a = float((q[b, 8 * h:8 * h + 8].double().abs() @ k.abs().t()).max()) / 8
                d = 2 * (D + 4) * 2.0 ** -24 * a + 2.0 ** -21
                tol = (d + 2.0 ** -17 + n * 2.0 ** -24) * mag + 2.0 ** -8 * ref.abs()
                err = (o[b, 8 * h:8 * h + 8].double() - ref).abs()
                assert bool((err <= tol).all()), (layout, b, h, float((err - tol).max()))
                w = p.sum(0)
                assert bool(((sums[b, h, :n].double() - w).abs() <= (d + n * 2.0 ** -24) * w + 2.0 ** -23 * w).all())
            assert not sums[b, :, n:].any()


def test_offsets_past_32_bits(fa, gpu):
    """Pages 4 GiB apart: a pool of all layers, of which this is one layer's view."""
    P, Hkv, page, D = 3, 2, 16, 64
    step = 2 ** 31  # elements
    pools = [torch.empty(2 * step + Hkv * page * D, dtype=torch.bfloat16, device=gpu).as_strided((P, Hkv, page, D), (step, page * D, D, 1))
             for _ in range(2)]
    small = [torch.randn(P, Hkv, page, D, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16) for i in range(2)]
    for x, y in zip(pools, small):
        x.copy_(y)
    table = torch.tensor([[2, 1]], dtype=torch.int32)
    lens = torch.tensor([21], dtype=torch.int32)
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(1, Hkv, D, generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(1, 4, D, generator=g).to(torch.bfloat16)
    fa.paged_append(k.to(gpu), v.to(gpu), *pools, table.to(gpu), lens.to(gpu))
    small = oracle.append(k, v, *small, table, lens)
    o = fa.paged_attention(q.to(gpu), *pools, table.to(gpu), lens.to(gpu))
    ref, mag, _ = oracle.attention(q, *small, table, lens)
    check_attention(o, dict(q=q, kp=small[0], vp=small[1], table=table, lens=lens, descale=(1, 1)), ref, mag, "bf16", D, 21, 0.125)
    sums = torch.rand(1, Hkv, 32, generator=g)
    new_table = torch.tensor([[0]], dtype=torch.int32)
    want = oracle.evict(*small, table, lens, sums, 12, new_table, 1, 2)
    left, new = fa.paged_evict(*pools, table.to(gpu), lens.to(gpu), sums.to(gpu), 12, new_table.to(gpu), 1, 2)
    same(new, want[3])
    same(pools[0].contiguous(), want[0])
    same(pools[1].contiguous(), want[1])


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_attention_scale(fa, gpu, scale):
    c = make(3, "bf16", "bf16", 64, 8, 2, 16, "hnd", (70, 600))
    ref, mag, _ = oracle.attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], scale=scale)
    o = fa.paged_attention(c["q"].to(gpu), c["kp"].to(gpu), c["vp"].to(gpu), c["table"].to(gpu), c["lens"].to(gpu), scale=scale)
    check_attention(o, c, ref, mag, "bf16", 64, 600, scale)


def test_masked_places_hold_anything(fa, gpu):
    """Keys and values outside the window and the sinks: infinities and NaN; the result is as without them."""
    c = make(4, "bf16", "bf16", 64, 8, 1, 16, "hnd", (300, 900, 40))
    args = lambda: (c["q"].to(gpu), c["kp"].to(gpu), c["vp"].to(gpu), c["table"].to(gpu), c["lens"].to(gpu), 128, 3)
    o = fa.paged_attention(*args())
    for b, n in enumerate((300, 900, 40)):
        for pos in range(3, n - 128):
            p, s = oracle.entry(c["table"], b, pos, 16, c["kp"].shape[0])
            c["kp"][p, :, s] = [math.nan, math.inf, -math.inf, 3e38][pos % 4]
            c["vp"][p, :, s] = [math.inf, math.nan, 3e38, -math.inf][pos % 4]
    same(fa.paged_attention(*args()), o)


def test_entries_that_are_no_page(fa, gpu):
    """Table entries outside [0, pages) are masked for reading and left out for writing, wherever they stand."""
    c = make(5, "bf16", "bf16", 64, 8, 2, 16, "nhd", (300, 900, 40, 64))
    P = c["kp"].shape[0]
    c["table"][0, 3], c["table"][1, 40], c["table"][1, 0], c["table"][2, 2] = -1, P, 2 ** 31 - 1, -2 ** 31
    c["table"][3, :4] = P + 7  # nothing to see at all
    ref, mag, _ = oracle.attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], sinks=c["sinks"])
    assert not ref[3].any()
    o = fa.paged_attention(c["q"].to(gpu), on_gpu(c["kp"], gpu), on_gpu(c["vp"], gpu), c["table"].to(gpu), c["lens"].to(gpu),
                           sinks=c["sinks"].to(gpu))
    check_attention(o, c, ref, mag, "bf16", 64, 900, 0.125)
    g = c["g"]
    k, v = (torch.randn(4, 2, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    c["table"][0, 18] = -5
    want = oracle.append(k, v, c["kp"], c["vp"], c["table"], c["lens"])
    kp, vp = on_gpu(c["kp"], gpu), on_gpu(c["vp"], gpu)
    fa.paged_append(k.to(gpu), v.to(gpu), kp, vp, c["table"].to(gpu), c["lens"].to(gpu))
    same(kp, want[0])
    same(vp, want[1])


def test_lens_outside_the_table(fa, gpu):
    """Lengths below 0 count as 0 and are cut off at the table's tokens and at max_seqlen."""
    c = make(6, "bf16", "bf16", 64, 8, 1, 16, "hnd", (600, 600, 600))
    t = lambda lens: torch.tensor(lens, dtype=torch.int32, device=gpu)
    run = lambda lens, **kw: fa.paged_attention(c["q"].to(gpu), c["kp"].to(gpu), c["vp"].to(gpu), c["table"].to(gpu), t(lens), **kw)
    vis = 38 * 16  # the table's tokens; the last page's rest is NaN, so look at 600 by max_seqlen
    same(run((-7, 2 ** 31 - 1, 601), max_seqlen=600), run((0, 600, 600), max_seqlen=600))
    assert vis == 608 and not run((-7, 5, 600))[0].any()
    o = run((3, 600, 599))
    same(o, run((3, 600, 599), max_seqlen=600))


APPEND = [
    # dtype, cache, D, Hkv, page, layout, lens (new rows included), new (None: one each)
    ("bf16", "bf16", 64, 8, 16, "hnd", (1, 16, 17, 0, 33), None),
    ("bf16", "bf16", 64, 2, 16, "nhd", (40, 16, 17, 3, 100), (40, 1, 0, 2, 77)),
    ("fp16", "fp16", 16, 3, 5, "hnd", (40, 16, 17, 3), (40, 16, 17, 3)),
    ("fp32", "fp32", 128, 2, 16, "nhd", (40, 16, 1), (9, 16, 1)),
    ("fp32", "fp32", 16, 1, 16, "hnd", (40, 16, 1), None),
    ("bf16", "bf16", 128, 4, 64, "hnd", (200, 64, 1), (129, 64, 1)),
    ("fp16", "fp16", 32, 4, 64, "hnd", (200, 64, 1), (129, 64, 1)),
    ("bf16", "fp8", 64, 8, 16, "hnd", (1, 16, 17, 0, 33), None),
    ("fp16", "fp8", 64, 2, 16, "nhd", (40, 16, 17), (40, 1, 3)),
    ("bf16", "fp8", 128, 3, 24, "nhd", (40, 16, 17), (40, 1, 3)),
    ("fp16", "fp8", 128, 1, 16, "hnd", (40, 16, 17), (40, 1, 3)),
    ("bf16", "bf16", 64, 1, 16, "hnd", tuple(range(1, 131)), tuple(1 + i // 2 for i in range(130))),
]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(str(x) for x in c[:6]) + f"-{len(c[6])}")
def test_append(fa, gpu, case):
    dtype, cache, D, Hkv, page, layout, lens, new = case
    print(case, flush=True)
    c = make(11, dtype, cache, D, Hkv, Hkv, page, layout, lens)
    n = [1] * len(lens) if new is None else list(new)
    cu = None if new is None else torch.tensor([0] + n).cumsum(0)
    k, v = ((torch.randn(sum(n), Hkv, D, generator=c["g"]) * 4).to(DT[dtype]) for _ in range(2))
    if cache == "fp8":  # values past the largest code, on borders between codes, and what has no code
        edge = torch.tensor([math.inf, -math.inf, math.nan, -math.nan, 0.0, -0.0, 1e4, -1e4, 6.5, 8.5 * 0.013]).to(DT[dtype])
        k.view(-1)[:10] = edge
        v.view(-1)[-10:] = edge
    want = oracle.append(k, v, c["kp"], c["vp"], c["table"], c["lens"], cu, c["descale"])
    for where in ("host", "device"):
        kp, vp = on_gpu(c["kp"], gpu), on_gpu(c["vp"], gpu)
        off = None if cu is None else (cu if where == "host" else cu.to(gpu, torch.int32))
        # K as a slice of a fused projection's rows
        fused = torch.cat((k, v), 1).to(gpu)
        fa.paged_append(fused[:, :Hkv], fused[:, Hkv:], kp, vp, c["table"].to(gpu), c["lens"].to(gpu), cu_seqlens=off, descale=c["descale"])
        if cache == "fp8":  # (the sign of a NaN's code is the product's)
            same_codes(kp, want[0])
            same_codes(vp, want[1])
        else:
            same(kp, want[0])
            same(vp, want[1])


def same_codes(a, b):
    x, y = a.cpu().float(), b.float()
    assert torch.equal(x.isnan(), y.isnan()) and torch.equal(bits(a.cpu())[~x.isnan()], bits(b)[~x.isnan()])


def test_append_rows_of_no_sequence(fa, gpu):
    """Rows before the first offset and behind the last one are left out, and a sequence without room gets what fits."""
    c = make(12, "bf16", "bf16", 64, 2, 2, 16, "hnd", (30, 5, 16))
    k, v = (torch.randn(40, 2, 64, generator=c["g"]).to(torch.bfloat16) for _ in range(2))
    cu = torch.tensor([3, 8, 8, 26], dtype=torch.int32)
    c["lens"] = torch.tensor([3, 5, 35], dtype=torch.int32)  # two rows before position 0; rows past the table
    want = oracle.append(k, v, c["kp"], c["vp"], c["table"], c["lens"], cu)
    kp, vp = c["kp"].to(gpu), c["vp"].to(gpu)
    fa.paged_append(k.to(gpu), v.to(gpu), kp, vp, c["table"].to(gpu), c["lens"].to(gpu), cu_seqlens=cu.to(gpu))
    same(kp, want[0])
    same(vp, want[1])
    fa.paged_append(k[:0].to(gpu), v[:0].to(gpu), kp, vp, c["table"].to(gpu), c["lens"].to(gpu), cu_seqlens=torch.zeros(4, dtype=torch.int32))
    same(kp, want[0])


EVICT = [
    # cache, D, Hkv, page, layout, lens, keep, sink, recent
    ("bf16", 64, 2, 16, "hnd", (100, 64, 63, 65, 0, 1, 300), 64, 4, 16),
    ("bf16", 64, 3, 16, "nhd", (1500, 64, 2000, 65), 130, 0, 0),
    ("fp16", 16, 1, 5, "hnd", (100, 33), 33, 33, 0),
    ("fp32", 128, 2, 16, "nhd", (100, 33), 40, 0, 40),
    ("bf16", 128, 2, 64, "hnd", (5000, 4097, 4096), 1024, 4, 256),
    ("fp8", 64, 2, 16, "hnd", (100, 33), 1, 0, 0),
    ("fp8", 128, 2, 24, "nhd", (1100, 33), 100, 1, 1),
    ("fp32", 16, 1, 16, "hnd", (100, 33), 50, 10, 40),
    # more entries than a workgroup of the selection holds
    ("fp16", 16, 2, 64, "nhd", (40000, 16385, 5, 20000, 16384), 3000, 4, 100),
    ("bf16", 16, 1, 16, "hnd", (40001, 33000), 20000, 17000, 0),
    ("bf16", 16, 1, 16, "hnd", (49153, 32769), 20000, 0, 17000),
    # more (sequence, KV head) than one workgroup each fills the card with
    ("bf16", 16, 24, 16, "nhd", (20001, 16385, 100), 3000, 1, 30),
    ("bf16", 16, 48, 16, "hnd", (20001, 16385, 8193), 3000, 1, 30),
]


def weights(g, kind, shape):
    w = torch.exp(2 * torch.randn(shape, generator=g) - 4)
    if kind == "ties":
        w = torch.randint(0, 4, shape, generator=g).float()
    elif kind == "zero":
        w = torch.zeros(shape)
    elif kind == "odd":  # every kind of number
        w = torch.randn(shape, generator=g) * torch.exp(20 * torch.randn(shape, generator=g))
        pick = torch.randint(0, 12, shape, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42)):
            w = torch.where(pick == i, torch.tensor(x), w)
    return w


@pytest.mark.parametrize("kind", ["weights", "ties", "zero", "odd"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: "-".join(str(x) for x in c[:5]) + f"-{c[6]}-{c[7]}-{c[8]}")
def test_evict(fa, gpu, case, kind):
    cache, D, Hkv, page, layout, lens, keep, sink, recent = case
    print(case, kind, flush=True)
    c = make(21, "bf16", cache, D, Hkv, Hkv, page, layout, lens, nan=False)
    B, P = len(lens), c["kp"].shape[0]
    width = -(-keep // page) + 1
    need = B * width
    more = lambda x: torch.cat((x, x[:1].expand(need, *x.shape[1:])), 0)
    kp, vp = more(bits(c["kp"])).view(c["kp"].dtype), more(bits(c["vp"])).view(c["kp"].dtype)
    new_table = (P + torch.randperm(need, generator=c["g"]).view(B, width)).to(torch.int32)
    sums = weights(c["g"], kind, (B, Hkv, c["table"].shape[1] * page + 3))
    want = oracle.evict(kp, vp, c["table"], c["lens"], sums, keep, new_table, sink, recent)
    gk, gv = (on_gpu(x.transpose(1, 2).contiguous().transpose(1, 2) if layout == "nhd" else x, gpu) for x in (kp, vp))
    gs = sums.to(gpu)
    left, new = fa.paged_evict(gk, gv, c["table"].to(gpu), c["lens"].to(gpu), gs, keep, new_table.to(gpu), sink, recent)
    same(left, want[2])
    same(new, want[3], "sums")
    same(gk, want[0])
    same(gv, want[1])
    same(gs, sums, "the old sums stay")


def test_evict_entries_that_are_no_page(fa, gpu):
    c = make(22, "bf16", "bf16", 64, 2, 2, 16, "hnd", (100, 90), nan=False)
    P = c["kp"].shape[0]
    kp, vp = (torch.cat((x, x[:8])) for x in (c["kp"], c["vp"]))
    new_table = torch.tensor([[P, P + 1, -1], [P + 8, P + 2, P + 3]], dtype=torch.int32)
    c["table"][0, 2] = -1
    sums = torch.rand(2, 2, 112, generator=c["g"])
    want = oracle.evict(kp, vp, c["table"], c["lens"], sums, 48, new_table, 2, 9)
    gk, gv = kp.to(gpu), vp.to(gpu)
    left, new = fa.paged_evict(gk, gv, c["table"].to(gpu), c["lens"].to(gpu), sums.to(gpu), 48, new_table.to(gpu), 2, 9)
    same(new, want[3])
    same(gk, want[0])
    same(gv, want[1])


def test_a_conversation(fa, gpu):
    """Prompts into the cache, decoding with accumulated weights, eviction, more decoding: every step as the oracle has it."""
    dev, Hq, Hkv, D, page, keep = gpu, 8, 2, 64, 16, 40
    g = torch.Generator().manual_seed(31)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)
    prompt = [70, 9, 33]
    cu = torch.tensor([0, 70, 79, 112])
    P, width = 40, 6
    order = torch.randperm(P, generator=g).to(torch.int32)
    table, new_table = order[:18].view(3, 6), order[18:30].view(3, 4)
    kp = torch.zeros(P, Hkv, page, D, dtype=torch.bfloat16)
    vp = kp.clone()
    sums = torch.zeros(3, Hkv, width * page)
    G = dict(kp=kp.to(dev), vp=vp.to(dev), table=table.to(dev), sums=sums.to(dev), lens=torch.tensor(prompt, dtype=torch.int32, device=dev))
    lens = torch.tensor(prompt, dtype=torch.int32)
    k, v, q = r(112, Hkv, D), r(112, Hkv, D), r(112, Hq, D)
    fa.paged_append(k.to(dev), v.to(dev), G["kp"], G["vp"], G["table"], G["lens"], cu_seqlens=cu)
    kp, vp = oracle.append(k, v, kp, vp, table, lens, cu)
    same(G["kp"], kp)
    # the prompt's last row through the prefill kernels and through the cache: the same attention
    full = fa.flash_swda_with_sink_varlen(q.to(dev), k.to(dev), v.to(dev), cu, None, None)
    last = fa.paged_attention(q.to(dev)[cu[1:].to(dev) - 1], G["kp"], G["vp"], G["table"], G["lens"])
    assert float((full[cu[1:].to(dev) - 1].float() - last.float()).abs().max()) < 2.0 ** -6  # (two roundings of values below 4, P in 16 bits)
    sinks = torch.randn(Hq, generator=g)

    def steps(count):
        nonlocal kp, vp, sums, lens
        for _ in range(count):
            k, v, q = r(3, Hkv, D), r(3, Hkv, D), r(3, Hq, D)
            G["lens"] += 1
            lens = lens + 1
            fa.paged_append(k.to(dev), v.to(dev), G["kp"], G["vp"], G["table"], G["lens"])
            kp, vp = oracle.append(k, v, kp, vp, table, lens)
            o = fa.paged_attention(q.to(dev), G["kp"], G["vp"], G["table"], G["lens"], sinks=sinks.to(dev), weight_sums=G["sums"])
            ref, mag, new = oracle.attention(q, kp, vp, table, lens, sinks=sinks, sums=sums)
            check_attention(o, dict(q=q, kp=kp, vp=vp, table=table, lens=lens, descale=(1, 1)), ref, mag, "bf16", D, 96, 0.125)
            assert torch.allclose(G["sums"].cpu().double(), new, atol=1e-4, rtol=1e-4)
            sums = G["sums"].cpu()

    steps(4)
    kp, vp, lens, sums = oracle.evict(kp, vp, table, lens, sums, keep, new_table, 2, 8)
    G["lens"], G["sums"] = fa.paged_evict(G["kp"], G["vp"], G["table"], G["lens"], G["sums"], keep, new_table.to(dev), 2, 8)
    table, G["table"] = new_table, new_table.to(dev)
    same(G["lens"], lens)
    same(G["sums"], sums)
    same(G["kp"], kp)
    steps(4)
    assert lens.tolist() == [44, 17, 41]


def test_captured_step(fa, gpu):
    """A captured step (append, attention with and without weights, eviction), replayed with new inputs between eager calls."""
    def inputs(seed, lens):
        c = make(seed, "bf16", "bf16", 64, 8, 2, 16, "hnd", lens, extra=60, nan=False)
        return c
    c = inputs(41, (700, 300, 900, 0))
    P = c["kp"].shape[0]
    st = {n: c[n].to(gpu) for n in ("q", "table", "lens", "sinks")}
    st["kp"], st["vp"] = (torch.cat((c[n], c[n][:40])).to(gpu) for n in ("kp", "vp"))
    st["k"], st["v"] = (torch.randn(4, 2, 64, generator=c["g"]).to(torch.bfloat16).to(gpu) for _ in range(2))
    st["sums"] = torch.rand(4, 2, c["table"].shape[1] * 16, generator=c["g"]).to(gpu)
    st["new_table"] = (P + torch.arange(40, dtype=torch.int32).view(4, 10)).to(gpu)

    def step(s):
        fa.paged_append(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["lens"])
        a = fa.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], sinks=s["sinks"], weight_sums=s["sums"])
        b = fa.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"], 128)
        left, new = fa.paged_evict(s["kp"], s["vp"], s["table"], s["lens"], s["sums"], 150, s["new_table"], 4, 20)
        return a, b, left, new
    step({n: x.clone() for n, x in st.items()})
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(st)
    first = {n: x.clone() for n, x in st.items()}
    for i, lens in enumerate(((700, 300, 900, 0), (701, 1, 17, 640), (0, 0, 0, 0), (700, 300, 900, 0))):
        other = inputs(50 + i, (700, 300, 900, 0))
        fresh = {n: x.clone() for n, x in first.items()}
        fresh["q"] = other["q"].to(gpu)
        fresh["lens"] = torch.tensor(lens, dtype=torch.int32, device=gpu)
        for n, x in fresh.items():
            st[n].copy_(x)
        want = step(fresh)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            same(x, y, f"replay {i}")
        for n in ("kp", "vp", "sums"):
            same(st[n], fresh[n], f"replay {i} {n}")


def test_two_streams(fa, gpu):
    """Calls on two streams at once give what they give alone."""
    cs = [make(60 + i, "bf16", "bf16", 64, 16, 2, 16, "hnd", (1500, 800, 30 + i)) for i in range(2)]
    st = [{n: c[n].to(gpu) for n in ("q", "kp", "vp", "table", "lens")} for c in cs]
    run = lambda s: fa.paged_attention(s["q"], s["kp"], s["vp"], s["table"], s["lens"])
    want = [run(s) for s in st]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, x in zip(streams, st):
            with torch.cuda.stream(s):
                got.append(run(x))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        same(x, want[i % 2])


@pytest.mark.parametrize("binding", [True, False])
def test_refusals(fa, gpu, monkeypatch, binding):
    ops = load_mod("_ops")
    if not binding:
        monkeypatch.setattr(ops, "_BINDING", None)
    bf = torch.bfloat16
    kp = torch.zeros(6, 2, 16, 64, dtype=bf, device=gpu)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device=gpu), torch.ones(2, dtype=torch.int32, device=gpu)
    x, q = torch.zeros(2, 2, 64, dtype=bf, device=gpu), torch.zeros(2, 4, 64, dtype=bf, device=gpu)
    sums, nt = torch.zeros(2, 2, 48, device=gpu), torch.ones(2, 1, dtype=torch.int32, device=gpu)
    att = lambda **kw: fa.paged_attention(**{**dict(q=q, k_pages=kp, v_pages=kp, block_table=table, lens=lens), **kw})
    app = lambda **kw: fa.paged_append(**{**dict(k=x, v=x, k_pages=kp, v_pages=kp, block_table=table, lens=lens), **kw})
    evi = lambda **kw: fa.paged_evict(**{**dict(k_pages=kp, v_pages=kp, block_table=table, lens=lens, weight_sums=sums, keep=16,
                                               new_table=nt), **kw})
    for f in (att, app, evi):
        for kw, err in ((dict(k_pages=kp[0]), ValueError), (dict(v_pages=kp[:5]), ValueError), (dict(v_pages=kp.half()), ValueError),
                        (dict(k_pages=kp.double(), v_pages=kp.double()), ValueError), (dict(block_table=table.long()), ValueError),
                        (dict(block_table=table[0]), ValueError), (dict(lens=lens.long()), ValueError), (dict(lens=lens[:1]), ValueError),
                        (dict(lens=lens.cpu()), RuntimeError), (dict(block_table=table.cpu()), RuntimeError),
                        (dict(v_pages=kp.cpu()), RuntimeError), (dict(k_pages=kp[..., :48], v_pages=kp[..., :48]), ValueError),
                        (dict(k_pages=kp.transpose(2, 3), v_pages=kp.transpose(2, 3)), ValueError),
                        (dict(k_pages=kp[:0], v_pages=kp[:0]), ValueError)):
            with pytest.raises(err):
                f(**kw)
    odd = torch.zeros(6 * 2 * 16 * 64 + 1, dtype=bf, device=gpu)[1:].view(6, 2, 16, 64)
    for f in (att, app, evi):
        with pytest.raises(ValueError, match="in place"):
            f(k_pages=odd)
    for kw, err in ((dict(q=q[:1]), ValueError), (dict(q=q[:, :3]), ValueError), (dict(q=q.half()), ValueError), (dict(q=q[..., :32]), ValueError),
                    (dict(q=q.cpu()), RuntimeError), (dict(window_size=0), ValueError), (dict(scale=math.nan), ValueError),
                    (dict(sinks=torch.zeros(3, device=gpu)), ValueError), (dict(sinks=torch.zeros(4)), RuntimeError),
                    (dict(descale=(2.0, 1.0)), ValueError), (dict(max_seqlen=0), ValueError), (dict(weight_sums=sums[:, :1]), ValueError),
                    (dict(weight_sums=sums.half()), ValueError), (dict(weight_sums=sums[..., :47].contiguous()), ValueError),
                    (dict(weight_sums=sums.cpu()), RuntimeError), (dict(weight_sums=torch.zeros(2, 48, 2, device=gpu).transpose(1, 2)), ValueError)):
        with pytest.raises(err):
            att(**kw)
    wide = kp[:1].expand(6, 2, 16, 64)
    for f, kw in ((app, dict(k_pages=wide)), (app, dict(v_pages=wide)), (evi, dict(k_pages=wide)), (evi, dict(v_pages=wide)),
                  (att, dict(weight_sums=sums[:1].expand(2, 2, 48)))):
        with pytest.raises(ValueError, match="share memory"):
            f(**kw)
    att(k_pages=wide, v_pages=wide)  # (reading them is well defined)
    q8 = torch.zeros(6, 2, 16, 64, device=gpu).to(torch.float8_e4m3fn)
    with pytest.raises(ValueError):
        att(q=q.float(), k_pages=q8, v_pages=q8)
    with pytest.raises(ValueError):
        app(k_pages=q8, v_pages=q8, descale=(0.0, 1.0))
    for kw in (dict(k=x[:1]), dict(k=x[:1], v=x[:1]), dict(v=x.half()), dict(k=q, v=q), dict(cu_seqlens=torch.tensor([0, 1])),
               dict(cu_seqlens=torch.tensor([0, 2, 1])), dict(cu_seqlens=torch.tensor([0, 1, 3]))):
        with pytest.raises(ValueError):
            app(**kw)
    for kw in (dict(keep=0), dict(keep=17), dict(sink_size=-1), dict(recent=-1), dict(sink_size=9, recent=8), dict(new_table=table),
               dict(new_table=nt[:1]), dict(new_table=nt.long()), dict(weight_sums=sums[..., :40].contiguous()), dict(weight_sums=sums.half())):
        with pytest.raises(ValueError):
            evi(**kw)
    with pytest.raises(RuntimeError):
        evi(new_table=nt.cpu())
    torch.cuda.synchronize()


def test_ctypes_path(fa, gpu, monkeypatch):
    """Without the C++ binding: the same results, version counters included."""
    c = make(71, "bf16", "fp8", 64, 8, 2, 16, "nhd", (700, 33), nan=False)
    P = c["kp"].shape[0]
    x = torch.randn(2, 2, 64, generator=c["g"]).to(torch.bfloat16).to(gpu)
    nt = torch.tensor([[P - 1], [P - 2]], dtype=torch.int32, device=gpu)
    c["table"] = c["table"] % (P - 3)

    def run():
        kp, vp = on_gpu(c["kp"], gpu), on_gpu(c["vp"], gpu)
        sums = torch.zeros(2, 2, c["table"].shape[1] * 16, device=gpu)
        t, lens = c["table"].to(gpu), c["lens"].to(gpu)
        before = [y._version for y in (kp, vp, sums)]
        fa.paged_append(x, x, kp, vp, t, lens, descale=c["descale"])
        o = fa.paged_attention(c["q"].to(gpu), kp, vp, t, lens, sinks=c["sinks"].to(gpu), descale=c["descale"], weight_sums=sums)
        left, new = fa.paged_evict(kp, vp, t, lens, sums, 16, nt, 2, 3)
        assert all(y._version > z for y, z in zip((kp, vp, sums), before))
        return o, sums, kp, vp, left, new
    a = run()
    monkeypatch.setattr(load_mod("_ops"), "_BINDING", None)
    for y, z in zip(a, run()):
        same(y, z)


def test_inputs_in_other_layouts(fa, gpu):
    """q, k, v, the table and lens as views: slices of a fused projection, unaligned, strided."""
    c = make(81, "bf16", "bf16", 64, 8, 2, 16, "hnd", (700, 33, 5), nan=False)
    kp, vp, t, lens = (c[n].to(gpu) for n in ("kp", "vp", "table", "lens"))
    q = c["q"].to(gpu)
    want = fa.paged_attention(q, kp, vp, t, lens)
    k, v = (torch.randn(3, 2, 64, generator=c["g"]).to(torch.bfloat16).to(gpu) for _ in range(2))
    fused = torch.cat((q, k, v), 1)  # [B, Hq + 2 Hkv, D]
    odd = torch.zeros(3 * 8 * 64 + 1, dtype=torch.bfloat16, device=gpu)[1:].view(3, 8, 64).copy_(q)
    by_dim = q.transpose(1, 2).contiguous().transpose(1, 2)
    one = torch.zeros(3, 8, 64, 2, dtype=torch.bfloat16, device=gpu)[..., 0].copy_(q)
    wide = torch.zeros(3, t.shape[1], 2, dtype=torch.int32, device=gpu)[..., 1].copy_(t)
    turned = t.t().contiguous().t()
    far = torch.zeros(3, 2, dtype=torch.int32, device=gpu)[:, 1].copy_(lens)
    for x in (fused[:, :8], odd, by_dim, one, q.unsqueeze(2).expand(3, 8, 5, 64)[:, :, 3]):
        for tt in (t, wide, turned):
            same(fa.paged_attention(x, kp, vp, tt, far), want)
    a, b = (kp.clone(), vp.clone()), (kp.clone(), vp.clone())
    fa.paged_append(k, v, *a, t, lens)
    strange = torch.zeros(3, 2, 64, 3, dtype=torch.bfloat16, device=gpu)[..., 2].copy_(k)
    fa.paged_append(strange, fused[:, 10:], *b, wide, far)
    same(a[0], b[0])
    same(a[1], b[1])


def test_shared_prefix(fa, gpu):
    """Two sequences share the pages of a prefix: attention reads them, eviction leaves them whole."""
    c = make(82, "bf16", "bf16", 64, 4, 2, 16, "hnd", (100, 90), nan=False)
    c["table"][1, :4] = c["table"][0, :4]
    P = c["kp"].shape[0]
    kp, vp = (torch.cat((x, x[:6])) for x in (c["kp"], c["vp"]))
    sums = torch.rand(2, 2, 112, generator=c["g"])
    new_table = torch.arange(P, P + 6, dtype=torch.int32).view(2, 3)
    t, lens, gk, gv, gs = c["table"].to(gpu), c["lens"].to(gpu), kp.to(gpu), vp.to(gpu), sums.to(gpu)
    ref, mag, ref_sums = oracle.attention(c["q"], kp, vp, c["table"], c["lens"], sums=sums)
    o = fa.paged_attention(c["q"].to(gpu), gk, gv, t, lens, weight_sums=gs)
    check_attention(o, dict(c, kp=kp, vp=vp), ref, mag, "bf16", 64, 100, 0.125)
    assert torch.allclose(gs.cpu().double(), ref_sums, rtol=1e-5, atol=1e-6)
    want = oracle.evict(kp, vp, c["table"], c["lens"], gs.cpu(), 48, new_table, 4, 8)
    left, new = fa.paged_evict(gk, gv, t, lens, gs, 48, new_table.to(gpu), 4, 8)
    same(gk, want[0])
    same(gv, want[1])
    same(new, want[3])


def test_traced_calls_are_refused(fa, gpu):
    kp = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16, device=gpu)
    t, lens = torch.zeros(1, 2, dtype=torch.int32, device=gpu), torch.ones(1, dtype=torch.int32, device=gpu)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: fa.paged_attention(x, kp, kp, t, lens), (q,), check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        torch.func.vmap(lambda x: fa.paged_attention(x, kp, kp, t, lens))(q.unsqueeze(0))


def test_inference_mode(fa, gpu):
    """Inference tensors have no version counters to raise."""
    c = make(91, "bf16", "bf16", 64, 4, 2, 16, "hnd", (40, 9), nan=False)
    with torch.inference_mode():
        kp, vp, t, lens = (c[n].to(gpu) for n in ("kp", "vp", "table", "lens"))
        x = torch.randn(2, 2, 64, generator=c["g"]).to(torch.bfloat16).to(gpu)
        sums = torch.zeros(2, 2, t.shape[1] * 16, device=gpu)
        fa.paged_append(x, x, kp, vp, t, lens)
        fa.paged_attention(c["q"].to(gpu), kp, vp, t, lens, weight_sums=sums)
        nt = torch.arange(c["used"], c["used"] + 2, dtype=torch.int32, device=gpu).view(2, 1)
        left, new = fa.paged_evict(kp, vp, t, lens, sums, 16, nt)
        assert left.tolist() == [16, 9] and float(sums.sum()) > 0


def test_pools_of_different_layouts_and_narrow_sums(fa, gpu):
    """K pages with the heads first, V pages as half of a fused pool with the slots first; sums as wide as max_seqlen."""
    c = make(95, "bf16", "bf16", 64, 8, 2, 16, "hnd", (700, 33, 1300), nan=False)
    P = c["kp"].shape[0]
    fused = torch.zeros(P, 16, 2, 2, 64, dtype=torch.bfloat16, device=gpu)  # [pages, slots, K/V, heads, D]
    vp = fused[:, :, 1].transpose(1, 2)
    vp.copy_(c["vp"])
    kp, t, lens = c["kp"].to(gpu), c["table"].to(gpu), c["lens"].to(gpu)
    w = torch.rand(2, 3, 1500, generator=c["g"]).to(gpu)[:, :, 100:1400].transpose(0, 1)  # [B, Hkv, 1300], unaligned
    w0 = w.clone()
    ref, mag, ref_sums = oracle.attention(c["q"], c["kp"], c["vp"], c["table"], c["lens"], 1250, 7, sums=torch.zeros(3, 2, 1312))
    o = fa.paged_attention(c["q"].to(gpu), kp, vp, t, lens, 1250, 7, max_seqlen=1300, weight_sums=w)
    check_attention(o, c, ref, mag, "bf16", 64, 1300, 0.125, 1250, 7)
    assert torch.allclose((w - w0).cpu().double(), ref_sums[..., :1300], atol=1e-5)
    x = torch.randn(3, 2, 64, generator=c["g"]).to(torch.bfloat16)
    want = oracle.append(x, x, c["kp"], c["vp"], c["table"], c["lens"])
    fa.paged_append(x.to(gpu), x.to(gpu), kp, vp, t, lens)
    same(kp, want[0])
    same(vp, want[1])
    assert not fused[:, :, 0].any()
