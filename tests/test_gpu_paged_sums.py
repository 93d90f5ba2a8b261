"""Accumulated weights to float32's accuracy at every width and type, one long sequence among short ones, and e4m3 codes bit for
bit.

Tolerance of the weights against the float64 oracle: a head's score is off by at most (D + 4) 2^-24 a, with a = scale *
sum_i |q_i k_i| of its own keys (products are exact in float32; D roundings of the sum, those of the scale and of the maximum's
difference), exp2 by 2^-22, and the sum of n weights by n 2^-24: a weight by the factor d = 2 max_k (D + 4) 2^-24 a[k] +
2^-21 + n 2^-24.  float32 products are not exact: D roundings more.  G weights are added to a sum: (G + 1) 2^-24 of the result."""
import math

import pytest
import torch

from oracle import paged as oracle
from test_gpu_paged import DT, bits, make, on_gpu

pytestmark = pytest.mark.gpu

CASES = [
    # dtype, cache, D, Hq, Hkv, page, layout, lens, window, sink, learned
    ("bf16", "bf16", 128, 8, 2, 32, "nhd", (1, 64, 999, 0, 555), None, 0, True),
    ("fp16", "fp16", 128, 20, 1, 64, "hnd", (300, 1, 1600), None, 0, False),
    ("bf16", "fp8", 64, 8, 1, 16, "hnd", (70, 1, 1800, 0), None, 0, True),
    ("fp16", "fp8", 128, 34, 1, 16, "nhd", (1030, 5), None, 0, True),
    ("bf16", "fp8", 128, 8, 2, 24, "hnd", (70, 33, 777), 300, 4, False),
    ("fp32", "fp32", 128, 18, 1, 20, "hnd", (70, 32, 700), None, 0, True),
    ("bf16", "bf16", 16, 5, 1, 16, "nhd", (70, 1, 800), 100, 2, False),
    # one long sequence among many short ones
    ("bf16", "bf16", 64, 16, 2, 16, "hnd", (20000,) + tuple(range(0, 320, 10)), None, 0, True),
    ("fp16", "fp8", 64, 16, 2, 16, "nhd", tuple(range(0, 320, 10)) + (17000,), None, 0, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:7]) + f"-{len(c[7])}-W{c[8]}-S{c[9]}")
def test_weight_sums(fa, gpu, case):
    dtype, cache, D, Hq, Hkv, page, layout, lens, W, S, learned = case
    print(case, flush=True)
    c = make(51, dtype, cache, D, Hq, Hkv, page, layout, lens)
    w0 = torch.rand(len(lens), Hkv, c["table"].shape[1] * page, generator=c["g"])
    w = w0.to(gpu)
    fa.paged_attention(c["q"].to(gpu), on_gpu(c["kp"], gpu), on_gpu(c["vp"], gpu), c["table"].to(gpu), c["lens"].to(gpu), W, S,
                       c["sinks"].to(gpu) if learned else None, descale=c["descale"], weight_sums=w)
    w, G = w.double().cpu(), Hq // Hkv
    for b, n in enumerate(lens):
        pos = [k for k in range(n) if W is None or n - 1 - k < W or k < S]
        keys = oracle.gather(c["kp"], c["table"], b, pos)[0] * c["descale"][0]
        want, tol = w0[b].double(), torch.zeros(Hkv, w0.shape[2], dtype=torch.float64)
        for h in range(Hq if pos else 0):
            q, k = c["q"][b, h].double(), keys[:, h // G]
            s = k @ q / math.sqrt(D)
            a = float((k.abs() @ q.abs()).max()) / math.sqrt(D)
            p = torch.softmax(torch.cat((s, c["sinks"][h:h + 1].double())) if learned else s, 0)[:len(pos)]
            d = 2 * ((2 if dtype == "fp32" else 1) * D + 4) * 2.0 ** -24 * a + 2.0 ** -21 + len(pos) * 2.0 ** -24
            want[h // G, pos] += p
            tol[h // G, pos] += d * p
        tol += (G + 1) * 2.0 ** -24 * want
        err = (w[b] - want).abs()
        assert bool((err <= tol).all()), (b, n, float((err - tol).max()), float(err.max()))
        unseen = torch.ones(w0.shape[2], dtype=torch.bool)
        unseen[pos] = False
        assert torch.equal(w[b][:, unseen], w0[b].double()[:, unseen])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128])
def test_codes_are_those_of_quantize_fp8(fa, gpu, dtype, D):
    """Every 16-bit number, NaNs of both signs among them: all bits of the codes."""
    x = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(DT[dtype]).view(-1, 1, D).to(gpu)
    rows = x.shape[0]
    pages = [torch.zeros(rows // 16, 1, 16, D, device=gpu).to(torch.float8_e4m3fn) for _ in range(2)]
    table = torch.arange(rows // 16, dtype=torch.int32, device=gpu).view(1, -1)
    fa.paged_append(x, x.flip(0), *pages, table, torch.tensor([rows], dtype=torch.int32, device=gpu), cu_seqlens=torch.tensor([0, rows]),
                    descale=(0.013, 1.7))
    for y, p, f in zip((x, x.flip(0)), pages, (0.013, 1.7)):
        assert torch.equal(bits(fa.quantize_fp8(y.contiguous(), f)[0]).view(-1), bits(p).view(-1))
