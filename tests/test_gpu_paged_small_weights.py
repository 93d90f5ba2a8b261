"""Long caches in which one key outweighs each of the others by far, and they count by their number.

Tolerance, against the float64 oracle, as in test_gpu_paged.py: d mag for scores and sums, half a step of the output, and what a
16-bit weight loses: float16 has no numbers below 2^-24, so each key at most half of that, 2^-25, of weights of which the largest
is at least 2^7: 2^-32 max |v| a key."""
import pytest
import torch

from oracle import paged as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1000, 20000])
@pytest.mark.parametrize("dtype,cache", [("fp16", "fp16"), ("fp16", "fp8"), ("bf16", "bf16"), ("fp32", "fp32")])
def test_many_small_weights(fa, gpu, n, dtype, cache):
    DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
    D, page = 64, 64
    g = torch.Generator().manual_seed(n)
    P = -(-n // page)
    table, lens = torch.randperm(P, generator=g).view(1, P).to(torch.int32), torch.tensor([n], dtype=torch.int32)
    k, v = torch.zeros(n, 1, D), 1 + torch.rand(n, 1, D, generator=g)
    at = n // 3  # the heavy key, of value 0
    k[at, 0, 0], v[at] = 18, 0
    kp, vp = (torch.zeros(P, 1, page, D, dtype=DT[cache]) for _ in range(2))
    kp, vp = oracle.append(k, v, kp, vp, table, lens, torch.tensor([0, n]))
    q = torch.zeros(1, 3, D)
    q[0, :, 0] = torch.tensor([8.0, 7.0, 5.0])  # the others weigh 2^-26, 2^-22.7 and 2^-16.2 of it
    q = q.to(DT[dtype])
    ref, mag, _ = oracle.attention(q, kp, vp, table, lens)
    o = fa.paged_attention(*(x.to(gpu) for x in (q, kp, vp, table, lens)))
    d = 2 * (D + 4) * 2.0 ** -24 * 18 + 2.0 ** -21
    eps = torch.finfo(DT[dtype]).eps
    tol = (d + 2.0 ** -17 + n * 2.0 ** -24) * mag + eps / 2 * ref.abs()
    if dtype == "fp16":
        tol = tol + n * 2.0 ** -32 * float(v.max()) + 2.0 ** -25
    err = (o.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), (float(err.max()), float((err - tol).max()), float(ref.max()))
