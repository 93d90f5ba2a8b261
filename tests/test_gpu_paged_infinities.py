"""Infinite values at visible places: o is infinite or NaN where the formula says so, and as without them elsewhere."""
import math

import pytest
import torch

from test_gpu_paged import make, on_gpu, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("lens,Hq", [((300, 70, 33), 8), ((2500, 4000, 1), 8), ((300, 2500, 40), 40)])
def test_infinite_values(fa, gpu, dtype, D, lens, Hq):
    c = make(7, dtype, dtype, D, Hq, 1, 16, "hnd", lens)
    c["q"] = (c["q"].float() / 4).to(c["q"].dtype)  # (no weight is so small that 16 bits do not hold it)
    run = lambda vp: fa.paged_attention(c["q"].to(gpu), on_gpu(c["kp"], gpu), on_gpu(vp, gpu), c["table"].to(gpu), c["lens"].to(gpu)).cpu()
    clean = run(c["vp"])
    vp, want = c["vp"].clone(), clean.clone()
    for b, n in enumerate(lens):
        # dim 0: infinities of one sign all over, dim 1: of the other at one key, dim 2: of both signs, dim 3: NaN
        keys = [n // 2] if n < 50 else [n // 5, n // 2, n - 1]
        for i, k in enumerate(keys):
            row = vp[c["table"][b, k // 16], 0, k % 16]
            row[0] = math.inf
            if i == 0:
                row[1] = -math.inf
                row[3] = math.nan
            if len(keys) > 1:
                row[2] = math.inf if i else -math.inf
        want[b, :, 0], want[b, :, 1], want[b, :, 3] = math.inf, -math.inf, math.nan
        if len(keys) > 1:
            want[b, :, 2] = math.nan
    o = run(vp)
    assert torch.equal(o.isnan(), want.isnan()), [(int(x), int(y)) for x, y in zip(o.isnan().sum((0, 1)), want.isnan().sum((0, 1)))][:4]
    same(o[..., :2], want[..., :2])
    same(o[..., 4:], clean[..., 4:], "other dims")
