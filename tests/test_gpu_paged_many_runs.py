"""Calls over pages with the slots first that are cut into twice as many runs, and short ones whose table would allow as much: against
float64, with weights.  Tolerances as in test_gpu_paged.py."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [(150001, 60000, 0, 7), (3000, 60000, 130, 1), (0, 1, 0, 0)])
def test_slots_first(fa, gpu, lens):
    Hq, Hkv, D, page, width = 16, 8, 64, 64, 2400
    g = torch.Generator(device=gpu).manual_seed(6)
    B, used = len(lens), [-(-n // page) for n in lens]
    P = sum(used) + 1
    order = torch.randperm(P, generator=g, device=gpu).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device=gpu)
    for b in range(B):
        table[b, :used[b]] = order[sum(used[:b]):sum(used[:b + 1])]
    q = torch.randn(B, Hq, D, generator=g, device=gpu).to(torch.bfloat16) * 2
    kp, vp = (torch.randn(P, page, Hkv, D, generator=g, device=gpu).to(torch.bfloat16).transpose(1, 2) for _ in range(2))
    sinks, sums = torch.randn(Hq, generator=g, device=gpu), torch.zeros(B, Hkv, width * page, device=gpu)
    tl = torch.tensor(lens, dtype=torch.int32, device=gpu)
    o = fa.paged_attention(q, kp, vp, table, tl, sinks=sinks, weight_sums=sums)
    same = fa.paged_attention(q, kp, vp, table, tl, sinks=sinks, weight_sums=torch.zeros_like(sums))
    assert torch.equal(o, same)
    for b, n in enumerate(lens):
        assert not sums[b, :, n:].any()
        if not n:
            assert not o[b].any()
            continue
        at = table[b, :used[b]].long()
        for h in range(Hkv):
            k, v = (x[at, h].reshape(-1, D)[:n].double() for x in (kp, vp))
            qh = q[b, 2 * h:2 * h + 2].double()
            s = torch.cat((qh @ k.t() / 8, sinks[2 * h:2 * h + 2, None].double()), -1)
            p = torch.softmax(s, -1)[:, :n]
            a = float((qh.abs() @ k.abs().t()).max()) / 8
            d = 2 * (D + 4) * 2.0 ** -24 * a + 2.0 ** -21
            tol = (d + 2.0 ** -17 + n * 2.0 ** -24) * (p @ v.abs()) + 2.0 ** -8 * (p @ v).abs()
            err = (o[b, 2 * h:2 * h + 2].double() - p @ v).abs()
            assert bool((err <= tol).all()), (b, h, float((err - tol).max()))
            w = p.sum(0)
            assert bool(((sums[b, h, :n].double() - w).abs() <= (d + n * 2.0 ** -24) * w + 2.0 ** -23 * w).all())
