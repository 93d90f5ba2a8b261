"""Eviction on the GPU of sequences with pages that the table does not name, against the oracle: copies and sums are exact."""
import pytest
import torch

from oracle import paged as oracle
from test_gpu_paged import check_attention, make, on_gpu, same, weights

pytestmark = pytest.mark.gpu

CASES = [
    # cache, D, Hkv, page, layout, lens, keep, sink, recent, share of pages that are missing
    ("bf16", 64, 2, 16, "hnd", (100, 64, 63, 65, 0, 1, 300), 64, 4, 16, 0.3),
    ("bf16", 64, 2, 16, "nhd", (12, 16, 200), 200, 0, 0, 0.4),  # nothing is evicted
    ("fp16", 16, 3, 5, "hnd", (100, 33, 5), 33, 33, 0, 0.5),
    ("fp32", 128, 2, 16, "nhd", (100, 33, 640), 40, 0, 40, 0.2),
    ("fp8", 64, 2, 16, "hnd", (100, 33), 30, 15, 15, 1.0),  # nothing is left
    ("bf16", 128, 2, 64, "hnd", (5000, 4097, 4096), 1024, 4, 256, 0.1),
    ("bf16", 16, 1, 1, "hnd", (3000, 2500), 1000, 100, 100, 0.5),
    # several workgroups a head
    ("fp16", 16, 2, 64, "nhd", (40000, 16385, 5, 20000, 16384), 3000, 4, 100, 0.2),
    ("bf16", 16, 1, 16, "hnd", (40001, 33000), 20000, 17000, 0, 0.1),
    ("bf16", 16, 1, 16, "hnd", (49153, 32769), 20000, 0, 17000, 0.6),
    ("bf16", 16, 24, 16, "nhd", (20001, 16385, 100), 3000, 1, 30, 0.05),
]


def evicted(c, seed, page, keep, missing):
    """The case's pages with room for a new table, pages of its table taken away, the new table."""
    g = torch.Generator().manual_seed(seed)
    B, P = c["table"].shape[0], c["kp"].shape[0]
    gone = torch.rand(c["table"].shape, generator=g) < missing
    c["table"][gone] = torch.tensor([-1, 2 * P + 10 ** 6, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)[torch.randint(0, 4, (int(gone.sum()),), generator=g)]
    width = -(-keep // page) + 1
    more = lambda x: torch.cat((x, x[:1].expand(B * width, *x.shape[1:])), 0)
    kp, vp = (more(x.view(torch.uint8)).view(x.dtype) if x.element_size() == 1 else more(x) for x in (c["kp"].contiguous(), c["vp"].contiguous()))
    return kp, vp, (P + torch.randperm(B * width, generator=g).view(B, width)).to(torch.int32)


@pytest.mark.parametrize("kind", ["weights", "ties", "odd"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:5]) + f"-{c[6]}-{c[7]}-{c[8]}")
def test_evict(fa, gpu, case, kind):
    cache, D, Hkv, page, layout, lens, keep, sink, recent, missing = case
    print(case, kind, flush=True)
    c = make(23, "bf16", cache, D, Hkv, Hkv, page, "hnd", lens, nan=False)
    kp, vp, new_table = evicted(c, 24, page, keep, missing)
    sums = weights(c["g"], kind, (len(lens), Hkv, c["table"].shape[1] * page + 3))
    want = oracle.evict(kp, vp, c["table"], c["lens"], sums, keep, new_table, sink, recent)
    gk, gv = (on_gpu(x.transpose(1, 2).contiguous().transpose(1, 2) if layout == "nhd" else x, gpu) for x in (kp, vp))
    left, new = fa.paged_evict(gk, gv, c["table"].to(gpu), c["lens"].to(gpu), sums.to(gpu), keep, new_table.to(gpu), sink, recent)
    same(left, want[2])
    same(new, want[3], "sums")
    same(gk, want[0])
    same(gv, want[1])


@pytest.mark.parametrize("keep", [16, 320])
def test_attention_after_eviction(fa, gpu, keep):
    """Fresh pages hold NaN: attention over the new table sees kept entries only."""
    c = make(25, "bf16", "bf16", 64, 4, 2, 16, "hnd", (300, 12, 40))
    kp, vp, new_table = evicted(c, 26, 16, keep, 0.0)
    kp[c["kp"].shape[0]:], vp[c["kp"].shape[0]:] = float("nan"), float("nan")
    c["table"][0, 0] = c["table"][0, 7] = c["table"][1, 0] = c["table"][2, 1] = -1
    t, lens, nt, q, gk, gv = (x.to(gpu) for x in (c["table"], c["lens"], new_table, c["q"], kp, vp))
    sums = torch.zeros(3, 2, c["table"].shape[1] * 16, device=gpu)
    fa.paged_attention(q, gk, gv, t, lens, weight_sums=sums)
    sums = sums.cpu()
    kp, vp, left, _ = oracle.evict(kp, vp, c["table"], c["lens"], sums, keep, new_table, 3, 4)
    new_lens, _ = fa.paged_evict(gk, gv, t, lens, sums.to(gpu), keep, nt, 3, 4)
    same(new_lens, left)
    o = fa.paged_attention(q, gk, gv, nt, new_lens)
    ref, mag, _ = oracle.attention(c["q"], kp, vp, new_table, left)
    check_attention(o, dict(c, kp=kp, vp=vp, table=new_table, lens=left), ref, mag, "bf16", 64, 320, 0.125)
    if keep == 320:  # nothing was evicted: as before the call
        ref, mag, _ = oracle.attention(c["q"], kp, vp, c["table"], c["lens"])
        check_attention(o, dict(c, kp=kp, vp=vp), ref, mag, "bf16", 64, 320, 0.125)
    assert not o[1].any()
