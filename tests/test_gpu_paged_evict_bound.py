"""paged_evict with max_seqlen: sums as wide as that, as paged_attention accumulates them, and lens cut off there."""
import pytest
import torch

from conftest import load_mod
from oracle import paged as oracle
from test_gpu_paged import make, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("lens,width,bound", [((1000, 400, 0), 1000, 1000), ((20000, 16385, 300), 20001, 20001), ((700, 650, 30), 640, 640),
                                              ((40000, 700, 30), 1000, 690), ((100, 90, 80), 40000, 2 ** 31)])
def test_narrow_sums(fa, gpu, monkeypatch, binding, lens, width, bound):
    if not binding:
        monkeypatch.setattr(load_mod("_ops"), "_BINDING", None)
    c = make(31, "bf16", "bf16", 16, 2, 2, 16, "hnd", lens, nan=False, extra=1)
    P, keep = c["kp"].shape[0], 90
    kp, vp = (torch.cat((c[n], c[n][:1].expand(18, -1, -1, -1))) for n in ("kp", "vp"))
    new_table = (P + torch.randperm(18, generator=c["g"]).view(3, 6)).to(torch.int32)
    sums = torch.rand(3, 2, width, generator=c["g"])
    cut = c["lens"].clamp(max=min(bound, 2 ** 31 - 1))
    want = oracle.evict(kp, vp, c["table"], cut, sums, keep, new_table, 3, 40)
    gk, gv = kp.to(gpu), vp.to(gpu)
    left, new = fa.paged_evict(gk, gv, c["table"].to(gpu), c["lens"].to(gpu), sums.to(gpu), keep, new_table.to(gpu), 3, 40, max_seqlen=bound)
    same(left, want[2])
    same(new, want[3])
    same(gk, want[0])
    same(gv, want[1])


def test_refusals(fa, gpu):
    c = make(32, "bf16", "bf16", 16, 2, 2, 16, "hnd", (100, 90), nan=False)
    args = [c[n].to(gpu) for n in ("kp", "vp", "table", "lens")]
    nt = torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    for width, bound in ((99, 100), (99, None), (112, 0), (112, -1)):
        with pytest.raises(ValueError):
            fa.paged_evict(*args, torch.zeros(2, 2, width, device=gpu), 48, nt, max_seqlen=bound)
