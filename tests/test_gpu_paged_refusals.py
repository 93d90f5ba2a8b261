"""Refused calls of the paged operators leave nothing behind."""
import pytest
import torch

from conftest import load_mod

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("binding", [True, False])
def test_a_refused_eviction_allocates_no_workspace(fa, gpu, monkeypatch, binding):
    """keep far past the new table ("no limit") is the documented error, before room is made for that many entries."""
    if not binding:
        monkeypatch.setattr(load_mod("_ops"), "_BINDING", None)
    kp = torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16, device=gpu)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device=gpu), torch.ones(2, dtype=torch.int32, device=gpu)
    sums, nt = torch.zeros(2, 2, 48, device=gpu), torch.ones(2, 1, dtype=torch.int32, device=gpu)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="new table"):
        fa.paged_evict(kp, kp.clone(), table, lens, sums, 2 ** 26, nt)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20
