"""Transformed calls of the paged operators are refused by name, before anything else is looked at: whichever tensor carries the
tangent, with the C++ binding and without it."""
import pytest
import torch
from torch.autograd import forward_ad

from conftest import load_mod

_ops = load_mod("_ops")


@pytest.mark.parametrize("binding", [True, False])
def test_tangents_and_vmap(fa, monkeypatch, binding):
    if not binding:
        monkeypatch.setattr(_ops, "_BINDING", None)
    pages, q, sinks = torch.zeros(4, 2, 16, 64), torch.zeros(1, 4, 64), torch.zeros(4)
    table, lens, sums = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, 32)
    x = torch.zeros(1, 2, 64)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: fa.paged_attention(dual(q), pages, pages, table, lens),
                     lambda: fa.paged_attention(q, pages, pages, table, lens, sinks=dual(sinks)),
                     lambda: fa.paged_attention(q, pages, pages, table, lens, weight_sums=dual(sums)),
                     lambda: fa.paged_attention(q, pages, dual(pages), table, lens),
                     lambda: fa.paged_append(x, dual(x), pages, pages, table, lens),
                     lambda: fa.paged_evict(pages, pages, table, lens, dual(sums), 16, table.clone())):
            with pytest.raises(RuntimeError, match="traced or transformed"):
                call()
    with pytest.raises(RuntimeError, match="traced or transformed"):
        torch.func.vmap(lambda n: fa.paged_attention(q, pages, pages, table, n))(lens.unsqueeze(0))
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        fa.paged_attention(q, pages, pages, table, lens)
