"""The paged oracle (oracle/paged.py) against independent statements: SDPA over the gathered keys with an explicit mask,
sorting for eviction, plain indexing for appending."""
import math

import pytest
import torch

from oracle import paged


def _case(seed=0, B=3, H=2, P=12, S=4, D=8, lens=(9, 0, 16)):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(P, H, S, D, generator=g) for _ in range(2))
    table = torch.randperm(P, generator=g)[:B * 4].view(B, 4).to(torch.int32)
    return g, k, v, table, torch.tensor(lens, dtype=torch.int32)


@pytest.mark.parametrize("window,sink", [(None, 0), (5, 0), (3, 2), (0, 3), (100, 100)])
@pytest.mark.parametrize("learned", [False, True])
def test_attention_is_sdpa(window, sink, learned):
    g, k, v, table, lens = _case()
    q = torch.randn(3, 4, 8, generator=g)
    sinks = torch.randn(4, generator=g) if learned else None
    o, mag, sums = paged.attention(q, k, v, table, lens, window, sink, sinks, sums=torch.zeros(3, 2, 16))
    for b in range(3):
        n = int(lens[b])
        if n == 0:
            assert not o[b].any() and not sums[b].any()
            continue
        kd = k[table[b].long()].transpose(0, 1).reshape(2, 16, 8)[:, :n].repeat_interleave(2, 0).double()
        vd = v[table[b].long()].transpose(0, 1).reshape(2, 16, 8)[:, :n].repeat_interleave(2, 0).double()
        i = torch.arange(n)
        seen = (n - 1 - i < (n if window is None else window)) | (i < sink)
        mask = torch.where(seen, 0.0, -math.inf).double().expand(4, 1, n)
        if learned:  # one zero key more, whose mask holds the logit
            kd, vd = (torch.cat((x, torch.zeros(4, 1, 8).double()), 1) for x in (kd, vd))
            mask = torch.cat((mask, sinks.double().view(4, 1, 1)), 2)
        ref = torch.nn.functional.scaled_dot_product_attention(q[b].double()[:, None], kd, vd, attn_mask=mask)[:, 0]
        assert torch.allclose(o[b], ref, atol=1e-12)
        assert bool((mag[b] >= o[b].abs() - 1e-12).all())
        if not learned:
            assert torch.allclose(sums[b].sum(-1), torch.full((2,), 2.0).double())


def test_append_and_bad_entries():
    g, k, v, table, lens = _case(lens=(9, 0, 16))
    table[2, 3] = -1  # the last page of sequence 2 does not exist
    nk, nv = (torch.randn(3, 2, 8, generator=g) for _ in range(2))
    kp, vp = paged.append(nk, nv, k, v, table, lens)
    want = k.clone()
    want[table[0, 2].long(), :, 0] = nk[0]
    assert torch.equal(kp, want)
    kp, _ = paged.append(nk, nv, k, v, table, torch.tensor([2, 1, 0]), cu=torch.tensor([0, 2, 3, 3]))
    assert torch.equal(kp[table[0, 0].long(), :, :2], nk[:2].transpose(0, 1)) and torch.equal(kp[table[1, 0].long(), :, 0], nk[2])


def test_kept_is_a_stable_sort():
    g = torch.Generator().manual_seed(3)
    for _ in range(50):
        w = torch.randint(0, 6, (30,), generator=g).float()
        n, keep, sink, recent = 27, 12, 3, 4
        x = w[:n].clone()
        x[:sink] = x[n - recent:] = math.inf
        want = sorted(torch.sort(x, descending=True, stable=True).indices[:keep].tolist())
        assert paged.kept(w, n, keep, sink, recent) == want
    w = torch.tensor([0.0, math.nan, math.inf, -0.0, -1.0, math.nan])
    assert paged.kept(w, 6, 3, 0, 0) == [1, 2, 5]
    assert paged.kept(torch.tensor([-0.0, 0.0, -0.0]), 3, 1, 0, 0) == [0]
    assert paged.kept(w, 6, 4, 2, 2) == [0, 1, 4, 5]


def test_evict_moves_entries_in_order():
    g, k, v, table, lens = _case(P=24, lens=(9, 3, 16))
    new_table = torch.tensor([[20, 21], [22, 23], [18, 19]], dtype=torch.int32)
    new_table = torch.tensor([p for p in range(24) if p not in set(table.view(-1).tolist())][:6], dtype=torch.int32).view(3, 2)
    sums = torch.rand(3, 2, 16, generator=g)
    kp, vp, left, new = paged.evict(k, v, table, lens, sums, 6, new_table, 1, 2)
    assert left.tolist() == [6, 3, 6]
    for b in range(3):
        for h in range(2):
            at = paged.kept(sums[b, h], int(lens[b]), 6, 1, 2)
            old = k[table[b].long(), h].reshape(16, 8)[at]
            assert torch.equal(kp[new_table[b].long(), h].reshape(8, 8)[:len(at)], old)
            assert torch.equal(new[b, h, :len(at)], sums[b, h, at]) and not new[b, h, len(at):].any()
