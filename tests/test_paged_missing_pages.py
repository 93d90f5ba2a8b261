"""Eviction of sequences with pages that the table does not name (handed back, or never given): the oracle on the CPU."""
import math

import pytest
import torch

from oracle import paged


def case(seed, gaps, lens=(12, 30), page=4):
    """Two sequences over shuffled pages, entry p of sequence b's row no page where (b, p) is in gaps.  new_table names pages of
    NaN."""
    g = torch.Generator().manual_seed(seed)
    width = 8
    used = torch.randperm(2 * width, generator=g)
    table = used.view(2, width).to(torch.int32)
    kp, vp = (torch.randn(4 * width, 2, page, 8, generator=g) for _ in range(2))
    kp[2 * width:], vp[2 * width:] = math.nan, math.nan
    for b, p in gaps:
        table[b, p] = [-1, 4 * width, 2 ** 31 - 1, -2 ** 31][p % 4]
    new_table = (2 * width + torch.randperm(2 * width, generator=g)).view(2, width).to(torch.int32)
    q, sums = torch.randn(2, 4, 8, generator=g), torch.rand(2, 2, width * page, generator=g)
    return q, kp, vp, table, torch.tensor(lens, dtype=torch.int32), sums, new_table


@pytest.mark.parametrize("gaps", [[(0, 0)], [(0, 2), (1, 7)], [(0, 0), (0, 1), (0, 2), (1, 1), (1, 6)]])
def test_nothing_evicted_leaves_attention_as_it_was(gaps):
    q, kp, vp, table, lens, sums, new_table = case(1, gaps)
    before = paged.attention(q, kp, vp, table, lens)[0]
    nk, nv, left, new = paged.evict(kp, vp, table, lens, sums, 32, new_table)
    after = paged.attention(q, nk, nv, new_table, left)[0]
    assert torch.allclose(before, after, atol=1e-12)
    assert left.tolist() == [int(n) - sum(max(0, min(4, int(n) - 4 * p)) for c, p in gaps if c == b) for b, n in enumerate(lens)]


def test_entries_that_stay_are_on_pages():
    """The first and last positions stay where they are on a page; the others make room for as many more."""
    q, kp, vp, table, lens, sums, new_table = case(2, [(1, 0), (1, 3), (1, 7)])
    nk, nv, left, new = paged.evict(kp, vp, table, lens, sums, 12, new_table, 6, 5)
    assert left.tolist() == [8 + 4, 12]
    live = [i for i in range(30) if i // 4 not in (0, 3, 7)]
    for h in range(2):
        held = [i for i in live if i < 6 or i >= 25]
        rest = sorted((i for i in live if 6 <= i < 25), key=lambda i: (-float(sums[1, h, i]), i))
        want = sorted(held + rest[:12 - len(held)])
        rows = kp[table[1].long().clamp(0, 31)].transpose(1, 2).reshape(32, 2, 8)[want, h]
        assert torch.equal(nk[new_table[1].long()].transpose(1, 2).reshape(32, 2, 8)[:12, h], rows)
        assert torch.equal(new[1, h, :12], sums[1, h, want]) and not new[1, h, 12:].any()
