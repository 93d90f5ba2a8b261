"""Oracle of the paged key-value cache in float64 on the CPU: appending rows, attention of one new token a
sequence, eviction by accumulated weight.  Loops over sequences, heads and tokens, written from the definitions;
it knows pages only through `entry`."""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def entry(table, b, pos, page_size, pages):
    """(page, slot) of position pos of sequence b, or None where the table names no page."""
    if pos < 0 or pos >= table.shape[1] * page_size:
        return None
    p = int(table[b, pos // page_size])
    return (p, pos % page_size) if 0 <= p < pages else None


def codes(x, dtype, descale):
    """x as pages of `dtype` store it; e4m3: codes of clamp(x * fl32(1 / descale))."""
    if dtype != torch.float8_e4m3fn:
        return x.to(dtype)
    inv = torch.tensor(1.0 / descale, dtype=torch.float64).to(torch.float32)
    return (x.float() * inv).clamp(-E4M3_MAX, E4M3_MAX).to(dtype)


def append(k, v, k_pages, v_pages, table, lens, cu=None, descale=(1.0, 1.0)):
    """New contents of (k_pages, v_pages); every argument is a CPU tensor."""
    kp, vp = k_pages.clone(), v_pages.clone()
    B = table.shape[0]
    cu = list(range(B + 1)) if cu is None else cu.tolist()
    ck, cv = codes(k, kp.dtype, descale[0]), codes(v, vp.dtype, descale[1])
    for b in range(B):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            at = entry(table, b, int(lens[b]) - n + i, kp.shape[2], kp.shape[0])
            if at is not None:
                kp[at[0], :, at[1]] = ck[cu[b] + i]
                vp[at[0], :, at[1]] = cv[cu[b] + i]
    return kp, vp


def gather(pages, table, b, positions):
    """float64 [n, Hkv, D] of sequence b's positions, and which of them are on a page."""
    P, H, S, D = pages.shape
    x, ok = torch.zeros(len(positions), H, D, dtype=torch.float64), []
    for i, pos in enumerate(positions):
        at = entry(table, b, pos, S, P)
        ok.append(at is not None)
        if at is not None:
            x[i] = pages[at[0], :, at[1]].double()
    return x, torch.tensor(ok, dtype=torch.bool)


def attention(q, k_pages, v_pages, table, lens, window=None, sink=0, sinks=None, scale=None, descale=(1.0, 1.0), sums=None):
    """(o float64 [B, Hq, D], |o|'s scale: sum of p |v| of the same shape, new sums or None)."""
    B, Hq, D = q.shape
    P, H, S, _ = k_pages.shape
    G = Hq // H
    scale = 1 / math.sqrt(D) if scale is None else scale
    o, mag = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    sums = None if sums is None else sums.double().clone()
    for b in range(B):
        n = max(0, min(int(lens[b]), table.shape[1] * S))
        pos = [k for k in range(n) if window is None or n - 1 - k < window or k < sink]
        k, ok = gather(k_pages, table, b, pos)
        v, _ = gather(v_pages, table, b, pos)
        pos = [p for p, y in zip(pos, ok.tolist()) if y]
        k, v = k[ok] * descale[0], v[ok] * descale[1]
        for h in range(Hq):
            s = scale * (k[:, h // G] @ q[b, h].double())
            if sinks is not None:
                s = torch.cat((s, sinks[h].double().view(1)))
            if s.numel() == 0 or not pos:
                continue
            p = torch.softmax(s, 0)[:len(pos)]
            o[b, h], mag[b, h] = p @ v[:, h // G], p @ v[:, h // G].abs()
            if sums is not None:
                sums[b, h // G, pos] += p
    return o, mag, sums


def kept(w, n, keep, sink, recent, live=None):
    """Positions that stay of one (sequence, KV head) with weights w; live: those on a page (None: all of n)."""
    live = list(range(n)) if live is None else live
    if len(live) <= keep:
        return live
    held = [i for i in live if i < sink or i >= n - recent]
    rest = [i for i in live if sink <= i < n - recent]
    key = [math.inf if math.isnan(x) else x for x in w[:n].tolist()]
    first = [0 if math.isnan(x) else 1 for x in w[:n].tolist()]  # (a NaN above every number)
    rest.sort(key=lambda i: (first[i], -key[i], i))
    return sorted(held + rest[:keep - len(held)])


def evict(k_pages, v_pages, table, lens, sums, keep, new_table, sink=0, recent=0):
    """New contents of (k_pages, v_pages), new lens, new sums.  Positions on no page are none of the sequence's."""
    kp, vp = k_pages.clone(), v_pages.clone()
    P, H, S, _ = kp.shape
    new, left = torch.zeros_like(sums), []
    for b in range(table.shape[0]):
        n = max(0, min(int(lens[b]), table.shape[1] * S))
        live = [i for i in range(n) if entry(table, b, i, S, P) is not None]
        left.append(min(len(live), keep))
        for h in range(H):
            for r, i in enumerate(kept(sums[b, h], n, keep, sink, recent, live)):
                new[b, h, r] = sums[b, h, i]
                src, dst = entry(table, b, i, S, P), entry(new_table, b, r, S, P)
                if dst is not None:
                    kp[dst[0], h, dst[1]] = k_pages[src[0], h, src[1]]
                    vp[dst[0], h, dst[1]] = v_pages[src[0], h, src[1]]
    return kp, vp, torch.tensor(left, dtype=torch.int32), new
