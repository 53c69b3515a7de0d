"""Paged K/V cache oracle: plain torch in 64 bits, one sequence and one row at a
time where it matters, on whatever device its inputs are.

Key j is visible to the query at position i when j <= i, j < seq_len, its page
is present and (no window, i - j <= window, or j < prefix).
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch


def slots(table, seq_lens, q_start, page_size: int, num_pages: int):
    """(row, page, offset) of every new row that is stored."""
    tab, lens = table.tolist(), seq_lens.tolist()
    starts = list(range(len(lens) + 1)) if q_start is None else q_start.tolist()
    out = []
    for b, n in enumerate(lens):
        for r in range(starts[b], starts[b + 1]):
            pos = n - (starts[b + 1] - r)
            if 0 <= pos < len(tab[b]) * page_size and 0 <= tab[b][pos // page_size] < num_pages:
                out.append((r, tab[b][pos // page_size], pos % page_size))
    return out


def gather(pages, row, n: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first n rows of a sequence ``[n, Hkv, D]`` in 64 bits (rows of absent
    pages are zero) and which of them are present ``[n]``."""
    P, H, ps, D = pages.shape
    pos = torch.arange(n, device=pages.device)
    page = row.to(pages.device).long()[pos // ps]
    there = (page >= 0) & (page < P)
    rows = pages[page.clamp(0, P - 1), :, pos % ps].double()
    return torch.where(there[:, None, None], rows, torch.zeros_like(rows)), there


def attention(q, k_pages, v_pages, table, seq_lens, q_start=None, *, window: Optional[int] = None, prefix: int = 0,
              scale: Optional[float] = None):
    """q ``[N, Hq, D]`` -> ``(out, spread, ds)`` in 64 bits, zeros where nothing is
    visible. spread = sum_j p_j |v_j| and ds = max_j scale * sum_d |q_d k_jd|
    ``[N, Hq]`` are what error bounds are made of."""
    N, Hq, D = q.shape
    Hkv, ps = k_pages.shape[1], k_pages.shape[2]
    g = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(N, Hq, D, dtype=torch.float64, device=q.device)
    spread, ds = torch.zeros_like(out), torch.zeros(N, Hq, dtype=torch.float64, device=q.device)
    lens = seq_lens.tolist()
    starts = list(range(len(lens) + 1)) if q_start is None else q_start.tolist()
    cap = table.shape[1] * ps
    for b, length in enumerate(lens):
        n = min(max(length, 0), cap)
        new = starts[b + 1] - starts[b]
        if n == 0 or new == 0:
            continue
        k, there = gather(k_pages, table[b], n)
        v, _ = gather(v_pages, table[b], n)
        i = torch.arange(length - new, length, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)[None]
        see = (j <= i) & there[None]
        if window is not None:
            see = see & ((i - j <= window) | (j < prefix))
        some = see.any(1)
        for h in range(Hq):
            rows = slice(starts[b], starts[b + 1])
            qh, kh, vh = q[rows, h].double(), k[:, h // g], v[:, h // g]
            s = (qh @ kh.T * scale).masked_fill(~see, float("-inf"))
            p = torch.softmax(torch.where(some[:, None], s, torch.zeros_like(s)), -1)
            p = torch.where(see, p, torch.zeros_like(p))
            out[rows, h] = p @ vh
            spread[rows, h] = p @ vh.abs()
            ds[rows, h] = (qh.abs() @ kh.abs().T * abs(scale)).masked_fill(~see, 0.0).amax(1)
    return out, spread, ds
