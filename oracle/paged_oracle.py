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


# ---------------------------------------------------------------------------
# block tables from lengths, and attention over selected pages
# ---------------------------------------------------------------------------

def extend(new, table, lens, free, count, page_size: int, num_pages: int, rows: int, max_len: Optional[int] = None):
    """(fits, table, lens, count, starts, slots, positions) as lists; all arguments
    lists too. Where it does not fit, everything is as before and no row has a place.
    max_len: rows that a sequence may have, beside what its table row holds."""
    table, lens = [list(t) for t in table], list(lens)
    need = [-(-(n + m) // page_size) - -(-n // page_size) if n >= 0 and m >= 0 else 0 for n, m in zip(lens, new)]
    fits = all(n >= 0 and m >= 0 and n + m <= len(t) * page_size for n, m, t in zip(lens, new, table))
    fits = fits and 0 <= count <= len(free) and sum(need) <= count and sum(new) <= rows
    fits = fits and (max_len is None or all(n + m <= max_len for n, m in zip(lens, new)))
    starts, slots, positions = [0], [], []
    for b, m in enumerate(new if fits else [0] * len(new)):
        for pos in range(lens[b], lens[b] + m):
            if pos % page_size == 0:
                count -= 1
                table[b][pos // page_size] = free[count] if 0 <= free[count] < num_pages else -1
            page = table[b][pos // page_size]
            slots.append(page * page_size + pos % page_size if 0 <= page < num_pages else -1)
            positions.append(pos)
        lens[b] += m if fits else 0
        starts.append(len(slots))
    pad = rows - len(slots)
    return fits, table, lens, count, starts, slots + [-1] * pad, positions + [0] * pad


def key_means(k_pages, table, seq_lens, q_start=None):
    """{page: mean [Hkv, D] in 64 bits} of the pages that the new rows fill."""
    P, ps = k_pages.shape[0], k_pages.shape[2]
    tab, lens = table.tolist(), seq_lens.tolist()
    starts = list(range(len(lens) + 1)) if q_start is None else q_start.tolist()
    out = {}
    for b, n in enumerate(lens):
        new, n = starts[b + 1] - starts[b], min(max(n, 0), len(tab[b]) * ps)
        for p in range(max(0, min(lens[b] - new, n)) // ps, n // ps):
            if 0 <= tab[b][p] < P:
                out[tab[b][p]] = k_pages[tab[b][p]].double().mean(1)
    return out


def query_blocks(seq_lens, q_start, block: int):
    """(sequence, first row, rows, first position) of every query block."""
    lens = seq_lens.tolist()
    starts = list(range(len(lens) + 1)) if q_start is None else q_start.tolist()
    out = []
    for b, n in enumerate(lens):
        for r in range(starts[b], starts[b + 1], block):
            m = min(block, starts[b + 1] - r)
            out.append((b, r, m, n - (starts[b + 1] - r)))
    return out


def select(q, means, table, seq_lens, q_start=None, *, page_size: int, topk: int, block: int = 1, window: int = 0,
           prefix: int = 0):
    """Per query block and KV head the ascending list of columns it reads."""
    P, Hkv, D = means.shape
    g = q.shape[1] // Hkv
    tab = table.tolist()
    cap = table.shape[1] * page_size
    out = []
    for b, r, m, pos in query_blocks(seq_lens, q_start, block):
        n = max(0, min(int(seq_lens[b]), cap, pos + m))
        there = [p for p in range(-(-n // page_size)) if 0 <= tab[b][p] < P]
        low = max(0, max(pos, 0) - window) // page_size
        always = [p for p in there if p >= low or p * page_size < prefix]
        rest = [p for p in there if p not in set(always)]
        lists = []
        for h in range(Hkv):
            qs = q[r:r + m, h * g:(h + 1) * g].double().sum((0, 1))
            score = (means[[tab[b][p] for p in rest], h].double() @ qs).float().tolist() if rest else []
            order = sorted(range(len(rest)), key=lambda i: (score[i] != score[i], -score[i] if score[i] == score[i]
                                                            else 0.0, rest[i]))
            lists.append(sorted(always + [rest[i] for i in order[:topk]]))
        out.append(lists)
    return out


def listed_attention(q, k_pages, v_pages, table, seq_lens, lists, counts, q_start=None, *, block: int = 1,
                     scale: Optional[float] = None):
    """As :func:`attention`, each block seeing the rows j <= i of its listed columns."""
    N, Hq, D = q.shape
    P, Hkv, ps, _ = k_pages.shape
    g = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(N, Hq, D, dtype=torch.float64, device=q.device)
    spread, ds = torch.zeros_like(out), torch.zeros(N, Hq, dtype=torch.float64, device=q.device)
    cols = table.shape[1]
    lists, counts = lists.tolist(), counts.tolist()
    for i, (b, r, m, pos) in enumerate(query_blocks(seq_lens, q_start, block)):
        n = min(max(int(seq_lens[b]), 0), cols * ps)
        if n == 0:
            continue
        keys, there = gather(k_pages, table[b], n)
        values, _ = gather(v_pages, table[b], n)
        for h in range(Hkv):
            mine = lists[i][h][:max(0, min(counts[i][h], len(lists[i][h])))]
            use = [c for x, c in enumerate(mine) if 0 <= c < cols and (x == 0 or mine[x - 1] < c)]
            at = torch.tensor([c * ps + x for c in use for x in range(ps) if c * ps + x < n], dtype=torch.long,
                              device=q.device)
            see = (at[None] <= torch.arange(pos, pos + m, device=q.device)[:, None]) & there[at][None]
            some = see.any(1)
            k, v = keys[at, h], values[at, h]
            for head in range(h * g, (h + 1) * g):
                qh = q[r:r + m, head].double()
                s = (qh @ k.T * scale).masked_fill(~see, float("-inf"))
                p = torch.softmax(torch.where(some[:, None], s, torch.zeros_like(s)), -1)
                p = torch.where(see, p, torch.zeros_like(p))
                out[r:r + m, head] = p @ v
                spread[r:r + m, head] = p @ v.abs()
                if at.numel():
                    ds[r:r + m, head] = (qh.abs() @ k.abs().T * abs(scale)).masked_fill(~see, 0.0).amax(1)
    return out, spread, ds
