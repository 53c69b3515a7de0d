"""Selected pages of the paged cache: what is measured of the operators.

Five operators let a step over the paged cache run without the host and read
only a part of long sequences:

* ``paged_extend``: block tables and slot maps from request lengths. Each
  sequence's new rows get pages from a stack of free ones, and every row its
  place in the pool and its position.
* ``paged_key_means``: the mean key of each page that the new rows fill.
* ``paged_select``: for every query block and KV head the pages it reads, as
  ascending lists: those of the first ``prefix`` tokens, those that hold a key
  at most ``window`` before one of its queries (its own included), and of the
  others the ``topk`` best by the block's summed queries times the page's mean
  key (sums in 64 bits, rounded to 32; ties to the lower page).
* ``paged_decode_listed`` and ``paged_prefill_listed``: attention of one new
  token per sequence, and of a ragged batch of new rows in query blocks, over
  the listed pages: key j is visible to the query at position i when j <= i and
  its page is listed.

``run`` with ``own`` false computes them with elementary torch operations;
with ``own`` true it calls this repository's kernels.
"""

import bisect
import random

import numpy as np
import torch

own = False

HEAD_DIM = 128
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# (query heads, KV heads): the 1.3B, 6.7B and 33B layers, and one of eight
# tensor-parallel shards of the 33B layer.
HEADS = ((16, 16), (32, 32), (56, 8), (7, 1))
PAGE_SIZES = (16, 32, 64, 128)


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # One decode step of a serving batch: a row for each of 64 sequences.
        dict(name="extend_step", op="extend", batch=64, new_min=1, new_max=1, past_min=0, past_max=16383,
             page_size=64, pad=0, lens_seed=1),
        # Four prompts of odd lengths and the turns of twelve cached ones, 16-row
        # pages, with room for more rows than there are.
        dict(name="extend_prompts", op="extend", batch=16, new_min=0, new_max=8191, past_min=0, past_max=700,
             page_size=16, pad=37, lens_seed=2),
        # The same decode step on the 33B cache: a page in 16 gets full.
        dict(name="means_step", op="means", batch=64, new_min=1, new_max=1, past_min=0, past_max=16383, heads_kv=8,
             page_size=16, dtype="bf16", lens_seed=3),
        # The benched 6.7B prompt: all its pages.
        dict(name="means_prompt", op="means", batch=1, new_min=16384, new_max=16384, past_min=0, past_max=0,
             heads_kv=32, page_size=64, dtype="f16", lens_seed=4),
        # One sequence of the benched 1.3B prompt's decode (latency).
        dict(name="select_one", op="select", batch=1, new_min=1, new_max=1, past_min=12288, past_max=12288,
             heads_q=16, heads_kv=16, page_size=64, block=1, topk=8, window=256, prefix=64, dtype="bf16", pad=0,
             lens_seed=5),
        # A serving batch of the 33B model, lengths from one token to 16K.
        dict(name="select_batch_gqa", op="select", batch=32, new_min=1, new_max=1, past_min=0, past_max=16383,
             heads_q=56, heads_kv=8, page_size=16, block=1, topk=64, window=255, prefix=128, dtype="bf16", pad=0,
             lens_seed=6),
        # The benched 1.3B prompt: blocks of 128 queries, the sink block, a window
        # of four blocks and the top eight.
        dict(name="select_prompt", op="select", batch=1, new_min=12288, new_max=12288, past_min=0, past_max=0,
             heads_q=16, heads_kv=16, page_size=64, block=128, topk=8, window=256, prefix=64, dtype="bf16", pad=0,
             lens_seed=7),
        # The 1.3B decode step over its selected pages.
        dict(name="decode_one", op="decode", batch=1, new_min=1, new_max=1, past_min=12288, past_max=12288,
             heads_q=16, heads_kv=16, page_size=64, block=1, topk=8, window=256, prefix=64, dtype="bf16", pad=0,
             lens_seed=8),
        # The 33B serving batch: 16 pages of 128 rows each beside prefix and window.
        dict(name="decode_batch_gqa", op="decode", batch=64, new_min=1, new_max=1, past_min=0, past_max=16383,
             heads_q=56, heads_kv=8, page_size=128, block=1, topk=16, window=511, prefix=128, dtype="f16", pad=0,
             lens_seed=9),
        # The benched 1.3B prompt over its selected pages.
        dict(name="prefill_prompt", op="prefill", batch=1, new_min=12288, new_max=12288, past_min=0, past_max=0,
             heads_q=16, heads_kv=16, page_size=64, block=128, topk=8, window=256, prefix=64, dtype="bf16", pad=0,
             lens_seed=10),
        # One chunk of a long 33B prompt on what is cached already.
        dict(name="prefill_chunk_gqa", op="prefill", batch=1, new_min=512, new_max=512, past_min=15872,
             past_max=15872, heads_q=56, heads_kv=8, page_size=128, block=16, topk=16, window=512, prefix=128,
             dtype="bf16", pad=0, lens_seed=11),
        # Short continuations of cached contexts (a forked prompt's new turns).
        dict(name="prefill_turns", op="prefill", batch=16, new_min=1, new_max=200, past_min=100, past_max=8000,
             heads_q=32, heads_kv=32, page_size=16, block=64, topk=32, window=200, prefix=128, dtype="f16", pad=19,
             lens_seed=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("extend", "means", "select", "select", "decode", "decode", "prefill", "prefill"))
    heads_q, heads_kv = rng.choice(HEADS)
    case = dict(op=op, page_size=rng.choice(PAGE_SIZES), lens_seed=rng.randrange(1 << 30))
    step = op == "decode" or (op != "prefill" and rng.random() < 0.5)
    if step:
        case.update(batch=_log_int(rng, 1, 64), new_min=1, new_max=1, past_min=0, past_max=_log_int(rng, 1, 16384))
    else:
        hi = _log_int(rng, 1, 8000)
        case.update(batch=_log_int(rng, 1, 16), new_min=_log_int(rng, 1, hi), new_max=hi, past_min=0,
                    past_max=rng.choice((0, 100, 2000, 8000)))
    if op == "extend":
        case.update(pad=rng.choice((0, 0, 13)))
        if not step:
            case["new_min"] = rng.choice((0, case["new_min"]))
        return case
    case.update(heads_kv=heads_kv, dtype=rng.choice(tuple(DTYPES)))
    if op == "means":
        # Some page is filled at least.
        hi = _log_int(rng, case["page_size"], 8000)
        case.update(new_min=_log_int(rng, case["page_size"], hi), new_max=hi, past_max=rng.choice((0, 100, 2000, 8000)))
        while sum(n for n, _ in _lens(case)) * heads_kv > 700000:
            case["batch"] = max(1, case["batch"] // 2)
        return case
    blocks = [b for b in (16, 32, 64, 128) if b * (heads_q // heads_kv) <= 128]
    case.update(heads_q=heads_q, block=1 if step else rng.choice(blocks), topk=_log_int(rng, 1, 64),
                window=rng.choice((0, 64, 255, 1000)), prefix=rng.choice((0, 1, 64, 128, 200)),
                pad=0 if step else rng.choice((0, 0, 13)))
    if op == "select":
        # Long enough that the scores decide: more pages than are read anyway.
        case["past_min"] = case["window"] + case["prefix"] + (case["topk"] + 3) * case["page_size"]
        case["past_max"] = case["past_min"] + case["past_max"]
    most = dict(select="select_batch_gqa" if step else "select_prompt", decode="decode_batch_gqa",
                prefill="prefill_prompt")[op]
    most = work(next(c for c in listed() if c["name"] == most))
    while work(case)["flops"] > most["flops"] or work(case)["bytes"] > most["bytes"]:
        if case["batch"] > 1:
            case["batch"] //= 2
        elif case["new_max"] > 1:
            case["new_max"] //= 2
            case["new_min"] = min(case["new_min"], case["new_max"])
        else:
            case["past_max"] = max(case["past_min"], case["past_max"] // 2)
    return case


def _lens(case):
    """Per sequence: cached length after the call, and its new rows."""
    rng = random.Random(case["lens_seed"])
    out = []
    for _ in range(case["batch"]):
        new = rng.randint(case["new_min"], case["new_max"])
        out.append((rng.randint(case["past_min"], case["past_max"]) + new, new))
    return out


def _blocks(case):
    """(sequence, first row within it, rows, first position) of every query block."""
    out = []
    for b, (n, new) in enumerate(_lens(case)):
        for r in range(0, new, case["block"]):
            out.append((b, r, min(case["block"], new - r), n - new + r))
    return out


def _pages_of(case, i0, i1):
    """Pages that a query block at positions i0 .. i1 reads: (those before its own
    that it always reads, the first of its own, the last of its own)."""
    ps = case["page_size"]
    own0, last = i0 // ps, i1 // ps
    first = max(0, i0 - case["window"]) // ps
    always = own0 - first + min(first, -(-case["prefix"] // ps))
    return always, own0, last


def work(case):
    lens = _lens(case)
    if case["op"] == "extend":
        ps = case["page_size"]
        pages = sum(-(-n // ps) - -(-(n - new) // ps) for n, new in lens)
        # New and old lengths in, lengths and starts out, a page id in and out, a
        # slot and a position for each row.
        return {"bytes": 16 * len(lens) + 8 * pages + 16 * sum(new for _, new in lens), "flops": 0}
    row = HEAD_DIM * 2
    if case["op"] == "means":
        ps = case["page_size"]
        pages = sum(n // ps - (n - new) // ps for n, new in lens)
        return {"bytes": pages * case["heads_kv"] * (ps * row + HEAD_DIM * 4),
                "flops": pages * case["heads_kv"] * ps * HEAD_DIM}
    nbytes = flops = 0
    group = case["heads_q"] // case["heads_kv"]
    seen = {}
    for b, _, rows, pos in _blocks(case):
        always, own0, last = _pages_of(case, pos, pos + rows - 1)
        picked = min(own0, always + case["topk"])  # before its own
        if case["op"] == "select":
            flops += case["heads_q"] * rows * HEAD_DIM + 2 * HEAD_DIM * case["heads_kv"] * (own0 - always)
            nbytes += case["heads_q"] * rows * row + 4 * case["heads_kv"] * (picked + last - own0 + 2)
            seen[b] = max(seen.get(b, 0), own0)
        else:
            keys = rows * picked * case["page_size"]
            keys += sum(i - own0 * case["page_size"] + 1 for i in range(pos, pos + rows))
            flops += 4 * HEAD_DIM * case["heads_kv"] * group * keys
            nbytes += 2 * case["heads_q"] * rows * row
            have = lens[b][0] - 1
            seen[b] = min(have + 1, seen.get(b, 0) + picked * case["page_size"] +
                          min(have, pos + rows - 1) - own0 * case["page_size"] + 1)
    if case["op"] == "select":
        nbytes += sum(seen.values()) * case["heads_kv"] * HEAD_DIM * 4
    else:
        nbytes += sum(seen.values()) * case["heads_kv"] * 2 * row
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed * 7919 + 1)
    lens = _lens(case)
    ps, op = case["page_size"], case["op"]
    cols = max(1, max(-(-n // ps) for n, _ in lens))
    need = sum(-(-n // ps) for n, _ in lens)
    spare = 200 if op == "extend" else 3
    ids = list(range(need + spare))
    rng.shuffle(ids)
    table = torch.full((len(lens), cols), -1, dtype=torch.int32)
    for b, (n, new) in enumerate(lens):
        have = n - new if op == "extend" else n
        for p in range(-(-have // ps)):
            table[b, p] = ids.pop()
    st = dict(case=case, lens=lens, table=table.to(dev))
    starts = [0]
    for _, new in lens:
        starts.append(starts[-1] + new)
    st["starts"] = starts

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    if op == "extend":
        st.update(new=ints([new for _, new in lens]), old=ints([n - new for n, new in lens]),
                  free=ints(ids + [0] * 5), count=ints([len(ids)]), rows=starts[-1] + case["pad"],
                  num_pages=need + spare, lens_out=ints([0] * len(lens)), count_out=ints([0]))
        return st
    st.update(seq_lens=ints([n for n, _ in lens]), q_start=ints(starts))
    dt, hk = DTYPES[case["dtype"]], case["heads_kv"]
    if op == "means":
        st["k_pages"] = torch.randn(need + spare, hk, ps, HEAD_DIM, generator=gen, device=dev, dtype=dt)
        st["means"] = torch.zeros(need + spare, hk, HEAD_DIM, device=dev)
        return st
    if case["block"] == 1:
        st["q_start"] = None
    rows = starts[-1] + case["pad"]
    st["q"] = torch.randn(rows, case["heads_q"], HEAD_DIM, generator=gen, device=dev, dtype=dt)
    if op == "select":
        # Means of rows with unit variance.
        st["means"] = torch.randn(need + spare, hk, HEAD_DIM, generator=gen, device=dev) * ps ** -0.5
        return st
    st["k_pages"] = torch.randn(need + spare, hk, ps, HEAD_DIM, generator=gen, device=dev, dtype=dt)
    st["v_pages"] = torch.randn(need + spare, hk, ps, HEAD_DIM, generator=gen, device=dev, dtype=dt)
    st["out"] = torch.zeros_like(st["q"])
    # The lists that a selection would have made, by random scores.
    width = _width(case, cols)
    blocks = _blocks(case)
    st["lists"] = torch.full((_block_rows(case, rows), hk, width), -1, dtype=torch.int32, device=dev)
    st["counts"] = torch.zeros(st["lists"].shape[0], hk, dtype=torch.int32, device=dev)
    for i in range(0, len(blocks), 64):
        part = blocks[i:i + 64]
        scores = torch.rand(len(part), hk, cols, generator=gen, device=dev)
        lists, counts = _choose(case, part, scores, width)
        st["lists"][i:i + len(part)] = lists
        st["counts"][i:i + len(part)] = counts
    return st


def _width(case, cols):
    """Entries of a list: the most pages that a query block can read."""
    ps = case["page_size"]
    return min(cols, case["topk"] + -(-case["prefix"] // ps) + (case["window"] + case["block"] + ps - 2) // ps + 1)


def _block_rows(case, rows):
    """Query blocks that so many rows of the batch can have at most."""
    k = min(rows, case["batch"])
    return (rows - k) // case["block"] + k


def _choose(case, blocks, scores, width):
    """Lists and counts of some query blocks from their scores [blocks, Hkv, pages]."""
    ps, dev = case["page_size"], scores.device
    pos = torch.tensor([p for _, _, _, p in blocks], device=dev)[:, None, None]
    end = torch.tensor([p + r - 1 for _, _, r, p in blocks], device=dev)[:, None, None]
    page = torch.arange(scores.shape[-1], device=dev)
    there = (page * ps <= end).expand_as(scores)
    always = there & ((page * ps < case["prefix"]) | ((page + 1) * ps > pos - case["window"]))
    key = scores.masked_fill(always, float("inf")).masked_fill(~there, float("-inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    many = (always.sum(-1, keepdim=True) + case["topk"]).minimum(there.sum(-1, keepdim=True))
    picked = torch.zeros_like(there).scatter_(-1, order, torch.arange(scores.shape[-1], device=dev) < many)
    page = torch.where(picked, page, scores.shape[-1]).sort(dim=-1).values[..., :width]
    return (torch.where(page < scores.shape[-1], page, -1).int(), picked.sum(-1).int())


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    return (_own if own else _plain)[op](st)


def _own_extend(st):
    from sabrecoder_b200 import kernels as K
    q_start, slots, positions = K.paged_extend(st["new"], st["table"], st["old"], st["free"], st["count"],
                                               page_size=st["case"]["page_size"], num_pages=st["num_pages"],
                                               num_rows=st["rows"], seq_lens_out=st["lens_out"],
                                               free_count_out=st["count_out"])
    return st["table"], st["lens_out"], st["count_out"], q_start, slots, positions


def _own_means(st):
    from sabrecoder_b200 import kernels as K
    K.paged_key_means(st["k_pages"], st["means"], st["table"], st["seq_lens"], st["q_start"],
                      num_rows=st["starts"][-1])
    return st["means"]


def _own_select(st):
    from sabrecoder_b200 import kernels as K
    c = st["case"]
    return K.paged_select(st["q"], st["means"], st["table"], st["seq_lens"], st["q_start"], page_size=c["page_size"],
                          topk=c["topk"], query_block=c["block"], window_size=c["window"],
                          num_prefix_tokens=c["prefix"])


def _own_decode(st):
    from sabrecoder_b200 import kernels as K
    return K.paged_decode_listed(st["q"], st["k_pages"], st["v_pages"], st["table"], st["seq_lens"], st["lists"],
                                 st["counts"], out=st["out"])


def _own_prefill(st):
    from sabrecoder_b200 import kernels as K
    return K.paged_prefill_listed(st["q"], st["k_pages"], st["v_pages"], st["table"], st["seq_lens"], st["q_start"],
                                  st["lists"], st["counts"], query_block=st["case"]["block"], out=st["out"])


_own = dict(extend=_own_extend, means=_own_means, select=_own_select, decode=_own_decode, prefill=_own_prefill)


def _plain_extend(st):
    ps, dev = st["case"]["page_size"], st["table"].device
    new, old, table = st["new"].long(), st["old"].long(), st["table"]
    zero = torch.zeros(1, dtype=torch.long, device=dev)
    have, want = (old + ps - 1) // ps, (old + new + ps - 1) // ps
    ends = (want - have).cumsum(0)
    column = torch.arange(table.shape[1], device=dev)
    taken = column - have[:, None] + (ends - (want - have))[:, None]
    fresh = st["free"][(st["count"].long() - 1 - taken).clamp(0, st["free"].shape[0] - 1)]
    table.copy_(torch.where((column >= have[:, None]) & (column < want[:, None]), fresh, table))
    st["lens_out"].copy_(old + new)
    st["count_out"].copy_(st["count"] - ends[-1])
    q_start = torch.cat([zero, new.cumsum(0)])
    row = torch.arange(st["rows"], device=dev)
    seq = (row[:, None] >= q_start[None, 1:]).sum(1)
    real = seq < new.shape[0]
    seq = seq.clamp(max=new.shape[0] - 1)
    pos = torch.where(real, old[seq] + row - q_start[seq], 0)
    slots = torch.where(real, table[seq, pos // ps].long() * ps + pos % ps, -1)
    return table, st["lens_out"], st["count_out"], q_start.int(), slots, pos


def _plain_means(st):
    ps = st["case"]["page_size"]
    for b, (n, new) in enumerate(st["lens"]):
        for p0 in range((n - new) // ps, n // ps, 64):
            page = st["table"][b, p0:min(p0 + 64, n // ps)].long()
            st["means"][page] = st["k_pages"][page].float().sum(2) / ps
    return st["means"]


def _plain_select(st):
    c, dev = st["case"], st["q"].device
    hk, cols = c["heads_kv"], st["table"].shape[1]
    width = _width(c, cols)
    q = st["q"].double().view(-1, hk, c["heads_q"] // hk, HEAD_DIM).sum(2)
    blocks = _blocks(c)
    lists = torch.full((_block_rows(c, st["q"].shape[0]), hk, width), -1, dtype=torch.int32, device=dev)
    counts = torch.zeros(lists.shape[:2], dtype=torch.int32, device=dev)
    i = 0
    while i < len(blocks):
        b, j = blocks[i][0], i
        while j < len(blocks) and blocks[j][0] == b and j < i + 64:
            j += 1
        means = st["means"][st["table"][b].clamp(min=0).long()].double()
        sums = torch.stack([q[st["starts"][b] + r:st["starts"][b] + r + m].sum(0) for _, r, m, _ in blocks[i:j]])
        scores = torch.matmul(sums.transpose(0, 1), means.permute(1, 2, 0)).transpose(0, 1).float()
        lists[i:j], counts[i:j] = _choose(c, blocks[i:j], scores, width)
        i = j
    return lists, counts


def _plain_rows(st, i, q, b, pos):
    """Attention of the rows q, at positions pos, pos + 1, ... of sequence b, over list i."""
    c, dev = st["case"], q.device
    ps, hk = c["page_size"], c["heads_kv"]
    entry = st["lists"][i].long()
    page = st["table"][b][entry.clamp(min=0)].long()
    head = torch.arange(hk, device=dev)[:, None]
    keys = st["k_pages"][page, head].float().flatten(1, 2)
    values = st["v_pages"][page, head].float().flatten(1, 2)
    at = (entry[:, :, None] * ps + torch.arange(ps, device=dev)).flatten(1)
    listed_keys = (torch.arange(entry.shape[1], device=dev) < st["counts"][i][:, None])[:, :, None].expand(-1, -1, ps)
    row = torch.arange(pos, pos + q.shape[0], device=dev)
    see = (at[:, None, :] <= row[:, None]) & listed_keys.flatten(1)[:, None]
    g = c["heads_q"] // hk
    qh = q.float().view(-1, hk, g, HEAD_DIM).permute(1, 2, 0, 3).reshape(hk, -1, HEAD_DIM)
    s = torch.matmul(qh, keys.transpose(1, 2)) * HEAD_DIM ** -0.5
    s = s.view(hk, g, q.shape[0], -1).masked_fill_(~see[:, None], float("-inf"))
    p = (s - s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p.view(hk, -1, p.shape[-1]), values).view(hk, g, q.shape[0], HEAD_DIM) / p.sum(-1, keepdim=True)
    return o.permute(2, 0, 1, 3).reshape(q.shape)


def _plain_attend(st):
    for i, (b, r, m, pos) in enumerate(_blocks(st["case"])):
        row = st["starts"][b] + r
        st["out"][row:row + m] = _plain_rows(st, i, st["q"][row:row + m], b, pos).to(st["out"].dtype)
    return st["out"]


_plain = dict(extend=_plain_extend, means=_plain_means, select=_plain_select, decode=_plain_attend,
              prefill=_plain_attend)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return dict(extend=_exact_extend, means=_exact_means, select=_exact_select, decode=_exact_attend,
                prefill=_exact_attend)[case["op"]](case, st)


def _exact_extend(case, st):
    ps = case["page_size"]
    table, free, top = st["table"].tolist(), st["free"].tolist(), int(st["count"])
    starts, slots, positions, lens = [0], [], [], []
    for b, (n, new) in enumerate(st["lens"]):
        for pos in range(n - new, n):
            if pos % ps == 0:
                top -= 1
                table[b][pos // ps] = free[top]
            slots.append(table[b][pos // ps] * ps + pos % ps)
            positions.append(pos)
        lens.append(n)
        starts.append(len(slots))
    extra = st["rows"] - len(slots)
    i32 = torch.int32
    return (torch.tensor(table, dtype=i32), torch.tensor(lens, dtype=i32), torch.tensor([top], dtype=i32),
            torch.tensor(starts, dtype=i32), torch.tensor(slots + [-1] * extra), torch.tensor(positions + [0] * extra))


def _exact_means(case, st):
    ps, out = case["page_size"], st["means"].double()
    table = st["table"].tolist()
    for b, (n, new) in enumerate(st["lens"]):
        filled = [table[b][pos // ps] for pos in range(n - new, n) if pos % ps == ps - 1]
        for page in filled:
            out[page] = st["k_pages"][page].double().mean(1)
    return out


def _exact_select(case, st):
    ps, hk = case["page_size"], case["heads_kv"]
    g = case["heads_q"] // hk
    cols = st["table"].shape[1]
    width = _width(case, cols)
    q = st["q"].double().cpu().numpy()
    means, table = st["means"].cpu().numpy(), st["table"].cpu().numpy()
    shape = (_block_rows(case, q.shape[0]), hk, width)
    lists, counts = np.full(shape, -1, np.int32), np.zeros(shape[:2], np.int32)
    if shape[0] * hk * cols > 4000000:
        return None
    for i, (b, r, m, pos) in enumerate(_blocks(case)):
        row = st["starts"][b] + r
        last = (pos + m - 1) // ps
        low = max(0, pos - case["window"]) // ps
        for h in range(hk):
            total = q[row:row + m, h * g:(h + 1) * g].sum((0, 1))
            rest = [p for p in range(low) if p * ps >= case["prefix"]]
            score = (means[table[b, rest], h].astype(np.float64) @ total).astype(np.float32)
            best = np.lexsort((np.array(rest, np.int64), -score))[:case["topk"]]
            chosen = [rest[x] for x in best]
            for p in range(last + 1):
                if p >= low or p * ps < case["prefix"]:
                    bisect.insort(chosen, p)
            chosen.sort()
            lists[i, h, :len(chosen)] = chosen
            counts[i, h] = len(chosen)
    return torch.from_numpy(lists), torch.from_numpy(counts)


def _exact_attend(case, st):
    q = st["q"].double()
    out = torch.zeros_like(q)
    ps, hk = case["page_size"], case["heads_kv"]
    g = case["heads_q"] // hk
    blocks = _blocks(case)
    if len(blocks) * hk > 8000:
        return None
    lists, counts = st["lists"].cpu(), st["counts"].cpu()
    table = st["table"].cpu()
    for i, (b, r, m, pos) in enumerate(blocks):
        row = st["starts"][b] + r
        for h in range(hk):
            entry = lists[i, h, :int(counts[i, h])].long()
            page = table[b, entry].long().to(q.device)
            k = st["k_pages"][page, h].reshape(-1, HEAD_DIM).double()
            v = st["v_pages"][page, h].reshape(-1, HEAD_DIM).double()
            at = (entry.view(-1, 1) * ps + torch.arange(ps)).view(1, -1).to(q.device)
            hidden = at > torch.arange(pos, pos + m, device=q.device).view(-1, 1)
            logits = torch.einsum("mgd,td->gmt", q[row:row + m, h * g:(h + 1) * g], k) / HEAD_DIM ** 0.5
            weights = torch.softmax(logits.masked_fill(hidden, float("-inf")), -1)
            out[row:row + m, h * g:(h + 1) * g] = torch.einsum("gmt,td->mgd", weights, v)
    return out
