"""The paged key/value cache operators: what is measured of them.

Four operators serve one page pool: ``paged_store`` (new rows into pages),
``paged_decode`` (one new token per sequence over the pages), ``paged_prefill``
(a ragged batch of prompt rows over the pages, causal, with an optional
sliding window and first tokens that stay visible) and ``copy_pages`` (whole
pages for forks and compaction). Key j is visible to the query at position i
when j <= i and (there is no window, or i - j <= window, or j < prefix), and
its page is present.

``run`` with ``own`` false computes them with elementary torch operations in
fp32; with ``own`` true it calls this repository's kernels.
"""

import random

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
        # The 33B cache's store in one decode step of 64 sequences: a row each.
        dict(name="store_step", op="store", batch=64, new_min=1, new_max=1, past_min=0, past_max=16383, heads_kv=8,
             page_size=64, dtype="bf16", pad=0, lens_seed=1),
        # Four 1.3B prompts of odd lengths entering the cache, 16-row pages,
        # in a buffer with padding rows behind the last prompt.
        dict(name="store_prompts", op="store", batch=4, new_min=2500, new_max=8191, past_min=0, past_max=700,
             heads_kv=16, page_size=16, dtype="f16", pad=37, lens_seed=2),
        # One short completion (latency).
        dict(name="decode_short", op="decode", batch=1, len_min=300, len_max=300, heads_q=16, heads_kv=16,
             page_size=16, window=-1, prefix=0, dtype="bf16", lens_seed=3),
        # The benched 1.3B prompt's decode step: one sequence, long axis.
        dict(name="decode_long", op="decode", batch=1, len_min=12289, len_max=12289, heads_q=16, heads_kv=16,
             page_size=64, window=-1, prefix=0, dtype="bf16", lens_seed=4),
        # A serving batch of the 33B model, lengths from one token to 16K.
        dict(name="decode_batch_gqa", op="decode", batch=32, len_min=1, len_max=16384, heads_q=56, heads_kv=8,
             page_size=64, window=-1, prefix=0, dtype="bf16", lens_seed=5),
        # A windowed 6.7B cache that has dropped its middle pages.
        dict(name="decode_window", op="decode", batch=64, len_min=40, len_max=16000, heads_q=32, heads_kv=32,
             page_size=128, window=1023, prefix=128, dtype="f16", lens_seed=6),
        # The benched 1.3B prompt, dense causal.
        dict(name="prefill_prompt", op="prefill", batch=1, new_min=12288, new_max=12288, past_min=0, past_max=0,
             heads_q=16, heads_kv=16, page_size=64, window=-1, prefix=0, dtype="bf16", pad=0, lens_seed=7),
        # One chunk of a long 33B prompt on what is cached already.
        dict(name="prefill_chunk_gqa", op="prefill", batch=1, new_min=512, new_max=512, past_min=15872,
             past_max=15872, heads_q=56, heads_kv=8, page_size=128, window=-1, prefix=0, dtype="bf16", pad=0,
             lens_seed=8),
        # Ragged 6.7B prompts with a sliding window and prefix tokens.
        dict(name="prefill_window", op="prefill", batch=4, new_min=3500, new_max=12001, past_min=0, past_max=0,
             heads_q=32, heads_kv=32, page_size=64, window=1024, prefix=128, dtype="f16", pad=0, lens_seed=9),
        # Short continuations of cached contexts (a forked prompt's new turns).
        dict(name="prefill_turns", op="prefill", batch=16, new_min=1, new_max=200, past_min=100, past_max=8000,
             heads_q=16, heads_kv=16, page_size=16, window=-1, prefix=0, dtype="bf16", pad=19, lens_seed=10),
        # One sequence of the 33B cache forked: its last, part-filled page, all layers.
        dict(name="copy_fork", op="copy", buffers=124, pages=64, moves=1, heads_kv=8, page_size=16, dtype="bf16"),
        # The 1.3B cache compacted: scattered pages to the front, all layers.
        dict(name="copy_compact", op="copy", buffers=48, pages=190, moves=81, heads_kv=16, page_size=64,
             dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("store", "decode", "decode", "prefill", "prefill", "copy"))
    heads_q, heads_kv = rng.choice(HEADS)
    case = dict(op=op, heads_kv=heads_kv, page_size=rng.choice(PAGE_SIZES), dtype=rng.choice(tuple(DTYPES)))
    windowed = rng.random() < 0.4
    window = _log_int(rng, 17, 4000) if windowed else -1
    prefix = rng.choice((0, 1, 64, 128, 200)) if windowed else 0
    if op == "store":
        case.update(batch=_log_int(rng, 1, 64), new_min=1, new_max=_log_int(rng, 1, 1200), past_min=0,
                    past_max=rng.randint(0, 4000), pad=rng.choice((0, 0, 13)), lens_seed=rng.randrange(1 << 30))
    elif op == "decode":
        hi = _log_int(rng, 1, 16384)
        case.update(batch=_log_int(rng, 1, 64), len_min=_log_int(rng, 1, hi), len_max=hi, heads_q=heads_q,
                    window=window, prefix=prefix, lens_seed=rng.randrange(1 << 30))
        while _sum_lengths(case) * heads_kv > 2200000:
            case["batch"] = max(1, case["batch"] // 2)
    elif op == "prefill":
        hi = _log_int(rng, 1, 8000)
        case.update(batch=_log_int(rng, 1, 16), new_min=_log_int(rng, 1, hi), new_max=hi, past_min=0,
                    past_max=rng.choice((0, 100, 2000, 8000)), heads_q=heads_q, window=window, prefix=prefix,
                    pad=rng.choice((0, 0, 13)), lens_seed=rng.randrange(1 << 30))
        limit = work(listed()[6])["flops"]
        while work(case)["flops"] > limit:
            if case["batch"] > 1:
                case["batch"] //= 2
            else:
                case["new_max"] = max(1, case["new_max"] // 2)
                case["new_min"] = min(case["new_min"], case["new_max"])
    else:
        page_bytes = heads_kv * case["page_size"] * HEAD_DIM * 2
        buffers = rng.choice((2, 48, 64, 124))
        most = max(2, min(400, 2000000000 // (page_bytes * buffers)))
        pages = _log_int(rng, 2, most)
        case.update(buffers=buffers, pages=pages, moves=rng.randint(1, max(1, (pages * 2) // 5)))
    return case


def _lens(case):
    """Per sequence: cached length after the call, and its new rows."""
    rng = random.Random(case["lens_seed"])
    out = []
    for _ in range(case["batch"]):
        if case["op"] == "decode":
            out.append((rng.randint(case["len_min"], case["len_max"]), 1))
        else:
            new = rng.randint(case["new_min"], case["new_max"])
            out.append((rng.randint(case["past_min"], case["past_max"]) + new, new))
    return out


def _sum_lengths(case):
    return sum(n for n, _ in _lens(case))


def _visible_sum(n, new, window, prefix):
    """Number of (query, visible key) pairs over the last `new` positions of n."""
    a, b = n - new, n - 1
    edge = b if window < 0 else min(b, window + prefix)  # up to here everything is visible
    total = 0
    if a <= edge:
        total += (edge - a + 1) * (a + edge + 2) // 2
    if edge < b:
        total += (b - max(a, edge + 1) + 1) * (prefix + window + 1)
    return total


def work(case):
    if case["op"] == "copy":
        page = case["heads_kv"] * case["page_size"] * HEAD_DIM * 2
        return {"bytes": 2 * page * case["buffers"] * case["moves"], "flops": 0}
    row = HEAD_DIM * 2
    if case["op"] == "store":
        return {"bytes": 4 * row * case["heads_kv"] * sum(new for _, new in _lens(case)), "flops": 0}
    nbytes = flops = 0
    for n, new in _lens(case):
        pairs = _visible_sum(n, new, case["window"], case["prefix"])
        first = n - new - case["window"] if case["window"] >= 0 else 0
        keys = n if first <= case["prefix"] else case["prefix"] + n - first
        nbytes += 2 * row * case["heads_q"] * new + 2 * row * case["heads_kv"] * keys
        flops += 4 * HEAD_DIM * case["heads_q"] * pairs
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed * 7919 + 1)
    dt = DTYPES[case["dtype"]]
    hk, ps = case["heads_kv"], case["page_size"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dt)

    if case["op"] == "copy":
        pages = torch.empty(case["buffers"], case["pages"], hk, ps, HEAD_DIM, device=dev, dtype=dt)
        for m in range(case["buffers"]):
            pages[m] = randn(case["pages"], hk, ps, HEAD_DIM)
        # Distinct pages: the sources live in the back, the free ones in front.
        order = rng.sample(range(case["pages"]), 2 * case["moves"])
        order.sort()
        free, used = order[:case["moves"]], order[case["moves"]:]
        rng.shuffle(used)
        return dict(case=case, pages=pages, src=used, dst=free)

    lens = _lens(case)
    cap = max((n + ps - 1) // ps for n, _ in lens)
    window, prefix = case.get("window", -1), case.get("prefix", 0)
    rows = []
    need = 0
    for n, new in lens:
        live = [True] * ((n + ps - 1) // ps)
        if window >= 0:
            # Pages that no new row can see have been given back.
            first = n - new - window
            live = [p * ps < prefix or (p + 1) * ps > first for p in range(len(live))]
        rows.append(live)
        need += sum(live)
    ids = list(range(need + 3))
    rng.shuffle(ids)
    table = torch.full((len(lens), cap), -1, dtype=torch.int32)
    for b, live in enumerate(rows):
        for p, keep in enumerate(live):
            if keep:
                table[b, p] = ids.pop()
    st = dict(case=case, lens=lens, table=table.to(dev),
              seq_lens=torch.tensor([n for n, _ in lens], dtype=torch.int32, device=dev),
              k_pages=randn(need + 3, hk, ps, HEAD_DIM), v_pages=randn(need + 3, hk, ps, HEAD_DIM))
    if case["op"] == "decode":
        st["q"] = randn(len(lens), case["heads_q"], HEAD_DIM)
        return st
    starts = [0]
    for _, new in lens:
        starts.append(starts[-1] + new)
    st["starts"] = starts
    st["q_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    total = starts[-1] + case["pad"]
    if case["op"] == "store":
        # As a projection leaves them: one row holds the heads of a token.
        st["k"], st["v"] = randn(total, hk, HEAD_DIM), randn(total, hk, HEAD_DIM)
    else:
        st["q"] = randn(total, case["heads_q"], HEAD_DIM)
        st["out"] = torch.zeros_like(st["q"])
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    return (_own if own else _plain)[op](st)


def _window_args(case):
    return dict(window_size=None if case["window"] < 0 else case["window"], num_prefix_tokens=case["prefix"])


def _own_store(st):
    from sabrecoder_b200 import kernels as K
    K.paged_store(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["seq_lens"], st["q_start"])
    return st["k_pages"], st["v_pages"]


def _own_decode(st):
    from sabrecoder_b200 import kernels as K
    return K.paged_decode(st["q"], st["k_pages"], st["v_pages"], st["table"], st["seq_lens"],
                          **_window_args(st["case"]))


def _own_prefill(st):
    from sabrecoder_b200 import kernels as K
    return K.paged_prefill(st["q"], st["k_pages"], st["v_pages"], st["table"], st["seq_lens"], st["q_start"],
                           out=st["out"], **_window_args(st["case"]))


def _own_copy(st):
    from sabrecoder_b200 import kernels as K
    K.copy_pages(st["pages"], st["src"], st["dst"])
    return st["pages"]


_own = dict(store=_own_store, decode=_own_decode, prefill=_own_prefill, copy=_own_copy)


def _plain_copy(st):
    dev = st["pages"].device
    src, dst = torch.tensor(st["src"], device=dev), torch.tensor(st["dst"], device=dev)
    st["pages"][:, dst] = st["pages"][:, src]
    return st["pages"]


def _plain_store(st):
    ps = st["case"]["page_size"]
    n = st["starts"][-1]
    row = torch.arange(n, device=st["k"].device)
    seq = (row[:, None] >= st["q_start"][None, 1:]).sum(1)
    pos = st["seq_lens"][seq] - st["q_start"][seq + 1] + row
    page = st["table"][seq, pos // ps].long()
    st["k_pages"][page, :, pos % ps] = st["k"][:n]
    st["v_pages"][page, :, pos % ps] = st["v"][:n]
    return st["k_pages"], st["v_pages"]


def _plain_attend(q, keys, values, visible):
    """q [R, Hq, D], keys / values [T, Hkv, D] in fp32, visible [R, T]."""
    g = q.shape[1] // keys.shape[1]
    qh = q.view(q.shape[0], keys.shape[1], g, HEAD_DIM).permute(1, 2, 0, 3).reshape(keys.shape[1], -1, HEAD_DIM)
    s = torch.matmul(qh, keys.permute(1, 2, 0)) * HEAD_DIM ** -0.5
    s = s.view(keys.shape[1], g, q.shape[0], -1).masked_fill_(~visible, float("-inf"))
    p = (s - s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p.view(keys.shape[1], -1, p.shape[-1]), values.transpose(0, 1))
    o = o.view(keys.shape[1], g, q.shape[0], HEAD_DIM) / p.sum(-1, keepdim=True)
    return o.permute(2, 0, 1, 3).reshape(q.shape)


def _plain_rows(st, b, q, first):
    """Attention of the rows q, at positions first, first + 1, ... of sequence b."""
    ps, window, prefix = (st["case"][k] for k in ("page_size", "window", "prefix"))
    dev = q.device
    last = first + q.shape[0] - 1
    lo = max(0, first - window) if window >= 0 else 0
    keep = min(prefix, lo)
    key = torch.cat([torch.arange(keep, device=dev), torch.arange(lo, last + 1, device=dev)])
    page = st["table"][b, key // ps].long()
    keys, values = st["k_pages"][page, :, key % ps].float(), st["v_pages"][page, :, key % ps].float()
    pos = torch.arange(first, last + 1, device=dev)[:, None]
    visible = key[None] <= pos
    if window >= 0:
        visible &= (pos - key[None] <= window) | (key[None] < prefix)
    return _plain_attend(q.float(), keys, values, visible)


def _plain_decode(st):
    out = torch.empty_like(st["q"])
    for b, (n, _) in enumerate(st["lens"]):
        out[b] = _plain_rows(st, b, st["q"][b:b + 1], n - 1)[0].to(out.dtype)
    return out


def _plain_prefill(st):
    out = st["out"]
    for b, (n, new) in enumerate(st["lens"]):
        r0 = st["starts"][b]
        for r in range(0, new, 1024):
            m = min(1024, new - r)
            out[r0 + r:r0 + r + m] = _plain_rows(st, b, st["q"][r0 + r:r0 + r + m], n - new + r).to(out.dtype)
    return out


_plain = dict(store=_plain_store, decode=_plain_decode, prefill=_plain_prefill, copy=_plain_copy)


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] in ("store", "copy"):
        return None  # rows are moved, nothing is computed
    st = prepare(case, seed)
    q = st["q"].double()
    out = torch.zeros_like(q)
    ps, hk = case["page_size"], case["heads_kv"]
    g = case["heads_q"] // hk
    row = 0
    for b, (n, new) in enumerate(st["lens"]):
        pages = st["table"][b, :(n + ps - 1) // ps].long()
        held = (pages >= 0).repeat_interleave(ps)[:n]
        step = max(1, min(new, 100000000 // n))
        for h in range(hk):
            k = st["k_pages"][pages.clamp(min=0), h].reshape(-1, HEAD_DIM)[:n].double()
            v = st["v_pages"][pages.clamp(min=0), h].reshape(-1, HEAD_DIM)[:n].double()
            for r in range(0, new, step):
                m = min(step, new - r)
                i = (torch.arange(m, device=q.device) + (n - new + r)).view(-1, 1)
                j = torch.arange(n, device=q.device).view(1, -1)
                see = (j <= i) & held
                if case["window"] >= 0:
                    see = see & ((i - j <= case["window"]) | (j < case["prefix"]))
                bias = torch.zeros(m, n, dtype=torch.float64, device=q.device)
                bias[~see] = float("-inf")
                for head in range(h * g, (h + 1) * g):
                    logits = q[row + r:row + r + m, head] @ k.T / HEAD_DIM ** 0.5 + bias
                    out[row + r:row + r + m, head] = torch.softmax(logits, -1) @ v
        row += new
    return out
