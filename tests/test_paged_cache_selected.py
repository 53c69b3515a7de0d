"""Host logic of SabrePagedKVCache with selected pages and with pages lent to the
device, on the CPU: the kernels it calls are replaced by the oracle's loops."""

import copy
import random

import pytest
import torch

from oracle import paged_oracle as PO
from sabrecoder_b200 import paged_cache as PC

H, D, PS = 2, 8, 16


@pytest.fixture(autouse=True)
def plain_kernels(monkeypatch):
    def copy_pages(pages, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst) and pages.dim() >= 4
        pages[..., dst, :, :, :] = pages[..., src, :, :, :]

    def store(k, v, kp, vp, table, lens, starts=None):
        for r, page, off in PO.slots(table, lens, starts, kp.shape[2], kp.shape[0]):
            kp[page, :, off], vp[page, :, off] = k[r], v[r]

    def store_slots(k, v, kp, vp, slots):
        for r, s in enumerate(slots.tolist()):
            if s >= 0:
                kp[s // PS, :, s % PS], vp[s // PS, :, s % PS] = k[r], v[r]

    def extend(new, table, lens, free, count, *, page_size, num_pages, num_rows):
        _, t, n, c, starts, slots, pos = PO.extend(new.tolist(), table.tolist(), lens.tolist(), free.tolist(), int(count),
                                                   page_size, num_pages, num_rows)
        table.copy_(torch.tensor(t))
        lens.copy_(torch.tensor(n))
        count.fill_(c)
        return torch.tensor(starts, dtype=torch.int32), torch.tensor(slots), torch.tensor(pos)

    def key_means(kp, means, table, lens, starts=None, *, num_rows=None):
        assert starts is None or int(starts[-1]) <= num_rows
        for page, m in PO.key_means(kp, table, lens, starts).items():
            means[page] = m

    def select(q, means, table, lens, starts=None, *, page_size, topk, query_block=1, window_size=0,
               num_prefix_tokens=0):
        rows = PO.select(q, means, table, lens, starts, page_size=page_size, topk=topk, block=query_block,
                         window=window_size, prefix=num_prefix_tokens)
        width = max((len(x) for r in rows for x in r), default=1)
        lists = torch.tensor([[x + [-1] * (width - len(x)) for x in r] for r in rows], dtype=torch.int32)
        return lists, torch.tensor([[len(x) for x in r] for r in rows], dtype=torch.int32)

    def listed(q, kp, vp, table, lens, *args, query_block=1, softmax_scale=None, out=None):
        starts = args[0] if len(args) == 3 else None
        return PO.listed_attention(q, kp, vp, table, lens, *args[-2:], starts, block=query_block, scale=softmax_scale)[0]

    for name, fn in dict(copy_pages=copy_pages, paged_store=store, paged_store_slots=store_slots, paged_extend=extend,
                         paged_key_means=key_means, paged_select=select, paged_decode_listed=listed,
                         paged_prefill_listed=listed).items():
        monkeypatch.setattr(PC.K, name, fn)


def cache(**kw):
    a = dict(batch_size=3, max_seq_len=400, page_size=PS, num_layers=2, num_kv_heads=H, head_dim=D, device="cpu",
             dtype=torch.float32)
    a.update(kw)
    c = PC.SabrePagedKVCache(**a)
    c.pool.fill_(float("nan"))
    if c.key_means is not None:
        c.key_means.fill_(float("nan"))
    return c


def consistent(c, rows=None):
    """Tables, references and free pages agree, and the device's copies with them."""
    seen = {}
    for b, table in enumerate(c.tables):
        assert c.page_table[b].tolist() == c._host[b].tolist() == table + [-1] * (c.max_pages - len(table))
        assert len(table) == -(-c.lengths[b] // PS)
        for p in table:
            if p >= 0:
                seen[p] = seen.get(p, 0) + 1
    assert [seen.get(p, 0) for p in range(c.num_pages)] == c.refs
    assert sorted(c.unused) == [p for p in range(c.num_pages) if p not in seen]
    assert c.seq_lens.tolist() == c.lengths
    if c.key_means is not None:  # of every full page
        for layer in c.layers:
            for b, table in enumerate(c.tables):
                for p in range(c.lengths[b] // PS):
                    if table[p] >= 0:
                        assert torch.allclose(layer.key_means[table[p]], layer.k_pages[table[p]].mean(1), atol=1e-6)


def add(c, new, gen):
    n = max(new)
    if len(set(new)) == 1:
        for i in range(2):
            c.append(i, *torch.randn(2, c.batch_size, n, H, D, generator=gen))
        return
    c.extend(new)
    starts = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
    for i, layer in enumerate(c.layers):
        k, v = torch.randn(2, sum(new), H, D, generator=gen)
        PC.K.paged_store(k, v, layer.k_pages, layer.v_pages, c.page_table, c.seq_lens, starts)
        if layer.key_means is not None:
            PC.K.paged_key_means(layer.k_pages, layer.key_means, c.page_table, c.seq_lens, starts, num_rows=sum(new))


@pytest.mark.parametrize("window,prefix", [(None, 0), (20, 17)])
def test_means_follow_their_pages(window, prefix):
    """Forks, copies on write, truncations, compaction and a copy of the cache; no page
    is dropped although there is a window."""
    gen = torch.Generator().manual_seed(1)
    c = cache(topk_pages=2, window_size=window, num_prefix_tokens=prefix)
    add(c, [150, 150, 150], gen)
    consistent(c)
    c.fork(0, 2)
    add(c, [1, 1, 1], gen)
    consistent(c)
    c.truncate(0, 90)
    c.free(1)
    add(c, [30, 5, 64], gen)
    consistent(c)
    assert c.compact() > 0
    consistent(c)
    d = copy.deepcopy(c)
    consistent(d)
    add(d, [16, 0, 3], gen)
    consistent(d)
    consistent(c)
    assert all(p >= 0 for t in c.tables for p in t)


def test_decode_and_prompts_over_selected_pages():
    gen = torch.Generator().manual_seed(2)
    c = cache(topk_pages=2, window_size=10, num_prefix_tokens=5, query_block=8)
    add(c, [170, 170, 170], gen)
    c.truncate(1, 60)
    add(c, [20, 20, 20], gen)
    q = torch.randn(3, 20, 2 * H, D, generator=gen)
    assert c.block_rows(2 * H) == 8 and c.block_rows(64 * H) == 2
    got = c.prefill(1, q)
    starts = torch.tensor([0, 20, 40, 60], dtype=torch.int32)
    layer = c.layers[1]
    args = (layer.key_means, c.page_table, c.seq_lens)
    lists, counts = PC.K.paged_select(q.reshape(60, 2 * H, D), *args, starts, page_size=PS, topk=2, query_block=8,
                                      window_size=10, num_prefix_tokens=5)
    want = PO.listed_attention(q.reshape(60, 2 * H, D), layer.k_pages, layer.v_pages, c.page_table, c.seq_lens, lists,
                               counts, starts, block=8)[0]
    assert torch.equal(got.reshape(60, 2 * H, D), want)
    lists, counts = c.select(0, q[:, 0])
    # The page of the prefix, the one that holds positions 179 to 189, and two.
    assert counts[0].tolist() == [4] * H and lists.shape[:2] == (3, H)
    assert torch.isfinite(c.decode(0, q[:, 0])).all()


@pytest.mark.parametrize("kw", [dict(topk_pages=-1), dict(query_block=8), dict(topk_pages=3, query_block=0),
                                dict(topk_pages=3, query_block=129), dict(topk_pages=3, max_seq_len=32769 * PS,
                                                                          num_pages=4)])
def test_constructor_refusals(kw):
    with pytest.raises(ValueError):
        cache(**kw)


def test_selection_needs_topk_pages_and_gathering_refuses_it():
    c = cache()
    with pytest.raises(ValueError, match="topk_pages"):
        c.select(0, torch.zeros(3, H, D))
    c = cache(topk_pages=1)
    with pytest.raises(ValueError, match="topk_pages"):
        c.layers[0].update(torch.zeros(3, H, 1, D), torch.zeros(3, H, 1, D))


def test_a_mask_must_show_all_keys_with_selected_pages():
    c = cache(topk_pages=1, window_size=3)
    add(c, [40, 40, 40], torch.Generator().manual_seed(3))
    mask = torch.ones(3, 41)
    c.check_step(0, 1, None, mask)
    mask[:, 2] = 0  # outside the window, but a page there may be selected
    with pytest.raises(ValueError, match="mask"):
        c.check_step(0, 1, None, mask)


# -- pages lent to the device ---------------------------------------------

@pytest.mark.parametrize("seed,topk", [(0, None), (1, 2), (2, None), (3, 2)])
def test_random_steps_on_the_device(seed, topk):
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    c = cache(topk_pages=topk, num_pages=60)
    rows = [torch.zeros(0, H, D) for _ in range(3)]

    def check_rows():
        for b in range(3):
            k, there = PO.gather(c.layers[1].k_pages, c.page_table[b], len(rows[b]))
            assert there.all() and torch.equal(k, rows[b].double())

    for _ in range(12):
        op = rng.choice(("lend", "fork", "truncate", "compact"))
        if op == "fork":
            a, b = rng.sample(range(3), 2)
            c.fork(a, b)
            rows[b] = rows[a]
        elif op == "truncate":
            b = rng.randrange(3)
            n = rng.randint(0, c.lengths[b])
            c.truncate(b, n)
            rows[b] = rows[b][:n]
        elif op == "compact":
            c.compact()
        else:
            n = c.lend(rng.choice((None, len(c.unused) // 2)))
            assert int(c.free_count) == n
            for _ in range(rng.randint(0, 4)):
                new = [rng.choice((0, 1, 1, 17)) for _ in range(3)]
                before = c.seq_lens.clone()
                num = sum(new) + rng.randint(0, 3)
                q_start, slots, pos = c.extend_on_device(torch.tensor(new, dtype=torch.int32), num)
                k = torch.randn(num, H, D, generator=gen)
                for i in range(2):
                    c.store_rows(i, k, -k, q_start, slots)
                if torch.equal(before, c.seq_lens):
                    assert (slots == -1).all()
                    continue
                for b in range(3):
                    mine = slice(int(q_start[b]), int(q_start[b + 1]))
                    assert pos[mine].tolist() == list(range(len(rows[b]), len(rows[b]) + new[b]))
                    rows[b] = torch.cat([rows[b], k[mine]])
            c.settle()
        consistent(c)
        check_rows()
    assert c.lengths == [len(r) for r in rows]


def test_shared_last_pages_are_copied_before_pages_are_lent():
    gen = torch.Generator().manual_seed(4)
    c = cache(num_pages=8)
    add(c, [20, 0, 0], gen)
    c.fork(0, 1)
    c.fork(0, 2)
    assert c.pages_in_use == 2
    with pytest.raises(ValueError, match="cannot be lent"):
        c.lend(5)  # six are free, two go to the copies
    assert c.pages_in_use == 2
    assert c.lend() == 4
    assert len({t[1] for t in c.tables}) == 3 and len({t[0] for t in c.tables}) == 1
    c.settle()
    consistent(c)
    k, _ = PO.gather(c.layers[0].k_pages, c.page_table[2], 20)
    assert torch.equal(k, PO.gather(c.layers[0].k_pages, c.page_table[0], 20)[0])


@pytest.mark.parametrize("call", [lambda c: c.extend([1, 1, 1]), lambda c: c.fork(0, 1), lambda c: c.truncate(0, 3),
                                  lambda c: c.free(0), lambda c: c.compact(), lambda c: c.crop(2), lambda c: c.reset(),
                                  lambda c: c.batch_select_indices([0]), lambda c: copy.deepcopy(c), lambda c: c.lend(),
                                  lambda c: c.append(0, torch.zeros(3, 1, H, D), torch.zeros(3, 1, H, D))])
def test_sequences_are_the_devices_while_pages_are_lent(call):
    c = cache()
    add(c, [20, 20, 20], torch.Generator().manual_seed(5))
    c.lend(3)
    tables = [list(t) for t in c.tables]
    with pytest.raises(ValueError, match="settle"):
        call(c)
    assert c.tables == tables and c.lengths == [20] * 3
    c.settle()
    consistent(c)
    c.settle()  # nothing lent, nothing done
    consistent(c)


def test_settling_refuses_tables_that_do_not_match():
    c = cache()
    c.lend(5)
    c.extend_on_device(torch.tensor([20, 0, 1], dtype=torch.int32), 21)
    good = c.page_table.clone()
    c.page_table[0, 1] = c.page_table[0, 0]
    with pytest.raises(ValueError, match="do not match"):
        c.settle()
    c.page_table.copy_(good)
    c.settle()
    consistent(c)
    assert c.lengths == [20, 0, 1]
    with pytest.raises(ValueError, match="lend"):
        c.extend_on_device(torch.tensor([1, 1, 1], dtype=torch.int32), 3)


def test_a_step_after_settling_changes_nothing():
    """A graph of an earlier loan, replayed: also where a row fits into a last page."""
    c = cache()
    one = torch.ones(3, dtype=torch.int32)
    c.lend()
    c.extend_on_device(one, 3)
    c.settle()
    _, slots, _ = PC.K.paged_extend(one, c.page_table, c.seq_lens, c.free_pages, c.free_count, page_size=PS,
                                    num_pages=c.num_pages, num_rows=3)
    assert (slots == -1).all() and c.lengths == [1, 1, 1]
    consistent(c)


def test_lending_inside_a_capture_is_refused(monkeypatch):
    c = cache()
    monkeypatch.setattr(PC, "_capturing", lambda pool: True)
    with pytest.raises(ValueError, match="capture"):
        c.lend()
    with pytest.raises(ValueError, match="capture"):
        c.settle()


def test_steps_on_the_device_read_the_whole_table():
    c = cache(topk_pages=1)
    add(c, [20, 20, 20], torch.Generator().manual_seed(6))
    assert c._columns_in_use().shape[1] == 2
    c.lend()
    assert c._columns_in_use() is c.page_table
    c.settle()
    assert c._columns_in_use().shape[1] == 2
