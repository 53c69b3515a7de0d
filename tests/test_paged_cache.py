"""Host logic of SabrePagedKVCache on the CPU: the two kernels it calls are
replaced by plain loops."""

import random

import pytest
import torch

from oracle import paged_oracle as PO
from sabrecoder_b200 import paged_cache as PC

H, D = 2, 8


@pytest.fixture(autouse=True)
def plain_kernels(monkeypatch):
    def copy_pages(pages, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        pages[..., dst, :, :, :] = pages[..., src, :, :, :]

    def paged_store(k, v, kp, vp, table, lens, starts=None):
        for r, page, off in PO.slots(table, lens, starts, kp.shape[2], kp.shape[0]):
            kp[page, :, off], vp[page, :, off] = k[r], v[r]

    monkeypatch.setattr(PC.K, "copy_pages", copy_pages)
    monkeypatch.setattr(PC.K, "paged_store", paged_store)


def cache(**kw):
    a = dict(batch_size=3, max_seq_len=200, page_size=16, num_layers=2, num_kv_heads=H, head_dim=D, device="cpu",
             dtype=torch.float32)
    a.update(kw)
    return PC.SabrePagedKVCache(**a)


class Mirror:
    """Every sequence's rows as plain lists; checks the cache against them."""

    def __init__(self, c):
        self.c, self.rows, self.next = c, [[] for _ in range(c.batch_size)], 0

    def add(self, new):
        c = self.c
        c.extend(new)
        fresh = []
        for b, n in enumerate(new):
            vals = [self.next + i for i in range(n)]
            self.next += n
            self.rows[b] += vals
            fresh += vals
        starts = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
        rows = torch.tensor(fresh, dtype=torch.float32).view(-1, 1, 1).expand(-1, H, D)
        for i, layer in enumerate(c.layers):
            PC.K.paged_store(rows + 1000 * i, -rows - 1000 * i, layer.k_pages, layer.v_pages, c.page_table, c.seq_lens,
                             starts)

    def check(self):
        c = self.c
        assert c.lengths == [len(r) for r in self.rows] == c.seq_lens.tolist()
        seen = {}
        for b, table in enumerate(c.tables):
            assert c.page_table[b].tolist() == table + [-1] * (c.max_pages - len(table))
            for p in table:
                if p >= 0:
                    seen[p] = seen.get(p, 0) + 1
        assert [seen.get(p, 0) for p in range(c.num_pages)] == c.refs
        assert sorted(c.unused) == [p for p in range(c.num_pages) if p not in seen]
        for i, layer in enumerate(c.layers):
            for b, want in enumerate(self.rows):
                k, there = PO.gather(layer.k_pages, c.page_table[b], len(want))
                v, _ = PO.gather(layer.v_pages, c.page_table[b], len(want))
                n = len(want)
                must = torch.ones(n, dtype=torch.bool)
                if c.window_size is not None and n:  # what the last query sees
                    j = torch.arange(n)
                    must = (n - 1 - j <= c.window_size) | (j < c.num_prefix_tokens)
                assert there[must].all()
                full = torch.tensor(want, dtype=torch.float64) + 1000 * i
                assert torch.equal(k[there][:, 0, 0], full[there]) and torch.equal(v[there][:, 0, 0], -full[there])


def test_extend_fork_copy_on_write_and_compact():
    c = cache(num_pages=20)
    m = Mirror(c)
    m.add([40, 16, 0])
    m.check()
    assert c.pages_in_use == 4
    c.fork(0, 2)
    m.rows[2] = list(m.rows[0])
    m.check()
    assert c.pages_in_use == 4  # shared
    m.add([1, 1, 2])  # both 0 and 2 write the shared page: one of them gets a copy
    m.check()
    assert c.pages_in_use == 6 and c.tables[0][:2] == c.tables[2][:2] and c.tables[0][2] != c.tables[2][2]
    c.free(0)
    m.rows[0] = []
    m.check()
    c.compact()
    m.check()
    assert all(c.refs[p] for p in range(c.pages_in_use))
    c.truncate(2, 17)
    m.rows[2] = m.rows[2][:17]
    m.check()
    m.add([200, 3, 4])
    m.check()
    c.reset()
    m.rows = [[], [], []]
    m.check()
    assert c.pages_in_use == 0


def test_full_pool_and_full_sequence_change_nothing():
    c = cache(num_pages=5)
    m = Mirror(c)
    m.add([30, 30, 0])
    with pytest.raises(ValueError, match="out of pages"):
        c.extend([0, 3, 17])
    m.check()
    with pytest.raises(ValueError, match="full"):
        c.extend([171, 0, 0])
    m.check()
    c.fork(0, 2)
    m.rows[2] = list(m.rows[0])
    m.add([0, 2, 1])  # the copy on write takes the last page
    m.check()
    with pytest.raises(ValueError, match="out of pages"):
        c.extend([3, 0, 0])
    m.check()
    with pytest.raises(ValueError, match="counts"):
        c.extend([1, 1])
    with pytest.raises(ValueError, match="counts"):
        c.extend([1, -1, 0])


@pytest.mark.parametrize("window,prefix", [(20, 0), (0, 0), (33, 5), (16, 32), (15, 16)])
def test_window_drops_pages_nobody_will_see(window, prefix):
    c = cache(window_size=window, num_prefix_tokens=prefix, max_seq_len=2000, num_pages=30)
    m = Mirror(c)
    for n in [7, 30, 1, 1, 1, 16, 50] + [1] * 40:
        m.add([n, n // 2, 0])
        m.check()
    keep = -(-prefix // 16) + (window + 1 + 15) // 16 + 1
    assert sum(p >= 0 for p in c.tables[0]) <= keep
    with pytest.raises(ValueError, match="dropped already"):
        c.truncate(0, 60)
    m.check()
    c.fork(0, 2)
    m.rows[2] = list(m.rows[0])
    m.add([1, 0, 20])
    m.check()


@pytest.mark.parametrize("seed,window", [(0, None), (1, None), (2, 25), (3, 70)])
def test_random_use(seed, window):
    rng = random.Random(seed)
    c = cache(batch_size=4, max_seq_len=600, num_pages=40, window_size=window, num_prefix_tokens=10 if window else 0)
    m = Mirror(c)
    full = 0
    for _ in range(150):
        op = rng.choice(("add", "add", "add", "fork", "truncate", "free", "compact", "select"))
        try:
            if op == "add":
                m.add([rng.choice((0, 1, 1, 5, 40)) for _ in range(4)])
            elif op == "fork":
                a, b = rng.randrange(4), rng.randrange(4)
                c.fork(a, b)
                m.rows[b] = list(m.rows[a])
            elif op == "truncate":
                b = rng.randrange(4)
                n = rng.randint(0, len(m.rows[b]))
                c.truncate(b, n)
                m.rows[b] = m.rows[b][:n]
            elif op == "free" and rng.random() < 0.5:
                b = rng.randrange(4)
                c.free(b)
                m.rows[b] = []
            elif op == "compact":
                c.compact()
                assert all(c.refs[p] for p in range(c.pages_in_use))
            elif op == "select":
                idx = [rng.randrange(4) for _ in range(4)]
                c.reorder_cache(torch.tensor(idx))
                m.rows = [list(m.rows[i]) for i in idx]
        except ValueError:
            full += 1
        m.check()
    assert full < 100


def test_transformers_protocol():
    c = cache(batch_size=2)
    assert c.get_seq_length() == 0 and c.get_mask_sizes(5, 0) == (5, 0) and c.max_cache_len == 200
    assert c.max_batch_size == 2 and not any(c.is_sliding)
    k = torch.randn(2, H, 20, D)
    kk, vv = c.update(k, k + 1, 0)
    assert torch.equal(kk, k) and torch.equal(vv, k + 1)
    assert c.get_seq_length(0) == 20 and c.get_seq_length(1) == 0
    with pytest.raises(ValueError, match="out of step"):
        c.update(k[:, :, :3], k[:, :, :3], 1)
    c.update(k, k, 1)
    assert c.get_seq_length(1) == 20
    c.update(k[:, :, :1], k[:, :, :1], 0)
    kk, _ = c.update(k[:, :, :1], k[:, :, :1], 1)
    assert kk.shape == (2, H, 21, D) and torch.equal(kk[:, :, 20:], k[:, :, :1])
    c.batch_repeat_interleave(2)
    assert c.batch_size == 4 and c.page_table.shape[0] == 4 and c.tables[0] == c.tables[1]
    c.crop(-1)
    assert c.lengths == [20] * 4
    with pytest.raises(ValueError, match="sequences"):
        c.update(k, k, 0)
    with pytest.raises(ValueError, match="patched attention"):
        cache(window_size=4).update(k, k, 0)


def test_a_step_cut_off_by_an_error_and_a_reset():
    c = cache(batch_size=1)
    k = torch.randn(1, H, 5, D)
    c.update(k, k, 0)  # layer 1 never gets there
    c.reset()
    for i in (0, 1):
        kk, _ = c.update(k, k, i)
        assert torch.equal(kk, k)


def test_deepcopy_is_a_cache_of_its_own():
    import copy
    c = cache(num_pages=20)
    m = Mirror(c)
    m.add([40, 16, 0])
    c.fork(0, 2)
    m.rows[2] = list(m.rows[0])
    d = copy.deepcopy(c)
    n = Mirror(d)
    n.rows, n.next = [list(r) for r in m.rows], m.next
    m.add([1, 2, 3])
    n.check()
    n.add([7, 0, 7])
    m.check()
    n.check()
    assert d.layers[0]._cache is d and d.layers[0].k_pages.data_ptr() != c.layers[0].k_pages.data_ptr()


@pytest.mark.parametrize("kw", [dict(page_size=24), dict(page_size=8), dict(batch_size=0), dict(max_seq_len=0),
                                dict(num_pages=0), dict(window_size=-1), dict(num_prefix_tokens=-1),
                                dict(num_layers=None)])
def test_constructor_refusals(kw):
    with pytest.raises(ValueError):
        cache(**kw)


def test_the_pool_goes_with_the_cache():
    import gc
    import weakref
    gc.disable()
    try:
        c = cache()
        ref = weakref.ref(c)
        del c
        assert ref() is None
    finally:
        gc.enable()


def test_row_starts_stay_where_a_captured_call_found_them(monkeypatch):
    """A captured prefill keeps the address of its row starts: they are the same
    tensor after any number of other row counts, and those first asked for inside
    a capture (whose fill only runs on replay) are not handed to eager calls."""
    c = cache(batch_size=2)
    first = c._row_starts(5)
    for n in range(1, 150):
        assert c._row_starts(n).tolist() == [0, n, 2 * n]
    assert c._row_starts(5) is first
    capturing = True
    monkeypatch.setattr(PC, "_capturing", lambda pool: capturing, raising=False)
    inside = c._row_starts(170)
    assert c._row_starts(5) is first
    capturing = False
    assert c._row_starts(170) is not inside and c._row_starts(170) is c._row_starts(170)


def test_sequences_of_different_lengths_in_a_model():
    """Attention that does not read pages cannot tell the rows a shorter sequence
    does not have; the patched one needs every sequence's own positions."""
    c = cache(batch_size=2)
    k = torch.randn(2, H, 20, D)
    for i in (0, 1):
        c.update(k, k, i)
    c.check_step(0, 3, torch.arange(20, 23)[None])
    c.truncate(1, 10)
    with pytest.raises(ValueError, match="different lengths"):
        c.update(k[:, :, :1], k[:, :, :1], 0)
    assert c.lengths == [20, 10]
    for ids in (None, torch.tensor([[20, 21]]), torch.tensor([[20, 21], [20, 21]]), torch.tensor([[20], [10]])):
        with pytest.raises(ValueError, match="position_ids"):
            c.check_step(0, 2, ids)
    own = torch.tensor([[20, 21], [10, 11]])
    c.check_step(0, 2, own)
    c.append(0, k[:, :, :2].transpose(1, 2), k[:, :, :2].transpose(1, 2))
    c.check_step(1, 2, own)  # the same step: nothing new to check
    c.append(1, k[:, :, :2].transpose(1, 2), k[:, :, :2].transpose(1, 2))
    assert c.lengths == [22, 12]


def test_masks_that_say_more_than_the_cache_are_refused():
    """Attention over pages is causal within the cache's window: a mask that hides
    more, shows more or adds a bias would be dropped without a word."""
    lo = torch.finfo(torch.float32).min

    def causal(B=2, n=4, T=24, window=None):
        i, j = torch.arange(T - n, T)[:, None], torch.arange(T)[None]
        see = (j <= i) & (i - j <= (T if window is None else window))
        return see.expand(B, 1, n, T).clone()

    c = cache(batch_size=2)
    k = torch.randn(2, H, 20, D)
    for i in (0, 1):
        c.update(k, k, i)
    ids = torch.arange(20, 24)[None]
    good = causal()
    left, right, future, bias = good.clone(), good.clone(), good.clone(), torch.where(good, 0.0, lo)
    left[1, :, :, :3] = False
    right[0, :, :, 22:] = False
    future[:, :, 0] = True
    assert (bias == 0).any()
    bias[0, 0, 2, 5] = -0.5
    pad = torch.ones(2, 24, dtype=torch.long)
    pad[1, :3] = 0

    def added(see):
        return torch.where(see, 0.0, lo)

    for ok in (None, good, good[:1], added(good), added(good).expand(2, H, 4, 24), torch.ones(2, 24, dtype=torch.long),
               torch.nn.functional.pad(good, (0, 8))):
        c.check_step(0, 4, ids, ok)
    for wrong in (left, right, future, bias, added(left), added(future), pad, pad.bool(), causal(window=10),
                  good[..., :20], good[0, 0], good[:, 0]):
        with pytest.raises(ValueError, match="mask"):
            c.check_step(0, 4, ids, wrong)
    w = cache(batch_size=2, window_size=10)
    for i in (0, 1):
        w.append(i, k.transpose(1, 2), k.transpose(1, 2))
    for ok in (good, causal(window=10), added(causal(window=15))):
        w.check_step(0, 4, ids, ok)
    for wrong in (left & causal(window=2), causal(window=9)):
        with pytest.raises(ValueError, match="mask"):
            w.check_step(0, 4, ids, wrong)
    # Each sequence's own rows and positions, the mask of the longest.
    c.truncate(1, 10)
    own = torch.tensor([[20, 21, 22, 23], [10, 11, 12, 13]])
    c.check_step(0, 4, own, good)
    short = good.clone()
    short[1, :, :, 14:] = False
    c.check_step(0, 4, own, short)
    short[1, :, :, 13:] = False
    with pytest.raises(ValueError, match="mask"):
        c.check_step(0, 4, own, short)


def test_attention_is_planned_by_the_rows_that_are_there(monkeypatch):
    """The prompt kernel plans its work by the table's width: eager calls pass the
    columns in use, captured ones the whole table, which may fill by the replay."""
    seen, capturing = [], False
    monkeypatch.setattr(PC, "_capturing", lambda pool: capturing)
    monkeypatch.setattr(PC.K, "paged_prefill", lambda q, kp, vp, table, *a, **kw: seen.append(table) or q)
    c = cache(batch_size=2, max_seq_len=1000)

    def width():
        seen.clear()
        c.prefill(0, torch.zeros(c.batch_size, 1, 4, D))
        t, = seen
        assert t.data_ptr() == c.page_table.data_ptr() and t.stride() == c.page_table.stride()
        assert t.shape[0] == c.batch_size
        return t.shape[1]

    assert width() == 1
    c.extend([16, 3])
    assert width() == 1
    c.extend([1, 1])
    assert width() == 2
    capturing = True
    assert width() == 63
    capturing = False
    c.extend([200, 300])
    assert width() == 19
    c.batch_select_indices([0])
    assert width() == 14
    c.truncate(0, 0)
    assert width() == 1


def test_crop_takes_the_last_rows_of_every_sequence():
    c = cache(num_pages=30)
    m = Mirror(c)
    m.add([40, 7, 90])
    c.crop(-10)
    m.rows = [r[:max(0, len(r) - 10)] for r in m.rows]
    assert c.lengths == [30, 0, 80]
    m.check()
    c.crop(50)
    m.rows = [r[:50] for r in m.rows]
    m.check()
    c.crop(0)
    assert c.lengths == [0, 0, 0] and c.pages_in_use == 0


@pytest.mark.parametrize("call", [lambda c: c.batch_select_indices([0, 3]),
                                  lambda c: c.reorder_cache(torch.tensor([1, 7, 0])),
                                  lambda c: c.batch_select_indices([-4, 0]), lambda c: c.batch_select_indices([]),
                                  lambda c: c.batch_repeat_interleave(0), lambda c: c.fork(0, 3),
                                  lambda c: c.fork(-4, 1),
                                  lambda c: c.truncate(3, 0), lambda c: c.free(5)])
def test_sequences_that_are_not_there_change_nothing(call):
    c = cache(num_pages=20)
    m = Mirror(c)
    m.add([40, 16, 5])
    c.fork(0, 2)
    m.rows[2] = list(m.rows[0])
    with pytest.raises((ValueError, IndexError), match="sequence"):
        call(c)
    m.check()
    m.add([1, 2, 3])
    m.check()


def test_refused_rows_leave_the_step_undone(monkeypatch):
    """Rows that the store would refuse do not make room: the same step can be given
    again."""
    c = cache(batch_size=2, num_pages=20)
    m = Mirror(c)
    m.add([10, 3, 0][:2])
    k = torch.randn(2, 4, H, D)
    for kk, vv in ((k[:, :, :1], k[:, :, :1]), (k, k[:, :3]), (k.double(), k.double()), (k[..., :4], k[..., :4]),
                   (k, k.double()), (k[:1], k[:1]), (k.to("meta"), k.to("meta"))):
        with pytest.raises(ValueError, match="SabrePagedKVCache"):
            c.append(0, kk, vv)
        m.check()
        assert (c.step, c.layers[0].step) == (0, 0)
    c.append(0, k, -k)
    c.append(1, k, -k)
    assert c.lengths == [14, 7]
    c.append(0, k, k)
    monkeypatch.setattr(PC.K, "paged_store", lambda *a: (_ for _ in ()).throw(RuntimeError("refused")))
    with pytest.raises(RuntimeError, match="refused"):
        c.append(1, k, k)
    monkeypatch.undo()
    assert c.lengths == [18, 11] and (c.step, c.layers[1].step) == (2, 1)


def test_a_step_without_rows():
    c = cache(batch_size=2)
    k = torch.randn(2, 3, H, D)
    for n in (3, 0, 1):
        for i in (0, 1):
            c.append(i, k[:, :n], k[:, :n])
    assert c._row_starts(0).tolist() == [0, 0, 0] and c.lengths == [4, 4]


@pytest.mark.parametrize("call", [lambda c: c.extend([1, 1, 1]), lambda c: c.fork(0, 1), lambda c: c.truncate(0, 3),
                                  lambda c: c.compact(), lambda c: c.reorder_cache(torch.tensor([1, 0, 2])),
                                  lambda c: c.crop(2), lambda c: c.reset(),
                                  lambda c: c.append(0, torch.zeros(3, 1, H, D), torch.zeros(3, 1, H, D))])
def test_the_host_state_does_not_change_inside_a_capture(monkeypatch, call):
    """Inside a capture the device's tables and lengths are only recorded: the host's
    would run ahead of them, and every replay would move them once more."""
    c = cache(num_pages=20)
    m = Mirror(c)
    m.add([40, 16, 5])
    c.free(1)
    m.rows[1] = []
    monkeypatch.setattr(PC, "_capturing", lambda pool: True)
    with pytest.raises(ValueError, match="capture"):
        call(c)
    m.check()
    assert c.step == 0


def test_masks_that_are_not_tensors_are_refused():
    c = cache(batch_size=2)
    with pytest.raises(ValueError, match="mask"):
        c.check_step(0, 4, None, {"full_attention": None})
