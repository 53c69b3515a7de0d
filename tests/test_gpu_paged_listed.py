"""GPU tests of block tables built from lengths, mean keys, page selection and
attention over listed pages, against the 64-bit oracle. Every row of a pool that
no sequence owns holds NaN, so a read of one shows."""

import random

import pytest
import torch

from oracle import paged_oracle as PO
from test_gpu_paged import BF, D, FP, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from sabrecoder_b200 import kernels
    return kernels


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------
# tables and slots
# ---------------------------------------------------------------------------

EXTEND = [
    # old lengths, new rows, page_size, extra rows, extra free pages, extra columns
    ([0], [1], 16, 0, 0, 0),
    ([0], [0], 16, 0, 0, 1),
    ([0], [0], 16, 7, 3, 1),
    ([15, 16, 17, 0, 31], [1, 1, 1, 1, 1], 16, 0, 0, 0),
    ([15, 16, 17, 0, 31], [1, 0, 15, 16, 33], 16, 5, 2, 1),
    ([100, 0, 3000, 64], [900, 0, 77, 0], 64, 13, 1, 0),
    ([0, 5], [8191, 2500], 16, 3, 10, 2),
    ([1023, 1024, 1], [1, 1, 1023], 1024, 0, 0, 0),
    ([(37 * i) % 300 for i in range(600)], [(i * i) % 4 for i in range(600)], 32, 9, 5, 1),
    ([(11 * i) % 40 for i in range(1500)], [1] * 1500, 16, 0, 0, 0),
    ([0] * 3, [40000, 1, 30000], 128, 1, 1, 1),
    ([i % 33 for i in range(16384)], [i % 2 for i in range(16384)], 16, 3, 1, 0),
    ([0, 0, 7, 0], [0, 2049, 0, 0], 16, 0, 0, 0),
]


def extend_state(case, ps, extra_rows, extra_free, extra_cols, seed):
    old, new = case
    rng = random.Random(seed)
    cols = max(1, max(-(-(n + m) // ps) for n, m in zip(old, new))) + extra_cols
    held = sum(-(-n // ps) for n in old)
    need = sum(-(-(n + m) // ps) - -(-n // ps) for n, m in zip(old, new))
    pool = held + need + extra_free + 2
    ids = list(range(pool))
    rng.shuffle(ids)
    table = [[ids.pop() if p < -(-n // ps) else -1 for p in range(cols)] for n in old]
    free = ids[:need + extra_free]
    return table, free + [0, 0, 0], len(free), pool, sum(new) + extra_rows


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", range(len(EXTEND)))
def test_extend_vs_oracle(K, case, in_place):
    old, new, ps, extra_rows, extra_free, extra_cols = EXTEND[case]
    table, free, count, pool, rows = extend_state((old, new), ps, extra_rows, extra_free, extra_cols, case)
    fits, *want = PO.extend(new, table, old, free, count, ps, pool, rows)
    assert fits
    t, lens, cnt = i32(table), i32(old), i32([count])
    lens_out, cnt_out = (None, None) if in_place else (i32([7] * len(old)), i32([7]))
    starts, slots, positions = K.paged_extend(i32(new), t, lens, i32(free), cnt, page_size=ps, num_pages=pool,
                                              num_rows=rows, seq_lens_out=lens_out, free_count_out=cnt_out)
    got = (t, lens if in_place else lens_out, cnt if in_place else cnt_out, starts, slots, positions)
    for g, w in zip(got, ([*want[:2], [want[2]], *want[3:]])):
        assert g.tolist() == w
    if not in_place:
        assert lens.tolist() == old and cnt.tolist() == [count]
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("why", ["pages", "columns", "rows", "length", "new", "count", "count_low"])
@pytest.mark.parametrize("rows_extra", [0, 5000])
def test_extend_that_does_not_fit_changes_nothing(K, why, rows_extra):
    old, new, ps = [20, 0, 64], [30, 16, 1], 16
    table, free, count, pool, rows = extend_state((old, new), ps, 2 + rows_extra, 0, 0, 3)
    table = [t + [-1] for t in table]
    if why == "pages":
        count -= 1
    elif why == "columns":
        new[0] = 6 * 16 - 20 + 1
        free, count = list(range(40)), 40
        rows = 200
    elif why == "rows":
        rows = sum(new) - 1
    elif why == "length":
        old[1] = -3
    elif why == "new":
        new[2] = -1
    elif why == "count":
        count = len(free) + 1
    else:
        count = -1
    t, lens, cnt = i32(table), i32(old), i32([count])
    starts, slots, positions = K.paged_extend(i32(new), t, lens, i32(free), cnt, page_size=ps, num_pages=pool,
                                              num_rows=rows)
    assert (t.tolist(), lens.tolist(), cnt.tolist()) == (table, old, [count])
    assert (starts == 0).all() and (slots == -1).all() and (positions == 0).all()
    assert K.device_status(clear=True) == 8


def test_extend_with_pages_outside_the_pool(K):
    """A free page that is none and a last page that is absent: their rows have no
    place, the others have theirs."""
    table, free = [[-1, -1, -1], [2, -1, -1]], [1, 99, 0]
    want = PO.extend([20, 20], table, [5, 5], free, 3, 16, 4, 45)
    t, lens, cnt = i32(table), i32([5, 5]), i32([3])
    starts, slots, positions = K.paged_extend(i32([20, 20]), t, lens, i32(free), cnt, page_size=16, num_pages=4,
                                              num_rows=45)
    assert want[0] and t.tolist() == want[1] and slots.tolist() == want[5] and positions.tolist() == want[6]
    assert starts.tolist() == [0, 20, 40] and cnt.tolist() == [1]
    assert K.device_status(clear=True) == 4


def test_extend_on_a_table_slice_of_another_stream(K):
    """A table that is a slice of a wider one, on a stream of its own."""
    wide = torch.full((3, 20), -5, dtype=torch.int32, device="cuda")
    wide[:, 4:10] = -1
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _, slots, _ = K.paged_extend(i32([17, 1, 90]), wide[:, 4:10], i32([0, 0, 0]), i32(list(range(20))),
                                     i32([20]), page_size=16, num_pages=20, num_rows=108)
    stream.synchronize()
    want = PO.extend([17, 1, 90], [[-1] * 6] * 3, [0] * 3, list(range(20)), 20, 16, 20, 108)
    assert wide[:, 4:10].tolist() == want[1] and slots.tolist() == want[5]
    assert (wide[:, :4] == -5).all() and (wide[:, 10:] == -5).all()


# ---------------------------------------------------------------------------
# store by slots
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("Hkv,ps,dtype", [(1, 16, BF), (2, 64, FP), (8, 32, BF), (16, 128, FP)])
def test_store_by_slots_is_the_store_by_tables(K, Hkv, ps, dtype):
    lens, news = [300, 0, 77, 130], [200, 0, 77, 1]
    q, kp, vp, table, sl, starts = make(3, lens, news, Hkv, Hkv, ps, dtype)
    n = int(starts[-1])
    rows = torch.randn(n + 3, 2 * Hkv, D, device="cuda").to(dtype)
    k, v = rows[:, :Hkv], rows[:, Hkv:]
    slots = torch.full((n + 3,), -1, dtype=torch.int64)
    for r, page, off in PO.slots(table, sl, starts, ps, kp.shape[0]):
        slots[r] = page * ps + off
    ka, va, kb, vb = kp.clone(), vp.clone(), kp.clone(), vp.clone()
    K.paged_store(k, v, ka, va, table, sl, starts)
    K.paged_store_slots(k, v, kb, vb, slots.cuda())
    for a, b in ((ka, kb), (va, vb)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    assert K.device_status(clear=True) == 0
    slots[5] = kp.shape[0] * ps  # past the pool
    slots[6] = 2 ** 40
    before = kb.clone()
    K.paged_store_slots(k[5:7], v[5:7], kb, vb, slots[5:7].cuda())
    assert torch.equal(kb.view(torch.int16), before.view(torch.int16)) and K.device_status(clear=True) == 4


# ---------------------------------------------------------------------------
# mean keys
# ---------------------------------------------------------------------------

MEANS = [
    # lens, news, Hkv, page_size, dtype, layout
    ([16], [1], 1, 16, BF, "phtd"),
    ([15, 16, 17, 0, 32, 64], [1, 1, 1, 0, 1, 1], 3, 16, FP, "phtd"),
    ([1000, 5, 64, 300], [900, 5, 64, 0], 8, 64, BF, "ptkhd"),
    ([2100, 1024], [2100, 1], 9, 1024, FP, "phtd"),
    ([4000], [4000], 32, 32, BF, "phtd"),
    (list(range(100)), [i % 3 for i in range(100)], 2, 16, BF, "phtd"),
]


def check_means(got, before, want):
    """fp32 sums of up to 1024 values in at most 513 additions of rounded partial
    sums: each 2^-24 of the sum of magnitudes, which is at most page_size times
    the largest; the scaling by a power of two is exact."""
    for page in range(got.shape[0]):
        if page in want:
            mean, size = want[page]
            tol = 514 * 2.0 ** -24 * size
            assert ((got[page].double() - mean).abs() <= tol).all()
        else:
            assert torch.equal(got[page], before[page])


@pytest.mark.parametrize("case", range(len(MEANS)))
@pytest.mark.parametrize("strided", [False, True])
def test_key_means_vs_oracle(K, case, strided):
    lens, news, Hkv, ps, dtype, layout = MEANS[case]
    _, kp, _, table, sl, starts = make(40 + case, lens, news, Hkv, Hkv, ps, dtype, layout=layout)
    if strided:
        means = torch.full((Hkv, kp.shape[0], 2 * D), 7.0, device="cuda")[:, :, D:].transpose(0, 1)
    else:
        means = torch.full((kp.shape[0], Hkv, D), 7.0, device="cuda")
    before = means.clone()
    K.paged_key_means(kp, means, table, sl, starts, num_rows=int(starts[-1]) + 3 * case)
    want = {p: (m, kp[p].double().abs().mean(1)) for p, m in PO.key_means(kp, table, sl, starts).items()}
    check_means(means, before, want)
    assert K.device_status(clear=True) == 0


def test_key_means_one_row_each_and_odd_lengths(K):
    _, kp, _, table, sl, _ = make(50, [32, 31, 16, 1], [1] * 4, 2, 2, 16, BF)
    means = torch.full((kp.shape[0], 2, D), 7.0, device="cuda")
    before = means.clone()
    K.paged_key_means(kp, means, table, sl)
    want = {p: (m, kp[p].double().abs().mean(1)) for p, m in PO.key_means(kp, table, sl).items()}
    assert len(want) == 2
    check_means(means, before, want)
    # Lengths past the table, negative ones and absent pages: nothing to fill.
    means.copy_(before)
    table[2] = -1
    sl.copy_(i32([2 ** 31 - 1, -2 ** 31, 16, 0]))
    K.paged_key_means(kp, means, table, sl)
    assert torch.equal(means, before) and K.device_status(clear=True) == 0


# ---------------------------------------------------------------------------
# selection
# ---------------------------------------------------------------------------

SELECT = [
    # lens, news, Hq, Hkv, page_size, dtype, block, topk, window, prefix
    ([1], [1], 1, 1, 16, BF, 1, 4, 0, 0),
    ([700], [1], 16, 16, 16, BF, 1, 8, 100, 33),
    ([700, 0, 63, 64, 65, 3000], [1] * 6, 4, 2, 64, FP, 1, 5, 0, 1),
    ([700, 0, 63, 64, 65, 3000], [1] * 6, 4, 2, 16, FP, 1, 0, 70, 40),
    ([5000, 2], [1, 1], 7, 1, 32, BF, 1, 64, 255, 128),
    ([5000, 900], [1, 1], 56, 8, 16, BF, 1, 1, 0, 0),
    ([9000], [1], 2, 1, 16, FP, 1, 40, 17, 5),
    ([1500, 40, 700], [1200, 40, 3], 4, 4, 64, BF, 128, 3, 128, 64),
    ([1500, 0, 700], [1200, 0, 300], 7, 1, 16, FP, 16, 30, 40, 20),
    ([2500], [77], 8, 1, 1024, BF, 16, 1, 0, 0),
    ([900, 1300], [900, 200], 6, 2, 32, BF, 33, 4, 1000, 5000),
    ([600] * 40, [i % 5 for i in range(40)], 2, 2, 16, BF, 2, 3, 16, 16),
    ([3000, 260], [2049, 260], 2, 2, 32, BF, 64, 12, 31, 0),
    # Enough blocks that groups of four share the means they read.
    ([3000, 0, 777, 2500], [2900, 0, 700, 2500], 16, 16, 16, BF, 16, 6, 30, 20),
    ([2600, 5, 900], [2600, 2, 800], 56, 8, 32, FP, 5, 9, 0, 0),
    ([2600], [2600], 16, 2, 16, BF, 3, 200, 100, 64),
    ([7 * i % 90 + 150 for i in range(200)], [i % 7 for i in range(200)], 4, 4, 16, BF, 2, 2, 16, 16),
    ([20000], [1300], 4, 4, 16, FP, 4, 700, 0, 0),
    ([4000, 900], [3000, 900], 32, 32, 1024, BF, 128, 1, 0, 0),
]


@pytest.mark.parametrize("lens,news,Hq,Hkv", [([900, 0, 30, 500], [200, 0, 30, 1], 8, 8), ([700], [600], 56, 8)])
def test_select_for_each_row_of_a_prompt(K, lens, news, Hq, Hkv):
    """Blocks of one row, alone and in groups."""
    q, kp, _, table, sl, starts = make(83, lens, news, Hq, Hkv, 16, BF)
    means = torch.randn(kp.shape[0], Hkv, D, device="cuda")
    kw = dict(page_size=16, topk=4, window_size=20, num_prefix_tokens=16)
    lists, counts = K.paged_select(q, means, table, sl, starts, query_block=1, **kw)
    check_lists(lists, counts, PO.select(q, means, table, sl, starts, page_size=16, topk=4, block=1, window=20, prefix=16))


def lists_of(lists, counts):
    return [[lists[i, h, :int(counts[i, h])].tolist() for h in range(lists.shape[1])] for i in range(lists.shape[0])]


def check_lists(lists, counts, want):
    got = lists_of(lists.cpu(), counts.cpu())
    assert got[:len(want)] == want
    assert (counts[len(want):] == 0).all()
    past = torch.arange(lists.shape[2], device=lists.device) >= counts[:, :, None]
    assert (lists[past] == -1).all()


@pytest.mark.parametrize("case", range(len(SELECT)))
def test_select_vs_oracle(K, case):
    lens, news, Hq, Hkv, ps, dtype, block, topk, window, prefix = SELECT[case]
    q, kp, _, table, sl, starts = make(60 + case, lens, news, Hq, Hkv, ps, dtype)
    means = torch.randn(kp.shape[0], Hkv, D, device="cuda")
    kw = dict(page_size=ps, topk=topk)
    pad = torch.full((3, Hq, D), float("nan"), dtype=dtype, device="cuda")
    qs = starts if block > 1 else None
    qq = torch.cat([q, pad]) if block > 1 else q
    lists, counts = K.paged_select(qq, means, table, sl, qs, query_block=block, window_size=window,
                                   num_prefix_tokens=prefix, **kw)
    want = PO.select(q, means, table, sl, qs, block=block, window=window, prefix=prefix, **kw)
    check_lists(lists, counts, want)
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("lens,news,Hq,Hkv,block,topk", [
    ([2000, 900], [1900, 700], 16, 16, 16, 5), ([2000, 900], [1900, 700], 16, 16, 16, 60), ([3000], [1], 4, 2, 1, 40),
    ([3000, 2000], [40, 30], 8, 1, 16, 7)])
def test_select_among_many_equal_scores(K, lens, news, Hq, Hkv, block, topk):
    """Queries and means of small whole numbers: scores are exact and many are equal."""
    q, kp, _, table, sl, starts = make(79, lens, news, Hq, Hkv, 16, BF)
    gen = torch.Generator(device="cuda").manual_seed(7)
    q = torch.randint(-1, 2, q.shape, generator=gen, device="cuda").to(BF)
    means = torch.randint(-1, 2, (kp.shape[0], Hkv, D), generator=gen, device="cuda").float()
    means[..., 8:] = 0
    starts = starts if block > 1 else None
    lists, counts = K.paged_select(q, means, table, sl, starts, page_size=16, topk=topk, query_block=block)
    check_lists(lists, counts, PO.select(q, means, table, sl, starts, page_size=16, topk=topk, block=block))


@pytest.mark.parametrize("lens,news,Hkv,block", [([2000, 900], [1900, 700], 16, 16), ([2000, 900], [2, 3], 2, 1)])
def test_select_with_odd_values_in_queries_and_means(K, lens, news, Hkv, block):
    """NaN, infinities and numbers at the ends of their ranges, in some queries and pages."""
    q, kp, _, table, sl, starts = make(78, lens, news, Hkv, Hkv, 16, BF)
    gen = torch.Generator(device="cuda").manual_seed(8)
    means = torch.randn(kp.shape[0], Hkv, D, generator=gen, device="cuda")
    for x, bad in ((means, float("nan")), (means, float("inf")), (means, -float("inf")), (means, 3e38), (means, 1e-44),
                   (q, float("nan")), (q, float("inf")), (q, 3e38), (q, -1e-38)):
        for _ in range(3):
            i, h, d = (int(torch.randint(0, n, (1,), generator=gen, device="cuda")) for n in x.shape)
            x[i, h, d] = bad
    lists, counts = K.paged_select(q, means, table, sl, starts, page_size=16, topk=9, query_block=block)
    check_lists(lists, counts, PO.select(q, means, table, sl, starts, page_size=16, topk=9, block=block))


def test_select_scores_that_only_64_bits_tell_apart(K):
    """Means that differ in their last bit, and queries whose sum cancels."""
    q, kp, _, table, sl, starts = make(77, [3000, 3000], [64, 64], 4, 4, 16, BF)
    gen = torch.Generator(device="cuda").manual_seed(9)
    q[1::2] = -q[::2]
    q[::16, :, :4] += 0.0625
    base = torch.randn(4, D, generator=gen, device="cuda")
    ulp = torch.randint(-3, 4, (kp.shape[0], 4, D), generator=gen, device="cuda").float() * 2.0 ** -24
    means = base * (1 + ulp)
    for block, starts_ in ((16, starts), (64, starts)):
        lists, counts = K.paged_select(q, means, table, sl, starts_, page_size=16, topk=20, query_block=block)
        check_lists(lists, counts, PO.select(q, means, table, sl, starts_, page_size=16, topk=20, block=block))


def test_select_equal_scores_and_odd_ones(K):
    """Ties go to the earlier page; infinities order as numbers, NaN last."""
    q, kp, _, table, sl, _ = make(80, [1000], [1], 2, 2, 16, BF)
    means = torch.zeros(kp.shape[0], 2, D, device="cuda")
    page = table[0].long()
    for topk in (1, 3, 30, 60, 100):
        lists, counts = K.paged_select(q, means, table, sl, page_size=16, topk=topk)
        assert lists_of(lists, counts)[0] == [list(range(min(topk, 62))) + [62]] * 2
    q.fill_(1.0)
    means[page[7], 0] = -0.0
    means[page[9], 0, 0] = float("inf")
    means[page[11], 0, 0] = -float("inf")
    means[page[0], 0, 5] = float("nan")
    means[page[20], 1, 127] = -1e-30
    means[page[61], 1, 64] = 1e-30
    want = PO.select(q, means, table, sl, page_size=16, topk=1)
    for topk in (1, 2, 8, 59, 60, 61, 62):
        lists, counts = K.paged_select(q, means, table, sl, page_size=16, topk=topk)
        want = PO.select(q, means, table, sl, page_size=16, topk=topk)
        check_lists(lists, counts, want)
    assert 9 in want[0][0] and 0 in want[0][0]
    lists, counts = K.paged_select(q, means, table, sl, page_size=16, topk=61)
    assert 0 not in lists_of(lists, counts)[0][0] and 11 in lists_of(lists, counts)[0][0]


def test_select_leaves_absent_pages_out(K):
    q, kp, _, table, sl, starts = make(81, [900, 500], [300, 20], 6, 2, 32, BF, extra_cols=4)
    means = torch.randn(kp.shape[0], 2, D, device="cuda")
    table[0, 0] = table[0, 5] = table[0, 28] = table[1, 3] = -1  # a prefix page, others, an own one
    kw = dict(page_size=32, topk=4)
    lists, counts = K.paged_select(q, means, table, sl, starts, query_block=32, window_size=40, num_prefix_tokens=33,
                                   **kw)
    check_lists(lists, counts, PO.select(q, means, table, sl, starts, block=32, window=40, prefix=33, **kw))
    assert K.device_status(clear=True) == 0
    table[1, 4] = kp.shape[0]
    lists, counts = K.paged_select(q, means, table, sl, starts, query_block=32, window_size=40, num_prefix_tokens=33,
                                   **kw)
    check_lists(lists, counts, PO.select(q, means, table, sl, starts, block=32, window=40, prefix=33, **kw))
    assert K.device_status(clear=True) == 4


def test_select_of_rows_before_their_sequence_and_odd_lengths(K):
    q, kp, _, table, sl, starts = make(82, [900, 500, 100], [100, 20, 50], 2, 2, 16, BF)
    means = torch.randn(kp.shape[0], 2, D, device="cuda")
    for lens in ([30, 0, -5], [2 ** 31 - 1, 500, 100], [-2 ** 31, 10, 49]):
        sl.copy_(i32(lens))
        lists, counts = K.paged_select(q, means, table, sl, starts, page_size=16, topk=2, query_block=16,
                                       window_size=20, num_prefix_tokens=16)
        check_lists(lists, counts, PO.select(q, means, table, sl, starts, page_size=16, topk=2, block=16, window=20,
                                             prefix=16))
    assert K.device_status(clear=True) == 0


# ---------------------------------------------------------------------------
# attention over lists
# ---------------------------------------------------------------------------

def random_lists(seed, args, Hkv, ps, block, starts, width, share=0.5, own=True):
    """Ascending lists of a random part of the pages that each block could read; those
    of blocks that the rows could make but do not hold what no call may use."""
    rng = random.Random(seed)
    q, _, _, table, sl, _ = args
    blocks = PO.query_blocks(sl, starts, block)
    k = min(q.shape[0], len(sl))
    most = (q.shape[0] - k) // block + k
    lists = torch.full((most, Hkv, width), -1, dtype=torch.int32)
    counts = torch.zeros(lists.shape[:2], dtype=torch.int32)
    lists[len(blocks):], counts[len(blocks):] = 2 ** 30, 99
    for i, (_, _, m, pos) in enumerate(blocks):
        pages = min(table.shape[1], max(0, -(-(pos + m) // ps)))
        for h in range(Hkv):
            pick = [p for p in range(pages) if rng.random() < share or (own and p == pages - 1)]
            pick = sorted(rng.sample(pick, min(len(pick), width)))
            lists[i, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
            counts[i, h] = len(pick)
    return lists.cuda(), counts.cuda()


def check(got, args, lists, counts, starts=None, block=1, scale=None):
    """The bounds of test_gpu_paged.check(), the keys being those that are listed."""
    q, kp, vp, table, lens, _ = args
    want, spread, ds = PO.listed_attention(q, kp, vp, table, lens, lists, counts, starts, block=block, scale=scale)
    u = torch.finfo(q.dtype).eps / 2
    n = float(lists.shape[2] * kp.shape[2])
    rel = u + 2 * (129 * ds + 16) * 2.0 ** -23 + n * 2.0 ** -23
    tol = rel[..., None] * spread + u * want.abs() + 2.0 ** -25 * n * (q.dtype == FP) * 6.0 + 1e-7
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    bad = err > tol * 1.01
    assert not bad.any(), f"{int(bad.sum())} off, worst {(err / tol).max():.2f} of its bound, err {err.max():.3e}"


DECODE = [
    # lens, Hq, Hkv, page_size, dtype, width, share, layout
    ([1], 1, 1, 16, BF, 1, 1.0, "phtd"),
    ([300], 16, 16, 16, BF, 20, 0.5, "phtd"),
    ([63, 64, 65, 0, 1], 4, 2, 64, BF, 3, 1.0, "phtd"),
    ([5000, 1, 777, 0, 0, 64, 2049], 7, 1, 32, FP, 100, 0.5, "phtd"),
    ([1500, 2600, 3, 129], 56, 8, 64, BF, 24, 0.5, "ptkhd"),
    ([4097, 15, 16, 17], 8, 1, 128, FP, 12, 0.3, "phtd"),
    ([900, 70, 1200, 200, 201, 66], 6, 2, 16, BF, 9, 0.1, "phtd"),
    ([2000, 500, 129, 1], 5, 1, 1024, BF, 2, 1.0, "ptkhd"),
    (list(range(0, 300)), 2, 2, 16, BF, 7, 0.4, "phtd"),
    ([40000], 32, 32, 128, BF, 200, 0.5, "phtd"),
    ([70001, 2], 7, 1, 64, FP, 900, 0.8, "phtd"),
    # A cluster a pair: up to 37 pairs of two to 32 key tiles.
    ([2000], 1, 1, 64, BF, 2, 0.9, "phtd"),
    ([3000, 0, 5, 64, 2049], 7, 1, 64, BF, 32, 0.9, "ptkhd"),
    ([3000, 700, 1], 24, 12, 16, FP, 128, 0.7, "phtd"),
    ([100, 3000], 16, 16, 1024, BF, 2, 1.0, "phtd"),
    ([2100] * 37, 8, 1, 32, FP, 9, 0.2, "phtd"),
    ([2100] * 38, 8, 1, 32, FP, 9, 0.2, "phtd"),  # a pair too many
]


@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode_listed_vs_oracle(K, case):
    lens, Hq, Hkv, ps, dtype, width, share, layout = DECODE[case]
    args = make(200 + case, lens, [1] * len(lens), Hq, Hkv, ps, dtype, layout=layout)
    q, kp, vp, table, sl, _ = args
    lists, counts = random_lists(case, args, Hkv, ps, 1, None, width, share)
    out = K.paged_decode_listed(q, kp, vp, table, sl, lists, counts)
    check(out, args, lists, counts)
    assert torch.equal(out, K.paged_decode_listed(q, kp, vp, table, sl, lists, counts))
    assert K.device_status(clear=True) == 0


PREFILL = [
    # lens, news, Hq, Hkv, page_size, dtype, block, width, share, layout
    ([1], [1], 1, 1, 16, BF, 1, 1, 1.0, "phtd"),
    ([64], [64], 2, 2, 64, BF, 64, 1, 1.0, "phtd"),
    ([130, 128, 7], [130, 128, 7], 4, 4, 32, BF, 128, 4, 0.7, "phtd"),
    ([700, 300, 1000], [130, 1, 257], 7, 1, 16, FP, 16, 40, 0.5, "phtd"),
    ([200, 0, 333, 500], [5, 0, 333, 20], 56, 8, 64, BF, 18, 6, 0.6, "ptkhd"),
    ([1100], [1000], 16, 16, 128, BF, 100, 9, 0.5, "phtd"),
    ([2100], [600], 6, 1, 32, BF, 21, 30, 0.4, "phtd"),
    ([9000], [20], 2, 2, 64, BF, 32, 100, 0.5, "phtd"),     # parts of long lists
    ([9000, 31], [3, 2], 7, 1, 16, FP, 1, 400, 0.6, "phtd"),
    ([6000, 4000, 0, 40], [70, 33, 0, 9], 8, 1, 1024, BF, 16, 6, 0.8, "phtd"),
    (list(range(1, 120)), list(range(1, 120)), 2, 1, 16, BF, 64, 5, 0.5, "phtd"),
    ([3000], [2049], 2, 2, 256, BF, 37, 12, 0.4, "ptkhd"),
]


@pytest.mark.parametrize("case", range(len(PREFILL)))
def test_prefill_listed_vs_oracle(K, case):
    lens, news, Hq, Hkv, ps, dtype, block, width, share, layout = PREFILL[case]
    args = make(300 + case, lens, news, Hq, Hkv, ps, dtype, layout=layout)
    q, kp, vp, table, sl, starts = args
    lists, counts = random_lists(case, args, Hkv, ps, block, starts, width, share, own=case % 2 == 0)
    pad = 5
    qq = torch.cat([q, torch.full((pad,) + tuple(q.shape[1:]), float("nan"), dtype=dtype, device=q.device)])
    blocks = K.lib().sabre_paged_query_blocks(qq.shape[0], len(lens), block)
    assert lists.shape[0] == K.lib().sabre_paged_query_blocks(q.shape[0], len(lens), block)
    more = torch.full((blocks - lists.shape[0],) + tuple(lists.shape[1:]), 2 ** 30, dtype=torch.int32, device="cuda")
    all_lists = torch.cat([lists, more])
    all_counts = torch.cat([counts, torch.full((more.shape[0], Hkv), 99, dtype=torch.int32, device="cuda")])
    out = torch.full_like(qq, 7.0)
    K.paged_prefill_listed(qq, kp, vp, table, sl, starts, all_lists, all_counts, query_block=block, out=out)
    assert (out[q.shape[0]:] == 7.0).all(), "rows behind the last sequence were written"
    check(out[:q.shape[0]], args, lists, counts, starts, block)
    again = torch.full_like(qq, 7.0)
    K.paged_prefill_listed(qq, kp, vp, table, sl, starts, all_lists, all_counts, query_block=block, out=again)
    assert torch.equal(out, again)
    assert K.device_status(clear=True) == 0


def test_all_pages_listed_is_dense_attention(K):
    args = make(400, [900, 1300, 80], [300, 200, 80], 4, 2, 64, BF)
    q, kp, vp, table, sl, starts = args
    lists, counts = random_lists(0, args, 2, 64, 64, starts, 21, 1.0)
    got = K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=64)
    want, spread, ds = PO.attention(q, kp, vp, table, sl, starts)
    other, _, _ = PO.listed_attention(q, kp, vp, table, sl, lists, counts, starts, block=64)
    assert torch.allclose(want, other, rtol=1e-12, atol=1e-12)
    check(got, args, lists, counts, starts, 64)


def test_one_list_for_all_heads_and_blocks(K):
    args = make(401, [900, 1300, 80], [30, 20, 40], 4, 2, 16, BF)
    q, kp, vp, table, sl, starts = args
    one = i32([0, 1, 4, 9, 40, 41, 56, 80])
    n = K.lib().sabre_paged_query_blocks(q.shape[0], 3, 16)
    lists, counts = one.expand(n, 2, 8), i32([7]).expand(n, 2)
    check(K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=16), args, lists, counts,
          starts, 16)
    last = (q[starts[1:].long() - 1],) + args[1:]
    lists, counts = one.expand(3, 2, 8), i32([8]).expand(3, 2)
    check(K.paged_decode_listed(last[0], kp, vp, table, sl, lists, counts), last, lists, counts)
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("ps", [16, 64, 128])
def test_odd_lists(K, ps):
    """Entries twice, out of order, negative, past the table, of absent pages, past
    the sequence; counts past the list and below zero; empty lists give zeros."""
    args = make(402, [700, 700, 700, 300, 700], [40, 40, 40, 40, 40], 4, 2, ps, BF, extra_cols=2)
    q, kp, vp, table, sl, starts = args
    table[0, 1] = -1
    n = 700 // ps
    rows = [[0, 0, 1, 1, 2, n], [2, 1, 0, 3, 3, n], [-7, 0, 2, 2 ** 30, 2 ** 31 - 1, -1], [0, 1, 2, 3, 4, 2 * n],
            [-1] * 6]
    lists = i32(rows)[:, None].repeat(1, 2, 1)
    counts = i32([[6, 3], [6, 99], [6, 1], [99, 2], [0, -4]])
    big = K.lib().sabre_paged_query_blocks(q.shape[0], 5, 64)
    assert big > 5
    pl = torch.cat([lists, lists[:1].repeat(big - 5, 1, 1)])
    pc = torch.cat([counts, counts[:1].repeat(big - 5, 1)])
    out = K.paged_prefill_listed(q, kp, vp, table, sl, starts, pl, pc, query_block=64)
    check(out, args, lists, counts, starts, 64)
    assert (out[160:] == 0).all()
    assert K.device_status(clear=True) == 4
    last = (q[starts[1:].long() - 1],) + args[1:]
    out = K.paged_decode_listed(last[0], kp, vp, table, sl, lists, counts)
    check(out, last, lists, counts)
    assert (out[4] == 0).all() and K.device_status(clear=True) == 4


def test_listed_rows_that_see_nothing_give_zeros(K):
    args = make(403, [40, 100, 64], [40, 100, 64], 4, 2, 16, BF)
    q, kp, vp, table, sl, starts = args
    lists, counts = random_lists(1, args, 2, 16, 32, starts, 7, 1.0)
    sl[0] = 10  # 30 of the 40 rows lie before the sequence
    table[1] = -1
    out = K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=32)
    assert (out[:30] == 0).all() and (out[40:140] == 0).all() and (out[140:] != 0).any()
    check(out, args, lists, counts, starts, 32)
    for lens in ([0, 0, 0], [-5, -2 ** 31, 2 ** 31 - 1]):
        sl.copy_(i32(lens))
        out = K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=32)
        assert torch.isfinite(out).all() and (out[:140] == 0).all()
        out = K.paged_decode_listed(q[:3], kp, vp, table, sl, lists[:3], counts[:3])
        assert torch.isfinite(out).all() and (out[:2] == 0).all()
    assert K.device_status(clear=True) == 0


def test_nan_in_what_a_listed_query_sees(K):
    """A NaN key that is listed is a NaN result for the heads and rows that see it,
    however the work is split; a page that is not listed may hold anything."""
    args = make(404, [2000, 900], [70, 40], 4, 2, 16, BF)
    q, kp, vp, table, sl, starts = args
    lists, counts = random_lists(2, args, 2, 16, 32, starts, 60, 0.5)
    clean = K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=32)
    listed_pages = [set(lists[:3, h].flatten().tolist()) - {-1} for h in range(2)]
    free = next(p for p in range(100) if p not in listed_pages[0] and p not in listed_pages[1])
    kp[table[0, free]] = vp[table[0, free]] = float("nan")
    got = K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=32)
    assert torch.equal(got, clean)
    page = int(lists[0, 1, 0])
    kp[table[0, page], 1, 3] = float("nan")
    got = K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=32)
    hit = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
    for i in range(3):
        if page in lists[i, 1].tolist():
            hit[32 * i:min(32 * i + 32, 70), 2:] = True
    assert got[hit].isnan().all() and torch.equal(got[~hit], clean[~hit])
    last = q[starts[1:].long() - 1]
    got = K.paged_decode_listed(last, kp, vp, table, sl, lists[[0, 3]], counts[[0, 3]])
    assert got[0, 2:].isnan().all() and torch.isfinite(got[0, :2]).all() and torch.isfinite(got[1]).all()


def test_listed_results_into_any_layout_and_scale(K):
    args = make(405, [900, 1300, 77], [90, 211, 77], 16, 2, 64, BF)
    q, kp, vp, table, sl, starts = args
    lists, counts = random_lists(3, args, 2, 64, 16, starts, 12, 0.5)
    base = torch.full((16, q.shape[0] + 2, 2 * D), 7.0, dtype=BF, device="cuda")
    out = base[:, 1:-1, D:].transpose(0, 1)
    K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=16, softmax_scale=0.3, out=out)
    check(out, args, lists, counts, starts, 16, scale=0.3)
    assert (base[..., :D] == 7.0).all() and (base[:, 0] == 7.0).all() and (base[:, -1] == 7.0).all()
    fused = torch.randn(3, 20, D, device="cuda").to(BF)
    dec = (fused[:, 2:18],) + args[1:]
    check(K.paged_decode_listed(dec[0], kp, vp, table, sl, lists[:3], counts[:3], softmax_scale=0.02), dec, lists[:3],
          counts[:3], scale=0.02)


# ---------------------------------------------------------------------------
# a step of them together
# ---------------------------------------------------------------------------

def serve(K, st, new, k, v, q, block, topk, window, prefix):
    """One step: room for the rows, the rows, their pages' means, attention."""
    starts, slots, positions = K.paged_extend(new, st["table"], st["lens"], st["free"], st["count"],
                                              page_size=st["ps"], num_pages=st["kp"].shape[0], num_rows=k.shape[0])
    K.paged_store_slots(k, v, st["kp"], st["vp"], slots)
    K.paged_key_means(st["kp"], st["means"], st["table"], st["lens"], starts, num_rows=k.shape[0])
    kw = dict(page_size=st["ps"], topk=topk, window_size=window, num_prefix_tokens=prefix)
    if block is None:
        lists, counts = K.paged_select(q, st["means"], st["table"], st["lens"], **kw)
        return lists, counts, K.paged_decode_listed(q, st["kp"], st["vp"], st["table"], st["lens"], lists, counts)
    lists, counts = K.paged_select(q, st["means"], st["table"], st["lens"], starts, query_block=block, **kw)
    return lists, counts, K.paged_prefill_listed(q, st["kp"], st["vp"], st["table"], st["lens"], starts, lists, counts,
                                                 query_block=block)


def state(B, Hkv, ps, pages, cols, dtype=BF):
    ids = random.Random(1).sample(range(pages), pages)
    nan = torch.full((pages, Hkv, ps, D), float("nan"), dtype=dtype, device="cuda")
    return dict(ps=ps, table=torch.full((B, cols), -1, dtype=torch.int32, device="cuda"), lens=i32([0] * B),
                free=i32(ids), count=i32([pages]), kp=nan, vp=nan.clone(),
                means=torch.full((pages, Hkv, D), float("nan"), device="cuda"))


@pytest.mark.parametrize("Hq,Hkv,ps,block", [(4, 4, 16, 64), (7, 1, 32, 16), (16, 2, 64, 16)])
def test_prompts_then_steps_and_a_captured_step(K, Hq, Hkv, ps, block):
    """Prompts of several lengths, a chunk more, then steps of one token each, first
    eagerly and then as one graph that makes its own room; all against the oracle
    over the rows that were given."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    B, topk, window, prefix = 3, 3, 40, 20
    st = state(B, Hkv, ps, 3 * 800 // ps + 9, -(-800 // ps))
    rows = [[], [], []]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(BF)

    def verify(q, starts, lists, counts, out, block):
        want = PO.select(q, st["means"], st["table"], st["lens"], starts, page_size=ps, topk=topk, block=block,
                         window=window, prefix=prefix)
        check_lists(lists, counts, want)
        check(out, (q, st["kp"], st["vp"], st["table"], st["lens"], starts), lists, counts, starts, block)
        for b in range(B):
            k, _ = PO.gather(st["kp"], st["table"][b], int(st["lens"][b]))
            assert torch.equal(k, torch.cat(rows[b]).double())

    for news in ([300, 1, 517], [20, 200, 0]):
        n = sum(news)
        k, v, q = randn(n, Hkv, D), randn(n, Hkv, D), randn(n, Hq, D)
        starts = i32([0, news[0], news[0] + news[1], n])
        for b in range(B):
            rows[b].append(k[int(starts[b]):int(starts[b + 1])])
        verify(q, starts, *serve(K, st, i32(news), k, v, q, block, topk, window, prefix), block)
    one = i32([1] * B)
    k, v, q = (torch.empty(B, h, D, dtype=BF, device="cuda") for h in (Hkv, Hkv, Hq))
    graph, outs = torch.cuda.CUDAGraph(), None
    for step in range(70):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        for b in range(B):
            rows[b].append(k[b:b + 1].clone())
        if step == 2:
            with torch.cuda.graph(graph):
                outs = serve(K, st, one, k, v, q, None, topk, window, prefix)
        if step < 2:
            outs = serve(K, st, one, k, v, q, None, topk, window, prefix)
        else:
            graph.replay()
        if step % 9 < 3:
            verify(q, None, *outs, 1)
    assert st["lens"].tolist() == [320 + 70, 201 + 70, 517 + 70]
    assert K.device_status(clear=True) == 0


def test_two_streams_at_once(K):
    """Two states served on two streams give what each gives alone."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    ins = [[torch.randn(333, h, D, generator=gen, device="cuda").to(BF) for h in (2, 2, 14)] for _ in range(2)]

    def both(streams):
        outs = []
        states = [state(2, 2, 16, 60, 30) for _ in ins]
        torch.cuda.synchronize()
        for (k, v, q), st, s in zip(ins, states, streams):
            with torch.cuda.stream(s):
                for _ in range(2):
                    outs.append(serve(K, st, i32([33, 100]), k[:133], v[:133], q[:133], 16, 2, 10, 5))
        torch.cuda.synchronize()
        return outs

    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for x, y in zip(both((a, b)), both((a, a))):
        for s, t in zip(x, y):
            assert torch.equal(s, t)
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("call", ["clusters", "shares", "prompt", "parts"])
def test_listed_waits_that_run_out_end_the_call(K, call):
    """A wait limit shorter than any load: the call ends, records it and leaves the
    device usable."""
    lens, news = ([5000, 3000], [1, 1]) if call in ("clusters", "shares") else ([5000, 3000], [70, 40])
    args = make(407, lens, news, 4, 2, 64, BF)
    q, kp, vp, table, sl, starts = args
    block = 1 if call in ("clusters", "shares") else 32
    lists, counts = random_lists(5, args, 2, 64, block, starts, dict(clusters=20, shares=70, prompt=6, parts=70)[call],
                                 0.9)

    def run():
        if block == 1:
            return K.paged_decode_listed(q, kp, vp, table, sl, lists, counts)
        return K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=block)

    K.device_status(clear=True)
    K.set_wait_limit_ns(1000)
    try:
        run()
        torch.cuda.synchronize()
    finally:
        K.set_wait_limit_ns(0)
    assert K.device_status(clear=True) & 1
    out = run()
    assert K.device_status(clear=True) == 0
    check(out, args, lists, counts, starts, block)


def test_two_streams_and_two_captured_graphs_of_listed_calls(K):
    """Calls on two streams, and two captured calls replayed at once, each with the
    workspace of its own that it allocates."""
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    jobs, graphs, outs = [], [], []
    for i, side in enumerate(sides):
        args = make(408 + i, [3000 + 77 * i, 2900], [60, 5], 4, 2, 64, BF)
        q, kp, vp, table, sl, starts = args
        long = random_lists(i, args, 2, 64, 32, starts, 40, 0.9)
        short = [t[[0, 2]] for t in long]
        wide = random_lists(9 + i, (q[:2],) + args[1:], 2, 64, 1, None, 46, 0.95)
        jobs.append((args, long, short, wide))

        def run(args=args, long=long, short=short, wide=wide):
            q, kp, vp, table, sl, starts = args
            return (K.paged_prefill_listed(q, kp, vp, table, sl, starts, *long, query_block=32),
                    K.paged_decode_listed(q[:2], kp, vp, table, sl, short[0][:, :, :20], short[1]),
                    K.paged_decode_listed(q[:2], kp, vp, table, sl, *wide))

        run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(run())
        graphs.append((g, run))
    for kind in ("streams", "graphs"):
        got = [None, None]
        for _ in range(5):
            for i, side in enumerate(sides):
                with torch.cuda.stream(side):
                    if kind == "graphs":
                        graphs[i][0].replay()
                        got[i] = outs[i]
                    else:
                        got[i] = graphs[i][1]()
        torch.cuda.synchronize()
        for (args, long, short, wide), (a, b, c) in zip(jobs, got):
            check(a, args, *long, args[5], 32)
            two = (args[0][:2],) + args[1:]
            check(b, two, short[0][:, :, :20], short[1])
            check(c, two, *wide)
    assert K.device_status(clear=True) == 0


def test_launches_of_listed_calls_are_counted(K):
    """LAUNCHES grows by the kernels of a call: those of its captured graph."""
    from cuda.bindings import runtime

    def kernels(call):
        graph = torch.cuda.CUDAGraph(keep_graph=True)
        before = K.LAUNCHES[0]
        with torch.cuda.graph(graph):
            call()
        counted = K.LAUNCHES[0] - before
        err, _, n = runtime.cudaGraphGetNodes(graph.raw_cuda_graph())
        assert err == runtime.cudaError_t.cudaSuccess
        assert counted == n
        return n

    args = make(406, [900, 300], [40, 16], 4, 2, 16, BF)
    q, kp, vp, table, sl, starts = args
    means = torch.zeros(kp.shape[0], 2, D, device="cuda")
    n = K.lib().sabre_paged_query_blocks(q.shape[0], 2, 16)
    lists, counts = i32(list(range(64))).expand(n, 2, 64), i32([2]).expand(n, 2)
    new, free, count = i32([1, 1]), i32(list(range(8))), i32([8])
    slots = torch.arange(q.shape[0], device="cuda")
    assert kernels(lambda: K.paged_extend(new, table, sl, free, count, page_size=16, num_pages=8, num_rows=2)) == 1
    assert kernels(lambda: K.paged_store_slots(q[:, :2], q[:, 2:], kp, vp, slots)) == 1
    assert kernels(lambda: K.paged_store_slots(q[:0, :2], q[:0, 2:], kp, vp, slots[:0])) == 0
    assert kernels(lambda: K.paged_key_means(kp, means, table, sl, starts, num_rows=56)) == 1
    assert kernels(lambda: K.paged_key_means(kp, means, table, sl, starts, num_rows=0)) == 0
    assert kernels(lambda: K.paged_select(q, means, table, sl, starts, page_size=16, topk=2, query_block=16)) == 1
    assert kernels(lambda: K.paged_select(q[:2], means, table, sl, page_size=16, topk=2)) == 1
    assert kernels(lambda: K.paged_select(q[:0], means, table, sl, starts, page_size=16, topk=2)) == 0
    assert kernels(lambda: K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=16)) == 2
    assert kernels(lambda: K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists[:, :, :2], counts,
                                                  query_block=16)) == 1
    # A cluster a pair up to 32 key tiles; parts and a joining kernel beyond them.
    assert kernels(lambda: K.paged_decode_listed(q[:2], kp, vp, table, sl, lists[:2], counts[:2])) == 1
    long = i32(list(range(132))).expand(2, 2, 132)
    assert kernels(lambda: K.paged_decode_listed(q[:2], kp, vp, table, sl, long, counts[:2])) == 2
    assert kernels(lambda: K.paged_decode_listed(q[:1, :2], kp[:, :1], vp[:, :1], table[:1], sl[:1], lists[:1, :1, :4],
                                                 counts[:1, :1])) == 1
