"""GPU tests of selected pages and of steps on the device where ranges end: values
whose squares underflow, rows far before their sequence, lengths that are no
multiple of the page, row starts that do not ascend, other streams."""

import pytest
import torch

from oracle import paged_oracle as PO
from sabrecoder_b200 import _lib
from test_gpu_paged import BF, D, make
from test_gpu_paged_listed import K, check, check_lists, i32  # noqa: F401 (K: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,news,block", [([3000, 3000], [64, 64], 16), ([3000, 2800], [1, 1], 1),
                                             ([3000, 3000], [1900, 1100], 16)])
@pytest.mark.parametrize("of_means,of_queries", [(-80, 0), (0, -80), (-80, 33), (-60, -60), (-75, -75)])
def test_select_of_tiny_means_and_queries(K, lens, news, block, of_means, of_queries):
    """Scores that only 64 bits tell apart, of vectors whose squares are nothing in 32
    bits: factors of two change no order as long as the scores stay in range."""
    q, kp, _, table, sl, starts = make(85, lens, news, 4, 4, 16, BF)
    gen = torch.Generator(device="cuda").manual_seed(10)
    base = torch.randn(4, D, generator=gen, device="cuda")
    ulp = torch.randint(-3, 4, (kp.shape[0], 4, D), generator=gen, device="cuda").float() * 2.0 ** -24
    means = base * (1 + ulp) * 2.0 ** of_means
    q = q * 2.0 ** of_queries
    starts = None if block == 1 else starts
    lists, counts = K.paged_select(q, means, table, sl, starts, page_size=16, topk=20, query_block=block)
    check_lists(lists, counts, PO.select(q, means, table, sl, starts, page_size=16, topk=20, block=block))


@pytest.mark.parametrize("starts,rows,block", [([0, 12800, 0, 12800], 12800, 16), ([0, 700, 3, 700, 0, 700], 700, 1),
                                               ([0, 640] * 20, 640, 4)])
def test_select_with_row_starts_that_do_not_ascend(K, starts, rows, block):
    """Sequences that share rows count more blocks than the rows can make: no list or
    count behind the last is written."""
    B, H, ps = len(starts) - 1, 16, 16
    L = K.lib()
    blocks, cols = L.sabre_paged_query_blocks(rows, B, block), -(-rows // ps)
    width = L.sabre_paged_select_width(ps, cols, 3, block, 0, 0)
    q = torch.randn(rows, H, D, device="cuda").to(BF)
    means = torch.randn(cols, H, D, device="cuda")
    table = torch.arange(cols, dtype=torch.int32, device="cuda").repeat(B, 1)
    lens, start = i32([rows] * B), i32(starts)
    lists = torch.full((2 * blocks + B * rows, H, width), -7, dtype=torch.int32, device="cuda")
    counts = torch.full((2 * blocks + B * rows, H), -7, dtype=torch.int32, device="cuda")
    st = L.sabre_paged_select(q.data_ptr(), means.data_ptr(), table.data_ptr(), lens.data_ptr(), start.data_ptr(),
                              lists[blocks:].data_ptr(), counts[blocks:].data_ptr(), rows, B, H, H, D, cols, ps, cols,
                              3, block, 0, 0, _lib.i64([H * D, D]), _lib.i64([H * D, D]), cols, 0,
                              torch.cuda.current_stream().cuda_stream)
    assert st == 0
    for t in (lists, counts):
        assert (t[:blocks] == -7).all() and (t[2 * blocks:] == -7).all()
    mine = counts[blocks:2 * blocks]
    assert ((mine >= 0) & (mine <= width) | (mine == -7)).all() and (mine > 0).any()
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("width", [1, 300])
def test_listed_rows_far_before_their_sequence_give_zeros(K, width):
    """A block of 128 rows of which 108 lie before the sequence, whatever they hold; also
    in parts of long lists."""
    args = make(406, [128, 200], [128, 128], 2, 2, 16, BF)
    q, kp, vp, table, sl, starts = args
    sl[0] = 20
    q[:108] = float("nan")
    lists = torch.full((3, 2, width), -1, dtype=torch.int32, device="cuda")  # the rows could make three blocks
    lists[:, :, 0] = 0
    counts = i32([[1, 1]] * 3)
    out = K.paged_prefill_listed(q, kp, vp, table, sl, starts, lists, counts, query_block=128)
    assert (out[:108] == 0).all()
    clean = (q.nan_to_num(0.0),) + args[1:]
    check(out, clean, lists, counts, starts, 128)
    assert K.device_status(clear=True) == 0


def test_settling_waits_for_steps_on_other_streams(K):
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    c = SabrePagedKVCache(batch_size=3, max_seq_len=64, page_size=16, num_layers=1, num_kv_heads=1, head_dim=D)
    new = i32([20, 0, 1])
    c.lend()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.extend_on_device(new, 21)
        torch.cuda._sleep(200_000_000)  # a tenth of a second or so
        c.extend_on_device(new, 21)
    c.settle()
    assert c.lengths == [40, 0, 2] == c.seq_lens.tolist() and c.pages_in_use == 4
    c.extend([1, 1, 1])
    assert c.seq_lens.tolist() == [41, 1, 3] and K.device_status(clear=True) == 0
    c.lend()
    c.settle()
    with torch.cuda.stream(side):  # not ordered behind it: nothing is lent all the same
        _, slots, _ = K.paged_extend(new, c.page_table, c.seq_lens, c.free_pages, c.free_count, page_size=16,
                                     num_pages=c.num_pages, num_rows=21)
    side.synchronize()
    assert (slots == -1).all() and c.seq_lens.tolist() == c.lengths and K.device_status(clear=True) == 8


@pytest.mark.parametrize("extra_rows", [0, 3000])
@pytest.mark.parametrize("new,fits", [([10, 2, 0, 700], True), ([10, 3, 0, 700], False), ([0, 0, 1, 0], False),
                                      ([0, 0, 0, 0], True)])
def test_extend_within_a_greatest_length(K, new, fits, extra_rows):
    """1000 rows at most on pages of 16; one sequence is there already."""
    old, ps, pool = [5, 998, 1000, 300], 16, 300
    table = [[63 * b + p if p * ps < n else -1 for p in range(63)] for b, n in enumerate(old)]
    free, rows = list(range(260, 300)) + list(range(10, 62)), sum(new) + 2 + extra_rows
    want = PO.extend(new, table, old, free, len(free), ps, pool, rows, 1000)
    assert want[0] == fits
    t, lens, count = i32(table), i32(old), i32([len(free)])
    starts, slots, positions = K.paged_extend(i32(new), t, lens, i32(free), count, page_size=ps, num_pages=pool,
                                              num_rows=rows, max_seq_len=1000)
    for got, w in zip((t, lens, count, starts, slots, positions), (*want[1:3], [want[3]], *want[4:])):
        assert got.tolist() == w
    assert K.device_status(clear=True) == (0 if fits else 8)


def test_captured_steps_keep_max_seq_len(K):
    """A replayed step stands still at max_seq_len, as the host's would raise."""
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    c = SabrePagedKVCache(batch_size=2, max_seq_len=40, page_size=16, num_layers=1, num_kv_heads=1, head_dim=D)
    one, k = i32([1, 1]), torch.ones(2, 1, D, device="cuda", dtype=BF)
    c.extend([30, 30])
    c.truncate(1, 20)
    c.lend()
    c.extend_on_device(one, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        starts, slots, _ = c.extend_on_device(one, 2)
        c.store_rows(0, k, k, starts, slots)
    for _ in range(9):
        graph.replay()
    assert K.device_status(clear=True) == 0
    graph.replay()
    assert slots.tolist() == [-1, -1] and K.device_status(clear=True) == 8
    c.settle()
    assert c.lengths == [40, 30]
    c.extend([0, 10])
    assert c.lengths == c.seq_lens.tolist() == [40, 40]


def test_reading_rows_while_pages_are_lent(K):
    """gather() and the length that a model asks for follow the steps on the device."""
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    c = SabrePagedKVCache(batch_size=2, max_seq_len=64, page_size=16, num_layers=1, num_kv_heads=2, head_dim=D)
    rows = torch.randn(40, 2, D, device="cuda").to(BF)
    c.append(0, rows[None, :10].repeat(2, 1, 1, 1), -rows[None, :10].repeat(2, 1, 1, 1))
    c.lend()
    starts, slots, _ = c.extend_on_device(i32([30, 1]), 31)
    c.store_rows(0, torch.cat([rows[10:], rows[10:11]]), -torch.cat([rows[10:], rows[10:11]]), starts, slots)
    assert c.get_seq_length() == 40 and c.get_mask_sizes(1, 0) == (41, 0)
    k, v = c.gather(0)
    assert torch.equal(k[0], rows.transpose(0, 1)) and torch.equal(v, -k)
    assert torch.equal(k[1, :, :11], rows[:11].transpose(0, 1)) and (k[1, :, 11:] == 0).all()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(ValueError, match="capture"), torch.cuda.graph(graph):
        c.gather(0)
    torch.cuda.synchronize()
    c.settle()
    assert torch.equal(c.gather(0)[0], k) and c.get_seq_length() == 40


def test_new_outputs_go_through_torch(K):
    """Outputs of the listed calls are filled in deterministic mode and seen by dispatch
    modes, as those of the other calls."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        count = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.count += "empty" in str(func)
            return func(*args, **(kwargs or {}))

    args = make(407, [100, 60], [40, 30], 2, 2, 16, BF)
    q, kp, vp, table, sl, starts = args
    lists, counts = i32([[[0, 1], [0, 2]]] * 2), i32([[2, 2], [2, 1]])
    pad = torch.cat([q, q[:5]])
    more = K.lib().sabre_paged_query_blocks(75, 2, 64) - 2
    lists, counts = (torch.cat([t, t[:1].repeat(more, *[1] * (t.dim() - 1))]) for t in (lists, counts))

    def call():
        return K.paged_prefill_listed(pad, kp, vp, table, sl, starts, lists, counts, query_block=64)

    want = call()
    before = torch.are_deterministic_algorithms_enabled(), torch.utils.deterministic.fill_uninitialized_memory
    try:
        torch.use_deterministic_algorithms(True)
        torch.utils.deterministic.fill_uninitialized_memory = True
        out = call()
    finally:
        torch.use_deterministic_algorithms(before[0])
        torch.utils.deterministic.fill_uninitialized_memory = before[1]
    assert torch.equal(out[:70], want[:70]) and out[70:].isnan().all()
    with Seen() as seen:
        out = call()
    assert seen.count >= 1 and torch.equal(out[:70], want[:70])


@pytest.mark.parametrize("tiles", [1, 2, 32, 33])
@pytest.mark.parametrize("pairs", [27, 28, 29, 30])
def test_decode_listed_where_clusters_end(K, pairs, tiles):
    """Clusters of up to 28 pairs of two to 32 key tiles, and shares with a joining kernel
    past them: results, and the kernels that are counted."""
    args = make(500 + pairs, [tiles * 64 + 10 - b for b in range(pairs)], [1] * pairs, 3, 1, 64, BF)
    q, kp, vp, table, sl, _ = args
    lists = torch.arange(tiles, dtype=torch.int32, device="cuda").expand(pairs, 1, tiles)
    counts = torch.full((pairs, 1), tiles, dtype=torch.int32, device="cuda")
    before = K.LAUNCHES[0]
    out = K.paged_decode_listed(q, kp, vp, table, sl, lists, counts)
    assert K.LAUNCHES[0] - before == (1 if pairs <= 28 and 2 <= tiles <= 32 else 2)
    check(out, args, lists, counts)
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("Hq,Hkv,max_len", [(4, 2, 300), (7, 1, 1000)])
def test_a_ragged_prompt_on_the_device(K, Hq, Hkv, max_len):
    """Prompts and turns of different lengths in one step on the device: room, rows,
    means, selection and attention, captured and replayed, against the oracle."""
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    gen = torch.Generator(device="cuda").manual_seed(11)
    c = SabrePagedKVCache(batch_size=3, max_seq_len=max_len, num_pages=3 * 1008 // 16, page_size=16, num_layers=2,
                          num_kv_heads=Hkv, head_dim=D, topk_pages=2, window_size=20, num_prefix_tokens=5)
    c.pool.fill_(float("nan"))
    c.key_means.fill_(float("nan"))
    n = 160
    new = i32([0, 0, 0])
    q = torch.empty(2, n, Hq, D, dtype=BF, device="cuda")
    k, v = (torch.empty(2, n, Hkv, D, dtype=BF, device="cuda") for _ in range(2))
    outs = [torch.full((n, Hq, D), 7.0, dtype=BF, device="cuda") for _ in range(2)]

    def step():
        q_start, slots, _ = c.extend_on_device(new, n)
        lists, counts = [], []
        for i, layer in enumerate(c.layers):
            c.store_rows(i, k[i], v[i], q_start, slots)
            li, co = c.select(i, q[i], q_start)
            K.paged_prefill_listed(q[i], layer.k_pages, layer.v_pages, c.page_table, c.seq_lens, q_start, li, co,
                                   query_block=c.block_rows(Hq), out=outs[i])
            lists.append(li)
            counts.append(co)
        return q_start, lists, counts

    c.lend()
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q_start, lists, counts = step()
    before = [0, 0, 0]
    for rows in ([130, 1, 29], [0, 0, 0], [3, 150, 0], [17, 1, 142]):
        new.copy_(i32(rows))
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        before = [a + b for a, b in zip(before, rows)]
        assert c.seq_lens.tolist() == before and q_start.tolist()[-1] == sum(rows)
        for i, layer in enumerate(c.layers):
            args = (q[i, :sum(rows)], layer.k_pages, layer.v_pages, c.page_table, c.seq_lens, q_start)
            block = c.block_rows(Hq)
            check_lists(lists[i], counts[i], PO.select(q[i], layer.key_means, c.page_table, c.seq_lens, q_start,
                                                       page_size=16, topk=2, block=block, window=20, prefix=5))
            if sum(rows):
                check(outs[i][:sum(rows)], args, lists[i], counts[i], q_start, block)
            assert (outs[i][sum(rows):] == 7.0).all()
    c.settle()
    assert c.lengths == before and K.device_status(clear=True) == 0
