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
                              lists[blocks:].data_ptr(), counts[blocks:].data_ptr(), rows, B, H, H, D, cols, ps, cols, 3,
                              block, 0, 0, _lib.i64([H * D, D]), _lib.i64([H * D, D]), cols, 0,
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
