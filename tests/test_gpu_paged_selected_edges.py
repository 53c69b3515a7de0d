"""GPU tests of selected pages and of steps on the device where ranges end: values
whose squares underflow, rows far before their sequence, lengths that are no
multiple of the page, row starts that do not ascend, other streams."""

import pytest
import torch

from oracle import paged_oracle as PO
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
