"""Pages lent to the device, on the CPU: sequences whose greatest length is no
multiple of the page."""

import pytest
import torch

from oracle import paged_oracle as PO
from sabrecoder_b200 import _lib
from sabrecoder_b200 import paged_cache as PC
from test_paged_cache_selected import PS, add, cache, consistent, plain_kernels  # noqa: F401 (a fixture)
from test_paged_listed_refusals import args, c_extend, extend, status


@pytest.fixture(autouse=True)
def extend_within(plain_kernels, monkeypatch):  # noqa: F811
    def fn(new, table, lens, free, count, *, page_size, num_pages, num_rows, max_seq_len=None):
        _, t, n, c, starts, slots, pos = PO.extend(new.tolist(), table.tolist(), lens.tolist(), free.tolist(), int(count),
                                                   page_size, num_pages, num_rows, max_seq_len)
        table.copy_(torch.tensor(t))
        lens.copy_(torch.tensor(n))
        count.fill_(c)
        return torch.tensor(starts, dtype=torch.int32), torch.tensor(slots), torch.tensor(pos)
    monkeypatch.setattr(PC.K, "paged_extend", fn)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


def test_steps_on_the_device_keep_max_seq_len():
    """40 rows at most, on pages that hold 48: what the host refuses the device has no
    room for, and the cache goes on."""
    c = cache(max_seq_len=40)
    add(c, [38, 38, 10], torch.Generator().manual_seed(7))
    with pytest.raises(ValueError, match="full"):
        c.extend([3, 0, 0])
    c.lend()
    _, slots, _ = c.extend_on_device(i32([3, 0, 0]), 3)
    assert (slots == -1).all() and c.seq_lens.tolist() == [38, 38, 10]
    starts, slots, pos = c.extend_on_device(i32([2, 1, 30]), 33)
    assert starts.tolist() == [0, 2, 3, 33] and (slots >= 0).all() and pos.tolist() == [38, 39, 38, *range(10, 40)]
    c.settle()
    consistent(c)
    assert c.lengths == [40, 39, 40]
    c.extend([0, 1, 0])
    assert c.lengths == [40, 40, 40]


def test_settling_refuses_lengths_past_the_greatest():
    c = cache(max_seq_len=40)
    c.lend()
    c.extend_on_device(i32([40, 0, 0]), 40)
    c.seq_lens[0] = 41
    with pytest.raises(ValueError, match="went from 0 rows to 41"):
        c.settle()
    c.seq_lens[0] = 40
    c.settle()
    consistent(c)


def test_greatest_length_refusals(monkeypatch):
    monkeypatch.undo()
    for bad in (0, -5):
        with pytest.raises(_lib.SabreError, match="max_seq_len"):
            extend(args(), max_seq_len=bad)
    with pytest.raises(_lib.SabreError, match="CUDA tensor"):
        extend(args(), max_seq_len=2 ** 40)
    a = [16, 32, 48, 48, 64, 80, 80, 96, 112, 128, 3, 3, 5, 16, 2, 7]
    for changed, code, match in (({}, -1, b"max_len"), ({0: None}, -1, b"null"), ({13: 24}, -2, b"page_size")):
        b = [changed.get(i, x) for i, x in enumerate(a)]
        got, msg = status("sabre_paged_extend_within", [*b, 9 if changed else -1, 2, None])
        assert got == code and match in msg and b"extend_within" in msg
    assert b"sabre_paged_extend:" in c_extend(page_size=24)[1]
