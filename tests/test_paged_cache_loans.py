"""Pages lent to the device, on the CPU: what reads the sequences meanwhile, and
sequences whose greatest length is no multiple of the page."""

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
        _, t, n, c, starts, slots, pos = PO.extend(new.tolist(), table.tolist(), lens.tolist(), free.tolist(),
                                                   int(count), page_size, num_pages, num_rows, max_seq_len)
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


def test_rows_and_lengths_follow_the_device_while_pages_are_lent():
    """What the device added is gathered, and is in the length that a model asks for."""
    gen = torch.Generator().manual_seed(8)
    c = cache()
    add(c, [38, 38, 10], gen)
    c.lend()
    starts, slots, _ = c.extend_on_device(i32([5, 0, 2]), 7)
    rows = torch.randn(7, 2, 8, generator=gen)
    for i in range(2):
        c.store_rows(i, rows, -rows, starts, slots)
    for _ in range(2):  # during the loan and after it
        k, v = c.gather(0)
        assert k.shape == (3, 2, 43, 8)
        assert torch.equal(k[0, :, 38:], rows[:5].transpose(0, 1)) and torch.equal(v[0, :, 38:], -k[0, :, 38:])
        assert torch.equal(k[2, :, 10:12], rows[5:].transpose(0, 1)) and (k[2, :, 12:] == 0).all()
        assert c.get_seq_length() == 43 and c.get_mask_sizes(1, 0) == (44, 0)
        c.settle()
    assert c.lengths == [43, 38, 12]


@pytest.mark.parametrize("call", [lambda c: c.append(1, torch.zeros(3, 1, 2, 8), torch.zeros(3, 1, 2, 8)),
                                  lambda c: c.check_step(0, 1, None), lambda c: c.check_step(1, 1, None),
                                  lambda c: c.layers[0].update(torch.zeros(3, 2, 1, 8), torch.zeros(3, 2, 1, 8))])
def test_steps_of_the_host_wait_for_the_end_of_the_loan(call):
    """Also those whose first layer was stored before it."""
    c = cache()
    add(c, [20, 20, 20], torch.Generator().manual_seed(9))
    c.append(0, torch.ones(3, 1, 2, 8), torch.ones(3, 1, 2, 8))
    c.lend()
    pool = c.pool.clone()
    with pytest.raises(ValueError, match="settle"):
        call(c)
    assert torch.equal(pool.nan_to_num(7.0), c.pool.nan_to_num(7.0)) and c.lengths == [21] * 3
    c.settle()
    c.append(1, torch.ones(3, 1, 2, 8), torch.ones(3, 1, 2, 8))
    consistent(c)


def test_a_capture_cannot_read_lengths_that_are_the_devices(monkeypatch):
    c = cache()
    add(c, [20, 20, 20], torch.Generator().manual_seed(10))
    monkeypatch.setattr(PC, "_capturing", lambda pool: True)
    assert c.get_seq_length() == 20 and c.gather(0)[0].shape[2] == 20
    monkeypatch.setattr(PC, "_capturing", lambda pool: False)
    c.lend()
    monkeypatch.setattr(PC, "_capturing", lambda pool: True)
    for call in (c.get_seq_length, lambda: c.gather(0)):
        with pytest.raises(ValueError, match="capture"):
            call()
