"""What the calls over selected pages, and those that build tables on the device,
refuse, without a GPU."""

import pytest
import torch

from sabrecoder_b200 import _lib
from sabrecoder_b200 import kernels as K

D = 128
BF = torch.bfloat16


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def args(**kw):
    a = dict(q=torch.zeros(3, 4, D, dtype=BF), k=torch.zeros(3, 2, D, dtype=BF), v=torch.zeros(3, 2, D, dtype=BF),
             k_pages=torch.zeros(5, 2, 16, D, dtype=BF), v_pages=torch.zeros(5, 2, 16, D, dtype=BF),
             key_means=torch.zeros(5, 2, D), page_table=i32(3, 2), seq_lens=i32(3), q_start=i32(4),
             lists=i32(3, 2, 6), counts=i32(3, 2), new_rows=i32(3), free_pages=i32(7), free_count=i32(1),
             slots=torch.zeros(3, dtype=torch.int64))
    a.update(kw)
    return a


def extend(a, **kw):
    K.paged_extend(a["new_rows"], a["page_table"], a["seq_lens"], a["free_pages"], a["free_count"],
                   **dict(dict(page_size=16, num_pages=5, num_rows=3), **kw))


def store(a):
    K.paged_store_slots(a["k"], a["v"], a["k_pages"], a["v_pages"], a["slots"])


def means(a, **kw):
    K.paged_key_means(a["k_pages"], a["key_means"], a["page_table"], a["seq_lens"], a["q_start"],
                      **dict(dict(num_rows=3), **kw))


def select(a, **kw):
    K.paged_select(a["q"], a["key_means"], a["page_table"], a["seq_lens"], a["q_start"],
                   **dict(dict(page_size=16, topk=2, query_block=16), **kw))


def decode(a, **kw):
    K.paged_decode_listed(a["q"], a["k_pages"], a["v_pages"], a["page_table"], a["seq_lens"], a["lists"], a["counts"],
                          **kw)


def prefill(a, **kw):
    K.paged_prefill_listed(a["q"], a["k_pages"], a["v_pages"], a["page_table"], a["seq_lens"], a["q_start"], a["lists"],
                           a["counts"], **dict(dict(query_block=16), **kw))


TABLES = [
    (dict(page_table=i32(3, 0)), "page_table"),
    (dict(page_table=i32(2, 3).t()), "column"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int64)), "int32"),
    (dict(seq_lens=i32(2)), "seq_lens"),
    (dict(seq_lens=i32(6)[::2]), "contiguous"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(), "CUDA tensor"),
]


@pytest.mark.parametrize("call", [extend, means, select, decode, prefill])
@pytest.mark.parametrize("i", range(len(TABLES)))
def test_tables_are_checked(call, i):
    kw, match = TABLES[i]
    with pytest.raises(_lib.SabreError, match=match):
        call(args(**kw))


@pytest.mark.parametrize("call", [means, select, prefill])
def test_row_starts_are_checked(call):
    for bad, match in ((i32(3), "q_start"), (torch.zeros(4, dtype=torch.int64), "int32")):
        with pytest.raises(_lib.SabreError, match=match):
            call(args(q_start=bad))


EXTEND = [
    (dict(page_table=None), {}, "page_table must be a tensor"),
    (dict(seq_lens=[0, 0, 0]), {}, "seq_lens must be a tensor"),
    (dict(new_rows=i32(2)), {}, "new_rows"),
    (dict(new_rows=torch.zeros(3)), {}, "new_rows|int32"),
    (dict(free_pages=i32(7, 1)), {}, "free_pages"),
    (dict(free_pages=torch.zeros(7, dtype=torch.int64)), {}, "int32"),
    (dict(free_count=i32(2)), {}, "free_count"),
    (dict(page_table=i32(0, 2), seq_lens=i32(0), new_rows=i32(0)), {}, "CUDA tensor|no sequences"),
    ({}, dict(page_size=0), "page_size"),
    ({}, dict(num_pages=0), "num_pages"),
    ({}, dict(num_rows=-1), "num_rows"),
    ({}, dict(seq_lens_out=i32(2)), "seq_lens_out"),
    ({}, dict(free_count_out=torch.zeros(1)), "int32"),
]


@pytest.mark.parametrize("i", range(len(EXTEND)))
def test_extend_refuses(i):
    a, kw, match = EXTEND[i]
    with pytest.raises(_lib.SabreError, match=match):
        extend(args(**a), **kw)


@pytest.mark.parametrize("a,match", [
    (dict(k_pages=torch.zeros(5, 2, 16, dtype=BF)), "must both be"),
    (dict(v_pages=torch.zeros(5, 2, 32, D, dtype=BF)), "must both be"),
    (dict(k=torch.zeros(3, 2, D)), "share dtype"),
    (dict(k=torch.zeros(3, 4, D, dtype=BF), v=torch.zeros(3, 4, D, dtype=BF)), "must both be"),
    (dict(v=torch.zeros(2, 2, D, dtype=BF)), "must both be"),
    (dict(k=torch.zeros(3, D, 2, dtype=BF).transpose(1, 2), v=torch.zeros(3, D, 2, dtype=BF).transpose(1, 2)), "unit"),
    (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots"),
    (dict(slots=torch.zeros(2, dtype=torch.int64)), "slots"),
    (dict(slots=[0, 1, 2]), "slots"),
    (dict(), "CUDA tensor"),
])
def test_store_by_slots_refuses(a, match):
    with pytest.raises(_lib.SabreError, match=match):
        store(args(**a))


@pytest.mark.parametrize("call", [means, select])
@pytest.mark.parametrize("bad", [torch.zeros(5, 2, D, dtype=BF), torch.zeros(5, 2, 64), torch.zeros(5, 2 * D),
                                 torch.zeros(5, D, 2).transpose(1, 2)])
def test_key_means_are_checked(call, bad):
    with pytest.raises(_lib.SabreError, match="key_means must be fp32"):
        call(args(key_means=bad))


def test_key_means_refuses():
    with pytest.raises(_lib.SabreError, match="needs num_rows"):
        means(args(), num_rows=None)
    with pytest.raises(_lib.SabreError, match="num_rows"):
        means(args(), num_rows=-1)
    with pytest.raises(_lib.SabreError, match="key_means must be fp32"):  # of another pool
        means(args(key_means=torch.zeros(4, 2, D)))
    with pytest.raises(_lib.SabreError, match="k_pages"):
        means(args(k_pages=torch.zeros(5, 2, 16, D)))


@pytest.mark.parametrize("kw,match", [(dict(topk=-1), "topk"), (dict(window_size=-1), "window_size"),
                                      (dict(num_prefix_tokens=-1), "num_prefix_tokens"),
                                      (dict(query_block=0), "query_block"),
                                      (dict(page_size=0), "page_size")])
def test_select_sizes_are_checked(kw, match):
    with pytest.raises(_lib.SabreError, match=match):
        select(args(), **kw)


def test_select_refuses():
    with pytest.raises(_lib.SabreError, match="need q_start"):
        select(args(q_start=None))
    with pytest.raises(_lib.SabreError, match="q .* must be"):
        select(args(q=torch.zeros(3, 4, D)))
    with pytest.raises(_lib.SabreError, match="q .* must be"):
        select(args(q=torch.zeros(3, D, dtype=BF)))


LISTS = [
    (dict(lists=i32(3, 2)), "lists must be"),
    (dict(lists=torch.zeros(3, 2, 6)), "lists must be"),
    (dict(counts=i32(3)), "counts must be"),
    (dict(counts=torch.zeros(3, 2, dtype=torch.int64)), "counts must be"),
    (dict(lists=[1]), "lists must be"),
]


@pytest.mark.parametrize("call", [decode, prefill])
@pytest.mark.parametrize("i", range(len(LISTS)))
def test_lists_are_checked(call, i):
    a, match = LISTS[i]
    with pytest.raises(_lib.SabreError, match=match):
        call(args(**a))


def test_prefill_listed_refuses():
    with pytest.raises(_lib.SabreError, match="needs q_start"):
        prefill(args(q_start=None))
    with pytest.raises(_lib.SabreError, match="query_block"):
        prefill(args(), query_block=0)


# -- the C entries, with pointers that are never read ---------------------

S3, S2 = _lib.i64([4096, 2048, 128]), _lib.i64([256, 128])
M2, L2, C2 = _lib.i64([256, 128]), _lib.i64([12, 6]), _lib.i64([2, 1])


def status(name, a):
    L = _lib.lib()
    return getattr(L, name)(*a), L.sabre_last_error()


def c_extend(**kw):
    a = dict(new_rows=16, table=32, lens=48, lens_out=48, free=64, count=80, count_out=80, starts=96, slots=112, pos=128,
             rows=3, batch=3, num_pages=5, page_size=16, max_pages=2, free_size=7, stride=2)
    a.update(kw)
    return status("sabre_paged_extend", [*a.values(), None])


@pytest.mark.parametrize("kw,code,match", [
    (dict(new_rows=None), -1, b"null"), (dict(free=None), -1, b"null"), (dict(slots=None), -1, b"null"),
    (dict(lens_out=16), -1, b"same"), (dict(rows=-1), -1, b"sizes"), (dict(batch=0), -1, b"sizes"),
    (dict(free_size=-1), -1, b"sizes"), (dict(page_size=24), -2, b"page_size"),
    (dict(page_size=2048), -2, b"page_size"),
    (dict(page_size=1024, max_pages=2 ** 21, stride=2 ** 21), -2, b"2^30"), (dict(batch=16385, stride=2), -2, b"16384"),
    (dict(stride=1), -1, b"overlap"), (dict(rows=2 ** 30 + 1), -2, b"2^30"),
])
def test_c_extend_rejects(kw, code, match):
    got, msg = c_extend(**kw)
    assert got == code and match in msg


def c_means(**kw):
    a = dict(k=16, means=16, table=16, lens=16, starts=None, rows=3, batch=3, heads=2, dim=128, num_pages=5, page_size=16,
             max_pages=2, ks=S3, ms=M2, stride=2, dtype=0)
    a.update(kw)
    return status("sabre_paged_key_means", [*a.values(), None])


@pytest.mark.parametrize("kw,code,match", [
    (dict(k=None), -1, b"null"), (dict(means=None), -1, b"null"), (dict(rows=0), -1, b"rows"),
    (dict(rows=4), -1, b"q_start"),
    (dict(dim=64), -2, b"head_dim"), (dict(means=8), -3, b"key_means"), (dict(ms=_lib.i64([256, 126])), -3, b"key_means"),
    (dict(ms=_lib.i64([-256, 128])), -3, b"key_means"), (dict(dtype=2), -1, b"dtype"),
])
def test_c_key_means_rejects(kw, code, match):
    got, msg = c_means(**kw)
    assert got == code and match in msg


def c_select(**kw):
    a = dict(q=16, means=16, table=16, lens=16, starts=16, lists=16, counts=16, rows=3, batch=3, heads_q=4, heads_kv=2,
             dim=128, num_pages=5, page_size=16, max_pages=2, topk=2, block=16, window=0, prefix=0,
             qs=_lib.i64([512, 128]), ms=M2, stride=2, dtype=0)
    a.update(kw)
    return status("sabre_paged_select", [*a.values(), None])


@pytest.mark.parametrize("kw,code,match", [
    (dict(q=None), -1, b"null"), (dict(lists=None), -1, b"null"), (dict(heads_q=0), -1, b"sizes"),
    (dict(rows=0), -1, b"sizes"),
    (dict(heads_q=3), -2, b"integer"), (dict(topk=-1), -1, b"topk"), (dict(block=0), -1, b"query_block"),
    (dict(block=1025), -1, b"query_block"), (dict(window=-1), -1, b"window"), (dict(starts=None), -1, b"q_start"),
    (dict(starts=None, block=1, rows=4), -1, b"q_start"), (dict(max_pages=32769, stride=32769), -2, b"32768"),
    (dict(q=8), -3, b"aligned"), (dict(qs=_lib.i64([512, 4])), -3, b"aligned"), (dict(means=4), -3, b"key_means"),
    (dict(qs=_lib.i64([2 ** 31, 128])), -2, b"strides"), (dict(heads_q=2050), -2, b"1024"),
])
def test_c_select_rejects(kw, code, match):
    got, msg = c_select(**kw)
    assert got == code and match in msg


def c_decode(**kw):
    a = dict(q=16, k=16, v=16, o=16, table=16, lens=16, lists=16, counts=16, entries=6, batch=3, heads_q=4, heads_kv=2,
             dim=128, num_pages=5, page_size=16, max_pages=2, qs=_lib.i64([512, 128]), ks=S3, vs=S3,
             os=_lib.i64([512, 128]), ls=L2, cs=C2, stride=2, scale=0.0, dtype=0, ws=16, wb=1 << 30)
    a.update(kw)
    return status("sabre_paged_decode_listed", [*a.values(), None])


def c_prefill(**kw):
    a = dict(q=16, k=16, v=16, o=16, table=16, lens=16, starts=16, lists=16, counts=16, entries=6, rows=3, batch=3,
             heads_q=4, heads_kv=2, dim=128, num_pages=5, page_size=16, max_pages=2, block=16, qs=_lib.i64([512, 128]),
             ks=S3, vs=S3, os=_lib.i64([512, 128]), ls=L2, cs=C2, stride=2, scale=0.0, dtype=0, ws=16, wb=1 << 30)
    a.update(kw)
    return status("sabre_paged_prefill_listed", [*a.values(), None])


BOTH = [
    (dict(lists=None), -1, b"null"), (dict(counts=None), -1, b"null"), (dict(entries=0), -1, b"entries"),
    (dict(ls=_lib.i64([-12, 6])), -1, b"strides"), (dict(cs=_lib.i64([2, -1])), -1, b"strides"),
    (dict(q=None), -1, b"null"),
    (dict(heads_q=5), -2, b"integer"), (dict(heads_q=18), -2, b"integer"), (dict(dim=64), -2, b"head_dim"),
    (dict(page_size=1024, entries=2 ** 20 + 1), -2, b"2^30"),
]


@pytest.mark.parametrize("call", [c_decode, c_prefill])
@pytest.mark.parametrize("kw,code,match", BOTH)
def test_c_listed_attention_rejects(call, kw, code, match):
    got, msg = call(**kw)
    assert got == code and match in msg


@pytest.mark.parametrize("kw,code,match", [
    (dict(starts=None), -1, b"null"), (dict(rows=0), -1, b"rows"), (dict(block=0), -2, b"query_block"),
    (dict(block=65), -2, b"query_block"), (dict(block=2 ** 31 - 1), -2, b"query_block"),
    (dict(entries=1000, ws=None), -5, b"workspace"), (dict(entries=1000, wb=100), -5, b"workspace"),
    (dict(entries=1000, ws=8), -3, b"workspace"),
])
def test_c_prefill_listed_rejects(kw, code, match):
    got, msg = c_prefill(**kw)
    assert got == code and match in msg


@pytest.mark.parametrize("kw,code", [(dict(ws=None), -5), (dict(wb=100), -5), (dict(ws=8), -3)])
def test_c_decode_listed_workspace(kw, code):
    assert c_decode(**kw)[0] == code


def test_sizes_that_callers_ask_for():
    L = _lib.lib()
    assert L.sabre_paged_query_blocks(0, 3, 16) == 0 and L.sabre_paged_query_blocks(100, 1, 16) == 7
    assert L.sabre_paged_query_blocks(100, 200, 16) == 100  # a row each at most
    for ps, block, window in ((16, 1, 0), (16, 16, 15), (64, 128, 256), (32, 33, 1000)):
        width = L.sabre_paged_select_width(ps, 1 << 20, 5, block, window, 40)
        # Pages that a span of window + block tokens can touch, wherever it begins.
        most = max((s + window + block - 1) // ps - s // ps + 1 for s in range(ps))
        assert width == 5 + -(-40 // ps) + most
    assert L.sabre_paged_select_width(16, 7, 100, 1, 0, 0) == 7
    assert L.sabre_paged_select_width(16, 0, 1, 1, 0, 0) == 0
    assert L.sabre_paged_prefill_listed_workspace_size(3, 3, 4, 2, 128, 16, 16, 6) == 0
    assert L.sabre_paged_prefill_listed_workspace_size(3, 3, 4, 2, 128, 16, 16, 1000) > 0
    assert L.sabre_paged_prefill_listed_workspace_size(3, 3, 4, 2, 64, 16, 16, 1000) == 0
