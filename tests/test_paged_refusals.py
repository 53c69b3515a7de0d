"""What the paged cache calls refuse, without a GPU."""

import ctypes

import pytest
import torch

from sabrecoder_b200 import _lib
from sabrecoder_b200 import kernels as K

D = 128


def args(**kw):
    a = dict(k=torch.zeros(3, 2, D, dtype=torch.bfloat16), v=torch.zeros(3, 2, D, dtype=torch.bfloat16),
             q=torch.zeros(3, 4, D, dtype=torch.bfloat16), k_pages=torch.zeros(5, 2, 16, D, dtype=torch.bfloat16),
             v_pages=torch.zeros(5, 2, 16, D, dtype=torch.bfloat16), page_table=torch.zeros(3, 2, dtype=torch.int32),
             seq_lens=torch.zeros(3, dtype=torch.int32), q_start=torch.zeros(4, dtype=torch.int32))
    a.update(kw)
    return a


def store(a):
    K.paged_store(a["k"], a["v"], a["k_pages"], a["v_pages"], a["page_table"], a["seq_lens"], a["q_start"])


def decode(a, **kw):
    K.paged_decode(a["q"], a["k_pages"], a["v_pages"], a["page_table"], a["seq_lens"], **kw)


def prefill(a, **kw):
    K.paged_prefill(a["q"], a["k_pages"], a["v_pages"], a["page_table"], a["seq_lens"], a["q_start"], **kw)


SHARED = [
    (dict(v_pages=torch.zeros(5, 2, 32, D, dtype=torch.bfloat16)), "must both be"),
    (dict(k_pages=torch.zeros(5, 2, 16, dtype=torch.bfloat16)), "must both be"),
    (dict(page_table=torch.zeros(3, 0, dtype=torch.int32)), "page_table"),
    (dict(page_table=torch.zeros(2, 3, dtype=torch.int32).t()), "column"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int64)), "int32"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int32)), "seq_lens"),
    (dict(seq_lens=torch.zeros(6, dtype=torch.int32)[::2]), "contiguous"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(k_pages=torch.zeros(5, 2, 16, D), v_pages=torch.zeros(5, 2, 16, D), q=torch.zeros(3, 4, D),
          k=torch.zeros(3, 2, D), v=torch.zeros(3, 2, D)), "bf16 or f16"),
    (dict(q=torch.zeros(3, 4, D, dtype=torch.float16), k=torch.zeros(3, 2, D, dtype=torch.float16)), "pages are"),
    (dict(), "CUDA tensor"),
]


@pytest.mark.parametrize("call", [store, decode, prefill])
@pytest.mark.parametrize("i", range(len(SHARED)))
def test_shared_argument_checks(call, i):
    kw, match = SHARED[i]
    with pytest.raises(_lib.SabreError, match=match):
        call(args(**kw))


@pytest.mark.parametrize("call", [store, prefill])
def test_row_starts_are_checked(call):
    with pytest.raises(_lib.SabreError, match="q_start"):
        call(args(q_start=torch.zeros(3, dtype=torch.int32)))
    with pytest.raises(_lib.SabreError, match="int32"):
        call(args(q_start=torch.zeros(4, dtype=torch.int64)))


def test_prefill_needs_row_starts():
    with pytest.raises(_lib.SabreError, match="needs q_start"):
        prefill(args(q_start=None))


def test_rows_are_checked():
    half = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(_lib.SabreError, match="unit last"):
        decode(args(q=half))
    with pytest.raises(_lib.SabreError, match="unit last"):
        decode(args(q=torch.zeros(3, D, 4, dtype=torch.bfloat16).transpose(1, 2)))
    with pytest.raises(_lib.SabreError, match="unit last"):
        prefill(args(q=torch.zeros(3, D, dtype=torch.bfloat16)))


@pytest.mark.parametrize("call", [decode, prefill])
def test_windows_are_checked(call):
    with pytest.raises(_lib.SabreError, match="must not be negative"):
        call(args(), window_size=-1)
    with pytest.raises(_lib.SabreError, match="must not be negative"):
        call(args(), num_prefix_tokens=-1)


def i64(*v):
    return _lib.i64(v)


def c_decode(**kw):
    a = dict(q=16, kp=16, vp=16, o=16, table=16, lens=16, batch=2, hq=8, hkv=2, d=128, pages=4, ps=64, cols=3, window=-1,
             prefix=0, qs=i64(1024, 128), ks=i64(16384, 8192, 128), vs=i64(16384, 8192, 128), os=i64(1024, 128),
             ts=3, scale=0.0, dtype=0, ws=None, wsb=0)
    a.update(kw)
    return _lib.lib().sabre_paged_decode(*a.values(), None)


def c_prefill(**kw):
    a = dict(q=16, kp=16, vp=16, o=16, table=16, lens=16, starts=16, rows=7, batch=2, hq=8, hkv=2, d=128, pages=4, ps=64,
             cols=3, window=-1, prefix=0, qs=i64(1024, 128), ks=i64(16384, 8192, 128), vs=i64(16384, 8192, 128),
             os=i64(1024, 128), ts=3, scale=0.0, dtype=0, ws=None, wsb=0)
    a.update(kw)
    return _lib.lib().sabre_paged_prefill(*a.values(), None)


def c_store(**kw):
    a = dict(k=16, v=16, kp=16, vp=16, table=16, lens=16, starts=None, rows=2, batch=2, hkv=2, d=128, pages=4, ps=64,
             cols=3, rs=i64(256, 128), vrs=i64(256, 128), ks=i64(16384, 8192, 128), vs=i64(16384, 8192, 128), ts=3,
             dtype=0)
    a.update(kw)
    return _lib.lib().sabre_paged_store(*a.values(), None)


C_SHARED = [
    (dict(kp=None), -1, b"null"), (dict(table=None), -1, b"null"), (dict(lens=None), -1, b"null"),
    (dict(ks=None), -1, b"null"), (dict(batch=0), -1, b"positive"), (dict(hkv=0), -1, b""),
    (dict(pages=0), -1, b"positive"), (dict(cols=0), -1, b"positive"), (dict(d=64), -2, b"head_dim"),
    (dict(ps=48), -2, b"page_size"), (dict(ps=8), -2, b"page_size"), (dict(ps=2048), -2, b"page_size"),
    (dict(cols=1 << 25, ts=1 << 25), -2, b"2^30"), (dict(dtype=2), -1, b"dtype"), (dict(kp=24), -3, b"aligned"),
    (dict(vp=8), -3, b"aligned"), (dict(ks=i64(16384, 8192, 100)), -3, b"multiples"),
    (dict(vs=i64(16384, 0, 128)), -3, b"multiples"), (dict(ts=2), -1, b"overlap"),
]


@pytest.mark.parametrize("call", [c_store, c_decode, c_prefill])
@pytest.mark.parametrize("i", range(len(C_SHARED)))
def test_c_entries_check_before_launch(call, i):
    kw, status, text = C_SHARED[i]
    assert call(**kw) == status and text in _lib.lib().sabre_last_error()


@pytest.mark.parametrize("call", [c_decode, c_prefill])
def test_c_attention_checks(call):
    err = _lib.lib().sabre_last_error
    assert call(q=None) == -1 and call(o=None) == -1 and call(qs=None) == -1 and call(os=None) == -1
    assert call(hq=7) == -2 and b"integer" in err()
    assert call(hq=18) == -2 and b"integer" in err()
    assert call(hq=0) == -1
    assert call(prefix=-1) == -1 and b"num_prefix_tokens" in err()
    assert call(q=20) == -3 and call(o=20) == -3
    assert call(qs=i64(1024, 100)) == -3 and call(os=i64(100, 128)) == -3


def test_c_decode_workspace_and_size():
    err = _lib.lib().sabre_last_error
    need = _lib.lib().sabre_paged_decode_workspace_size(2, 8, 2, 128)
    assert need > 0
    assert c_decode(ws=None) == -5 and c_decode(ws=16, wsb=need - 1) == -5 and b"workspace" in err()
    assert c_decode(ws=24, wsb=need) == -3
    assert c_decode(batch=1 << 24, cols=1 << 20, ts=1 << 20, ws=16, wsb=1 << 40) == -2 and b"2^37" in err()


def test_c_store_and_prefill_rows():
    err = _lib.lib().sabre_last_error
    assert c_store(k=None) == -1 and c_store(rs=None) == -1
    assert c_store(rows=3) == -1 and b"need q_start" in err()
    assert c_store(starts=16, rows=0) == -1
    assert c_store(rs=i64(256, 100)) == -3 and c_store(v=40) == -3
    assert c_prefill(starts=None) == -1 and b"null" in err()
    assert c_prefill(rows=0) == -1


def c_copy(a_, b_, **kw):
    n = len(a_)
    a = dict(pages=16, buffers=2, bs=1 << 20, num=8, pst=1 << 17, pb=1 << 17, src=(ctypes.c_int32 * n)(*a_),
             dst=(ctypes.c_int32 * n)(*b_), n=n)
    a.update(kw)
    return _lib.lib().sabre_copy_pages(*a.values(), None)


def test_copy_pages_refusals():
    err = _lib.lib().sabre_last_error
    assert c_copy([0], [8]) == -1 and b"outside" in err()
    assert c_copy([-1], [2]) == -1 and b"outside" in err()
    assert c_copy([0, 1], [2, 2]) == -1 and b"written twice" in err()
    assert c_copy([0, 2], [2, 3]) == -1 and b"read and written" in err()
    assert c_copy([3], [3]) == -1 and b"read and written" in err()
    assert c_copy([0], [1], pages=None) == -1 and c_copy([0], [1], src=None) == -1
    assert c_copy([0], [1], buffers=0) == -1 and c_copy([0], [1], pb=0) == -1
    assert c_copy([0], [1], buffers=70000) == -2
    assert c_copy([0], [1], pages=24) == -3 and c_copy([0], [1], pb=1000) == -3 and c_copy([0], [1], bs=8) == -3
    assert c_copy([0], [1], pst=1 << 16) == -1 and b"overlap" in err()
    assert c_copy([], []) == 0
    pages = torch.zeros(2, 4, 1, 16, D)
    for a, b, match in (([0], [1, 2], "destinations"), ([0], [4], "outside"), ([-1], [1], "outside"),
                        ([0], [1], "CUDA tensor"), (torch.zeros(2), [1, 2], "integer"),
                        (torch.zeros(1, 1, dtype=torch.int64), [1], "1-D")):
        with pytest.raises(_lib.SabreError, match=match):
            K.copy_pages(pages, a, b)
    with pytest.raises(_lib.SabreError, match="must be"):
        K.copy_pages(pages[0, 0], [0], [1])


def test_prompts_whose_key_tiles_pass_int32_do_not_run_in_shares():
    """A call in shares counts the key tiles of all its row tiles in 32 bits (one row
    tile sees up to 2^24 of them): the plan, seen in the workspace it asks for, is a
    CTA for each pair where the sum could pass."""
    def size(rows, ps, cols, batch=1, hq=8, hkv=1):
        return _lib.lib().sabre_paged_prefill_workspace_size(rows, batch, hq, hkv, D, ps, cols, -1, 0)

    assert size(16, 1024, 1 << 20) > 0 and size(127 * 16, 1024, 1 << 20) > 0  # 127 tiles of 2^24
    assert size(128 * 16, 1024, 1 << 20) == 0 and size(148 * 16, 1024, 1 << 20) == 0
    assert size(148 * 16, 1024, 1 << 19) > 0
    assert size(147, 1024, 1 << 20, batch=128) == 0


def test_outputs_that_overlap_themselves_are_refused():
    """Rows or heads of an expanded output would be written by several CTAs at once."""
    row = torch.zeros(1, 4, D, dtype=torch.bfloat16).expand(3, 4, D)
    head = torch.zeros(3, 1, D, dtype=torch.bfloat16).expand(3, 4, D)
    for call in (decode, prefill):
        for out in (row, head):
            with pytest.raises(_lib.SabreError, match="overlap"):
                call(args(), out=out)
