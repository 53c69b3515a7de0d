"""GPU tests of the paged K/V cache kernels against the 64-bit oracle. Every row
of a pool that no sequence owns holds NaN, so a read of one shows."""

import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

D = 128
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from sabrecoder_b200 import kernels
    return kernels


def make(seed, lens, news, Hq, Hkv, ps, dtype, window=None, prefix=0, layout="phtd", extra_cols=1, drop=True,
         spare=3):
    """Pools, tables and queries of a ragged batch on the GPU. With a window,
    pages that no new row can see are absent (drop)."""
    gen = torch.Generator().manual_seed(seed)
    cap = max(max((n + ps - 1) // ps for n in lens), 1) + extra_cols
    table = torch.full((len(lens), cap), -1, dtype=torch.int32)
    live = []
    for b, (n, new) in enumerate(zip(lens, news)):
        for p in range((n + ps - 1) // ps):
            if drop and window is not None and p * ps >= prefix and (p + 1) * ps <= n - new - window:
                continue
            live.append((b, p))
    P = len(live) + spare
    ids = torch.randperm(P, generator=gen).tolist()
    if layout == "phtd":
        kp, vp = (torch.full((P, Hkv, ps, D), float("nan"), dtype=dtype) for _ in range(2))
    else:  # K and V interleaved, heads inside a row: [P, ps, 2, Hkv, D]
        both = torch.full((P, ps, 2, Hkv, D), float("nan"), dtype=dtype)
        kp, vp = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    for (b, p), page in zip(live, ids):
        table[b, p] = page
        m = min(ps, lens[b] - p * ps)
        kp[page, :, :m] = torch.randn(Hkv, m, D, generator=gen).to(dtype)
        vp[page, :, :m] = torch.randn(Hkv, m, D, generator=gen).to(dtype)
    starts = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32)
    q = torch.randn(int(starts[-1]), Hq, D, generator=gen).to(dtype)
    if layout == "phtd":
        kp, vp = kp.cuda(), vp.cuda()
    else:
        both = both.cuda()
        kp, vp = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    return (q.cuda(), kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), starts.cuda())


def check(got, args, window=None, prefix=0, scale=None, starts=None):
    """|got - exact| against the arithmetic of the kernels, each factor a bound:
    a weight p is rounded to the type once (u = eps / 2 relative), the result
    once; a score is a sum of 128 products (128 additions, up to 2^-23 each of
    the sum of magnitudes ds, and 2^-23 for the scaling), and p moves by twice
    that; ex2 and the joining of partial sums add 16 * 2^-23; the sums over n keys
    n * 2^-23 of the magnitudes. f16 weights below its normal range are off by
    half the smallest step, 2^-25, each."""
    q, kp, vp, table, lens, _ = args
    want, spread, ds = PO.attention(q, kp, vp, table, lens, starts, window=window, prefix=prefix, scale=scale)
    u = torch.finfo(q.dtype).eps / 2
    n = float(lens.max())
    rel = u + 2 * (129 * ds + 16) * 2.0 ** -23 + n * 2.0 ** -23
    tol = rel[..., None] * spread + u * want.abs() + 2.0 ** -25 * n * (q.dtype == FP) * 6.0 + 1e-7
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    bad = err > tol * 1.01
    assert not bad.any(), f"{int(bad.sum())} off, worst {(err / tol).max():.2f} of its bound, err {err.max():.3e}"


DECODE = [
    # lens, Hq, Hkv, page_size, dtype, window, prefix, layout
    ([1], 1, 1, 16, BF, None, 0, "phtd"),
    ([300], 16, 16, 16, BF, None, 0, "phtd"),
    ([63, 64, 65, 0, 1], 4, 2, 64, BF, None, 0, "phtd"),
    ([5000, 1, 777, 0, 0, 64, 2049], 7, 1, 32, FP, None, 0, "phtd"),
    ([1500, 2600, 3, 129], 56, 8, 64, BF, None, 0, "ptkhd"),
    ([4097, 15, 16, 17], 8, 1, 128, FP, None, 0, "phtd"),
    ([900, 70, 1200, 200, 201, 66], 6, 2, 16, BF, 100, 0, "phtd"),
    ([900, 70, 1200, 200, 201, 1100], 4, 4, 64, FP, 64, 33, "phtd"),
    ([2000, 500, 129], 10, 2, 256, BF, 0, 5, "phtd"),
    ([2000, 500, 129, 1], 5, 1, 1024, BF, 700, 200, "ptkhd"),
    ([3000, 31, 400], 3, 1, 32, BF, 1000, 5000, "phtd"),
    (list(range(0, 300)), 2, 2, 16, BF, None, 0, "phtd"),
    ([40000], 32, 32, 128, BF, None, 0, "phtd"),
    ([70001, 2], 7, 1, 64, FP, None, 0, "phtd"),
]


@pytest.mark.parametrize("case", range(len(DECODE)))
def test_paged_decode_vs_oracle(K, case):
    lens, Hq, Hkv, ps, dtype, window, prefix, layout = DECODE[case]
    args = make(case, lens, [1] * len(lens), Hq, Hkv, ps, dtype, window, prefix, layout)
    q, kp, vp, table, sl, _ = args
    out = K.paged_decode(q, kp, vp, table, sl, window_size=window, num_prefix_tokens=prefix)
    check(out, args, window, prefix)
    again = K.paged_decode(q, kp, vp, table, sl, window_size=window, num_prefix_tokens=prefix)
    assert torch.equal(out, again)
    assert K.device_status(clear=True) == 0


PREFILL = [
    # lens, news, Hq, Hkv, page_size, dtype, window, prefix, layout
    ([1], [1], 1, 1, 16, BF, None, 0, "phtd"),
    ([64], [64], 2, 2, 64, BF, None, 0, "phtd"),
    ([130, 128, 7], [130, 128, 7], 4, 4, 32, BF, None, 0, "phtd"),
    ([700, 300, 1000], [130, 1, 257], 7, 1, 16, FP, None, 0, "phtd"),
    ([200, 0, 333, 500], [5, 0, 333, 20], 56, 8, 64, BF, None, 0, "ptkhd"),
    ([1100], [1000], 16, 16, 128, BF, None, 0, "phtd"),
    ([900, 1300, 80], [900, 200, 80], 4, 2, 64, BF, 100, 0, "phtd"),
    ([900, 1300, 80], [900, 200, 80], 3, 1, 16, FP, 64, 33, "phtd"),
    ([900, 1300, 80], [300, 200, 80], 8, 1, 64, BF, 0, 0, "phtd"),
    ([900, 1300, 80], [300, 200, 80], 5, 1, 1024, BF, 257, 128, "ptkhd"),
    ([2100], [600], 6, 1, 32, BF, 500, 700, "phtd"),
    ([9000], [20], 2, 2, 64, BF, None, 0, "phtd"),
    ([9000, 31], [3, 2], 7, 1, 16, FP, None, 0, "phtd"),
    (list(range(1, 120)), list(range(1, 120)), 2, 1, 16, BF, None, 0, "phtd"),
    # Few row tiles over a long table: the call runs in shares of the key tiles.
    ([3000, 5000, 100], [300, 129, 100], 4, 2, 64, BF, None, 0, "phtd"),
    ([2500, 0, 6000, 4096], [1, 0, 700, 64], 7, 1, 16, FP, None, 0, "ptkhd"),
    ([8000, 3000], [200, 3000], 2, 2, 128, BF, 2500, 100, "phtd"),
    ([20000], [130], 56, 8, 64, BF, None, 0, "phtd"),
    ([4000, 30, 2100, 2], [40, 30, 1, 2], 8, 1, 1024, BF, 2050, 0, "phtd"),
    ([17 * i % 400 + 2100 for i in range(128)], [i % 3 for i in range(128)], 3, 1, 16, BF, None, 0, "phtd"),
    ([17 * i % 400 + 2100 for i in range(129)], [i % 3 for i in range(129)], 3, 1, 16, FP, None, 0, "phtd"),
]


@pytest.mark.parametrize("case", range(len(PREFILL)))
def test_paged_prefill_vs_oracle(K, case):
    lens, news, Hq, Hkv, ps, dtype, window, prefix, layout = PREFILL[case]
    args = make(100 + case, lens, news, Hq, Hkv, ps, dtype, window, prefix, layout)
    q, kp, vp, table, sl, starts = args
    pad = 5
    qq = torch.cat([q, torch.full((pad,) + tuple(q.shape[1:]), float("nan"), dtype=dtype, device=q.device)])
    out = torch.full_like(qq, 7.0)
    K.paged_prefill(qq, kp, vp, table, sl, starts, window_size=window, num_prefix_tokens=prefix, out=out)
    assert (out[q.shape[0]:] == 7.0).all(), "rows behind the last sequence were written"
    check(out[:q.shape[0]], args, window, prefix, starts=starts)
    again = K.paged_prefill(q, kp, vp, table, sl, starts, window_size=window, num_prefix_tokens=prefix)
    assert torch.equal(out[:q.shape[0]], again)
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("lens,news,Hq,Hkv,ps,window,prefix", [
    ([8400], [400], 56, 8, 64, None, 0),              # equal shares that cut pairs anywhere
    ([900, 1300, 77], [900, 211, 77], 7, 1, 32, None, 0),
    ([900, 1300, 77], [900, 211, 77], 16, 2, 64, 300, 40),
])
def test_results_into_any_layout(K, lens, news, Hq, Hkv, ps, window, prefix):
    """Outputs with heads outermost and rows apart; what lies between stays."""
    args = make(31, lens, news, Hq, Hkv, ps, BF, window, prefix)
    q, kp, vp, table, sl, starts = args
    base = torch.full((Hq, q.shape[0] + 2, 2 * D), 7.0, dtype=BF, device="cuda")
    out = base[:, 1:-1, D:].transpose(0, 1)
    K.paged_prefill(q, kp, vp, table, sl, starts, window_size=window, num_prefix_tokens=prefix, out=out)
    check(out, args, window, prefix, starts=starts)
    assert (base[..., :D] == 7.0).all() and (base[:, 0] == 7.0).all() and (base[:, -1] == 7.0).all()
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("extra_cols", [1, 300])  # 300: the call runs in shares
def test_rows_that_see_nothing_give_zeros(K, extra_cols):
    """Sequences shorter than their new rows, absent pages under every visible
    key, lengths of zero."""
    q, kp, vp, table, sl, starts = make(5, [40, 100, 64], [40, 100, 64], 4, 2, 16, BF, extra_cols=extra_cols)
    table[1] = -1
    sl[0] = 10  # 30 of the 40 rows lie before the sequence
    out = K.paged_prefill(q, kp, vp, table, sl, starts)
    assert (out[:30] == 0).all() and (out[40:140] == 0).all() and (out[140:] != 0).any()
    check(out, (q, kp, vp, table, sl, starts), starts=starts)
    sl[1] = 0  # a whole row tile before the sequence
    out = K.paged_prefill(q, kp, vp, table, sl, starts)
    assert (out[:30] == 0).all() and (out[40:140] == 0).all() and (out[140:] != 0).any()
    check(out, (q, kp, vp, table, sl, starts), starts=starts)
    sl[1], sl[2] = 100, 0
    out = K.paged_decode(q[:3], kp, vp, table, sl)
    assert (out[1:] == 0).all() and (out[0] != 0).any()


@pytest.mark.parametrize("ps,extra_cols", [(16, 1), (64, 1), (128, 1), (16, 300), (64, 50)])
def test_absent_pages_inside_a_tile(K, ps, extra_cols):
    """Pages missing at the start, inside and at the end are not visible."""
    args = make(6, [1000, 900], [1, 1], 6, 2, ps, BF, extra_cols=extra_cols)
    q, kp, vp, table, sl, _ = args
    for b, p in ((0, 0), (0, 3), (0, 4), (1, 1), (1, 899 // ps)):
        if table[b, p] >= 0:
            kp[table[b, p]] = float("nan")
            vp[table[b, p]] = float("nan")
        table[b, p] = -1
    check(K.paged_decode(q, kp, vp, table, sl), args)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    check(K.paged_prefill(q, kp, vp, table, sl, starts), args)
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("ps,window,prefix", [(16, 100, 33), (64, 129, 0), (128, 700, 70), (32, 0, 1), (64, 127, 64)])
@pytest.mark.parametrize("extra_cols", [1, 200])
def test_rows_no_query_sees_may_hold_anything(K, ps, window, prefix, extra_cols):
    """NaN and infinities in rows of present pages that lie before every query's
    window and behind the prefix."""
    lens, news = [1500, 2100, 901], [300, 1, 130]
    args = make(18, lens, news, 6, 2, ps, BF, window, prefix, drop=False, extra_cols=extra_cols)
    q, kp, vp, table, sl, starts = args
    for b, (n, new) in enumerate(zip(lens, news)):
        for j in range(prefix, n - new - window):
            bad = float("nan") if j % 3 else float("inf")
            kp[table[b, j // ps], :, j % ps] = bad
            vp[table[b, j // ps], :, j % ps] = bad
    clean = (q, torch.nan_to_num(kp, 0.0, 0.0), torch.nan_to_num(vp, 0.0, 0.0), table, sl, starts)
    kw = dict(window_size=window, num_prefix_tokens=prefix)
    check(K.paged_prefill(q, kp, vp, table, sl, starts, **kw), clean, window, prefix, starts=starts)
    for b, (n, new) in enumerate(zip(lens, news)):  # and what the last row alone does not see
        for j in range(max(prefix, n - new - window), n - 1 - window):
            kp[table[b, j // ps], :, j % ps] = vp[table[b, j // ps], :, j % ps] = float("nan")
    last = (q[starts[1:].long() - 1],) + clean[1:]
    check(K.paged_decode(last[0], kp, vp, table, sl, **kw), last, window, prefix)
    assert K.device_status(clear=True) == 0


def test_pages_outside_the_pool_are_absent_and_recorded(K):
    args = make(7, [200, 300], [1, 1], 4, 2, 32, BF)
    q, kp, vp, table, sl, _ = args
    table[0, 2] = kp.shape[0]
    table[1, 1] = -5
    check(K.paged_decode(q, kp, vp, table, sl), args)
    assert K.device_status(clear=True) == 4
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    check(K.paged_prefill(q, kp, vp, table, sl, starts), args)
    assert K.device_status(clear=True) == 4
    sl[0] = 96  # the new row would go to the bad page
    before = kp.clone()
    K.paged_store(q[:, :2], q[:, 2:], kp, vp, table, sl)
    assert K.device_status(clear=True) == 4
    changed = (kp != before) & ~(kp.isnan() & before.isnan())
    assert changed.flatten(1).any(1).nonzero().flatten().tolist() == [int(table[1, 299 // 32])]


def test_lengths_past_the_table_read_only_what_it_holds(K):
    args = make(8, [128, 256], [1, 1], 2, 2, 64, BF, extra_cols=0)
    q, kp, vp, table, sl, _ = args
    sl[1] = 100000
    check(K.paged_decode(q, kp, vp, table, sl), (q, kp, vp, table, sl, None))
    K.paged_store(q, q, kp, vp, table, sl)  # the second row has no place
    assert K.device_status(clear=True) == 4


def test_strided_rows_scale_and_output(K):
    """q a slice of a fused projection, out a view of a wider buffer, scores at
    another scale."""
    args = make(9, [500, 77, 130], [200, 77, 1], 4, 2, 32, BF)
    q, kp, vp, table, sl, starts = args
    fused = torch.randn(q.shape[0], 8, D, device="cuda").to(BF)
    fused[:, 2:6] = q
    wide = torch.full((q.shape[0], 8, D), 3.0, dtype=BF, device="cuda")
    K.paged_prefill(fused[:, 2:6], kp, vp, table, sl, starts, softmax_scale=0.21, out=wide[:, 1:5])
    check(wide[:, 1:5], args, scale=0.21, starts=starts)
    assert (wide[:, 0] == 3.0).all() and (wide[:, 5:] == 3.0).all()
    wide.fill_(3.0)
    K.paged_decode(fused[:3, 2:6], kp, vp, table, sl, softmax_scale=0.21, out=wide[:3, 1:5])
    check(wide[:3, 1:5], (q[:3],) + args[1:], scale=0.21)
    assert (wide[:, 0] == 3.0).all() and (wide[:, 5:] == 3.0).all()


def test_large_scores_stay_finite(K):
    """Scores in the hundreds, rising along the sequence, in both types."""
    for dtype in (BF, FP):
        args = make(10, [700, 90], [150, 90], 4, 1, 16, dtype)
        q, kp, vp, table, sl, starts = args
        q *= 40
        check(K.paged_prefill(q, kp, vp, table, sl, starts), args, starts=starts)
        last = (q[starts[1:].long() - 1],) + args[1:]
        check(K.paged_decode(*last[:5]), last)


@pytest.mark.parametrize("dtype,ps,layout", [(BF, 16, "phtd"), (FP, 64, "ptkhd"), (BF, 1024, "phtd")])
def test_paged_store_writes_its_rows_and_nothing_else(K, dtype, ps, layout):
    lens, news = [1, 70, 300, 90, 64, 0], [1, 7, 290, 0, 64, 0]
    args = make(11, lens, news, 1, 3, ps, dtype, layout=layout)
    _, kp, vp, table, sl, starts = args
    kp.fill_(0.5), vp.fill_(-0.5)
    table[2, 1] = -1  # dropped silently
    n = int(starts[-1])
    k = torch.randn(n + 9, 6, D, device="cuda").to(dtype)[:, ::2]
    v = torch.randn(n + 9, 3, D, device="cuda").to(dtype)
    wk, wv = kp.clone(), vp.clone()
    for r, page, off in PO.slots(table, sl, starts, ps, kp.shape[0]):
        wk[page, :, off] = k[r]
        wv[page, :, off] = v[r]
    K.paged_store(k, v, kp, vp, table, sl, starts)
    assert torch.equal(kp, wk) and torch.equal(vp, wv)
    assert K.device_status(clear=True) == 0
    # One row per sequence without starts.
    B = len(lens)
    sl2 = (sl + 1).clamp(max=table.shape[1] * ps)
    for r, page, off in PO.slots(table, sl2, None, ps, kp.shape[0]):
        wk[page, :, off] = k[r]
        wv[page, :, off] = v[r]
    K.paged_store(k[:B], v[:B], kp, vp, table, sl2)
    assert torch.equal(kp, wk) and torch.equal(vp, wv)


@pytest.mark.parametrize("shape,moves", [((5, 2, 9, 3, 16, D), 4), ((7, 1, 16, D), 2), ((2, 1300, 1, 16, D), 600),
                                         ((3, 40, 8, 128, D), 17)])
def test_copy_pages(K, shape, moves):
    gen = torch.Generator().manual_seed(12)
    pages = torch.randn(*shape, generator=gen).to(BF).cuda()
    order = torch.randperm(shape[-4], generator=gen)
    src, dst = order[:moves], order[moves:2 * moves]
    want = pages.clone()
    want[..., dst.cuda(), :, :, :] = want[..., src.cuda(), :, :, :]
    K.copy_pages(pages, src, dst.tolist())
    assert torch.equal(pages, want)


def test_copy_pages_one_source_many_targets_strided_pool_other_type(K):
    pool = torch.randint(-100, 100, (3, 12, 4, 2, 16, D), dtype=torch.int8, device="cuda")
    pages = pool[:, :, 1]  # pages at a wider stride
    want = pool.clone()
    for d in (2, 5, 11):
        want[:, d, 1] = want[:, 7, 1]
    K.copy_pages(pages, [7, 7, 7], [2, 5, 11])
    assert torch.equal(pool, want)
    with pytest.raises(K.SabreError, match="written twice"):
        K.copy_pages(pages, [1, 3], [4, 4])
    with pytest.raises(K.SabreError, match="read and written"):
        K.copy_pages(pages, [1, 4], [4, 6])
    assert torch.equal(pool, want)


def test_captured_step_replays_with_new_tables(K):
    """Store and decode captured once; replays follow the tensors' contents, and
    an eager call on another stream between them changes nothing."""
    args = make(13, [200, 64, 900], [1, 1, 1], 4, 2, 32, BF)
    q, kp, vp, table, sl, _ = args
    k, v = (torch.randn(3, 2, D, device="cuda").to(BF) for _ in range(2))
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.paged_store(k, v, kp, vp, table, sl)
        K.paged_decode(q, kp, vp, table, sl, out=out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.paged_store(k, v, kp, vp, table, sl)
        K.paged_decode(q, kp, vp, table, sl, out=out)
    for step in range(3):
        if step:
            sl.sub_(1)
            table.copy_(table.roll(1, 0))  # the sequences trade places
            sl.copy_(sl.roll(1, 0))
            q.copy_(torch.randn(q.shape, device="cuda").to(BF))
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            K.paged_decode(q[:1], kp, vp, table[:1], sl[:1])
        torch.cuda.current_stream().wait_stream(side)
        graph.replay()
        torch.cuda.synchronize()
        check(out, (q, kp, vp, table, sl, None))
    assert K.device_status(clear=True) == 0


def test_pool_past_32_bit_offsets(K):
    """Pages that start past 2^31 elements of the pool."""
    Hkv, ps = 8, 128
    P = 2 ** 31 // (Hkv * ps * D) + 40
    kp = torch.empty(P, Hkv, ps, D, dtype=BF, device="cuda")
    vp = torch.empty(P, Hkv, ps, D, dtype=BF, device="cuda")
    kp[:40], vp[:40], kp[-40:], vp[-40:] = 9.0, 9.0, 0.0, 0.0
    lens = [700, 129]
    table = torch.full((2, 7), -1, dtype=torch.int32)
    table[0, :6] = torch.arange(P - 1, P - 7, -1)
    table[1, :2] = torch.tensor([P - 20, P - 10])
    table = table.cuda()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 700, 829], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(829, Hkv, D, device="cuda").to(BF) for _ in range(2))
    K.paged_store(k, v, kp, vp, table, sl, starts)
    assert torch.equal(PO.gather(kp, table[0], 700)[0], k[:700].double())
    q = torch.randn(829, Hkv, D, device="cuda").to(BF)
    args = (q, kp, vp, table, sl, starts)
    check(K.paged_prefill(q, kp, vp, table, sl, starts), args, starts=starts)
    last = (q[[699, 828]],) + args[1:]
    check(K.paged_decode(*last[:5]), last)
    K.copy_pages(kp, [P - 1, P - 20], [P - 30, 3])
    assert torch.equal(kp[P - 30], kp[P - 1]) and torch.equal(kp[3], kp[P - 20])
    assert (kp[:3] == 9.0).all() and (kp[4:40] == 9.0).all()


def test_empty_calls(K):
    q, kp, vp, table, sl, starts = make(14, [20], [20], 2, 1, 16, BF)
    e = torch.empty(0, 2, D, dtype=BF, device="cuda")
    none = torch.empty(0, 2, dtype=torch.int32, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert K.paged_decode(e, kp, vp, none, zero[:0]).shape == (0, 2, D)
    assert K.paged_prefill(e, kp, vp, none, zero[:0], zero).shape == (0, 2, D)
    K.paged_store(e[:, :1], e[:, :1], kp, vp, none, zero[:0], zero)
    K.copy_pages(kp, [], [])


@pytest.mark.parametrize("call", ["decode", "prefill", "shares"])
def test_waits_that_run_out_end_the_call_and_the_next_one_is_correct(K, call):
    """Under a wait limit of 1 us the waits for copies and MMAs run out: the call
    completes, the status word says so, and a call at the default limit is right.
    (Every wait is bounded; nothing faults or hangs.)"""
    lens, news = ([9000, 3000], [1, 1]) if call == "decode" else ([2000, 900], [1900, 900])
    args = make(15, lens, news if call != "shares" else [70, 30], 8, 2, 64, BF)
    q, kp, vp, table, sl, starts = args

    def run():
        if call == "decode":
            return K.paged_decode(q, kp, vp, table, sl)
        return K.paged_prefill(q, kp, vp, table, sl, starts)

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
    check(out, args, starts=None if call == "decode" else starts)


def test_two_streams_and_two_captured_graphs_at_once(K):
    """Calls on two streams, and two captured calls replayed at once, each with the
    workspace of its own that it allocates."""
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    jobs = [make(16 + i, [3000 + 77 * i, 2900], [60, 5], 4, 2, 64, BF) for i in range(2)]
    graphs, outs = [], []
    for (q, kp, vp, table, sl, starts), side in zip(jobs, sides):
        K.paged_prefill(q, kp, vp, table, sl, starts)
        K.paged_decode(q[:2], kp, vp, table, sl)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append((K.paged_prefill(q, kp, vp, table, sl, starts), K.paged_decode(q[:2], kp, vp, table, sl)))
        graphs.append(g)
    for kind in ("streams", "graphs"):
        got = [None, None]
        for _ in range(5):
            for i, side in enumerate(sides):
                with torch.cuda.stream(side):
                    if kind == "graphs":
                        graphs[i].replay()
                        got[i] = outs[i]
                    else:
                        q, kp, vp, table, sl, starts = jobs[i]
                        got[i] = (K.paged_prefill(q, kp, vp, table, sl, starts), K.paged_decode(q[:2], kp, vp, table, sl))
        torch.cuda.synchronize()
        for job, (a, b) in zip(jobs, got):
            check(a, job, starts=job[5])
            check(b, (job[0][:2],) + job[1:])
    assert K.device_status(clear=True) == 0


def within(got, want, spread, ds, n):
    """The bound of `check` over n keys for results whose exact value is a number."""
    u = torch.finfo(got.dtype).eps / 2
    rel = u + 2 * (129 * ds + 16) * 2.0 ** -23 + n * 2.0 ** -23
    tol = rel[..., None] * spread + u * want.abs() + 2.0 ** -25 * n * (got.dtype == FP) * 6.0 + 1e-7
    some = ~want.isnan()
    err = (got.double() - want).abs()
    assert (err <= tol * 1.01)[some].all(), f"worst {(err / tol)[some].max():.2f} of its bound"


def poisoned(got, args, clean, window=None, prefix=0, starts=None):
    """NaN in exactly the results where the oracle has it; the others within the
    bound of `check` (score magnitudes without the bad values: a score of -inf is
    exact, its weight zero)."""
    kw = dict(window=window, prefix=prefix)
    want, spread, _ = PO.attention(*args[:5], starts, **kw)
    bad = want.isnan()
    assert not bad.all()
    assert torch.equal(got.isnan(), bad), f"{int(got.isnan().sum())} NaN for {int(bad.sum())}"
    within(got, want, spread, PO.attention(*clean[:5], starts, **kw)[2], float(args[4].max()))
    return int(bad.sum())


@pytest.mark.parametrize("what", ["q", "q inf", "k", "k inf"])
@pytest.mark.parametrize("lens,news,Hq,Hkv,ps,dtype,window,extra_cols", [
    ([130, 128, 70], [130, 128, 70], 4, 2, 32, BF, None, 1),        # a CTA each
    ([900, 1300, 80], [300, 200, 80], 4, 2, 64, BF, 100, 1),
    ([9000, 31], [20, 9], 7, 1, 16, FP, None, 1),                   # parts of pairs
    ([8400], [400], 56, 8, 64, BF, None, 1),                        # equal shares
    ([300, 20], [1, 1], 16, 8, 16, BF, None, 1),                    # decode: pairs whole and cut
    ([40000, 33], [1, 1], 7, 1, 64, BF, None, 1),
    ([2000, 900, 77] * 20, [1] * 60, 2, 2, 32, FP, 300, 1),
])
def test_nan_in_what_a_query_sees_reaches_its_result(K, what, lens, news, Hq, Hkv, ps, dtype, window, extra_cols):
    """A query with a NaN or an infinity, and a visible K row with one: the queries
    that meet it answer NaN, whatever way the work is split, and no other does."""
    clean = make(40, lens, news, Hq, Hkv, ps, dtype, window, extra_cols=extra_cols, drop=False)
    q, kp, vp, table, sl, starts = clean
    bad = float("inf") if "inf" in what else float("nan")
    if what[0] == "q":
        q = q.clone()
        q[q.shape[0] // 2, Hq - 1, 17] = bad
    else:  # in the first window of the last row of sequence 0, and in sight of few rows or many
        kp = kp.clone()
        j = lens[0] - 1 - min(news[0], 7)
        kp[table[0, j // ps], 0, j % ps, 100] = bad
    args = (q, kp, vp, table, sl, starts)
    calls = [(K.paged_prefill(*args, window_size=window), starts)]
    if max(news) == 1:
        calls.append((K.paged_decode(*args[:5], window_size=window), None))
    for got, st in calls:
        assert poisoned(got, args, clean, window, starts=st) or what == "k inf"
    assert K.device_status(clear=True) == 0


FAR = 2 ** 31 - 1


@pytest.mark.parametrize("window,prefix", [(100, 5000), (0, FAR), (FAR - 300, 33), (FAR - 300, FAR), (FAR - 1, 0),
                                           (100, 0), (None, 0)])
@pytest.mark.parametrize("times,extra_cols", [(40, 0), (10, 60)])  # 60: wide windows run in shares
def test_lengths_far_past_the_table(K, window, prefix, times, extra_cols):
    """Lengths up to the largest int32 over a table of a few rows: what the table
    holds of the window and the prefix is seen, the other sequences are as ever."""
    lens, news = [128, 256, 70] * times, [1, 3, 1] * times
    args = make(19, lens, news, 4, 2, 64, BF, extra_cols=extra_cols, drop=False)
    q, kp, vp, table, sl, starts = args
    sl[::3] = FAR
    sl[1::9] = FAR - 40
    n = table.shape[1] * 64
    table[:, 4:] = table[:, :1]  # the places past the rows hold some page of the pool
    kp.nan_to_num_(0.25), vp.nan_to_num_(0.5)
    kw = dict(window_size=window, num_prefix_tokens=prefix)
    o = dict(window=window, prefix=prefix)
    within(K.paged_prefill(q, kp, vp, table, sl, starts, **kw), *PO.attention(*args[:5], starts, **o), n)
    last = q[starts[1:].long() - 1]
    within(K.paged_decode(last, kp, vp, table, sl, **kw), *PO.attention(last, *args[1:5], **o), n)
    assert K.device_status(clear=True) == 0


@pytest.mark.parametrize("window", [FAR - 1, FAR - 2, FAR - 5, None])
@pytest.mark.parametrize("extra_cols", [1, 100])
def test_rows_before_their_sequence_under_the_widest_windows(K, window, extra_cols):
    """New rows that lie before their sequence see nothing, and hide nothing from the
    others of their row tile."""
    args = make(20, [40, 100, 64], [40, 100, 64], 4, 2, 16, BF, extra_cols=extra_cols)
    q, kp, vp, table, sl, starts = args
    sl[0], sl[2] = 10, 63
    out = K.paged_prefill(q, kp, vp, table, sl, starts, window_size=window)
    assert (out[:30] == 0).all() and (out[30:40] != 0).any(-1).all()
    check(out, args, window, starts=starts)
    assert K.device_status(clear=True) == 0


def test_launches_are_counted_as_they_are(K):
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

    def one(lens, news, Hq, Hkv, ps, extra_cols=0):
        return make(22, lens, news, Hq, Hkv, ps, BF, extra_cols=extra_cols)

    q, kp, vp, table, sl, starts = one([1], [1], 2, 1, 16)
    assert kernels(lambda: K.paged_decode(q, kp, vp, table, sl)) == 1
    assert kernels(lambda: K.paged_store(q[:, :1], q[:, 1:], kp, vp, table, sl)) == 1
    assert kernels(lambda: K.copy_pages(kp, [0, 1], [2, 3])) == 1
    assert kernels(lambda: K.copy_pages(kp, [], [])) == 0
    none, zero = table[:0], torch.zeros(1, dtype=torch.int32, device="cuda")
    assert kernels(lambda: K.paged_decode(q[:0], kp, vp, none, sl[:0])) == 0
    assert kernels(lambda: K.paged_prefill(q[:0], kp, vp, none, sl[:0], zero)) == 0
    assert kernels(lambda: K.paged_store(q[:0, :1], q[:0, :1], kp, vp, none, sl[:0], zero)) == 0
    pool = torch.zeros(2000, 1, 16, D, device="cuda", dtype=BF)
    assert kernels(lambda: K.copy_pages(pool, list(range(961)), list(range(1000, 1961)))) == 3
    for shape in (([70], [1], 2, 1, 16), ([9, 5], [1, 1], 2, 1, 16), ([9], [1], 2, 2, 16)):
        q, kp, vp, table, sl, starts = one(*shape)
        assert kernels(lambda: K.paged_decode(q, kp, vp, table, sl)) == 2
    for shape, n in ((([300], [300], 2, 1, 16), 1), (([9000], [20], 2, 2, 64), 2), (([100], [100], 2, 1, 16, 200), 2)):
        q, kp, vp, table, sl, starts = one(*shape)
        assert kernels(lambda: K.paged_prefill(q, kp, vp, table, sl, starts)) == n


def test_outputs_that_overlap_themselves_are_refused(K):
    q, kp, vp, table, sl, starts = make(23, [20, 9], [1, 1], 4, 2, 16, BF)
    for out in (q[:1].clone().expand(2, 4, D), q[:, :1].clone().expand(2, 4, D)):
        before = out.clone()
        with pytest.raises(K.SabreError, match="overlap"):
            K.paged_decode(q, kp, vp, table, sl, out=out)
        with pytest.raises(K.SabreError, match="overlap"):
            K.paged_prefill(q, kp, vp, table, sl, starts, out=out)
        assert torch.equal(out, before)
    one = torch.empty(1, 4, D, dtype=BF, device="cuda").expand(1, 4, D)  # a size of one repeats nothing
    K.paged_decode(q[:1], kp, vp, table[:1], sl[:1], out=one)
    check(one, (q[:1], kp, vp, table[:1], sl[:1], None))
