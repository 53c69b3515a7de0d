"""GPU tests of SabrePagedKVCache: the operators together, as a serving loop and
as the patched model use them."""

import pytest
import torch

from oracle import paged_oracle as PO
from test_gpu_api import _tiny_llama
from test_gpu_paged import check

pytestmark = pytest.mark.gpu

D = 128
BF = torch.bfloat16


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


@pytest.mark.parametrize("Hq,Hkv,ps,window,prefix", [(4, 4, 16, None, 0), (7, 1, 64, None, 0), (8, 2, 32, 150, 40)])
def test_serving_loop(cuda, Hq, Hkv, ps, window, prefix):
    """Prompts of different lengths, a fork, continuations, decode steps, pages
    given back and the pool compacted: every step's attention against the
    64-bit oracle over the same rows held contiguously."""
    from sabrecoder_b200 import kernels as K
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    gen = torch.Generator().manual_seed(ps)
    c = SabrePagedKVCache(batch_size=4, max_seq_len=2048, num_pages=3 * 2048 // ps, page_size=ps, num_layers=2,
                          num_kv_heads=Hkv, head_dim=D, window_size=window, num_prefix_tokens=prefix)
    c.pool.fill_(float("nan"))
    rows = [[torch.zeros(0, 2, Hkv, D, dtype=BF) for _ in range(4)] for _ in range(2)]

    def step(new):
        n = sum(new)
        c.extend(new)
        starts = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=cuda)
        for i, layer in enumerate(c.layers):
            kv = torch.randn(n, 2, Hkv, D, generator=gen).to(BF)
            for b in range(4):
                rows[i][b] = torch.cat([rows[i][b], kv[starts[b]:starts[b + 1]]])
            kv = kv.cuda()
            q = torch.randn(n, Hq, D, generator=gen).to(BF).cuda()
            K.paged_store(kv[:, 0], kv[:, 1], layer.k_pages, layer.v_pages, c.page_table, c.seq_lens, starts)
            if all(m == 1 for m in new):
                out = c.decode(i, q)
            else:
                out = K.paged_prefill(q, layer.k_pages, layer.v_pages, c.page_table, c.seq_lens, starts,
                                      window_size=window, num_prefix_tokens=prefix)
            # The oracle's cache: one page per sequence holding all its rows.
            T = max(max(c.lengths), 1)
            full = torch.zeros(4, 2, Hkv, T, D, dtype=BF)
            for b in range(4):
                full[b, :, :, :c.lengths[b]] = rows[i][b].permute(1, 2, 0, 3)
            full = full.cuda()
            check(out, (q, full[:, 0], full[:, 1], torch.arange(4, dtype=torch.int32, device=cuda)[:, None], c.seq_lens,
                        None), window, prefix, starts=starts)

    def copy(a, b):
        for i in range(2):
            rows[i][b] = rows[i][a]

    step([300, 77, 0, 500])
    step([1, 1, 1, 1])
    c.fork(3, 1)
    copy(3, 1)
    step([5, 40, 130, 1])
    for _ in range(ps + 3):
        c.extend([1, 1, 1, 1])
        c.truncate(0, c.lengths[0] - 1)
        for b in (1, 2, 3):
            c.truncate(b, c.lengths[b] - 1)
    step([1, 1, 1, 1])
    c.free(0)
    for i in range(2):
        rows[i][0] = rows[i][0][:0]
    c.fork(1, 2)
    copy(1, 2)
    c.compact()
    step([64, 1, 200, 3])
    step([1, 1, 1, 1])
    c.batch_select_indices([2, 2, 0, 1])
    for i in range(2):
        rows[i][:] = [rows[i][j] for j in (2, 2, 0, 1)]
    step([1, 1, 1, 1])
    step([2, 3, 0, 700])
    assert K.device_status(clear=True) == 0


def _model(cuda, H=4, Hkv=2):
    from sabrecoder_b200 import sabrecoder_llama as SL
    model = _tiny_llama(H, Hkv).to(cuda)
    SL.patch_model_with_sabrecoder_attention(model, None, block_size=64, window_size=192, num_prefix_tokens=64,
                                             num_suffix_tokens=128, global_last_k_chunks=0, max_chunk_tokens=128,
                                             verbose=False)
    return model


def _close(a, b):
    """bf16 models whose attention differs by rounding and order: within 3 % of the
    largest logit, the bound the model tests use."""
    assert (a.float() - b.float()).abs().max() <= 0.03 * b.float().abs().max()


@pytest.mark.parametrize("H,Hkv", [(2, 2), (4, 2), (8, 1)])
def test_patched_model_with_pages_matches_dynamic_cache(cuda, H, Hkv):
    """Sparse prompt, then decode steps over the pages, in lockstep with
    transformers' DynamicCache; a fork and a compaction on the way change nothing."""
    from transformers import DynamicCache

    from sabrecoder_b200 import sabrecoder_llama as SL
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    from sabrecoder_b200.sabrecoder_attention import StructureAwareMaskBuilder
    from sabrecoder_b200.spans import make_spans
    L = 500
    model = _model(cuda, H, Hkv)
    mb = StructureAwareMaskBuilder(None, block_size=64, window_size=192, num_prefix_tokens=64, num_suffix_tokens=128,
                                   global_last_k_chunks=0, max_chunk_tokens=128)
    bi, bc, _ = mb.build_block_indices_from_spans(make_spans(L, 8), cuda)
    ids = torch.randint(0, 512, (1, L), generator=torch.Generator().manual_seed(1)).to(cuda)
    ca = DynamicCache()
    cb = SabrePagedKVCache(model.config, batch_size=1, max_seq_len=L + 40, page_size=32, device=cuda)
    SL.set_current_code("<prompt>")
    SL.set_precomputed_blocks(bi, bc)
    try:
        with torch.no_grad():
            a = model(input_ids=ids, past_key_values=ca, use_cache=True, logits_to_keep=1).logits
            b = model(input_ids=ids, past_key_values=cb, use_cache=True, logits_to_keep=1).logits
            assert torch.equal(a, b)  # the same kernels on the same rows
            for step in range(20):
                tok = a[:, -1].argmax(-1, keepdim=True)
                a = model(input_ids=tok, past_key_values=ca, use_cache=True).logits
                b = model(input_ids=tok, past_key_values=cb, use_cache=True).logits
                _close(b, a)
                if step == 7:
                    cb.compact()
    finally:
        SL.clear_current_code()
        SL.clear_precomputed_blocks()
    assert cb.get_seq_length() == ca.get_seq_length() == L + 20


def test_prompt_in_chunks_and_a_forked_batch(cuda):
    """A prompt without structure in uneven chunks gives the whole prompt's logits;
    two forks of it continue apart, as two separate prompts would."""
    from transformers import DynamicCache

    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    model = _model(cuda)
    ids = torch.randint(0, 512, (1, 413), generator=torch.Generator().manual_seed(2)).to(cuda)
    tails = torch.randint(0, 512, (2, 30), generator=torch.Generator().manual_seed(3)).to(cuda)
    cache = SabrePagedKVCache(model.config, batch_size=1, max_seq_len=600, num_pages=40, page_size=16, device=cuda)
    with torch.no_grad():
        want = model(input_ids=ids, past_key_values=DynamicCache(), use_cache=True).logits
        got = [model(input_ids=part, past_key_values=cache, use_cache=True).logits for part in ids.split([200, 1, 212], 1)]
        _close(torch.cat(got, 1), want)
        cache.batch_repeat_interleave(2)
        assert cache.pages_in_use == -(-413 // 16)  # shared
        got = model(input_ids=tails, past_key_values=cache, use_cache=True).logits
        both = torch.cat([ids.expand(2, -1), tails], 1)
        want = model(input_ids=both, past_key_values=DynamicCache(), use_cache=True).logits[:, 413:]
        _close(got, want)


def test_generate_with_pages_and_a_window(cuda):
    """model.generate over a windowed paged cache, against the same steps fed one by
    one; the middle pages are given back."""
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    model = _model(cuda)
    ids = torch.randint(0, 512, (1, 600), generator=torch.Generator().manual_seed(4)).to(cuda)

    def new():
        return SabrePagedKVCache(model.config, batch_size=1, max_seq_len=700, page_size=16, window_size=128,
                                 num_prefix_tokens=32, device=cuda)

    with torch.no_grad():
        cache = new()
        # The ids hold the pad id: without a mask generate would take those for padding.
        out = model.generate(input_ids=ids, attention_mask=torch.ones_like(ids), past_key_values=cache,
                             max_new_tokens=10, min_new_tokens=10, do_sample=False, pad_token_id=0)
        assert out.shape == (1, 610) and cache.get_seq_length() == 609
        assert cache.pages_in_use <= 2 + 10
        again = new()
        # The head over one row, as generate runs it: the steps are then the same
        # kernels on the same values, and the tokens equal.
        logits = model(input_ids=ids, past_key_values=again, use_cache=True, logits_to_keep=1).logits
        for i in range(600, 609):
            assert int(logits[0, -1].float().argmax()) == int(out[0, i])
            logits = model(input_ids=out[:, i:i + 1], past_key_values=again, use_cache=True).logits


def test_sparse_generation_refuses_pages(cuda):
    from sabrecoder_b200 import sabrecoder_llama as SL
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    model = _tiny_llama(2, 2).to(cuda)
    SL.patch_model_with_sabrecoder_attention(model, None, use_sparse_for_generation=True, verbose=False)
    cache = SabrePagedKVCache(model.config, max_seq_len=64, device=cuda)
    with pytest.raises(ValueError, match="contiguous cache"):
        model(input_ids=torch.zeros(1, 8, dtype=torch.long, device=cuda), past_key_values=cache, use_cache=True)
    assert cache.get_seq_length() == 0


@pytest.mark.parametrize("eager_first", [True, False])
def test_captured_prefill_replays_after_many_other_lengths(cuda, eager_first):
    """A captured step of 6 rows (store and attention) keeps answering right after
    the cache served 99 other row counts and the memory they left was reused; and
    when 6 rows were first seen inside the capture, an eager step before the first
    replay is right too."""
    from sabrecoder_b200 import kernels as K
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    B, Hq, Hkv, n = 3, 4, 2, 6
    gen = torch.Generator().manual_seed(9)
    c = SabrePagedKVCache(batch_size=B, max_seq_len=512, page_size=16, num_layers=1, num_kv_heads=Hkv, head_dim=D)
    c.pool.zero_()
    layer = c.layers[0]
    q = torch.randn(B, n, Hq, D, generator=gen).to(BF).cuda()
    c.extend([40, 3, 100])
    c.pool.normal_()
    c.extend([n] * B)

    def right(out):
        starts = torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32, device=cuda)
        check(out.reshape(B * n, Hq, D), (q.view(B * n, Hq, D), layer.k_pages, layer.v_pages, c.page_table, c.seq_lens,
                                          None), starts=starts)

    if eager_first:
        right(c.prefill(0, q))
    else:
        c.prefill(0, q[:, :1])  # the kernels are loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.prefill(0, q)
    right(c.prefill(0, q))
    for m in range(1, 100):
        c._row_starts(m)
    junk = [torch.full((B + 1,), 10 ** 6, dtype=torch.int32, device=cuda) for _ in range(200)]
    for _ in range(3):
        c.extend([n, n, n])
        q.copy_(torch.randn(q.shape, generator=gen).to(BF))
        graph.replay()
        right(out)
    del junk
    assert K.device_status(clear=True) == 0


def test_model_steps_on_sequences_of_different_lengths(cuda):
    """A batch whose second sequence was cut back continues as two separate ones
    when it is given each sequence's positions, and is refused without them."""
    from transformers import DynamicCache

    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    model = _model(cuda)
    ids = torch.randint(0, 512, (2, 90), generator=torch.Generator().manual_seed(5)).to(cuda)
    cache = SabrePagedKVCache(model.config, batch_size=2, max_seq_len=200, page_size=16, device=cuda)
    with torch.no_grad():
        model(input_ids=ids[:, :70], past_key_values=cache, use_cache=True)
        cache.truncate(1, 33)
        with pytest.raises(ValueError, match="position_ids"):
            model(input_ids=ids[:, 70:75], past_key_values=cache, use_cache=True)
        assert cache.lengths == [70, 33]
        tokens = [list(ids[0, :70].tolist()), list(ids[1, :33].tolist())]
        for n in (5, 1, 1, 12):
            new = torch.stack([ids[0, 70:70 + n], ids[1, 40:40 + n]])
            at = torch.tensor([[len(t)] for t in tokens], device=cuda) + torch.arange(n, device=cuda)
            got = model(input_ids=new, past_key_values=cache, use_cache=True, position_ids=at).logits
            for b in range(2):
                tokens[b] += new[b].tolist()
                want = model(input_ids=torch.tensor([tokens[b]], device=cuda), past_key_values=DynamicCache(),
                             use_cache=True).logits[0, -n:]
                _close(got[b], want)
    assert cache.lengths == [89, 52]


def test_padded_batches_are_refused_and_plain_masks_are_not(cuda):
    """A left-padded batch in generate raises before a row is stored; the mask that
    eager attention always builds changes nothing."""
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    model = _model(cuda)
    ids = torch.randint(1, 512, (2, 50), generator=torch.Generator().manual_seed(6)).to(cuda)
    mask = torch.ones_like(ids)
    mask[1, :9] = 0

    def new():
        return SabrePagedKVCache(model.config, batch_size=2, max_seq_len=80, page_size=16, device=cuda)

    cache = new()
    with pytest.raises(ValueError, match="mask"):
        model.generate(input_ids=ids, attention_mask=mask, past_key_values=cache, max_new_tokens=4, do_sample=False,
                       pad_token_id=0)
    assert cache.lengths == [0, 0]
    with torch.no_grad():
        ca, cb = new(), new()
        for part in ids.split([30, 1, 19], 1):
            a = model(input_ids=part, past_key_values=ca, use_cache=True).logits
            model.config._attn_implementation = "eager"
            b = model(input_ids=part, past_key_values=cb, use_cache=True).logits
            model.config._attn_implementation = "sdpa"
            assert torch.equal(a, b)


@pytest.mark.parametrize("window,prefix", [(None, 0), (70, 20)])
def test_captured_step_stores_new_rows_where_the_tables_now_say(cuda, window, prefix):
    """Store and decode captured once: every replay writes the rows that k and v then
    hold to the places that table and lengths then name, and nothing else; decode sees
    them. Between replays extend takes pages, a sequence is forked, cut and the pool
    compacted. A decode on another stream at the same time answers as it would alone."""
    from sabrecoder_b200 import kernels as K
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    B, Hq, Hkv = 3, 8, 2
    gen = torch.Generator().manual_seed(21)
    c = SabrePagedKVCache(batch_size=B, max_seq_len=400, num_pages=60, page_size=16, num_layers=1, num_kv_heads=Hkv,
                          head_dim=D, window_size=window, num_prefix_tokens=prefix)
    layer = c.layers[0]

    def rand(*shape):
        return torch.randn(*shape, generator=gen).to(BF).cuda()

    c.pool.copy_(rand(*c.pool.shape))
    k, v, q = rand(B, Hkv, D), rand(B, Hkv, D), rand(B, Hq, D)
    c.extend([100, 31, 203])
    c.extend([1, 1, 1])
    K.paged_store(k, v, layer.k_pages, layer.v_pages, c.page_table, c.seq_lens)
    c.decode(0, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="capture"):
            c.append(0, k[:, None], v[:, None])
        K.paged_store(k, v, layer.k_pages, layer.v_pages, c.page_table, c.seq_lens)
        out = c.decode(0, q)
    side = torch.cuda.Stream()
    for step in range(20):
        if step == 5:
            c.fork(2, 0)
        if step == 9:
            c.truncate(1, 3)
        if step == 12:
            c.compact()
        c.extend([1, 1, 1])
        for t in (k, v, q):
            t.copy_(rand(*t.shape))
        out.fill_(9.0)
        table = c.page_table
        want = c.pool.clone()
        placed = PO.slots(table, c.seq_lens, None, 16, c.num_pages)
        assert len(placed) == B and len({p[1:] for p in placed}) == B
        for r, page, off in placed:
            want[0, 0, page, :, off], want[0, 1, page, :, off] = k[r], v[r]
        # Another decode meanwhile, over a copy of the pool and all rows but the last.
        before = (c.seq_lens - 1).clamp(min=0)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = K.paged_decode(q, want[0, 0], want[0, 1], table, before)
        torch.cuda.synchronize()
        assert torch.equal(c.pool, want)
        check(out, (q, want[0, 0], want[0, 1], table, c.seq_lens, None), window, prefix)
        check(beside, (q, want[0, 0], want[0, 1], table, before, None))
    assert K.device_status(clear=True) == 0
