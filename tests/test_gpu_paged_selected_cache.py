"""GPU tests of SabrePagedKVCache with selected pages and with pages lent to the
device, as a serving loop and as the patched model use it."""

import pytest
import torch

from oracle import paged_oracle as PO
from test_gpu_paged_cache import _close, _model
from test_gpu_paged_listed import check, check_lists

pytestmark = pytest.mark.gpu

D = 128
BF = torch.bfloat16


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda")


@pytest.mark.parametrize("Hq,Hkv,ps,topk,window,prefix,block", [(4, 4, 16, 3, None, 0, None), (7, 1, 64, 2, 70, 20, 16),
                                                                (16, 2, 32, 5, 40, 0, 5)])
def test_serving_loop_over_selected_pages(cuda, Hq, Hkv, ps, topk, window, prefix, block):
    """Prompts, a fork, chunks, steps, truncation and compaction: what each step
    selects and attends against the oracle over the pages and means that are there."""
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    gen = torch.Generator(device="cuda").manual_seed(ps)
    c = SabrePagedKVCache(batch_size=3, max_seq_len=2048, num_pages=3 * 1200 // ps, page_size=ps, num_layers=2,
                          num_kv_heads=Hkv, head_dim=D, topk_pages=topk, window_size=window, num_prefix_tokens=prefix,
                          query_block=block)
    c.pool.fill_(float("nan"))
    c.key_means.fill_(float("nan"))

    def step(n):
        for i, layer in enumerate(c.layers):
            k, v = (torch.randn(3, n, Hkv, D, generator=gen, device=cuda).to(BF) for _ in range(2))
            q = torch.randn(3, n, Hq, D, generator=gen, device=cuda).to(BF)
            c.append(i, k, v)
            for t, length in zip(c.tables, c.lengths):
                for p in range(length // ps):
                    want = layer.k_pages[t[p]].double().mean(1)
                    # 513 additions of fp32 at most, 2^-24 each of the sum of magnitudes.
                    size = layer.k_pages[t[p]].double().abs().mean(1)
                    assert ((layer.key_means[t[p]].double() - want).abs() <= 514 * 2.0 ** -24 * size).all()
            rows = q.reshape(3 * n, Hq, D)
            out = c.decode(i, q[:, 0]) if n == 1 else c.prefill(i, q)
            starts = None if n == 1 else torch.arange(4, dtype=torch.int32, device=cuda) * n
            b = 1 if n == 1 else c.block_rows(Hq)
            lists, counts = c.select(i, rows, starts)
            check_lists(lists, counts, PO.select(rows, layer.key_means, c.page_table, c.seq_lens, starts, page_size=ps,
                                                 topk=topk, block=b, window=window or 0, prefix=prefix))
            args = (rows, layer.k_pages, layer.v_pages, c.page_table, c.seq_lens, starts)
            check(out.reshape(3 * n, Hq, D), args, lists, counts, starts, b)

    step(300)
    step(1)
    c.truncate(0, 150)
    c.fork(2, 1)
    step(77)
    c.free(2)
    step(40)
    c.compact()
    for _ in range(3):
        step(1)
    assert all(p >= 0 for t in c.tables for p in t)


def test_all_pages_selected_is_the_dense_model(cuda):
    """topk_pages past the sequence: the model's logits are those of DynamicCache, over
    a prompt without structure, a chunk and decode steps."""
    from transformers import DynamicCache

    from sabrecoder_b200 import sabrecoder_llama as SL
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    model = _model(cuda, 8, 2)
    ids = torch.randint(0, 512, (1, 400), generator=torch.Generator().manual_seed(1)).to(cuda)
    ca = DynamicCache()
    cb = SabrePagedKVCache(model.config, batch_size=1, max_seq_len=500, page_size=16, device=cuda, topk_pages=100)
    dense, sparse = SL._DENSE_CALL_COUNT, SL._SPARSE_CALL_COUNT
    with torch.no_grad():
        a = model(input_ids=ids, past_key_values=ca, use_cache=True, logits_to_keep=1).logits
        b = model(input_ids=ids[:, :300], past_key_values=cb, use_cache=True, logits_to_keep=1).logits
        b = model(input_ids=ids[:, 300:], past_key_values=cb, use_cache=True, logits_to_keep=1).logits
        _close(b, a)
        before = SL._SPARSE_CALL_COUNT
        for _ in range(20):
            tok = a[:, -1].argmax(-1, keepdim=True)
            a = model(input_ids=tok, past_key_values=ca, use_cache=True).logits
            dense = SL._DENSE_CALL_COUNT
            b = model(input_ids=tok, past_key_values=cb, use_cache=True).logits
            assert SL._DENSE_CALL_COUNT == dense
            _close(b, a)
    assert SL._SPARSE_CALL_COUNT - before == 20 * model.config.num_hidden_layers and before > sparse
    assert cb.get_seq_length() == 420


def test_generate_over_selected_pages_with_sparse_generation(cuda):
    """use_sparse_for_generation takes a paged cache that selects pages; a copy of the
    cache goes on as the cache does."""
    import copy

    from sabrecoder_b200 import sabrecoder_llama as SL
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    model = _model(cuda, 4, 2)
    for layer in model.model.layers:
        layer.self_attn.use_sparse_for_generation = True
    ids = torch.randint(0, 512, (2, 300), generator=torch.Generator().manual_seed(2)).to(cuda)
    c = SabrePagedKVCache(model.config, batch_size=2, max_seq_len=400, page_size=16, device=cuda, topk_pages=2,
                          window_size=48, num_prefix_tokens=16)
    SL.clear_current_code()
    with torch.no_grad():
        model(input_ids=ids, past_key_values=c, use_cache=True, logits_to_keep=1)
        d = copy.deepcopy(c)
        c.compact()
        tok = ids[:, :1]
        for _ in range(18):
            a = model(input_ids=tok, past_key_values=c, use_cache=True).logits
            b = model(input_ids=tok, past_key_values=d, use_cache=True).logits
            assert torch.equal(a, b) and torch.isfinite(a).all()
            tok = a[:, -1].argmax(-1, keepdim=True)
    c = SabrePagedKVCache(model.config, batch_size=2, max_seq_len=400, page_size=16, device=cuda, topk_pages=2)
    # Without a mask transformers takes the tokens that are the padding's for padding,
    # which pages refuse.
    out = model.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=c, max_new_tokens=8,
                         do_sample=False, pad_token_id=0)
    assert out.shape == (2, 308)


@pytest.mark.parametrize("topk", [None, 3])
def test_captured_steps_make_their_own_room(cuda, topk):
    """A graph of whole steps (room, rows, means, attention of two layers) against the
    same rows appended by the host; then the host goes on from where it ended."""
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    gen = torch.Generator(device="cuda").manual_seed(9)
    B, Hq, Hkv, ps = 4, 14, 2, 16

    def new():
        return SabrePagedKVCache(batch_size=B, max_seq_len=512, num_pages=100, page_size=ps, num_layers=2,
                                 num_kv_heads=Hkv, head_dim=D, topk_pages=topk, window_size=40 if topk else None)

    a, b = new(), new()
    kv = torch.empty(2, 2, B, Hkv, D, dtype=BF, device=cuda)
    q = torch.empty(2, B, Hq, D, dtype=BF, device=cuda)
    prompt = torch.randn(2, 2, B, 100, Hkv, D, generator=gen, device=cuda).to(BF)
    for c in (a, b):
        for i in range(2):
            c.append(i, prompt[i, 0], prompt[i, 1])
        c.truncate(1, 37)
    b.fork(0, 3)
    a.fork(0, 3)
    one = torch.ones(B, dtype=torch.int32, device=cuda)

    def on_device():
        starts, slots, positions = b.extend_on_device(one, B)
        outs = []
        for i in range(2):
            b.store_rows(i, kv[i, 0], kv[i, 1], starts, slots)
            outs.append(b.decode(i, q[i]))
        return outs, positions

    def by_host():
        outs = []
        for i in range(2):
            a.append(i, kv[i, 0][:, None], kv[i, 1][:, None])
            outs.append(a.decode(i, q[i]))
        return outs

    def fill():
        for t in (kv, q):
            t.copy_(torch.randn(t.shape, generator=gen, device=cuda))

    b.lend()
    fill()
    got, _ = on_device()
    for x, y in zip(got, by_host()):
        assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, positions = on_device()
    for _ in range(60):
        fill()
        graph.replay()
        assert positions.tolist() == a.lengths
        for x, y in zip(got, by_host()):
            assert torch.equal(x, y)
    b.settle()
    assert a.lengths == b.lengths and a.pages_in_use == b.pages_in_use
    a.truncate(2, 90)
    b.truncate(2, 90)
    b.compact()
    for _ in range(20):
        fill()
        ours = []
        for i in range(2):
            b.append(i, kv[i, 0][:, None], kv[i, 1][:, None])
            ours.append(b.decode(i, q[i]))
        for x, y in zip(ours, by_host()):
            assert torch.equal(x, y)
    b.lend(5)
    graph.replay()  # the graph's tensors are the cache's still
    b.settle()
    assert b.lengths == [n + 1 for n in a.lengths]


def test_a_graph_that_runs_out_of_pages_stands_still(cuda):
    """Steps without room change nothing and write nowhere; after more pages are lent
    the same graph goes on."""
    from sabrecoder_b200 import kernels as K
    from sabrecoder_b200.paged_cache import SabrePagedKVCache
    c = SabrePagedKVCache(batch_size=2, max_seq_len=64, num_pages=4, page_size=16, num_layers=1, num_kv_heads=1,
                          head_dim=D, topk_pages=1)
    c.pool.zero_()
    c.lend(2)
    one = torch.ones(2, dtype=torch.int32, device=cuda)
    k = torch.ones(2, 1, D, dtype=BF, device=cuda)

    def step():
        starts, slots, _ = c.extend_on_device(one, 2)
        c.store_rows(0, k, k, starts, slots)
        return slots

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots = step()
    for _ in range(15):
        graph.replay()
    assert c.seq_lens.tolist() == [16, 16] and K.device_status(clear=True) == 0
    pool = c.pool.clone()
    graph.replay()
    assert slots.tolist() == [-1, -1] and torch.equal(pool, c.pool) and K.device_status(clear=True) == 8
    c.settle()
    assert c.lengths == [16, 16]
    c.lend()
    graph.replay()
    c.settle()
    assert c.lengths == [17, 17] and K.device_status(clear=True) == 0
    graph.replay()  # nothing is lent: no row is added, although the last pages have room
    assert slots.tolist() == [-1, -1] and c.seq_lens.tolist() == [17, 17] and K.device_status(clear=True) == 8
