"""Paged KV cache for the patched model and for serving loops.

Sequences of different lengths share one pool of pages, allocated once:
``pool[layer, 0 | 1 (K | V), page, kv head, row, d]``. The host keeps the free
list, the pages' reference counts and every sequence's table; the device
tensors ``page_table`` and ``seq_lens`` (static addresses, so a captured step
follows them) are what the kernels read.

* :meth:`extend` makes room for new rows; a page that another sequence still
  shares is copied first (all layers in one launch).
* :meth:`fork` lets a sequence continue another one's rows without a copy.
* :meth:`truncate`, :meth:`free` and :meth:`compact` give pages back and move the
  live ones to the front of the pool.
* With ``window_size`` (and ``num_prefix_tokens`` first tokens that stay
  visible) a query at position i sees key j <= i when ``i - j <= window_size``
  or ``j < num_prefix_tokens``; pages that no later query can see are released.
* With ``topk_pages`` queries read selected pages: those of the window and the
  prefix (the window's pages are the query's own without ``window_size``) and the
  ``topk_pages`` others whose mean key suits them best. All pages are kept.
* :meth:`lend` hands free pages to the device, where :meth:`extend_on_device`
  makes room for rows, also inside a capture, until :meth:`settle` brings the host
  up to date (``lengths`` and ``tables`` stand still meanwhile).

As a transformers ``Cache`` it takes the same number of new rows for every
sequence of the batch; the patched attention writes its rows through
:meth:`append` and attends with :meth:`decode` / :meth:`prefill`. Padding masks
are refused: sequences of different lengths keep their own lengths, and a model
that continues them needs ``position_ids`` that go on from each.
"""

from __future__ import annotations

import weakref
from typing import Dict, List, Optional, Sequence, Tuple

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from . import kernels as K


def _capturing(pool: torch.Tensor) -> bool:
    """Whether calls on the current stream are being captured into a graph."""
    return pool.is_cuda and torch.cuda.is_current_stream_capturing()


class SabrePagedCacheLayer(CacheLayerMixin):
    """One layer of a :class:`SabrePagedKVCache`: its pages and the step it is at."""

    is_compileable = False
    is_sliding = False

    def __init__(self, cache: "SabrePagedKVCache", index: int):
        super().__init__()
        self._ref, self.index, self.step = weakref.ref(cache), index, 0
        self.max_cache_len = cache.max_seq_len
        self.k_pages, self.v_pages = cache.pool[index, 0], cache.pool[index, 1]
        self.key_means = None if cache.key_means is None else cache.key_means[index]
        self.dtype, self.device = cache.pool.dtype, cache.pool.device
        self.keys = self.values = None  # never held as one tensor
        self.is_initialized = True

    @property
    def _cache(self) -> "SabrePagedKVCache":
        cache = self._ref()
        if cache is None:
            raise ValueError("the SabrePagedKVCache of this layer is gone")
        return cache

    @property
    def max_batch_size(self) -> int:
        return self._cache.batch_size

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        return None

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args, **kwargs):
        """Stores new rows ``[B, Hkv, n, D]`` and returns all rows gathered into
        ``[B, Hkv, T, D]`` (for attention that does not read pages)."""
        c = self._cache
        if c.window_size is not None:
            raise ValueError("SabrePagedKVCache with a window serves the patched attention only (pages are dropped)")
        if c.topk_pages is not None:
            raise ValueError("SabrePagedKVCache with topk_pages serves the patched attention only")
        c._not_lent()
        if len(set(c.lengths)) > 1:
            raise ValueError(f"SabrePagedKVCache: sequences of different lengths ({c.lengths}) serve the patched "
                             f"attention only (its mask knows one length)")
        c.append(self.index, key_states.transpose(1, 2), value_states.transpose(1, 2))
        return c.gather(self.index)

    def get_seq_length(self) -> int:
        c = self._cache
        return max(c._lengths_now(), default=0) - (c.step_rows if self.step < c.step else 0)

    def get_mask_sizes(self, query_length) -> Tuple[int, int]:
        n = query_length if isinstance(query_length, int) else query_length.shape[0]
        return self.get_seq_length() + n, 0

    def get_max_cache_shape(self) -> int:
        return self._cache.max_seq_len

    def reset(self) -> None:
        self._cache.reset()

    def crop(self, max_length: int) -> None:
        self._cache.crop(max_length)

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        self._cache.reorder_cache(beam_idx)


class SabrePagedKVCache(Cache):
    """``SabrePagedKVCache(config, batch_size=B, num_pages=P, max_seq_len=T)`` or
    with explicit ``num_layers`` / ``num_kv_heads`` / ``head_dim``.

    ``num_pages`` is shared by all sequences (default: enough for every
    sequence at ``max_seq_len``). ``topk_pages``: attention over selected pages,
    one choice for each KV head and up to ``query_block`` new rows (default: the
    largest power of two that fills a row tile of the prompt kernel, 128 rows over
    the heads of a group)."""

    def __init__(self, config=None, *, batch_size: int = 1, max_seq_len: int, num_pages: Optional[int] = None,
                 page_size: int = 64, window_size: Optional[int] = None, num_prefix_tokens: int = 0, device="cuda",
                 dtype: torch.dtype = torch.bfloat16, num_layers: Optional[int] = None,
                 num_kv_heads: Optional[int] = None, head_dim: Optional[int] = None, topk_pages: Optional[int] = None,
                 query_block: Optional[int] = None):
        if config is not None:
            num_layers = num_layers or config.num_hidden_layers
            num_kv_heads = num_kv_heads or config.num_key_value_heads
            head_dim = head_dim or getattr(config, "head_dim", None) or config.hidden_size // config.num_attention_heads
        if not (num_layers and num_kv_heads and head_dim):
            raise ValueError("SabrePagedKVCache needs a config or num_layers/num_kv_heads/head_dim")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} must be a power of two from 16 to 1024")
        if batch_size < 1 or max_seq_len < 1:
            raise ValueError("SabrePagedKVCache needs batch_size >= 1 and max_seq_len >= 1")
        if (window_size is not None and window_size < 0) or num_prefix_tokens < 0:
            raise ValueError("window_size and num_prefix_tokens must not be negative")
        if topk_pages is not None and topk_pages < 0:
            raise ValueError(f"topk_pages {topk_pages} must not be negative")
        if query_block is not None and (topk_pages is None or not 1 <= query_block <= 128):
            raise ValueError(f"query_block {query_block} goes with topk_pages, from 1 to 128")
        self.page_size, self.max_seq_len = int(page_size), int(max_seq_len)
        self.topk_pages, self.query_block = topk_pages, query_block
        self.window_size, self.num_prefix_tokens = window_size, int(num_prefix_tokens)
        self.max_pages = -(-self.max_seq_len // self.page_size)
        self.num_pages = int(num_pages) if num_pages is not None else batch_size * self.max_pages
        if self.num_pages < 1:
            raise ValueError("SabrePagedKVCache needs at least one page")
        if topk_pages is not None and self.max_pages > 32768:
            raise ValueError(f"topk_pages selects among at most 32768 pages of a sequence, not {self.max_pages}")
        self.pool = torch.empty(num_layers, 2, self.num_pages, num_kv_heads, self.page_size, head_dim, dtype=dtype,
                                device=device)
        # The mean key of every full page; other pages' are not read.
        self.key_means = None
        if topk_pages is not None:
            self.key_means = torch.empty(num_layers, self.num_pages, num_kv_heads, head_dim, dtype=torch.float32,
                                         device=device)
        # Pages lent to the device, as a stack, and how many of them it still has (-1:
        # none are lent, and a graph that extends on the device changes nothing).
        self.free_pages = torch.zeros(self.num_pages, dtype=torch.int32, device=device)
        self.free_count = torch.full((1,), -1, dtype=torch.int32, device=device)
        self._lent: Optional[List[int]] = None
        self.refs: List[int] = [0] * self.num_pages
        self.unused: List[int] = list(range(self.num_pages - 1, -1, -1))  # the lowest page is taken first
        self.step = 0       # steps begun (a step: new rows of every layer)
        self.step_rows = 0  # new rows per sequence of the last step
        self._starts: dict = {}
        # Table entries before `tops` are not looked at for dropping any more.
        self._top0 = -(-self.num_prefix_tokens // self.page_size)
        self._batch([[] for _ in range(batch_size)], [0] * batch_size, [self._top0] * batch_size)
        super().__init__(layers=[SabrePagedCacheLayer(self, i) for i in range(num_layers)])

    # -- host state -------------------------------------------------------

    def _batch(self, tables: List[List[int]], lengths: List[int], tops: List[int]) -> None:
        """Takes over the sequences' tables; new device tensors when their number changes."""
        grown = getattr(self, "tables", None) is None or len(tables) != len(self.tables)
        self.tables, self.lengths, self.tops = tables, lengths, tops
        if grown:
            dev = self.pool.device
            self._host = torch.full((len(tables), self.max_pages), -1, dtype=torch.int32)
            self.page_table = self._host.to(dev, copy=True)
            self.seq_lens = torch.zeros(len(tables), dtype=torch.int32, device=dev)
            self._starts.clear()
            self._columns = self.max_pages, self.page_table
        self._upload(range(len(tables)))

    def _upload(self, seqs) -> None:
        """Brings the device's tables and lengths in line; `seqs`: the tables that changed."""
        rows = self._host.numpy()
        for b in seqs:
            n = len(self.tables[b])
            rows[b, :n] = self.tables[b]
            rows[b, n:] = -1
        self.page_table.copy_(self._host)
        self.seq_lens.copy_(torch.tensor(self.lengths, dtype=torch.int32))

    def _release(self, page: int) -> None:
        if page >= 0:
            self.refs[page] -= 1
            if self.refs[page] == 0:
                self.unused.append(page)

    def _outside_captures(self) -> None:
        """Tables and lengths change on the host and the device together: inside a
        capture the device's part would only be recorded, and run at every replay."""
        if _capturing(self.pool):
            raise ValueError("SabrePagedKVCache: sequences do not change inside a capture (extend, and the like, go "
                             "between replays; a captured step stores with paged_store)")
        self._not_lent()

    def _not_lent(self) -> None:
        """For what needs the sequences' lengths on the host."""
        if self._lent is not None:
            raise ValueError("SabrePagedKVCache: pages are lent to the device, which changes the sequences; settle() "
                             "comes first")

    def _lengths_now(self) -> List[int]:
        """The sequences' lengths; while pages are lent those on the device, behind what
        the current stream does."""
        if self._lent is None:
            return self.lengths
        if _capturing(self.pool):
            raise ValueError("SabrePagedKVCache: pages are lent to the device, whose lengths a capture cannot read")
        return self.seq_lens.tolist()

    def _seq(self, seq: int) -> int:
        """A sequence's index (from the end when negative)."""
        n = self.batch_size
        if not -n <= seq < n:
            raise ValueError(f"SabrePagedKVCache has no sequence {seq} (it holds {n})")
        return int(seq) % n

    @property
    def batch_size(self) -> int:
        return len(self.lengths)

    @property
    def pages_in_use(self) -> int:
        return self.num_pages - len(self.unused)

    @property
    def _drop_window(self) -> Optional[int]:
        """The window outside of which pages are given back."""
        return self.window_size if self.topk_pages is None else None

    # -- sequences --------------------------------------------------------

    def extend(self, new: Sequence[int]) -> None:
        """Makes room for ``new[b]`` more rows of each sequence (to be stored at
        its end). Raises ValueError, changing nothing, when a sequence or the
        pool is full."""
        self._outside_captures()
        ps, w = self.page_size, self._drop_window
        if len(new) != self.batch_size or min(new, default=0) < 0:
            raise ValueError(f"extend needs {self.batch_size} row counts >= 0")
        need, dropped, shared = 0, [], {}
        for b, n in enumerate(new):
            length, table = self.lengths[b], self.tables[b]
            if length + n > self.max_seq_len:
                raise ValueError(f"SabrePagedKVCache: sequence {b} is full: {length} + {n} > {self.max_seq_len}")
            if n == 0:
                continue
            need += -(-(length + n) // ps) - len(table)
            if length % ps:  # the last page is written: its own copy, unless it is the last to share it
                page = table[length // ps]
                shared[page] = shared.get(page, 0) + 1
            if w is not None:
                # What the last row sees is kept too: it may be asked again (truncate).
                dropped += [(b, p) for p in range(self.tops[b], max(0, length - 1 - w) // ps)]
        need += sum(min(count, self.refs[page] - 1) for page, count in shared.items())
        freed = {}
        for b, p in dropped:
            freed[self.tables[b][p]] = freed.get(self.tables[b][p], 0) + 1
        room = len(self.unused) + sum(1 for page, count in freed.items() if count == self.refs[page])
        if need > room:
            raise ValueError(f"SabrePagedKVCache is out of pages: {need} needed, {room} free")
        for b, p in dropped:
            self._release(self.tables[b][p])
            self.tables[b][p] = -1
            self.tops[b] = p + 1
        src, dst = [], []
        changed = {b for b, _ in dropped}
        for b, n in enumerate(new):
            length, table = self.lengths[b], self.tables[b]
            if n and length % ps and self.refs[table[length // ps]] > 1:
                page = self.unused.pop()
                src.append(table[length // ps])
                dst.append(page)
                self.refs[page] = 1
                self._release(table[length // ps])
                table[length // ps] = page
                changed.add(b)
            while len(table) * ps < length + n:
                page = self.unused.pop()
                self.refs[page] = 1
                table.append(page)
                changed.add(b)
            self.lengths[b] = length + n
        if src:
            K.copy_pages(self.pool, src, dst)
        if changed or len(set(new)) > 1:
            self._upload(changed)
        else:
            self.seq_lens.add_(new[0])

    def fork(self, src: int, dst: int) -> None:
        """Sequence ``dst`` gives its rows back and continues those of ``src``; the
        pages are shared until one of them writes."""
        self._outside_captures()
        src, dst = self._seq(src), self._seq(dst)
        if src == dst:
            return
        for page in self.tables[src]:
            if page >= 0:
                self.refs[page] += 1
        for page in self.tables[dst]:
            self._release(page)
        self.tables[dst], self.lengths[dst], self.tops[dst] = list(self.tables[src]), self.lengths[src], self.tops[src]
        self._upload([dst])

    def truncate(self, seq: int, length: int) -> None:
        """Drops the rows of a sequence from ``length`` on."""
        self._truncate({self._seq(seq): length})

    def _truncate(self, lengths: Dict[int, int]) -> None:
        """{sequence: new length}; raises, changing nothing, where rows that the new
        last row sees are dropped already."""
        self._outside_captures()
        ps = self.page_size
        for b, length in lengths.items():
            lengths[b] = length = max(0, min(int(length), self.lengths[b]))
            if self._drop_window is not None:
                first = max(0, length - 1 - self.window_size) // ps
                if any(p < 0 for p in self.tables[b][first:-(-length // ps)]):
                    raise ValueError(f"SabrePagedKVCache: rows in the window before {length} of sequence {b} are "
                                     f"dropped already")
        for b, length in lengths.items():
            keep = -(-length // ps)
            for page in self.tables[b][keep:]:
                self._release(page)
            del self.tables[b][keep:]
            self.lengths[b], self.tops[b] = length, max(self._top0, min(self.tops[b], keep))
        self._upload(lengths)

    def free(self, seq: int) -> None:
        """Gives all rows of a sequence back."""
        self.truncate(seq, 0)

    def compact(self) -> int:
        """Moves the live pages to the lowest places of the pool (all layers in one
        launch per 480 pages); returns how many moved."""
        self._outside_captures()
        live = self.pages_in_use
        src = [p for p in range(live, self.num_pages) if self.refs[p]]
        dst = [p for p in range(live) if not self.refs[p]]
        if not src:
            return 0
        K.copy_pages(self.pool, src, dst)
        if self.key_means is not None:
            K.copy_pages(self.key_means.unsqueeze(3), src, dst)
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        for t in self.tables:
            t[:] = [to.get(p, p) for p in t]
        self.unused = list(range(self.num_pages - 1, live - 1, -1))
        self._upload(range(self.batch_size))
        return len(src)

    # -- steps without the host -------------------------------------------

    def lend(self, num_pages: Optional[int] = None) -> int:
        """Hands free pages (all of them by default) to the device, which takes them
        in :meth:`extend_on_device`; returns how many. Until :meth:`settle` the
        sequences are the device's: calls that change them raise. Last pages that
        sequences share are copied first."""
        self._outside_captures()
        ps = self.page_size
        copies, count = [], {}
        for b, n in enumerate(self.lengths):
            if n % ps:
                page = self.tables[b][n // ps]
                count[page] = count.get(page, 0) + 1
                if self.refs[page] - count[page] > 0:  # all but the last to share it get their own
                    copies.append((b, page))
        free = len(self.unused) - len(copies)
        want = free if num_pages is None else int(num_pages)
        if want < 0 or want > free:
            raise ValueError(f"SabrePagedKVCache: {want} pages cannot be lent: {len(self.unused)} are free and "
                             f"{len(copies)} are needed for copies of shared pages")
        src, dst = [], []
        for b, page in copies:
            src.append(page)
            dst.append(self.unused.pop())
            self.refs[dst[-1]] = 1
            self._release(page)
            self.tables[b][self.lengths[b] // ps] = dst[-1]
        if src:
            K.copy_pages(self.pool, src, dst)
            self._upload([b for b, _ in copies])
        self._lent = self.unused[len(self.unused) - want:]
        del self.unused[len(self.unused) - want:]
        self.free_pages[:want].copy_(torch.tensor(self._lent, dtype=torch.int32))
        self.free_count.fill_(want)
        return want

    def extend_on_device(self, new_rows: torch.Tensor, num_rows: int
                         ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Makes room for ``new_rows`` (int32 ``[B]``, on the device) more rows of each
        sequence, num_rows or fewer in all, from the pages lent: ``(q_start, slots,
        positions)`` as :func:`kernels.paged_extend` gives them. May be captured. A
        sequence has no room past max_seq_len rows."""
        if self._lent is None:
            raise ValueError("SabrePagedKVCache: lend() pages to the device first")
        # Where whole pages make up max_seq_len the table's width is the limit.
        limit = dict(max_seq_len=self.max_seq_len) if self.max_seq_len % self.page_size else {}
        return K.paged_extend(new_rows, self.page_table, self.seq_lens, self.free_pages, self.free_count,
                              page_size=self.page_size, num_pages=self.num_pages, num_rows=num_rows, **limit)

    def store_rows(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, q_start: torch.Tensor,
                   slots: torch.Tensor) -> None:
        """Stores the rows k, v ``[num_rows, Hkv, D]`` of a step on the device in one
        layer, where :meth:`extend_on_device` made room for them."""
        layer = self.layers[layer_idx]
        K.paged_store_slots(k, v, layer.k_pages, layer.v_pages, slots)
        if layer.key_means is not None:
            K.paged_key_means(layer.k_pages, layer.key_means, self.page_table, self.seq_lens, q_start,
                              num_rows=k.shape[0])

    def settle(self) -> None:
        """Takes over what the device did with the pages lent and takes the others back.
        Waits for all of the device's streams: steps may have been replayed on any of
        them, and later ones, on any of them, find nothing lent. Nothing happens when
        none are lent."""
        if _capturing(self.pool):
            raise ValueError("SabrePagedKVCache: settle() reads from the device, which a capture cannot")
        if self._lent is None:
            return
        wait = torch.cuda.synchronize if self.pool.is_cuda else lambda device: None
        wait(self.pool.device)
        ps, lent = self.page_size, self._lent
        left = int(self.free_count)
        lengths, rows = self.seq_lens.tolist(), self.page_table.tolist()
        taken = {}
        for b, n in enumerate(lengths):
            if n < self.lengths[b] or n > self.max_seq_len:
                raise ValueError(f"SabrePagedKVCache: sequence {b} went from {self.lengths[b]} rows to {n} on the device")
            for col in range(len(self.tables[b]), -(-n // ps)):
                taken[rows[b][col]] = taken.get(rows[b][col], 0) + 1
        if taken != {page: 1 for page in lent[left:]} or not 0 <= left <= len(lent):
            raise ValueError("SabrePagedKVCache: the device's tables do not match the pages lent to it")
        for b, n in enumerate(lengths):
            self.tables[b] += rows[b][len(self.tables[b]):-(-n // ps)]
        for page in taken:
            self.refs[page] = 1
        self.unused += lent[:left]
        self.lengths, self._lent = lengths, None
        self.free_count.fill_(-1)
        wait(self.pool.device)
        # The host's copies of the tables; the device has them.
        host = self._host.numpy()
        for b, t in enumerate(self.tables):
            host[b, :len(t)] = t

    # -- one step ---------------------------------------------------------

    def check_step(self, layer_idx: int, n: int, position_ids: Optional[torch.Tensor],
                   attention_mask: Optional[torch.Tensor] = None) -> None:
        """Raises ValueError when a step of n rows cannot be what the model takes it
        for. A model derives its positions from the longest sequence; when the lengths
        differ it must have been given each sequence's own. A mask (if there is one:
        additive, boolean, or one flag a key) may not say more than the cache does:
        it must show the keys that each query sees here and none of its future. Both
        are read from the device, once a step."""
        self._not_lent()
        if self.layers[layer_idx].step != self.step:
            return
        if len(set(self.lengths)) > 1:
            own = [[length + i for i in range(n)] for length in self.lengths]
            if position_ids is None or position_ids.tolist() != own:
                raise ValueError(f"SabrePagedKVCache holds sequences of different lengths ({self.lengths}): their new "
                                 f"rows need position_ids that go on from each one's length")
        if attention_mask is not None and not self._mask_fits(attention_mask, n):
            raise ValueError("SabrePagedKVCache: attention over pages is causal (within the cache's window) over all "
                             "rows of a sequence; this attention mask is not (padding must not be stored: give each "
                             "sequence its own rows)")

    def _mask_fits(self, mask: torch.Tensor, n: int) -> bool:
        top = max(self.lengths)
        if not isinstance(mask, torch.Tensor):
            return False
        if mask.shape[-1] < top + n or mask.dim() not in (2, 4) or (mask.dim() == 4 and mask.shape[2] != n):
            return False
        see = (mask == 0 if mask.is_floating_point() and mask.dim() == 4 else mask != 0)[..., :top + n]
        if mask.dim() == 2:
            see = see[:, None, None]
        lengths = torch.tensor(self.lengths if len(set(self.lengths)) > 1 else self.lengths[:1], device=mask.device)
        row = torch.arange(n, device=mask.device)[:, None]
        j = torch.arange(top + n, device=mask.device)
        i = lengths[:, None, None, None] + row
        own = j <= i
        if self._drop_window is not None:
            own = own & ((i - j <= self.window_size) | (j < self.num_prefix_tokens))
        wrong = own & ~see
        if mask.dim() == 4:
            wrong = wrong | (see & (j > top + row))
        return not bool(wrong.any())

    def append(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """Stores the rows k, v ``[B, n, Hkv, D]`` of a step in one layer; the
        step's first layer makes room for them."""
        layer = self.layers[layer_idx]
        B, n = k.shape[:2]
        if B != self.batch_size:
            raise ValueError(f"SabrePagedKVCache holds {self.batch_size} sequences (got rows of {B})")
        self._not_lent()  # a step that was begun before the loan does not go on in it
        if layer.step == self.step:
            pool = self.pool
            for x in (k, v):  # before room is made for them
                if x.shape != (B, n, pool.shape[3], pool.shape[5]) or x.dtype != pool.dtype or x.device != pool.device:
                    raise ValueError(f"SabrePagedKVCache: rows {tuple(x.shape)} ({x.dtype}, {x.device}) for pages of "
                                     f"{pool.shape[3]} heads of {pool.shape[5]} ({pool.dtype}, {pool.device})")
            self.extend([n] * B)
            self.step, self.step_rows = self.step + 1, n
        elif layer.step != self.step - 1 or n != self.step_rows:
            raise ValueError(f"SabrePagedKVCache: layer {layer_idx} is out of step")
        K.paged_store(k.reshape(B * n, *k.shape[2:]), v.reshape(B * n, *v.shape[2:]), layer.k_pages, layer.v_pages,
                      self.page_table, self.seq_lens, self._row_starts(n))
        if layer.key_means is not None:
            K.paged_key_means(layer.k_pages, layer.key_means, self.page_table, self.seq_lens, self._row_starts(n),
                              num_rows=B * n)
        layer.step = self.step

    def _row_starts(self, n: int) -> torch.Tensor:
        """Row starts of a step of n rows each. Kept while the number of sequences
        stays, since a captured call holds their address (at most max_seq_len small
        tensors). First asked for inside a capture they belong to its graph, which
        fills them on every replay, and to nobody else."""
        t = self._starts.get(n)
        if t is None:
            t = torch.arange(self.batch_size + 1, dtype=torch.int32, device=self.pool.device) * n
            if not _capturing(self.pool):
                self._starts[n] = t
        return t

    def decode(self, layer_idx: int, q: torch.Tensor, softmax_scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of one new token per sequence, q ``[B, Hq, D]``, over a layer."""
        layer = self.layers[layer_idx]
        if self.topk_pages is not None:
            table = self._columns_in_use()
            lists, counts = self.select(layer_idx, q)
            return K.paged_decode_listed(q, layer.k_pages, layer.v_pages, table, self.seq_lens, lists, counts,
                                         softmax_scale=softmax_scale, out=out)
        return K.paged_decode(q, layer.k_pages, layer.v_pages, self.page_table, self.seq_lens,
                              window_size=self.window_size, num_prefix_tokens=self.num_prefix_tokens,
                              softmax_scale=softmax_scale, out=out)

    def select(self, layer_idx: int, q: torch.Tensor, q_start: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
        """The pages (as lists of table columns) that the rows q ``[N, Hq, D]`` of a
        step read in a layer: one new token per sequence, or the last
        ``q_start[b+1] - q_start[b]`` rows of each in blocks of :meth:`block_rows`."""
        if self.topk_pages is None:
            raise ValueError("SabrePagedKVCache selects pages with topk_pages only")
        layer = self.layers[layer_idx]
        return K.paged_select(q, layer.key_means, self._columns_in_use(), self.seq_lens, q_start,
                              page_size=self.page_size, topk=self.topk_pages,
                              query_block=1 if q_start is None else self.block_rows(q.shape[1]),
                              window_size=self.window_size or 0, num_prefix_tokens=self.num_prefix_tokens)

    def block_rows(self, num_heads: int) -> int:
        """Rows of a query block for so many query heads."""
        most = max(1, 128 // max(1, num_heads // self.pool.shape[3]))
        return min(self.query_block or 128, 1 << (most.bit_length() - 1))

    def _columns_in_use(self) -> torch.Tensor:
        """The columns of the page table that are in use: the prompt kernel plans its
        work by the table's width. Inside a capture, and while pages are lent, all of
        them, since the device may find more rows."""
        if _capturing(self.pool) or self._lent is not None:
            return self.page_table
        n = max(1, -(-max(self.lengths) // self.page_size))
        if self._columns[0] != n:
            self._columns = n, self.page_table[:, :n]
        return self._columns[1]

    def prefill(self, layer_idx: int, q: torch.Tensor, softmax_scale: Optional[float] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of a step's rows, q ``[B, n, Hq, D]``, over a layer."""
        layer = self.layers[layer_idx]
        B, n, Hq, D = q.shape
        if self.topk_pages is not None:
            rows, starts = q.reshape(B * n, Hq, D), self._row_starts(n)
            lists, counts = self.select(layer_idx, rows, starts)
            return K.paged_prefill_listed(rows, layer.k_pages, layer.v_pages, self._columns_in_use(), self.seq_lens,
                                          starts, lists, counts, query_block=self.block_rows(Hq),
                                          softmax_scale=softmax_scale,
                                          out=None if out is None else out.view(B * n, Hq, D)).view(B, n, Hq, D)
        res = K.paged_prefill(q.reshape(B * n, Hq, D), layer.k_pages, layer.v_pages, self._columns_in_use(),
                              self.seq_lens, self._row_starts(n), window_size=self.window_size,
                              num_prefix_tokens=self.num_prefix_tokens, softmax_scale=softmax_scale,
                              out=None if out is None else out.view(B * n, Hq, D))
        return res.view(B, n, Hq, D)

    def gather(self, layer_idx: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """All rows of a layer as ``[B, Hkv, T, D]`` (T the longest length; rows a
        sequence does not have are zero)."""
        T = max(self._lengths_now())
        pages = self.page_table[:, :-(-T // self.page_size)].long()
        have = torch.arange(T, device=pages.device)[None] < self.seq_lens[:, None]
        out = []
        for kv in (0, 1):
            x = self.pool[layer_idx, kv][pages.clamp(min=0)].transpose(1, 2).flatten(2, 3)[:, :, :T]
            out.append(torch.where(have[:, None, :, None], x, torch.zeros_like(x)))
        return out[0], out[1]

    # -- transformers -----------------------------------------------------

    def reset(self) -> None:
        self._truncate({b: 0 for b in range(self.batch_size)})
        for layer in self.layers:  # a step that an error cut off is over
            layer.step = self.step

    def __deepcopy__(self, memo) -> "SabrePagedKVCache":
        """A cache of its own with the same contents, as prompts are reused."""
        if self._lent is not None:
            raise ValueError("SabrePagedKVCache: pages are lent to the device; settle() comes before a copy")
        _, _, n, heads, _, dim = self.pool.shape
        new = SabrePagedKVCache(batch_size=self.batch_size, max_seq_len=self.max_seq_len, num_pages=n,
                                page_size=self.page_size, window_size=self.window_size,
                                num_prefix_tokens=self.num_prefix_tokens, device=self.pool.device,
                                dtype=self.pool.dtype, num_layers=self.pool.shape[0], num_kv_heads=heads,
                                head_dim=dim, topk_pages=self.topk_pages, query_block=self.query_block)
        memo[id(self)] = new
        new.pool.copy_(self.pool)
        if self.key_means is not None:
            new.key_means.copy_(self.key_means)
        new.refs, new.unused = list(self.refs), list(self.unused)
        new.step, new.step_rows = self.step, self.step_rows
        for a, b in zip(new.layers, self.layers):
            a.step = b.step
        new._batch([list(t) for t in self.tables], list(self.lengths), list(self.tops))
        return new

    def crop(self, max_length: int) -> None:
        """Cuts every sequence to max_length rows; -n drops the last n of each."""
        self._truncate({b: max_length if max_length >= 0 else n + max_length for b, n in enumerate(self.lengths)})

    def batch_select_indices(self, indices) -> None:
        """The sequences become copies (shared pages) of the listed ones."""
        self._outside_captures()
        idx = [self._seq(int(i)) for i in (indices.tolist() if isinstance(indices, torch.Tensor) else indices)]
        if not idx:
            raise ValueError("SabrePagedKVCache needs at least one sequence")
        for i in idx:
            for page in self.tables[i]:
                if page >= 0:
                    self.refs[page] += 1
        for t in self.tables:
            for page in t:
                self._release(page)
        self._batch([list(self.tables[i]) for i in idx], [self.lengths[i] for i in idx], [self.tops[i] for i in idx])

    def batch_repeat_interleave(self, repeats: int) -> None:
        self.batch_select_indices([b for b in range(self.batch_size) for _ in range(repeats)])

    def reorder_cache(self, beam_idx: torch.LongTensor) -> None:
        self.batch_select_indices(beam_idx)
