"""KV cache of the generation path.

The reference keeps `past_key_values` as per-layer tuples of `[B, H, L, hd]` tensors that grow by `torch.cat` on every
step (modeling_cogvlm.py:253-262), padding positions included. Here one allocation per model holds every layer:
`k`, `v` `[n_layers, B, max_len, H*hd]` bf16 — token-major rows in the same format as the packed qkv rows of the training
path — plus one int32 length per sample. Only VALID tokens are stored (the packed layout never materialises padding), so a
right-padded prompt batch decodes correctly and the decode attention needs no mask. A step appends one row per sample and
layer with `vm_scatter_rows`; nothing is reallocated, and the only host-side state is an upper bound of the lengths (the
launch geometry), so a decode step never synchronises with the device."""
from __future__ import annotations

import torch

from ... import kernels as K


class KVCache:
    def __init__(self, n_layers: int, batch: int, max_len: int, width: int, device, dtype=torch.bfloat16):
        self.k = torch.empty(n_layers, batch, max_len, width, dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)       # tokens cached per sample (device)
        self.max_len = max_len
        self.len_bound = 0            # host upper bound of lens (max over samples)
        # launch bound of the decode attention: None = len_bound + 1 (eager); a captured decode step (hipGraph) is replayed
        # with one fixed geometry, so it is sized for the whole cache and the chunks past a sample's length exit at once
        self.launch_bound: int | None = None
        self._slots: torch.Tensor | None = None
        self._pending: torch.Tensor | None = None
        # constants of a decode step (one row per sample), created once: nothing is uploaded inside a step
        self.rows = torch.arange(batch, device=device, dtype=torch.int32)
        self.zeros = torch.zeros(batch, device=device, dtype=torch.int32)
        self.ones = torch.ones(batch, device=device, dtype=torch.int32)
        self.cu_rows = torch.arange(batch + 1, device=device, dtype=torch.int32)
        self.decode_counts = torch.tensor([0, batch, 1, 0], dtype=torch.int32, device=device)     # no vision rows

    @property
    def batch(self) -> int:
        return self.k.shape[1]

    def __len__(self) -> int:         # `if past_key_values:` of the reference's prepare_inputs_for_generation
        return self.k.shape[0] if self.len_bound > 0 else 0

    def begin(self, seq_of_row: torch.Tensor, offset_in_seq: torch.Tensor, rows_per_seq: torch.Tensor, max_new: int):
        """declare the rows of one forward call: row r belongs to sample seq_of_row[r] and is its offset_in_seq[r]-th new
        token (both int32, device); rows_per_seq int32[B]; max_new: host upper bound of rows_per_seq"""
        if self.len_bound + max_new > self.max_len:
            raise ValueError(f'KV cache overflow: {self.len_bound} + {max_new} > {self.max_len}')
        seq = seq_of_row.long()
        self._slots = (seq * self.max_len + self.lens[seq].long() + offset_in_seq.long()).to(torch.int32).contiguous()
        self._pending = rows_per_seq.to(torch.int32)
        self._pending_bound = max_new

    def append(self, layer: int, qkv: torch.Tensor, width: int, nrows: torch.Tensor | None = None):
        """store the (rotated) K and V thirds of the packed qkv rows of this call into layer `layer`"""
        flat_k = self.k[layer].view(-1, width)
        flat_v = self.v[layer].view(-1, width)
        K.scatter_rows(qkv[:, width:2 * width], self._slots, flat_k, nrows=nrows)
        K.scatter_rows(qkv[:, 2 * width:], self._slots, flat_v, nrows=nrows)

    def lens_after(self) -> torch.Tensor:
        return self.lens + self._pending

    def attn_bound(self) -> int:
        return self.launch_bound if self.launch_bound is not None else self.len_bound + 1

    def commit(self):
        """all layers have appended: advance the lengths"""
        self.lens.add_(self._pending)
        self.len_bound += self._pending_bound
        self._slots = self._pending = None


class PagedKVCache:
    """KV cache in pages, for conversations that go on: several samples of different lengths share one pool of pages per layer, a chunk of
    any number of new tokens may follow what is cached (`CogVLMModel.forward` with a non-empty cache), and the cache can be cut to a budget
    by the attention weight its tokens have received.

    `k`, `v` `[n_layers, n_pages, n_heads, page_size, head_dim]` bf16: a page holds the same tokens in every layer, so there is one
    `block_table` int32 `[batch, pages per sample]` (token j of a sample lies in page `block_table[b, j // page_size]`), kept on the host
    (which owns the list of free pages) and uploaded when it changes. As in `KVCache` only valid tokens are stored and lengths live on the
    device. The host knows an upper bound of each sample's length and hands out pages by it; a step that needs no new page uploads nothing
    and does not synchronise — `reserve` ahead of a captured step. Where the bounds ask for more than the pool or `max_len` holds, the lengths
    are read back (one synchronisation) before the call is refused. `track_weights` keeps `weights` fp32 `[n_layers, batch, n_heads, tokens]`
    (`max_len` of them for every sample), which `evict` needs."""

    def __init__(self, n_layers: int, batch: int, max_len: int, n_heads: int, head_dim: int, device, *, page_size: int = 64,
                 n_pages: int | None = None, track_weights: bool = False, dtype=torch.bfloat16):
        if dtype != torch.bfloat16:
            raise TypeError(f'the paged cache is bf16, not {dtype}')
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f'page size {page_size}: a power of two in 16 .. 1024')
        self.page_size = page_size
        cols = max(1, -(-max_len // page_size))
        self.max_len = cols * page_size
        n_pages = batch * cols if n_pages is None else n_pages
        self.k = torch.empty(n_layers, n_pages, n_heads, page_size, head_dim, dtype=dtype, device=device)
        self.v = torch.empty_like(self.k)
        self.n_heads, self.head_dim = n_heads, head_dim
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.block_table = torch.full((batch, cols), -1, dtype=torch.int32, device=device)
        self.weights = torch.zeros(n_layers, batch, n_heads, self.max_len, dtype=torch.float32, device=device) if track_weights else None
        self._bounds = [0] * batch    # host upper bounds of lens
        self.pos_bound = 0            # host upper bound of the rotary positions: all of them so far are below it
        self._pos_reserved = 0        # ... and those that reserve_positions() has announced
        self.launch_bound: int | None = None            # as in KVCache
        self.launch_new: list[int] | None = None        # of a captured step: new tokens per sample that prepare_step() has found pages for
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: list[list[int]] = [[] for _ in range(batch)]
        self._reserved = [0] * batch  # tokens whose pages stay until tighten()
        self._pending: torch.Tensor | None = None
        self._counting = False        # this call has added to `weights`
        self._miscounted = False      # a call that was dropped has
        self.rows = torch.arange(batch, device=device, dtype=torch.int32)
        self.zeros = torch.zeros(batch, device=device, dtype=torch.int32)
        self.ones = torch.ones(batch, device=device, dtype=torch.int32)
        self.cu_rows = torch.arange(batch + 1, device=device, dtype=torch.int32)
        self.decode_counts = torch.tensor([0, batch, 1, 0], dtype=torch.int32, device=device)     # no vision rows

    @property
    def batch(self) -> int:
        return len(self._pages)

    def __len__(self) -> int:
        return self.k.shape[0] if self.len_bound > 0 else 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def len_bound(self) -> int:
        """host upper bound of the longest sample's length"""
        return max(self._bounds, default=0)

    @len_bound.setter
    def len_bound(self, n: int):
        self._bounds = [n] * self.batch

    @property
    def len_bounds(self) -> list[int]:
        """the same for every sample"""
        return list(self._bounds)

    @len_bounds.setter
    def len_bounds(self, n: list[int]):
        self._bounds = list(n)

    def _up(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    def _take(self, tokens: int) -> list[int]:
        return [self._free.pop() for _ in range(self._up(tokens))]

    def _capturing(self) -> bool:
        return self.block_table.is_cuda and torch.cuda.is_current_stream_capturing()

    def _not_captured(self):
        if self._capturing():
            raise RuntimeError('the block table changes inside a captured step: reserve() the pages first')

    def _upload(self, pages: list[list[int]], table: torch.Tensor):
        host = torch.full(tuple(table.shape), -1, dtype=torch.int32)
        for b, p in enumerate(pages):
            host[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        table.copy_(host)

    def _grant(self, want: list[int]) -> bool:
        """pages for want[b] tokens of sample b; False, and nothing changes, if there is no room for all"""
        short = [max(0, self._up(n) - len(p)) for n, p in zip(want, self._pages)]
        if max(want, default=0) > self.max_len or sum(short) > len(self._free):
            return False
        if any(short):
            self._not_captured()
            for p, n in zip(self._pages, short):
                p.extend(self._take(n * self.page_size))
            self._upload(self._pages, self.block_table)
        return True

    def _overflow(self, want: list[int]) -> ValueError:
        if max(want) > self.max_len:
            return ValueError(f'KV cache overflow: {max(want)} > {self.max_len}')
        short = sum(max(0, self._up(n) - len(p)) for n, p in zip(want, self._pages))
        return ValueError(f'KV cache overflow: {short} pages wanted, {len(self._free)} free')

    def reserve(self, tokens: int):
        """pages for `tokens` tokens of every sample (those it has counted), and rotary tables for positions that go on as far: later steps up
        to that length upload nothing. The pages stay, over further turns and evictions, until tighten(); tables that have to grow for it do
        so in the next step, which then must not be a captured one. The replays of a step of one's own are not counted by the host: settle()
        before the next call or eviction."""
        want = [tokens] * self.batch
        if not self._grant(want):
            raise self._overflow(want)
        self.reserve_positions(self.pos_bound + max(0, tokens - min(self._bounds, default=0)))
        self._reserved = [max(n, tokens) for n in self._reserved]

    def reserve_positions(self, n: int):
        """rotary positions below n are to come"""
        self._pos_reserved = max(self._pos_reserved, n)

    def rope_len(self, least: int) -> int:
        """rows of rotary tables that hold the positions so far and the announced ones: `least`, doubled as often as it takes"""
        while least < max(self.pos_bound, self._pos_reserved):
            least *= 2
        return least

    def _room(self, most: list[int], rows_per_seq) -> list[int]:
        """pages for at most most[b] further tokens of sample b, or, where the bounds leave no room for so many, for the rows there are (read
        from the device by rows_per_seq()) behind the lengths there are -> host upper bounds of the new tokens"""
        want = [n + m for n, m in zip(self._bounds, most)]
        if self._grant(want):
            return most
        if not self._capturing():
            self.settle()
            most = rows_per_seq()
            want = [n + m for n, m in zip(self._bounds, most)]
            if self._grant(want):
                return most
        raise self._overflow(want)

    def begin(self, seq_of_row: torch.Tensor, offset_in_seq: torch.Tensor, rows_per_seq: torch.Tensor, max_new: int):
        """as KVCache.begin: row r of the call is the offset_in_seq[r]-th new token of sample seq_of_row[r] (-1: of none, nothing is stored);
        a sample without new rows is left out of the call altogether (its queries see nothing and count nowhere)"""
        self.abort()
        self.in_capture = self._capturing()
        self._pending_bounds = self._room([max_new] * self.batch if self.launch_new is None else self.launch_new, rows_per_seq.tolist)
        self._row_seq = seq_of_row.to(torch.int32).contiguous()
        self._row_index = (self.lens[self._row_seq.long()] + offset_in_seq.to(torch.int32)).contiguous()
        self._pending = rows_per_seq.to(torch.int32)
        self._lens_after = torch.where(self._pending > 0, self.lens + self._pending, self.zeros)

    def prepare_step(self, done: torch.Tensor):
        """ahead of the capture or a replay of a decode step: pages for its tokens (done bool [batch]: the samples that have none)"""
        self.launch_new = self._room([1] * self.batch, lambda: [int(not d) for d in done.tolist()])

    def count_step(self):
        """a captured step has been replayed: its tokens"""
        self.pos_bound += 1
        self._bounds = [n + m for n, m in zip(self._bounds, self.launch_new)]

    def append(self, layer: int, qkv: torch.Tensor, row_pos: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               nrows: torch.Tensor | None = None) -> torch.Tensor:
        """the rows of this call into layer `layer`, rotary positions included -> rotated q"""
        return K.kv_append_paged(qkv, self._row_seq, self._row_index, self.block_table, self.k[layer], self.v[layer], row_pos, cos, sin,
                                 self.n_heads, nrows=nrows)

    def attend(self, layer: int, q: torch.Tensor, cu_q: torch.Tensor, row_of_pos: torch.Tensor | None, max_q: int, scale: float) -> torch.Tensor:
        """attention of the appended rows over everything cached (their own tokens included, causally)"""
        w = self.weights[layer] if self.weights is not None else None
        self._counting = w is not None and not self.in_capture
        return K.attn_paged(q, self.k[layer], self.v[layer], self.block_table, cu_q, self._lens_after, scale, max_q, self.attn_bound(),
                            row_of_pos=row_of_pos, weights=w)[0]

    def lens_after(self) -> torch.Tensor:
        """cached tokens a sample of this call attends to, the new ones included"""
        return self._lens_after

    def attn_bound(self) -> int:
        return self.launch_bound if self.launch_bound is not None else max((n + m for n, m in zip(self._bounds, self._pending_bounds)), default=0)

    def commit(self):
        self.lens.add_(self._pending)
        self._bounds = [n + m for n, m in zip(self._bounds, self._pending_bounds)]
        self._pending = None
        self._counting = False

    def abort(self):
        """drop the call that begin() has declared, if there is one: the lengths stay what they are, what it has stored lies behind them. The
        weights that its layers have added up are not taken back: evict() refuses from then on."""
        self._miscounted |= self._counting
        self._pending = None
        self._counting = False

    def settle(self) -> list[int]:
        """read the lengths back (synchronises), give pages behind them back that are not reserved -> lengths"""
        assert self._pending is None, 'settle() between begin() and commit()'
        lens = self.lens.tolist()
        self._bounds = list(lens)
        changed = False
        for p, n, r in zip(self._pages, lens, self._reserved):
            keep = self._up(max(n, r))
            changed |= len(p) > keep
            while len(p) > keep:
                self._free.append(p.pop())
        if changed:
            self._upload(self._pages, self.block_table)
        return lens

    def tighten(self) -> list[int]:
        """settle(), and reserved pages go back too: a step that was captured on them must not be replayed any more -> lengths"""
        assert self._pending is None, 'tighten() between begin() and commit()'
        self._reserved = [0] * self.batch
        return self.settle()

    def pages_to_evict(self, budget: int) -> int:
        """free pages that evict() to `budget` tokens needs while it runs: those of the samples that are over it"""
        return sum(self._up(budget) for n in self._bounds if n > budget)

    def evict(self, budget: int, recent: int):
        """cut every sample to the `budget` tokens (per layer and head) that are among its `recent` newest or have received the most
        attention; they keep their order and their rotary positions. Needs ceil(budget / page_size) free pages for every sample over the
        budget while it runs; the others stay where they are."""
        assert self._pending is None, 'evict() between begin() and commit()'
        if self.weights is None:
            raise ValueError('evict() needs the received attention weights: track_weights=True')
        if self._miscounted:
            raise RuntimeError('the received weights are those of a call that failed half way: this cache cannot be evicted from, start another one')
        if budget <= 0 or not 0 <= recent <= budget:
            raise ValueError(f'budget {budget}, recent {recent}: 0 <= recent <= budget, budget > 0')
        need = self.pages_to_evict(budget)
        if need == 0:
            return                                       # nobody is over the budget
        if need > len(self._free):
            raise ValueError(f'KV cache overflow: eviction to {budget} tokens wants {need} pages, {len(self._free)} free')
        self._not_captured()
        # (who is not over the budget keeps every token in its place: source and destination are the same rows)
        pages = [self._take(budget) if n > budget else p for n, p in zip(self._bounds, self._pages)]
        layer = 0
        try:
            table = torch.full_like(self.block_table, -1)
            self._upload(pages, table)
            for layer in range(self.k.shape[0]):
                w, lens, _ = K.kv_evict_paged(self.k[layer], self.v[layer], self.weights[layer], self.block_table, self.lens, table, budget, recent)
                self.weights[layer].copy_(w)
        except BaseException:                            # nothing has moved out of the old pages; the weights of the first layers have
            self._free.extend(i for n, p in zip(self._bounds, pages) if n > budget for i in p)
            self._miscounted |= layer > 0
            raise
        self.lens.copy_(lens)
        self.block_table.copy_(table)                    # (in place: a captured step reads these buffers)
        for n, p in zip(self._bounds, self._pages):
            if n > budget:
                self._free.extend(p)
        self._pages = pages
        self._bounds = [min(n, budget) for n in self._bounds]
        self._grant([max(n, r) for n, r in zip(self._bounds, self._reserved)])      # (out of the pages that have just come back)
