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
    (which owns the list of free pages) and uploaded when it changes. As in `KVCache` only valid tokens are stored, lengths live on the
    device, the host knows upper bounds (`len_bound`), and a step that needs no new page uploads nothing and does not synchronise — `reserve`
    ahead of a captured step. `track_weights` keeps `weights` fp32 `[n_layers, batch, n_heads, tokens]`, which `evict` needs."""

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
        self.len_bound = 0            # host upper bound of lens
        self.launch_bound: int | None = None            # as in KVCache
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: list[list[int]] = [[] for _ in range(batch)]
        self._pending: torch.Tensor | None = None
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

    def _take(self, tokens: int) -> list[int]:
        n = -(-tokens // self.page_size)
        return [self._free.pop() for _ in range(n)]

    def _not_captured(self):
        if self.block_table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError('the block table changes inside a captured step: reserve() the pages first')

    def _upload(self, pages: list[list[int]], table: torch.Tensor):
        host = torch.full(tuple(table.shape), -1, dtype=torch.int32)
        for b, p in enumerate(pages):
            host[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        table.copy_(host)

    def reserve(self, tokens: int):
        """pages for `tokens` tokens of every sample (those it has counted): later steps up to that length upload nothing"""
        if tokens > self.max_len:
            raise ValueError(f'KV cache overflow: {tokens} > {self.max_len}')
        want = -(-tokens // self.page_size)
        short = sum(max(0, want - len(p)) for p in self._pages)
        if short > len(self._free):
            raise ValueError(f'KV cache overflow: {short} pages wanted, {len(self._free)} free')
        if short:
            self._not_captured()
            for p in self._pages:
                p.extend(self._take((want - len(p)) * self.page_size) if want > len(p) else [])
            self._upload(self._pages, self.block_table)

    def begin(self, seq_of_row: torch.Tensor, offset_in_seq: torch.Tensor, rows_per_seq: torch.Tensor, max_new: int):
        """as KVCache.begin: row r of the call is the offset_in_seq[r]-th new token of sample seq_of_row[r] (-1: of none, nothing is stored);
        a sample without new rows is left out of the call altogether (its queries see nothing and count nowhere)"""
        self.reserve(self.len_bound + max_new)
        self._row_seq = seq_of_row.to(torch.int32).contiguous()
        self._row_index = (self.lens[self._row_seq.long()] + offset_in_seq.to(torch.int32)).contiguous()
        self._pending = rows_per_seq.to(torch.int32)
        self._pending_bound = max_new
        self._lens_after = torch.where(self._pending > 0, self.lens + self._pending, self.zeros)

    def append(self, layer: int, qkv: torch.Tensor, row_pos: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
               nrows: torch.Tensor | None = None) -> torch.Tensor:
        """the rows of this call into layer `layer`, rotary positions included -> rotated q"""
        return K.kv_append_paged(qkv, self._row_seq, self._row_index, self.block_table, self.k[layer], self.v[layer], row_pos, cos, sin,
                                 self.n_heads, nrows=nrows)

    def attend(self, layer: int, q: torch.Tensor, cu_q: torch.Tensor, row_of_pos: torch.Tensor | None, max_q: int, scale: float) -> torch.Tensor:
        """attention of the appended rows over everything cached (their own tokens included, causally)"""
        w = self.weights[layer] if self.weights is not None else None
        return K.attn_paged(q, self.k[layer], self.v[layer], self.block_table, cu_q, self._lens_after, scale, max_q, self.attn_bound(),
                            row_of_pos=row_of_pos, weights=w)[0]

    def lens_after(self) -> torch.Tensor:
        """cached tokens a sample of this call attends to, the new ones included"""
        return self._lens_after

    def attn_bound(self) -> int:
        return self.launch_bound if self.launch_bound is not None else self.len_bound + self._pending_bound

    def commit(self):
        self.lens.add_(self._pending)
        self.len_bound += self._pending_bound
        self._pending = None

    def tighten(self) -> list[int]:
        """read the lengths back (the one call that synchronises), give pages behind them back -> lengths"""
        assert self._pending is None, 'tighten() between begin() and commit()'
        lens = self.lens.tolist()
        self.len_bound = max(lens, default=0)
        changed = False
        for p, n in zip(self._pages, lens):
            keep = -(-n // self.page_size)
            changed |= len(p) > keep
            while len(p) > keep:
                self._free.append(p.pop())
        if changed:
            self._upload(self._pages, self.block_table)
        return lens

    def evict(self, budget: int, recent: int):
        """cut every sample to the `budget` tokens (per layer and head) that are among its `recent` newest or have received the most
        attention; they keep their order and their rotary positions. Needs ceil(budget / page_size) free pages per sample while it runs."""
        assert self._pending is None, 'evict() between begin() and commit()'
        if self.weights is None:
            raise ValueError('evict() needs the received attention weights: track_weights=True')
        if budget <= 0 or not 0 <= recent <= budget:
            raise ValueError(f'budget {budget}, recent {recent}: 0 <= recent <= budget, budget > 0')
        left = min(budget, self.len_bound)
        if left == self.len_bound:
            return                                       # nobody is over the budget
        need = -(-left // self.page_size) * self.batch
        if need > len(self._free):
            raise ValueError(f'KV cache overflow: eviction to {budget} tokens wants {need} pages, {len(self._free)} free')
        self._not_captured()
        pages = [self._take(left) for _ in range(self.batch)]
        table = torch.full_like(self.block_table, -1)
        self._upload(pages, table)
        for layer in range(self.k.shape[0]):
            w, lens, _ = K.kv_evict_paged(self.k[layer], self.v[layer], self.weights[layer], self.block_table, self.lens, table, budget, recent)
            self.weights[layer].copy_(w)
        self.lens.copy_(lens)
        self.block_table.copy_(table)                    # (in place: a captured step reads these buffers)
        for p in self._pages:
            self._free.extend(p)
        self._pages = pages
        self.len_bound = left
