"""Paged KV cache of a batch of sequences: the host's side of csrc/paged_kv.hip and csrc/paged_attention.hip.

The static cache (Engine/Llama_KV.py) holds one sequence in fixed slots; this one holds many, of any lengths, in pages of a common
pool.  The host owns the page tables, so that what the kernels read on the device is right by construction: no page belongs to
two sequences, and a batch is refused before anything changes when the pool cannot hold it.  Roll-back after a verification is a
shorter length, as `kv_offset` is for the static cache."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ..ops import get_ops


@dataclass
class PagedBatch:
    """One step's ragged batch on the device: what the paged operators take (ops.rope_kv_write_paged, ops.paged_attention)."""
    page_table: torch.Tensor       # int32 [sequences, width]
    seq_lens: torch.Tensor         # int32 [sequences]: rows stored before the step
    cu_rows: torch.Tensor          # int32 [sequences + 1]: the step's rows of sequence b are [cu_rows[b], cu_rows[b + 1])
    position_ids: torch.Tensor     # int64 [rows]
    n_rows: int
    max_rows: int
    max_len: int


class PagedKVCache:
    def __init__(self, config, n_pages: int, page_size: int = 64, device: str = "cuda:0", dtype=torch.float16, quantised: bool = False):
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"page_size {page_size}: expected 16, 32, 64, 128 or 256")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"dtype {dtype}: the paged kernels take fp16 and bf16 rows (e4m3 pages: quantised=True)")
        if n_pages < 1:
            raise ValueError("n_pages: expected at least one page")
        self.page_size, self.n_pages, self.device, self.dtype, self.quantised = page_size, n_pages, device, dtype, quantised
        self.num_layers, self.num_kv_heads = config.num_hidden_layers, config.num_key_value_heads
        self.head_dim = config.hidden_size // config.num_attention_heads
        shape = (self.num_layers, n_pages, self.num_kv_heads, page_size, self.head_dim)
        kind = torch.float8_e4m3fn if quantised else dtype
        self.k_pages, self.v_pages = (torch.zeros(shape, dtype=torch.uint8 if quantised else dtype, device=device).view(kind) for _ in range(2))
        self.k_scales = self.v_scales = None
        if quantised:
            self.k_scales, self.v_scales = (torch.full(shape[:4], 127, dtype=torch.uint8, device=device) for _ in range(2))
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._length: dict[int, int] = {}
        self._next_id = 0

    # ---- sequences ------------------------------------------------------------------------------
    def add_sequence(self) -> int:
        seq, self._next_id = self._next_id, self._next_id + 1
        self._pages[seq], self._length[seq] = [], 0
        return seq

    def free_sequence(self, seq: int):
        self._free += self._pages.pop(seq)
        del self._length[seq]

    def length(self, seq: int) -> int:
        return self._length[seq]

    def free_pages(self) -> int:
        return len(self._free)

    def set_length(self, seq: int, length: int):
        """Rows [0, length) are stored; pages behind them return to the pool.  `length` may not pass the pages reserved."""
        pages = self._pages[seq]
        if not 0 <= length <= len(pages) * self.page_size:
            raise ValueError(f"sequence {seq}: length {length} is outside its {len(pages)} reserved pages")
        keep = -(-length // self.page_size)
        self._free += pages[keep:]
        del pages[keep:]
        self._length[seq] = length

    # ---- one step -------------------------------------------------------------------------------
    def batch(self, seqs, counts) -> PagedBatch:
        """Reserves pages for counts[i] new rows behind sequence seqs[i] and builds the step's device arrays.  The lengths stay
        until set_length() says what the step left."""
        seqs, counts = list(seqs), [int(c) for c in counts]
        if not seqs or len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or min(counts) < 0:
            raise ValueError("batch: one count >= 0 for each of one or more different sequences")
        totals = [self._length[s] + c for s, c in zip(seqs, counts)]
        need = {s: max(0, -(-t // self.page_size) - len(self._pages[s])) for s, t in zip(seqs, totals)}
        if sum(need.values()) > len(self._free):
            raise RuntimeError(f"paged KV cache: {sum(need.values())} more pages wanted, {len(self._free)} free")
        for s, n in need.items():
            self._pages[s] += [self._free.pop() for _ in range(n)]
        width = max(1, max(len(self._pages[s]) for s in seqs))
        table = [self._pages[s] + [0] * (width - len(self._pages[s])) for s in seqs]
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        position = [self._length[s] + i for s, c in zip(seqs, counts) for i in range(c)]
        put = lambda v, dt: torch.tensor(v, dtype=dt, device=self.device)
        return PagedBatch(put(table, torch.int32), put([self._length[s] for s in seqs], torch.int32), put(cu, torch.int32),
                          put(position, torch.int64), cu[-1], max(counts), max(1, max(totals)))

    def layer(self, layer_idx: int) -> dict:
        """One layer's pages, as keyword arguments of the paged operators."""
        s = self.k_scales is not None
        return dict(k_pages=self.k_pages[layer_idx], v_pages=self.v_pages[layer_idx],
                    k_scales=self.k_scales[layer_idx] if s else None, v_scales=self.v_scales[layer_idx] if s else None)

    def export(self, seq: int, kv_cache):
        """Copies a sequence's rows into the static cache `kv_cache` (Engine/Llama_KV.py) and sets its length: the single-sequence
        engines continue from there."""
        n = self._length[seq]
        if n > kv_cache.max_length:
            raise ValueError(f"sequence {seq} holds {n} rows, the static cache {kv_cache.max_length}")
        if self.dtype != kv_cache.dtype or kv_cache.k_cache.shape[0] != self.num_layers:
            raise ValueError("export: the caches hold different element types or numbers of layers")
        if n:
            pages = torch.tensor([self._pages[seq]], dtype=torch.int32, device=self.device)
            start, count = (torch.tensor([v], dtype=torch.int32, device=self.device) for v in (0, n))
            for i in range(self.num_layers):
                get_ops().kv_read_paged(k_out=kv_cache.k_cache[i], v_out=kv_cache.v_cache[i], page_table=pages, starts=start, counts=count,
                                        max_count=n, **self.layer(i))
        kv_cache.set_kv_len(n)
        kv_cache.dirty_end = max(kv_cache.dirty_end, n)
