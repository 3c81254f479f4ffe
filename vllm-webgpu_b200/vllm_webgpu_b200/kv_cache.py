"""The paged key-value cache of a model: its pages on the GPU and, on the host, which
sequence holds which of them.

The reference allocates one cache per layer for a single sequence and passes its slot
mapping and block table to the shaders (vllm_webgpu/models/llama.py:181-206,
run_inference.py:305-321); here any number of sequences share the pages, and ``extend``
makes the step's device tensors for all of them in one host-to-device copy.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class CacheStep:
    """What one forward step needs to know of its sequences, on the GPU (see ``PagedKVCache.extend``)."""

    cache: "PagedKVCache"
    positions: torch.Tensor     # int64 [tokens]
    slots: torch.Tensor         # int64 [tokens]
    block_tables: torch.Tensor  # int32 [sequences, pages of the longest]
    lens: torch.Tensor          # int32 [sequences], the new tokens included
    q_starts: torch.Tensor      # int32 [sequences + 1]
    max_q: int

    @property
    def decode(self) -> bool:
        """One new token for every sequence."""
        return self.positions.shape[0] == self.lens.shape[0] and self.max_q == 1


class PagedKVCache:
    """``k[layer]`` and ``v[layer]``: [pages, kv heads, page size, head_dim] of f16 or bf16.

    A page holds ``page_size`` consecutive tokens of one sequence, each kv head's rows side
    by side, so that a head's part of a page is one contiguous run."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str | None = None) -> None:
        if page_size < 8 or page_size % 8:
            raise ValueError(f"page_size must be a positive multiple of 8, not {page_size}")
        if head_dim % 8 or not 8 <= head_dim <= 256:
            raise ValueError(f"head_dim must be a multiple of 8 up to 256, not {head_dim}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"the cache holds float16 or bfloat16, not {dtype}")
        if num_layers < 1 or num_pages < 1 or num_kv_heads < 1:
            raise ValueError("a cache needs at least one layer, page and head")
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.page_size, self.num_pages, self.dtype = page_size, num_pages, dtype
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=self.device)
        self.v = torch.empty(shape, dtype=dtype, device=self.device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict = {}
        self._lens: dict = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq) -> int:
        """Tokens that sequence ``seq`` holds (0 for one that is not there)."""
        return self._lens.get(seq, 0)

    def extend(self, seqs: list, counts: list[int]) -> CacheStep:
        """Give each sequence of ``seqs`` room for its next ``counts`` tokens and return the
        step that writes and reads them. A new name starts a sequence. RuntimeError, with
        nothing changed, when the free pages do not suffice."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 1 for c in counts):
            raise ValueError("extend takes distinct sequences and a count of at least one new token for each")
        need = [-(-(self.length(s) + c) // self.page_size) - len(self._pages.get(s, ())) for s, c in zip(seqs, counts)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {sum(need)} are needed")
        positions, slots = [], []
        for s, c, n in zip(seqs, counts, need):
            pages = self._pages.setdefault(s, [])
            pages.extend(self._free.pop() for _ in range(n))
            first = self._lens.get(s, 0)
            self._lens[s] = first + c
            positions.extend(range(first, first + c))
            slots.extend(pages[p // self.page_size] * self.page_size + p % self.page_size for p in range(first, first + c))
        width = max(len(self._pages[s]) for s in seqs) if seqs else 0
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        # one pinned buffer, one copy: int64 positions and slots, then int32 tables, lens, starts
        t, b = starts[-1], len(seqs)
        small = [p for s in seqs for p in self._pages[s] + [0] * (width - len(self._pages[s]))]
        small += [self._lens[s] for s in seqs] + starts
        if len(small) % 2:
            small.append(0)
        wide = torch.tensor(positions + slots, dtype=torch.int64)
        host = torch.cat([wide, torch.tensor(small, dtype=torch.int32).view(torch.int64)])
        dev = (host.pin_memory() if self.device.type == "cuda" else host).to(self.device, non_blocking=True)
        i32 = dev[2 * t:].view(torch.int32)
        return CacheStep(self, dev[:t], dev[t:2 * t], i32[:b * width].view(b, width), i32[b * width:b * width + b],
                         i32[b * width + b:b * width + 2 * b + 1], max(counts, default=0))

    def release(self, seq) -> None:
        """Forget a sequence and free its pages."""
        self._free.extend(reversed(self._pages.pop(seq, [])))
        self._lens.pop(seq, None)
