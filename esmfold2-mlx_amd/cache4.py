"""Keys and values in 4 bits, in pages of 64 keys, beside ``kernels.packed_attention`` on caches in 16 bits.

A value stands as step (code - zero) with a step (bf16) and a whole zero per key, head and 64 values: 4.5 bits in all, half a
step of a fifteenth of the 64 values' range off at most. Heads are filled up to 64 or 128 values: with 64 or 128 a cache takes
0.28 of its 16 bits' memory, with 96 0.38, 80 0.45, 72 0.50, 32 0.56, and with 16 or fewer more than 16 bits would. Where a model
bears the error, a step of generation, which is bound by reading the cache, takes about as much less time on long contexts.

The sequences of a batch are given to every call as int32 tensors on the GPU, so that calls may be captured into a HIP graph and
replayed with other contents: ``cu`` [n + 1], the first of each sequence's rows in the call and the end of the last; ``lens``
[n], its keys with those rows; ``table`` [n, width], its pages, key j in table[i, j // 64]. Which pages are whose is the
caller's to keep; one page may serve several sequences that only read it.
"""

from __future__ import annotations

import torch

from . import capi, kernels

PAGE = 64


class Cache4:
    page = PAGE  # keys in a page

    def __init__(self, pages: int, heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, device=None):
        """Room for ``pages`` pages of 64 keys and values of ``heads`` heads of ``head_dim`` (a multiple of 8 up to 128);
        ``dtype``: fp16 or bf16, of the rows that go in and the queries."""
        if pages < 0 or heads <= 0 or head_dim <= 0 or head_dim % 8 or head_dim > 128 or dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"Cache4: {pages} pages of {heads} heads of {head_dim} (a multiple of 8 up to 128) in {dtype}")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.data = torch.zeros(int(capi.lib().cache4_bytes(pages, heads, head_dim)), dtype=torch.uint8, device=dev)
        self.pages, self.heads, self.head_dim, self.dtype = pages, heads, head_dim, dtype

    def _check(self, t: torch.Tensor, name: str, heads=None):
        if t.dim() != 3 or t.dtype is not self.dtype or t.shape[2] != self.head_dim or (heads is not None and t.shape[1] != heads):
            raise ValueError(f"Cache4: {name} {t.dtype} {tuple(t.shape)}, holds heads of {self.head_dim} in {self.dtype}")

    def append(self, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor, table: torch.Tensor) -> None:
        """Rows k, v [T, heads, head_dim] become the last of their sequences' keys (``lens`` counts them already)."""
        self._check(k, "k", self.heads)
        self._check(v, "v", self.heads)
        kernels.cache4_append(self.data, k, v, cu, lens, table)

    def read(self, cu: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, rows: int | None = None):
        """(k, v) [T, heads, head_dim] as the cache holds them, of the rows that ``append`` with these arguments writes.
        ``rows``: T, where the caller knows it (else it is read from the GPU)."""
        T = int(cu[-1]) if rows is None else int(rows)
        return kernels.cache4_read(self.data, T, self.heads, self.head_dim, self.dtype, cu, lens, table)

    def attend(self, q: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, causal: bool = True,
               scale: float | None = None, out=None) -> torch.Tensor:
        """softmax(q k^T scale) v of q [T, H, head_dim] over each sequence's keys; ``causal``: its last row sees the last. Sums
        are fp32: values below 2^96."""
        self._check(q, "q")
        return kernels.cache4_attention(self.data, q, self.heads, cu, lens, table, causal, scale, out)
