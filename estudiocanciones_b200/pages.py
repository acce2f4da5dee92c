"""A paged KV cache that takes of one prompt share.

The static cache of the engine (``Block.kc/vc [B, Hk, L, hd]``, ``app/engine.py:119-121``) holds
the prompt once per row.  A :class:`PagePool` holds it once per prompt: its sequences list the
pages they hold, :meth:`PagePool.fork` lets a take share its prompt's full pages (only a partial
last page is copied), and :func:`estudiocanciones_b200.kernels.prefix_attn` reads the shared
pages once for all takes.  Typical use, with every call on the device (capturable):

    pool = PagePool(layers=28, n_pages=512, kv_heads=8, hd=128, max_seqs=10, max_len=2048)
    pool.grow([0], P)                       # sequence 0: the prompt, written per layer by
    kernels.rope_pages(..., *pool.layer(i), pool.table, S=P, ...)
    pool.fork([0, 0, 0, 0], [2, 3, 4, 5])   # four takes
    pool.grow(takes, 1)                     # every frame: a slot for the new position
    pool.free(takes); pool.compact()        # the takes end; live pages move to the front
"""
from __future__ import annotations

import torch

from . import kernels
from ._lib import HMError


class PagePool:
    """K and V pages of every layer and the bookkeeping of the sequences that hold them.

    ``k``, ``v`` ``[layers, n_pages, kv_heads, page, hd]``; ``table [max_seqs, max_pages]`` int32
    (-1 = none); ``lens [max_seqs]`` int64; ``refs [n_pages]`` int32 (0 = free).

    The page calls and ``rope_pages`` take any ``page`` up to 1024 and any ``hd`` that is a multiple of 8;
    ``prefix_attn`` reads pages of 16, 32 or a multiple of 64 positions with ``hd`` 64, 128 or 256."""

    def __init__(self, layers: int, n_pages: int, kv_heads: int, hd: int, max_seqs: int, max_len: int, page: int = 64,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        if min(layers, n_pages, kv_heads, hd, max_seqs, max_len, page) < 1:
            raise HMError("PagePool: every size is at least 1")
        if dtype not in (torch.float16, torch.bfloat16):
            raise HMError("PagePool: fp16 or bf16")
        if page > 1024 or hd % 8:
            raise HMError("PagePool: pages of at most 1024 positions, hd a multiple of 8")
        shape = (layers, n_pages, kv_heads, page, hd)
        self.page = page
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.table = torch.full((max_seqs, -(-max_len // page)), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(max_seqs, dtype=torch.int64, device=device)
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device=device)

    def layer(self, i: int):
        """K and V pages of layer ``i``, ``[n_pages, kv_heads, page, hd]``."""
        return self.k[i], self.v[i]

    def grow(self, seqs, n: int = 1) -> None:
        kernels.pages_grow(self.table, self.lens, self.refs, self.page, seqs, n)

    def fork(self, src, dst) -> None:
        kernels.pages_fork(self.k, self.v, self.table, self.lens, self.refs, src, dst)

    def free(self, seqs) -> None:
        kernels.pages_free(self.table, self.lens, self.refs, seqs)

    def copy(self, src, dst) -> None:
        kernels.pages_copy(self.k, self.v, src, dst)

    def compact(self) -> torch.Tensor:
        return kernels.pages_compact(self.k, self.v, self.table, self.refs)

    def free_pages(self) -> int:
        """Free pages now (reads the device)."""
        return int((self.refs == 0).sum())
