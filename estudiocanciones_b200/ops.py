"""The decode entry points as ``torch.library`` custom operators (namespace ``heartmula_b200``).

Each operator calls the same C-ABI launch as the function of the same name in
:mod:`estudiocanciones_b200.kernels` (the drop-in for ``app/kernels.py``), on the current
CUDA stream, so ``torch.cuda.graph`` captures it.  Registering them lets torch tooling
see the kernels as opaque operators with known output shapes (a fake implementation
per operator) and known in-place arguments (``mutates_args``), instead of untraceable
ctypes calls:

* ``int8_mm(x, w, s, res)`` -> ``[..., N]``       (``app/kernels.py:40-54``)
* ``rms(x, w, eps)`` -> ``[R, D]``                  (``app/kernels.py:70-74``)
* ``rope_cache(qkv, rope, pos, q_out, kc, vc, S, Hq, Hk, L)``, writes q_out / kc / vc
                                                    (``app/kernels.py:79-107``)
* ``attn(q, kc, vc, pos, o, S, Hq, Hk, L, scale, nsplit)``, writes o
                                                    (``app/kernels.py:112-167``)
* ``silu_mul(a)`` -> ``[R, F]``                     (``app/kernels.py:172-180``)
* ``gemm_i8w(a, w, s, res, silu)`` -> ``[M, N or N/2]`` (the ``M > 16`` branch of ``int8_mm``)
* ``prefill_attn(q, kc, vc, P)`` -> like ``q``      (``Block.__call__`` causal attention)
* ``int8_mm_a8(x, w, s, res, silu)`` -> ``[..., N or N/2]``, ``quant_tokens(x)`` -> ``(q, sx)`` and
  ``gemm_i8a8(q, sx, w, s, res, silu, dtype)``     (``int8_mm`` with the activations in 8 bits)
* ``prefix_attn(q, k, v, table, pos, gstart, owner, plen, S, scale, seqs)`` -> like ``q``, and
  ``rope_pages(...)``, writes q_out / k / v           (``attn`` and ``rope_cache`` over pages)
* ``pages_grow`` / ``pages_free`` / ``pages_fork`` / ``pages_copy`` / ``pages_compact``, write the cache's
  state in place

Importing this module registers them; nothing is loaded onto a GPU until an operator runs.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import kernels

NS = "heartmula_b200"


@torch.library.custom_op(f"{NS}::int8_mm", mutates_args=())
def int8_mm(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, res: Optional[torch.Tensor] = None) -> torch.Tensor:
    return kernels.int8_mm(x, w, s, res)


@int8_mm.register_fake
def _(x, w, s, res=None):
    return x.new_empty(*x.shape[:-1], w.shape[0])


@torch.library.custom_op(f"{NS}::rms", mutates_args=())
def rms(x: torch.Tensor, w: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    return kernels.rms(x, w, eps)


@rms.register_fake
def _(x, w, eps=1e-5):
    return torch.empty_like(x)


@torch.library.custom_op(f"{NS}::rope_cache", mutates_args=("q_out", "kc", "vc"))
def rope_cache(qkv: torch.Tensor, rope: torch.Tensor, pos: torch.Tensor, q_out: torch.Tensor, kc: torch.Tensor,
               vc: torch.Tensor, S: int, Hq: int, Hk: int, L: int) -> None:
    kernels.rope_cache(qkv, rope, pos, q_out, kc, vc, S, Hq, Hk, L)


@rope_cache.register_fake
def _(qkv, rope, pos, q_out, kc, vc, S, Hq, Hk, L):
    return None


@torch.library.custom_op(f"{NS}::attn", mutates_args=("o",))
def attn(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, pos: torch.Tensor, o: torch.Tensor, S: int, Hq: int,
         Hk: int, L: int, scale: float, nsplit: int = 16) -> None:
    kernels.attn(q, kc, vc, pos, o, S, Hq, Hk, L, scale, nsplit=nsplit)


@attn.register_fake
def _(q, kc, vc, pos, o, S, Hq, Hk, L, scale, nsplit=16):
    return None


@torch.library.custom_op(f"{NS}::silu_mul", mutates_args=())
def silu_mul(a: torch.Tensor) -> torch.Tensor:
    return kernels.silu_mul(a)


@silu_mul.register_fake
def _(a):
    return a.new_empty(a.shape[0], a.shape[1] // 2)


@torch.library.custom_op(f"{NS}::gemm_i8w", mutates_args=())
def gemm_i8w(a: torch.Tensor, w: torch.Tensor, s: torch.Tensor, res: Optional[torch.Tensor] = None,
             silu: bool = False) -> torch.Tensor:
    return kernels.gemm_i8w(a, w, s, res=res, silu=silu)


@gemm_i8w.register_fake
def _(a, w, s, res=None, silu=False):
    return a.new_empty(a.shape[0], w.shape[0] // 2 if silu else w.shape[0])


@torch.library.custom_op(f"{NS}::prefill_attn", mutates_args=())
def prefill_attn(q: torch.Tensor, kc: torch.Tensor, vc: torch.Tensor, P: int) -> torch.Tensor:
    return kernels.prefill_attn(q, kc, vc, P)


@prefill_attn.register_fake
def _(q, kc, vc, P):
    return torch.empty_like(q)


@torch.library.custom_op(f"{NS}::quant_tokens", mutates_args=())
def quant_tokens(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    return kernels.quant_tokens(x)


@quant_tokens.register_fake
def _(x):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[0], dtype=torch.float32)


@torch.library.custom_op(f"{NS}::gemm_i8a8", mutates_args=())
def gemm_i8a8(q: torch.Tensor, sx: torch.Tensor, w: torch.Tensor, s: torch.Tensor, res: Optional[torch.Tensor] = None,
              silu: bool = False, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    return kernels.gemm_i8a8(q, sx, w, s, res=res, silu=silu, dtype=dtype)


@gemm_i8a8.register_fake
def _(q, sx, w, s, res=None, silu=False, dtype=torch.float16):
    return q.new_empty(q.shape[0], w.shape[0] // 2 if silu else w.shape[0], dtype=dtype)


@torch.library.custom_op(f"{NS}::int8_mm_a8", mutates_args=())
def int8_mm_a8(x: torch.Tensor, w: torch.Tensor, s: torch.Tensor, res: Optional[torch.Tensor] = None,
               silu: bool = False) -> torch.Tensor:
    return kernels.int8_mm_a8(x, w, s, res, silu=silu)


@int8_mm_a8.register_fake
def _(x, w, s, res=None, silu=False):
    return x.new_empty(*x.shape[:-1], w.shape[0] // 2 if silu else w.shape[0])


@torch.library.custom_op(f"{NS}::prefix_attn", mutates_args=())
def prefix_attn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, pos: torch.Tensor,
                gstart: Optional[torch.Tensor] = None, owner: Optional[torch.Tensor] = None,
                plen: Optional[torch.Tensor] = None, S: int = 1, scale: Optional[float] = None,
                seqs: Optional[torch.Tensor] = None) -> torch.Tensor:
    return kernels.prefix_attn(q, k, v, table, pos, gstart, owner, plen, S, scale=scale, seqs=seqs)


@prefix_attn.register_fake
def _(q, k, v, table, pos, gstart=None, owner=None, plen=None, S=1, scale=None, seqs=None):
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{NS}::rope_pages", mutates_args=("q_out", "k", "v"))
def rope_pages(qkv: torch.Tensor, rope: torch.Tensor, pos: torch.Tensor, q_out: torch.Tensor, k: torch.Tensor,
               v: torch.Tensor, table: torch.Tensor, S: int, Hq: int, Hk: int,
               seqs: Optional[torch.Tensor] = None) -> None:
    kernels.rope_pages(qkv, rope, pos, q_out, k, v, table, S, Hq, Hk, seqs)


@rope_pages.register_fake
def _(qkv, rope, pos, q_out, k, v, table, S, Hq, Hk, seqs=None):
    return None


@torch.library.custom_op(f"{NS}::pages_grow", mutates_args=("table", "lens", "refs"))
def pages_grow(table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, page: int, seqs: torch.Tensor,
               n: int = 1) -> None:
    kernels.pages_grow(table, lens, refs, page, seqs, n)


@pages_grow.register_fake
def _(table, lens, refs, page, seqs, n=1):
    return None


@torch.library.custom_op(f"{NS}::pages_free", mutates_args=("table", "lens", "refs"))
def pages_free(table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, seqs: torch.Tensor) -> None:
    kernels.pages_free(table, lens, refs, seqs)


@pages_free.register_fake
def _(table, lens, refs, seqs):
    return None


@torch.library.custom_op(f"{NS}::pages_fork", mutates_args=("k", "v", "table", "lens", "refs"))
def pages_fork(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor,
               src: torch.Tensor, dst: torch.Tensor) -> None:
    kernels.pages_fork(k, v, table, lens, refs, src, dst)


@pages_fork.register_fake
def _(k, v, table, lens, refs, src, dst):
    return None


@torch.library.custom_op(f"{NS}::pages_copy", mutates_args=("k", "v"))
def pages_copy(k: torch.Tensor, v: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    kernels.pages_copy(k, v, src, dst)


@pages_copy.register_fake
def _(k, v, src, dst):
    return None


@torch.library.custom_op(f"{NS}::pages_compact", mutates_args=("k", "v", "table", "refs"))
def pages_compact(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, refs: torch.Tensor) -> torch.Tensor:
    return kernels.pages_compact(k, v, table, refs)


@pages_compact.register_fake
def _(k, v, table, refs):
    return refs.new_empty(1)
