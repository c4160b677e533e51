"""Token embedding with scaling, and the gradient of its table (`csrc/embedding.cu`).

`y[n] = scale * table[tokens[n]]`; the gradient of row `v` is `scale` times the sum of `dy` over the positions that hold
token `v`, taken in fp32 in ascending order of position (positions sorted by token), so it does not change from run to
run, and rounded once to the table's type. Every row of the gradient is written: rows of unseen tokens are zero.
"""

from __future__ import annotations

import ctypes as C
from functools import lru_cache

import torch
from torch import Tensor

from param_decomp_b200.ops import native as nv
from param_decomp_b200.ops.elementwise import _FLOAT, _check, _dense, _flat_rows, _on_current_device, _s


@lru_cache(maxsize=1)
def _lib():
    lib = nv.lib()
    P, LL, I, F = C.c_void_p, C.c_longlong, C.c_int, C.c_float
    lib.pd_embedding.argtypes = [P, I, P, P, P, LL, LL, I, F, I, I, P, P, P]
    lib.pd_embedding_grad.argtypes = [P, P, P, LL, LL, I, F, I, I, P, P, P]
    lib.pd_embedding_grad_ints.argtypes, lib.pd_embedding_grad_ints.restype = [LL, LL], LL
    lib.pd_embedding_grad_floats.argtypes, lib.pd_embedding_grad_floats.restype = [LL, I], LL
    return lib


@lru_cache(maxsize=256)
def _scratch(n: int, rows: int, d: int) -> tuple[int, int]:
    """Ints and floats of the gradient's scratch."""
    return _lib().pd_embedding_grad_ints(n, rows), _lib().pd_embedding_grad_floats(n, d)


def _lookup(table: Tensor, tokens: Tensor, scale: float, out_dtype: torch.dtype, ids: Tensor | None) -> Tensor:
    """`tokens [n]` -> `[n, d]`; `ids [n]` int32 (or None) receives the tokens, unknown ones as -1."""
    n, (rows, d) = tokens.numel(), table.shape
    y = torch.empty(n, d, device=table.device, dtype=out_dtype)
    if n > 0:
        _check(_lib().pd_embedding(tokens.data_ptr(), tokens.dtype is torch.int64, table.data_ptr(), y.data_ptr(),
                                   None if ids is None else ids.data_ptr(), n, rows, d, scale, table.dtype is torch.float32,
                                   out_dtype is torch.float32,
                                   nv.status_word().data_ptr(), nv.refused_ptr(), _s()), "embedding")
    return y


def _grad(ids: Tensor, dy: Tensor, rows: int, scale: float, dtype: torch.dtype) -> Tensor:
    n, d = dy.shape
    dE = torch.empty(rows, d, device=dy.device, dtype=dtype)
    ints, floats = _scratch(n, rows, d)
    scratch = torch.empty(ints + floats, device=dy.device, dtype=torch.float32)
    _check(_lib().pd_embedding_grad(ids.data_ptr(), dy.data_ptr(), dE.data_ptr(), n, rows, d, scale,
                                    dy.dtype is torch.float32, dtype is torch.float32, scratch.data_ptr() + 4 * floats,
                                    scratch.data_ptr(), _s()), "embedding_grad")
    nv.count_launch()
    return dE


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table: Tensor, tokens: Tensor, scale: float, out_dtype: torch.dtype) -> Tensor:  # type: ignore[override]
        ids = torch.empty(tokens.shape[0], device=tokens.device, dtype=torch.int32)
        ctx.save_for_backward(ids)
        ctx.cfg = (table.shape[0], scale, table.dtype)
        return _lookup(_dense(table), tokens, scale, out_dtype, ids)

    @staticmethod
    def backward(ctx, dy: Tensor):  # type: ignore[override]
        rows, scale, dtype = ctx.cfg
        return _grad(ctx.saved_tensors[0], _flat_rows(dy, dy.shape[-1]), rows, scale, dtype), None, None, None


def embedding(tokens: Tensor, table: Tensor, scale: float = 1.0, out_dtype: torch.dtype | None = None) -> Tensor:
    """`scale * table[tokens]`: `tokens [...]` int32 or int64 in `[0, rows)`, `table [rows, d]` bf16 or fp32, the result
    `[..., d]` in `out_dtype` (the table's type by default); differentiable in `table`.

    A token outside the table is refused: its row is zero and takes no part in the gradient, `native.raise_refused` (made
    by the next call) raises, `native.check_status` raises at once."""
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"embedding: token ids are int32 or int64, not {tokens.dtype}")
    if table.dim() != 2 or table.dtype not in _FLOAT or 0 in table.shape:
        raise ValueError(f"embedding: the table is [rows, d] in bf16 or fp32, not {tuple(table.shape)} {table.dtype}")
    out_dtype = table.dtype if out_dtype is None else out_dtype
    if out_dtype not in _FLOAT:
        raise ValueError(f"embedding: the result is bf16 or fp32, not {out_dtype}")
    if tokens.numel() >= 1 << 30 or table.shape[0] >= 1 << 30:
        raise ValueError(f"embedding: fewer than 2^30 tokens and 2^30 rows, not {tokens.numel()} and {table.shape[0]}")
    _on_current_device("embedding", tokens, table)
    nv.raise_refused()
    flat = tokens if tokens.dim() == 1 else tokens.reshape(-1)
    flat = _dense(flat)
    if table.requires_grad and torch.is_grad_enabled():
        y = _Embedding.apply(table, flat, scale, out_dtype)
    else:
        y = _lookup(_dense(table), flat, scale, out_dtype, None)
    return y if tokens.dim() == 1 else y.view(*tokens.shape, table.shape[1])
