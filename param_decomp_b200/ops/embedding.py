"""Token embedding with scaling, and the gradient of its table (`csrc/embedding.cu`).

`y[n] = scale * table[tokens[n]]`; the gradient of row `v` is `scale` times the sum of `dy` over the positions that hold
token `v`, taken in fp32 and rounded once to the table's type. Positions are sorted by token: up to 32 of a token are added
in ascending order, more by groups of threads over 32 places of the sorted order each, whose sums are added in their order;
either way the order depends on the sizes and the tokens alone, so the gradient does not change from run to run. Every row of
it is written: rows of unseen tokens are zero.
"""

from __future__ import annotations

import torch
from torch import Tensor

from param_decomp_b200.ops import native as nv
from param_decomp_b200.ops.elementwise import _FLOAT, _on_current_device


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
    return nv.autograd().embedding(tokens, table, scale, out_dtype is torch.float32, nv.status_ptr(), nv.refused_ptr())
