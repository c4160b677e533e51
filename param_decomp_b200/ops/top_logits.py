"""The top logits of a teacher, and the distillation loss that reads them (`csrc/top_logits.cu`, `csrc/top_kl.cu`).

A teacher's row of `V` logits is kept as its `k` largest (`top_logits`), their columns and `tail`, the logarithm of the
sum of exponentials of all others: a distribution over `k + 1` events. `top_kl` is the divergence from it to the student's
softmax, grouped into the same events. At `k = V - 1` and at `k = V` it is the divergence over the whole vocabulary that
`vocab_kl` computes, below that never more; it reads one row of logits a position instead of two.

With one slot and no tail, `top_kl` is the cross entropy of a target: `next_token_loss`.

The `eager_*` functions are the same definitions in plain torch, for any device.
"""

from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import NamedTuple

import torch
from torch import Tensor

from param_decomp_b200.ops import native as nv
from param_decomp_b200.ops.elementwise import _FLOAT, _dense, _flat_rows, _on_current_device

MAX_K = 256


class TopLogits(NamedTuple):
    values: Tensor  # [..., k] the k largest logits, descending, in the logits' type
    indices: Tensor  # [..., k] int32 columns; equal logits in the order of their columns
    tail: Tensor  # [...] fp32 logsumexp of all other logits over the temperature (-inf where k is the whole row)


@lru_cache(maxsize=4)
def _max_columns(what: str, fp32: bool) -> int:
    """The widest row that a cluster's shared memory holds."""
    f = nv.lib().pd_top_logits_max_columns if what == "top_logits" else nv.lib().pd_top_kl_max_columns
    f.argtypes, f.restype = [C.c_int], C.c_longlong
    return f(fp32)


def _check_width(what: str, logits: Tensor) -> None:
    limit = _max_columns(what, logits.dtype is torch.float32)
    if logits.shape[-1] > limit:
        raise ValueError(f"{what}: rows of at most {limit} {logits.dtype} logits, not {logits.shape[-1]}")


def _rows_of(logits: Tensor) -> Tensor:
    """`[rows, V]` view with neighbouring columns and rows that do not overlap (a copy where there is none)."""
    V = logits.shape[-1]
    z = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if not z.is_contiguous() and ((V > 1 and z.stride(1) != 1) or (z.shape[0] > 1 and z.stride(0) < V)):
        z = z.contiguous()
    return z


def _pitch(z: Tensor) -> int:
    return z.stride(0) if z.shape[0] > 1 else z.shape[1]


def _check_logits(what: str, logits: Tensor, temperature: float) -> None:
    if logits.dtype not in _FLOAT:
        raise ValueError(f"{what}: logits are bf16 or fp32, not {logits.dtype}")
    if logits.dim() < 1 or not 1 <= logits.shape[-1] < 1 << 31:
        raise ValueError(f"{what}: logits of shape {tuple(logits.shape)}")
    if logits.numel() // logits.shape[-1] >= 1 << 28:
        raise ValueError(f"{what}: fewer than 2^28 rows")
    if not 2.0**-120 <= temperature <= 2.0**120:  # its inverse is taken in fp32
        raise ValueError(f"{what}: a temperature from 2^-120 to 2^120, not {temperature}")


def top_logits(logits: Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The `k` largest of each row of `logits [..., V]` (bf16 or fp32, `1 <= k <= min(V, 256)`), their columns and the
    logsumexp of `logits / temperature` (2^-120 to 2^120) over the rest of the row. NaN counts as the largest. Not
    differentiable."""
    _check_logits("top_logits", logits, temperature)
    V = logits.shape[-1]
    if not 1 <= k <= min(V, MAX_K):
        raise ValueError(f"top_logits: k from 1 to {min(V, MAX_K)}, not {k}")
    _on_current_device("top_logits", logits)
    _check_width("top_logits", logits)
    return TopLogits(*nv.autograd().top_logits(_rows_of(logits.detach()), logits.shape[:-1], k, temperature, nv.status_ptr()))


def _arguments(what: str, logits: Tensor, indices: Tensor, values: Tensor, tail: Tensor | None, temperature: float):
    _check_logits(what, logits, temperature)
    lead = logits.shape[:-1]
    if indices.dtype not in (torch.int32, torch.int64) or indices.shape[:-1] != lead or indices.dim() != logits.dim():
        raise ValueError(f"{what}: columns are int32 or int64 of shape {tuple(lead)} + [k], not {indices.dtype} "
                         f"{tuple(indices.shape)}")
    k = indices.shape[-1]
    if not 1 <= k <= MAX_K:
        raise ValueError(f"{what}: 1 to {MAX_K} slots a row, not {k}")
    if values.dtype not in _FLOAT or values.shape != indices.shape:
        raise ValueError(f"{what}: values are bf16 or fp32 of shape {tuple(indices.shape)}, not {values.dtype} "
                         f"{tuple(values.shape)}")
    if tail is not None and (tail.dtype != torch.float32 or tail.shape != lead):
        raise ValueError(f"{what}: the tail is fp32 of shape {tuple(lead)}, not {tail.dtype} {tuple(tail.shape)}")
    _on_current_device(what, logits, indices, values, tail)
    _check_width(what, logits)
    nv.raise_refused()
    return (_rows_of(logits), _flat_rows(indices, k), _flat_rows(values.detach(), k),
            None if tail is None else _dense(tail.detach().reshape(-1)))


def top_kl(logits: Tensor, indices: Tensor, values: Tensor, tail: Tensor | None = None, temperature: float = 1.0) -> Tensor:
    """Divergence of every row from its teacher, `[...]` fp32, differentiable in `logits`.

    `logits [..., V]` bf16 or fp32: the student's. `indices`, `values [..., k]`: the teacher's logits and their columns
    (int32 or int64; negative: an unused slot; one that is not below `V` is refused like an unused slot and reported as
    `native.raise_refused` does). `tail [...]`: the teacher's logsumexp of all other logits over the temperature; without it
    the teacher has its `k` slots alone. Both sides are taken at `temperature` (2^-120 to 2^120). A row whose teacher has no
    mass counts zero, with a zero gradient; a NaN that takes part on either side makes the row's loss and gradient NaN.

    The loss is a sum over slots, `p_k (log p_k - log q_k)` each. The slots of a column that is named more than once share its
    gradient with the sum of their probabilities, but each counts by its own `p_k`: the loss is then below the divergence by
    what the split of the column costs, a number that does not depend on `logits`."""
    z, indices, values, tail = _arguments("top_kl", logits, indices, values, tail, temperature)
    loss = nv.autograd().top_kl(z, indices, values, tail, temperature, nv.status_ptr(), nv.refused_ptr())
    return loss if logits.dim() == 2 else loss.view(logits.shape[:-1])


def top_kl_rows(logits: Tensor, indices: Tensor, values: Tensor, tail: Tensor | None = None, temperature: float = 1.0,
                want_grad: bool = True) -> tuple[Tensor, Tensor | None]:
    """`top_kl` of `[rows, V]` logits and (optionally) its gradient with respect to them, each row's by its own loss, in
    one pass over the logits (the counterpart of `elementwise.vocab_kl_rows`; no autograd)."""
    if logits.dim() != 2:
        raise ValueError(f"top_kl_rows: logits [rows, V], not {tuple(logits.shape)}")
    z, indices, values, tail = _arguments("top_kl_rows", logits.detach(), indices, values, tail, temperature)
    return nv.autograd().top_kl_rows(z, indices, values, tail, temperature, want_grad, nv.status_ptr(), nv.refused_ptr())


def next_token_loss(logits: Tensor, targets: Tensor) -> Tensor:
    """Mean cross entropy of `targets [...]` (int32 or int64; negative: no target here, as it counts for nothing, not for
    the mean either) under `logits [..., V]`."""
    loss = top_kl(logits, targets.unsqueeze(-1), torch.zeros(*targets.shape, 1, device=logits.device))
    return loss.sum() / (targets >= 0).sum()


# ---- plain torch ----------------------------------------------------------------------------------------------------

def eager_top_logits(logits: Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    indices = torch.sort(logits.detach(), dim=-1, descending=True, stable=True)[1][..., :k]
    rest = (logits.detach().float() / temperature).scatter(-1, indices, float("-inf"))
    return TopLogits(torch.gather(logits.detach(), -1, indices), indices.to(torch.int32), torch.logsumexp(rest, -1))


def eager_top_kl(logits: Tensor, indices: Tensor, values: Tensor, tail: Tensor | None = None,
                 temperature: float = 1.0) -> Tensor:
    used = indices >= 0
    columns = indices.long().clamp(min=0)
    z = logits if logits.dtype == torch.float64 else logits.float()
    top = z.detach().amax(-1, keepdim=True)  # taken off first: the type's lowest value over a temperature may leave fp32
    logq = torch.log_softmax((z - torch.where(top.isfinite(), top, 0.0)) / temperature, -1)
    low = torch.full_like(logq[..., :1], float("-inf"))
    teacher = torch.where(used, values.double() / temperature, low.double())
    teacher = torch.cat([teacher, (low if tail is None else tail.unsqueeze(-1)).double()], -1)
    live = (teacher > float("-inf")).any(-1, keepdim=True)
    logp = torch.log_softmax(torch.where(live, teacher, 0.0), -1).to(logq.dtype)
    # unused slots point at column 0 and must not name it
    named = torch.zeros_like(logq).scatter_add_(-1, columns, used.to(logq.dtype)) > 0
    others = logq.masked_fill(named, float("-inf"))
    some = (others > float("-inf")).any(-1, keepdim=True)
    rest = torch.where(some, torch.logsumexp(torch.where(some, others, 0.0), -1, keepdim=True), low)
    events = torch.cat([torch.gather(logq, -1, columns), rest], -1)
    counts = live & (logp > float("-inf"))
    return torch.where(counts, logp.exp() * (logp - torch.where(counts, events, 0.0)), 0.0).sum(-1)
