"""The device operators of a training step over an embedding table, through
libfgemma's C ABI on CUDA tensors (the reference trains on the CPU with its
autograd, tensor/autograd.go):

- ``Embedding``: rows of a table by token id, scaled; ``EmbeddingGrad`` and
  ``EmbeddingGradRows``: the table's gradient, whole or only the rows met;
- ``LogProbs``: log probabilities of given columns of logit rows (a
  similarity matrix for a contrastive loss, or a vocabulary), with entropy
  and the most probable columns; ``LogProbsGrad``: the logits' gradient;
- ``ClipGradNorm``: the global norm of many gradients and their clipping.

The operators run on the current stream of their tensors' device and do not
synchronise. Values are float32, bfloat16 or float16 in memory, sums in 32
bits or more; ids and targets are int32. An id or a target outside its range
is skipped, and reported by ``Check``. Shape and type errors raise
``TensorError``.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib
from .tensor import TensorError, _fail

_DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


def _run(name: str, device: torch.device, *args) -> None:
    """Calls an entry point on the device's current stream, its last argument."""
    stream = torch.cuda.current_stream(device).cuda_stream
    fn = getattr(_lib.lib(), name)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _dtype(op: str, name: str, t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype) if isinstance(t, torch.Tensor) and t.is_cuda else None
    if code is None:
        _fail(op, f"{name} must be a float32, bfloat16 or float16 CUDA tensor")
    return code


def _int32(op: str, name: str, t: torch.Tensor, device: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device:
        _fail(op, f"{name} must be an int32 tensor on {device}")
    return t.contiguous()


def _float32(op: str, name: str, t: torch.Tensor, rows: int, device: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != device or t.numel() != rows:
        _fail(op, f"{name} must be {rows} float32 values on {device}")
    return t.contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous rows at a stride of at least their length."""
    if t.stride(1) != 1 and t.shape[1] > 1 or t.stride(0) < t.shape[1] and t.shape[0] > 1:
        return t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def Check(device=None) -> None:
    """Waits for the device's work and raises what its kernels reported: an
    id or a target out of range (status FG_EINVAL)."""
    index = torch.cuda.current_device() if device is None else torch.device(device).index or 0
    _lib.check(_lib.lib().fg_synchronize(index))


def Embedding(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding: int = -1,
              dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """scale · table[ids] for a table [vocab, dim] and int32 ids of any shape:
    [*ids, dim] of ``dtype`` (the table's where None). A token whose id is
    ``padding`` has a zero row; -1 stands for empty slots."""
    op = "Embedding"
    code = _dtype(op, "table", table)
    if table.dim() != 2 or table.shape[1] == 0:
        _fail(op, f"table must be 2-D, got {list(table.shape)}")
    dtype = table.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        _fail(op, f"no output type {dtype}")
    ids = _int32(op, "ids", ids, table.device)
    table = _rows(table)
    vocab, dim = table.shape
    out = torch.empty((*ids.shape, dim), dtype=dtype, device=table.device)
    _run("fg_embedding", table.device, table.data_ptr(), code, vocab, dim, _ld(table), ids.data_ptr(), ids.numel(),
         scale, padding, out.data_ptr(), _DTYPES[dtype], dim)
    return out


def _grad_args(op: str, dy: torch.Tensor, ids: torch.Tensor, vocab: int, dtype: Optional[torch.dtype]):
    code = _dtype(op, "dy", dy)
    if dy.dim() < 2 or dy.shape[-1] == 0:
        _fail(op, f"dy must be [tokens, dim], got {list(dy.shape)}")
    ids = _int32(op, "ids", ids, dy.device)
    if dy.shape[:-1] != ids.shape:
        _fail(op, f"dy {list(dy.shape)} does not match ids {list(ids.shape)}")
    if vocab < 0:
        _fail(op, f"vocabulary of {vocab}")
    if dtype is not None and dtype not in _DTYPES:
        _fail(op, f"no output type {dtype}")
    if dy.dim() != 2:
        dy = dy.reshape(-1, dy.shape[-1])
    return code, _rows(dy), ids


def EmbeddingGrad(dy: torch.Tensor, ids: torch.Tensor, vocab: int, scale: float = 1.0, padding: int = -1,
                  dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                  accumulate: bool = False) -> torch.Tensor:
    """The gradient [vocab, dim] of ``Embedding``'s table: row v is scale ·
    the sum of dy's rows whose id is v. Written to ``out`` where given, or
    added to it with ``accumulate`` (then rows without a token are not
    touched); otherwise a new tensor of ``dtype`` (dy's where None)."""
    op = "EmbeddingGrad"
    code, dy, ids = _grad_args(op, dy, ids, vocab, dtype)
    dim = dy.shape[1]
    if out is None:
        if accumulate:
            _fail(op, "accumulate needs out")
        out_dtype = dy.dtype if dtype is None else dtype
    else:
        _dtype(op, "out", out)
        if out.device != dy.device or tuple(out.shape) != (vocab, dim) or dtype not in (None, out.dtype):
            _fail(op, f"out must be [{vocab}, {dim}] on {dy.device}, got {out.dtype} {list(out.shape)}")
        if out.stride(1) != 1 and dim > 1 or out.stride(0) < dim and vocab > 1:
            _fail(op, "out must have contiguous rows")
        out_dtype = out.dtype
    if out is None:
        out = torch.empty((vocab, dim), dtype=out_dtype, device=dy.device)
    _run("fg_embedding_grad", dy.device, dy.data_ptr(), code, _ld(dy), ids.data_ptr(), ids.numel(), vocab, dim, scale,
         padding, out.data_ptr(), _DTYPES[out_dtype], _ld(out), int(accumulate))
    return out


class RowsGrad(NamedTuple):
    """A table's gradient without the rows that no token met: Ids [n] int32
    ascending, -1 past the count; Rows [n, dim], zero past it; Count [1]."""
    Ids: torch.Tensor
    Rows: torch.Tensor
    Count: torch.Tensor


def EmbeddingGradRows(dy: torch.Tensor, ids: torch.Tensor, vocab: int, scale: float = 1.0, padding: int = -1,
                      dtype: Optional[torch.dtype] = None) -> RowsGrad:
    """``EmbeddingGrad``'s rows that have tokens, on the device without a
    synchronisation: room for as many rows as there are tokens."""
    op = "EmbeddingGradRows"
    code, dy, ids = _grad_args(op, dy, ids, vocab, dtype)
    n, dim = dy.shape
    out_dtype = dy.dtype if dtype is None else dtype
    row_ids = torch.empty(n + 1, dtype=torch.int32, device=dy.device)
    rows = torch.empty((n, dim), dtype=out_dtype, device=dy.device)
    at = row_ids.data_ptr()
    _run("fg_embedding_grad_rows", dy.device, dy.data_ptr(), code, _ld(dy), ids.data_ptr(), n, vocab, dim, scale,
         padding, at, rows.data_ptr(), _DTYPES[out_dtype], dim, at + 4 * n)
    return RowsGrad(row_ids[:n], rows, row_ids[n:])


class LogProbsResult(NamedTuple):
    """LogProb, Entropy and LogSum [rows] float32; TopIndex (int32) and
    TopLogProb [rows, top], None where no alternatives were asked for."""
    LogProb: torch.Tensor
    Entropy: torch.Tensor
    LogSum: torch.Tensor
    TopIndex: Optional[torch.Tensor]
    TopLogProb: Optional[torch.Tensor]


def _logits(op: str, logits: torch.Tensor, targets: torch.Tensor, scale: float):
    code = _dtype(op, "logits", logits)
    if logits.dim() != 2 or logits.shape[1] == 0:
        _fail(op, f"logits must be [rows, width], got {list(logits.shape)}")
    targets = _int32(op, "targets", targets, logits.device)
    if targets.numel() != logits.shape[0]:
        _fail(op, f"{targets.numel()} targets for {logits.shape[0]} rows")
    if not 0 < scale < float("inf"):
        _fail(op, f"scale {scale} must be positive and finite")
    return code, _rows(logits), targets


def LogProbs(logits: torch.Tensor, targets: torch.Tensor, scale: float = 1.0, top: int = 0) -> LogProbsResult:
    """log softmax(scale · logits)[r, targets[r]] of every row (0 where the
    target is negative), with the rows' entropies, log sums and ``top`` most
    probable columns (equal logits by ascending index)."""
    op = "LogProbs"
    code, logits, targets = _logits(op, logits, targets, scale)
    rows, width = logits.shape
    if not 0 <= top <= min(width, _lib.MAX_TOP):
        _fail(op, f"{top} alternatives of {width} columns (at most {_lib.MAX_TOP})")
    out = torch.empty((3, rows), dtype=torch.float32, device=logits.device)
    at = out.data_ptr()
    index = value = None
    if top:
        index = torch.empty((rows, top), dtype=torch.int32, device=logits.device)
        value = torch.empty((rows, top), dtype=torch.float32, device=logits.device)
    _run("fg_log_probs", logits.device, logits.data_ptr(), code, rows, width, _ld(logits), targets.data_ptr(), scale,
         top, at, at + 4 * rows, at + 8 * rows, index.data_ptr() if top else None, value.data_ptr() if top else None)
    logprob, entropy, lse = out
    return LogProbsResult(logprob, entropy, lse, index, value)


def LogProbsGrad(logits: torch.Tensor, targets: torch.Tensor, lse: torch.Tensor, dlogprob: torch.Tensor,
                 entropy: Optional[torch.Tensor] = None, dentropy: Optional[torch.Tensor] = None,
                 scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits' gradient of ``LogProbs`` from its LogSum (and Entropy) and
    the gradients of its log probabilities and, where ``dentropy`` is given,
    of its entropies. ``out`` may be the logits themselves."""
    op = "LogProbsGrad"
    code, x, targets = _logits(op, logits, targets, scale)
    rows, width = x.shape
    lse = _float32(op, "lse", lse, rows, x.device)
    dlogprob = _float32(op, "dlogprob", dlogprob, rows, x.device)
    if dentropy is not None:
        dentropy = _float32(op, "dentropy", dentropy, rows, x.device)
        if entropy is None:
            _fail(op, "dentropy needs entropy")
        entropy = _float32(op, "entropy", entropy, rows, x.device)
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.dtype != x.dtype or out.device != x.device or out.shape != x.shape:
            _fail(op, f"out must be {x.dtype} [{rows}, {width}] on {x.device}")
        if out.stride(1) != 1 and width > 1 or out.stride(0) < width and rows > 1:
            _fail(op, "out must have contiguous rows")
    if out is None:
        out = torch.empty((rows, width), dtype=x.dtype, device=x.device)
    _run("fg_log_probs_grad", x.device, x.data_ptr(), code, rows, width, _ld(x), targets.data_ptr(), scale,
         lse.data_ptr(), None if dentropy is None else entropy.data_ptr(), dlogprob.data_ptr(),
         None if dentropy is None else dentropy.data_ptr(), out.data_ptr(), _ld(out))
    return out


def ClipGradNorm(grads: Sequence[torch.Tensor], max_norm: float,
                 out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """The Euclidean norm of all gradients together (a float32 scalar on
    their device), and every gradient times max_norm / norm where the norm is
    finite and larger: in place, or into the tensors of ``out``. A norm that
    is not finite changes nothing. The tensors are contiguous and on one
    device; their types may differ."""
    op = "ClipGradNorm"
    if not max_norm >= 0:
        _fail(op, f"max_norm {max_norm} must be at least 0")
    n = len(grads)
    if n == 0:
        _fail(op, "no gradients")
    device = grads[0].device
    try:
        codes = [_DTYPES[g.dtype] for g in grads]
    except (KeyError, AttributeError):
        _fail(op, "gradients must be float32, bfloat16 or float16 tensors")
    if not all([g.device == device and g.is_contiguous() for g in grads]) or device.type != "cuda":
        _fail(op, "gradients must be contiguous tensors on one CUDA device")
    outs = None
    if out is not None:
        if len(out) != n or not all([o.dtype == g.dtype and o.shape == g.shape and o.device == device and
                                     o.is_contiguous() for o, g in zip(out, grads)]):
            _fail(op, "out must match the gradients' shapes, types and device, contiguous")
        outs = (C.c_void_p * n)(*[o.data_ptr() for o in out])
    norm = torch.empty((), dtype=torch.float32, device=device)
    _run("fg_clip_grad_norm", device, n, (C.c_void_p * n)(*[g.data_ptr() for g in grads]),
         (C.c_int64 * n)(*[g.numel() for g in grads]), (C.c_int * n)(*codes), outs, max_norm, norm.data_ptr())
    return norm
