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

from array import array
from operator import attrgetter
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib
from .tensor import TensorError, _fail

_TYPE_OF = attrgetter("dtype")
_DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


def _run(name: str, index: int, *args) -> None:
    """Calls an entry point of the library on device `index`, with that
    device's current stream as the last argument."""
    fn = getattr(_lib.lib(), name)
    stream = torch._C._cuda_getCurrentRawStream(index)  # current_stream(index).cuda_stream without its object
    if torch.cuda.current_device() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _dtype(op: str, name: str, t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype) if isinstance(t, torch.Tensor) and t.is_cuda else None
    if code is None:
        _fail(op, f"{name} must be a float32, bfloat16 or float16 CUDA tensor")
    return code


def _int32(op: str, name: str, t: torch.Tensor, index: int) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.get_device() != index:
        _fail(op, f"{name} must be an int32 tensor on cuda:{index}")
    return t if t.is_contiguous() else t.contiguous()


def _padding(op: str, padding: int) -> int:
    if not -2 ** 31 <= padding < 2 ** 31:  # the call would take its lower 32 bits
        _fail(op, f"padding {padding} is not an int32")
    return padding


def _float32(op: str, name: str, t: torch.Tensor, rows: int, index: int) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.get_device() != index or t.numel() != rows:
        _fail(op, f"{name} must be {rows} float32 values on cuda:{index}")
    return t if t.is_contiguous() else t.contiguous()


def _stride(t: torch.Tensor, rows: int, cols: int) -> int:
    """The distance of t's rows, 0 where they are not contiguous or overlap."""
    s0, s1 = t.stride()
    if s1 != 1 and cols > 1 or s0 < cols and rows > 1:
        return 0
    return s0 if s0 > cols else cols


def _rows(t: torch.Tensor, rows: int, cols: int):
    """t with contiguous rows, and their distance."""
    ld = _stride(t, rows, cols)
    return (t, ld) if ld else (t.contiguous(), cols)


def Check(device=None) -> None:
    """Waits for the work of a device (the current one where none or "cuda" is
    given) and raises what its kernels reported: an id or a target out of
    range (status FG_EINVAL). The current device stays what it is."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        _fail("Check", f"{device} is not a CUDA device")
    index = torch.cuda.current_device() if device.index is None else device.index
    with torch.cuda.device(index):  # fg_synchronize makes its device the current one
        rc = _lib.lib().fg_synchronize(index)
    _lib.check(rc)


def Embedding(table: torch.Tensor, ids: torch.Tensor, scale: float = 1.0, padding: int = -1,
              dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """scale · table[ids] for a table [vocab, dim] and int32 ids of any shape:
    [*ids, dim] of ``dtype`` (the table's where None). A token whose id is
    ``padding`` has a zero row; -1 stands for empty slots."""
    op = "Embedding"
    code = _dtype(op, "table", table)
    shape = table.shape
    if len(shape) != 2 or shape[1] == 0:
        _fail(op, f"table must be 2-D, got {list(shape)}")
    vocab, dim = shape
    if dtype is None:
        dtype = table.dtype
    out_code = _DTYPES.get(dtype)
    if out_code is None:
        _fail(op, f"no output type {dtype}")
    index = table.get_device()
    ids = _int32(op, "ids", ids, index)
    table, ld = _rows(table, vocab, dim)
    out = table.new_empty((*ids.shape, dim), dtype=dtype)
    _run("fg_embedding", index, table.data_ptr(), code, vocab, dim, ld, ids.data_ptr(), ids.numel(), scale,
         _padding(op, padding), out.data_ptr(), out_code, dim)
    return out


def _grad_args(op: str, dy: torch.Tensor, ids: torch.Tensor, vocab: int, dtype: Optional[torch.dtype]):
    code = _dtype(op, "dy", dy)
    shape = dy.shape
    if len(shape) < 2 or shape[-1] == 0:
        _fail(op, f"dy must be [tokens, dim], got {list(shape)}")
    index = dy.get_device()
    ids = _int32(op, "ids", ids, index)
    if shape[:-1] != ids.shape:
        _fail(op, f"dy {list(shape)} does not match ids {list(ids.shape)}")
    if vocab < 0:
        _fail(op, f"vocabulary of {vocab}")
    if dtype is not None and dtype not in _DTYPES:
        _fail(op, f"no output type {dtype}")
    if len(shape) != 2:
        dy = dy.reshape(-1, shape[-1])
    n, dim = ids.numel(), shape[-1]
    dy, ld = _rows(dy, n, dim)
    return code, dy, ld, ids, n, dim, index


def EmbeddingGrad(dy: torch.Tensor, ids: torch.Tensor, vocab: int, scale: float = 1.0, padding: int = -1,
                  dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None,
                  accumulate: bool = False) -> torch.Tensor:
    """The gradient [vocab, dim] of ``Embedding``'s table: row v is scale ·
    the sum of dy's rows whose id is v. Written to ``out`` where given, or
    added to it with ``accumulate`` (then rows without a token are not
    touched); otherwise a new tensor of ``dtype`` (dy's where None)."""
    op = "EmbeddingGrad"
    code, dy, ld, ids, n, dim, index = _grad_args(op, dy, ids, vocab, dtype)
    if out is None:
        if accumulate:
            _fail(op, "accumulate needs out")
        out, ldo = dy.new_empty((vocab, dim), dtype=dtype), dim
    else:
        _dtype(op, "out", out)
        if out.get_device() != index or tuple(out.shape) != (vocab, dim) or dtype not in (None, out.dtype):
            _fail(op, f"out must be [{vocab}, {dim}] on cuda:{index}, got {out.dtype} {list(out.shape)}")
        ldo = _stride(out, vocab, dim)
        if not ldo:
            _fail(op, "out must have contiguous rows")
    _run("fg_embedding_grad", index, dy.data_ptr(), code, ld, ids.data_ptr(), n, vocab, dim, scale,
         _padding(op, padding), out.data_ptr(), _DTYPES[out.dtype], ldo, int(accumulate))
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
    code, dy, ld, ids, n, dim, index = _grad_args(op, dy, ids, vocab, dtype)
    row_ids, count = ids.new_empty(n), ids.new_empty(1)
    rows = dy.new_empty((n, dim), dtype=dtype)
    _run("fg_embedding_grad_rows", index, dy.data_ptr(), code, ld, ids.data_ptr(), n, vocab, dim, scale,
         _padding(op, padding), row_ids.data_ptr(), rows.data_ptr(), _DTYPES[rows.dtype], dim, count.data_ptr())
    return RowsGrad(row_ids, rows, count)


class _LogProbsFields(NamedTuple):
    LogProb: torch.Tensor
    Entropy: torch.Tensor
    LogSum: torch.Tensor
    TopIndex: Optional[torch.Tensor]
    TopLogProb: Optional[torch.Tensor]


class LogProbsResult(_LogProbsFields):
    """LogProb, Entropy and LogSum [rows] float32; TopIndex (int32) and
    TopLogProb [rows, top], None where no alternatives were asked for. Beside
    these five, Peak [2, rows] float32: every row's largest logit and that
    one's log probability."""
    _sums: torch.Tensor  # [3, rows], the first three; the peak lies between its first two rows

    @property
    def Peak(self) -> torch.Tensor:
        rows = self._sums.shape[1]
        return self._sums.as_strided((2, rows), (rows, 1), self._sums.storage_offset() + rows)


def _logits(op: str, logits: torch.Tensor, targets: torch.Tensor, scale: float):
    code = _dtype(op, "logits", logits)
    shape = logits.shape
    if len(shape) != 2 or shape[1] == 0:
        _fail(op, f"logits must be [rows, width], got {list(shape)}")
    rows, width = shape
    index = logits.get_device()
    targets = _int32(op, "targets", targets, index)
    if targets.numel() != rows:
        _fail(op, f"{targets.numel()} targets for {rows} rows")
    if not 0 < scale < float("inf"):
        _fail(op, f"scale {scale} must be positive and finite")
    logits, ld = _rows(logits, rows, width)
    return code, logits, ld, targets, rows, width, index


def LogProbs(logits: torch.Tensor, targets: torch.Tensor, scale: float = 1.0, top: int = 0) -> LogProbsResult:
    """log softmax(scale · logits)[r, targets[r]] of every row (0 where the
    target is negative), with the rows' entropies, log sums and ``top`` most
    probable columns (equal logits by ascending index)."""
    op = "LogProbs"
    code, logits, ld, targets, rows, width, index = _logits(op, logits, targets, scale)
    if scale > _lib.MAX_SCALE:
        _fail(op, f"scale {scale} is too large")
    if not 0 <= top <= min(width, _lib.MAX_TOP):
        _fail(op, f"{top} alternatives of {width} columns (at most {_lib.MAX_TOP})")
    # three rows with room for two between them: one allocation, and three views in one call
    out = logits.new_empty_strided((3, rows), (3 * rows, 1), dtype=torch.float32)
    at = out.data_ptr()
    place = value = place_at = value_at = None
    if top:
        place, value = targets.new_empty((rows, top)), out.new_empty((rows, top))
        place_at, value_at = place.data_ptr(), value.data_ptr()
    _run("fg_log_probs_peak", index, logits.data_ptr(), code, rows, width, ld, targets.data_ptr(), scale, top, at,
         at + 12 * rows, at + 24 * rows, at + 4 * rows, place_at, value_at)
    result = LogProbsResult(*out.unbind(), place, value)
    result._sums = out
    return result


def LogProbsGrad(logits: torch.Tensor, targets: torch.Tensor, lse: Optional[torch.Tensor], dlogprob: torch.Tensor,
                 entropy: Optional[torch.Tensor] = None, dentropy: Optional[torch.Tensor] = None,
                 scale: float = 1.0, out: Optional[torch.Tensor] = None,
                 peak: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits' gradient of ``LogProbs`` from its LogSum or its Peak (and
    Entropy) and the gradients of its log probabilities and, where
    ``dentropy`` is given, of its entropies. ``out`` may be the logits
    themselves; a new tensor has their rows' distance where that is little
    more than their length.

    A LogSum far from 0 has no room in 32 bits for what tells a row's
    probabilities (for a row of the type's lowest value, or logits with an
    offset of 1e6): its rounding is a relative error of about 2^-24 |lse| in
    all of them. With ``peak`` such rows are as exact as others; ``lse`` is not
    looked at then and may be None."""
    op = "LogProbsGrad"
    code, x, ld, targets, rows, width, index = _logits(op, logits, targets, scale)
    if peak is None:
        sums = _float32(op, "lse", lse, rows, index)
    else:
        sums = _float32(op, "peak", peak, 2 * rows, index)
    dlogprob = _float32(op, "dlogprob", dlogprob, rows, index)
    entropy_at = dentropy_at = None
    if dentropy is not None:
        dentropy = _float32(op, "dentropy", dentropy, rows, index)
        if entropy is None:
            _fail(op, "dentropy needs entropy")
        entropy = _float32(op, "entropy", entropy, rows, index)
        entropy_at, dentropy_at = entropy.data_ptr(), dentropy.data_ptr()
    if out is None:
        # rows as far apart as the logits' own, so that both lie alike in memory
        ldo = ld if ld - width < 64 else width
        out = x.new_empty((rows, ldo))
        if ldo != width:
            out = out[:, :width]
    else:
        if not isinstance(out, torch.Tensor) or out.dtype != x.dtype or out.get_device() != index or out.shape != x.shape:
            _fail(op, f"out must be {x.dtype} [{rows}, {width}] on cuda:{index}")
        ldo = _stride(out, rows, width)
        if not ldo:
            _fail(op, "out must have contiguous rows")
    _run("fg_log_probs_grad" if peak is None else "fg_log_probs_grad_peak", index, x.data_ptr(), code, rows, width, ld,
         targets.data_ptr(), scale, sums.data_ptr(), entropy_at, dlogprob.data_ptr(), dentropy_at, out.data_ptr(), ldo)
    return out


def _packed(grads: Sequence[torch.Tensor]) -> Optional[list]:
    """The gradients with packed copies of those whose rows lie apart, None
    where one has no such rows."""
    got = []
    for g in grads:
        if not g.is_contiguous():
            if g.dim() != 2 or not _stride(g, *g.shape):
                return None
            g = g.contiguous()
        got.append(g)
    return got


def ClipGradNorm(grads: Sequence[torch.Tensor], max_norm: float,
                 out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """The Euclidean norm of all gradients together (a float32 scalar on
    their device), and every gradient times max_norm / norm where the norm is
    finite and larger: in place, or into the tensors of ``out``. A norm that
    is not finite changes nothing. The tensors are on one device and
    contiguous, or matrices with rows apart (as ``LogProbsGrad`` has for padded
    logits), which go through a packed copy; their types may differ. Those of
    ``out`` are contiguous."""
    op = "ClipGradNorm"
    if not max_norm >= 0:
        _fail(op, f"max_norm {max_norm} must be at least 0")
    n = len(grads)
    if n == 0:
        _fail(op, "no gradients")
    # one pass of C calls for each thing asked of the tensors: there may be hundreds
    T = torch.Tensor
    try:
        types = list(map(_TYPE_OF, grads))
        codes = list(map(_DTYPES.__getitem__, types))
        index = grads[0].get_device()
        alike = index >= 0 and set(map(T.get_device, grads)) == {index}
        packed = grads if all(map(T.is_contiguous, grads)) else _packed(grads)
        sizes = list(map(T.numel, grads))
    except (KeyError, AttributeError, TypeError):
        _fail(op, "gradients must be float32, bfloat16 or float16 tensors")
    if not alike or packed is None:
        _fail(op, "gradients must be tensors on one CUDA device, contiguous or matrices with rows apart")
    outs = outs_at = None
    if out is not None:
        if len(out) != n or list(map(_TYPE_OF, out)) != types or list(map(T.numel, out)) != sizes or \
                set(map(T.get_device, out)) != {index} or not all(map(T.is_contiguous, out)):
            _fail(op, "out must match the gradients' sizes, types and device, contiguous")
        outs = array("Q", map(T.data_ptr, out))
        outs_at = outs.buffer_info()[0]
    ins, sizes, codes = array("Q", map(T.data_ptr, packed)), array("q", sizes), array("i", codes)
    norm = grads[0].new_empty((), dtype=torch.float32)
    _run("fg_clip_grad_norm", index, n, ins.buffer_info()[0], sizes.buffer_info()[0], codes.buffer_info()[0], outs_at,
         max_norm, norm.data_ptr())
    if packed is not grads and out is None:
        with torch.no_grad():
            for g, p in zip(grads, packed):
                if p is not g:
                    g.copy_(p)
    return norm
