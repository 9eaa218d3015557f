"""Operators on dense tensors next to the sparse kernel: what a model with an embedding table needs to learn from the
neighbourhood model's top-k lists, and to be served with the same selectors.

    embed_rows(table, indices, indptr, data)          rows of a CSR (user histories) times an embedding table; a plain lookup
                                                      when ``indptr`` is left out.  Differentiable in ``table``.
    embed_rows_grad(grad, indices, n_vocab, ...)      its gradient, by sorted ids (equal calls give equal bits)
    adjust_scores(scores, ...)                        penalties for repeated ids, biases and masks on dense scores: ``targets``,
                                                      ``filter_cols`` and ``target_cols`` as in the similarity functions
    distill_loss(student, cols, values, counts)       divergence of dense scores from top-k lists in the layout DeviceProblem.run
                                                      writes.  Differentiable in ``student``.
    distill_grad(student, stats, cols, values, ...)   its gradient from the row statistics the forward pass left
    distill_loss_grad(student, cols, values, ...)     loss and gradient in one call

The compute is hand-written HIP behind include/sp_dense.h; torch is the tensors, the streams and the autograd graph.  Calls are
asynchronous on torch's current stream of the tensors' device; outputs and workspaces come from torch's allocator, so a call may
be captured into a graph.  Dense tensors are float32, bfloat16 or float16 with contiguous rows (any distance between rows);
everything is summed in float32 or wider and rounded once.  There is no CPU fallback.  A call that needs more threads than a launch has
(2^32) is refused: 2^23 rows of distillation, 2^24 rows of scores by segments of 16 384 columns, 2^26 embedding rows by slabs of 1 KB (include/
sp_dense.h has the numbers).  An output that is given may share memory with no operand but where its function says so (columns beside
an input's in one store are not shared); it counts as changed in place for autograd.

Autograd and graph capture: inside a capture the functions that build an autograd graph refuse inputs that require a gradient
(the backward pass of a captured graph would meet leaves whose gradients belong to another stream): capture the explicit
``embed_rows_grad``, ``distill_grad`` or ``distill_loss_grad`` instead.  Operands with a forward-mode tangent are refused, and so
are calls inside ``torch.jit.trace``, ``make_fx`` and ``torch.export``; ``torch.compile`` runs them between its graphs.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _abi

__all__ = ["embed_rows", "embed_rows_grad", "adjust_scores", "distill_loss", "distill_grad", "distill_loss_grad"]

_Pattern = Optional[Tuple[torch.Tensor, torch.Tensor]]
_PerRow = Union[float, torch.Tensor]

_DT = {torch.float32: _abi.SP_DT_F32, torch.bfloat16: _abi.SP_DT_BF16, torch.float16: _abi.SP_DT_F16}
_INT = (torch.int32, torch.int64)
_EMBED_SIZE, _ADJUST_SIZE, _DISTILL_SIZE = (C.sizeof(s) for s in (_abi.SpEmbedArgs, _abi.SpAdjustArgs, _abi.SpDistillArgs))


# ---- argument checks ---------------------------------------------------------------------------------------------------------

# (the checks of one operand are one condition on the way through: a small call's time is mostly this file's)

def _dense(name: str, t, ndim: int = 2):
    """A dense operand: a supported type on a HIP device, rows contiguous."""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _DT and t.dim() == ndim and (ndim == 1 or t.stride(1) == 1 or t.shape[1] <= 1):
        return t
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in _DT:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimension(s), got shape {tuple(t.shape)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a HIP device (similaripy_amd has no CPU fallback), got {t.device}")
    raise ValueError(f"{name} must have contiguous rows (stride 1 in its last dimension), got strides {t.stride()}")


def _same_device(name: str, t, device) -> None:
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other operands are on {device}")


def _ints(name: str, t, device, dtypes=_INT):
    """An index operand, contiguous."""
    if isinstance(t, torch.Tensor) and t.dtype in dtypes and t.device == device:
        return t if t.is_contiguous() else t.contiguous()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, got {t.dtype}")
    raise ValueError(f"{name} is on {t.device}, the other operands are on {device}")


def _floats(name: str, t, device, numel: int, dtype=torch.float32):
    if isinstance(t, torch.Tensor) and t.dtype == dtype and t.numel() == numel and t.device == device and not t.requires_grad:
        return t if t.is_contiguous() else t.contiguous()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {str(dtype).replace('torch.', '')}, got {t.dtype}")
    if t.numel() != numel:
        raise ValueError(f"{name} must have {numel} elements, got shape {tuple(t.shape)}")
    _same_device(name, t, device)
    if torch.is_grad_enabled():
        raise ValueError(f"{name} has no gradient here: detach it")
    return t.contiguous()


def _ld(t) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _out(name: str, out, shape, dtype, device, operands, in_place=None):
    """The caller's output, or a new one.  It may be `in_place` (same start, same rows), and shares memory with no other operand: the kernels
    read lists, weights and statistics while they write."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _dense(name, out)
    _same_device(name, out, device)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)}, got {out.dtype} of shape {tuple(out.shape)}")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} must not require a gradient")
    if shape[0] > 1 and out.stride(0) < shape[1]:
        raise ValueError(f"the rows of {name} overlap")
    if not out.numel():
        return out
    if in_place is not None and not (in_place.data_ptr() == out.data_ptr() and (shape[0] <= 1 or in_place.stride(0) == out.stride(0))):
        operands = (in_place, *operands)
    for t in operands:
        if t is not None and t.numel() and _overlap(out, t):
            raise ValueError(f"{name} shares memory with an input")
    return out


def _overlap(out, t) -> bool:
    """Whether rows of `out` and of `t` share memory: columns of one store that lie beside each other do not.  (With different distances
    between rows only what is apart altogether counts as apart.)"""
    a0, a1 = _extent(out)
    b0, b1 = _extent(t)
    if a1 <= b0 or b1 <= a0:
        return False
    a, b = _row_bytes(out), _row_bytes(t)
    steps = {x.stride(0) * x.element_size() for x in (out, t) if x.dim() == 2 and x.shape[0] > 1}
    if a is None or b is None or len(steps) != 1:
        return True
    step = steps.pop()
    at = (a0 - b0) % step if step else 0
    return at < b or at + a > step


def _row_bytes(t):
    """Bytes of one row of a matrix, or of all of a vector; None where they are not next to each other."""
    last = t.shape[-1] if t.dim() else 1
    return None if t.dim() > 2 or last > 1 and t.stride(-1) != 1 else last * t.element_size()


def _extent(t):
    first = t.data_ptr()
    return first, first + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _nothing(t) -> int:
    """The pointer of an operand that has none: an empty one.  A wrapper tensor has none either; 0 would say that the operand is not given."""
    if t.numel():
        raise TypeError(f"an operand has no memory of its own ({type(t).__name__}): pass the tensor that it wraps")
    return 0


# the caller's output has been written behind torch's back: its version goes up, so that a backward pass that has saved it raises
_written = torch.autograd.graph.increment_version


def _stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# torch's own way to a stream's handle costs as much as a launch; torch.compile's generated code uses this one
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    def _stream(device, _raw=torch._C._cuda_getCurrentRawStream) -> int:  # noqa: F811
        return _raw(device.index)


def _no_grad_here(name: str, t) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} builds no autograd graph: detach its inputs or call it under torch.no_grad()")


def _fixed(name: str, t) -> None:
    """An operand that gets no gradient, checked before an autograd graph is built (inside one, grad mode is off)."""
    if isinstance(t, torch.Tensor) and t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} has no gradient here: detach it")


def _number(name: str, v) -> float:
    if isinstance(v, torch.Tensor):
        _fixed(name, v)
    return float(v)


def _not_capturing(name: str, instead: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{name} on tensors that require a gradient cannot be captured into a graph: capture {instead} on detached tensors")


_is_tracing, _modes, _in_keys, _compiling = (torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._dispatch_tls_is_dispatch_key_included,
                                             torch.compiler.is_dynamo_compiling)
_PROXY, _PRE_DISPATCH = torch._C._TorchDispatchModeKey.PROXY, torch._C.DispatchKey.PreDispatch


def _plain(*operands) -> None:
    """Every entry begins with this.  The kernels read and write memory behind torch's back: a tangent would be dropped (a derivative of 0),
    and a recorded graph (torch.jit.trace, make_fx, torch.export) would hold the allocation of the output and nothing else.  torch.compile breaks
    its graph at these calls and needs no refusal."""
    if _is_tracing() or (_modes() and torch._C._get_dispatch_mode(_PROXY) is not None) or (not _compiling() and _in_keys(_PRE_DISPATCH)):
        raise RuntimeError("the dense operators cannot be traced: a recorded graph would not hold their kernels")
    if forward_ad._current_level >= 0:
        for t in operands:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("the dense operators have no forward-mode derivative: an operand has a tangent")


# ---- embedding rows ------------------------------------------------------------------------------------------------------------

def _rows(t):
    """All but the last dimension as one (reshape(-1, d) does not work for d = 0)."""
    return t if t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


def _csr_of(indices, indptr, data, device):
    """(indices, indptr, data, rows, output shape without the last dimension)."""
    indices = _ints("indices", indices, device)
    if indptr is None:
        if data is not None:
            raise ValueError("data needs indptr: a lookup has no weights")
        return indices, None, None, indices.numel(), tuple(indices.shape)
    if indices.dim() != 1:
        raise ValueError(f"indices must have 1 dimension with indptr, got shape {tuple(indices.shape)}")
    indptr = _ints("indptr", indptr, device, (indices.dtype,))
    if indptr.dim() != 1 or indptr.numel() < 1:
        raise ValueError(f"indptr must have 1 dimension and at least one element, got shape {tuple(indptr.shape)}")
    if data is not None:
        data = _floats("data", data, device, indices.numel())
    return indices, indptr, data, indptr.numel() - 1, (indptr.numel() - 1,)


def _embed_args(src, out, indices, indptr, data, n_rows, n_vocab, dim, scale, accumulate=0):
    dev = src.device
    return _abi.SpEmbedArgs(_EMBED_SIZE, 0, dev.index, _DT[src.dtype], _DT[out.dtype], 1 if indices.dtype == torch.int64 else 0, accumulate, scale,
                            n_rows, n_vocab, dim, indices.numel(), _ld(src), _ld(out), src.data_ptr(), indices.data_ptr(),
                            None if indptr is None else indptr.data_ptr() or _nothing(indptr), None if data is None else data.data_ptr() or _nothing(data), out.data_ptr(), _stream(dev))


def _embed_forward(table, indices, indptr, data, scale, out):
    indices, indptr, data, n_rows, lead = _csr_of(indices, indptr, data, table.device)
    dim = table.shape[1]
    if out is not None and not isinstance(out, torch.Tensor):
        raise TypeError(f"out must be a torch.Tensor, got {type(out).__name__}")
    if out is not None and tuple(out.shape) != lead + (dim,):
        raise ValueError(f"out must have shape {lead + (dim,)}, got {tuple(out.shape)}")
    flat = None if out is None else out.view(n_rows, dim) if out.dim() != 2 else out
    res = _out("out", flat, (n_rows, dim), table.dtype, table.device, (table, indices, indptr, data))
    _abi.call_dense("sp_embed_rows", _embed_args(table, res, indices, indptr, data, n_rows, table.shape[0], dim, scale))
    if out is not None:
        _written(out)
        return out
    return res if len(lead) == 1 else res.view(lead + (dim,))


class _EmbedRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, indices, indptr, data, scale):
        ctx.save_for_backward(indices, indptr, data)
        ctx.scale, ctx.n_vocab = scale, table.shape[0]
        return _embed_forward(table, indices, indptr, data, scale, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        _not_capturing("embed_rows' backward pass", "embed_rows_grad")
        indices, indptr, data = ctx.saved_tensors
        grad = _rows(grad)
        if grad.shape[1] > 1 and grad.stride(1) != 1:
            grad = grad.contiguous()
        return embed_rows_grad(grad, indices, ctx.n_vocab, indptr, data, scale=ctx.scale), None, None, None, None


def embed_rows(table: torch.Tensor, indices: torch.Tensor, indptr: Optional[torch.Tensor] = None, data: Optional[torch.Tensor] = None, *,
               scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of a CSR times an embedding table, scaled.

    ``out[i] = scale * sum(data[j] * table[indices[j]] for j in indptr[i] .. indptr[i + 1])`` — with ``indptr`` left out a plain
    lookup, ``out[...] = scale * table[indices[...]]`` for indices of any shape.

    table     [n_vocab, dim] float32 / bfloat16 / float16
    indices   int32 or int64; an id outside ``[0, n_vocab)`` contributes nothing (a padding id gives a row of zeros)
    indptr    [n_rows + 1] of the same type as ``indices``; rows may be empty
    data      [nnz] float32 weights (the CSR's data), default ones
    out       optional output (no autograd graph is built then)
    """
    _plain(table, data, scale, out)
    _dense("table", table)
    if type(scale) is not float:
        scale = _number("scale", scale)
    if data is not None:
        _fixed("data", data)
    if out is None and table.requires_grad and torch.is_grad_enabled():
        _not_capturing("embed_rows", "embed_rows and embed_rows_grad")
        return _EmbedRows.apply(table, indices, indptr, data, scale)
    if out is not None:
        _no_grad_here("embed_rows with out", table)
    return _embed_forward(table, indices, indptr, data, scale, out)


def embed_rows_grad(grad: torch.Tensor, indices: torch.Tensor, n_vocab: int, indptr: Optional[torch.Tensor] = None,
                    data: Optional[torch.Tensor] = None, *, scale: float = 1.0, dtype: Optional[torch.dtype] = None,
                    out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """Gradient of the table of :func:`embed_rows`: ``out[v] = scale * sum(data[j] * grad[row of j] for indices[j] == v)``.

    The entries are sorted by id and summed in float32, in ascending order within a chunk of the sorted entries and then chunk by chunk: no
    atomics, equal calls give equal bits.

    grad        [n_rows, dim] gradient of the rows (a lookup's with its leading dimensions flattened or not)
    n_vocab     rows of the table
    dtype       of the result: ``grad.dtype`` (default) or float32
    out         optional [n_vocab, dim] output
    accumulate  add to ``out``; rows of ids that do not occur are neither read nor written
    """
    _plain(grad, data, scale, out)
    if not isinstance(grad, torch.Tensor):
        raise TypeError(f"grad must be a torch.Tensor, got {type(grad).__name__}")
    if indptr is None and grad.dim() != 2 and grad.dim() > 0:
        grad = _rows(grad)
    _dense("grad", grad)
    _no_grad_here("embed_rows_grad", grad)
    indices, indptr, data, n_rows, _ = _csr_of(indices, indptr, data, grad.device)
    n_vocab, dim = int(n_vocab), grad.shape[1]
    if n_vocab < 0:
        raise ValueError(f"n_vocab must not be negative, got {n_vocab}")
    if grad.shape[0] != n_rows:
        raise ValueError(f"grad has {grad.shape[0]} rows, the indices make {n_rows}")
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    dtype = dtype or (grad.dtype if out is None else out.dtype)
    if dtype not in (grad.dtype, torch.float32):
        raise ValueError(f"the result must be {grad.dtype} or float32, got {dtype}")
    res = _out("out", out, (n_vocab, dim), dtype, grad.device, (grad, indices, indptr, data))
    a = _embed_args(grad, res, indices, indptr, data, n_rows, n_vocab, dim, _number("scale", scale), 1 if accumulate else 0)
    need = _abi.call_dense("sp_embed_rows_grad_workspace_bytes", a)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=grad.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _abi.call_dense("sp_embed_rows_grad", a)
    if out is not None:
        _written(out)
    return res


# ---- score adjustment ------------------------------------------------------------------------------------------------------------

_NO_PATTERN = _abi.SpCsrPattern()


def _pattern(name: str, csr, device, keep):
    if csr is None:
        return _NO_PATTERN
    if not isinstance(csr, (tuple, list)) or len(csr) != 2:
        raise TypeError(f"{name} must be a pair (indptr, indices)")
    indptr, indices = csr
    indices = _ints(name, indices, device)
    indptr = _ints(name, indptr, device, (indices.dtype,))
    if indptr.dim() != 1 or indptr.numel() < 1 or indices.dim() != 1:
        raise ValueError(f"{name}: indptr and indices must have 1 dimension, indptr at least one element")
    keep += (indptr, indices)
    return _abi.SpCsrPattern(indptr.data_ptr() or _nothing(indptr), indices.data_ptr(), indptr.numel() - 1, indices.numel(), 1 if indices.dtype == torch.int64 else 0)


def _per_row(name: str, v, device, n, keep):
    """(pointer, value for all rows) of a number or one float32 per row.  A tensor of no dimensions on a device is not read here, which would wait
    for the device: the rows share it."""
    if not isinstance(v, torch.Tensor):
        return None, float(v)
    if v.dim() == 0:
        _fixed(name, v)
        if not v.is_cuda:
            return None, float(v)
        v = v.to(device, torch.float32).expand(n)
    v = _floats(name, v, device, n)
    keep.append(v)
    return v.data_ptr() or _nothing(v), 0.0


def adjust_scores(scores: torch.Tensor, *, targets: Optional[torch.Tensor] = None, history: _Pattern = None, repetition: _PerRow = 1.0,
                  presence: _PerRow = 0.0, frequency: _PerRow = 0.0, bias: Optional[torch.Tensor] = None, allowed: Optional[torch.Tensor] = None,
                  filter_cols: _Pattern = None, target_cols: _Pattern = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties for repeated ids, biases and masks on rows of dense scores, in one pass over them.

    A column listed ``c > 0`` times in the row's history: ``y = (s > 0 ? s / repetition : s * repetition) - presence - frequency * c``;
    then ``y += bias``; then ``-inf`` where a mask says so (whatever the score was, NaN included).  A row whose masks leave nothing
    is all ``-inf``.

    scores       [n, n_cols] float32 / bfloat16 / float16
    targets      [n] int32 / int64: the row of ``history``, ``filter_cols`` and ``target_cols`` each row of scores belongs to (absolute
                 row ids, as ``target_rows`` of the similarity functions); default ``0 .. n-1``.  A row outside a pattern is empty there.
    history      (indptr, indices) of a CSR pattern: ids in any order, repeats count, ids outside the columns are passed over
    repetition, presence, frequency   a number (or a tensor of no dimensions), or one float32 per row (repetition positive; tensors on a device are not
                 checked)
    bias         [n_cols] or [n, n_cols], any of the three types
    allowed      int32 words of packed bits, [words] or [n, words] with ``words = ceil(n_cols / 32)``: column c stays where bit ``c % 32``
                 of word ``c // 32`` is set
    filter_cols  (indptr, indices): listed columns become ``-inf`` (the items a user has seen)
    target_cols  (indptr, indices): columns that are not listed become ``-inf``
    out          optional output; may be ``scores`` itself
    """
    _plain(scores, repetition, presence, frequency, bias, out)
    _dense("scores", scores)
    if scores.requires_grad:
        _no_grad_here("adjust_scores", scores)
    n, n_cols = scores.shape
    device = scores.device
    keep = []
    tptr, t64 = None, 0
    if targets is not None:
        targets = _ints("targets", targets, device)
        if targets.dim() != 1 or targets.numel() != n:
            raise ValueError(f"targets must have {n} elements, got shape {tuple(targets.shape)}")
        keep.append(targets)
        tptr, t64 = targets.data_ptr() or _nothing(targets), 1 if targets.dtype == torch.int64 else 0
    h = _pattern("history", history, device, keep)
    f = _pattern("filter_cols", filter_cols, device, keep)
    t = _pattern("target_cols", target_cols, device, keep)
    rep, rep_all = _per_row("repetition", repetition, device, n, keep)
    if rep is None and not rep_all >= 2.0 ** -149:      # (float32's smallest: what is below becomes 0)
        raise ValueError(f"repetition must be positive, got {repetition}")
    pres, pres_all = _per_row("presence", presence, device, n, keep)
    freq, freq_all = _per_row("frequency", frequency, device, n, keep)
    bptr, bdt, ldb = None, 0, 0
    if bias is not None:
        _dense("bias", bias, 2 if isinstance(bias, torch.Tensor) and bias.dim() == 2 else 1)
        if bias.device != device or bias.requires_grad:
            _same_device("bias", bias, device)
            _no_grad_here("adjust_scores", bias)
        if tuple(bias.shape) not in ((n_cols,), (n, n_cols)):
            raise ValueError(f"bias must have shape {(n_cols,)} or {(n, n_cols)}, got {tuple(bias.shape)}")
        if bias.dim() == 1 and not bias.is_contiguous():
            bias = bias.contiguous()
        keep.append(bias)
        bptr, bdt, ldb = bias.data_ptr() or _nothing(bias), _DT[bias.dtype], 0 if bias.dim() == 1 else bias.stride(0)
    aptr, lda = None, 0
    if allowed is not None:
        words = (n_cols + 31) // 32
        allowed = _ints("allowed", allowed, device, (torch.int32,))
        if tuple(allowed.shape) not in ((words,), (n, words)):
            raise ValueError(f"allowed must have shape {(words,)} or {(n, words)}, got {tuple(allowed.shape)}")
        keep.append(allowed)
        aptr, lda = allowed.data_ptr() or _nothing(allowed), 0 if allowed.dim() == 1 else words
    res = _out("out", out, (n, n_cols), scores.dtype, device, keep, scores)
    a = _abi.SpAdjustArgs(_ADJUST_SIZE, 0, device.index, _DT[scores.dtype], n, n_cols, _ld(scores), _ld(res), scores.data_ptr(), res.data_ptr(), tptr, t64, bdt,
                          h, f, t, rep, pres, freq, rep_all, pres_all, freq_all, 0, bptr, ldb, aptr, lda, _stream(device))
    _abi.call_dense("sp_adjust_scores", a)
    if out is not None:
        _written(out)
    return res


# ---- distillation ------------------------------------------------------------------------------------------------------------------

def _distill_args(student, cols, values, counts, temperature, teacher_lse):
    """The arguments every distillation call shares, and the tensors they point to."""
    _dense("student", student)
    n, n_cols = student.shape
    device = student.device
    cols = _ints("cols", cols, device)
    if cols.numel() % max(1, n) or (n == 0 and cols.numel()):
        raise ValueError(f"cols must hold the same number of slots for each of the {n} rows, got shape {tuple(cols.shape)}")
    k = cols.numel() // n if n else 0
    if n and cols.dim() != 1 and cols.shape != (n, k):
        raise ValueError(f"cols must have shape ({n}, k) or ({n} * k,), got {tuple(cols.shape)}")
    if k > _abi.SP_DISTILL_KMAX:
        raise ValueError(f"lists of {k} slots: at most {_abi.SP_DISTILL_KMAX} are supported")
    if not isinstance(values, torch.Tensor):
        raise TypeError(f"values must be a torch.Tensor, got {type(values).__name__}")
    if values.dtype not in _DT:
        raise TypeError(f"values must be float32, bfloat16 or float16, got {values.dtype}")
    if values.dim() != 1 and n and values.shape != (n, k):
        raise ValueError(f"values must have shape ({n}, {k}) or ({n * k},), got {tuple(values.shape)}")
    values = _floats("values", values, device, cols.numel(), values.dtype)
    if counts is not None:
        counts = _ints("counts", counts, device, (torch.int32,))
        if counts.numel() != n:
            raise ValueError(f"counts must have {n} elements, got shape {tuple(counts.shape)}")
    if teacher_lse is not None:
        teacher_lse = _floats("teacher_lse", teacher_lse, device, n)
    temperature = _number("temperature", temperature)
    if not 1e-30 < temperature < 1e30:
        raise ValueError(f"temperature must be positive, got {temperature}")
    a = _abi.SpDistillArgs(_DISTILL_SIZE, 0, device.index, _DT[student.dtype], n, n_cols, _ld(student), 0, k, 1 if cols.dtype == torch.int64 else 0,
                           _DT[values.dtype], temperature, student.data_ptr(), cols.data_ptr(), values.data_ptr(),
                           None if counts is None else counts.data_ptr() or _nothing(counts),
                           None if teacher_lse is None else teacher_lse.data_ptr() or _nothing(teacher_lse))
    a.stream = _stream(device)
    return a, (cols, values, counts, teacher_lse)


def _workspace(a, device):
    need = _abi.call_dense("sp_distill_workspace_bytes", a)
    if not need:
        return None
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    return ws


def _distill_forward(student, cols, values, counts, temperature, teacher_lse, want_stats):
    a, keep = _distill_args(student, cols, values, counts, temperature, teacher_lse)
    n = student.shape[0]
    loss = torch.empty(n, dtype=torch.float32, device=student.device)
    stats = torch.empty(n, 2, dtype=torch.float32, device=student.device) if want_stats else None
    a.loss, a.stats = loss.data_ptr(), None if stats is None else stats.data_ptr()
    ws = _workspace(a, student.device)
    _abi.call_dense("sp_distill_loss", a)
    del ws, keep
    return loss, stats


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, student, cols, values, counts, temperature, teacher_lse):
        loss, stats = _distill_forward(student, cols, values, counts, temperature, teacher_lse, True)
        ctx.save_for_backward(student, stats, cols, values, counts, teacher_lse)
        ctx.temperature = temperature
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss, _):
        _not_capturing("distill_loss' backward pass", "distill_grad or distill_loss_grad")
        student, stats, cols, values, counts, teacher_lse = ctx.saved_tensors
        grad = distill_grad(student.detach(), stats, cols, values, counts, grad_loss=grad_loss, temperature=ctx.temperature, teacher_lse=teacher_lse)
        return grad, None, None, None, None, None


def distill_loss(student: torch.Tensor, cols: torch.Tensor, values: torch.Tensor, counts: Optional[torch.Tensor] = None, *,
                 temperature: float = 1.0, teacher_lse: Optional[torch.Tensor] = None, return_stats: bool = False):
    """Divergence of a student's scores from a teacher's top-k lists, one float32 per row.

    With ``p`` the softmax of ``values / temperature`` over a row's list and ``q`` the softmax of ``student / temperature`` over all
    columns: ``loss = temperature**2 * sum(p * (log p - log q[cols]))``.  A row with an empty list has loss 0 (and gradient 0, whatever
    its scores hold); ``p = 0`` contributes 0; a listed column whose score is ``-inf`` makes the loss ``inf``.

    student      [n, n_cols] float32 / bfloat16 / float16
    cols, values [n, k] or flat [n * k]: the lists as DeviceProblem.run writes them (int32 or int64 ids; any of the three types); an id
                 outside the columns is not in the list; at most 4096 slots
    counts       [n] int32: valid slots of each list, default all
    teacher_lse  [n] float32: log-sum-exp of ALL the teacher's scores / temperature; ``p = exp(values / temperature - teacher_lse)`` then keeps
                 the mass that the teacher gives the list instead of being normalised over it
    return_stats also return [n, 2] float32, every row's maximum ``m`` and the sum of ``exp((student - m) / temperature)``, which
                 :func:`distill_grad` takes (their log-sum-exp ``m / temperature + log(sum)`` in two parts)
    """
    _plain(student, values, temperature, teacher_lse)
    _fixed("values", values)
    if isinstance(temperature, torch.Tensor):
        _fixed("temperature", temperature)
    if teacher_lse is not None:
        _fixed("teacher_lse", teacher_lse)
    if isinstance(student, torch.Tensor) and student.requires_grad and torch.is_grad_enabled():
        _not_capturing("distill_loss", "distill_loss and distill_grad, or distill_loss_grad,")
        loss, stats = _DistillLoss.apply(student, cols, values, counts, float(temperature), teacher_lse)
    else:
        loss, stats = _distill_forward(student, cols, values, counts, temperature, teacher_lse, return_stats)
    return (loss, stats) if return_stats else loss


def _grad_outputs(a, student, grad_loss, out, operands):
    n = student.shape[0]
    if grad_loss is not None:
        grad_loss = _floats("grad_loss", grad_loss, student.device, n)
    grad = _out("out", out, tuple(student.shape), student.dtype, student.device, (grad_loss, *operands), student)
    a.grad_loss, a.grad, a.ld_grad = None if grad_loss is None else grad_loss.data_ptr() or _nothing(grad_loss), grad.data_ptr(), _ld(grad)
    return grad, grad_loss


def distill_grad(student: torch.Tensor, stats: torch.Tensor, cols: torch.Tensor, values: torch.Tensor, counts: Optional[torch.Tensor] = None, *,
                 grad_loss: Optional[torch.Tensor] = None, temperature: float = 1.0, teacher_lse: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of :func:`distill_loss` in ``student``, from the row statistics it returned: ``grad_loss * temperature * (q * sum(p) - p)``.

    stats      [n, 2] float32, what ``distill_loss(..., return_stats=True)`` left
    grad_loss  [n] float32 gradient of every row's loss, default ones
    out        optional output; may be ``student`` itself
    """
    _plain(student, stats, values, grad_loss, temperature, teacher_lse, out)
    a, keep = _distill_args(student, cols, values, counts, temperature, teacher_lse)
    _no_grad_here("distill_grad", student)
    n = student.shape[0]
    stats = _floats("stats", stats, student.device, 2 * n)
    if stats.dim() != 1 and stats.shape != (n, 2):
        raise ValueError(f"stats must have shape ({n}, 2) or ({2 * n},), got {tuple(stats.shape)}")
    grad, g = _grad_outputs(a, student, grad_loss, out, (stats, *keep))
    a.stats = stats.data_ptr()
    _abi.call_dense("sp_distill_grad", a)
    if out is not None:
        _written(out)
    del keep, g
    return grad


def distill_loss_grad(student: torch.Tensor, cols: torch.Tensor, values: torch.Tensor, counts: Optional[torch.Tensor] = None, *,
                      grad_loss: Optional[torch.Tensor] = None, temperature: float = 1.0, teacher_lse: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Loss and gradient of :func:`distill_loss` in one call, for a training step that knows the gradient of the losses beforehand
    (``1 / n`` for their mean).  Arguments as in :func:`distill_grad`."""
    _plain(student, values, grad_loss, temperature, teacher_lse, out)
    a, keep = _distill_args(student, cols, values, counts, temperature, teacher_lse)
    _no_grad_here("distill_loss_grad", student)
    loss = torch.empty(student.shape[0], dtype=torch.float32, device=student.device)
    grad, g = _grad_outputs(a, student, grad_loss, out, keep)
    a.loss = loss.data_ptr()
    ws = _workspace(a, student.device)
    _abi.call_dense("sp_distill_loss_grad", a)
    if out is not None:
        _written(out)
    del ws, keep, g
    return loss, grad
