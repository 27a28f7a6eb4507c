"""Operators on lists of matrices, for optimizers that treat a weight as one matrix: the momentum pass and the
orthogonalisation of updates.  Host side of ``fsadam_momentum_pass`` and ``fsadam_orthogonalize`` (include/fsadam.h);
``fairscale_amd.optim.Muon`` runs both and the parameter update in one call.

The reference has no such operator (its optimizers are elementwise).  Everything runs on torch's current stream, keeps
nothing between calls and does not wait for the GPU; scratch memory comes from torch's allocator, so a call may be
captured into a graph.
"""
from __future__ import annotations

import ctypes
from typing import List, NamedTuple, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _cabi, _rows

__all__ = ["MomentumStats", "momentum_pass", "orthogonalize"]

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # quintic of the usual Newton-Schulz iteration: slope 3.4 at 0, about 0.7..1.2 from 0.05 on

TYPE_CODE = {torch.float32: _cabi.TYPE_F32, torch.float16: _cabi.TYPE_F16, torch.bfloat16: _cabi.TYPE_BF16}
_PRODUCTS = {"half": _cabi.PRODUCTS_HALF, "split": _cabi.PRODUCTS_SPLIT}


class MomentumStats(NamedTuple):
    """Device-resident results of one momentum pass."""

    updates: List[torch.Tensor]  # one per gradient, of its shape
    norms: torch.Tensor          # float32[n]: L2 norm of each update as stored
    found_inf: torch.Tensor      # float32[1]: 1.0 when a stored update is +-inf/NaN (never cleared here)


def orth_options(steps: int, coefficients: Sequence[float], eps: float, products: str) -> _cabi.FsOrthOptions:
    if len(coefficients) != 3:
        raise ValueError(f"coefficients must be three numbers (a, b, c), got {coefficients}")
    if products not in _PRODUCTS:
        raise ValueError(f"products must be 'half' or 'split', got {products!r}")
    if not -2**31 <= steps < 2**31 or int(steps) != steps:  # the call's own range is 1 to 32; what does not fit its field would be cut
        raise ValueError(f"steps must be a whole number, got {steps}")
    a, b, c = (float(v) for v in coefficients)
    return _cabi.FsOrthOptions(a, b, c, float(eps), int(steps), _PRODUCTS[products])


def scale_arguments(scale: Union[float, torch.Tensor], device: torch.device) -> Tuple[float, Optional[int]]:
    """(value, device pointer) of a gradient scale given as a number or as a tensor that the kernel reads."""
    if not isinstance(scale, torch.Tensor):
        return float(scale), None
    if scale.dtype != torch.float32 or scale.numel() != 1 or scale.device != device:
        raise RuntimeError("a tensor scale must be float32 with one element on the gradients' device")
    return 1.0, scale.data_ptr()


def workspace_size(size_call, *arguments) -> int:
    size = ctypes.c_int64(0)
    _cabi.check(size_call(*arguments, ctypes.byref(size)))
    return int(size.value)


def empty_workspace(size: int, device: torch.device) -> torch.Tensor:
    return torch.empty(max(size, 256), dtype=torch.uint8, device=device)


def workspace_for(size_call, device: torch.device, *arguments) -> Tuple[torch.Tensor, int]:
    size = workspace_size(size_call, *arguments)
    return empty_workspace(size, device), size


def refuse_shared(written: Sequence[torch.Tensor], read: Sequence[torch.Tensor] = ()) -> None:
    """Raises when a tensor that is written shares memory with another one (all contiguous)."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), w) for ts, w in ((written, True), (read, False)) for t in ts if t.numel()]
    end = written_end = 0
    for start, stop, writes in sorted(spans):
        if start < (end if writes else written_end):
            raise RuntimeError("a tensor that is written shares memory with another one of the call (the same tensor twice, or overlapping views)")
        end = max(end, stop)
        written_end = max(written_end, stop) if writes else written_end


def fill_rows(lists: Sequence[Optional[List[torch.Tensor]]], dtypes: Sequence[torch.dtype], written: Tuple[int, ...], device: torch.device,
              rows: np.ndarray, with_numel: bool = False) -> bool:
    """The lists' pointers into ``rows``, with every check that can be made of them, in one C++ loop.  False when the helper is not
    built or found something to refuse: the Python checks of the caller then name it."""
    native = _rows.native
    return native is not None and native.fill_matrix_rows(tuple(lists), tuple(TYPE_CODE[d] for d in dtypes), written, device.index,
                                                          rows.ctypes.data, rows.shape[1], with_numel)[0] >= 0


def rows_pointer(rows: np.ndarray, row_type):
    return ctypes.cast(rows.ctypes.data, ctypes.POINTER(row_type))


def _check_momentum_lists(grads, momenta, updates, device, dtype, update_dtype) -> None:
    for g, m in zip(grads, momenta):
        if g.device != device or g.dtype != dtype or m.device != device:
            raise RuntimeError("gradients of one pass must share dtype, and device with their momenta")
        if g.layout != torch.strided or m.layout != torch.strided or not g.is_contiguous() or not m.is_contiguous():
            raise RuntimeError("gradients and momenta must be dense, contiguous device tensors")
        if m.dtype != torch.float32 or m.shape != g.shape:
            raise RuntimeError("momenta must be float32 tensors of the gradients' shapes")
    for g, u in zip(grads, updates):
        if u.dtype != update_dtype or u.device != device or u.shape != g.shape or u.layout != torch.strided or not u.is_contiguous():
            raise RuntimeError("updates must be dense, contiguous tensors of one dtype with the gradients' shapes and device")
    in_place = [u.data_ptr() == g.data_ptr() and u.element_size() == g.element_size() for g, u in zip(grads, updates)]
    refuse_shared([*momenta, *updates], [g for g, own in zip(grads, in_place) if not own])


@torch.no_grad()
def momentum_pass(grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor], momentum: float = 0.95, *, nesterov: bool = True,
                  scale: Union[float, torch.Tensor] = 1.0, updates: Optional[Sequence[torch.Tensor]] = None,
                  found_inf: Optional[torch.Tensor] = None) -> MomentumStats:
    """Moving average of a list of gradients and the update it gives, in one pass over them.

    Per element, in fp32: ``r = g / scale``; ``m <- m + (r - m) * (1 - momentum)``;
    ``u = r + (m - r) * momentum`` with ``nesterov``, else ``u = m``.

    Arguments:
        grads: tensors of one device and dtype (fp32, fp16 or bf16), dense and contiguous; any shapes.
        momenta: fp32 tensors of the same shapes, updated in place.
        scale: the gradients are divided by this: a float, or a one-element float32 tensor the kernel reads when it runs.
        updates: tensors to write the updates to, of one dtype (any of the three); each may be its own gradient, if
            their elements have one size, but share memory with nothing else.  Made in the gradients' dtype when None.
        found_inf: float32[1] device tensor to raise; a zeroed one is made when None.  The momenta have taken the values in by then: gradients
            that may not be finite go through ``grad_pass`` or a ``GradScaler`` first.
    """
    grads, momenta = list(grads), list(momenta)
    if len(grads) == 0:
        raise RuntimeError("momentum_pass needs at least one gradient")
    if len(momenta) != len(grads) or (updates is not None and len(updates) != len(grads)):
        raise RuntimeError("grads, momenta and updates must be lists of the same length")
    device, dtype = grads[0].device, grads[0].dtype
    if dtype not in TYPE_CODE:
        raise RuntimeError(f"gradients must be float32, float16 or bfloat16, got {dtype}")
    if device.type != "cuda":
        raise RuntimeError("gradients must be dense, contiguous device tensors")
    if updates is None:
        updates = [torch.empty_like(g, memory_format=torch.contiguous_format) for g in grads]
    updates = list(updates)
    update_dtype = updates[0].dtype
    if update_dtype not in TYPE_CODE:
        raise RuntimeError(f"updates must be float32, float16 or bfloat16, got {update_dtype}")
    rows = np.empty((len(grads), 4), dtype=np.int64)
    if not fill_rows((grads, momenta, updates), (dtype, torch.float32, update_dtype), (1, 2), device, rows, True):
        _check_momentum_lists(grads, momenta, updates, device, dtype, update_dtype)
        rows[:] = [(g.data_ptr(), m.data_ptr(), u.data_ptr(), g.numel()) for g, m, u in zip(grads, momenta, updates)]
    fresh = found_inf is None
    if fresh:
        found_inf = torch.empty(1, dtype=torch.float32, device=device)  # the call clears it
    elif found_inf.dtype != torch.float32 or found_inf.device != device or found_inf.numel() != 1:
        raise RuntimeError("found_inf must be a float32 tensor with one element on the gradients' device")
    value, pointer = scale_arguments(scale, device)
    lib = _cabi.lib()
    pointer_to_rows = rows_pointer(rows, _cabi.FsMomentumTensor)
    with torch.cuda.device(device):
        workspace, size = workspace_for(lib.fsadam_momentum_workspace, device, pointer_to_rows, len(grads))
        norms = torch.empty(len(grads), dtype=torch.float32, device=device)
        _cabi.check(lib.fsadam_momentum_pass(
            pointer_to_rows, len(grads), TYPE_CODE[dtype], TYPE_CODE[update_dtype], float(momentum), 1 if nesterov else 0, value, pointer,
            norms.data_ptr(), found_inf.data_ptr(), 1 if fresh else 0, workspace.data_ptr(), size, int(torch.cuda.current_stream(device).cuda_stream)))
    return MomentumStats(updates, norms, found_inf)


def _layout(t: torch.Tensor) -> Optional[Tuple[bool, int, int]]:
    """(turned, ld, stride) of a batch of matrices whose rows (turned: columns) have neighbouring elements; None if it is none."""
    sizes, strides = list(t.shape), list(t.stride())
    stride = 0
    if t.dim() > 2:
        stride = strides[-3]
        reach = None  # the leading dimensions have to step through the matrices evenly
        for n, st in zip(reversed(sizes[:-2]), reversed(strides[:-2])):
            if n == 1:
                continue
            if reach is None:
                stride = st
            elif st != reach:
                return None
            reach = st * n
    rows, cols = sizes[-2:]
    row_step, col_step = strides[-2:]
    if col_step == 1 or cols == 1:
        ld = row_step if rows > 1 else cols
        if ld >= cols:
            return False, ld, stride
    if row_step == 1 or rows == 1:
        ld = col_step if cols > 1 else rows
        if ld >= rows:
            return True, ld, stride
    return None


@torch.no_grad()
def orthogonalize(matrices: Sequence[torch.Tensor], *, steps: int = 5, coefficients: Sequence[float] = NS_COEFFICIENTS, eps: float = 1e-7,
                  products: Optional[str] = None, out: Optional[Sequence[torch.Tensor]] = None) -> List[torch.Tensor]:
    """Matrices with (nearly) the same singular vectors and all singular values brought near 1, by Newton-Schulz products.

    Each matrix ``U`` is divided by ``max(norm(U), eps)`` (Frobenius) and then taken ``steps`` times through
    ``X <- a X + (b X X^T + c (X X^T)^2) X``, ``(a, b, c) = coefficients``.  A matrix of zeros stays zeros; a matrix
    with an entry that is not finite gives NaN everywhere, without touching the others.  Not differentiable.

    Arguments:
        matrices: tensors of one device and dtype (fp32, fp16 or bf16) with at least two dimensions; leading dimensions
            count matrices (experts, heads: ``w.view(heads, -1, w.shape[-1])``).  Rows or columns must have neighbouring
            elements: slices of rows or columns and transposed matrices are taken as they are, others are refused.
        products: ``"split"`` multiplies 22 bits of the operands: errors like fp32 products, at three times the matrix work.
            ``"half"`` multiplies 11 bits.  With the default coefficients and steps its error is about 2e-3 of the result's norm, the
            size of bf16's own rounding, where the roundings average over many singular directions (Gaussian matrices 2e-3, some
            non-zero rows or equal rows up to 4e-3); it is up to 3e-2 for matrices of a few entries, diagonal ones and those of rank one
            with entries of one size.  22 bits are taken in its place where the short side is 128 or less and for coefficients and
            steps that would multiply the error (a first-order bound over 1/16: six of the default steps).
            None: ``"half"`` for bf16, ``"split"`` for fp16 and fp32.  Ask for ``"split"`` where bf16 matrices of few or aligned
            directions have to be exact to their rounding.
        out: tensors to write the results to (of the same shapes, dtype and order of strides).  Each may be its own matrix, but share
            memory with no other one of the call; side by side in the columns of one tensor is no sharing.
    """
    matrices = list(matrices)
    if out is not None and len(out) != len(matrices):
        raise RuntimeError("out must be as long as the list of matrices")
    if len(matrices) == 0:
        return []
    device, dtype = matrices[0].device, matrices[0].dtype
    if dtype not in TYPE_CODE:
        raise RuntimeError(f"matrices must be float32, float16 or bfloat16, got {dtype}")
    if device.type != "cuda":
        raise RuntimeError("matrices must be device tensors")
    options = orth_options(steps, coefficients, eps, products or ("half" if dtype == torch.bfloat16 else "split"))
    layouts = []
    for t in matrices:
        if t.device != device or t.dtype != dtype:
            raise RuntimeError("matrices of one call must share device and dtype")
        if t.layout != torch.strided or t.dim() < 2:
            raise RuntimeError("matrices must be dense tensors with at least two dimensions")
        layout = _layout(t) if t.numel() else (False, t.shape[-1], 0)
        if layout is None:
            raise RuntimeError(f"a matrix needs rows or columns of neighbouring elements, got strides {tuple(t.stride())} for {tuple(t.shape)}")
        layouts.append(layout)
    given = out is not None
    if not given:
        out = [torch.empty(t.shape[:-2] + (t.shape[-1], t.shape[-2]), dtype=dtype, device=device).transpose(-2, -1) if layout[0]
               else torch.empty(t.shape, dtype=dtype, device=device) for t, layout in zip(matrices, layouts)]
    out = list(out)
    rows = (_cabi.FsMatrix * len(matrices))()
    for row, t, o, (turned, ld, stride) in zip(rows, matrices, out, layouts):
        if o.dtype != dtype or o.device != device or o.shape != t.shape or o.layout != torch.strided:
            raise RuntimeError("out must hold dense tensors with the matrices' shapes, dtype and device")
        if t.numel() == 0:
            continue
        into = _layout(o)
        if into is not None and into[0] != turned:  # a single row or column can be read either way
            into = _layout_as(o, turned)
        if into is None:
            raise RuntimeError("out must have neighbouring elements along the same dimension as its matrix")
        m, n = t.shape[-2:]
        row.src, row.dst, row.batch = t.data_ptr(), o.data_ptr(), t.numel() // (m * n)
        row.rows, row.cols = (n, m) if turned else (m, n)
        row.src_ld, row.src_stride, row.dst_ld, row.dst_stride = ld, stride, into[1], into[2]
    if given:
        _refuse_overlap(rows, matrices[0].element_size())
    lib = _cabi.lib()
    with torch.cuda.device(device):
        workspace, size = workspace_for(lib.fsadam_orth_workspace, device, rows, len(matrices), ctypes.byref(options))
        _cabi.check(lib.fsadam_orthogonalize(rows, len(matrices), TYPE_CODE[dtype], ctypes.byref(options), workspace.data_ptr(), size,
                                             int(torch.cuda.current_stream(device).cuda_stream)))
    return out


def _refuse_overlap(rows, size: int) -> None:
    """Raises when a result may lie over another matrix or result of the call.  Tensors of interleaved rows (slices of columns of one
    tensor) are told apart by their columns where their rows are equally far apart; other interleavings are refused."""
    spans = []
    for k, r in enumerate(rows):
        if not r.batch:
            continue
        in_place = (r.src, r.src_ld) == (r.dst, r.dst_ld) and (r.batch == 1 or r.src_stride == r.dst_stride)
        for start, ld, stride, writes in ((r.dst, r.dst_ld, r.dst_stride, True),) + (() if in_place else ((r.src, r.src_ld, r.src_stride, False),)):
            step = ld if r.rows > 1 else stride if r.batch > 1 else 0  # from row to row; 0: a single one, -1: not even
            if r.rows > 1 and r.batch > 1 and stride % ld:
                step = -1
            spans.append((start, start + ((r.batch - 1) * stride + (r.rows - 1) * ld + r.cols) * size, writes, step, r.cols))
    spans.sort()
    live = []
    for span in spans:
        start, _, writes, step, cols = span
        live = [s for s in live if s[1] > start]
        for _start, _, _writes, _step, _cols in live:
            if not (writes or _writes):
                continue
            shift, rest = divmod(start - _start, size)
            apart = not rest and _step > 0 and step in (0, _step) and _cols <= shift % _step <= _step - cols
            if not apart:
                raise RuntimeError("out shares memory with another matrix of the call (only a matrix's own result may lie over it)")
        live.append(span)


def _layout_as(t: torch.Tensor, turned: bool) -> Optional[Tuple[bool, int, int]]:
    """``_layout`` of a tensor seen as the other orientation, where its strides allow that too."""
    other = _layout(t.transpose(-2, -1))
    return (turned, other[1], other[2]) if other is not None and not other[0] and turned else \
        (turned, other[1], other[2]) if other is not None and other[0] and not turned else None
