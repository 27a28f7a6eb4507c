"""``Muon``: momentum whose update is orthogonalised before it is applied, on the gfx950 matrix kernels.

For weights that are matrices.  Everything else in a model (embeddings and heads as one prefers, biases, norms) belongs to
``fairscale_amd.optim.Adam``; both take the same gradients, loss scales and scalers.  The constructor follows
``torch.optim.Muon``, the precision modes, ``step(scale=...)`` and ``fp32_param_groups`` follow ``Adam`` of this package.  The
reference has no counterpart.
"""
from __future__ import annotations

import ctypes
import math
from typing import Any, Callable, Dict, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from .. import _cabi
from ..matrix_ops import NS_COEFFICIENTS, TYPE_CODE, empty_workspace, fill_rows, orth_options, refuse_shared, rows_pointer, scale_arguments, workspace_size
from .adam import Precision

__all__ = ["Muon"]

_SETTINGS = ("lr", "weight_decay", "momentum", "nesterov", "ns_coefficients", "eps", "ns_steps", "adjust_lr_fn", "row_blocks")


class Muon(torch.optim.Optimizer):
    """Momentum orthogonalised by Newton-Schulz products. GPU-only.

    Per matrix, with ``r = grad / scale``: ``m <- m + (r - m) * (1 - momentum)``; ``u = r + (m - r) * momentum`` (``nesterov``) or
    ``m``; ``O = orthogonalize(u)``; ``p <- p * (1 - lr * weight_decay) - lr * ratio * O``.  One call covers a group; the
    update of the parameters happens inside the last product.

    Arguments:
        params: parameters of one dtype with at least two dimensions, or groups of them.  The last two dimensions
            are the matrix, leading ones count matrices (experts).  A convolution's weight is passed as a parameter of two
            dimensions over its memory, ``Parameter(w.detach().view(len(w), -1))``, that is given ``w.grad.view(len(w), -1)`` before a step.
        lr, weight_decay, momentum, nesterov, ns_coefficients, eps, ns_steps: as in the formulas above and in
            ``fairscale_amd.optim.orthogonalize``.
        adjust_lr_fn: ``ratio`` by the matrix's shape: None or ``"original"`` sqrt(max(1, rows / cols)),
            ``"match_rms_adamw"`` 0.2 * sqrt(max(rows, cols)).
        row_blocks: every matrix of the group is split into this many blocks of rows, each orthogonalised on its own (the
            query, key and value parts of one projection; heads).  ``ratio`` goes by the block.
        precision: FULL_PRECISION (fp32 parameters and gradients), MIXED_PRECISION (fp16 or bf16 parameters and gradients,
            fp32 master copies in ``fp32_param_groups``) or MEMORY_EFFICIENT_MIXED_PRECISION (fp16 or bf16, no master copies).
            The momentum is fp32 in all of them; PURE_FP16 is refused, since an average that takes in 5 % of a
            gradient a step loses most of it in 11 bits.  Inferred from the first parameter when None, as ``Adam`` does.
        products: ``"half"`` or ``"split"`` (see ``orthogonalize`` for what each is off by).  None: ``"split"`` where the parameters
            are updated in fp32, ``"half"`` where they are stored in 16 bits without masters: the update is then off by about 2e-3 of its
            norm, for gradients of few entries or aligned directions by up to 3e-2.
    """

    def __init__(
        self,
        params: Any,
        lr: float = 1e-3,
        weight_decay: float = 0.1,
        momentum: float = 0.95,
        nesterov: bool = True,
        ns_coefficients: Sequence[float] = NS_COEFFICIENTS,
        eps: float = 1e-7,
        ns_steps: int = 5,
        adjust_lr_fn: Optional[str] = None,
        row_blocks: int = 1,
        *,
        precision: Optional[Precision] = None,
        products: Optional[str] = None,
    ):
        if products not in (None, "half", "split"):
            raise ValueError(f"products must be None, 'half' or 'split', got {products!r}")
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                      ns_coefficients=tuple(ns_coefficients), eps=eps, ns_steps=ns_steps,
                                      adjust_lr_fn=adjust_lr_fn, row_blocks=row_blocks))
        first_dtype = self.param_groups[0]["params"][0].dtype
        if precision is None:
            precision = Precision.FULL_PRECISION if first_dtype == torch.float32 else Precision.MIXED_PRECISION
        if precision is Precision.PURE_FP16:
            raise ValueError("Muon keeps its momentum in fp32: PURE_FP16 is not supported (MEMORY_EFFICIENT_MIXED_PRECISION is)")
        allowed = (torch.float32,) if precision is Precision.FULL_PRECISION else (torch.float16, torch.bfloat16)
        if first_dtype not in allowed:
            raise ValueError(f"{precision.name} needs parameters of {' or '.join(str(d) for d in allowed)}, got {first_dtype}")
        self.precision = precision
        self.products = products or ("half" if precision is Precision.MEMORY_EFFICIENT_MIXED_PRECISION else "split")
        self._dtype = first_dtype
        for group in self.param_groups:
            self._check_group(group)
        self._make_masters(self.param_groups)

    @property
    def fp32_param_groups(self) -> List[Dict[str, Any]]:
        """The groups with their fp32 master copies in place of the parameters; empty without masters.  A view: the masters live in
        ``state[p]["master"]`` alone, which is what the step updates, ``state_dict`` saves and a resuming program assigns."""
        if not self.mixed_precision:
            return []
        return [{**group, "params": [self._master(p) for p in group["params"]]} for group in self.param_groups]

    @property
    def mixed_precision(self) -> bool:
        return self.precision is Precision.MIXED_PRECISION

    @property
    def supports_memory_efficient_fp16(self) -> bool:
        return True

    def __getstate__(self) -> Dict[str, Any]:  # of copies and pickles
        return {**super().__getstate__(), "precision": self.precision, "products": self.products, "_dtype": self._dtype}

    # ------------------------------------------------------------------ groups and state

    def _check_group(self, group: Dict[str, Any], gi: int = -1) -> None:
        """Raises ValueError for settings the step cannot take; before a step (of group ``gi``) only when they changed since the last."""
        settings = tuple(group[name] for name in _SETTINGS) + (self.products,)
        checked = self.__dict__.setdefault("_checked", {})
        step = gi >= 0
        if step and checked.get(gi) == settings:
            return
        if not 0.0 <= group["lr"] < math.inf:
            raise ValueError(f"Invalid learning rate: {group['lr']}")
        if not 0.0 <= group["weight_decay"] < math.inf:
            raise ValueError(f"Invalid weight_decay value: {group['weight_decay']}")
        if not 0.0 <= group["momentum"] < 1.0:
            raise ValueError(f"Invalid momentum value: {group['momentum']}")
        if group["adjust_lr_fn"] not in (None, "original", "match_rms_adamw"):
            raise ValueError(f"adjust_lr_fn must be None, 'original' or 'match_rms_adamw', got {group['adjust_lr_fn']!r}")
        if not 0.0 < group["eps"] < math.inf:
            raise ValueError(f"Invalid epsilon value: {group['eps']}")
        options = orth_options(group["ns_steps"], group["ns_coefficients"], group["eps"], self.products)
        size = ctypes.c_int64(0)
        if _cabi.lib().fsadam_muon_workspace(None, 0, ctypes.byref(options), ctypes.byref(size)) != 0:
            raise ValueError(_cabi.lib().fsadam_last_error().decode("utf-8", "replace"))
        blocks = group["row_blocks"]
        if int(blocks) != blocks or blocks < 1:
            raise ValueError(f"row_blocks must be a positive whole number, got {blocks}")
        for p in group["params"]:
            if p.dtype != self._dtype:
                raise ValueError(f"all parameters must share one dtype, got {self._dtype} and {p.dtype}")
            self._check_shape(p, blocks)
        if step:
            checked[gi] = settings

    @staticmethod
    def _check_shape(p: torch.Tensor, blocks: int) -> None:
        if p.dim() < 2:
            raise ValueError(f"Muon optimizes matrices, got a parameter of shape {tuple(p.shape)} (Adam takes it)")
        if p.shape[-2] % blocks:
            raise ValueError(f"{p.shape[-2]} rows cannot be split into {blocks} blocks")

    def _master(self, p: torch.Tensor) -> torch.Tensor:
        """The fp32 master copy of a parameter; made from the parameter where its state has none (a state of another precision)."""
        state = self.state[p]
        master = state.get("master")
        if master is None:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a graph that makes a master copy would make it again at every replay: step once before the capture")
            master = state["master"] = p.detach().to(torch.float32, memory_format=torch.contiguous_format, copy=True)
        return master

    def _make_masters(self, groups: Sequence[Dict[str, Any]]) -> None:
        if self.mixed_precision:
            for group in groups:
                for p in group["params"]:
                    self._master(p)

    def add_param_group(self, param_group: Dict[str, Any]) -> None:
        super().add_param_group(param_group)
        if "precision" in self.__dict__:  # not during construction, which checks all groups at its end
            group = self.param_groups[-1]
            try:
                self._check_group(group)
            except Exception:
                self.param_groups.pop()
                raise
            self._make_masters([group])

    def load_state_dict(self, state_dict: Dict[str, Any]) -> None:
        """Restores momentum and master copies bit for bit (torch alone casts them to the parameters' dtype).

        Settings that a checkpoint does not hold (``row_blocks`` in one of ``torch.optim.Muon``) stay as they are.  All of it is
        checked before anything is replaced: a checkpoint that is refused leaves the optimizer as it was.
        """
        saved_groups = state_dict["param_groups"]
        if [len(g["params"]) for g in saved_groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the checkpoint's parameter groups are not those of the optimizer")
        saved_groups = [{**{name: group[name] for name in _SETTINGS}, **saved} for group, saved in zip(self.param_groups, saved_groups)]
        restored = []  # (parameter, key, tensor)
        for group, saved in zip(self.param_groups, saved_groups):
            self._check_group({**saved, "params": group["params"]})
            for p, pid in zip(group["params"], saved["params"]):
                state = state_dict["state"].get(pid, {})
                for key in ("momentum_buffer", "master") if self.mixed_precision else ("momentum_buffer",):
                    if key in state:
                        restored.append((p, key, state[key].detach().to(device=p.device, dtype=torch.float32, copy=True).contiguous()))
        super().load_state_dict({**state_dict, "param_groups": saved_groups})
        for p, key, tensor in restored:
            self.state[p][key] = tensor
        if not self.mixed_precision:
            for state in self.state.values():
                state.pop("master", None)  # no step would keep it up to date
        self._make_masters(self.param_groups)

    # ------------------------------------------------------------------ the step

    def _gather(self, group: Dict[str, Any]) -> Dict[torch.device, Tuple[List[torch.Tensor], ...]]:
        """(parameters or masters, gradients, momenta, copies) of what takes part, by device.  Changes nothing but for momenta and masters that are made."""
        batches: Dict[torch.device, Tuple[List[torch.Tensor], ...]] = {}
        mixed = self.mixed_precision
        for p in group["params"]:
            grad = p.grad
            if grad is None:
                continue
            state = self.state[p]
            buf = state.get("momentum_buffer")
            if buf is None:
                self._check_row(p, p, grad, None)
                self._check_shape(p, int(group["row_blocks"]))
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("a graph that makes the momentum would clear it at every replay: step once before the capture")
                buf = state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            if not mixed:
                state.pop("master", None)  # assigned with a state of another precision: no step keeps it up to date
            lists = batches.get(p.device)
            if lists is None:
                lists = batches[p.device] = ([], [], [], [])
            lists[0].append(self._master(p) if mixed else p)
            lists[1].append(grad)
            lists[2].append(buf)
            lists[3].append(p)
        return batches

    def _check_row(self, p: torch.Tensor, like: torch.Tensor, grad: torch.Tensor, buf: Optional[torch.Tensor]) -> None:
        """What the kernels rely on, by name (the native walk checks the same of all rows in one loop)."""
        if grad.layout != torch.strided:
            raise RuntimeError("Muon does not support sparse gradients")
        if not like.is_cuda or not like.is_contiguous() or not grad.is_contiguous() or grad.device != like.device:
            raise RuntimeError("parameters and gradients must be dense, contiguous tensors on one device each")
        if grad.dtype != like.dtype or grad.shape != like.shape:
            raise RuntimeError("gradients must have their parameter's dtype and shape")
        if like.dtype != self._dtype:
            raise RuntimeError(f"a parameter has changed its dtype from {self._dtype} to {like.dtype}")
        for t in ((buf,) if p is like else (buf, p)):
            if t is not None and (t.dtype != torch.float32 or t.device != like.device or t.shape != like.shape or not t.is_contiguous()):
                raise RuntimeError("momentum and master copies must be contiguous float32 tensors with their parameter's shape and device")

    def _rows(self, gi: int, group: Dict[str, Any], device: torch.device, lists: Tuple[List[torch.Tensor], ...]) -> np.ndarray:
        """FsMuonTensor rows of one call."""
        params, grads, bufs, likes = lists
        blocks, how = int(group["row_blocks"]), group["adjust_lr_fn"]
        rows = np.empty((len(params), 8), dtype=np.int64)
        copies = likes if self.mixed_precision else None
        stored = torch.float32 if self.mixed_precision else self._dtype
        if device.type != "cuda" or not fill_rows((params, grads, bufs, copies), (stored, self._dtype, torch.float32, self._dtype), (0, 2, 3), device, rows):
            for p, like, grad, buf in zip(params, likes, grads, bufs):
                self._check_row(p, like, grad, buf)
            refuse_shared([*params, *bufs, *(copies or ())], grads)
            rows[:, :4] = [(p.data_ptr(), g.data_ptr(), m.data_ptr(), c.data_ptr() if copies else 0) for p, g, m, c in zip(params, grads, bufs, likes)]
        # batch, rows, cols and ratio go by the shapes alone
        shapes = (blocks, how, tuple(p.shape for p in params))
        cached = self.__dict__.setdefault("_geometry", {}).get((gi, device))
        if cached is None or cached[0] != shapes:
            cells = np.empty((len(params), 4), dtype=np.int64)
            ratios = cells.view(np.float64)
            for k, p in enumerate(params):
                self._check_shape(p, blocks)
                height, cols = p.shape[-2] // blocks, p.shape[-1]
                cells[k, :3] = p.numel() // (height * cols) if p.numel() else 0, height, cols
                if how == "match_rms_adamw":
                    ratios[k, 3] = 0.2 * math.sqrt(max(height, cols))
                else:
                    ratios[k, 3] = math.sqrt(max(1.0, height / cols)) if cols else 1.0
            cached = self._geometry[gi, device] = (shapes, cells)
        rows[:, 4:] = cached[1]
        return rows

    def step(self, closure: Optional[Callable[[], float]] = None, *, scale: Union[float, torch.Tensor] = 1.0) -> Optional[float]:
        """One optimization step.

        Arguments:
            closure: re-evaluates the model and returns the loss.
            scale: gradients are divided by this inside the kernels, as in ``Adam.step``: a float, or a one-element float32
                tensor on the parameters' device (``clip_grad_norm_(..., fold="device")``).

        May be captured into a graph after one eager step; a replay then repeats the recorded lr, weight decay and (float) scale.
        """
        loss = closure() if closure is not None else None
        calls = []
        for gi, group in enumerate(self.param_groups):
            self._check_group(group, gi)
            for device, lists in self._gather(group).items():
                calls.append((group, device, self._rows(gi, group, device, lists), *scale_arguments(scale, device)))
        if torch.autograd._profiler_enabled():
            with torch.autograd.profiler.record_function("fairscale_amd::muon::fused_step"):
                self._launch(calls)
        else:
            self._launch(calls)
        return loss

    def _launch(self, calls: Sequence[Tuple[Dict[str, Any], torch.device, np.ndarray, float, Optional[int]]]) -> None:
        lib = _cabi.lib()
        code = TYPE_CODE[self._dtype]
        # Every call's list is checked, and there is memory for all of them, before the first one runs: a refused step changes nothing.
        # Calls of one device follow each other on its stream, so the largest workspace serves them all.
        options, workspaces = [], {}
        for group, device, rows, _, _ in calls:
            options.append(orth_options(group["ns_steps"], group["ns_coefficients"], group["eps"], self.products))
            size = workspace_size(lib.fsadam_muon_workspace, rows_pointer(rows, _cabi.FsMuonTensor), len(rows), ctypes.byref(options[-1]))
            workspaces[device] = max(size, workspaces.get(device, 0))
        for device, size in workspaces.items():
            workspaces[device] = empty_workspace(size, device), size
        for (group, device, rows, scale, scale_pointer), how in zip(calls, options):
            with torch.cuda.device(device):
                workspace, size = workspaces[device]
                _cabi.check(lib.fsadam_muon_step(
                    rows_pointer(rows, _cabi.FsMuonTensor), len(rows), _cabi.TYPE_F32 if self.mixed_precision else code, code,
                    code if self.mixed_precision else -1, ctypes.byref(how), float(group["lr"]), float(group["momentum"]), 1 if group["nesterov"] else 0,
                    float(group["weight_decay"]), scale, scale_pointer, workspace.data_ptr(), size, int(torch.cuda.current_stream(device).cuda_stream)))
