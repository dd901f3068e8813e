"""AdamW over all tensors of a model in one launch, moments in 32 bits or in 8.

The alpha / beta loops have their own fused Adam steps (`bf_alpha_adam_step`, `bf_shared_adam_step`: the reference's torch.optim.Adam over ReLU parameters,
runtime/alpha_beta_crown.py:747-923).  `AdamW` is the step for the network's own tensors between queries: what stays in full precision around frozen
4-bit layers, say.  A chain that has been compiled from these tensors follows them (`network.CudaChain`).
"""
from __future__ import annotations

import array
import itertools
import operator
from typing import Any, Dict, Iterable, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from .weights4 import _Entry

_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16, torch.float16: _lib.TYPE_F16}
_PAIRS = {(p, g) for p in _TYPES for g in _TYPES if p == g or p == torch.float32}
_SIZE = {torch.float32: 4, torch.bfloat16: 2, torch.float16: 2}
_GRAD, _SHAPE, _DTYPE, _BYTES = (operator.attrgetter(n) for n in ("grad", "shape", "dtype", "nbytes"))
_POINTER, _CONTIGUOUS, _INDEX = torch.Tensor.data_ptr, torch.Tensor.is_contiguous, torch.Tensor.get_device
_ADAMW_STEP, _ADAMW_MOMENTS = _Entry("bf_adamw_step"), _Entry("bf_adamw_moments")
_BLOCK = 256  # moments that share an exponent; a tensor's moments begin at a whole block
_ENTRY = np.dtype([("p", np.uint64), ("g", np.uint64), ("n", np.int64), ("first", np.int64), ("lr", np.float32), ("weight_decay", np.float32)])


class AdamW:
    """p = p (1 - lr weight_decay) - lr m^ / (sqrt(v^) + eps), m and v the running means of the gradient and its square, ^ their bias correction.

    `params`: tensors, or dicts {"params": [...], "lr": ..., "weight_decay": ...} whose options replace the defaults (lr and weight_decay are read again
    at every step, so that a schedule may change them in `param_groups`).  fp32, bf16 or fp16 tensors, contiguous, on one CUDA device.  Gradients have
    the tensor's type, or any of the three beside fp32 tensors.

    `state_bits=8` holds the moments in a byte each with an exponent for every 256 elements (1.004 bytes instead of 4): exponent and 3 mantissa bits,
    rounded up or down in proportion by a hash of element and step, so that two runs give the same bits; the step's root and quotient are good to 2^-22 then (with 32 bits rounded to the
    nearest).  A block whose gradients hold an infinity
    or a NaN is NaN from then on, as its parameters are.

    The step count is on the device: a step that was captured into a graph counts as it is replayed (with the gradients' memory and lr of
    its capture).  All tensors share it; one without a gradient is left as it is by that step."""

    def __init__(self, params: Iterable[Any], lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 *, state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits={state_bits!r}: 8 or 32")
        self.betas, self.eps = self._constants(betas, eps)
        given = [params] if torch.is_tensor(params) else list(params)
        groups = [dict(g) for g in given] if given and isinstance(given[0], dict) else [{"params": given}]
        self.param_groups: List[Dict[str, Any]] = []
        self._params: List[torch.Tensor] = []
        self._group_of: List[int] = []
        for i, g in enumerate(groups):
            tensors = [g["params"]] if torch.is_tensor(g["params"]) else list(g["params"])
            unknown = set(g) - {"params", "lr", "weight_decay"}
            if unknown:
                raise ValueError(f"AdamW: group {i} has options {sorted(unknown)}; lr and weight_decay can differ between groups")
            self.param_groups.append({"params": tensors, "lr": float(g.get("lr", lr)), "weight_decay": float(g.get("weight_decay", weight_decay))})
            self._params += tensors
            self._group_of += [i] * len(tensors)
        if not self._params:
            raise ValueError("AdamW: no parameters")
        for k, p in enumerate(self._params):
            if not torch.is_tensor(p) or p.dtype not in _TYPES:
                raise TypeError(f"AdamW: parameter {k} is no fp32, bf16 or fp16 tensor")
            if not p.is_cuda or p.device != self._params[0].device:
                raise RuntimeError(f"AdamW: parameter {k} is on {p.device}; all have to be on one CUDA device")
            if not p.is_contiguous():
                raise ValueError(f"AdamW: parameter {k} is not contiguous")
        self._refuse_overlap()
        self._options()
        self.state_bits, self.device = state_bits, self._params[0].device
        self._sizes, self._types = [p.numel() for p in self._params], [p.dtype for p in self._params]
        self._bytes, self._one_type = [n * _SIZE[t] for n, t in zip(self._sizes, self._types)], len(set(self._types)) == 1
        self._inference = any(p.is_inference() for p in self._params)
        self._first = np.concatenate([[0], np.cumsum([-(-n // _BLOCK) * _BLOCK for n in self._sizes])]).astype(np.int64)
        total = max(_BLOCK, int(self._first[-1]))
        kind = torch.float32 if state_bits == 32 else torch.uint8
        self.exp_avg, self.exp_avg_sq = (torch.zeros(total, dtype=kind, device=self.device) for _ in range(2))
        self.exp_avg_exponent = self.exp_avg_sq_exponent = None
        if state_bits == 8:
            self.exp_avg_exponent, self.exp_avg_sq_exponent = (torch.zeros(total // _BLOCK, dtype=torch.uint8, device=self.device) for _ in range(2))
        self._state = torch.empty(4, dtype=torch.float64, device=self.device)
        self._set_step(0)
        self._table = np.zeros(len(self._params), dtype=_ENTRY)
        self._table["n"], self._table["first"] = self._sizes, self._first[:-1]

    # ---- checks -----------------------------------------------------------------
    @staticmethod
    def _constants(betas: Any, eps: Any) -> Tuple[Tuple[float, float], float]:
        b1, b2 = (float(b) for b in betas)
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0) or not float(eps) >= 0.0:
            raise ValueError(f"betas={betas!r}, eps={eps!r}: betas in [0, 1) and eps >= 0 are wanted")
        return (b1, b2), float(eps)

    def _check_moments(self, step: int, moments: Dict[str, torch.Tensor]) -> List[str]:
        names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_exponent", "exp_avg_sq_exponent"] if self.state_bits == 8 else [])
        if set(moments) != set(names) or int(step) < 0:
            raise ValueError(f"load_flat_moments: step >= 0 and {names} are wanted, got step={step} and {sorted(moments)}")
        for name in names:
            buf, t = getattr(self, name), moments[name]
            if t.shape != buf.shape or t.dtype != buf.dtype:
                raise ValueError(f"load_flat_moments: {name} is {tuple(t.shape)} {t.dtype}, {tuple(buf.shape)} {buf.dtype} is wanted")
        return names

    def _refuse_overlap(self) -> None:
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size(), k) for k, p in enumerate(self._params) if p.numel())
        for (_, end, a), (start, _, b) in zip(spans, spans[1:]):
            if start < end:
                raise ValueError(f"AdamW: parameters {a} and {b} share memory")

    def _options(self) -> Tuple[List[float], List[float]]:
        lr, decay = [], []
        for i, g in enumerate(self.param_groups):
            lr.append(float(g["lr"]))
            decay.append(float(g["weight_decay"]))
            if not lr[-1] >= 0.0 or not decay[-1] >= 0.0:
                raise ValueError(f"AdamW: group {i} has lr={lr[-1]} and weight_decay={decay[-1]}; both have to be >= 0")
        return lr, decay

    def _set_step(self, step: int) -> None:
        self._state.copy_(torch.tensor([1.0, 1.0, 0.0, 0.0] if step == 0 else [self.betas[0] ** step, self.betas[1] ** step, float(step), 0.0],
                                       dtype=torch.float64))

    # ---- the step -----------------------------------------------------------------
    def step(self, grads: Optional[Sequence[Optional[torch.Tensor]]] = None, *, grad_scale: Optional[torch.Tensor] = None) -> None:
        """One step with the tensors' `.grad`, or with `grads` (one for each tensor, in order; None leaves that one as it is).  `grad_scale`: a device
        tensor of one fp32 element that the gradients are multiplied by (a clip factor, one over a loss scale)."""
        params, device = self._params, self.device
        given = list(map(_GRAD, params)) if grads is None else list(grads)
        if len(given) != len(params):
            raise ValueError(f"AdamW.step: {len(given)} gradients for {len(params)} tensors")
        scale = None
        if grad_scale is not None:
            if not torch.is_tensor(grad_scale) or grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != device:
                raise ValueError(f"AdamW.step: grad_scale is one fp32 element on {device}")
            scale = grad_scale.data_ptr()
        lr, decay = self._options()
        live, moved, sizes, ptypes = range(len(params)), params, self._sizes, self._types
        if any(map(operator.is_, given, itertools.repeat(None))):
            live = [k for k, g in enumerate(given) if g is not None]
            if not live:
                return
            moved, given, sizes, ptypes = ([xs[k] for k in live] for xs in (params, given, sizes, ptypes))
        index = [device.index] * len(given)
        if list(map(_INDEX, moved)) != index:
            raise ValueError(f"AdamW.step: a tensor has left {device}")
        shapes = list(map(_SHAPE, moved)) if grads is not None else None  # (a tensor's .grad has its shape and type)
        if list(map(_INDEX, given)) != index or (shapes is not None and list(map(_SHAPE, given)) != shapes):
            k, g = next((k, g) for k, g in zip(live, given) if g.shape != params[k].shape or g.device != device)
            raise ValueError(f"AdamW.step: gradient {k} is {tuple(g.shape)} on {g.device}, not {tuple(params[k].shape)} on {device}")
        if not all(map(_CONTIGUOUS, given)):
            if any(g.layout is not torch.strided for g in given):
                raise ValueError("AdamW.step: gradients have to be strided tensors")
            given = [g.contiguous() for g in given]  # (copies live until the launch)
        gtypes = list(map(_DTYPE, given))
        one = self._one_type and gtypes.count(gtypes[0]) == len(gtypes)
        kinds = [(ptypes[0], gtypes[0])] if one else list(zip(ptypes, gtypes))
        for k, (pt, gt) in zip(live, kinds):
            if (pt, gt) not in _PAIRS:
                raise TypeError(f"AdamW.step: gradient {k} is {gt} for a tensor of {pt}")
        if moved is params:
            wanted = self._bytes
            given_bytes = wanted if one and ptypes[0] == gtypes[0] else [n * _SIZE[t] for n, t in zip(sizes, gtypes)]
        else:
            wanted, given_bytes = [n * _SIZE[t] for n, t in zip(sizes, ptypes)], [n * _SIZE[t] for n, t in zip(sizes, gtypes)]
        if list(map(_BYTES, moved)) != wanted or list(map(_BYTES, given)) != given_bytes or not all(map(_CONTIGUOUS, moved)):
            raise ValueError("AdamW.step: a tensor has changed its shape, type or strides")
        table = self._table if moved is params else self._table[live]
        table["p"], table["g"] = array.array("Q", map(_POINTER, moved)), array.array("Q", map(_POINTER, given))
        if len(lr) == 1:
            table["lr"], table["weight_decay"] = lr[0], decay[0]
        else:
            table["lr"], table["weight_decay"] = [lr[self._group_of[k]] for k in live], [decay[self._group_of[k]] for k in live]
        buckets = [(kinds[0], table)] if one else [(kind, np.ascontiguousarray(table[[i for i, other in enumerate(kinds) if other == kind]])) for kind in dict.fromkeys(kinds)]
        m8, v8 = (None, None) if self.state_bits == 32 else (self.exp_avg_exponent.data_ptr(), self.exp_avg_sq_exponent.data_ptr())
        for n, ((pt, gt), part) in enumerate(buckets):
            _ADAMW_STEP(device, part.ctypes.data, len(part), _TYPES[pt], _TYPES[gt], self.state_bits, self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), m8, v8,
                        self.betas[0], self.betas[1], self.eps, scale, self._state.data_ptr(), 1 if n + 1 == len(buckets) else 0)
        torch.autograd.graph.increment_version(moved if not self._inference else [p for p in moved if not p.is_inference()])

    def zero_grad(self, set_to_none: bool = True) -> None:
        for p in self._params:
            if p.grad is not None:
                if set_to_none:
                    p.grad = None
                else:
                    p.grad.detach_().zero_()

    # ---- state ------------------------------------------------------------------------
    @property
    def steps(self) -> int:
        """Steps taken (waits for the device)."""
        return int(self._state[2].item())

    def flat_moments(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """Both moments of all tensors, each tensor's at a whole multiple of 256 elements (`moment_offsets`): the buffers themselves, or for 8-bit states
        the values that they stand for, in bf16 (which holds them exactly)."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        m, v = (torch.empty(self.exp_avg.numel(), dtype=torch.bfloat16, device=self.device) for _ in range(2))
        _ADAMW_MOMENTS(self.device, self.exp_avg.data_ptr(), self.exp_avg_sq.data_ptr(), self.exp_avg_exponent.data_ptr(), self.exp_avg_sq_exponent.data_ptr(),
                       m.data_ptr(), v.data_ptr(), m.numel())
        return m, v

    @property
    def moment_offsets(self) -> List[int]:
        return [int(v) for v in self._first[:-1]]

    def load_flat_moments(self, step: int, **moments: torch.Tensor) -> None:
        """Sets the step count and the flat buffers (`exp_avg`, `exp_avg_sq` and, for 8-bit states, `exp_avg_exponent`, `exp_avg_sq_exponent`)."""
        names = self._check_moments(step, moments)
        for name in names:
            getattr(self, name).copy_(moments[name])
        self._set_step(int(step))

    def state_dict(self) -> Dict[str, Any]:
        names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_exponent", "exp_avg_sq_exponent"] if self.state_bits == 8 else [])
        return {"step": self.steps, "state_bits": self.state_bits, "sizes": list(self._sizes), "betas": self.betas, "eps": self.eps,
                "groups": [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups],
                "moments": {n: getattr(self, n).clone() for n in names}}

    def load_state_dict(self, state: Dict[str, Any]) -> None:
        if state["state_bits"] != self.state_bits or list(state["sizes"]) != self._sizes or len(state["groups"]) != len(self.param_groups):
            raise ValueError("AdamW.load_state_dict: the state is of other tensors, groups or state_bits")
        groups = [{"lr": float(g["lr"]), "weight_decay": float(g["weight_decay"])} for g in state["groups"]]
        if not all(v >= 0.0 for g in groups for v in g.values()):
            raise ValueError(f"AdamW.load_state_dict: groups {groups}; lr and weight_decay have to be >= 0")
        betas, eps = self._constants(state["betas"], state["eps"])
        self._check_moments(state["step"], state["moments"])
        self.betas, self.eps = betas, eps  # (from here on nothing is refused: a state that is leaves the optimiser as it was)
        self.load_flat_moments(state["step"], **state["moments"])
        for g, s in zip(self.param_groups, groups):
            g.update(s)
