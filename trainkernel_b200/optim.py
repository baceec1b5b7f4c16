"""AdamW over all tensors of a parameter tree, with moments held in 32 or in 8 bits.

Functional in the way the compiled steps are: an `AdamW` is a set of numbers, `init` makes the state
for a list of parameters, and `update` commits one step into the parameters and the state in place,
one launch for all tensors of the same types.  `compile_training(fn, inputs, optimizer=AdamW(...))`
runs it behind a compiled step.  The reference's only update is SGD inside the step
(reference: benchmarks/train_loop.py:35-45).
"""
from __future__ import annotations

import bisect
import ctypes
from dataclasses import dataclass
from typing import Any, Sequence

import torch
from torch.utils._pytree import keystr, tree_flatten, tree_flatten_with_path

from . import operators
from .operators import AdamWOptions, AdamWTensor

BLOCK = 256                 # elements that share one scale when moments are held in 8 bits
_COUNTERS = 4096            # copies of the step counter (TK_ADAMW_COUNTERS)


class AdamWState:
    """Moments of every parameter and the number of steps taken.

    The moments of all tensors are flat buffers: tensor `i` has elements `offsets[i]` to
    `offsets[i] + sizes[i]` in its own memory order, and offsets are multiples of 256.  With 32 bits
    `exp_avg` and `exp_avg_sq` are FP32.  With 8 bits `exp_avg` and `exp_avg_root` (the square root of
    the second moment) are e4m3 numbers that stand for themselves times the FP32 scale of their block
    of 256, `exp_avg_scale` and `exp_avg_root_scale`.  `paths` names the tensors by their place in the tree that
    `init` was given (None for a plain list).
    """

    def __init__(self, sizes: Sequence[int], bits: int, device: torch.device, paths: Sequence[str] | None = None) -> None:
        self.sizes = tuple(sizes)
        self.paths = None if paths is None else tuple(paths)
        self.bits = bits
        self.device = device
        offsets, total = [], 0
        for size in self.sizes:
            offsets.append(total)
            total += -(-size // BLOCK) * BLOCK
        self.offsets = tuple(offsets)
        dtype = torch.float32 if bits == 32 else torch.float8_e4m3fn
        self.exp_avg = torch.zeros(total, dtype=dtype, device=device)
        second = torch.zeros(total, dtype=dtype, device=device)
        if bits == 32:
            self.exp_avg_sq = second
            scales = (None, None)
        else:
            self.exp_avg_root = second
            self.exp_avg_scale = torch.zeros(total // BLOCK, dtype=torch.float32, device=device)
            self.exp_avg_root_scale = torch.zeros(total // BLOCK, dtype=torch.float32, device=device)
            scales = (self.exp_avg_scale, self.exp_avg_root_scale)
        # every block of the kernel reads and advances a counter of its own, so none can see another's new value
        self._counters = torch.zeros(_COUNTERS, dtype=torch.int64, device=device)
        self._second = second
        self._struct = operators.AdamWState(self.exp_avg.data_ptr(), second.data_ptr(), *(None if s is None else s.data_ptr() for s in scales),
                                            self._counters.data_ptr())
        self._struct_at = ctypes.addressof(self._struct)
        self._tensors = self.tensors()

    @property
    def step(self) -> torch.Tensor:
        """Steps taken so far, an int64 scalar on the device (do not write to it: use `set_step`)."""
        return self._counters[0]

    def set_step(self, step: int) -> None:
        if isinstance(step, bool) or not isinstance(step, int) or step < 0:
            raise ValueError("trainkernel: step must be a non-negative integer")
        self._counters.fill_(step)

    def tensors(self) -> tuple[torch.Tensor, ...]:
        """Everything a checkpoint or a snapshot has to copy."""
        if self.bits == 32:
            return (self.exp_avg, self.exp_avg_sq, self._counters)
        return (self.exp_avg, self.exp_avg_root, self.exp_avg_scale, self.exp_avg_root_scale, self._counters)

    def state_dict(self) -> dict[str, Any]:
        """Copies of the moments with the sizes they belong to, for a checkpoint."""
        return {"sizes": self.sizes, "bits": self.bits, "paths": self.paths, "tensors": tuple(t.clone() for t in self.tensors())}

    def load_state_dict(self, saved: dict[str, Any]) -> None:
        """Take over what `state_dict` of a state of the same sizes and bits returned."""
        if tuple(saved["sizes"]) != self.sizes or saved["bits"] != self.bits:
            raise ValueError("trainkernel: AdamW: the saved state belongs to other tensors or another number of bits")
        _check_places("the saved state", _names(saved.get("paths")), "the state", self.paths)
        for mine, theirs in zip(self.tensors(), saved["tensors"]):
            mine.copy_(theirs)

    def moments(self, index: int) -> tuple[torch.Tensor, torch.Tensor]:
        """First and second moment of tensor `index` as flat FP32 tensors."""
        begin, size = self.offsets[index], self.sizes[index]
        if self.bits == 32:
            return self.exp_avg[begin:begin + size].clone(), self.exp_avg_sq[begin:begin + size].clone()
        blocks = slice(begin // BLOCK, begin // BLOCK + -(-size // BLOCK))
        padded = -(-size // BLOCK) * BLOCK
        values = []
        for codes, scale in ((self.exp_avg, self.exp_avg_scale), (self.exp_avg_root, self.exp_avg_root_scale)):
            values.append((codes[begin:begin + padded].float().view(-1, BLOCK) * scale[blocks, None]).view(-1)[:size])
        return values[0], values[1].square()


def _leaves(tree: Any, what: str) -> list[torch.Tensor]:
    leaves = list(tree) if isinstance(tree, (list, tuple)) and all(isinstance(x, torch.Tensor) for x in tree) else tree_flatten(tree)[0]
    if not leaves or not all(isinstance(leaf, torch.Tensor) for leaf in leaves):
        raise TypeError(f"trainkernel: {what} must contain tensors only and cannot be empty")
    return leaves


def _paths(tree: Any) -> tuple[str, ...] | None:
    """Where every tensor of a tree stands; None for a tensor, for a plain list or tuple of them and for containers registered
    without keys, which go by position alone."""
    if isinstance(tree, torch.Tensor) or isinstance(tree, (list, tuple)) and all(isinstance(x, torch.Tensor) for x in tree):
        return None
    try:
        return tuple(keystr(path) for path, _ in tree_flatten_with_path(tree)[0])
    except ValueError:
        return None


def _names(paths: Any) -> tuple[str, ...] | None:
    return None if paths is None else tuple(paths)


def _check_places(what: str, paths: tuple[str, ...] | None, other: str, expected: tuple[str, ...] | None) -> None:
    """Tensors are paired by position, and a dictionary has the order in which its keys were set: equal shapes would hide a mix-up."""
    if paths is not None and expected is not None and paths != expected:
        raise ValueError(f"trainkernel: AdamW: {what} must have the structure of {other}, dictionary keys in the same order")


def _dense(tensor: torch.Tensor) -> bool:
    """Whether the elements fill one run of memory, in any order of dimensions."""
    if tensor.is_contiguous():
        return True
    expected = 1
    for stride, size in sorted((s, n) for s, n in zip(tensor.stride(), tensor.shape) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


def _span(tensor: torch.Tensor) -> tuple[int, int]:
    """First byte of a dense tensor and the one behind its last."""
    begin = tensor.data_ptr()
    return begin, begin + tensor.numel() * tensor.element_size()


def _check_apart(leaves: Sequence[torch.Tensor], gradients: Sequence[torch.Tensor], values: dict[str, Any]) -> None:
    """Nothing the launch writes may be written twice or read by another block: every param has memory of its own.  A
    gradient may be its own param's memory, where each element is read before it is written."""
    spans = sorted((*_span(leaf), i) for i, leaf in enumerate(leaves) if leaf.numel())
    for (a, end, i), (b, _, j) in zip(spans, spans[1:]):
        if a == b:
            raise ValueError(f"trainkernel: AdamW: param {max(i, j)} is listed twice")
        if b < end:
            raise ValueError(f"trainkernel: AdamW: params {i} and {j} overlap in memory")

    def over(tensor: torch.Tensor) -> int | None:
        """The first param that a tensor overlaps."""
        begin, end = _span(tensor)
        at = bisect.bisect_left(spans, (begin,))
        if at and spans[at - 1][1] > begin:
            at -= 1
        return spans[at][2] if at < len(spans) and spans[at][0] < end and spans[at][1] > begin else None

    for i, grad in enumerate(gradients):
        where = over(grad) if grad.numel() else None
        if where is not None and not (where == i and grad.data_ptr() == leaves[i].data_ptr() and grad.dtype == leaves[i].dtype):
            raise ValueError(f"trainkernel: AdamW: grad {i} overlaps param {where} in memory")
    for name, value in values.items():
        if isinstance(value, torch.Tensor) and over(value) is not None:
            raise ValueError(f"trainkernel: AdamW: {name} overlaps a param in memory")


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.stride() == b.stride() or all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


@dataclass(frozen=True)
class AdamW:
    """Numbers of an AdamW update.

    `lr` is a number, or a tensor of one FP32 value on the device that every launch (and every replay of a
    captured one) reads anew.  `weight_decay` is decoupled, one number or one per tensor.  `state_bits` 8 holds
    both moments in 8 bits with a scale per 256 elements; they are rounded stochastically, by a hash of
    place, step and `seed`, so equal runs give equal results.  Parameters are FP32 (or FP16 / BF16, which
    are rounded to nearest: steps below half of their spacing are lost).
    """

    lr: float | torch.Tensor = 1e-3
    betas: tuple[float, float] = (0.9, 0.999)
    eps: float = 1e-8
    weight_decay: float | Sequence[float] = 1e-2
    state_bits: int = 32
    seed: int = 0

    def __post_init__(self) -> None:
        def number(x) -> bool:
            return isinstance(x, (int, float)) and not isinstance(x, bool)
        if isinstance(self.lr, torch.Tensor):
            if self.lr.dtype != torch.float32 or self.lr.numel() != 1 or self.lr.device.type != "cuda":
                raise ValueError("trainkernel: AdamW: a tensor lr must hold one float32 value on a CUDA device")
        elif not number(self.lr) or not 0 <= self.lr < float("inf"):
            raise ValueError("trainkernel: AdamW: lr must be a non-negative number")
        if len(self.betas) != 2 or not all(number(b) and 0 <= b < 1 for b in self.betas):
            raise ValueError("trainkernel: AdamW: betas must be two numbers in [0, 1)")
        if not number(self.eps) or not 1e-30 <= self.eps < float("inf"):
            raise ValueError("trainkernel: AdamW: eps must be a number of at least 1e-30")
        decays = (self.weight_decay,) if number(self.weight_decay) else self.weight_decay
        if isinstance(decays, str) or not all(number(w) and 0 <= w < float("inf") for w in decays):
            raise ValueError("trainkernel: AdamW: weight_decay must be a non-negative number, or one per tensor")
        if not number(self.weight_decay):
            object.__setattr__(self, "weight_decay", tuple(map(float, decays)))
        object.__setattr__(self, "betas", tuple(self.betas))
        if self.state_bits not in (8, 32):
            raise ValueError("trainkernel: AdamW: state_bits must be 8 or 32")
        if isinstance(self.seed, bool) or not isinstance(self.seed, int) or not 0 <= self.seed < 2 ** 32:
            raise ValueError("trainkernel: AdamW: seed must be an integer in [0, 2^32)")

    def _decays(self, count: int) -> Sequence[float]:
        if isinstance(self.weight_decay, (int, float)):
            return (float(self.weight_decay),) * count
        if len(self.weight_decay) != count:
            raise ValueError(f"trainkernel: AdamW: {len(self.weight_decay)} weight decays for {count} tensors")
        return tuple(map(float, self.weight_decay))

    def init(self, params: Any) -> AdamWState:
        """Zero moments for `params` (a pytree of tensors); allocates, so not inside a stream capture."""
        leaves = _leaves(params, "params")
        device = leaves[0].device
        operators.require_device(device)
        self._decays(len(leaves))
        for leaf in leaves:
            self._check_param(leaf, device)
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("trainkernel: AdamW: init inside a stream capture would clear the moments in every replay")
        return AdamWState([leaf.numel() for leaf in leaves], self.state_bits, device, _paths(params))

    @staticmethod
    def _check_param(leaf: torch.Tensor, device: torch.device) -> None:
        if leaf.dtype not in operators.DTYPES:
            raise ValueError("trainkernel: AdamW: params must be float32, float16 or bfloat16")
        if leaf.device != device:
            raise ValueError("trainkernel: AdamW: all tensors must use one device")
        if leaf.layout != torch.strided or not _dense(leaf):
            raise ValueError("trainkernel: AdamW: params must be dense in memory")
        if leaf.requires_grad and not leaf.is_leaf:
            raise ValueError("trainkernel: AdamW: params must be detached from autograd")

    def update(self, params: Any, grads: Any, state: AdamWState, *, grad_scale: torch.Tensor | None = None) -> None:
        """One step, in place, on the current stream.

        `params` and `grads` are trees of the structure that `init` was given, or plain lists in the order of its leaves.
        `grads` matches `params` in shape and memory order (FP32, FP16 or BF16).  No two params overlap in memory, and
        nothing else overlaps one, but a gradient its own param.  `grad_scale` (one FP32 value on the device, for clipping
        or for undoing a loss scale) multiplies the gradients; when it is not finite the step does not happen: parameters,
        moments and step count stay as they are.
        """
        if operators.fast is not None and state.bits == self.state_bits and operators.fast.adamw_update(
                params, grads, state.sizes, state.offsets, self.weight_decay, state._struct_at, state._tensors, self.state_bits, self.lr, self.betas,
                self.eps, self.seed, grad_scale) is not None:
            return
        leaves, gradients = _leaves(params, "params"), _leaves(grads, "grads")
        device = state.device
        if state.bits != self.state_bits:
            raise ValueError(f"trainkernel: AdamW: the state holds {state.bits}-bit moments, this optimizer {self.state_bits}-bit ones")
        if len(leaves) != len(state.sizes) or len(gradients) != len(leaves):
            raise ValueError(f"trainkernel: AdamW: {len(leaves)} params and {len(gradients)} grads for a state of {len(state.sizes)} tensors")
        places = _paths(params)
        _check_places("params", places, "the tree that init was given", state.paths)
        _check_places("grads", _paths(grads), "params", places if places is not None else state.paths)
        decays = self._decays(len(leaves))
        groups: dict[tuple, list] = {}
        for i, (leaf, grad) in enumerate(zip(leaves, gradients)):
            self._check_param(leaf, device)
            if leaf.numel() != state.sizes[i]:
                raise ValueError(f"trainkernel: AdamW: param {i} has {leaf.numel()} elements, the state {state.sizes[i]}")
            if grad.dtype not in operators.DTYPES or grad.device != device or grad.shape != leaf.shape or grad.is_neg():
                raise ValueError(f"trainkernel: AdamW: grad {i} does not match its param in shape, device or type")
            if not _same_order(leaf, grad):
                raise ValueError(f"trainkernel: AdamW: grad {i} must have its param's memory order")
            groups.setdefault((leaf.dtype, grad.dtype), []).append((leaf.data_ptr(), grad.data_ptr(), state.offsets[i], state.sizes[i], decays[i], 0))
        for name, value in (("lr", self.lr), ("grad_scale", grad_scale)):
            if isinstance(value, torch.Tensor) and (value.device != device or value.dtype != torch.float32 or value.numel() != 1):
                raise ValueError(f"trainkernel: AdamW: a tensor {name} must hold one float32 value on the params' device")
        if grad_scale is not None and not isinstance(grad_scale, torch.Tensor):
            raise ValueError("trainkernel: AdamW: grad_scale must be a tensor of one float32 value")
        _check_apart(leaves, gradients, {"lr": self.lr, "grad_scale": grad_scale})
        by_tensor = isinstance(self.lr, torch.Tensor)
        options = AdamWOptions(self.lr.data_ptr() if by_tensor else None, None if grad_scale is None else grad_scale.data_ptr(),
                               0.0 if by_tensor else self.lr, *self.betas, self.eps, self.seed, self.state_bits)
        index = operators.require_device(device)
        lib, stream = operators.library(), torch._C._cuda_getCurrentRawStream(index)
        for position, ((param_dtype, grad_dtype), items) in enumerate(groups.items()):
            operators.check(lib.tk_adamw_update((AdamWTensor * len(items))(*items), len(items), operators.DTYPES[param_dtype], operators.DTYPES[grad_dtype],
                                                state._struct, options, int(position == len(groups) - 1), index, stream))
        torch.autograd.graph.increment_version([t for t in (*leaves, *state.tensors()) if not t.is_inference()])
