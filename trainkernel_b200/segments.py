"""Programs that call the package's own operators: generated kernels with operator launches between them.

A step that uses `losses.py` cannot be one kernel: the operators are hand-written kernels with a launch
shape of their own.  `split_at_operators` cuts the program at its operator calls.  A value belongs to the
segment after the last call it depends on, so everything up to the first loss (the forward pass) is one
generated kernel, the loss launches follow, and everything behind them (the backward pass and the update)
is the next kernel.  Values that cross a cut are dense tensors allocated per call, on the caller's
stream, so a captured step gets its own.  `OptimizedProgram` puts an optimizer's launches behind any
program.  No counterpart in the reference, which has no operators outside its kernels.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Sequence

import torch

from .ir import Operation, Program, TensorSpec, validate
from .losses import IMPLEMENTATIONS
from .passes import fuse_loss_gradients


def has_operators(program: Program) -> bool:
    return any(op.op in IMPLEMENTATIONS for op in program.operations)


@dataclass(frozen=True)
class Call:
    """One operator launch: its IR operations (one per used result) share operands and arguments."""

    results: tuple[Operation, ...]

    @property
    def op(self) -> str:
        return self.results[0].op


@dataclass(frozen=True)
class Segment:
    """One generated kernel: `program` with, for every output, the slot it fills.

    `slots[k]` is `("output", j)` when output k is program output j, `("value", buffer)` when it crosses a cut.
    """

    program: Program
    slots: tuple[tuple[str, Any], ...]
    inplace: dict[int, int]


def _operands(op: Operation) -> list[TensorSpec]:
    return [value for value in op.inputs if isinstance(value, TensorSpec)]


def split_at_operators(program: Program, inplace_outputs: dict[int, int] | None = None) -> tuple[list[Segment | Call], dict[int, int]]:
    """`(steps, late)`: segments and calls in launch order, and the in-place outputs a segment could not commit itself.

    A segment commits an in-place output directly only when no later step reads the input it overwrites; the
    others (`late`: output slot -> input) are computed into fresh tensors and copied after the last step.
    """
    validate(program)
    inplace_outputs = dict(inplace_outputs or {})
    level: dict[str, int] = {spec.buffer: 0 for spec in program.inputs}
    roots = {spec.buffer: spec for spec in program.inputs}
    ordinary: dict[int, list[Operation]] = {}
    calls: dict[int, dict[str, list[Operation]]] = {}
    made_by_call: set[str] = set()
    call_level: dict[str, int] = {}
    for op in program.operations:
        at = max((level[value.buffer] for value in _operands(op)), default=0)
        roots[op.output.buffer] = op.output
        if op.op in IMPLEMENTATIONS:
            at = call_level.setdefault(op.attrs["call"], at)
            calls.setdefault(at, {}).setdefault(op.attrs["call"], []).append(op)
            level[op.output.buffer] = at + 1
            made_by_call.add(op.output.buffer)
        else:
            ordinary.setdefault(at, []).append(op)
            level[op.output.buffer] = at
    depth = max([*ordinary, *(at + 1 for at in calls), 0])

    def computed(buffer: str) -> bool:
        return buffer not in made_by_call and buffer not in input_buffers

    input_buffers = {spec.buffer for spec in program.inputs}
    # the last step that reads a buffer: segment k is step 2k, the calls behind it are step 2k + 1
    last_read: dict[str, int] = {}
    for at, ops in ordinary.items():
        for op in ops:
            for value in _operands(op):
                last_read[value.buffer] = max(last_read.get(value.buffer, -1), 2 * at)
    for at, group in calls.items():
        for ops in group.values():
            for value in _operands(ops[0]):
                last_read[value.buffer] = max(last_read.get(value.buffer, -1), 2 * at + 1)
    for spec in program.outputs:
        if spec.buffer in input_buffers or spec.buffer in made_by_call:
            last_read[spec.buffer] = 2 * depth + 2               # windows of these are copied after the last step
    steps: list[Segment | Call] = []
    late: dict[int, int] = {}
    for at in range(depth + 1):
        ops = ordinary.get(at, [])
        made = {op.output.buffer for op in ops}
        outputs: list[TensorSpec] = []
        slots: list[tuple[str, Any]] = []
        inplace: dict[int, int] = {}
        reads = {value.buffer: None for op in ops for value in _operands(op) if value.buffer not in made}
        for slot, spec in enumerate(program.outputs):
            if spec.buffer not in made:
                continue
            if slot in inplace_outputs:
                target = program.inputs[inplace_outputs[slot]]
                if last_read.get(target.buffer, -1) > 2 * at:
                    late[slot] = inplace_outputs[slot]
                else:
                    reads[target.buffer] = None
                    inplace[len(outputs)] = target.buffer         # resolved to an input position below
            outputs.append(spec)
            slots.append(("output", slot))
        for op in ops:
            buffer = op.output.buffer
            if last_read.get(buffer, -1) > 2 * at:
                outputs.append(TensorSpec(buffer, op.output.shape, op.output.dtype, op.output.strides, buffer))
                slots.append(("value", buffer))
        if outputs:
            if not reads:                                        # constants only: a kernel takes at least one tensor
                reads[next((spec for spec in program.inputs if spec.dtype.startswith(("float", "bfloat"))), program.inputs[0]).buffer] = None
            inputs = tuple(TensorSpec(b, roots[b].shape, roots[b].dtype, roots[b].strides, b) for b in reads)
            position = {spec.buffer: i for i, spec in enumerate(inputs)}
            steps.append(Segment(Program(inputs, tuple(ops), tuple(outputs)), tuple(slots), {k: position[b] for k, b in inplace.items()}))
        steps.extend(Call(tuple(group)) for group in calls.get(at, {}).values())
    for slot, target in inplace_outputs.items():
        if not computed(program.outputs[slot].buffer):
            late[slot] = target
    return steps, late


class SegmentedProgram:
    """The call interface of `runtime.CompiledProgram` over several launches."""

    def __init__(self, program: Program, steps: Sequence[tuple[Any, Any]], device: torch.device, inplace_outputs: dict[int, int], late: dict[int, int]) -> None:
        self.program = program
        self.steps = list(steps)                       # (Segment, CompiledProgram) or (Call, None)
        self.device = device
        self.inplace_outputs = dict(inplace_outputs)
        self.late = dict(late)
        self._input_meta = [(spec.shape, spec.strides, getattr(torch, spec.dtype)) for spec in program.inputs]
        # values are dropped behind their last reader, so a long program does not hold all of them
        self._frees: list[tuple[str, ...]] = []
        last: dict[str, int] = {}
        for index, (step, _) in enumerate(self.steps):
            read = [s.buffer for s in step.program.inputs] if isinstance(step, Segment) else [v.buffer for v in _operands(step.results[0])]
            last.update({buffer: index for buffer in read})
        kept = {spec.buffer for spec in program.outputs}
        for index in range(len(self.steps)):
            self._frees.append(tuple(b for b, at in last.items() if at == index and b not in kept))

    # -- the parts of CompiledProgram's surface that front end and tools use ------------------------
    from .runtime import CompiledProgram as _Single
    _validate_inputs = _Single._validate_inputs
    del _Single

    @property
    def kernels(self) -> list[Any]:
        return [runner for _, runner in self.steps if runner is not None]

    @property
    def source(self) -> str:
        return "\n".join(runner.source for runner in self.kernels)

    def resource_usage(self) -> list[dict[str, int]]:
        return [runner.resource_usage() for runner in self.kernels]

    def status(self) -> list[tuple[int, int, int, int]]:
        return [runner.status() for runner in self.kernels]

    def invalidate_carried(self) -> None:
        for runner in self.kernels:
            runner.invalidate_carried()

    def _single_only(self, *args: Any, **kwargs: Any) -> Any:
        raise ValueError("trainkernel: a program that calls operators is several launches with buffers of their own; call it, or capture it")

    allocate = run_into = _single_only
    module = property(_single_only)
    generated = property(_single_only)

    @staticmethod
    def _window(root: torch.Tensor, spec: TensorSpec) -> torch.Tensor:
        return root if tuple(root.shape) == spec.shape and tuple(root.stride()) == spec.strides and spec.offset == 0 else \
            torch.as_strided(root, spec.shape, spec.strides, root.storage_offset() + spec.offset)

    @staticmethod
    def _dense(result: torch.Tensor) -> torch.Tensor:
        """An operator's result as the next generated kernel takes it: a gradient may have its logits' strides, and lie like them within 16 bytes."""
        result = result.contiguous()
        return result.clone() if result.data_ptr() % 16 else result

    def __call__(self, *inputs: torch.Tensor) -> tuple[torch.Tensor, ...]:
        self._validate_inputs(inputs)
        for index in self.inplace_outputs.values():
            target = inputs[index]
            if target.numel():
                storage = target.untyped_storage().data_ptr()
                for other, value in enumerate(inputs):
                    if other != index and value.numel() and value.untyped_storage().data_ptr() == storage:
                        raise ValueError("trainkernel: inplace target must not alias another input")
        values = {spec.buffer: tensor for spec, tensor in zip(self.program.inputs, inputs)}
        outputs: list[torch.Tensor | None] = [None] * len(self.program.outputs)
        with torch.no_grad():
            for index, (step, runner) in enumerate(self.steps):
                if isinstance(step, Segment):
                    arguments = tuple(values[spec.buffer] for spec in step.program.inputs)
                    buffers = runner._fresh_buffers(arguments)
                    runner._launch(arguments, buffers.outputs, buffers.workspace)
                    for (kind, where), tensor in zip(step.slots, buffers.outputs):
                        if kind == "output":
                            outputs[where] = tensor
                        else:
                            values[where] = tensor
                else:
                    first = step.results[0]
                    operands = [self._window(values[value.buffer], value) for value in first.inputs]
                    # The trace checked its own strides; here a value may lie in another order, and a kernel reads a row as one run.
                    if operands[0].shape[-1] != 1 and operands[0].stride(-1) != 1:
                        operands[0] = operands[0].contiguous()
                    arguments = [operands[value] if kind == "operand" else value for kind, value in first.attrs["arguments"]]
                    with torch.cuda.device(self.device):
                        results = IMPLEMENTATIONS[step.op](*arguments)
                    results = (results,) if isinstance(results, torch.Tensor) else results
                    for op in step.results:
                        values[op.output.buffer] = self._dense(results[op.attrs["result"]])
                for buffer in self._frees[index]:
                    values.pop(buffer, None)
            for slot, spec in enumerate(self.program.outputs):
                if outputs[slot] is None:                      # a window of an input or of an operator's result
                    outputs[slot] = self._window(values[spec.buffer], spec).clone(memory_format=torch.contiguous_format)
            for slot, target in self.late.items():
                inputs[target].copy_(outputs[slot])
                outputs[slot] = inputs[target]
        return tuple(outputs)


def compile_segments(program: Program, example_inputs: Sequence[torch.Tensor], *, inplace_outputs: dict[int, int] | None = None,
                     verbose: bool = False, **options: Any) -> SegmentedProgram:
    """Compile every segment of `program` for the examples' device."""
    from . import runtime
    inplace_outputs = dict(inplace_outputs or {})
    if any(example_inputs[i].requires_grad for i in inplace_outputs.values()):
        raise ValueError("trainkernel: inplace targets must be detached from autograd")
    program = fuse_loss_gradients(program)
    steps, late = split_at_operators(program, inplace_outputs)
    device = example_inputs[0].device
    examples = {spec.buffer: tensor for spec, tensor in zip(program.inputs, example_inputs)}
    compiled: list[tuple[Any, Any]] = []
    for step in steps:
        runner = None
        if isinstance(step, Segment):
            arguments = []
            for spec in step.program.inputs:
                if spec.buffer not in examples:
                    examples[spec.buffer] = torch.empty(spec.shape, dtype=getattr(torch, spec.dtype), device=device)
                arguments.append(examples[spec.buffer])
            runner = runtime.compile_program(step.program, tuple(arguments), inplace_outputs=step.inplace, verbose=verbose, **options)
        compiled.append((step, runner))
    runner = SegmentedProgram(program, compiled, device, inplace_outputs, late)
    runner._validate_inputs(tuple(example_inputs))
    return runner


class OptimizedProgram:
    """A compiled `(state..., data...) -> (loss, grads...)` program with an optimizer's update behind it."""

    def __init__(self, runner: Any, optimizer: Any, params: Sequence[torch.Tensor]) -> None:
        if any(param.requires_grad for param in params):
            raise ValueError("trainkernel: inplace targets must be detached from autograd")
        for param in params:
            if not param.is_contiguous():
                raise ValueError("trainkernel: an optimized state tensor must be contiguous")
        self.runner = runner
        self.optimizer = optimizer
        self.count = len(params)
        self.state = optimizer.init(list(params))
        self.program = runner.program
        self.device = runner.device
        self.inplace_outputs = {1 + self.count + i: i for i in range(self.count)}

    @property
    def source(self) -> str:
        return self.runner.source

    @property
    def kept_tensors(self) -> tuple[torch.Tensor, ...]:
        return self.state.tensors()

    def _validate_inputs(self, inputs: tuple[torch.Tensor, ...]) -> None:
        self.runner._validate_inputs(inputs)
        if any(param.requires_grad for param in inputs[:self.count]):
            raise ValueError("trainkernel: inplace targets must be detached from autograd")

    def resource_usage(self) -> Any:
        return self.runner.resource_usage()

    def status(self) -> Any:
        return self.runner.status()

    def invalidate_carried(self) -> None:
        self.runner.invalidate_carried()

    allocate = run_into = SegmentedProgram._single_only
    module = property(SegmentedProgram._single_only)

    @property
    def generated(self) -> Any:
        return self.runner.generated

    def __call__(self, *inputs: torch.Tensor) -> tuple[torch.Tensor, ...]:
        self._validate_inputs(inputs)
        params = inputs[:self.count]
        for index, param in enumerate(params):
            if param.numel():
                storage = param.untyped_storage().data_ptr()
                for other, value in enumerate(inputs):
                    if other != index and value.numel() and value.untyped_storage().data_ptr() == storage:
                        raise ValueError("trainkernel: inplace target must not alias another input")
        loss, *grads = self.runner(*inputs)
        self.optimizer.update(list(params), grads[:self.count], self.state)
        return (loss, *grads[:self.count], *params)
