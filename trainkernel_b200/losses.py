"""Token log-probabilities and the losses of language-model training, from logits, with their gradient.

Three operators, each in two forms:

* `token_logprobs`, `policy_loss`, `preference_loss` are differentiable in the logits: by `torch.func`
  transforms inside a step handed to `compile` / `compile_training` (where the call becomes an IR
  operation that runs between two generated kernels), by the same transforms in eager code, and by
  eager autograd; once, and in reverse mode only (forward-mode derivatives are refused).
* `token_logprobs_and_grad`, `policy_loss_and_grad`, `preference_loss_and_grad` return the gradient of
  the logits with the value, in the style of a compiled step.  They record no autograd history, read
  every logit from memory once where the mathematics allows it, and may be captured into a CUDA graph.

`logits` is `[batch, length, vocab]` (or `[rows, vocab]` for the first two), FP32, FP16 or BF16, of any
strides as long as one row is contiguous, so the usual shifted slice `logits[:, :-1]` needs no copy.
`targets` are int64 or int32.  `mask` is boolean, of the targets' shape; a row it excludes has
log-probability 0 and gradient 0 whatever its logits hold, NaN included.  A counted target outside
`[0, vocab)` reads nothing and gives NaN.  Log-probabilities, losses and sums are FP32; gradients have
the logits' type, and, for strided logits, their strides (inside a traced or transformed function they are dense).  Everything else that enters a loss is a constant: it must not require grad.
No counterpart in the reference, whose losses are means of squares (reference: benchmarks/train_loop.py:35-45).
"""
from __future__ import annotations

import functools
import math

import torch
from torch._functorch.pyfunctorch import temporarily_clear_interpreter_stack
from torch.autograd import forward_ad

from . import operators
from .operators import PolicyTerms, TokenArray, TokenGrad, TokenRows

AVERAGES = ("tokens", "sequences")
_TARGET_BYTES = {torch.int64: 8, torch.int32: 4}
_NO_ARRAY = (None, 0, 0)


# ---------------------------------------------------------------------------
# argument checks (metadata only: they hold for fake tensors too)
# ---------------------------------------------------------------------------

def _has_tangent(value: torch.Tensor) -> bool:
    """Whether a forward-mode derivative travels with the tensor (`forward_ad.make_dual`, `torch.func.jvp`)."""
    if forward_ad._current_level < 0:
        return False
    while True:
        if not torch._C._functorch.is_batchedtensor(value) and forward_ad.unpack_dual(value).tangent is not None:
            return True
        if not torch._C._functorch.is_functorch_wrapped_tensor(value):
            return False
        value = torch._C._functorch.get_unwrapped(value)


def _check_rows(who: str, logits, targets, mask, *, pairs: bool = False) -> None:
    if not isinstance(logits, torch.Tensor) or not isinstance(targets, torch.Tensor):
        raise TypeError(f"trainkernel: {who} takes tensors")
    if logits.dtype not in operators.DTYPES:
        raise ValueError(f"trainkernel: {who}: logits must be float32, float16 or bfloat16")
    if targets.dtype not in _TARGET_BYTES:
        raise ValueError(f"trainkernel: {who}: targets must be int64 or int32")
    rank = logits.dim()
    if rank != 3 if pairs else rank not in (2, 3):
        raise ValueError(f"trainkernel: {who}: logits must be {'[sequences, length, vocab]' if pairs else '[rows, vocab] or [batch, length, vocab]'}")
    shape = logits.shape
    if targets.shape != shape[:-1]:
        raise ValueError(f"trainkernel: {who}: targets must have the logits' shape without the vocabulary")
    if 0 in shape:
        raise ValueError(f"trainkernel: {who}: empty logits")
    if logits.stride(-1) != 1 and shape[-1] != 1:
        raise ValueError(f"trainkernel: {who}: the vocabulary must be contiguous in memory")
    if math.prod(shape[:-1]) > 0x7FFFFFFF or shape[-1] > 0x7FFFFFFF:
        raise ValueError(f"trainkernel: {who}: at most 2^31 - 1 rows and logits in a row")
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.bool or mask.shape != targets.shape:
            raise ValueError(f"trainkernel: {who}: mask must be a boolean tensor of the targets' shape")
    if pairs and shape[0] % 2:
        raise ValueError(f"trainkernel: {who}: an even number of sequences is required, the preferred half first")
    for value in (targets, mask):
        if value is not None and value.device != logits.device:
            raise ValueError(f"trainkernel: {who}: inputs must use one device")
    if logits.is_neg() or logits.is_conj():
        raise ValueError("trainkernel: resolve lazy negative or conjugate input views before execution")
    if _has_tangent(logits):
        raise RuntimeError(f"trainkernel: {who} has no forward-mode derivative")


def _check_constant(who: str, name: str, value, shape, device) -> torch.Tensor:
    """An FP32 constant, broadcast to `shape` as a strided view."""
    if not isinstance(value, torch.Tensor):
        raise TypeError(f"trainkernel: {who}: {name} must be a tensor")
    if value.dtype != torch.float32:
        raise ValueError(f"trainkernel: {who}: {name} must be float32")
    if value.device != device:
        raise ValueError(f"trainkernel: {who}: inputs must use one device")
    if value.requires_grad or _has_tangent(value):
        raise ValueError(f"trainkernel: {who}: no gradient flows to {name}; detach it")
    if value.is_neg():
        raise ValueError("trainkernel: resolve lazy negative or conjugate input views before execution")
    if value.shape != shape:
        try:
            value = value.expand(shape)
        except RuntimeError:
            raise ValueError(f"trainkernel: {who}: {name} does not broadcast to the targets' shape") from None
    return value


def _check_number(who: str, name: str, value, low: float, high: float) -> float:
    if isinstance(value, bool) or not isinstance(value, (int, float)) or not low <= value <= high:
        raise ValueError(f"trainkernel: {who}: {name} must be a number in [{low:g}, {high:g}]")
    return float(value)


def _check_scale(who: str, scale, device) -> tuple[float, torch.Tensor | None]:
    if isinstance(scale, torch.Tensor):
        if scale.dtype != torch.float32 or scale.numel() != 1 or scale.device != device:
            raise ValueError(f"trainkernel: {who}: a tensor grad_scale must hold one float32 value on the logits' device")
        if _has_tangent(scale):
            raise ValueError(f"trainkernel: {who}: no gradient flows to grad_scale; detach it")
        return 1.0, scale
    if isinstance(scale, bool) or not isinstance(scale, (int, float)):
        raise ValueError(f"trainkernel: {who}: grad_scale must be a number or a tensor of one float32 value")
    return float(scale), None


def _check_policy(who, logits, targets, old, advantages, ref, mask, clip, kl_weight, average):
    _check_rows(who, logits, targets, mask)
    old = _check_constant(who, "old_logprobs", old, targets.shape, logits.device)
    advantages = _check_constant(who, "advantages", advantages, targets.shape, logits.device)
    kl_weight = _check_number(who, "kl_weight", kl_weight, 0.0, 1e30)
    if ref is not None:
        ref = _check_constant(who, "ref_logprobs", ref, targets.shape, logits.device)
    elif kl_weight:
        raise ValueError(f"trainkernel: {who}: a KL term needs ref_logprobs")
    if not isinstance(clip, (tuple, list)) or len(clip) != 2:
        raise ValueError(f"trainkernel: {who}: clip is a pair (below, above)")
    low, high = _check_number(who, "clip below", clip[0], 0.0, 1.0), _check_number(who, "clip above", clip[1], 0.0, 1e30)
    if average not in AVERAGES:
        raise ValueError(f"trainkernel: {who}: average must be one of {', '.join(AVERAGES)}")
    return old, advantages, ref, low, high, kl_weight, AVERAGES.index(average)


# ---------------------------------------------------------------------------
# launches
# ---------------------------------------------------------------------------

def _outside_transforms(launch):
    """A launch on plain tensors inside a `torch.func` transform of something else: its results are allocated as the
    constants that they are, where the transform would wrap them."""
    @functools.wraps(launch)
    def run(*args, **kwargs):
        if torch._C._functorch.peek_interpreter_stack() is None:
            return launch(*args, **kwargs)
        with temporarily_clear_interpreter_stack():
            return launch(*args, **kwargs)
    return run


def _array(value: torch.Tensor | None, rank: int) -> tuple:
    """(pointer, batch stride, token stride) of a [batch, length] or [rows] tensor."""
    if value is None:
        return _NO_ARRAY
    strides = value.stride()
    return (value.data_ptr(), strides[0], strides[1]) if rank == 3 else (value.data_ptr(), 0, strides[0])


def _row_struct(logits: torch.Tensor, targets: torch.Tensor, mask: torch.Tensor | None) -> TokenRows:
    rank = logits.dim()
    shape, strides = logits.shape, logits.stride()
    lead = (strides[0], strides[1], shape[0], shape[1]) if rank == 3 else (0, strides[0], 1, shape[0])
    return TokenRows(logits.data_ptr(), *lead, shape[-1], operators.DTYPES[logits.dtype], _TARGET_BYTES[targets.dtype],
                     _array(targets, rank), _array(mask, rank))


def _pointer(value: torch.Tensor | None):
    return None if value is None else value.data_ptr()


def _place(logits: torch.Tensor) -> tuple:
    """(library, device ordinal, stream) of a launch."""
    device = operators.require_device(logits.device)
    return operators.library(), device, torch._C._cuda_getCurrentRawStream(device)


def _fp32(shape, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(shape, dtype=torch.float32, device=like.device)


def _grad_like(logits: torch.Tensor) -> torch.Tensor:
    """Room for the gradient.  It keeps the logits' row strides where that wastes little memory (a shifted slice of a
    longer batch does), because rows that lie alike in memory are read and written 16 bytes at a time; otherwise dense."""
    if logits.is_contiguous() and logits.storage_offset() * logits.element_size() % 16 == 0:
        return torch.empty_like(logits, memory_format=torch.contiguous_format)
    shape, strides = logits.shape, logits.stride()
    order = sorted((s, n) for s, n in zip(strides, shape) if n > 1)
    reach, apart = 1, True
    for stride, size in order:
        apart &= stride >= reach
        reach += stride * (size - 1)
    per = 16 // logits.element_size()
    lead = logits.data_ptr() % 16 // logits.element_size()
    if not apart or reach + per > 1.25 * logits.numel() + per:
        return torch.empty(shape, dtype=logits.dtype, device=logits.device)
    whole = torch.empty(lead + reach, dtype=logits.dtype, device=logits.device)
    return whole.as_strided(shape, strides, lead)


def _grad_struct(grad: torch.Tensor | None, scale: float, scale_at: torch.Tensor | None) -> TokenGrad:
    if grad is None:
        return TokenGrad(None, 0, 0, None, 1.0, 0)
    strides = grad.stride()
    return TokenGrad(grad.data_ptr(), strides[0] if grad.dim() == 3 else 0, strides[-2], _pointer(scale_at), scale, 0)


@_outside_transforms
def _logprobs_launch(logits, targets, mask, with_stats: bool):
    lib, device, stream = _place(logits)
    logprobs = _fp32(targets.shape, logits)
    stats = _fp32((*targets.shape, 2), logits) if with_stats else None
    operators.check(lib.tk_token_logprobs(_row_struct(logits, targets, mask), logprobs.data_ptr(), _pointer(stats), device, stream))
    return logprobs, stats


@_outside_transforms
def _logprobs_and_grad_launch(logits, targets, weights, mask, scale: float, scale_at):
    lib, device, stream = _place(logits)
    logprobs = _fp32(targets.shape, logits)
    grad = _grad_like(logits)
    operators.check(lib.tk_token_logprobs_and_grad(_row_struct(logits, targets, mask), TokenArray(*_array(weights, logits.dim())), logprobs.data_ptr(),
                                                   _grad_struct(grad, scale, scale_at), device, stream))
    return logprobs, grad


@_outside_transforms
def _logits_grad_launch(logits, targets, mask, coefficients, stats, scale_at):
    lib, device, stream = _place(logits)
    grad = _grad_like(logits)
    if coefficients.dim() < targets.dim():
        array = TokenArray(coefficients.data_ptr(), coefficients.stride(0), 0)          # one per sequence
    else:
        array = TokenArray(*_array(coefficients, logits.dim()))
    operators.check(lib.tk_token_logits_grad(_row_struct(logits, targets, mask), array, stats.data_ptr(),
                                             _grad_struct(grad, 1.0, scale_at), device, stream))
    return grad


@_outside_transforms
def _policy_launch(logits, targets, old, advantages, ref, mask, low, high, kl_weight, average: int, *, saved: bool, grad: bool,
                   scale: float = 1.0, scale_at=None):
    lib, device, stream = _place(logits)
    rank, shape = logits.dim(), targets.shape
    loss, logprobs = _fp32((), logits), _fp32(shape, logits)
    stats = _fp32((*shape, 2), logits) if saved else None
    coefficients = _fp32(shape, logits) if saved else None
    out = _grad_like(logits) if grad else None
    rows = _row_struct(logits, targets, mask)
    workspace = torch.empty(lib.tk_policy_workspace_bytes(rows.batch, rows.length), dtype=torch.uint8, device=logits.device)
    terms = PolicyTerms(_array(old, rank), _array(advantages, rank), _array(ref, rank), low, high, kl_weight, average)
    operators.check(lib.tk_policy_loss(rows, terms, loss.data_ptr(), logprobs.data_ptr(), _pointer(stats), _pointer(coefficients),
                                       _grad_struct(out, scale, scale_at), workspace.data_ptr(), device, stream))
    return loss, logprobs, stats, coefficients, out


@_outside_transforms
def _preference_launch(logits, targets, reference, mask, beta: float, smoothing: float, *, grad: bool, scale: float = 1.0, scale_at=None):
    lib, device, stream = _place(logits)
    shape = targets.shape
    loss, sums, coefficients, stats = _fp32((), logits), _fp32(shape[:1], logits), _fp32(shape[:1], logits), _fp32((*shape, 2), logits)
    out = _grad_like(logits) if grad else None
    rows = _row_struct(logits, targets, mask)
    workspace = torch.empty(lib.tk_preference_workspace_bytes(rows.batch, rows.length), dtype=torch.uint8, device=logits.device)
    operators.check(lib.tk_preference_loss(rows, reference.data_ptr(), reference.stride(0), beta, smoothing, loss.data_ptr(), sums.data_ptr(),
                                           stats.data_ptr(), coefficients.data_ptr(), _grad_struct(out, scale, scale_at),
                                           workspace.data_ptr(), device, stream))
    return loss, sums, stats, coefficients, out


# ---------------------------------------------------------------------------
# dispatcher operators: what a traced step records, and what its real tensors run
# ---------------------------------------------------------------------------

_ops = torch.library.Library("trainkernel", "DEF")
_ops.define("token_logprobs(Tensor logits, Tensor targets, Tensor? mask) -> (Tensor, Tensor)")
_ops.define("token_logprobs_and_grad(Tensor logits, Tensor targets, Tensor weights, Tensor? mask, float scale) -> (Tensor, Tensor)")
_ops.define("token_logits_grad(Tensor logits, Tensor targets, Tensor? mask, Tensor coefficients, Tensor stats, Tensor? scale) -> Tensor")
_ops.define("policy_loss(Tensor logits, Tensor targets, Tensor old_logprobs, Tensor advantages, Tensor? ref_logprobs, Tensor? mask, "
            "float clip_low, float clip_high, float kl_weight, int average) -> (Tensor, Tensor, Tensor, Tensor)")
_ops.define("policy_loss_and_grad(Tensor logits, Tensor targets, Tensor old_logprobs, Tensor advantages, Tensor? ref_logprobs, Tensor? mask, "
            "float clip_low, float clip_high, float kl_weight, int average, float scale) -> (Tensor, Tensor, Tensor)")
_ops.define("preference_loss(Tensor logits, Tensor targets, Tensor reference, Tensor? mask, float beta, float label_smoothing) "
            "-> (Tensor, Tensor, Tensor, Tensor)")
_ops.define("preference_loss_and_grad(Tensor logits, Tensor targets, Tensor reference, Tensor? mask, float beta, float label_smoothing, float scale) "
            "-> (Tensor, Tensor, Tensor)")


def _run_policy(logits, targets, old, advantages, ref, mask, low, high, kl_weight, average):
    return _policy_launch(logits, targets, old, advantages, ref, mask, low, high, kl_weight, average, saved=True, grad=False)[:4]


def _run_policy_and_grad(logits, targets, old, advantages, ref, mask, low, high, kl_weight, average, scale):
    loss, logprobs, _, _, grad = _policy_launch(logits, targets, old, advantages, ref, mask, low, high, kl_weight, average, saved=False, grad=True, scale=scale)
    return loss, logprobs, grad


def _run_preference(logits, targets, reference, mask, beta, smoothing):
    return _preference_launch(logits, targets, reference, mask, beta, smoothing, grad=False)[:4]


def _run_preference_and_grad(logits, targets, reference, mask, beta, smoothing, scale):
    loss, sums, _, _, grad = _preference_launch(logits, targets, reference, mask, beta, smoothing, grad=True, scale=scale)
    return loss, sums, grad


# name -> what runs on real tensors (also called, with the same arguments, by compiled programs)
IMPLEMENTATIONS = {
    "token_logprobs": lambda logits, targets, mask: _logprobs_launch(logits, targets, mask, True),
    "token_logprobs_and_grad": lambda logits, targets, weights, mask, scale: _logprobs_and_grad_launch(logits, targets, weights, mask, scale, None),
    "token_logits_grad": _logits_grad_launch,
    "policy_loss": _run_policy,
    "policy_loss_and_grad": _run_policy_and_grad,
    "preference_loss": _run_preference,
    "preference_loss_and_grad": _run_preference_and_grad,
}


def _like_fp32(shape, like):
    return like.new_empty(shape, dtype=torch.float32)


_SHAPES = {
    "token_logprobs": lambda logits, targets, *rest: (_like_fp32(targets.shape, logits), _like_fp32((*targets.shape, 2), logits)),
    "token_logprobs_and_grad": lambda logits, targets, *rest: (_like_fp32(targets.shape, logits), logits.new_empty(logits.shape)),
    "token_logits_grad": lambda logits, *rest: logits.new_empty(logits.shape),
    "policy_loss": lambda logits, targets, *rest: (_like_fp32((), logits), _like_fp32(targets.shape, logits),
                                                   _like_fp32((*targets.shape, 2), logits), _like_fp32(targets.shape, logits)),
    "policy_loss_and_grad": lambda logits, targets, *rest: (_like_fp32((), logits), _like_fp32(targets.shape, logits), logits.new_empty(logits.shape)),
    "preference_loss": lambda logits, targets, *rest: (_like_fp32((), logits), _like_fp32(targets.shape[:1], logits),
                                                       _like_fp32((*targets.shape, 2), logits), _like_fp32(targets.shape[:1], logits)),
    "preference_loss_and_grad": lambda logits, targets, *rest: (_like_fp32((), logits), _like_fp32(targets.shape[:1], logits), logits.new_empty(logits.shape)),
}


def _no_cpu(*args):
    raise RuntimeError("trainkernel: CUDA sm_100a GPU required; CPU IR inspection is available through capture()")


def _as_declared(run):
    """What a traced call runs on real tensors: results as dense as `_SHAPES` says, which a trace relies on."""
    def dense(*args):
        results = run(*args)
        return results.contiguous() if isinstance(results, torch.Tensor) else tuple(result.contiguous() for result in results)
    return dense


for _name, _run in IMPLEMENTATIONS.items():
    _ops.impl(_name, _as_declared(_run), "CUDA")
    _ops.impl(_name, _no_cpu, "CPU")
    torch.library.register_fake(f"trainkernel::{_name}", _SHAPES[_name], lib=_ops)

_call = torch.ops.trainkernel


# ---------------------------------------------------------------------------
# differentiation
# ---------------------------------------------------------------------------

class _LogitsGrad(torch.autograd.Function):
    """The gradient itself; differentiating it again is refused rather than answered with nothing."""

    @staticmethod
    def forward(logits, targets, mask, coefficients, stats, scale):
        if logits.is_cuda and _is_plain(logits, targets, mask, coefficients, stats, scale):
            return _logits_grad_launch(logits, targets, mask, coefficients, stats, scale)          # with the logits' strides
        return _call.token_logits_grad(logits, targets, mask, coefficients, stats, scale)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("trainkernel: the token losses are differentiable once")


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(logits, targets, mask):
        return _call.token_logprobs(logits, targets, mask)

    @staticmethod
    def setup_context(ctx, inputs, output):
        logits, targets, mask = inputs
        ctx.has_mask = mask is not None
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(output[1])
        ctx.save_for_backward(logits, targets, output[1], *([mask] if ctx.has_mask else []))

    @staticmethod
    def backward(ctx, grad_logprobs, _):
        if grad_logprobs is None:
            return None, None, None
        logits, targets, stats, *mask = ctx.saved_tensors
        return _LogitsGrad.apply(logits, targets, mask[0] if mask else None, grad_logprobs, stats, None), None, None


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(logits, targets, old, advantages, ref, mask, low, high, kl_weight, average):
        return _call.policy_loss(logits, targets, old, advantages, ref, mask, low, high, kl_weight, average)

    @staticmethod
    def setup_context(ctx, inputs, output):
        logits, targets, mask = inputs[0], inputs[1], inputs[5]
        ctx.has_mask = mask is not None
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*output[1:])
        ctx.save_for_backward(logits, targets, output[2], output[3], *([mask] if ctx.has_mask else []))

    @staticmethod
    def backward(ctx, grad_loss, *_):
        if grad_loss is None:
            return (None,) * 10
        logits, targets, stats, coefficients, *mask = ctx.saved_tensors
        grad = _LogitsGrad.apply(logits, targets, mask[0] if mask else None, coefficients, stats, grad_loss)
        return (grad, *(None,) * 9)


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(logits, targets, reference, mask, beta, smoothing):
        return _call.preference_loss(logits, targets, reference, mask, beta, smoothing)

    @staticmethod
    def setup_context(ctx, inputs, output):
        logits, targets, mask = inputs[0], inputs[1], inputs[3]
        ctx.has_mask = mask is not None
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*output[1:])
        ctx.save_for_backward(logits, targets, output[2], output[3], *([mask] if ctx.has_mask else []))

    @staticmethod
    def backward(ctx, grad_loss, *_):
        if grad_loss is None:
            return (None,) * 6
        logits, targets, stats, coefficients, *mask = ctx.saved_tensors
        grad = _LogitsGrad.apply(logits, targets, mask[0] if mask else None, coefficients, stats, grad_loss)
        return (grad, *(None,) * 5)


class NotFunctional(Exception):
    """Raised inside a functionalized trace: functionalization has no rule for a differentiable operator of this module,
    so `capture` traces such a function once more without it (nothing these operators do needs it)."""


def _differentiable(function: type[torch.autograd.Function], *args):
    stack = torch._C._functorch.peek_interpreter_stack()
    if stack is not None and any(level.key() == torch._C._functorch.TransformType.Functionalize for level in torch._C._functorch.get_interpreter_stack()):
        raise NotFunctional
    return function.apply(*args)


def _is_plain(*tensors: torch.Tensor | None) -> bool:
    """Real tensors, no tracing, no transform: the launch can be made directly (when there is no history to record)."""
    wrapped = torch._C._functorch.is_functorch_wrapped_tensor
    return not torch._C._len_torch_dispatch_stack() and all(
        t is None or type(t) in (torch.Tensor, torch.nn.Parameter) and not wrapped(t) for t in tensors)


def _records(who: str, logits: torch.Tensor) -> bool:
    """Whether eager autograd records this call.  Under stream capture that is refused: the recorded backward pass would
    meet leaves whose gradients an eager graph accumulates on another stream, which ends the process."""
    if not (logits.requires_grad and torch.is_grad_enabled()):
        return False
    if logits.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"trainkernel: {who}: autograd history cannot be recorded while a CUDA graph is captured; "
                           "use the _and_grad form, torch.func, or compile")
    return True


# ---------------------------------------------------------------------------
# public operators
# ---------------------------------------------------------------------------

def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, mask: torch.Tensor | None = None) -> torch.Tensor:
    """`log_softmax(logits)[targets]` in FP32, one value per row; differentiable in the logits."""
    if operators.fast is not None and (done := operators.fast.token_logprobs(logits, targets, mask)) is not None:
        return done
    _check_rows("token_logprobs", logits, targets, mask)
    if _is_plain(logits, targets, mask) and not _records("token_logprobs", logits):
        return _logprobs_launch(logits, targets, mask, False)[0]
    return _differentiable(_TokenLogprobs, logits, targets, mask)[0]


def token_logprobs_and_grad(logits: torch.Tensor, targets: torch.Tensor, weights: torch.Tensor, *, mask: torch.Tensor | None = None,
                            grad_scale: float | torch.Tensor = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """`(logprobs, grad)`: the gradient of `(weights * logprobs).sum()` in the logits, times `grad_scale`.

    With `weights = -1 / count` this is the cross entropy and its gradient in one pass over the logits.
    `weights` is FP32 and broadcasts to the targets' shape.
    """
    if operators.fast is not None and (done := operators.fast.token_logprobs_and_grad(logits, targets, weights, mask, grad_scale)) is not None:
        return done
    who = "token_logprobs_and_grad"
    _check_rows(who, logits, targets, mask)
    weights = _check_constant(who, "weights", weights, targets.shape, logits.device)
    scale, scale_at = _check_scale(who, grad_scale, logits.device)
    if _is_plain(logits, targets, weights, mask, scale_at):
        return _logprobs_and_grad_launch(logits, targets, weights, mask, scale, scale_at)
    _no_tensor_scale(who, scale_at)
    return _call.token_logprobs_and_grad(logits, targets, weights, mask, scale)


def policy_loss(logits: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, *,
                ref_logprobs: torch.Tensor | None = None, mask: torch.Tensor | None = None, clip: tuple[float, float] = (0.2, 0.2),
                kl_weight: float = 0.0, average: str = "tokens") -> tuple[torch.Tensor, torch.Tensor]:
    """`(loss, logprobs)` of the clipped policy objective with a KL penalty; the loss is differentiable in the logits,
    `logprobs` is a constant beside it.

    Per counted token, with `r = exp(logprob - old_logprob)`:
    `-min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_weight (exp(d) - d - 1)`, `d = ref_logprob - logprob`.
    `average="tokens"` averages over all counted tokens; `"sequences"` over the tokens of each sequence and then over
    all `batch` sequences (one without counted tokens contributes 0).  With nothing counted the loss is 0.  With a
    `kl_weight` of 0 `ref_logprobs` is not read.
    """
    if operators.fast is not None and (done := operators.fast.policy_loss(logits, targets, old_logprobs, advantages, ref_logprobs, mask, clip,
                                                                          kl_weight, average, None)) is not None:
        return done
    who = "policy_loss"
    old, advantages, ref, low, high, kl_weight, which = _check_policy(who, logits, targets, old_logprobs, advantages, ref_logprobs, mask, clip, kl_weight, average)
    if _is_plain(logits, targets, old, advantages, ref, mask) and not _records(who, logits):
        return _policy_launch(logits, targets, old, advantages, ref, mask, low, high, kl_weight, which, saved=False, grad=False)[:2]
    return _differentiable(_PolicyLoss, logits, targets, old, advantages, ref, mask, low, high, kl_weight, which)[:2]


def policy_loss_and_grad(logits: torch.Tensor, targets: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, *,
                         ref_logprobs: torch.Tensor | None = None, mask: torch.Tensor | None = None, clip: tuple[float, float] = (0.2, 0.2),
                         kl_weight: float = 0.0, average: str = "tokens",
                         grad_scale: float | torch.Tensor = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """`(loss, logprobs, grad)`: `policy_loss` with the gradient of `grad_scale * loss` in the logits, in one pass."""
    if operators.fast is not None and grad_scale is not None and (
            done := operators.fast.policy_loss(logits, targets, old_logprobs, advantages, ref_logprobs, mask, clip, kl_weight, average, grad_scale)) is not None:
        return done
    who = "policy_loss_and_grad"
    old, advantages, ref, low, high, kl_weight, which = _check_policy(who, logits, targets, old_logprobs, advantages, ref_logprobs, mask, clip, kl_weight, average)
    scale, scale_at = _check_scale(who, grad_scale, logits.device)
    if _is_plain(logits, targets, old, advantages, ref, mask, scale_at):
        loss, logprobs, _, _, grad = _policy_launch(logits, targets, old, advantages, ref, mask, low, high, kl_weight, which, saved=False, grad=True,
                                                    scale=scale, scale_at=scale_at)
        return loss, logprobs, grad
    _no_tensor_scale(who, scale_at)
    return _call.policy_loss_and_grad(logits, targets, old, advantages, ref, mask, low, high, kl_weight, which, scale)


def _check_preference(who, logits, targets, reference, mask, beta, label_smoothing):
    _check_rows(who, logits, targets, mask, pairs=True)
    if isinstance(reference, torch.Tensor) and reference.shape != logits.shape[:1]:
        raise ValueError(f"trainkernel: {who}: reference holds one summed log-probability per sequence")
    reference = _check_constant(who, "reference", reference, logits.shape[:1], logits.device)
    return reference, _check_number(who, "beta", beta, 0.0, 1e30), _check_number(who, "label_smoothing", label_smoothing, 0.0, 1.0)


def preference_loss(logits: torch.Tensor, targets: torch.Tensor, reference: torch.Tensor, *, mask: torch.Tensor | None = None,
                    beta: float = 0.1, label_smoothing: float = 0.0) -> tuple[torch.Tensor, torch.Tensor]:
    """`(loss, sums)` over pairs of sequences; the loss is differentiable in the logits, `sums` is a constant beside it.

    Sequence `i` is preferred over sequence `i + batch / 2`.  `sums[i]` is the sum of sequence i's counted
    log-probabilities, `reference[i]` the same sum under the reference model; with
    `h = (sums[i] - reference[i]) - (sums[j] - reference[j])` a pair's loss is
    `-(1 - label_smoothing) log sigmoid(beta h) - label_smoothing log sigmoid(-beta h)`, and the loss is their mean.
    """
    if operators.fast is not None and (
            done := operators.fast.preference_loss(logits, targets, reference, mask, beta, label_smoothing, None)) is not None:
        return done
    who = "preference_loss"
    reference, beta, label_smoothing = _check_preference(who, logits, targets, reference, mask, beta, label_smoothing)
    if _is_plain(logits, targets, reference, mask) and not _records(who, logits):
        return _preference_launch(logits, targets, reference, mask, beta, label_smoothing, grad=False)[:2]
    return _differentiable(_PreferenceLoss, logits, targets, reference, mask, beta, label_smoothing)[:2]


def preference_loss_and_grad(logits: torch.Tensor, targets: torch.Tensor, reference: torch.Tensor, *, mask: torch.Tensor | None = None,
                             beta: float = 0.1, label_smoothing: float = 0.0,
                             grad_scale: float | torch.Tensor = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """`(loss, sums, grad)`: `preference_loss` with the gradient of `grad_scale * loss` in the logits."""
    if operators.fast is not None and grad_scale is not None and (
            done := operators.fast.preference_loss(logits, targets, reference, mask, beta, label_smoothing, grad_scale)) is not None:
        return done
    who = "preference_loss_and_grad"
    reference, beta, label_smoothing = _check_preference(who, logits, targets, reference, mask, beta, label_smoothing)
    scale, scale_at = _check_scale(who, grad_scale, logits.device)
    if _is_plain(logits, targets, reference, mask, scale_at):
        loss, sums, _, _, grad = _preference_launch(logits, targets, reference, mask, beta, label_smoothing, grad=True, scale=scale, scale_at=scale_at)
        return loss, sums, grad
    _no_tensor_scale(who, scale_at)
    return _call.preference_loss_and_grad(logits, targets, reference, mask, beta, label_smoothing, scale)


def _no_tensor_scale(who: str, scale_at) -> None:
    if scale_at is not None:
        raise ValueError(f"trainkernel: {who}: inside a traced or transformed function grad_scale must be a number")
