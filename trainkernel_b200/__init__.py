"""B200-native (sm_100a) back end for TrainKernel-style compiled training steps.

Same public names as the reference package (reference: trainkernel/__init__.py:1-23).
"""
from .ir import Operation, Program, TensorSpec
from .frontend import (
    CapturedProgram,
    CompiledFunction,
    CompiledTrainingStep,
    capture,
    compile,
    compile_training,
)
from .losses import (
    policy_loss,
    policy_loss_and_grad,
    preference_loss,
    preference_loss_and_grad,
    token_logprobs,
    token_logprobs_and_grad,
)
from .optim import AdamW, AdamWState

__version__ = "0.1.0"

__all__ = [
    "TensorSpec",
    "Operation",
    "Program",
    "CapturedProgram",
    "CompiledFunction",
    "CompiledTrainingStep",
    "capture",
    "compile",
    "compile_training",
    "token_logprobs",
    "token_logprobs_and_grad",
    "policy_loss",
    "policy_loss_and_grad",
    "preference_loss",
    "preference_loss_and_grad",
    "AdamW",
    "AdamWState",
]
