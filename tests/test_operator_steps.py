"""Compiled steps that use the language-model operators: capture, cutting, merging, and the whole step on the GPU."""
import pytest
import torch
from torch.utils._pytree import tree_flatten

import trainkernel_b200 as tk
from oracle import interpreter
from tests import operator_cases as cases
from tests.helpers import rel_error
from trainkernel_b200 import segments
from trainkernel_b200.ir import Program
from trainkernel_b200.passes import fuse_loss_gradients

gpu = pytest.mark.gpu


def flat(args):
    return tree_flatten(args)[0]


def run_steps(program, steps, inputs):
    """The oracle on every segment and call in turn, as `SegmentedProgram` orders them."""
    values = {spec.buffer: tensor for spec, tensor in zip(program.inputs, inputs)}
    outputs = [None] * len(program.outputs)
    for step in steps:
        if isinstance(step, segments.Segment):
            results = interpreter.run(step.program, [values[spec.buffer] for spec in step.program.inputs])
            for (kind, where), tensor in zip(step.slots, results):
                if kind == "output":
                    outputs[where] = tensor
                else:
                    values[where] = tensor.contiguous()
        else:
            for op in step.results:
                sources = {value.buffer: program_spec(value) for value in op.inputs}
                alone = Program(tuple(sources.values()), (op,), (op.output,))
                values[op.output.buffer] = interpreter.run(alone, [values[b] for b in sources])[0]
    for slot, spec in enumerate(program.outputs):
        if outputs[slot] is None:
            outputs[slot] = torch.as_strided(values[spec.buffer], spec.shape, spec.strides, spec.offset)
    return outputs


def program_spec(value):
    from dataclasses import replace
    return replace(value, offset=0)


@pytest.mark.parametrize("name", cases.CASES)
def test_cutting_and_merging_keep_every_result(name):
    example = cases.data("cpu")
    program, _ = tk.capture(cases.CASES[name], example)
    assert segments.has_operators(program)
    expected = interpreter.run(program, flat(example))
    merged = fuse_loss_gradients(program)
    kinds = {op.op for op in merged.operations if op.op in segments.IMPLEMENTATIONS}
    assert kinds == {"policy": {"policy_loss_and_grad"}, "likelihood": {"token_logprobs", "token_logits_grad"},
                     "preference": {"preference_loss", "token_logits_grad"}}[name]
    inplace = {4 + i: i for i in range(3)}
    steps, late = segments.split_at_operators(merged, inplace)
    assert not late
    assert sorted(len(s.inplace) for s in steps if isinstance(s, segments.Segment)) [-1] == 3
    for got in (interpreter.run(merged, flat(example)), run_steps(merged, steps, flat(example))):
        for a, b in zip(got, expected):
            assert a.shape == b.shape and a.dtype == b.dtype
            torch.testing.assert_close(a, b, rtol=1e-6, atol=1e-9)


def test_eager_derivative_of_the_formulas_matches_the_captured_program():
    """The captured backward operations against autograd through the same loss written in plain operations."""
    params, x, ids, mask, old, ref, advantages = cases.data("cpu")
    program, _ = tk.capture(cases.policy_step, (params, x, ids, mask, old, ref, advantages))
    loss, *rest = interpreter.run(program, [*params, x, ids, mask, old, ref, advantages])

    def plain(p):
        logp = torch.log_softmax(cases.trunk(p, x).float(), -1).gather(-1, ids[:, None])[:, 0]
        ratio = torch.exp(logp - old)
        term = -torch.minimum(ratio * advantages, ratio.clamp(0.8, 1.3) * advantages) + 0.1 * (torch.exp(ref - logp) - (ref - logp) - 1)
        return (term * mask).sum() / mask.sum()

    grads, value = torch.func.grad_and_value(plain)(params)
    torch.testing.assert_close(loss, value, rtol=1e-5, atol=1e-6)
    for a, b in zip(rest[:3], grads):
        assert rel_error(a, b) <= 2e-2                      # two BF16 backward passes that round the logits' gradient once each


def test_an_output_that_is_still_read_is_committed_after_the_last_step():
    x, ids = torch.randn(5, 7), torch.zeros(5, dtype=torch.int64)

    def fn(w, ids):
        return w * 2.0, tk.token_logprobs(w, ids)           # the new value is ready before the operator reads the old one

    program, _ = tk.capture(fn, (x, ids))
    steps, late = segments.split_at_operators(program, {0: 0})
    assert late == {0: 0} and all(not s.inplace for s in steps if isinstance(s, segments.Segment))


def test_capture_refuses_what_the_operators_refuse():
    x, ids = torch.randn(5, 7), torch.zeros(5, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="int64 or int32"):
        tk.capture(lambda a, b: tk.token_logprobs(a, b), (x, x))
    with pytest.raises(RuntimeError, match="grad_scale must be a number"):
        tk.capture(lambda a, b, s: tk.token_logprobs_and_grad(a, b, torch.zeros_like(s).expand(5), grad_scale=s), (x, ids, torch.ones(())))
    with pytest.raises(ValueError, match="unsupported ATen op aten.mul_"):
        tk.capture(lambda a, b: torch.func.grad(lambda y: tk.token_logprobs(y.clone().mul_(2.0), b).sum())(a), (x, ids))
    with pytest.raises(TypeError, match="must be an AdamW"):
        tk.compile_training(lambda p: (p.sum(), p), (x,), optimizer="adamw")
    with pytest.raises(ValueError, match="must return loss, gradients"):
        tk.compile_training(lambda p: (p.sum(), p, p), (x,), optimizer=tk.AdamW())


def test_sharded_steps_refuse_the_operators():
    from trainkernel_b200 import dp
    example = cases.data("cpu")
    for form in (dp.ShardedTrainingStep, dp.FusedShardedTrainingStep):
        with pytest.raises(ValueError, match="cannot call the token operators"):
            form(cases.policy_step, example)


def test_masks_are_accepted_as_inputs_and_nothing_else_is_done_with_them():
    with pytest.raises(ValueError, match="unsupported"):
        tk.capture(lambda m: m & m, (torch.ones(3, dtype=torch.bool),))


# -- on the GPU ----------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("name", cases.CASES)
def test_compiled_steps_follow_the_oracle_and_replay(name):
    """Three steps and a captured one against the IR oracle (2e-2, the bound of every 16-bit-compute step here)."""
    example, host = cases.data("cuda"), cases.data("cpu")
    step = tk.compile_training(cases.CASES[name], example)
    program, _ = tk.capture(cases.CASES[name], host)
    state, want = example[0], host[0]
    for _ in range(3):
        loss, grads, state = step(state, *example[1:])
        expected = interpreter.run(program, [*want, *host[1:]])
        for a, b in zip([loss, *grads, *state], expected):
            assert rel_error(a, b) <= 2e-2
        assert all(a.data_ptr() == b.data_ptr() for a, b in zip(state, example[0]))
        want = tuple(p.cpu() for p in state)
    step.runner.status()
    captured = step.capture(state, *example[1:])
    for a, b in zip(state, want):
        assert torch.equal(a.cpu(), b)                        # capturing leaves the state alone
    loss, grads, new = captured.replay()
    torch.cuda.synchronize()
    expected = interpreter.run(program, [*want, *host[1:]])
    for a, b in zip([loss, *grads, *new], expected):
        assert rel_error(a, b) <= 2e-2


@gpu
def test_a_step_with_its_own_backward_pass_and_operator_results_as_outputs():
    example, host = cases.data("cuda"), cases.data("cpu")
    got = tk.compile(cases.explicit_step, example)(*example)
    program, _ = tk.capture(cases.explicit_step, host)
    for a, b in zip(got, interpreter.run(program, flat(host))):
        assert a.shape == b.shape and rel_error(a, b) <= 2e-2


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_policy_step_with_adamw_together(bits):
    """Loss, backward kernel and optimizer as they are used: five steps and three replays against the same parts called one by one."""
    example = cases.data("cuda")
    optimizer = tk.AdamW(lr=1e-2, weight_decay=0.1, state_bits=bits)
    step = tk.compile_training(cases.policy_gradients, example, optimizer=optimizer)
    gradients = tk.compile(cases.policy_gradients, example)
    params = tuple(p.clone() for p in example[0])
    state = optimizer.init(params)
    ours = example[0]
    for t in range(1, 6):
        loss, grads, ours = step(ours, *example[1:])
        want_loss, want_grads = gradients(params, *example[1:])
        optimizer.update(params, want_grads, state)
        assert torch.equal(loss, want_loss)
        for a, b in zip([*grads, *ours], [*want_grads, *params]):
            assert torch.equal(a, b)
        assert int(step.runner.state.step) == t
    captured = step.capture(ours, *example[1:])
    assert int(step.runner.state.step) == 5
    for t in range(6, 9):
        loss, grads, new = captured.replay()
        want_loss, want_grads = gradients(params, *example[1:])
        optimizer.update(params, want_grads, state)
        torch.cuda.synchronize()
        assert torch.equal(loss, want_loss) and int(step.runner.state.step) == t
        for a, b in zip(new, params):
            assert torch.equal(a, b)
    for a, b in zip(step.runner.state.tensors(), state.tensors()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@gpu
def test_eager_and_compiled_forms_of_a_step_agree():
    example = cases.data("cuda")
    eager = cases.policy_step(*example)
    compiled = tk.compile(cases.policy_step, example)(*example)
    for a, b in zip(flat(compiled), flat(eager)):
        assert rel_error(a, b) <= 2e-2


@gpu
def test_late_commit_and_optimizer_refusals():
    w, ids = torch.randn(5, 7, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda")
    kept = w.clone()
    runner = tk.compile(lambda w, ids: (w * 2.0, tk.token_logprobs(w, ids)), (w, ids), inplace_outputs={0: 0})
    doubled, logp = runner(w, ids)
    assert doubled.data_ptr() == w.data_ptr() and torch.equal(w, kept * 2.0) and torch.equal(logp, tk.token_logprobs(kept, ids))
    for use in (lambda: runner.runner.allocate(w, ids), lambda: runner.runner.run_into(w, ids, buffers=None), lambda: runner.runner.module):
        with pytest.raises(ValueError, match="several launches"):
            use()
    example = cases.data("cuda")
    step = tk.compile_training(cases.policy_gradients, example, optimizer=tk.AdamW())
    with pytest.raises(ValueError, match="shape, stride"):
        step(example[0], example[1][:-1], *example[2:])
    with pytest.raises(ValueError, match="alias"):
        params = (*example[0][:1], example[0][1], example[0][2])
        ref = params[0].view(-1)[:48]
        step(params, *example[1:5], ref, example[6])
