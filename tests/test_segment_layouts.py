"""Steps that call the operators on values whose memory is not what the trace saw."""
import contextlib

import pytest
import torch

import trainkernel_b200 as tk
from oracle import interpreter
from trainkernel_b200 import codegen, segments
from trainkernel_b200.passes import fuse_loss_gradients

gpu = pytest.mark.gpu
IDS = torch.tensor([3, 0, 6, 2, 5])


def by_columns(a, ids):
    """Row-major to the trace, which keeps the order of `a.t()` through the product; column-major in the IR, whose products are dense."""
    return tk.token_logprobs((a.t() * 2.0).t(), ids)


class OracleRunner:
    """A segment on the oracle, results as dense as the kernels write them."""

    def __init__(self, segment):
        self.segment = segment
        self.arguments = []

    def _fresh_buffers(self, arguments):
        self.arguments.append(arguments)
        outputs = tuple(t.contiguous() for t in interpreter.run(self.segment.program, arguments))
        return type("Buffers", (), {"outputs": outputs, "workspace": None})

    def _launch(self, *_):
        pass


def on_the_host(monkeypatch, fn, inputs, **operators):
    """A `SegmentedProgram` of `fn` whose kernels are the oracle's and whose operators are the given functions."""
    program, _ = tk.capture(fn, inputs)
    steps, late = segments.split_at_operators(program)
    for name, run in operators.items():
        monkeypatch.setitem(segments.IMPLEMENTATIONS, name, run)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    pairs = [(step, OracleRunner(step) if isinstance(step, segments.Segment) else None) for step in steps]
    return segments.SegmentedProgram(program, pairs, torch.device("cpu"), {}, late)


def test_an_operator_never_sees_logits_with_a_strided_vocabulary(monkeypatch):
    """The kernels read a row as one run of memory, so that is what the launch has to be handed."""
    a = torch.randn(5, 7)
    seen = []

    def launch(logits, targets, mask):
        seen.append(logits)
        return torch.log_softmax(logits, -1).gather(1, targets[:, None])[:, 0], torch.zeros(5, 2)

    (got,) = on_the_host(monkeypatch, by_columns, (a, IDS), token_logprobs=launch)(a, IDS)
    assert seen[0].stride(-1) == 1 and torch.equal(seen[0], a * 2.0)
    torch.testing.assert_close(got, torch.log_softmax(a * 2.0, -1).gather(1, IDS[:, None])[:, 0])


@gpu
def test_logits_by_columns_and_their_gradient():
    a, ids = torch.randn(5, 7, device="cuda"), IDS.cuda()
    want = torch.log_softmax(a.double() * 2.0, -1).gather(1, ids[:, None])[:, 0]
    torch.testing.assert_close(tk.compile(by_columns, (a, ids))(a, ids).double(), want, rtol=1e-5, atol=1e-5)

    weights = torch.ones(5, device="cuda")

    def gradient(a, ids, weights):
        return tk.token_logprobs_and_grad((a.t() * 2.0).t(), ids, weights)[1]

    got = tk.compile(gradient, (a, ids, weights))(a, ids, weights)
    hot = torch.zeros_like(a).scatter_(1, ids[:, None], 1.0)
    torch.testing.assert_close(got, hot - torch.softmax(a * 2.0, -1), rtol=1e-5, atol=1e-5)


def backward_product(x, h, ids, weights):
    """The gradient of the logits feeds a product, whose kernel reads its operands by tiles from 16-byte boundaries."""
    return h.t() @ tk.token_logprobs_and_grad(x, ids, weights)[1]


def at_an_odd_offset(*shape, dtype=torch.bfloat16, device="cpu"):
    count = torch.Size(shape).numel()
    return torch.randn(count + 1, device=device).to(dtype)[1:].view(shape)


def test_results_reach_the_next_kernel_on_16_byte_boundaries(monkeypatch):
    x, h, ids, weights = at_an_odd_offset(64, 128), torch.randn(64, 64).to(torch.bfloat16), torch.zeros(64, dtype=torch.int64), torch.ones(64)
    given = torch.randn(64, 128).to(torch.bfloat16)

    def launch(logits, targets, weights, mask, scale):
        grad = at_an_odd_offset(64, 128)                       # as the logits lie, so that both are read and written alike
        return torch.zeros(64), grad.copy_(given)

    program = on_the_host(monkeypatch, backward_product, (x, h, ids, weights), token_logprobs_and_grad=launch)
    (got,) = program(x, h, ids, weights)
    (arguments,) = program.steps[-1][1].arguments
    assert any(torch.equal(t, given) for t in arguments if t.shape == given.shape)
    assert all(t.data_ptr() % 16 == 0 for t in arguments)
    torch.testing.assert_close(got.float(), h.float().t() @ given.float(), rtol=2e-2, atol=2e-2)


@gpu
def test_logits_at_an_odd_offset_and_the_product_behind_them():
    x, h = at_an_odd_offset(64, 128, device="cuda"), torch.randn(64, 64, device="cuda").to(torch.bfloat16)
    ids, weights = torch.zeros(64, dtype=torch.int64, device="cuda"), torch.ones(64, device="cuda")
    got = tk.compile(backward_product, (x, h, ids, weights))(x, h, ids, weights)
    hot = torch.zeros(64, 128, device="cuda").scatter_(1, ids[:, None], 1.0)
    want = h.float().t() @ (hot - torch.softmax(x.float(), -1)).to(torch.bfloat16).float()
    assert float((got.float() - want).norm() / want.norm()) <= 2e-2


# -- segments that read nothing ----------------------------------------------------------------------------------

def summed(ids, logits):
    return torch.func.grad(lambda x: -tk.token_logprobs(x, ids).sum())(logits)


def averaged(ids, logits):
    return torch.func.grad_and_value(lambda x: -tk.token_logprobs(x, ids).mean())(logits)


@pytest.mark.parametrize("fn", [summed, averaged])
def test_every_segment_has_an_input(fn):
    """What flows back into the log-probabilities is a constant here: the kernel that writes it reads no tensor."""
    inputs = (IDS, torch.randn(5, 7))
    program, _ = tk.capture(fn, inputs)
    steps, _ = segments.split_at_operators(fuse_loss_gradients(program))
    parts = [step for step in steps if isinstance(step, segments.Segment)]
    assert parts and all(part.program.inputs for part in parts)
    for part in parts:
        assert part.program.inputs[0].dtype == "float32"
        codegen.generate(part.program)


@gpu
@pytest.mark.parametrize("fn", [summed, averaged])
def test_the_gradient_of_a_cross_entropy_alone(fn):
    ids, logits = IDS.cuda(), torch.randn(5, 7, device="cuda")
    got, scale = tk.compile(fn, (ids, logits))(ids, logits), 1.0
    if fn is averaged:
        got, value = got
        scale = 0.2
        torch.testing.assert_close(value, -torch.log_softmax(logits, -1).gather(1, ids[:, None]).mean(), rtol=1e-5, atol=1e-5)
    hot = torch.zeros_like(logits).scatter_(1, ids[:, None], 1.0)
    torch.testing.assert_close(got, (torch.softmax(logits, -1) - hot) * scale, rtol=1e-5, atol=1e-6)
