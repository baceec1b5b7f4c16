"""Steps that call the operators on values whose memory is not what the trace saw."""
import contextlib

import pytest
import torch

import trainkernel_b200 as tk
from oracle import interpreter
from trainkernel_b200 import segments

gpu = pytest.mark.gpu
IDS = torch.tensor([3, 0, 6, 2, 5])


def by_columns(a, ids):
    """Row-major to the trace, which keeps the order of `a.t()` through the product; column-major in the IR, whose products are dense."""
    return tk.token_logprobs((a.t() * 2.0).t(), ids)


def test_an_operator_never_sees_logits_with_a_strided_vocabulary(monkeypatch):
    """The kernels read a row as one run of memory, so that is what the launch has to be handed."""
    a = torch.randn(5, 7)
    program, _ = tk.capture(by_columns, (a, IDS))
    steps, late = segments.split_at_operators(program)
    seen = []

    def launch(logits, targets, mask):
        seen.append(logits)
        return torch.log_softmax(logits, -1).gather(1, targets[:, None])[:, 0], torch.zeros(5, 2)

    class Runner:
        """A segment on the oracle, results as dense as the kernels write them."""

        def __init__(self, segment):
            self.segment = segment

        def _fresh_buffers(self, arguments):
            outputs = tuple(t.contiguous() for t in interpreter.run(self.segment.program, arguments))
            return type("Buffers", (), {"outputs": outputs, "workspace": None})

        def _launch(self, *_):
            pass

    monkeypatch.setitem(segments.IMPLEMENTATIONS, "token_logprobs", launch)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    pairs = [(step, Runner(step) if isinstance(step, segments.Segment) else None) for step in steps]
    (got,) = segments.SegmentedProgram(program, pairs, torch.device("cpu"), {}, late)(a, IDS)
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
