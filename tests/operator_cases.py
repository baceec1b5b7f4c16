"""Training steps that use the language-model operators, buildable on any device (their kernels are built ahead)."""
from __future__ import annotations

import torch
from torch.utils._pytree import tree_flatten

import trainkernel_b200 as tk
from trainkernel_b200 import codegen, segments
from trainkernel_b200.passes import fuse_loss_gradients

BF16 = torch.bfloat16


def trunk(params, x):
    """Two layers, BF16 compute on FP32 masters: hidden states to logits."""
    q = [p.to(BF16) for p in params]
    return torch.relu(x @ q[0] + q[1]) @ q[2]


def data(device, rows=48, width=64, hidden=96, vocab=200, seed=0):
    gen = torch.Generator(device="cpu").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=gen) * scale

    params = (normal(width, hidden, scale=width ** -0.5), torch.zeros(hidden), normal(hidden, vocab, scale=hidden ** -0.5))
    x = normal(rows, width).to(BF16)
    ids = torch.randint(0, vocab, (rows,), generator=gen)
    mask = torch.rand(rows, generator=gen) < 0.8
    old, ref, advantages = -5.5 + normal(rows, scale=0.3), -5.5 + normal(rows, scale=0.3), normal(rows)
    move = lambda t: t.to(device)  # noqa: E731
    return tuple(map(move, params)), move(x), move(ids), move(mask), move(old), move(ref), move(advantages)


def policy_gradients(params, x, ids, mask, old, ref, advantages):
    def loss_fn(p):
        return tk.policy_loss(trunk(p, x), ids, old, advantages, ref_logprobs=ref, mask=mask, clip=(0.2, 0.3), kl_weight=0.1)[0]
    grads, loss = torch.func.grad_and_value(loss_fn)(params)
    return loss, grads


def policy_step(params, *rest):
    loss, grads = policy_gradients(params, *rest)
    return loss, grads, tuple(p - 0.05 * g for p, g in zip(params, grads))


def likelihood_step(params, x, ids, mask, old, ref, advantages):
    """Cross entropy through the differentiable log-probabilities: the coefficients are computed inside the step."""
    def loss_fn(p):
        return -(tk.token_logprobs(trunk(p, x), ids, mask=mask) * advantages).sum() * 0.02
    grads, loss = torch.func.grad_and_value(loss_fn)(params)
    return loss, grads, tuple(p - 0.05 * g for p, g in zip(params, grads))


def preference_step(params, x, ids, mask, old, ref, advantages):
    """8 sequences of 6 tokens, the preferred half first; the loss is scaled inside the step, so nothing merges."""
    def loss_fn(p):
        logits = trunk(p, x).view(8, 6, 200)
        return tk.preference_loss(logits, ids.view(8, 6), old.view(8, 6).sum(1), mask=mask.view(8, 6), beta=0.3)[0] * 2.0
    grads, loss = torch.func.grad_and_value(loss_fn)(params)
    return loss, grads, tuple(p - 0.05 * g for p, g in zip(params, grads))


def explicit_step(params, x, ids, mask, old, ref, advantages):
    """The `_and_grad` form inside a step that writes its own backward pass; the update of the last layer is also returned scaled."""
    q = [p.to(BF16) for p in params]
    h = torch.relu(x @ q[0] + q[1])
    loss, logp, d = tk.policy_loss_and_grad(h @ q[2], ids, old, advantages, mask=mask)
    grads = ((h.t() @ d).float(),)
    return loss, logp, d, params[2] - 0.05 * grads[0]


CASES = {"policy": policy_step, "likelihood": likelihood_step, "preference": preference_step}


def kernel_sources() -> dict[str, str]:
    """The generated source of every segment of every case."""
    example = data("cpu")
    sources: dict[str, str] = {}

    def add(name, fn, inplace):
        program, _ = tk.capture(fn, example)
        steps, _ = segments.split_at_operators(fuse_loss_gradients(program), inplace)
        for index, step in enumerate(steps):
            if isinstance(step, segments.Segment):
                sources[f"operators_{name}_{index}"] = codegen.generate(step.program, inplace_outputs=step.inplace).source

    count = len(tree_flatten(example[0])[0])
    for name, fn in CASES.items():
        add(name, fn, {1 + count + i: i for i in range(count)})
    add("gradients", policy_gradients, {})
    add("explicit", explicit_step, {})
    return sources
