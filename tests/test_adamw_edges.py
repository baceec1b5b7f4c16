"""AdamW: trees whose order differs, tensors that overlap, and what an earlier failed call leaves behind."""
from collections import OrderedDict

import pytest
import torch

import trainkernel_b200 as tk
from trainkernel_b200 import optim

gpu = pytest.mark.gpu


def state_of(tree, bits=32):
    """A state on the host, made as `init` makes one: the checks of `update` come before anything is launched."""
    leaves = optim._leaves(tree, "params")
    return optim.AdamWState([leaf.numel() for leaf in leaves], bits, leaves[0].device, optim._paths(tree))


def tree_of(order, device="cpu"):
    return {"layer": {name: torch.full((4, 4), float(ord(name)), device=device) for name in order}, "head": [torch.zeros(4, device=device)]}


@pytest.mark.parametrize("params,grads", [("qkv", "kqv"), ("kqv", "qkv"), ("kqv", "kqv")])
def test_trees_in_another_order_are_refused(params, grads):
    """Equal shapes: by position, each gradient or each moment would go to another weight."""
    state = state_of(tree_of("qkv"))
    with pytest.raises(ValueError, match="same order"):
        tk.AdamW().update(tree_of(params), tree_of(grads), state)


def test_trees_and_lists_that_name_the_same_tensors_are_accepted():
    """They reach the launch, which is refused on the host."""
    tree = tree_of("qkv")
    leaves = optim._leaves(tree, "params")
    nested = OrderedDict(layer=OrderedDict(tree["layer"]), head=tuple(tree["head"]))
    for state in (state_of(tree), state_of(leaves), state_of(tuple(leaves))):
        for params in (tree, nested, leaves, tuple(leaves)):
            for grads in (tree_of("qkv"), optim._leaves(tree_of("qkv"), "grads")):
                with pytest.raises(RuntimeError, match="sm_100a GPU required"):
                    tk.AdamW().update(params, grads, state)
    bare = torch.zeros(3)
    with pytest.raises(RuntimeError, match="sm_100a GPU required"):
        tk.AdamW().update(bare, [torch.zeros(3)], state_of(bare))


def test_a_saved_state_of_another_order_is_refused():
    state, other, listed = state_of(tree_of("qkv")), state_of(tree_of("kqv")), state_of(optim._leaves(tree_of("qkv"), "params"))
    saved = state.state_dict()
    with pytest.raises(ValueError, match="same order"):
        other.load_state_dict(saved)
    for target in (state_of(tree_of("qkv")), listed):
        target.load_state_dict(saved)
        target.load_state_dict({key: value for key, value in saved.items() if key != "paths"})       # saved without names


@gpu
def test_a_tree_is_updated_by_its_names():
    optimizer, params = tk.AdamW(lr=0.1, weight_decay=0.0), tree_of("qkv", "cuda")
    before = {name: value.clone() for name, value in params["layer"].items()}
    grads = {"layer": {name: torch.full((4, 4), sign, device="cuda") for name, sign in (("q", 1.0), ("k", -1.0), ("v", 2.0))}, "head": [torch.ones(4, device="cuda")]}
    state = optimizer.init(params)
    optimizer.update(params, grads, state)
    for name, sign in (("q", 1), ("k", -1), ("v", 1)):         # the first step is lr in the gradient's direction
        torch.testing.assert_close(params["layer"][name], before[name] - sign * 0.1, rtol=1e-5, atol=1e-5)
    with pytest.raises(ValueError, match="same order"):
        optimizer.update(params, {"head": grads["head"], "layer": grads["layer"]}, state)
    with pytest.raises(ValueError, match="same order"):
        optimizer.update({"layer": dict(reversed(params["layer"].items())), "head": params["head"]}, grads, state)
    assert int(state.step) == 1
