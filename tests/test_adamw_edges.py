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


def test_containers_without_keys_go_by_position():
    from torch.utils import _pytree

    class Pair:
        def __init__(self, a, b):
            self.a, self.b = a, b

    _pytree.register_pytree_node(Pair, lambda pair: ([pair.a, pair.b], None), lambda children, _: Pair(*children))
    tree = {"layer": Pair(torch.zeros(3), torch.zeros(4))}
    for params in (tree, [torch.zeros(3), torch.zeros(4)]):
        with pytest.raises(RuntimeError, match="sm_100a GPU required"):
            tk.AdamW().update(params, tree, state_of(tree))


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


# -- tensors that share memory (a race inside the launch: refused before it) --------------------------------------

ON = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])


def flat(count, device):
    return torch.zeros(count, device=device)


@ON
def test_overlapping_tensors_are_refused(device):
    whole, apart = flat(1000, device), flat(1000, device)
    number = flat(1, device)
    optimizer = tk.AdamW()
    if device == "cuda":
        optimizer.update([number], [apart[:1]], optimizer.init([number]))        # the compiled host path is asked first from here on
    cases = [
        ([whole[:300], whole[299:400]], [apart[:300], apart[:101]], None, "params 0 and 1 overlap"),
        ([whole[299:400], apart[:7], whole[:300]], [apart[10:111], apart[200:207], apart[300:600]], None, "overlap"),
        ([whole[100:110], whole[:300]], [apart[:10], apart[10:310]], None, "overlap"),
        ([whole[:300], whole[:300]], [apart[:300], apart[300:600]], None, "listed twice"),
        ([whole[:300]], [whole[1:301]], None, "grad 0 overlaps param 0"),
        ([whole[:300], apart[:5]], [apart[10:310], whole[295:300]], None, "grad 1 overlaps param 0"),
        ([whole[:256], whole[256:512]], [whole[256:512], whole[:256]], None, "overlaps param"),
        ([whole[:4].bfloat16().float()[:2], whole[:300]], [apart[:2], apart[:300]], whole[7:8], "grad_scale overlaps"),
    ]
    for params, grads, scale, message in cases:
        with pytest.raises(ValueError, match=message):
            optimizer.update(params, grads, state_of(params), grad_scale=scale)
    assert not bool(whole.any())


@ON
def test_neighbours_and_a_gradient_in_its_own_param_are_accepted(device):
    whole, apart = flat(1000, device) + 1.0, flat(1000, device) + 1.0
    optimizer = tk.AdamW(lr=0.5, weight_decay=0.0)
    cases = [([whole[:300], whole[300:301], whole[301:301], whole[301:1000]], [apart[:300], apart[300:301], apart[301:301], apart[301:1000]]),
             ([whole[:300], whole[300:600]], [whole[:300], whole[600:900]])]
    for params, grads in cases:
        if device == "cpu":
            with pytest.raises(RuntimeError, match="sm_100a GPU required"):
                optimizer.update(params, grads, state_of(params))
            continue
        whole.fill_(1.0)
        optimizer.update(params, grads, optimizer.init(params))
        torch.testing.assert_close(whole[:600], torch.full((600,), 0.5, device=device), rtol=1e-5, atol=0.0)


@gpu
def test_the_short_way_leaves_overlaps_to_the_long_one():
    from trainkernel_b200 import operators
    whole, apart = flat(1000, "cuda"), flat(1000, "cuda")
    optimizer = tk.AdamW()
    for params, grads, taken in (([whole[:300], whole[300:600]], [apart[:300], apart[300:600]], True), ([whole[:300], whole[299:600]], [apart[:300], apart[300:601]], False),
                                 ([whole[:300], apart[:5]], [apart[10:310], whole[295:300]], False)):
        state = optimizer.init(params)
        answer = operators.fast.adamw_update(params, grads, state.sizes, state.offsets, 0.0, state._struct_at, state._tensors, 32, 0.0, (0.9, 0.9), 1e-8, 0, None)
        assert bool(answer) == taken


@gpu
def test_an_earlier_call_s_error_is_not_this_call_s():
    """A call on a device that does not exist fails on the host; the update behind it is answered for itself."""
    from trainkernel_b200 import operators
    params, grads = [torch.ones(300, device="cuda")], [torch.ones(300, device="cuda")]
    optimizer = tk.AdamW(lr=0.5, weight_decay=0.0)
    state = optimizer.init(params)
    logits, targets, out = torch.zeros(2, 8, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, device="cuda")
    rows = operators.TokenRows(logits.data_ptr(), 0, 8, 1, 2, 8, 0, 8, operators.TokenArray(targets.data_ptr(), 0, 1), operators.TokenArray())
    lib = operators.library()
    assert lib.tk_token_logprobs(rows, out.data_ptr(), None, 63, None) not in (0, 100001) and b"selecting the device" in lib.tk_ops_last_error()
    optimizer.update(params, grads, state)
    assert int(state.step) == 1
    torch.testing.assert_close(params[0], torch.full((300,), 0.5, device="cuda"), rtol=1e-5, atol=0.0)
