"""The operator library loads without a GPU, exports what its header declares, and refuses bad arguments before any launch."""
import ctypes
import re
from pathlib import Path

from trainkernel_b200 import operators

HEADER = Path(__file__).resolve().parents[1] / "include" / "trainkernel_ops.h"


def test_library_exports_every_declared_symbol():
    declared = set(re.findall(r"\b(tk_[a-z_]+)\s*\(", HEADER.read_text()))
    assert {"tk_token_logprobs", "tk_policy_loss", "tk_preference_loss", "tk_adamw_update", "tk_ops_last_error"} <= declared
    library = ctypes.CDLL(str(operators.build_library()))
    for name in sorted(declared):
        assert hasattr(library, name), name


def test_structures_have_the_header_s_sizes():
    sizes = {operators.TokenArray: 24, operators.TokenRows: 104, operators.TokenGrad: 40, operators.PolicyTerms: 88,
             operators.AdamWTensor: 40, operators.AdamWState: 40, operators.AdamWOptions: 56}
    for structure, size in sizes.items():
        assert ctypes.sizeof(structure) == size, structure


def test_argument_errors_do_not_need_a_device():
    lib = operators.library()
    rows = operators.TokenRows()
    assert lib.tk_token_logprobs(rows, None, None, 0, None) == 100001 and b"invalid rows" in lib.tk_ops_last_error()
    rows = operators.TokenRows(16, 0, 8, 1, 4, 8, 0, 8, operators.TokenArray(16, 0, 1), operators.TokenArray())
    grad = operators.TokenGrad()
    assert lib.tk_token_logprobs_and_grad(rows, operators.TokenArray(), None, grad, 0, None) == 100001
    assert lib.tk_token_logits_grad(rows, operators.TokenArray(), None, grad, 0, None) == 100001
    assert lib.tk_policy_loss(rows, operators.PolicyTerms(), None, None, None, None, grad, None, 0, None) == 100001
    assert lib.tk_preference_loss(rows, None, 1, 0.1, 0.0, None, None, None, None, grad, None, 0, None) == 100001
    tensors = (operators.AdamWTensor * 1)(operators.AdamWTensor(16, 16, 3, 4, 0.0, 0))
    state = operators.AdamWState(16, 16, None, None, 16)
    good = operators.AdamWOptions(None, None, 0.1, 0.9, 0.9, 1e-8, 0, 32)
    assert lib.tk_adamw_update(tensors, 1, 0, 0, state, good, 1, 0, None) == 100001 and b"invalid tensor 0" in lib.tk_ops_last_error()
    for options in (operators.AdamWOptions(None, None, 0.1, 1.0, 0.9, 1e-8, 0, 32), operators.AdamWOptions(None, None, 0.1, 0.9, 0.9, 0.0, 0, 32),
                    operators.AdamWOptions(None, None, 0.1, 0.9, 0.9, 1e-8, 0, 8)):
        assert lib.tk_adamw_update(tensors, 1, 0, 0, state, options, 1, 0, None) == 100001
    assert lib.tk_policy_workspace_bytes(0, 5) == 0 and lib.tk_policy_workspace_bytes(2, 3) == 16 + 16 + 32


def test_host_path_loads_and_answers_none_for_tensors_on_the_host():
    import torch
    host = operators.host()
    logits, targets = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64)
    assert host.token_logprobs(logits, targets, None) is None and host.token_logprobs() is None
    assert host.policy_loss(logits, targets, logits, logits, None, None, (0.2, 0.2), 0.0, "tokens", None) is None
    assert host.token_logprobs(1, 2, 3) is None
