"""The language-model operators at the edges of their ranges: large logits, tangents, layouts, overlaps, errors.

Bounds are those of test_token_losses.py, derived there, unless a test says otherwise.
"""
import math

import pytest
import torch

import trainkernel_b200 as tk
from tests.test_token_losses import BF16, F16, F32, U, assert_grad, assert_logprobs, exact_preference, noise

gpu = pytest.mark.gpu


# -- rows whose largest logit is far from zero ---------------------------------------------------------------------

TOPS = [-1e5, -1e8, -1e9, -1e10, -1e20, -1e30, 1e5, 1e8, 1e10, 1e20, 1e30]


def far_rows(vocab, dtype, tops=TOPS):
    """Per top: a uniform row, a row that mixes it with its neighbours below, and one with a few of it among zeros or lower ones."""
    rows, targets = [], []
    place = torch.arange(vocab, device="cuda")
    for top in tops:
        value = torch.full((vocab,), top, dtype=dtype, device="cuda")
        below = value.float() - value.abs().float() * torch.finfo(dtype).eps * (place % 3)
        rest = torch.where(place % 97 == 5, value.float(), min(4.0 * top, 0.0))
        rows += [value, below.to(dtype), rest.to(dtype)]
        targets += [vocab // 2, vocab - vocab % 3 - 3, vocab // 97 // 2 * 97 + 5]
    return torch.stack(rows), torch.tensor(targets, device="cuda")


def crossing_rows(vocab, scale):
    """FP32 rows that pass from one side of +-2^16 to the other: up, down, by turns, and in runs of a vector, a block, a cluster's share."""
    place = torch.arange(vocab, device="cuda", dtype=torch.float64)
    forms = [place / vocab * 12 - 6, 6 - place / vocab * 12, (place % 2) * 3 - 1.5, (place // 4 % 2) * 3 - 1.5, (place // 1024 % 2) * 5 - 2.5, (place // (vocab / 8) % 2) * 5 - 2.5]
    rows = torch.stack([sign * 65536.0 + form * scale for sign in (1, -1) for form in forms]).float()
    return rows, torch.arange(len(rows), device="cuda") * (vocab // 13) + 1


# (vocab, repeats): few rows of a short and a long vocabulary (rows split over blocks), many rows of every block shape
PLACES = [(101, 1), (1003, 1), (1003, 60), (40001, 1), (20011, 40), (70001, 40)]


def check_rows(rows, targets):
    weights = noise((len(rows),), 1.0, 1)
    assert_logprobs(tk.token_logprobs(rows, targets), rows, targets)
    logp, grad = tk.token_logprobs_and_grad(rows, targets, weights)
    assert_logprobs(logp, rows, targets)
    assert_grad(grad, rows, targets, weights.double(), 2 * U)
    leaf = rows.clone().requires_grad_()                       # statistics saved by one kernel, the gradient from them by another
    (tk.token_logprobs(leaf, targets) * weights).sum().backward()
    assert_grad(leaf.grad, rows, targets, weights.double(), 2 * U)


@gpu
@pytest.mark.parametrize("vocab,times", PLACES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_large_logits(vocab, times, dtype):
    rows, targets = far_rows(vocab, dtype, TOPS if times == 1 or vocab < 20000 else TOPS[1::3])
    check_rows(rows.repeat(times, 1)[:1000], targets.repeat(times)[:1000])


@gpu
@pytest.mark.parametrize("vocab,times", PLACES)
@pytest.mark.parametrize("scale", [1.0, 1 / 16])
def test_rows_on_both_sides_of_the_switch(vocab, times, scale):
    rows, targets = crossing_rows(vocab, scale)
    check_rows(rows.repeat(times, 1)[:720], targets.repeat(times)[:720])


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_losses_of_rows_filled_with_a_large_negative_number(dtype):
    """Every choice excluded with a finite constant: the tokens are uniform, and losses and gradients are numbers."""
    vocab = 515
    logits = noise((4, 3, vocab), 1.0, 2).to(dtype)
    logits[:, 1] = -1e10
    logits[2, 2] = -1e30
    targets = torch.randint(0, vocab, (4, 3), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    logp = tk.token_logprobs(logits, targets)
    assert_logprobs(logp, logits, targets)
    old, advantages = logp.clone(), noise((4, 1), 1.0, 4)
    loss, _, grad = tk.policy_loss_and_grad(logits, targets, old, advantages)
    # the ratio is 1 up to two log-probabilities, each good to 60 u (its row is about 6 deep and has 515 logits)
    assert abs(float(loss) + float(advantages.mean())) <= 128 * U * float(advantages.abs().max())
    assert_grad(grad, logits, targets, (-advantages.double() / 12).expand(4, 3), 128 * U)
    reference = noise((4,), 2.0, 5)
    loss, sums, grad = tk.preference_loss_and_grad(logits, targets, reference, beta=0.5)
    want, want_sums, slope = exact_preference(logits, targets, reference, None, 0.5, 0.0)
    # three log-probabilities near -8 are added, each good to 64 u; z is off by half of four such sums, its sigmoid by a quarter of that
    assert bool(((sums.double() - want_sums).abs() <= 3 * 64 * U + want_sums.abs() * U).all())
    assert abs(float(loss) - float(want)) <= 0.5 * 4 * 192 * U + 16 * U * (1 + abs(float(want)))
    relative = 0.5 * 4 * 192 * U + 16 * U                     # d log sigmoid' = 1 - sigmoid <= 1
    assert_grad(grad, logits, targets, slope[:, None].expand(4, 3), relative)


# -- forward-mode derivatives --------------------------------------------------------------------------------------

ON = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])


def calls(logits, targets, old, reference):
    """Every operator on the given tensors: name -> (call of the logits, call of one constant or None)."""
    one = torch.ones((), device=logits.device)
    return {
        "token_logprobs": (lambda x: tk.token_logprobs(x, targets), None),
        "token_logprobs_and_grad": (lambda x: tk.token_logprobs_and_grad(x, targets, old), lambda c: tk.token_logprobs_and_grad(logits, targets, c)),
        "policy_loss": (lambda x: tk.policy_loss(x, targets, old, old), lambda c: tk.policy_loss(logits, targets, old, c)),
        "policy_loss_and_grad": (lambda x: tk.policy_loss_and_grad(x, targets, old, old), lambda c: tk.policy_loss_and_grad(logits, targets, c, old)),
        "policy_loss ref": (lambda x: tk.policy_loss(x, targets, old, old, ref_logprobs=old, kl_weight=0.1),
                            lambda c: tk.policy_loss(logits, targets, old, old, ref_logprobs=c, kl_weight=0.1)),
        "preference_loss": (lambda x: tk.preference_loss(x, targets, reference), lambda c: tk.preference_loss(logits, targets, c.sum(1))),
        "preference_loss_and_grad": (lambda x: tk.preference_loss_and_grad(x, targets, reference), lambda c: tk.preference_loss_and_grad(logits, targets, c.sum(1))),
        "grad_scale": (lambda x: tk.policy_loss_and_grad(x, targets, old, old, grad_scale=one),
                       lambda c: tk.policy_loss_and_grad(logits, targets, old, old, grad_scale=c.sum())),
    }


@ON
@pytest.mark.parametrize("name", calls(*[torch.zeros(1)] * 4))
def test_forward_mode_is_refused_everywhere(device, name):
    """A dropped tangent would read as a derivative of zero."""
    from torch.autograd import forward_ad
    logits, targets, old = torch.randn(2, 3, 5, device=device), torch.zeros((2, 3), dtype=torch.int64, device=device), torch.zeros((2, 3), device=device)
    of_logits, of_constant = calls(logits, targets, old, old.sum(1))[name]
    if device == "cuda":
        of_logits(logits)                                      # from here on the compiled host path is asked first
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            of_logits(forward_ad.make_dual(logits, torch.ones_like(logits)))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            of_logits(forward_ad.make_dual(logits, torch.ones_like(logits))[:, :, :4])             # a view carries its tangent
        if of_constant is not None:
            with pytest.raises(ValueError, match="detach"):
                of_constant(forward_ad.make_dual(old, torch.ones_like(old)))
        if device == "cuda":
            of_logits(logits)                                  # nothing else changes inside the level
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(of_logits, (logits,), (torch.ones_like(logits),))
    if of_constant is not None:
        with pytest.raises(ValueError, match="detach"):
            torch.func.jvp(of_constant, (old,), (torch.ones_like(old),))


# -- terms of weight zero ------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("grad", [False, True])
def test_a_kl_term_of_weight_zero_is_no_term(grad):
    """exp(ref - logprob) overflows FP32 from 89 on; its weight says that nothing of it is wanted."""
    logits, targets = noise((2, 3, 50), 1.0, 6), torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    old = tk.token_logprobs(logits, targets)
    form = tk.policy_loss_and_grad if grad else tk.policy_loss
    want = form(logits, targets, old, torch.ones_like(old))
    for ref in (old + 200.0, torch.full_like(old, float("inf")), torch.full_like(old, float("nan"))):
        for a, b in zip(form(logits, targets, old, torch.ones_like(old), ref_logprobs=ref, kl_weight=0.0), want):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("side", [0, 1])
def test_a_token_of_probability_zero_decides_its_pair(side):
    """With label_smoothing 0 a pair whose rejected sequence cannot occur has loss 0, one whose preferred sequence cannot has loss inf."""
    logits, targets = noise((2, 3, 50), 1.0, 7), torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    logits[side, 1, 0] = -float("inf")
    loss, sums, grad = tk.preference_loss_and_grad(logits, targets, torch.zeros(2, device="cuda"), beta=0.5)
    assert float(sums[side]) == -float("inf") and bool(torch.isfinite(sums[1 - side])) and bool(torch.isfinite(grad).all())
    assert float(loss) == (0.0 if side else float("inf"))
    assert bool((grad == 0).all()) == bool(side)
    # turned round by a smoothing of 1; with both terms, each infinite somewhere, the loss is infinite
    assert float(tk.preference_loss(logits, targets, torch.zeros(2, device="cuda"), beta=0.5, label_smoothing=1.0)[0]) == (float("inf") if side else 0.0)
    assert float(tk.preference_loss(logits, targets, torch.zeros(2, device="cuda"), beta=0.5, label_smoothing=0.5)[0]) == float("inf")


# -- layouts -------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("form", ["policy_loss_and_grad", "preference_loss_and_grad", "token_logprobs_and_grad", "backward"])
def test_a_trace_of_shifted_logits_meets_the_layout_that_it_saw(form):
    """A graph traced with fake tensors, run on real ones: `view` on the gradient is only possible where it is as dense as declared."""
    from torch.fx.experimental.proxy_tensor import make_fx
    logits = noise((4, 6, 33), 1.0, 8).to(BF16)[:, :-1]
    targets, old = torch.zeros((4, 5), dtype=torch.int64, device="cuda"), noise((4, 5), 0.1, 9) - 3.5

    def gradient(x):
        if form == "policy_loss_and_grad":
            return tk.policy_loss_and_grad(x, targets, old, old)[2]
        if form == "preference_loss_and_grad":
            return tk.preference_loss_and_grad(x, targets, old[:, 0])[2]
        if form == "token_logprobs_and_grad":
            return tk.token_logprobs_and_grad(x, targets, old)[1]
        return torch.func.grad(lambda y: (tk.token_logprobs(y, targets) * old).sum())(x)

    graph = make_fx(lambda x: gradient(x).view(-1) * 1.0, tracing_mode="fake", _allow_non_fake_inputs=True)(logits)
    got, want = graph(logits), gradient(logits)
    assert torch.equal(got, want.reshape(-1))
    assert want.stride() == logits.stride()                    # called directly, it lies as its logits do, without a copy


@gpu
def test_the_eager_gradient_of_shifted_logits_lies_as_they_do():
    whole = noise((4, 6, 33), 1.0, 10).requires_grad_()
    shifted = whole[:, :-1]
    seen = []
    shifted.register_hook(lambda grad: seen.append(grad.stride()))
    targets = torch.zeros((4, 5), dtype=torch.int64, device="cuda")
    tk.token_logprobs(shifted, targets).sum().backward()
    assert seen == [shifted.stride()]
    assert_grad(whole.grad[:, :-1], shifted.detach(), targets, torch.ones((4, 5), dtype=torch.float64, device="cuda"), 2 * U)
    assert bool((whole.grad[:, -1] == 0).all())


@gpu
def test_a_tensor_subclass_goes_the_long_way():
    """Its operations may mean something else, so the call is dispatched; the values are the same."""
    from trainkernel_b200 import operators

    class Marked(torch.Tensor):
        seen = 0

        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            cls.seen += "trainkernel" in str(func)
            return super().__torch_function__(func, types, args, kwargs or {})

    logits, targets = noise((3, 40), 1.0, 11), torch.zeros(3, dtype=torch.int64, device="cuda")
    want = tk.token_logprobs(logits, targets)                  # from here on the compiled host path is asked first
    marked = logits.as_subclass(Marked)
    for arguments in ((marked, targets, None), (logits, targets.as_subclass(Marked), None), (logits, targets, (targets == 0).as_subclass(Marked))):
        assert operators.fast.token_logprobs(*arguments) is None
    assert operators.fast.token_logprobs(torch.nn.Parameter(logits, requires_grad=False), targets, None) is not None
    logp, grad = tk.token_logprobs_and_grad(marked, targets, torch.ones(3, device="cuda"))
    assert Marked.seen and torch.equal(logp.as_subclass(torch.Tensor), want)
    assert torch.equal(tk.token_logprobs(marked, targets).as_subclass(torch.Tensor), want)


# -- many masked rows ----------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("rows,vocab,dtype", [(5000, 333, BF16), (16384, 40, F32), (1000, 20011, F16), (1024, 50257, BF16), (3000, 9001, F32)])
@pytest.mark.parametrize("counted", [1.0, 0.5, 0.01])
def test_policy_loss_of_many_rows_without_a_batch(rows, vocab, dtype, counted):
    """Rows that run at once, rows behind them and masked rows of both kinds; repeated, because their order is not fixed."""
    logits = noise((rows, vocab), 2.0, 12).to(dtype)
    targets = torch.randint(0, vocab, (rows,), generator=torch.Generator(device="cuda").manual_seed(13), device="cuda", dtype=torch.int32)
    mask = torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(14), device="cuda") < counted
    mask[0] = counted < 1                                      # the first row counts, or is the only one that does not
    every = tk.token_logprobs(logits, targets)
    old, advantages = every + noise((rows,), 0.1, 15), noise((rows,), 1.0, 16)
    logp = torch.log_softmax(logits.double(), -1).gather(1, targets.long()[:, None])[:, 0]
    ratio = torch.exp(logp - old)
    terms = -torch.minimum(ratio * advantages, ratio.clamp(0.5, 2.0) * advantages)
    want = float(terms[mask].mean())
    # a log-probability is off by d, its ratio by that and 4 u relative; ratios are below 2
    x = logits.double()
    d = float(U * (4 * (x.amax(-1) - x.amin(-1)).max() + vocab / 256 + 40))
    for _ in range(5):
        loss, got, grad = tk.policy_loss_and_grad(logits, targets, old, advantages, mask=mask, clip=(0.5, 1.0))
        assert torch.equal(got == 0, ~mask) and bool((grad[~mask] == 0).all()) and bool((grad[mask] != 0).any())
        assert abs(float(loss) - want) <= 2 * float(advantages.abs().max()) * (d + 8 * U) + 4 * U * abs(want)
        assert abs(float(tk.policy_loss(logits, targets, old, advantages, mask=mask, clip=(0.5, 1.0))[0]) - want) <= 2 * float(advantages.abs().max()) * (d + 8 * U) + 4 * U * abs(want)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_saved_statistics_are_what_the_header_says(dtype):
    """The sum is exact to rounding where the largest logit is 0 or beyond 2^16, elsewhere up to 2^(1/256) from it."""
    from trainkernel_b200 import losses
    tops = torch.tensor([0.0, 1.7, -3.3, 1000.1, -60000.7, 65535.9, 70000.0, -1e9, 1e30], device="cuda")
    logits = (tops[:, None] + torch.zeros(9, 3001, device="cuda")).to(dtype)
    logits[:, 1000:] = -float("inf")
    targets = torch.full((9,), 5, dtype=torch.int64, device="cuda")
    logp, stats = losses._logprobs_launch(logits, targets, None, True)
    assert torch.equal(stats[:, 0], logits[:, 5].float())
    ratio = (stats[:, 1].double() / 1000).log2().abs()
    assert bool((ratio <= 1 / 256 + 16 * U).all())
    assert bool((ratio[(logits[:, 5] == 0) | (logits[:, 5].float().abs() > 65536)] <= 16 * U).all())
    assert bool(((-logp.double() - math.log(1000)).abs() <= 64 * U).all())


# -- constants inside a transform ----------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("layout", ["dense", "shifted"])
@pytest.mark.parametrize("long_way", [False, True])
def test_constant_logits_inside_a_transform(layout, long_way, monkeypatch):
    """The reference model's log-probabilities are computed inside the function that is differentiated, from logits that are not."""
    from trainkernel_b200 import operators
    logits, constant = noise((4, 6, 33), 1.0, 17)[:, :5], noise((4, 6, 33), 1.0, 18)[:, :5]
    if layout == "dense":
        logits, constant = logits.contiguous(), constant.contiguous()
    targets = torch.randint(0, 33, (4, 5), generator=torch.Generator(device="cuda").manual_seed(19), device="cuda")
    ref = tk.token_logprobs(constant, targets)
    if long_way:
        monkeypatch.setattr(operators, "fast", None)

    def of_everything(x):
        inside = tk.token_logprobs(constant, targets)
        sums = tk.preference_loss(constant, targets, ref[:, 0])[1]
        other, also, grad = tk.policy_loss_and_grad(constant, targets, inside, inside)
        scored, weighed = tk.token_logprobs_and_grad(constant, targets, inside)
        total = grad.float().sum() + weighed.float().sum() + tk.preference_loss_and_grad(constant, targets, sums)[0] + tk.policy_loss(constant, targets, also, scored)[0]
        return tk.policy_loss(x, targets, inside, torch.ones_like(inside), ref_logprobs=inside, kl_weight=0.1)[0] + other + 0.0 * total

    def directly(x):
        return tk.policy_loss(x, targets, ref, torch.ones_like(ref), ref_logprobs=ref, kl_weight=0.1)[0] + tk.policy_loss(constant, targets, ref, ref)[0]

    leaf = logits.clone().requires_grad_()
    value = directly(leaf)
    value.backward()
    grad, got = torch.func.grad_and_value(of_everything)(logits)
    torch.testing.assert_close(got, value.detach(), rtol=16 * U, atol=16 * U)
    torch.testing.assert_close(grad, leaf.grad, rtol=16 * U, atol=1e-30)
    torch.func.jvp(lambda y: y * tk.token_logprobs(constant, targets).sum(), (ref,), (ref,))
    torch.testing.assert_close(torch.vmap(lambda y: y + tk.token_logprobs(constant, targets)[0, 0])(ref[0]), ref[0] + ref[0, 0])
