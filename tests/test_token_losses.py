"""Token log-probabilities, policy loss and preference loss against a 64-bit statement of their formulas.

Bounds, with u = 2^-24 (half a step of FP32) and h = `torch.finfo(type).eps / 2` (half a step of the logits' type):

* A log-probability is (x_t - top) - log S.  The subtraction and the result are off by u each, relative to
  themselves.  S is a sum of at most V positive terms, added in runs of at most V / 256 and then in a tree of about
  ten levels: relative error at most (V / 256 + 10) u, plus 4 u for every term's exponential (the hardware's 2^x is
  good to 2^-22) and 2 u |x - top| e^-(top - x) <= u for its argument; log turns that into the same absolute error.
  Together u (2 |x_t - top| + 2 |log S| + V / 256 + 20).
* A gradient element is c (delta - p).  p = 2^((x - top) log2 e) / S has the relative error of the two exponentials
  (4 u each), of S (above) and of the argument (3 u |x - top|); c is off by what its formula loses (`slack`, given
  where it is used); then one rounding to the type, h relative, or half of its smallest step below that.
"""
import math

import pytest
import torch

import trainkernel_b200 as tk

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
gpu = pytest.mark.gpu


# -- 64-bit statements of the formulas -----------------------------------------------------------------------

def exact_logprobs(logits, targets, mask=None):
    logp = torch.log_softmax(logits.double(), -1).gather(-1, targets.long().unsqueeze(-1)).squeeze(-1)
    return logp if mask is None else torch.where(mask, logp, torch.zeros_like(logp))


def exact_policy(logits, targets, old, advantages, ref, mask, clip, kl_weight, average):
    """(loss, d loss / d logprob)."""
    logp = torch.log_softmax(logits.double(), -1).gather(-1, targets.long().unsqueeze(-1)).squeeze(-1)
    keep = torch.ones_like(targets, dtype=torch.bool) if mask is None else mask
    logp = torch.where(keep, logp, torch.zeros_like(logp)).requires_grad_()
    old, advantages = old.double(), advantages.double().expand(targets.shape)
    old = torch.where(keep, old, torch.zeros_like(old))
    ratio = torch.exp(logp - old)
    low, high = 1 - torch.tensor(clip[0], dtype=F32).double(), 1 + torch.tensor(clip[1], dtype=F32).double()
    bounded = torch.minimum(torch.maximum(ratio, low.to(ratio)), high.to(ratio))
    terms = -torch.where(ratio * advantages <= bounded * advantages, ratio * advantages, (bounded * advantages).detach())
    if ref is not None:
        away = torch.where(keep, ref.double(), torch.zeros_like(old)) - logp
        terms = terms + kl_weight * (torch.exp(away) - away - 1)
    if average == "tokens":
        weight = keep.double() / keep.sum().clamp(min=1)
    elif targets.dim() == 1:
        weight = keep.double() / keep.sum().clamp(min=1)
    else:
        weight = keep.double() / (keep.sum(1, keepdim=True).clamp(min=1) * targets.shape[0])
    loss = torch.where(keep, weight * terms, torch.zeros_like(terms)).sum()
    (slope,) = torch.autograd.grad(loss, logp)
    return loss.detach(), torch.where(keep, slope, torch.zeros_like(slope))


def exact_preference(logits, targets, reference, mask, beta, smoothing):
    """(loss, sums, d loss / d sums)."""
    sums = exact_logprobs(logits, targets, mask).sum(1).requires_grad_()
    n = sums.shape[0] // 2
    margin = sums - reference.double()
    z = beta * (margin[:n] - margin[n:])
    logsig = torch.nn.functional.logsigmoid
    loss = (-(1 - smoothing) * logsig(z) - smoothing * logsig(-z)).mean()
    (slope,) = torch.autograd.grad(loss, sums)
    return loss.detach(), sums.detach(), slope


def exact_grad(logits, targets, coefficients):
    x = logits.double()
    hot = torch.zeros_like(x).scatter_(-1, targets.long().unsqueeze(-1), 1.0)
    return coefficients.unsqueeze(-1) * (hot - torch.softmax(x, -1))


def assert_logprobs(got, logits, targets, mask=None):
    want = exact_logprobs(logits, targets, mask)
    assert got.dtype == F32 and got.shape == targets.shape
    x = logits.double()
    far = x.amax(-1) - x.gather(-1, targets.long().unsqueeze(-1)).squeeze(-1)
    log_sum = torch.logsumexp(x, -1) - x.amax(-1)
    bound = U * (2 * far + 2 * log_sum + logits.shape[-1] / 256 + 20)
    wrong = (got.double() - want).abs() > bound
    if mask is not None:
        assert bool((got[~mask] == 0).all())
        wrong &= mask
    assert not bool(wrong.any()), float(((got.double() - want).abs() / bound).nan_to_num().max())


def assert_grad(got, logits, targets, coefficients, slack):
    """`slack`: bound of the relative error of the coefficients."""
    assert got.dtype == logits.dtype and got.shape == logits.shape
    want = exact_grad(logits, targets, coefficients)
    x = logits.double()
    p = torch.softmax(x, -1)
    c = coefficients.abs().unsqueeze(-1)
    info = torch.finfo(logits.dtype)
    lost = U * (8 + logits.shape[-1] / 256 + 20 + 3 * (x.amax(-1, keepdim=True) - x))
    bound = c * p * lost + want.abs() * (slack + info.eps / 2 + 4 * U) + c * 2 * U * (want.abs() > p * c * 0.999) + info.smallest_normal * info.eps
    excess = (got.double() - want).abs() / bound.clamp(min=1e-300)
    assert bool(torch.isfinite(got.float()).all())
    assert float(excess.max()) <= 1.0, float(excess.max())


def make(shape, vocab, dtype, seed=0, *, layout="dense", spread=2.0, masked=False, target_dtype=torch.int64):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lead = list(shape)
    if layout == "dense":
        logits = torch.randn((*lead, vocab), generator=gen, device="cuda").mul_(spread).to(dtype)
    elif layout == "shift":                                   # logits[:, :-1] of a batch of longer sequences
        logits = torch.randn((lead[0], lead[1] + 1, vocab), generator=gen, device="cuda").mul_(spread).to(dtype)[:, :-1]
    elif layout == "pitch":                                   # rows of a wider buffer, at an odd offset
        logits = torch.randn((*lead, vocab + 5), generator=gen, device="cuda").mul_(spread).to(dtype)[..., 3:3 + vocab]
    else:                                                     # "swapped": [length, batch, vocab] in memory
        logits = torch.randn((lead[1], lead[0], vocab), generator=gen, device="cuda").mul_(spread).to(dtype).transpose(0, 1)
    targets = torch.randint(0, vocab, lead, generator=gen, device="cuda").to(target_dtype)
    if layout == "swapped":
        targets = targets.t().contiguous().t()
    mask = None
    if masked:
        mask = torch.rand(lead, generator=gen, device="cuda") < 0.6
        if len(lead) == 2 and lead[0] > 1:
            mask[-1] = False                                  # a sequence without a counted token
        logits = logits.clone() if layout == "dense" else logits
        logits.masked_fill_(~mask.unsqueeze(-1), float("nan"))
    return logits, targets, mask


def clean(logits, mask):
    """The logits without what excluded rows hold, for the statements in 64 bits."""
    return logits if mask is None else torch.where(mask.unsqueeze(-1), logits, torch.zeros_like(logits))


def noise(shape, scale, seed):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale


SHAPES = [
    ((1,), 1, F32, "dense"), ((1,), 2, BF16, "dense"), ((3,), 7, F16, "dense"), ((5,), 8, BF16, "dense"), ((2, 1), 33, F32, "dense"),
    ((1, 3), 511, BF16, "dense"), ((2, 5), 513, F32, "shift"), ((4, 7), 1000, BF16, "shift"), ((3, 4), 4099, F16, "shift"), ((2, 3), 4097, BF16, "pitch"),
    ((2, 9), 6007, F32, "pitch"), ((2, 3), 32000, BF16, "swapped"), ((1, 2), 50257, BF16, "shift"), ((2, 2), 50257, F32, "shift"), ((3,), 65537, F16, "dense"),
    ((2,), 128256, BF16, "dense"), ((1, 2), 151937, F32, "dense"), ((1,), 262144, BF16, "dense"), ((1,), 300001, BF16, "pitch"), ((257, 3), 129, BF16, "dense"),
    ((700,), 24, F32, "dense"), ((31, 40), 520, F16, "shift"), ((40, 30), 20011, BF16, "shift"), ((500,), 33000, F32, "dense"), ((9, 100), 70001, F16, "shift"),
]
IDS = [f"{'x'.join(map(str, s))}x{v}-{str(d).split('.')[1]}-{lay}" for s, v, d, lay in SHAPES]


@gpu
@pytest.mark.parametrize("shape,vocab,dtype,layout", SHAPES, ids=IDS)
@pytest.mark.parametrize("masked", [False, True])
def test_logprobs_and_weighted_gradient(shape, vocab, dtype, layout, masked):
    logits, targets, mask = make(shape, vocab, dtype, 1, layout=layout, masked=masked, target_dtype=torch.int32 if vocab % 2 else torch.int64)
    assert_logprobs(tk.token_logprobs(logits, targets, mask=mask), clean(logits, mask), targets, mask)
    weights = noise(shape, 1.0, 2)
    logp, grad = tk.token_logprobs_and_grad(logits, targets, weights, mask=mask, grad_scale=0.5)
    assert_logprobs(logp, clean(logits, mask), targets, mask)
    counted = weights.double() * 0.5 if mask is None else torch.where(mask, weights.double() * 0.5, 0.0)
    assert_grad(grad, clean(logits, mask), targets, counted, 2 * U)
    if mask is not None:
        assert bool((grad[~mask] == 0).all())


@gpu
@pytest.mark.parametrize("shape,vocab,dtype,layout", [s for s in SHAPES if s[1] > 2], ids=[i for i, s in zip(IDS, SHAPES) if s[1] > 2])
@pytest.mark.parametrize("masked,average,kl", [(False, "tokens", 0.0), (True, "tokens", 0.1), (True, "sequences", 0.02)])
def test_policy_loss_and_gradient(shape, vocab, dtype, layout, masked, average, kl):
    logits, targets, mask = make(shape, vocab, dtype, 3, layout=layout, masked=masked)
    near = exact_logprobs(clean(logits, mask), targets, mask).float()
    old, ref = near + noise(shape, 0.2, 4), near + noise(shape, 0.3, 5) if kl else None
    advantages = noise((*shape[:-1], 1), 1.0, 6) if len(shape) == 2 else noise(shape, 1.0, 6)       # one per sequence, broadcast
    clip = (0.2, 0.3)
    # keep ratios off the clip's borders: there the slope depends on the last bit
    ratio = torch.exp(near - old)
    border = (ratio - 0.8).abs().minimum((ratio - 1.3).abs()) < 1e-3
    old = torch.where(border, near + 0.05, old)
    loss, logp, grad = tk.policy_loss_and_grad(logits, targets, old, advantages, ref_logprobs=ref, mask=mask, clip=clip, kl_weight=kl, average=average, grad_scale=2.0)
    want, slope = exact_policy(clean(logits, mask), targets, old, advantages, ref, mask, clip, kl, average)
    assert_logprobs(logp, clean(logits, mask), targets, mask)
    # a log-probability is off by d (bound above); the ratio and the KL slope by d + 8 u relative; slope also cancels between its two parts
    x = clean(logits, mask).double()
    d = float(U * (4 * (x.amax(-1) - x.amin(-1)).max() + vocab / 256 + 40))
    parts = (advantages.abs().double().expand(shape) * 1.5 + kl * 4).max()
    assert abs(float(loss) - float(want)) <= float(parts) * (d + 16 * U) * 1.5 + 4 * U
    scaled = slope * 2.0
    assert_slope_grad(grad, clean(logits, mask), targets, scaled, mask, float(parts) * (d + 16 * U), average, shape)
    only, logp2 = tk.policy_loss(logits, targets, old, advantages, ref_logprobs=ref, mask=mask, clip=clip, kl_weight=kl, average=average)
    # the form without a gradient may split a row between other threads and so add its terms in another order: it keeps to
    # the same bounds, not to the same bits
    assert_logprobs(logp2, clean(logits, mask), targets, mask)
    assert abs(float(only) - float(want)) <= float(parts) * (d + 16 * U) * 1.5 + 4 * U


def assert_slope_grad(got, logits, targets, scaled, mask, error, average, shape):
    """The coefficient of every row may be off by `error` times the row's weight: bound it row by row."""
    keep = torch.ones(shape, dtype=torch.bool, device="cuda") if mask is None else mask
    if average == "tokens" or len(shape) == 1:
        weight = keep.double() / keep.sum().clamp(min=1)
    else:
        weight = keep.double() / (keep.sum(1, keepdim=True).clamp(min=1) * shape[0])
    want = exact_grad(logits, targets, scaled)
    x = logits.double()
    p = torch.softmax(x, -1)
    hot = torch.zeros_like(x).scatter_(-1, targets.unsqueeze(-1), 1.0)
    info = torch.finfo(logits.dtype)
    lost = U * (28 + logits.shape[-1] / 256 + 3 * (x.amax(-1, keepdim=True) - x))
    c = scaled.abs().unsqueeze(-1)
    bound = (c * p * lost + c * 4 * U * hot + 2 * (weight * error).unsqueeze(-1) * (p + hot) + want.abs() * (info.eps / 2 + 8 * U)
             + info.smallest_normal * info.eps)
    assert bool(torch.isfinite(got.float()).all())
    assert float(((got.double() - want).abs() / bound).max()) <= 1.0
    assert bool((got[~keep] == 0).all())


@gpu
@pytest.mark.parametrize("pairs,length,vocab,dtype,layout", [(1, 1, 5, F32, "dense"), (2, 33, 4099, F16, "dense"), (3, 17, 1000, BF16, "shift"),
                                                             (2, 9, 50257, BF16, "shift"), (4, 300, 64, F32, "dense"), (1, 5, 4097, F32, "pitch"), (150, 3, 40, F32, "swapped")])
@pytest.mark.parametrize("masked,smoothing", [(False, 0.0), (True, 0.1)])
def test_preference_loss_and_gradient(pairs, length, vocab, dtype, layout, masked, smoothing):
    logits, targets, mask = make((2 * pairs, length), vocab, dtype, 7, layout=layout, masked=masked)
    data = clean(logits, mask)
    reference = exact_logprobs(data, targets, mask).sum(1).float() + noise((2 * pairs,), 4.0, 8)
    loss, sums, grad = tk.preference_loss_and_grad(logits, targets, reference, mask=mask, beta=0.2, label_smoothing=smoothing)
    beta = float(torch.tensor(0.2, dtype=F32))
    soft = float(torch.tensor(smoothing, dtype=F32))
    want, want_sums, slope = exact_preference(data, targets, reference, mask, beta, soft)
    x = data.double()
    d = float(U * (2 * (x.amax(-1) - x.amin(-1)).max() + 2 * math.log(vocab) + vocab / 256 + 20))       # of one log-probability
    assert bool(((sums.double() - want_sums).abs() <= length * d + want_sums.abs() * U).all())
    # z is off by beta 2 length d and its own rounding; softplus and sigmoid have slopes of at most 1 and 1/4
    z_error = beta * 2 * length * d + 2 * U * float((want_sums - reference.double()).abs().max()) * beta * 2
    assert abs(float(loss) - float(want)) <= z_error + 16 * U * (1 + abs(float(want)))
    coefficients = slope[:, None].expand(targets.shape)
    if mask is not None:
        coefficients = torch.where(mask, coefficients, 0.0)
    error = beta / pairs * (z_error / 4 + 8 * U)
    hot = torch.zeros_like(x).scatter_(-1, targets.unsqueeze(-1), 1.0)
    p = torch.softmax(x, -1)
    target = exact_grad(data, targets, coefficients)
    info = torch.finfo(dtype)
    c = coefficients.abs().unsqueeze(-1)
    lost = U * (28 + vocab / 256 + 3 * (x.amax(-1, keepdim=True) - x))
    bound = c * p * lost + c * 4 * U * hot + error * (p + hot) * (c > 0) + target.abs() * (info.eps / 2 + 8 * U) + info.smallest_normal * info.eps
    assert float(((grad.double() - target).abs() / bound).max()) <= 1.0
    only, sums2 = tk.preference_loss(logits, targets, reference, mask=mask, beta=0.2, label_smoothing=smoothing)
    assert torch.equal(only, loss) and torch.equal(sums, sums2)


@gpu
@pytest.mark.parametrize("vocab,times", [(1003, 1), (1003, 40), (40001, 1), (40001, 40), (70001, 40)])
def test_masked_vocabulary_and_extreme_logits(vocab, times):
    """Few rows and many, short and long: every block shape and the split rows."""
    lowest, inf = torch.finfo(BF16).min, float("inf")
    for dtype in (F32, BF16, F16):
        low = torch.finfo(dtype).min
        rows = torch.zeros((6, vocab), dtype=dtype, device="cuda")
        rows[0, 100:] = -inf                                   # part of the vocabulary excluded
        rows[1, :900] = low                                    # excluded with the type's lowest value, the target among them
        rows[2] = low                                          # everything excluded that way: uniform
        rows[3] = torch.finfo(dtype).max
        rows[4] = -inf                                         # nothing left: not a number
        rows[5, 7] = inf
        targets = torch.tensor([3, 950, 10, 0, 1, 2], device="cuda")
        weights = torch.ones(6, device="cuda")
        every = tk.token_logprobs_and_grad(rows.repeat(times, 1), targets.repeat(times), weights.repeat(times))
        logp, grad = every[0][-6:], every[1][-6:]
        if times > 1:
            assert torch.equal(every[0][:6].nan_to_num(), logp.nan_to_num()) and torch.equal(every[1][:6].nan_to_num(), grad.nan_to_num())
        want = torch.log_softmax(rows.double(), -1).gather(1, targets[:, None])[:, 0]
        assert bool(torch.isnan(want[4:]).all()) and bool(torch.isnan(logp[4:]).all())
        torch.testing.assert_close(logp[:4].double(), want[:4], rtol=8 * U, atol=(32 + vocab / 256) * U)
        expected = exact_grad(rows[:4], targets[:4], weights[:4].double())
        torch.testing.assert_close(grad[:4].double(), expected, rtol=torch.finfo(dtype).eps / 2 + (32 + vocab / 256) * U, atol=torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps)
        assert bool(torch.isnan(grad[4:]).all())
        # a target whose logit is -inf has log-probability -inf, and a gradient that is finite
        logp, grad = tk.token_logprobs_and_grad(rows[:1], torch.tensor([500], device="cuda"), weights[:1])
        assert float(logp) == -inf and bool(torch.isfinite(grad.float()).all())
    assert lowest < -3e38


@gpu
def test_targets_outside_the_vocabulary_read_nothing_and_show():
    logits, _, _ = make((4,), 100, F32, 9)
    targets = torch.tensor([-1, 100, 2 ** 40, 5], device="cuda")
    logp, grad = tk.token_logprobs_and_grad(logits, targets, torch.ones(4, device="cuda"))
    assert bool(torch.isnan(logp[:3]).all()) and bool(torch.isnan(grad[:3]).all())
    assert bool(torch.isfinite(logp[3])) and bool(torch.isfinite(grad[3]).all())
    masked = tk.token_logprobs(logits, targets, mask=torch.tensor([False, False, False, True], device="cuda"))
    assert masked[:3].tolist() == [0.0, 0.0, 0.0] and bool(torch.isfinite(masked[3]))


@gpu
def test_a_row_of_nan_stays_in_its_row_and_in_the_loss():
    logits, targets, _ = make((2, 3), 77, F32, 10)
    logits[1, 1, 5] = float("nan")
    old = torch.zeros((2, 3), device="cuda")
    loss, logp, grad = tk.policy_loss_and_grad(logits, targets, old, torch.ones_like(old))
    assert bool(torch.isnan(loss)) and bool(torch.isnan(logp[1, 1])) and bool(torch.isnan(grad[1, 1]).all())
    assert int(torch.isnan(logp).sum()) == 1 and int(torch.isnan(grad).sum()) == 77
    _, sums, grad = tk.preference_loss_and_grad(logits, targets, torch.zeros(2, device="cuda"))
    assert bool(torch.isnan(sums[1])) and bool(torch.isfinite(sums[0]))


@gpu
def test_nothing_counted_gives_zero():
    logits, targets, _ = make((2, 3), 50, BF16, 11)
    mask = torch.zeros((2, 3), dtype=torch.bool, device="cuda")
    logits.fill_(float("nan"))
    old = torch.full((2, 3), float("nan"), device="cuda")
    for average in ("tokens", "sequences"):
        loss, logp, grad = tk.policy_loss_and_grad(logits, targets, old, old, mask=mask, average=average)
        assert float(loss) == 0 and bool((logp == 0).all()) and bool((grad == 0).all())
    loss, sums, grad = tk.preference_loss_and_grad(logits, targets, torch.zeros(2, device="cuda"), mask=mask)
    assert abs(float(loss) - math.log(2)) <= 4 * U and bool((sums == 0).all()) and bool((grad == 0).all())


@gpu
def test_gradients_agree_with_differences():
    logits, targets, mask = make((4, 3), 11, F32, 12, masked=False)
    mask = torch.rand((4, 3), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.8
    old = tk.token_logprobs(logits, targets) + noise((4, 3), 0.05, 13)
    ref, adv = old + noise((4, 3), 0.2, 14), noise((4, 1), 1.0, 15)
    reference = noise((4,), 1.0, 16)
    forms = [
        lambda x: tk.policy_loss_and_grad(x, targets, old, adv, ref_logprobs=ref, mask=mask, kl_weight=0.1, average="sequences"),
        lambda x: tk.preference_loss_and_grad(x, targets, reference, mask=mask, beta=0.5, label_smoothing=0.1),
    ]
    for form in forms:
        grad = form(logits)[2]
        direction = noise(logits.shape, 1.0, 17)
        step = 2.0 ** -6
        up, down = form(logits + step * direction)[0].double(), form(logits - step * direction)[0].double()
        slope = float((up - down) / (2 * step))
        # a central difference is off by step^2 times the third derivative over 6, here of order 10, and by 2 u |loss| / step
        assert abs(slope - float((grad.double() * direction.double()).sum())) <= step ** 2 * 10 + 64 * U * (1 + abs(float(up))) / step


@gpu
def test_the_three_ways_to_a_gradient_agree():
    logits, targets, mask = make((3, 5), 777, BF16, 18, masked=True)
    old, adv = noise((3, 5), 0.3, 19) - 7, noise((3, 1), 1.0, 20)
    loss, _, grad = tk.policy_loss_and_grad(logits, targets, old, adv, mask=mask, grad_scale=3.0)

    def f(x):
        return 3.0 * tk.policy_loss(x, targets, old, adv, mask=mask)[0]

    transformed = torch.func.grad(f)(logits)
    leaf = logits.clone().requires_grad_()
    value = f(leaf)
    value.backward()
    # the same coefficients and statistics, added in the same order: at most the rounding of one product apart
    for other in (transformed, leaf.grad):
        torch.testing.assert_close(other.float(), grad.float(), rtol=torch.finfo(BF16).eps, atol=1e-30)
    assert abs(float(value.detach()) / 3 - float(loss)) <= 4 * U * abs(float(loss))
    leaf.grad = None
    out = tk.token_logprobs(leaf, targets, mask=mask)
    weights = noise((3, 5), 1.0, 21)
    (out * weights).sum().backward()
    torch.testing.assert_close(leaf.grad.float(), tk.token_logprobs_and_grad(logits, targets, weights, mask=mask)[1].float(), rtol=torch.finfo(BF16).eps, atol=1e-30)
    pair, ids, keep = make((4, 5), 333, F32, 22, masked=True)
    reference = noise((4,), 1.0, 23)
    want = tk.preference_loss_and_grad(pair, ids, reference, mask=keep)[2]
    got = torch.func.grad(lambda x: tk.preference_loss(x, ids, reference, mask=keep)[0])(pair)
    torch.testing.assert_close(got, want, rtol=8 * U, atol=0.0)


@gpu
def test_second_derivatives_are_refused():
    logits, targets, _ = make((3,), 20, F32, 24)
    leaf = logits.requires_grad_()
    (grad,) = torch.autograd.grad(tk.token_logprobs(leaf, targets).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        grad.sum().backward()


@gpu
def test_captured_calls_follow_their_inputs_and_share_nothing():
    logits, targets, mask = make((4, 6), 2000, BF16, 25)
    old, adv = noise((4, 6), 0.3, 26) - 8, noise((4, 1), 1.0, 27)
    reference = noise((4,), 1.0, 28)

    def policy():
        return tk.policy_loss_and_grad(logits, targets, old, adv)

    def preference():
        return tk.preference_loss_and_grad(logits, targets, reference)

    graphs = []
    for call in (policy, preference, policy):
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out, call))
    fresh, _, _ = make((4, 6), 2000, BF16, 29)
    logits.copy_(fresh)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):                                     # replayed side by side: each has a workspace of its own
        for stream, (graph, _, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for graph, out, call in graphs:
        for a, b in zip(out, call()):
            assert torch.equal(a, b)


@gpu
def test_calls_on_side_streams_and_repeated_calls_are_identical():
    logits, targets, _ = make((8, 16), 5000, F32, 30)
    old, adv = noise((8, 16), 0.3, 31) - 8, noise((8, 1), 1.0, 32)
    want = tk.policy_loss_and_grad(logits, targets, old, adv)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    results = []
    for _ in range(4):
        for stream in streams:
            with torch.cuda.stream(stream):
                results.append(tk.policy_loss_and_grad(logits, targets, old, adv))
    torch.cuda.synchronize()
    for result in results:
        for a, b in zip(result, want):
            assert torch.equal(a, b)


@gpu
def test_autograd_history_under_capture_is_refused():
    logits, targets, _ = make((3,), 20, F32, 33)
    leaf = logits.clone().requires_grad_()
    tk.token_logprobs(leaf, targets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="autograd history cannot be recorded"):
            tk.token_logprobs(leaf, targets)
        logp = tk.token_logprobs(logits, targets)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(logp, tk.token_logprobs(logits, targets))


@gpu
def test_tensor_scale_is_read_by_every_replay():
    logits, targets, _ = make((3, 2), 40, F32, 34)
    weights, scale = torch.ones(2, device="cuda"), torch.full((), 2.0, device="cuda")
    base = tk.token_logprobs_and_grad(logits, targets, weights)[1]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, grad = tk.token_logprobs_and_grad(logits, targets, weights, grad_scale=scale)
    for value in (2.0, 0.25):
        scale.fill_(value)
        graph.replay()
        assert torch.equal(grad, base * value)


@gpu
def test_offsets_beyond_32_bits():
    """A buffer of more than 2^32 logits: the last rows of a batch whose strides reach behind it."""
    vocab, batch = 1031, 3
    pitch = (2 ** 32 // 2 + 4096) // 1                       # elements between sequences: the third starts behind 2^32
    whole = torch.empty(2 * pitch + 4 * vocab, dtype=F16, device="cuda")
    logits = whole.as_strided((batch, 4, vocab), (pitch, vocab, 1))
    for b in range(batch):
        logits[b].normal_(generator=torch.Generator(device="cuda").manual_seed(b))
    targets = torch.randint(0, vocab, (batch, 4), device="cuda")
    weights = torch.ones(4, device="cuda")
    logp, grad = tk.token_logprobs_and_grad(logits, targets, weights)
    small = torch.stack([logits[b].clone() for b in range(batch)])
    assert_logprobs(logp, small, targets)
    assert_grad(grad, small, targets, weights.double().expand(batch, 4), 2 * U)


@gpu
def test_short_and_long_way_to_a_launch_agree(monkeypatch):
    from trainkernel_b200 import operators
    logits, targets, mask = make((2, 3), 50, F32, 39)
    old, one = torch.zeros((2, 3), device="cuda"), torch.ones((2, 1), device="cuda")
    tk.token_logprobs(logits, targets)
    for answer in (operators.fast.token_logprobs(logits, targets, None), operators.fast.token_logprobs_and_grad(logits, targets, old, None, 1.0),
                   operators.fast.policy_loss(logits, targets, old, one, None, None, (0.2, 0.2), 0.0, "tokens", 1.0),
                   operators.fast.preference_loss(logits, targets, one[:, 0], None, 0.1, 0.0, None)):
        assert answer is not None                              # an ordinary call does go the short way
    assert operators.fast.token_logprobs(logits.requires_grad_(), targets, None) is None
    results = []
    for long_way in (False, True):
        if long_way:
            monkeypatch.setattr(operators, "fast", None)
        taken = []
        for shape, vocab, dtype, layout, masked in (((4, 6), 1000, BF16, "dense", True), ((4, 6), 777, F32, "shift", False), ((2, 8), 40, F16, "pitch", True), ((12,), 129, F32, "dense", False)):
            logits, targets, mask = make(shape, vocab, dtype, 40, layout=layout, masked=masked)
            old, adv, reference = noise(shape, 0.3, 41) - 6, noise((*shape[:-1], 1), 1.0, 42) if len(shape) == 2 else noise(shape, 1.0, 42), noise(shape[:1], 1.0, 43)
            taken += [tk.token_logprobs(logits, targets, mask=mask), *tk.token_logprobs_and_grad(logits, targets, old, mask=mask, grad_scale=2)]
            taken += [*tk.policy_loss(logits, targets, old, adv, mask=mask), *tk.policy_loss_and_grad(logits, targets, old, adv, mask=mask, ref_logprobs=old, kl_weight=1)]
            if len(shape) == 2:
                taken += [*tk.preference_loss(logits, targets, reference, mask=mask), *tk.preference_loss_and_grad(logits, targets, reference, mask=mask, grad_scale=0.5)]
        results.append(taken)
    for a, b in zip(*results):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)


@gpu
def test_transformed_constants_are_refused():
    logits, targets, _ = make((3,), 20, F32, 44)
    with pytest.raises(ValueError, match="detach"):
        torch.func.grad(lambda a: tk.policy_loss_and_grad(logits, targets, torch.zeros(3, device="cuda"), a)[0])(torch.ones(3, device="cuda"))


@gpu
def test_gradients_behind_two_to_the_31_elements():
    rows, vocab = 20000, 120000                               # 2.4e9 logits, 4.8 GB, and as much for the gradient
    logits = torch.empty((rows, vocab), dtype=BF16, device="cuda")
    logits.normal_(0.0, 2.0, generator=torch.Generator(device="cuda").manual_seed(45))
    targets = torch.randint(0, vocab, (rows,), device="cuda")
    mask = torch.zeros(rows, dtype=torch.bool, device="cuda")
    mask[::997] = mask[-3:] = True
    logp, grad = tk.token_logprobs_and_grad(logits, targets, torch.ones(1, device="cuda"), mask=mask)
    at = torch.nonzero(mask)[:, 0]
    assert_logprobs(logp[at], logits[at], targets[at])
    assert_grad(grad[at], logits[at], targets[at], torch.ones(len(at), dtype=torch.float64, device="cuda"), 2 * U)
    assert bool((grad[-5] == 0).all()) and bool((logp[~mask] == 0).all())


@gpu
def test_inference_mode_and_parameters_as_logits():
    logits, targets, _ = make((6,), 700, F32, 46)
    want = tk.token_logprobs(logits, targets)
    with torch.inference_mode():
        assert torch.equal(tk.token_logprobs(logits, targets), want)
        inside = logits.clone()
        assert torch.equal(tk.token_logprobs(inside, targets), want)
        assert torch.equal(tk.policy_loss_and_grad(inside, targets, want, want)[1], want)
    leaf = torch.nn.Parameter(logits)
    with torch.no_grad():
        assert not tk.token_logprobs(leaf, targets).requires_grad
    assert not tk.token_logprobs_and_grad(leaf, targets, want)[1].requires_grad
    assert tk.token_logprobs(leaf, targets).requires_grad


@gpu
def test_logits_of_one_element_of_memory():
    """Expanded logits: every row the same memory; the gradient has memory of its own."""
    base = torch.randn((1, 1, 300), device="cuda")
    logits, targets = base.expand(3, 4, 300), torch.randint(0, 300, (3, 4), device="cuda")
    logp, grad = tk.token_logprobs_and_grad(logits, targets, torch.ones(4, device="cuda"))
    assert_logprobs(logp, logits, targets)
    assert_grad(grad, logits, targets, torch.ones((3, 4), dtype=torch.float64, device="cuda"), 2 * U)


# -- refusals (no GPU) ---------------------------------------------------------------------------------------

def _cpu(shape=(2, 3), vocab=5, device="cpu"):
    return torch.randn(*shape, vocab, device=device), torch.zeros(shape, dtype=torch.int64, device=device), torch.zeros(shape, device=device)


ON = pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])


def on_device(device):
    """On the GPU a first good call makes the compiled host path the one that is asked first."""
    if device == "cuda":
        logits, targets, _ = _cpu(device="cuda")
        tk.token_logprobs(logits, targets)
    return device


@ON
def test_refusals_of_rows(device):
    logits, targets, old = _cpu(device=on_device(device))
    bad = [
        (lambda: tk.token_logprobs(logits.double(), targets), "float32, float16 or bfloat16"),
        (lambda: tk.token_logprobs(logits, targets.float()), "int64 or int32"),
        (lambda: tk.token_logprobs(logits[0, 0], targets[0, 0]), "must be"),
        (lambda: tk.token_logprobs(logits[None], targets[None]), "must be"),
        (lambda: tk.token_logprobs(logits, targets[:, :2]), "without the vocabulary"),
        (lambda: tk.token_logprobs(logits[:, :0], targets[:, :0]), "empty"),
        (lambda: tk.token_logprobs(logits[..., :0], targets), "empty"),
        (lambda: tk.token_logprobs(logits.transpose(1, 2).contiguous().transpose(1, 2), targets), "contiguous"),
        (lambda: tk.token_logprobs(logits, targets, mask=torch.ones(2, 3, device=device)), "boolean"),
        (lambda: tk.token_logprobs(logits, targets, mask=torch.ones(2, 1, dtype=torch.bool, device=device)), "shape"),
        (lambda: tk.token_logprobs(logits, targets.to("meta")), "one device"),
        (lambda: tk.token_logprobs_and_grad(logits, targets, old.double()), "float32"),
        (lambda: tk.token_logprobs_and_grad(logits, targets, torch.zeros(7, device=device)), "broadcast"),
        (lambda: tk.token_logprobs_and_grad(logits, targets, old.requires_grad_()), "detach"),
        (lambda: tk.token_logprobs_and_grad(logits, targets, torch.zeros(3, device=device), grad_scale="big"), "grad_scale"),
        (lambda: tk.token_logprobs_and_grad(logits, targets, torch.zeros(3, device=device), grad_scale=torch.ones(2, device=device)), "grad_scale"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(TypeError, match="tensors"):
        tk.token_logprobs([1.0], targets)
    with pytest.raises(TypeError, match="must be a tensor"):
        tk.token_logprobs_and_grad(logits, targets, 1.0)


@ON
def test_refusals_of_the_losses(device):
    logits, targets, old = _cpu(device=on_device(device))
    bad = [
        (lambda: tk.policy_loss(logits, targets, old, old, kl_weight=0.1), "needs ref_logprobs"),
        (lambda: tk.policy_loss(logits, targets, old, old, kl_weight=-1.0, ref_logprobs=old), "kl_weight"),
        (lambda: tk.policy_loss(logits, targets, old, old, kl_weight=float("nan"), ref_logprobs=old), "kl_weight"),
        (lambda: tk.policy_loss(logits, targets, old, old, clip=0.2), "pair"),
        (lambda: tk.policy_loss(logits, targets, old, old, clip=(1.5, 0.2)), "clip below"),
        (lambda: tk.policy_loss(logits, targets, old, old, average="rows"), "average"),
        (lambda: tk.policy_loss(logits, targets, old, old.half()), "float32"),
        (lambda: tk.policy_loss_and_grad(logits, targets, old, torch.zeros(3, 2, device=device)), "broadcast"),
        (lambda: tk.preference_loss(logits[:1], targets[:1], torch.zeros(1, device=device)), "even number"),
        (lambda: tk.preference_loss(logits[0], targets[0], torch.zeros(3, device=device)), "sequences, length, vocab"),
        (lambda: tk.preference_loss(logits, targets, old), "one summed"),
        (lambda: tk.preference_loss(logits, targets, torch.zeros(2, device=device), beta=-0.1), "beta"),
        (lambda: tk.preference_loss(logits, targets, torch.zeros(2, device=device), label_smoothing=1.5), "label_smoothing"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()


def test_tensors_on_the_host_are_refused():
    logits, targets, old = _cpu()
    for call in (lambda: tk.token_logprobs(logits, targets), lambda: tk.policy_loss_and_grad(logits, targets, old, old),
                 lambda: tk.preference_loss(logits, targets, torch.zeros(2)), lambda: torch.func.grad(lambda x: tk.token_logprobs(x, targets).sum())(logits)):
        with pytest.raises(RuntimeError, match="sm_100a GPU required"):
            call()
