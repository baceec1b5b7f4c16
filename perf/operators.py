"""Cases of the language-model operators: token log-probabilities, the clipped policy loss, the preference loss and AdamW.

`run` computes an operator in its plain form (elementary PyTorch operations in 32 bits) or, with `own` set, through this
package's operators on the same inputs; `exact` computes the same outputs in 64 bits from the definitions.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CLIP = (0.2, 0.28)
KL_WEIGHT = 0.05
BETA = 0.1
SMOOTHING = 0.05
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01
BLOCK = 256                    # elements that share one scale when the moments are held in 8 bits
SLOT = 256                     # every tensor starts at a multiple of this many elements of the flat buffers
E4M3_MAX = 448.0


# -- cases ---------------------------------------------------------------------------------------------------

def listed():
    return [
        # scoring one token of each of a few decoded sequences
        {"name": "logprobs decode", "op": "logprobs", "grad": False, "batch": 8, "length": 1, "vocab": 32000, "dtype": "bf16", "shift": False, "masked": False},
        # scoring whole responses under a large vocabulary (the reference or old policy of a post-training step)
        {"name": "logprobs scoring", "op": "logprobs", "grad": False, "batch": 8, "length": 1024, "vocab": 128256, "dtype": "bf16", "shift": False, "masked": False},
        # weighted cross entropy of a language model with an odd vocabulary in 32 bits, next-token shifted
        {"name": "cross entropy fp32", "op": "logprobs", "grad": True, "batch": 4, "length": 511, "vocab": 50257, "dtype": "fp32", "shift": True, "masked": True},
        # a policy step on short answers with a small action vocabulary: latency counts
        {"name": "policy short", "op": "policy", "batch": 16, "length": 16, "vocab": 1000, "dtype": "fp32", "shift": False, "masked": False, "average": "tokens"},
        # a padded batch of sampled answers of different lengths
        {"name": "policy padded", "op": "policy", "batch": 16, "length": 500, "vocab": 32000, "dtype": "bf16", "shift": True, "masked": True, "average": "sequences"},
        # a long-context policy step under a large vocabulary
        {"name": "policy large", "op": "policy", "batch": 2, "length": 4096, "vocab": 128256, "dtype": "bf16", "shift": False, "masked": True, "average": "tokens"},
        # a few short pairs of a byte-pair vocabulary of odd size
        {"name": "preference short", "op": "preference", "batch": 8, "length": 33, "vocab": 4099, "dtype": "fp16", "shift": False, "masked": True},
        # a preference step on padded answers with an odd vocabulary
        {"name": "preference padded", "op": "preference", "batch": 16, "length": 512, "vocab": 50257, "dtype": "bf16", "shift": True, "masked": True},
        # update of the tiny online model (128-256-128)
        {"name": "adamw tiny", "op": "adamw", "bits": 32, "sizes": "32768,256,32768,128", "grads": "fp32", "params": "fp32"},
        # update of a model of many tensors of very different sizes, gradients of 16 bits
        {"name": "adamw many", "op": "adamw", "bits": 32, "sizes": ",".join(["1024," + "1048576," * 4 + "1024," + "2883584," * 2 + "2883584"] * 12), "grads": "bf16", "params": "fp32"},
        # update of the small model (1024-2048-2048-1024) with moments of 8 bits
        {"name": "adamw8 small", "op": "adamw", "bits": 8, "sizes": "2097152,2048,4194304,2048,2097152,1024", "grads": "fp32", "params": "fp32"},
        # update of the medium model (4096-8192-8192-8192-4096) with moments of 8 bits
        {"name": "adamw8 medium", "op": "adamw", "bits": 8, "sizes": "33554432,8192,67108864,8192,67108864,8192,33554432,4096", "grads": "fp32", "params": "fp32"},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "adamw"])
    if op == "adamw":
        total, count = _log_uniform(rng, 2000, 120_000_000), _log_uniform(rng, 1, 200)
        cuts = [rng.random() ** 2 + 1e-4 for _ in range(count)]
        sizes = [max(1, int(total * c / sum(cuts))) for c in cuts]
        return {"op": op, "bits": rng.choice([32, 8]), "sizes": ",".join(str(n) for n in sizes),
                "grads": rng.choice(["fp32", "bf16"]), "params": rng.choice(["fp32", "fp32", "bf16"])}
    vocab = _log_uniform(rng, 500, 200_000)
    if rng.random() < 0.5:
        vocab = -(-vocab // 64) * 64
    rows = max(2, min(16384, _log_uniform(rng, 2, 400_000_000 // vocab)))
    batch = min(64, _log_uniform(rng, 1, rows))
    batch += batch % 2 if op == "preference" else 0
    case = {"op": op, "batch": batch, "length": max(1, rows // batch), "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "shift": rng.random() < 0.3, "masked": rng.random() < 0.7}
    if op == "logprobs":
        case["grad"] = rng.random() < 0.5
    if op == "policy":
        case["average"] = rng.choice(["tokens", "sequences"])
    return case


# -- inputs --------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _prepare_adamw(case, seed):
    gen = _generator(seed)
    sizes = [int(n) for n in case["sizes"].split(",")]
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += -(-n // SLOT) * SLOT
    inside = torch.zeros(total, device="cuda")
    for a, n in zip(starts, sizes):
        inside[a:a + n] = 1.0

    def normal(scale):
        return torch.randn(total, generator=gen, device="cuda") * scale * inside

    # gradients whose sizes differ by orders of magnitude from weight to weight, and moments as after many such steps
    size = torch.exp(torch.randn(total, generator=gen, device="cuda") - 6.0)
    grads = (normal(1.0) * size).to(DTYPES[case["grads"]])
    params = normal(0.02).to(DTYPES[case["params"]])
    mean = normal(0.3) * size
    square = size * size * (0.5 + torch.rand(total, generator=gen, device="cuda")) * inside
    step = 1 + seed % 5000
    s = {"op": "adamw", "bits": case["bits"], "params": params, "grads": grads, "step": torch.full((), step, dtype=torch.int64, device="cuda")}
    if case["bits"] == 8:
        s["mean"], s["mean_scale"] = _to_nearest(mean)
        s["root"], s["root_scale"] = _to_nearest(square.sqrt())
    else:
        s["mean"], s["square"] = mean, square
    if own:
        import trainkernel_b200 as tk
        views = [[flat[a:a + n] for a, n in zip(starts, sizes)] for flat in (params, grads)]
        s["views"] = views
        s["optimizer"] = tk.AdamW(lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"])
        s["state"] = s["optimizer"].init(views[0])
        s["state"].set_step(step)
        s["state"].exp_avg.copy_(s["mean"])
        if case["bits"] == 8:
            s["state"].exp_avg_scale.copy_(s["mean_scale"])
            s["state"].exp_avg_root.copy_(s["root"])
            s["state"].exp_avg_root_scale.copy_(s["root_scale"])
        else:
            s["state"].exp_avg_sq.copy_(s["square"])
    return s


def _to_nearest(values):
    blocks = values.view(-1, BLOCK)
    top = blocks.abs().amax(1)
    factor = torch.where(top > 0, E4M3_MAX / top, torch.zeros_like(top))
    return (blocks * factor[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(-1), top / E4M3_MAX


def prepare(case, seed):
    if case["op"] == "adamw":
        return _prepare_adamw(case, seed)
    gen = _generator(seed)
    batch, length, vocab = case["batch"], case["length"], case["vocab"]
    extra = 1 if case["shift"] else 0
    whole = torch.empty((batch, length + extra, vocab), dtype=DTYPES[case["dtype"]], device="cuda")
    whole.normal_(0.0, 2.0, generator=gen)
    logits = whole[:, :length] if extra else whole
    ids = torch.randint(0, vocab, (batch, length + extra), generator=gen, device="cuda")
    targets = ids[:, extra:]
    # a sampled token is a likely one: lift each target's logit
    lift = torch.randn((batch, length, 1), generator=gen, device="cuda") + math.log(vocab)
    logits.scatter_(2, targets[:, :, None], lift.to(logits.dtype))
    s = {"op": case["op"], "grad": case.get("grad", True), "logits": logits, "targets": targets, "mask": None, "average": case.get("average")}
    if case["masked"]:
        lengths = torch.randint((length + 1) // 2, length + 1, (batch,), generator=gen, device="cuda")
        if batch > 4:
            lengths[1] = 0                     # an answer that was cut away altogether
        s["mask"] = torch.arange(length, device="cuda")[None, :] < lengths[:, None]

    def noise(scale, *shape):
        return torch.randn(shape, generator=gen, device="cuda") * scale

    if case["op"] == "logprobs":
        s["weights"] = noise(1.0, batch, length) / (batch * length)
        return s
    near = torch.cat([_logprobs(logits[i:i + 1], targets[i:i + 1])[0] for i in range(batch)])
    if case["op"] == "policy":
        s["old"] = near + noise(0.15, batch, length)
        s["reference"] = near + noise(0.3, batch, length)
        s["advantages"] = noise(1.0, batch, 1).expand(batch, length)
    else:
        counted = near if s["mask"] is None else near * s["mask"]
        s["reference"] = counted.sum(1) + noise(8.0, batch)
    return s


# -- plain forms ---------------------------------------------------------------------------------------------

def _logprobs(logits, targets):
    """Log-probability of every target, and the shifted exponentials and their sums that the gradient uses."""
    x = logits.float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    picked = x.gather(-1, targets.unsqueeze(-1))
    return (picked - top - torch.log(total)).squeeze(-1), e, total


def _logits_grad(e, total, targets, coefficient, dtype):
    """coefficient * (one_hot(target) - softmax), rounded once; zero where the coefficient is."""
    grad = e * (-coefficient.unsqueeze(-1) / total)
    grad.scatter_add_(-1, targets.unsqueeze(-1), coefficient.unsqueeze(-1))
    return grad.to(dtype)


def _plain_logprobs(s):
    logits, targets, mask = s["logits"], s["targets"], s["mask"]
    logp, e, total = _logprobs(logits, targets)
    if mask is not None:
        logp = torch.where(mask, logp, torch.zeros_like(logp))
    if not s["grad"]:
        return {"logprobs": logp}
    weights = s["weights"] if mask is None else torch.where(mask, s["weights"], torch.zeros_like(s["weights"]))
    return {"logprobs": logp, "grad": _logits_grad(e, total, targets, weights, logits.dtype)}


def _plain_policy(s):
    logits, targets, mask, advantages = s["logits"], s["targets"], s["mask"], s["advantages"]
    logp, e, total = _logprobs(logits, targets)
    keep = torch.ones_like(targets, dtype=torch.bool) if mask is None else mask
    if s["average"] == "tokens":
        weight = keep.float() / keep.sum().clamp(min=1)
    else:
        weight = keep.float() / (keep.sum(1, keepdim=True).clamp(min=1) * keep.shape[0])
    ratio = torch.exp(logp - s["old"])
    free = ratio * advantages
    bound = ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * advantages
    away = torch.exp(s["reference"] - logp)
    term = -torch.minimum(free, bound) + KL_WEIGHT * (away - (s["reference"] - logp) - 1)
    slope = torch.where(free <= bound, -free, torch.zeros_like(free)) + KL_WEIGHT * (1 - away)
    zero = torch.zeros_like(term)
    loss = torch.where(keep, weight * term, zero).sum()
    grad = _logits_grad(e, total, targets, torch.where(keep, weight * slope, zero), logits.dtype)
    return {"loss": loss, "logprobs": torch.where(keep, logp, zero), "grad": grad}


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _plain_preference(s):
    logits, targets, mask = s["logits"], s["targets"], s["mask"]
    logp, e, total = _logprobs(logits, targets)
    keep = torch.ones_like(targets, dtype=torch.bool) if mask is None else mask
    sums = torch.where(keep, logp, torch.zeros_like(logp)).sum(1)
    pairs = sums.shape[0] // 2
    ratio = sums - s["reference"]
    z = BETA * (ratio[:pairs] - ratio[pairs:])
    loss = ((1 - SMOOTHING) * _softplus(-z) + SMOOTHING * _softplus(z)).sum() / pairs
    slope = BETA / pairs * ((1 - SMOOTHING) * (torch.sigmoid(z) - 1) + SMOOTHING * torch.sigmoid(z))
    coefficient = torch.cat([slope, -slope]).unsqueeze(1) * keep
    return {"loss": loss, "sums": sums, "grad": _logits_grad(e, total, targets, coefficient, logits.dtype)}


def _hash(x):
    """A 32-bit mixing function of two multiplications, on int64 tensors that hold 32-bit values."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dither(count, step):
    """Two 16-bit numbers for every element of the flat buffers at this step."""
    salt = _hash(step & 0xFFFFFFFF)
    h = _hash((torch.arange(count, dtype=torch.int64, device="cuda") & 0xFFFFFFFF) ^ salt)
    return h & 0xFFFF, h >> 16


def _to_eight_bits(values, dither):
    """e4m3 codes and scales of blocks of values: stochastic rounding up with the probability of the part that is cut."""
    blocks = values.view(-1, BLOCK)
    top = blocks.abs().amax(1)
    factor = torch.where(top > 0, E4M3_MAX / top, torch.zeros_like(top))
    x = (blocks * factor[:, None]).view(-1)
    a = x.abs().clamp(max=E4M3_MAX)
    normal = ((a.view(torch.int32) + (dither << 4).to(torch.int32)) & -1048576).view(torch.float32)
    small = torch.floor(a * 512 + dither.float() / 65536) / 512
    q = torch.where(a >= 2.0 ** -6, normal, small)
    return torch.copysign(q, x), top / E4M3_MAX


def _plain_adamw(s):
    step = s["step"].add_(1)
    b1, b2 = BETAS
    t = step.double()
    c1, c2 = (1 - b1 ** t).float(), (1 - b2 ** t).float()
    g = s["grads"].float()
    if s["bits"] == 8:
        spread = lambda codes, scale: (codes.float().view(-1, BLOCK) * scale[:, None]).view(-1)  # noqa: E731
        mean = spread(s["mean"], s["mean_scale"])
        square = spread(s["root"], s["root_scale"]).square()
    else:
        mean, square = s["mean"], s["square"]
    mean = b1 * mean + (1 - b1) * g
    square = b2 * square + (1 - b2) * g * g
    root = square.sqrt()
    p = s["params"].float()
    p = p * (1 - LR * DECAY) - (LR / c1) * mean / (root / c2.sqrt() + EPS)
    s["params"].copy_(p)
    if s["bits"] == 32:
        s["mean"].copy_(mean)
        s["square"].copy_(square)
        return {"params": s["params"], "mean": s["mean"], "square": s["square"], "step": s["step"]}
    low, high = _dither(mean.numel(), step)
    codes, scale = _to_eight_bits(mean, low)
    s["mean"].copy_(codes.to(torch.float8_e4m3fn))
    s["mean_scale"].copy_(scale)
    codes, scale = _to_eight_bits(root, high)
    codes = torch.where(root > 0, codes.clamp(min=2.0 ** -9), codes)      # a second moment above zero stays above zero
    s["root"].copy_(codes.to(torch.float8_e4m3fn))
    s["root_scale"].copy_(scale)
    return {"params": s["params"], "mean": s["mean"], "mean_scale": s["mean_scale"], "root": s["root"], "root_scale": s["root_scale"], "step": s["step"]}


# -- one pass ------------------------------------------------------------------------------------------------

def _own_adamw(s):
    s["optimizer"].update(s["views"][0], s["views"][1], s["state"])
    state = s["state"]
    if s["bits"] == 32:
        return {"params": s["params"], "mean": state.exp_avg, "square": state.exp_avg_sq, "step": state.step}
    return {"params": s["params"], "mean": state.exp_avg, "mean_scale": state.exp_avg_scale, "root": state.exp_avg_root,
            "root_scale": state.exp_avg_root_scale, "step": state.step}


def run(s):
    if not own:
        return {"logprobs": _plain_logprobs, "policy": _plain_policy, "preference": _plain_preference, "adamw": _plain_adamw}[s["op"]](s)
    import trainkernel_b200 as tk
    if s["op"] == "adamw":
        return _own_adamw(s)
    if s["op"] == "logprobs":
        if not s["grad"]:
            return {"logprobs": tk.token_logprobs(s["logits"], s["targets"], mask=s["mask"])}
        logp, grad = tk.token_logprobs_and_grad(s["logits"], s["targets"], s["weights"], mask=s["mask"])
        return {"logprobs": logp, "grad": grad}
    if s["op"] == "policy":
        loss, logp, grad = tk.policy_loss_and_grad(s["logits"], s["targets"], s["old"], s["advantages"], ref_logprobs=s["reference"],
                                                   mask=s["mask"], clip=CLIP, kl_weight=KL_WEIGHT, average=s["average"])
        return {"loss": loss, "logprobs": logp, "grad": grad}
    loss, sums, grad = tk.preference_loss_and_grad(s["logits"], s["targets"], s["reference"], mask=s["mask"], beta=BETA, label_smoothing=SMOOTHING)
    return {"loss": loss, "sums": sums, "grad": grad}


# -- what a pass cannot do without ---------------------------------------------------------------------------

def work(case):
    width = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "adamw":
        n = sum(int(x) for x in case["sizes"].split(","))
        state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (2 * width[case["params"]] + width[case["grads"]] + state), "flops": 16 * n}
    rows = case["batch"] * case["length"]
    read = rows * (0.75 if case["masked"] else 1.0)             # rows behind an answer's end are not read, on average
    bytes_ = read * case["vocab"] * width[case["dtype"]] + rows * 12
    flops = 4 * read * case["vocab"]
    if case["op"] != "logprobs" or case["grad"]:
        bytes_ += rows * (case["vocab"] * width[case["dtype"]] + 12)
        flops += 3 * read * case["vocab"]
    return {"bytes": bytes_, "flops": flops}


# -- 64 bits -------------------------------------------------------------------------------------------------

def _exact_rows(s, coefficient):
    """Log-probabilities of all sequences, then, with `coefficient(logp)`, the gradient of the logits in 64 bits, sequence by sequence."""
    logits, targets = s["logits"], s["targets"]
    batch, length, vocab = logits.shape
    part = max(1, 100_000_000 // vocab)
    logp = torch.empty((batch, length), dtype=torch.float64, device="cuda")
    for b in range(batch):
        for i in range(0, length, part):
            x = logits[b, i:i + part].double()
            logp[b, i:i + part] = x.gather(1, targets[b, i:i + part, None])[:, 0] - torch.logsumexp(x, 1)
    keep = torch.ones_like(targets, dtype=torch.bool) if s["mask"] is None else s["mask"]
    if coefficient is None:
        return torch.where(keep, logp, 0.0), keep, None
    extra, c = coefficient(logp, keep)
    grad = torch.zeros((batch, length, vocab), dtype=torch.float32 if logits.dtype == torch.float32 else logits.dtype, device="cuda")
    for b in range(batch):
        for i in range(0, length, part):
            d = -torch.softmax(logits[b, i:i + part].double(), 1)
            d.scatter_add_(1, targets[b, i:i + part, None], torch.ones_like(d[:, :1]))
            grad[b, i:i + part] = (d * c[b, i:i + part, None]).to(grad.dtype)
    return torch.where(keep, logp, 0.0), extra, grad


def _exact_adamw(s):
    t = int(s["step"]) + 1
    n = s["params"].numel()
    g = s["grads"].double()
    (b1, b2), eight = BETAS, s["bits"] == 8
    if eight:
        mean = s["mean"].double() * s["mean_scale"].double().repeat_interleave(BLOCK)
        square = (s["root"].double() * s["root_scale"].double().repeat_interleave(BLOCK)) ** 2
    else:
        mean, square = s["mean"].double(), s["square"].double()
    mean = mean.mul_(b1).add_(g, alpha=1 - b1)
    square = square.mul_(b2).add_(g ** 2, alpha=1 - b2)
    p = s["params"].double()
    p -= LR * DECAY * p
    p -= LR * (mean / (1 - b1 ** t)) / (torch.sqrt(square / (1 - b2 ** t)) + EPS)
    out = {"params": p, "mean": None, "step": torch.tensor(t)}
    if not eight:
        return {**out, "mean": mean, "square": square}
    for name, values in (("mean", mean), ("root", torch.sqrt(square))):
        out[name] = None                                        # rounded by chance: a value on a border may go either way
        out[name + "_scale"] = values.abs().view(n // BLOCK, BLOCK).max(1).values / E4M3_MAX
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    if case["op"] == "adamw":
        return _exact_adamw(s)
    if case["op"] == "logprobs":
        if not case["grad"]:
            return {"logprobs": _exact_rows(s, None)[0]}
        logp, _, grad = _exact_rows(s, lambda lp, keep: (None, torch.where(keep, s["weights"].double(), 0.0)))
        return {"logprobs": logp, "grad": grad}
    if case["op"] == "policy":
        def policy(logp, keep):
            old, ref, adv = s["old"].double(), s["reference"].double(), s["advantages"].double()
            counts = keep.sum(1, keepdim=True).double()
            share = 1 / counts.sum().clamp(min=1) if case["average"] == "tokens" else 1 / (counts.clamp(min=1) * keep.shape[0])
            r = (logp - old).exp()
            clipped = (adv >= 0) & (r > 1 + CLIP[1]) | (adv < 0) & (r < 1 - CLIP[0])
            surrogate = torch.where(clipped, torch.where(adv >= 0, 1 + CLIP[1], 1 - CLIP[0]) * adv, r * adv)
            kl = torch.expm1(ref - logp) - (ref - logp)
            loss = (share * (KL_WEIGHT * kl - surrogate))[keep.nonzero(as_tuple=True)].sum() if case["average"] == "tokens" \
                else torch.where(keep, share * (KL_WEIGHT * kl - surrogate), 0.0).sum()
            slope = torch.where(clipped, 0.0, -r * adv) - KL_WEIGHT * torch.expm1(ref - logp)
            return loss, torch.where(keep, share * slope, 0.0)
        logp, loss, grad = _exact_rows(s, policy)
        return {"loss": loss, "logprobs": logp, "grad": grad}

    def preference(logp, keep):
        sums = torch.where(keep, logp, 0.0).sum(1)
        chosen, rejected = (sums - s["reference"].double()).chunk(2)
        z = BETA * (chosen - rejected)
        loss = (-(1 - SMOOTHING) * torch.nn.functional.logsigmoid(z) - SMOOTHING * torch.nn.functional.logsigmoid(-z)).mean()
        slope = BETA / len(z) * (SMOOTHING * torch.sigmoid(z) - (1 - SMOOTHING) * torch.sigmoid(-z))
        return (loss, sums), torch.where(keep, torch.cat([slope, -slope])[:, None], 0.0)
    _, (loss, sums), grad = _exact_rows(s, preference)
    return {"loss": loss, "sums": sums, "grad": grad}
