"""AdamW over many tensors against a 64-bit statement of its formulas, with 32-bit and 8-bit moments.

Bounds, with u = 2^-24: m' and v' are two products and a sum of FP32 numbers whose constants are rounded once, so each
is off by at most 4 u of the sum of its parts' sizes.  The update lr / c1 * m' / (sqrt(v') / sqrt(c2) + eps) adds the
square root, two quotients, two products and the bias corrections (each good to 4 u): 24 u of the update, plus what m'
lost relative to its parts; p' adds a product, a difference and the rounding to p's type.
"""
import math

import pytest
import torch

import trainkernel_b200 as tk

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
gpu = pytest.mark.gpu


def f32(x):
    return float(torch.tensor(x, dtype=F32))


def exact(p, g, m, v, t, lr, betas, eps, decay, scale=1.0):
    """New (p, m, v) in 64 bits and the bounds of their errors, from FP64 inputs."""
    g = g * scale
    b1, b2 = betas
    m_new, v_new = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    m_parts = (b1 * m).abs() + ((1 - b1) * g).abs()
    c1, c2 = 1 - b1 ** t, 1 - b2 ** t
    denominator = torch.sqrt(v_new / c2) + eps
    update = lr / c1 * m_new / denominator
    p_new = p * (1 - lr * decay) - update
    bound_m = 4 * U * m_parts + 1e-44
    bound_v = 6 * U * v_new + 1e-44
    bound_update = 24 * U * update.abs() + lr / c1 * bound_m / denominator
    return p_new, m_new, v_new, bound_update + 4 * U * p.abs(), bound_m, bound_v


def check_param(got, want, bound, label=""):
    info = torch.finfo(got.dtype)
    if got.dtype != F32:
        bound = bound + want.abs() * info.eps / 2 + info.smallest_normal * info.eps
    excess = (got.double() - want).abs() / bound.clamp(min=1e-300)
    assert float(excess.max()) <= 1.0, f"{label}: {float(excess.max())}"


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def tensors(sizes, dtype, scale, seed, *, shift=0):
    """One flat tensor per size, `shift` elements behind a 16-byte boundary."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for n in sizes:
        base = torch.empty(n + shift, dtype=dtype, device="cuda")
        base.copy_(torch.randn(n + shift, generator=gen, device="cuda") * scale)
        out.append(base[shift:])
    return out


SIZES = [[1], [255, 1, 257, 256], [2048, 2049, 7, 100003], [0, 5, 0, 4096], [33] * 130, [300] * 800, [5_000_000, 3]]
NAMES = ["one", "few", "odd", "empty", "many", "two-launches", "large"]


@gpu
@pytest.mark.parametrize("sizes", SIZES, ids=NAMES)
@pytest.mark.parametrize("params,grads,shift", [(F32, F32, 0), (F32, BF16, 1), (BF16, F32, 3), (F16, F16, 0), (F32, F16, 0), (BF16, BF16, 0)])
def test_three_steps_with_32_bit_moments(sizes, params, grads, shift):
    p, optimizer = tensors(sizes, params, 0.5, 1, shift=shift), tk.AdamW(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    state = optimizer.init(p)
    moments = [(torch.zeros(n, dtype=torch.float64, device="cuda"),) * 2 for n in sizes]
    for t in range(1, 4):
        g = tensors(sizes, grads, 0.1, 10 + t, shift=shift)
        before = [x.double() for x in p]
        optimizer.update(p, g, state)
        assert int(state.step) == t
        for i, n in enumerate(sizes):
            if not n:
                continue
            want = exact(before[i], g[i].double(), *moments[i], t, f32(1e-2), (f32(0.9), f32(0.95)), f32(1e-8), f32(0.1))
            # 1 - beta as the kernel has it: rounded from 64 bits, not from the rounded beta
            want = exact(before[i], g[i].double(), *moments[i], t, 1e-2, (0.9, 0.95), 1e-8, 0.1) if want else want
            m, v = state.moments(i)
            assert bool(((m.double() - want[1]).abs() <= want[4]).all()) and bool(((v.double() - want[2]).abs() <= want[5]).all())
            check_param(p[i], want[0], want[3], f"step {t} tensor {i}")
            moments[i] = (m.double(), v.double())


@gpu
@pytest.mark.parametrize("sizes", SIZES, ids=NAMES)
@pytest.mark.parametrize("params,grads,shift", [(F32, F32, 0), (F32, BF16, 1), (BF16, F16, 0)])
def test_three_steps_with_8_bit_moments(sizes, params, grads, shift):
    p, optimizer = tensors(sizes, params, 0.5, 2, shift=shift), tk.AdamW(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.01, state_bits=8, seed=77)
    state = optimizer.init(p)
    for t in range(1, 4):
        g = tensors(sizes, grads, 0.1, 20 + t, shift=shift)
        before, old = [x.double() for x in p], [state.moments(i) for i in range(len(sizes))]
        optimizer.update(p, g, state)
        for i, n in enumerate(sizes):
            if not n:
                continue
            m, v = (x.double() for x in old[i])
            want = exact(before[i], g[i].double(), m, v, t, 1e-2, (0.9, 0.95), 1e-8, 0.01)
            # the moments are two FP32 products (code times scale, squared for v) before the formula: 4 u more
            check_param(p[i], want[0], want[3] + 8 * U * (before[i] - want[0]).abs() + 8 * U * before[i].abs(), f"step {t} tensor {i}")
            root = want[2].sqrt()
            check_codes(state, i, want[1], root, t, 77, 2 * want[4], 2 * want[5] / root.clamp(min=1e-40))


def check_codes(state, i, mean, root, t, seed, mean_error, root_error):
    """Scales are the block maxima / 448; codes lie on the two neighbours of the value, on the one the hash says except next to its border."""
    begin, n = state.offsets[i], state.sizes[i]
    salt = mix(torch.tensor((t + seed * 0x9E3779B9) & 0xFFFFFFFF, device="cuda"))
    random = mix((torch.arange(begin, begin + n, device="cuda") & 0xFFFFFFFF) ^ salt)
    for codes, scales, values, dither, floor, error in ((state.exp_avg, state.exp_avg_scale, mean, random & 0xFFFF, False, mean_error),
                                                        (state.exp_avg_root, state.exp_avg_root_scale, root, random >> 16, True, root_error)):
        blocks = -(-n // 256)
        padded = torch.zeros(blocks * 256, dtype=torch.float64, device="cuda")
        padded[:n] = values
        top = padded.view(-1, 256).abs().amax(1)
        scale = scales[begin // 256:begin // 256 + blocks].double()
        assert bool(((scale - top / 448).abs() <= 16 * U * top / 448 + 1e-40).all())
        got = codes[begin:begin + blocks * 256].double()
        assert bool((got[n:] == 0).all())
        x = (padded.view(-1, 256) / torch.where(scale > 0, scale, 1.0)[:, None]).view(-1)[:n]
        got = got[:n]
        a = x.abs().clamp(max=448.0)
        exponent = torch.floor(torch.log2(a.clamp(min=2.0 ** -6)))
        spacing = torch.exp2(exponent - 3)
        low = torch.floor(a / spacing) * spacing
        part = (a - low) / spacing
        high = low + spacing
        up = part + dither.double() / 65536 >= 1.0
        want = torch.where(up, high, low)
        if floor:
            want = torch.where((values > 0) & (want < 2.0 ** -9), 2.0 ** -9, want)
        differs = got.abs() != want
        # The value that is rounded is off by what the moment is (b1 m and (1 - b1) g may cancel: u of the parts, not of their
        # sum, with the decoded moment's own rounding twice the bound above) and by the scale and one product, 16 u of itself:
        # only a part that near to the border may fall on its other side.
        reach = (error / torch.where(scale > 0, scale, 1.0).repeat_interleave(256)[:n] + 32 * U * a) / spacing + 2.0 ** -22
        near = ((part + dither.double() / 65536 - 1.0).abs() <= reach) | (part < reach) | (part > 1 - reach)
        assert not bool((differs & ~near).any())
        assert float(differs.double().mean()) <= 0.01 or n < 300
        assert bool((torch.sign(got) == torch.sign(x))[got != 0].all())


@gpu
def test_stochastic_rounding_is_unbiased_and_keeps_moving():
    """A second moment that rounding to nearest would freeze follows its exact course on average."""
    n = 256 * 512
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.1, device="cuda")
    g[::256] = 1.0                                          # holds every block's scale
    optimizer = tk.AdamW(lr=0.0, betas=(0.9, 0.99), weight_decay=0.0, state_bits=8)
    state = optimizer.init([p])
    for _ in range(5):
        optimizer.update([p], [g], state)
    small = g.clone()
    small[torch.arange(n, device="cuda") % 256 != 0] = 0.02
    m, v = (x.double() for x in state.moments(0))
    exact_v, exact_m, steps = v, m, 60
    for _ in range(steps):
        optimizer.update([p], [small], state)
        exact_v, exact_m = 0.99 * exact_v + 0.01 * small.double() ** 2, 0.9 * exact_m + 0.1 * small.double()
    m, v = (x.double() for x in state.moments(0))
    rest = torch.arange(n, device="cuda") % 256 != 0
    # Codes of the root are at most 1/8 apart relative to themselves, so one rounding has a variance of at most (1/16)^2 and
    # `steps` of them, decaying, well under 0.25 relative for one element; over 130560 elements the mean is good to 0.25 / 361 < 1e-3.
    # Squaring adds the variance of the root: each step up to (1/16)^2 = 0.4 % upwards, and about a third of that on average.
    ratio = float(v[rest].mean() / exact_v[rest].mean())
    assert 0.99 < ratio < 1.0 + steps * (1 / 16) ** 2
    assert float(v[rest].mean()) < 0.8 * float(0.01 * (1 - 0.99 ** 5) / 0.01)
    assert abs(float(m[rest].mean() / exact_m[rest].mean()) - 1) < 5e-3


@gpu
def test_weight_decay_per_tensor_and_device_learning_rate():
    sizes = [300, 5, 1000]
    p = tensors(sizes, F32, 1.0, 3)
    g = tensors(sizes, F32, 0.1, 4)
    lr = torch.full((), 0.5, device="cuda")
    optimizer = tk.AdamW(lr=lr, weight_decay=[0.0, 0.5, 0.25])
    state = optimizer.init(p)
    for t, value in enumerate((0.5, 0.125), 1):
        lr.fill_(value)
        before, old = [x.double() for x in p], [state.moments(i) for i in range(3)]
        optimizer.update(p, g, state)
        for i, decay in enumerate((0.0, 0.5, 0.25)):
            want = exact(before[i], g[i].double(), old[i][0].double(), old[i][1].double(), t, value, (0.9, 0.999), 1e-8, decay)
            check_param(p[i], want[0], want[3])


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_scale_of_gradients_and_skipped_steps(bits):
    p, g = tensors([4097, 3], F32, 1.0, 5), tensors([4097, 3], F32, 0.1, 6)
    optimizer = tk.AdamW(state_bits=bits)
    state = optimizer.init(p)
    scale = torch.full((1,), 0.25, device="cuda")
    q = [x.clone() for x in p]
    other = optimizer.init(q)
    optimizer.update(p, g, state, grad_scale=scale)
    optimizer.update(q, [x * 0.25 for x in g], other)              # a power of two: the same numbers
    for a, b in zip([*p, *state.tensors()], [*q, *other.tensors()]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    kept = [x.clone() for x in (*p, *state.tensors())]
    for value in (float("inf"), float("nan"), -float("inf")):
        scale.fill_(value)
        optimizer.update(p, g, state, grad_scale=scale)
    for a, b in zip((*p, *state.tensors()), kept):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert int(state.step) == 1


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_updates_advance(bits):
    sizes = [1000, 257, 70000]
    g = tensors(sizes, F32, 0.1, 7)
    eager, captured = tensors(sizes, F32, 1.0, 8), tensors(sizes, F32, 1.0, 8)
    optimizer = tk.AdamW(lr=1e-2, state_bits=bits)
    a, b = optimizer.init(eager), optimizer.init(captured)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optimizer.update(captured, g, b)
    for _ in range(4):
        graph.replay()
        optimizer.update(eager, g, a)
    torch.cuda.synchronize()
    assert int(b.step) == 4
    for x, y in zip([*eager, *a.tensors()], [*captured, *b.tensors()]):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@gpu
def test_mixed_types_advance_the_step_once_and_memory_order_is_kept():
    p = [torch.randn(16, 24, device="cuda").t(), torch.randn(40, device="cuda").to(BF16), torch.randn((), device="cuda"), torch.randn(2, 3, 4, 5, device="cuda").permute(0, 2, 3, 1)]
    g = [torch.randn(16, 24, device="cuda").t(), torch.randn(40, device="cuda"), torch.randn((), device="cuda").half(), torch.randn(2, 3, 4, 5, device="cuda").permute(0, 2, 3, 1)]
    optimizer = tk.AdamW(lr=0.1)
    state = optimizer.init({"a": p[0], "b": p[1], "c": p[2], "d": p[3]})
    before = [x.double() for x in p]
    versions = [x._version for x in p]
    optimizer.update(p, g, state)
    assert int(state.step) == 1 and all(x._version > v for x, v in zip(p, versions))
    for x, y, z in zip(p, before, g):
        zero = torch.zeros_like(y)
        want = exact(y, z.double(), zero, zero, 1, 0.1, (0.9, 0.999), 1e-8, 0.01)
        check_param(x, want[0], want[3])


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_neighbours_of_a_tensor_stay_as_they_were(bits):
    """Tensors that end inside a 256-block and start at odd places: nothing around them is written."""
    whole, gradient = torch.randn(5000, device="cuda"), torch.randn(5000, device="cuda")
    kept = whole.clone()
    spans = [(3, 17), (20, 277), (300, 2349), (2351, 2352), (4000, 4999)]
    optimizer = tk.AdamW(state_bits=bits)
    p, g = [whole[a:b] for a, b in spans], [gradient[a + 1:b + 1] for a, b in spans]
    state = optimizer.init(p)
    optimizer.update(p, g, state)
    inside = torch.zeros(5000, dtype=torch.bool, device="cuda")
    for a, b in spans:
        inside[a:b] = True
    assert torch.equal(whole[~inside], kept[~inside]) and not bool((whole[inside] == kept[inside]).all())


@gpu
def test_tiny_and_vanishing_moments_stay_numbers():
    p = [torch.ones(600, device="cuda")]
    optimizer = tk.AdamW(lr=1e-3, betas=(0.5, 0.5), state_bits=8)
    state = optimizer.init(p)
    gradient = torch.full((600,), 1e-20, device="cuda")
    gradient[300:] = 0
    for t in range(200):                                    # the first moment runs through the subnormal numbers to zero
        optimizer.update(p, [gradient if t < 2 else torch.zeros_like(gradient)], state)
    assert bool(torch.isfinite(p[0]).all())
    assert all(bool(torch.isfinite(x).all()) for x in state.moments(0))


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_short_and_long_way_to_a_launch_agree(bits, monkeypatch):
    from trainkernel_b200 import operators
    sizes = [300, 0, 5, 4096]
    results = []
    for long_way in (False, True):
        if long_way:
            monkeypatch.setattr(operators, "fast", None)
        p, g = tensors(sizes, F32, 1.0, 50), tensors(sizes, BF16, 0.1, 51)
        optimizer = tk.AdamW(weight_decay=(0.0, 0.1, 0.2, 0.3), state_bits=bits, seed=9)
        state = optimizer.init(p)
        if not long_way:
            assert operators.fast.adamw_update(p, g, state.sizes, state.offsets, 0.0, state._struct_at, state._tensors, bits, 0.0, (0.9, 0.9), 1e-8, 0, None)
            p, g = tensors(sizes, F32, 1.0, 50), tensors(sizes, BF16, 0.1, 51)
            state = optimizer.init(p)
        for _ in range(2):
            before = [x._version for x in (*p, *state.tensors())]
            optimizer.update(p, g, state, grad_scale=torch.full((), 0.5, device="cuda"))
            assert all(x._version > v for x, v in zip((*p, *state.tensors()), before))
        results.append([*p, *state.tensors()])
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# -- refusals ------------------------------------------------------------------------------------------------

def test_refusals_of_numbers():
    bad = [dict(lr=-1.0), dict(lr=float("nan")), dict(lr=torch.ones(1)), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(betas=(0.9,)), dict(eps=0.0), dict(eps=1e-40),
           dict(weight_decay=-0.1), dict(weight_decay=[0.1, "x"]), dict(state_bits=16), dict(seed=-1), dict(seed=2 ** 32)]
    for arguments in bad:
        with pytest.raises(ValueError, match="trainkernel: AdamW"):
            tk.AdamW(**arguments)


def test_parameters_on_the_host_are_refused():
    with pytest.raises(RuntimeError, match="sm_100a GPU required"):
        tk.AdamW().init([torch.zeros(3)])
    with pytest.raises(TypeError, match="tensors only"):
        tk.AdamW().init([1.0])


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_continues_where_it_was_taken(bits, tmp_path):
    sizes = [700, 3]
    p, g = tensors(sizes, F32, 1.0, 70), tensors(sizes, F32, 0.1, 71)
    optimizer = tk.AdamW(state_bits=bits)
    state = optimizer.init(p)
    optimizer.update(p, g, state)
    torch.save((p, state.state_dict()), tmp_path / "checkpoint")
    optimizer.update(p, g, state)
    q, saved = torch.load(tmp_path / "checkpoint", weights_only=False)
    other = optimizer.init(q)
    other.load_state_dict(saved)
    optimizer.update(q, g, other)
    for a, b in zip([*p, *state.tensors()], [*q, *other.tensors()]):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    with pytest.raises(ValueError, match="other tensors"):
        optimizer.init(q[:1]).load_state_dict(saved)


@gpu
def test_init_inside_a_capture_is_refused():
    p = [torch.zeros(4, device="cuda")]
    tk.AdamW().init(p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="clear the moments"):
            tk.AdamW().init(p)
        p[0].add_(1.0)


@gpu
@pytest.mark.parametrize("betas", [(0.0, 0.0), (0.9, 0.0), (0.0, 0.999)])
def test_betas_of_zero(betas):
    p, g = tensors([700], F32, 1.0, 60), tensors([700], F32, 0.1, 61)
    g[0][:5] = 0
    optimizer = tk.AdamW(lr=1e-2, betas=betas, weight_decay=0.0)
    state = optimizer.init(p)
    for t in (1, 2):
        before, old = p[0].double(), [x.double() for x in state.moments(0)]
        optimizer.update(p, g, state)
        want = exact(before, g[0].double(), *old, t, 1e-2, betas, 1e-8, 0.0)
        check_param(p[0], want[0], want[3])


@gpu
def test_an_update_leaves_gradients_and_follows_the_current_stream():
    p, g = tensors([5000, 3], F32, 1.0, 62), tensors([5000, 3], F32, 0.1, 63)
    kept = [x.clone() for x in g]
    optimizer = tk.AdamW()
    state, other = optimizer.init(p), [x.clone() for x in p]
    twin = optimizer.init(other)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            optimizer.update(p, g, state)
    for _ in range(3):
        optimizer.update(other, g, twin)
    torch.cuda.synchronize()
    for a, b in zip([*p, *state.tensors()], [*other, *twin.tensors()]):
        assert torch.equal(a, b)
    assert all(torch.equal(a, b) for a, b in zip(g, kept))


@gpu
def test_refusals_of_tensors():
    optimizer = tk.AdamW()
    p, g = [torch.zeros(4, 6, device="cuda"), torch.zeros(5, device="cuda")], [torch.zeros(4, 6, device="cuda"), torch.zeros(5, device="cuda")]
    state = optimizer.init(p)
    bad = [
        (lambda: optimizer.init([torch.zeros(3, dtype=torch.int32, device="cuda")]), "float32, float16"),
        (lambda: optimizer.init([torch.zeros(8, device="cuda")[::2]]), "dense"),
        (lambda: optimizer.init([torch.zeros(1, device="cuda").expand(4)]), "dense"),
        (lambda: tk.AdamW(weight_decay=[0.1]).init(p), "weight decays"),
        (lambda: optimizer.update(p[:1], g[:1], state), "for a state of 2"),
        (lambda: optimizer.update(p, g[:1], state), "1 grads"),
        (lambda: optimizer.update(p, [g[0].t().contiguous().t(), g[1]], state), "memory order"),
        (lambda: optimizer.update(p, [g[0].double(), g[1]], state), "does not match"),
        (lambda: optimizer.update(p, [g[0][:3], g[1]], state), "does not match"),
        (lambda: optimizer.update([p[1], p[0]], [g[1], g[0]], state), "elements"),
        (lambda: tk.AdamW(state_bits=8).update(p, g, state), "32-bit moments"),
        (lambda: optimizer.update(p, g, state, grad_scale=2.0), "grad_scale"),
        (lambda: optimizer.update(p, g, state, grad_scale=torch.ones(2, device="cuda")), "grad_scale"),
        (lambda: state.set_step(-1), "step"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
    twin = torch.zeros(4, 6, device="cuda")
    two = optimizer.init([twin, twin])
    with pytest.raises(ValueError, match="listed twice"):
        optimizer.update([twin, twin], [twin, twin], two)
    assert math.isfinite(float(p[0].sum()))
