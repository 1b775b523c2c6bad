"""AdamW over many tensors against the formulas in 64 bits.

Tolerances count roundings of u = 2^-24.  m = b1 m + (1 - b1) g: the two factors, the scaled gradient, a product and the
sum, 6 u of b1 |m| + (1 - b1) |g| with one to spare; v has the square besides, 8 u.  The update divides by a root whose
operand carries 8 u (4 u after the root), with root, quotient and eps' sum at 2 u each and the step's factors at 1 u:
below 2^-19 of the update's magnitude.  The parameter is decayed (2 u) and summed (1 u): 4 u.  A 16-bit copy adds
half a step.  An 8-bit code is what the formula gives for a value within those bounds."""
import math

import pytest
import torch

from fbcunn_b200 import AdamW, SpatialConvolutionFBFFT, capi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weightDecay=0.1)
SIZES = [1, 7, 255, 256, 257, 1000, 4096, 5003]


def _mix(x):
    for shift, odd in ((16, 0x6A09E667), (15, 0xBB67AE85), (16, 1)):
        x = ((x ^ (x >> shift)) * odd) & 0xFFFFFFFF
    return x


def _round(y, uniform):
    quantum = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
    return (torch.floor(y.abs() / quantum + uniform) * quantum).clamp(max=448) * torch.sign(y)


def _decode(opt, i, key):
    bits, at = opt.layout[i]
    n = opt.params[i].numel()
    if bits == 32:
        return opt.moments[{"m8": "m", "r8": "v"}[key]][at: at + n].double()
    codes = opt.moments[key][at: at + n].double()
    scale = opt.moments[key + "_scale"].double()[at // 256 + torch.arange(n, device="cuda") // 256]
    return codes * scale


def check_step(opt, do_step=None, grad_scale=1.0, lr=None):
    """One step of `opt`, compared with the formulas applied to what it held before."""
    b1, b2 = opt.betas
    lr = opt.lr if lr is None else lr
    t = opt.steps + 1
    before = []
    for i, (p, w, g) in enumerate(zip(opt.params, opt.masters, opt.grads)):
        m, v = _decode(opt, i, "m8"), _decode(opt, i, "r8")
        v = v ** 2 if opt.layout[i][0] == 8 else v
        before.append(((p if w is None else w).double().flatten(), g.double().flatten() * grad_scale, m, v))
    (do_step or opt.step)()
    assert opt.steps == t and int(opt._counter[1]) == 0
    for i, (x, g, m, v) in enumerate(before):
        if not x.numel():
            continue
        size1, size2 = b1 * m.abs() + (1 - b1) * g.abs(), b2 * v + (1 - b2) * g ** 2
        m, v = b1 * m + (1 - b1) * g, size2
        unit = lr / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + opt.eps)
        new = x * (1 - lr * opt.weightDecay) - unit * m
        tol = 4 * U * new.abs() + 4 * U * x.abs() + 2.0 ** -19 * unit * size1
        p, w = opt.params[i], opt.masters[i]
        if w is not None:
            assert bool(((w.double().flatten() - new).abs() <= tol).all())
            assert torch.equal(p, w.to(p.dtype))  # the copy is the master, rounded once
        else:
            half = 0 if p.dtype == torch.float32 else torch.finfo(p.dtype).eps / 2 * 1.001
            least = 0 if p.dtype != torch.float16 else 2.0 ** -25
            assert bool(((p.double().flatten() - new).abs() <= tol * 1.01 + half * new.abs() + least).all())
        bits, at = opt.layout[i]
        n = x.numel()
        if bits == 32:
            assert bool(((opt.moments["m"][at: at + n] - m).abs() <= 6 * U * size1).all())
            assert bool(((opt.moments["v"][at: at + n] - v).abs() <= 8 * U * size2).all())
            assert not opt.moments["m"][at + n: at + -(-n // 256) * 256].any()
            continue
        e = torch.arange(n, device="cuda")
        key = _mix(torch.tensor((opt.seed + t * 0x9E3779B9) & 0xFFFFFFFF, device="cuda"))
        bitset = _mix(e ^ _mix((key + i) & 0xFFFFFFFF))
        for name, value, off, uniform in (("m8", m, 6 * U * size1, bitset & 0xFFFF),
                                          ("r8", v.sqrt(), 8 * U * v.sqrt(), bitset >> 16)):
            top = torch.zeros(-(-n // 256), dtype=torch.float64, device="cuda")
            top.index_reduce_(0, e // 256, value.abs(), "amax")
            scale = opt.moments[name + "_scale"][at // 256: at // 256 + top.numel()].double()
            # the block's largest is known to `off` of some element; the scale to that and a quotient
            slack = torch.zeros_like(top).index_reduce_(0, e // 256, off, "amax") / 448 + 2 * U * top / 448
            assert bool(((scale - top / 448).abs() <= slack).all())
            per = (top / 448)[e // 256].clamp(min=1e-300)
            y, dy = value / per, (off + 4 * U * value.abs() + 448 * slack[e // 256] * value.abs() / (448 * per)) / per
            codes = opt.moments[name][at: at + n].double()
            least = 2.0 ** -9 if name == "r8" else -math.inf
            low = torch.where(y > 0, _round(y - dy, uniform / 65536).clamp(min=least), _round(y - dy, uniform / 65536))
            high = torch.where(y > 0, _round(y + dy, uniform / 65536).clamp(min=least), _round(y + dy, uniform / 65536))
            # below zero the magnitude is what is rounded: the two ends come in either order
            assert not int((codes < torch.minimum(low, high)).sum() + (codes > torch.maximum(low, high)).sum())
        tail = slice(at + n, at + -(-n // 256) * 256)
        assert not opt.moments["m8"][tail].double().any() and not opt.moments["r8"][tail].double().any()


def _tensors(sizes, dtype, grad_dtype, shift=0, seed=0):
    """Parameters and gradients as views of one tensor each, `shift` elements off a vector's alignment, with elements
    between them that nothing may touch."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(-(-n // 64) * 64 + 64 for n in sizes) + shift

    def flat(scale, dtype):
        return torch.empty(total, device="cuda").normal_(generator=gen).mul_(scale).to(dtype)

    fp, fg = flat(0.1, dtype), flat(0.01, grad_dtype)
    params, grads, at = [], [], shift
    for n in sizes:
        params.append(fp[at: at + n])
        grads.append(fg[at: at + n])
        at += -(-n // 64) * 64 + 64
    return params, grads, fp


def _set_moments(opt, seed=1):
    """Moments as after many steps."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for p, (bits, at) in zip(opt.params, opt.layout):
        n = p.numel()
        for key in ("m", "v") if bits == 32 else ("m8", "r8"):
            x = torch.empty(n, device="cuda").normal_(generator=gen)
            x = x * 1e-2 if key.startswith("m") else x.abs() * 1e-2
            if bits == 32:
                opt.moments[key][at: at + n] = x if key == "m" else x ** 2
            else:
                blocks = -(-n // 256)
                opt.moments[key][at: at + n] = (x * 1e4).clamp(-448, 448).to(torch.float8_e4m3fn)
                opt.moments[key + "_scale"][at // 256: at // 256 + blocks] = 1e-4
    opt._counter[0] = 41


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,grad_dtype,masters", [
    (torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False),
    (torch.bfloat16, torch.float32, True), (torch.float16, torch.float16, True), (torch.float32, torch.bfloat16, False),
    (torch.float16, torch.float32, False)])
def test_a_step_follows_the_formulas(dtype, grad_dtype, masters, bits, shift):
    params, grads, flat = _tensors(SIZES, dtype, grad_dtype, shift)
    outside = torch.ones(flat.numel(), dtype=torch.bool, device="cuda")
    for p in params:
        outside[p.storage_offset(): p.storage_offset() + p.numel()] = False
    untouched = flat[outside].clone()
    opt = AdamW(params, grads, stateBits=bits, min8bitSize=256, masters=True if masters else None, seed=7, **HYPER)
    _set_moments(opt)
    check_step(opt)
    check_step(opt, grad_scale=0.25, do_step=lambda: opt.step(gradScale=0.25))
    assert torch.equal(flat[outside], untouched)


@pytest.mark.parametrize("bits", [32, 8])
def test_first_steps_from_zero(bits):
    params, grads, _ = _tensors([3, 513, 2048], torch.float32, torch.float32)
    grads[1][:] = 0  # moments of zero stay zero, and 0 / (0 + eps) is no step
    grads[2][256:512] = 0
    opt = AdamW(params, grads, stateBits=bits, min8bitSize=1, **HYPER)
    still = params[1].clone()
    for _ in range(3):
        check_step(opt)
    decay = 1 - HYPER["lr"] * HYPER["weightDecay"]
    assert torch.allclose(params[1], still * decay ** 3, rtol=8 * U, atol=0)


@pytest.mark.parametrize("count", [44, 45, 400, 401, 1203])
def test_many_tensors(count):
    """Tables of every size, over one launch and several."""
    sizes = [(i * 37) % 300 for i in range(count)]  # empty ones among them
    params, grads, _ = _tensors(sizes, torch.float32, torch.float32)
    opt = AdamW(params, grads, stateBits=8, min8bitSize=128, **HYPER)
    _set_moments(opt)
    launches = capi.kernel_launches()
    p0 = [p.double() for p in params]
    m0 = [_decode(opt, i, "m8") for i in range(count)]
    v0 = [_decode(opt, i, "r8") ** (2 if opt.layout[i][0] == 8 else 1) for i in range(count)]
    opt.step()
    used = sum(n > 0 for n in sizes)
    assert capi.kernel_launches() - launches == -(-used // 400)
    assert opt.steps == 42
    for i in range(0, count, 7):
        m, v = 0.9 * m0[i] + 0.1 * grads[i].double(), 0.999 * v0[i] + 0.001 * grads[i].double() ** 2
        new = p0[i] * (1 - 1e-3) - 1e-2 / (1 - 0.9 ** 42) * m / ((v / (1 - 0.999 ** 42)).sqrt() + 1e-8)
        assert torch.allclose(params[i].double(), new, rtol=0, atol=2e-6)  # 2^-19 of updates up to 1e-2 x 7.3, 8 u of 0.5


def test_only_empty_tensors_still_count_a_step():
    p = torch.empty(0, device="cuda")
    opt = AdamW([p], [p.clone()])
    opt.step()
    assert opt.steps == 1


def test_rounding_is_unbiased():
    """The 8-bit roots of gradients that have halved decay as 32-bit moments do, where rounding to nearest would leave
    them (v would stay 1.24 times too large).  A step moves a root by the share p of its code's step q = 16/448 of the
    block's largest, which adds q^2 p (1 - p) to the mean of its square: over a way of 25 of those 448ths, from 224 to
    some 201, at most 16 * 25 / 201^2 = 1% in all.  The squares' spread is about 0.2, their mean's over 32768 elements
    1e-3."""
    n = 1 << 16
    g = torch.full((n,), 1e-2, device="cuda")
    g[::256] = 2e-2  # the blocks' largest, which the scales follow
    p = [torch.zeros(n, device="cuda") for _ in range(2)]
    a, b = (AdamW([p[i]], [g], stateBits=bits, **HYPER) for i, bits in ((0, 8), (1, 32)))
    b.moments["v"].copy_(g * g)
    a.moments["r8"].copy_((g * (224 / 1e-2)).to(torch.float8_e4m3fn))
    a.moments["r8_scale"].fill_(2e-2 / 448)
    g[1::2] = 5e-3
    for opt in (a, b):
        opt._counter[0] = 10 ** 6
        for _ in range(300):
            opt.step()
    ratio = float((_decode(a, 0, "r8")[1::2] ** 2).mean() / _decode(b, 0, "r8")[1::2].mean())
    assert 1 - 0.005 < ratio < 1.01 + 0.005


def test_non_finite_gradients_stay_in_their_block():
    for value in (float("nan"), float("inf")):
        params, grads, _ = _tensors([1024, 512], torch.float32, torch.float32)
        grads[0][300] = value
        opt = AdamW(params, grads, stateBits=8, min8bitSize=1, **HYPER)
        opt.step()
        assert not torch.isfinite(params[0][300])
        others = torch.arange(1024, device="cuda") != 300
        assert torch.isfinite(params[0][others]).all() and torch.isfinite(params[1]).all()
        m = _decode(opt, 0, "m8")
        assert not torch.isfinite(m[256:512]).any() and torch.isfinite(m[:256]).all() and torch.isfinite(m[512:]).all()


def test_captured_steps_count_and_read_their_scalars():
    params, grads, _ = _tensors(SIZES, torch.float32, torch.float32)
    twin = [p.clone() for p in params]
    opt, other = AdamW(params, grads, stateBits=8, **HYPER), AdamW(twin, grads, stateBits=8, **HYPER)
    scalars = torch.tensor([1e-2, 1.0], device="cuda")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            opt.step(scalars=scalars)
    torch.cuda.synchronize()
    assert opt.steps == 0
    for k in range(4):
        lr = 1e-2 / (k + 1)
        scalars.copy_(torch.tensor([lr, 0.5]))
        graph.replay()
        other.step(lr=float(scalars[0]), gradScale=0.5)
    assert opt.steps == other.steps == 4
    for a, b in zip(params, twin):
        assert torch.equal(a, b)
    for k in opt.moments:
        assert torch.equal(opt.moments[k].view(torch.uint8), other.moments[k].view(torch.uint8))


def test_state_moves_to_another_optimizer():
    params, grads, _ = _tensors([5000, 77], torch.bfloat16, torch.bfloat16)
    a = AdamW(params, grads, stateBits=8, seed=3, **HYPER)
    a.step()
    b = AdamW([p.clone() for p in params], grads, stateBits=8, seed=3, **HYPER)
    b.loadState(a.state())
    a.step()
    b.step()
    assert a.steps == b.steps == 2
    for p, q in zip(a.params, b.params):
        assert torch.equal(p, q)
    with pytest.raises(AssertionError):
        AdamW(params, grads, **HYPER).loadState(a.state())


def test_replaced_storage_is_noticed_and_gradients_exchanged():
    params, grads, _ = _tensors([600], torch.float32, torch.float32)
    opt = AdamW(params, grads, **HYPER)
    opt.step()
    old = params[0].clone()
    params[0].data = params[0].clone()
    grads[0].data = -grads[0].clone()
    opt.step()
    assert not torch.equal(params[0], old)
    opt.setGradients([torch.zeros(600, device="cuda")])
    check_step(opt)
    with pytest.raises(AssertionError):
        opt.setGradients([torch.zeros(601, device="cuda")])


def test_on_another_stream_than_the_current_one():
    params, grads, _ = _tensors([100000], torch.float32, torch.float32)
    twin = params[0].clone()
    opt, other = AdamW(params, grads, **HYPER), AdamW([twin], grads, **HYPER)
    other.step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        opt.step()
    stream.synchronize()
    assert torch.equal(params[0], twin)


def test_steps_the_parameters_of_convolutions():
    conv = SpatialConvolutionFBFFT(3, 5, 3, 3)
    x = torch.randn(2, 3, 9, 9, device="cuda")
    opt = AdamW([conv], **HYPER)
    assert [p.data_ptr() for p in opt.params] == [conv.weight.data_ptr(), conv.bias.data_ptr()]
    for _ in range(2):
        out = conv.updateOutput(x)
        conv.backward(x, torch.ones_like(out))
        check_step(opt)


def test_refusals_on_the_device():
    p, g = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    with pytest.raises(capi.FbfftconvError, match="share memory"):
        AdamW([p, p], [g, g])
    with pytest.raises(capi.FbfftconvError, match="share memory"):
        AdamW([p, p[299:]], [g, g[299:]])
    with pytest.raises(AssertionError):
        AdamW([p], [g.double()])
    with pytest.raises(AssertionError):
        AdamW([p[::2]], [g[::2]])
    with pytest.raises(AssertionError):
        AdamW([p], [g[:299]])
    with pytest.raises(AssertionError):
        AdamW([p], [g], masters=[p.bfloat16()])
    opt = AdamW([p], [g])
    with pytest.raises(capi.FbfftconvError, match="finite"):
        opt.step(lr=float("nan"))
    assert opt.steps == 0
    host = (capi.c_void_p * 1)(torch.zeros(300).data_ptr())
    assert capi.lib().fbfftconv_adamw_set_gradients(opt._handle, host, 1) == capi.ERR_INVALID_ARGUMENT
    opt.step()  # the handle still has its own gradients
    assert opt.steps == 1


def test_a_captured_step_of_many_tensors():
    """The large table of a launch's parameters in a graph, and two such graphs of two optimizers side by side."""
    made = []
    for seed in (0, 1):
        params, grads, _ = _tensors([(37 * i) % 900 + 1 for i in range(150)], torch.bfloat16, torch.float32, seed=seed)
        twin = [p.clone() for p in params]
        opts = [AdamW(p, grads, stateBits=8, min8bitSize=256, masters=True, **HYPER) for p in (params, twin)]
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            opts[0].step()
        made.append((graph, side, opts))
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, side, opts in made:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, (a, b) in made:
        for _ in range(3):
            b.step()
        assert a.steps == b.steps == 3
        assert all(torch.equal(p, q) for p, q in zip(a.params + a.masters, b.params + b.masters))


def test_a_run_goes_on_from_its_state():
    """Weights that live in masters made here are the state's: the steps after a resume are those of the run itself."""
    params, grads, _ = _tensors([5000, 77], torch.bfloat16, torch.bfloat16)
    a = AdamW(params, grads, stateBits=8, masters=True, seed=3, **HYPER)
    for _ in range(3):
        a.step()
    saved = [p.clone() for p in params]
    state = a.state()
    a.step()
    b = AdamW(saved, grads, stateBits=8, masters=True, seed=3, **HYPER)
    b.loadState(state)
    b.step()
    for p, q in zip(a.params + a.masters, b.params + b.masters):
        assert torch.equal(p, q)


def test_gradients_that_lie_in_what_is_stepped_are_refused():
    p, g = torch.zeros(300, device="cuda"), torch.zeros(300, device="cuda")
    for grad in (p, p[:]):
        with pytest.raises(capi.FbfftconvError, match="share memory"):
            AdamW([p], [grad])
    with pytest.raises(capi.FbfftconvError, match="share memory"):
        AdamW([p[:200]], [p[100:]])
    opt = AdamW([p], [g])
    inside = (capi.c_void_p * 1)(opt.moments["m"].data_ptr())
    assert capi.lib().fbfftconv_adamw_set_gradients(opt._handle, inside, 1) == capi.ERR_INVALID_ARGUMENT
    with pytest.raises(capi.FbfftconvError, match="share memory"):
        opt.setGradients([opt.moments["v"][:300]])
    assert opt.grads[0] is g
    opt.step()
    assert opt.steps == 1


@pytest.mark.parametrize("eps", [0.0, 1e-22, 1e-18, 1e-14, 1e-11])
@pytest.mark.parametrize("bits", [32, 8])
def test_small_gradients_and_eps(eps, bits):
    """Roots whose squares are below the normal numbers, where eps does not hide them.  A place of v is 2^-149 there: what
    64 bits make of the moments that are left is off by that, twice with the product's, beside a step's usual 2^-19; v of
    8-bit moments is the square of a root, which the codes round."""
    sizes = [300, 1000, 7]
    gen = torch.Generator(device="cuda").manual_seed(5)
    params = [torch.zeros(n, device="cuda") for n in sizes]
    grads = [torch.empty(n, device="cuda").uniform_(1e-19, 4e-18, generator=gen) for n in sizes]
    grads[0][::2] *= -1
    opt = AdamW(params, grads, lr=1.0, betas=(0.9, 0.999), eps=eps, weightDecay=0.0, stateBits=bits, min8bitSize=1)
    opt.step()
    for p, g in zip(params, grads):
        g = g.double()
        v = 0.001 * g ** 2
        off = 2.0 ** -148 / v  # of v, to its last place
        root = (v / 0.001).sqrt()
        want = -g / (root + eps)
        assert ((p.double() - want).abs() <= (2.0 ** -19 + off) * want.abs()).all()
    before, v = [p.double() for p in params], [_decode(opt, i, "r8") for i in range(3)]
    m = [_decode(opt, i, "m8") for i in range(3)]
    opt.step()
    for p, g, x, m, v in zip(params, grads, before, m, v):
        g, v = g.double(), v ** 2 if bits == 8 else v
        m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g ** 2
        root = (v / (1 - 0.999 ** 2)).sqrt()
        want = x - m / (1 - 0.9 ** 2) / (root + eps)
        assert ((p.double() - want).abs() <= (2.0 ** -18 + 3 * 2.0 ** -148 / v) * (want - x).abs() + 2.0 ** -22 * x.abs()).all()
