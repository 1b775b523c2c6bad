"""The norms around a residual block against their formulas in 64 bits.

Tolerances count roundings of u = 2^-24 (__expf and the sigmoid: 2^-20 relative).  A row's sum of d terms runs over at
most 16 in a thread and ten levels of a tree, so it is within 32 u of the sum of magnitudes; a normalised value takes
half of that from the deviation and all of it, times the mean magnitude, from the mean.  64 u of the magnitudes that
enter an output covers what is left.  The gradients of weights run over at most some 16 rows in a worker and the
workers' sums, some 600 in 32 strands: 64 u of the sum of magnitudes, on terms that are themselves within 64 u.  16-bit
outputs add half a step."""
import math

import pytest
import torch

from fbcunn_b200 import GatedResidualNorm, capi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _stat(x, kind, eps):
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    return mean, 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()


def _near(got, want, size, what):
    """|got - want| within 64 u of `size`, plus the type's half step."""
    eps = 0 if got.dtype == F32 else torch.finfo(got.dtype).eps / 2 * 1.001
    least = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    tol = 64 * U * (1 + eps) * size + eps * want.abs() + least
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got).all() and float(off.max()) <= 0, f"{what}: {float(off.max())} beyond {float(tol.max())}"


def check(m, table, grads, shared=None):
    """One step of module m on `table`, compared with the formulas."""
    u, r, gate = (table + [None])[:3] if len(table) > 1 else (None, table[0], None)
    out = m.updateOutput(table)
    r_out, v = (None, out) if u is None else (out, None) if m.pre is None else out
    d = lambda t: None if t is None else t.double()
    eps = m.eps
    x = d(r) * m.residualScale
    if u is not None:
        mean1, s1 = _stat(d(u), m.post, eps) if m.post else (0, 1)
        hat1 = (d(u) - mean1) * s1
        w1 = d(m.postWeight) if m.post else torch.ones(m.channels, dtype=torch.float64, device="cuda")
        b1 = d(m.postBias) if m.postBias is not None else 0 * w1
        n = hat1 * w1 + b1
        size_n = ((d(u).abs() + (d(u).abs().mean(-1, keepdim=True) if m.post == "layer" else 0)) * s1) * w1.abs() + b1.abs()
        act = 1 if gate is None else torch.sigmoid(d(gate)) if m.gate == "sigmoid" else d(gate)
        # where exp(-g) passes the largest number, 2^128, as at -100, the sigmoid 1 / (1 + exp(-g)) < 2^-128 is zero
        lost = 2.0 ** -128 / (64 * U) if m.gate == "sigmoid" else 0
        slack = 1 if gate is None else act.abs() + lost
        x = x + m.branchScale * act * n
        size_x = d(r).abs() * abs(m.residualScale) + abs(m.branchScale) * slack * size_n
        _near(r_out, x, size_x, "r")
    else:
        size_x = x.abs()
    if m.pre is not None:
        mean2, s2 = _stat(x, m.pre, eps)
        w2, b2 = d(m.preWeight), d(m.preBias) if m.preBias is not None else 0
        hat2 = (x - mean2) * s2
        size = (size_x + size_x.mean(-1, keepdim=True) + hat2.abs() * size_x.square().mean(-1, keepdim=True).sqrt()) * s2
        _near(v, hat2 * w2 + b2, size * w2.abs() + (b2.abs() if m.preBias is not None else 0), "v")
    if grads is None:
        return
    got = m.backward(table, grads if m.pre is not None and u is not None else grads[-1] if m.pre is not None else grads[0])
    D = 0 * x if u is None else d(grads[0])
    size_D = D.abs()
    rows = tuple(range(x.dim() - 1))
    if m.pre is not None:
        off2 = (size_x + size_x.mean(-1, keepdim=True)) * s2  # what an error of a few u in r' is worth
        dv = d(grads[1])
        gw = dv * w2
        D = D + s2 * (gw - hat2 * (gw * hat2).mean(-1, keepdim=True) - (gw.mean(-1, keepdim=True) if m.pre == "layer" else 0))
        size_D = size_D + s2 * (gw.abs() + off2 * (gw * hat2).abs().mean(-1, keepdim=True) + gw.abs().mean(-1, keepdim=True)
                                + hat2.abs() * (gw.abs() * off2).mean(-1, keepdim=True))
        _near(m.gradPreWeight, (dv * hat2).sum(rows), (dv.abs() * off2).sum(rows), "gradPreWeight")
        if m.preBias is not None:
            _near(m.gradPreBias, dv.sum(rows), dv.abs().sum(rows), "gradPreBias")
    dr = got if u is None else got[1]
    _near(dr, m.residualScale * D, abs(m.residualScale) * size_D, "dr")
    if u is None:
        return
    dn, size_dn = m.branchScale * act * D, abs(m.branchScale) * slack * size_D
    if gate is not None:
        slope = act * (1 - act) if m.gate == "sigmoid" else torch.ones_like(act)
        dg = m.branchScale * D * n * slope
        size_g = abs(m.branchScale) * (size_D * n.abs() + D.abs() * size_n) * slope.abs() * 2
        if m.gate == "sigmoid":
            # act (1 - act) of a saturated gate loses what 1 - act has: 2^-23 of act
            size_g = 9 * size_g + lost * size_D * size_n
        for dim, (a, b) in enumerate(zip(x.shape[:-1], (1,) * (x.dim() - gate.dim()) + tuple(gate.shape[:-1]))):
            if a != b:
                dg, size_g = dg.sum(dim, keepdim=True), size_g.sum(dim, keepdim=True)
        _near(got[2], dg.view(gate.shape), size_g.view(gate.shape), "dgate")
    du, size_du = dn, size_dn
    if m.post is not None:
        off1 = (d(u).abs() + (d(u).abs().mean(-1, keepdim=True) if m.post == "layer" else 0)) * s1
        gw, size_gw = dn * w1, size_dn * w1.abs()
        du = s1 * (gw - hat1 * (gw * hat1).mean(-1, keepdim=True) - (gw.mean(-1, keepdim=True) if m.post == "layer" else 0))
        size_du = s1 * (size_gw + off1 * (size_gw * off1).mean(-1, keepdim=True) * 2 + size_gw.mean(-1, keepdim=True))
        _near(m.gradPostWeight, (dn * hat1).sum(rows), (size_dn * off1 * 2).sum(rows), "gradPostWeight")
        if m.postBias is not None:
            _near(m.gradPostBias, dn.sum(rows), size_dn.sum(rows), "gradPostBias")
    _near(got[0], du, size_du, "du")


def build(shape, channels, dtype=F32, residual=None, per="token", seed=0, **kw):
    """A module with weights off their first values, its table and gradients."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s, dtype=dtype):
        return torch.empty(s, device="cuda").normal_(generator=gen).to(dtype)

    m = GatedResidualNorm(channels, residualScale=0.9, branchScale=0.5, **kw)
    for w in m.parameters()[0]:
        w.add_(0.2 * normal(channels, dtype=F32))
    residual = residual or dtype
    table = [normal(*shape, channels), 2 * normal(*shape, channels, dtype=residual)]
    if m.gate is not None:
        table.append(normal(*{"token": shape, "sequence": (shape[0],) + (1,) * (len(shape) - 1), "all": ()}[per], channels))
    return m, table, [normal(*shape, channels, dtype=residual), normal(*shape, channels)]


FORMS = [dict(), dict(post="layer", pre="layer", normBias=True), dict(gate="sigmoid"), dict(gate="linear", normBias=True),
         dict(post=None), dict(post=None, gate="sigmoid", pre="layer"), dict(pre=None), dict(pre=None, post="layer", gate="linear")]


@pytest.mark.parametrize("form", range(len(FORMS)))
@pytest.mark.parametrize("dtype,residual", [(F32, F32), (BF, BF), (BF, F32), (HF, HF), (HF, F32)])
def test_forms_and_types(form, dtype, residual):
    check(*build((3, 17), 200, dtype, residual, **FORMS[form]))
    check(*build((2, 5), 1000, dtype, residual, seed=1, **FORMS[form]))


@pytest.mark.parametrize("channels", [1, 2, 7, 31, 33, 255, 256, 264, 500, 513, 1024, 2056, 4096, 4097, 5120, 8192, 8200,
                                      12288, 16384])
def test_widths(channels):
    kw = dict(post="layer", gate="sigmoid", normBias=True)
    # one channel leaves a layer norm nothing: both formulas are all rounding there
    if channels == 1:
        kw["post"] = "rms"
    check(*build((5,), channels, F32, **kw))
    check(*build((3,), channels, BF, F32, seed=2, **kw))
    check(*build((2,), channels, HF, seed=3, gate="linear"))


@pytest.mark.parametrize("per", ["token", "sequence", "all"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 700), (5, 77), (700, 3), (2000, 1), (3, 1500), (4, 5, 6)])
def test_shared_gates(shape, per):
    check(*build(shape, 96, BF, F32, per=per, gate="sigmoid"))
    check(*build(shape, 1030, F32, per=per, gate="linear", post="layer", normBias=True, seed=4))


def test_entry_to_the_first_block():
    for kind in ("rms", "layer"):
        m, table, grads = build((4, 9), 320, BF, post=None, pre=kind, normBias=True)
        m.residualScale = 1.0
        check(m, [table[0]], grads)
        assert torch.equal(m.updateOutput(table[0]), m.updateOutput([table[0]]))


def test_strided_rows():
    """Parts of one projection's output, and sequences that are cut short where the rows stay evenly apart."""
    m, table, grads = build((4, 6), 256, BF, gate="sigmoid", seed=5)
    wide = torch.cat([table[2], table[0], table[2]], -1)
    rest = torch.cat([table[1], table[1]], -1)
    check(m, [wide[..., 256:512], rest[..., 256:], wide[..., :256]], grads)
    odd = torch.zeros(4, 6, 1 + 256, dtype=BF, device="cuda")
    odd[..., 1:] = table[0]
    check(m, [odd[..., 1:], table[1], table[2]], grads)
    with pytest.raises(AssertionError):
        m.updateOutput([torch.cat([table[0], table[0]], 1)[:, :6], table[1], table[2]])  # two distances between rows
    with pytest.raises(AssertionError):
        m.updateOutput([table[0][..., ::2], table[1], table[2]])
    with pytest.raises(AssertionError):
        m.updateOutput([table[0], table[1], table[2][:1].expand(4, 6, 256)])


def test_rows_of_zeros_and_extremes():
    m, table, grads = build((6,), 512, F32, gate="sigmoid")
    table[0][1] = 0  # eps alone
    table[1][1] = 0
    table[0][2] *= 1e15
    table[1][3] *= 1e-15
    table[2][4] = 100.0
    table[2][5] = -100.0
    check(m, table, grads)
    table[0][0, 7] = float("nan")
    out = m.updateOutput(table)
    assert torch.isnan(out[1][0]).all() and torch.isfinite(out[1][1:]).all()


def test_no_rows():
    m, table, grads = build((0, 3), 64, F32, gate="linear", normBias=True)
    m.gradPreWeight.fill_(3)
    out = m.updateOutput(table)
    assert out[0].shape == out[1].shape == (0, 3, 64)
    got = m.backward(table, grads)
    assert [t.shape for t in got] == [t.shape for t in table]
    assert not m.gradPreWeight.any() and not m.gradPostBias.any()


def test_gradients_against_differences():
    m, table, grads = build((3, 4), 48, F32, gate="sigmoid", post="layer", normBias=True, per="sequence")
    def loss():
        out = m.updateOutput(table)
        return float((out[0].double() * grads[0]).sum() + (out[1].double() * grads[1]).sum())
    loss()
    got = [g.clone() for g in m.backward(table, grads)]
    params, dparams = m.parameters()
    gen = torch.Generator(device="cuda").manual_seed(9)
    for t, g in list(zip(table, got)) + [(p, d.clone()) for p, d in zip(params, dparams)]:
        way = torch.empty_like(t).normal_(generator=gen)
        step, start = 2.0 ** -7, t.clone()
        t.copy_(start + step * way)
        up = loss()
        t.copy_(start - step * way)
        down = loss()
        t.copy_(start)
        # third derivatives of order one times step^2 / 6 = 1e-5, and 64 u of some 600 terms over the step: 3e-3
        want = float((g.double() * way).sum())
        assert abs((up - down) / (2 * step) - want) <= 1e-2 * max(1.0, float(g.norm()))


def test_accumulated_and_separate_passes():
    m, table, grads = build((5, 8), 160, BF, F32, gate="sigmoid", normBias=True)
    m.updateOutput(table)
    whole = [g.clone() for g in m.backward(table, grads, 0.5)]
    sums = [g.clone() for g in m.parameters()[1]]
    alone = m.updateGradInput(table, grads)
    assert all(torch.equal(a, b) for a, b in zip(whole, alone))
    kept = m.gradInput
    m.zeroGradParameters()
    m.accGradParameters(table, grads, 0.5)
    assert m.gradInput is kept and all(torch.equal(a, b) for a, b in zip(kept, whole))
    assert all(torch.equal(a, b) for a, b in zip(sums, m.parameters()[1]))
    m._accumulate = True
    m.backward(table, grads, 0.5)
    for a, b in zip(sums, m.parameters()[1]):
        assert torch.equal(2 * a, b)


def test_the_same_bits_every_time_and_when_replayed():
    m, table, grads = build((7, 300), 768, BF, gate="sigmoid", per="sequence", normBias=True)
    def outputs():
        out = m.updateOutput(table)
        return [t.clone() for t in out] + [t.clone() for t in m.backward(table, grads)] + [t.clone() for t in m.parameters()[1]]
    first = outputs()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, outputs()))
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        m.updateOutput(table)
        m.backward(table, grads)
    torch.cuda.synchronize()
    for t in m.output + m.gradInput + m.parameters()[1]:
        t.zero_()
    graph.replay()
    again = [t.clone() for t in m.output] + [t.clone() for t in m.gradInput] + [t.clone() for t in m.parameters()[1]]
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_backward_wants_the_forward_pass():
    m, table, grads = build((2, 3), 64)
    with pytest.raises(AssertionError):
        m.backward(table, grads)
    m.evaluate()
    m.updateOutput(table)
    with pytest.raises(AssertionError):
        m.backward(table, grads)
    m.training()
    m.updateOutput(table)
    with pytest.raises(AssertionError):
        m.backward([t[:1] for t in table], [g[:1] for g in grads])


def test_refusals():
    m, table, grads = build((2, 6), 64, BF, gate="sigmoid")
    with pytest.raises(AssertionError):
        m.updateOutput(table[:2])
    with pytest.raises(AssertionError):
        m.updateOutput([table[0], table[1][..., :32], table[2]])
    with pytest.raises(AssertionError):
        m.updateOutput([table[0], table[1].half(), table[2]])
    with pytest.raises(AssertionError):
        m.updateOutput([table[0].cpu(), table[1], table[2]])
    with pytest.raises(AssertionError):
        m.updateOutput([table[0], table[1], table[2][:1]])  # rows 0, 6 would share a gate row
    m.updateOutput(table)
    with pytest.raises(AssertionError):
        m.backward(table, [grads[0], grads[1].float()])
    lib, none = capi.lib(), [None] * 11
    rc = lib.fbfftconv_residual_norm(m._desc_ref, *none)
    assert rc == capi.ERR_INVALID_ARGUMENT
    host = torch.zeros(2, 6, 64, dtype=BF)
    launches = capi.kernel_launches()
    args = [t.data_ptr() for t in table] + [m.postWeight.data_ptr(), None, m.preWeight.data_ptr(), None,
                                            m.output[0].data_ptr(), host.data_ptr(), None, None]
    assert lib.fbfftconv_residual_norm(m._desc_ref, *args) == capi.ERR_INVALID_ARGUMENT
    assert "norm's output" in capi.last_error() and capi.kernel_launches() == launches


def test_graphs_of_several_shapes():
    """A graph captured for one batch is replayed after other batches have run through the module."""
    m = GatedResidualNorm(96, gate="sigmoid")
    made = {}
    for n in (3, 8):
        table = [torch.randn(n, 5, 96, device="cuda") for _ in range(3)]
        grads = [torch.randn(n, 5, 96, device="cuda") for _ in range(2)]

        def work(table=table, grads=grads):
            return [*m.updateOutput(table), *m.backward(table, grads), *m.parameters()[1]]

        work()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            outputs = work()
        torch.cuda.synchronize()
        made[n] = graph, outputs, work
    fill = [torch.full((n, 5, 96), 7.0, device="cuda") for n in range(1, 40)]
    for graph, outputs, work in made.values():
        graph.replay()
        got = [t.clone() for t in outputs]
        for a, b in zip(got, work()):
            assert torch.equal(a, b)
    assert all((t == 7).all() for t in fill)


def test_a_replaced_weight_is_looked_at():
    m, table, _ = build((2, 3), 64)
    m.updateOutput(table)
    m.preWeight = torch.ones(32, device="cuda")
    with pytest.raises(AssertionError):
        m.updateOutput(table)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("channels", [320, 321])
def test_no_scale_touches_the_entry_to_the_first_block(kind, channels):
    """v = pre(r) whatever residualScale is, and its gradients: the same bits as with a scale of one."""
    got = []
    for scale in (1.0, 0.9, 0.0):
        m, table, grads = build((4, 9), channels, BF, post=None, pre=kind, normBias=True)
        m.residualScale = scale
        v = m.updateOutput([table[0]])
        got.append([v, m.backward([table[0]], grads[1]), *m.parameters()[1]])
    x = table[0].double()
    mean, s = _stat(x, kind, m.eps)
    gw, hat = grads[1].double() * m.preWeight.double(), (x - mean) * s
    want = s * (gw - hat * (gw * hat).mean(-1, keepdim=True) - (gw.mean(-1, keepdim=True) if kind == "layer" else 0))
    off = (x.abs() + x.abs().mean(-1, keepdim=True)) * s
    size = s * (gw.abs() + off * (gw * hat).abs().mean(-1, keepdim=True) + gw.abs().mean(-1, keepdim=True)
                + hat.abs() * (gw.abs() * off).mean(-1, keepdim=True))
    _near(got[0][1], want, size, "dr")
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("gate", [(3, 1, 96), (1, 96), (96,)])
def test_the_gate_of_no_rows_has_a_gradient_of_zero(gate, dtype):
    """Sequences without rows leave a gate of each sequence, or of all rows, as it is: nothing has used it."""
    m = GatedResidualNorm(96, gate="linear")
    empty = torch.empty(3, 0, 96, dtype=dtype, device="cuda")
    table = [empty, empty.clone(), torch.ones(gate, dtype=dtype, device="cuda")]
    for _ in range(2):
        m.updateOutput(table)
        dgate = m.backward(table, [empty, empty])[2]
        assert dgate.shape == torch.Size(gate) and not dgate.any()
        dgate.fill_(float("nan"))


def test_one_module_at_several_borders():
    """A module that is shared by blocks takes its own outputs in; each backward pass has the inputs that it was given."""
    m, (u, r), grads = build((6,), 96, F32)
    twin, *_ = build((6,), 96, F32)
    r1, v1 = m.updateOutput([u, r])
    want = [t.clone() for t in (r1, v1)]
    second = m.updateOutput([v1, r1])
    assert torch.equal(r1, want[0]) and torch.equal(v1, want[1])
    got = [t.clone() for t in second + m.backward([v1, r1], grads)]
    table = want[::-1]
    for a, b in zip(got, twin.updateOutput(table) + twin.backward(table, grads)):
        assert torch.equal(a, b)
