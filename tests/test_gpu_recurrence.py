"""The gated linear recurrence against its formulas in 64 bits, row by row.

Tolerances, with u = 2^-24 and eps = (|g| + 4) 2^-23 the relative error of the smaller of a and 1 - a (exp's argument
carries |g| u, exp and quotient a few u).  a + (1 - a) = 1 to u / 2, so an error of the gate moves h by eps (1 - a)
|x - h|, in all at most 2 eps M with M the largest |x|, |h|; rounding and joining of stretches adds some 6 u M a row for
as many rows as the memory reaches, N = min(length, 1 / min(1 - a)).  D sums |e| with weights a: S_t = |e_t| + a_{t+1}
S_{t+1}, within S (6 u N + 4 eps).  Products add their factors' errors.  Below the normal numbers (|g| > 87) the smaller of a and 1 - a
is good to 2^-126 alone (`lost`), which is added to eps times it there.  16-bit outputs add half a step."""
import os
import subprocess
import sys

import pytest
import torch

from fbcunn_b200 import GatedLinearRecurrence, capi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


def _near(got, want, tol, what):
    eps = 0 if got.dtype == F32 else torch.finfo(got.dtype).eps / 2 * 1.001
    least = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got.double() - want).abs() - (tol * (1 + eps) + eps * want.abs() + least)
    assert torch.isfinite(got).all() and (not off.numel() or float(off.max()) <= 0), f"{what}: {float(off.max())} too far"


def reference(x, g, z, bias, offsets, state, dy=None, dstate=None):
    """Every output and its tolerance, on flat rows."""
    x, g, z, bias, state, dy, dstate = (None if t is None else t.double().cpu() for t in (x, g, z, bias, state, dy, dstate))
    g = g if bias is None else g + bias
    a, b = torch.sigmoid(g), torch.sigmoid(-g)
    n = len(offsets) - 1
    h, prev = torch.zeros_like(x), torch.zeros_like(x)
    final = torch.zeros(n, x.shape[1], dtype=torch.float64) if state is None else state.clone()
    reach, largest = torch.zeros_like(x), torch.zeros_like(x)
    eps = (g.abs() + 4) * 2.0 ** -23
    for i in range(n):
        lo, hi = offsets[i], offsets[i + 1]
        if lo == hi:
            continue
        cur = final[i]
        rows = slice(lo, hi)
        reach[rows] = (1 / b[rows].amin(0)).clamp(max=hi - lo)
        largest[rows] = torch.maximum(x[rows].abs().amax(0), cur.abs())
        for t in range(lo, hi):
            prev[t] = cur
            cur = a[t] * cur + b[t] * x[t]
            h[t] = cur
        final[i] = cur
        eps[rows] = eps[rows].amax(0)
    lost = 2.0 ** -126 * (g.abs() > 87)
    tol_h = largest * (2 * eps + 6 * U * reach + lost * reach)
    out = {}
    sz = torch.sigmoid(z) if z is not None else None
    soft = (z.abs() + 6) * 2.0 ** -22 if z is not None else None
    out["y"] = (h, tol_h) if z is None else (h * z * sz, (z * sz).abs() * (tol_h + largest * soft))
    last = [offsets[i + 1] - 1 for i in range(n) if offsets[i + 1] > offsets[i]]
    keep = [i for i in range(n) if offsets[i + 1] > offsets[i]]
    tol_f = torch.zeros_like(final)
    tol_f[keep] = tol_h[last]
    out["state"] = (final, tol_f)
    if dy is None:
        return out
    e = dy * z * sz if z is not None else dy.clone()
    size = e.abs() * (1 + (soft if soft is not None else 0))
    if dstate is not None:
        e[last] += dstate[keep]
        size[last] += dstate[keep].abs()
    soft_e = e.abs() * soft if soft is not None else 0 * e
    D, S, G = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    d0, s0 = (torch.zeros_like(final) if dstate is None else dstate.clone()), torch.zeros_like(final)
    for i in keep:
        flow, sums, slack = 0, 0, 0
        for t in reversed(range(offsets[i], offsets[i + 1])):
            D[t], S[t], G[t] = e[t] + flow, size[t] + sums, soft_e[t] + slack
            flow, sums, slack = a[t] * D[t], a[t] * S[t], a[t] * G[t]
        d0[i] = flow
        first = offsets[i]
        s0[i] = a[first] * (S[first] * (6 * U * reach[first] + 6 * eps[first]) + G[first]) + lost[first] * S[first]
    tol_D = S * (6 * U * reach + 4 * eps) + G
    out["dx"] = (b * D, b * (tol_D + S * 2 * eps) + lost * S)
    dg = D * (prev - x) * a * b
    tol_g = a * b * ((tol_D + S * 6 * eps) * 2 * largest + S * (tol_h + 4 * U * largest)) + lost * S * 2 * largest
    out["dg"] = (dg, tol_g)
    out["dbias"] = (dg.sum(0), tol_g.sum(0) + 64 * U * dg.abs().sum(0))
    out["dstate"] = (d0, s0)
    if z is not None:
        slope = sz * (1 + z * (1 - sz))
        out["dz"] = (dy * h * slope, dy.abs() * (1.1 * tol_h + largest * (z.abs() + 8) * 2.0 ** -21))
    return out


def make(rows, sequences, channels, dtype=F32, gate=True, state=True, seed=0, shift=0):
    """A module, its table as parts of one projection (`shift` channels off a pair's alignment), gradient, states."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s, dtype=F32):
        return torch.empty(s, device="cuda").normal_(generator=gen).to(dtype)

    parts = 3 if gate else 2
    wide = normal(*rows, parts * channels + shift, dtype=dtype)
    table = list(wide[..., shift:].split(channels, -1))
    m = GatedLinearRecurrence(channels, outputGate=gate)
    m.bias.copy_(torch.linspace(-2, 5, channels, device="cuda"))
    h0 = normal(sequences, channels) if state else None
    return m, table, normal(*rows, channels, dtype=dtype), h0, normal(sequences, channels) if state else None


def check(m, table, dy, h0, dlast, offsets=None, lengths=None):
    y = m.updateOutput(table, state=h0, offsets=offsets)
    grads = m.backward(table, dy, state=h0, offsets=offsets, gradState=dlast)
    d = m.channels
    borders = offsets.tolist() if offsets is not None else [i * table[0].shape[1] for i in range(table[0].shape[0] + 1)]
    flat = [t.reshape(-1, d) for t in table] + [None] * (3 - len(table))
    want = reference(*flat, m.bias, borders, h0, dy.reshape(-1, d), dlast)
    got = {"y": y, "state": m.state, "dbias": m.gradBias, **dict(zip(("dx", "dg", "dz"), grads))}
    if h0 is not None:
        got["dstate"] = m.gradState
    inside = slice(borders[0], borders[-1])
    for k, t in got.items():
        w, tol = want[k]
        if k in ("y", "dx", "dg", "dz"):
            _near(t.reshape(-1, d).cpu()[inside], w[inside], tol[inside], k)
        else:
            _near(t.cpu(), w, tol, k)


SHAPES = [(1, 1, 2), (3, 1, 64), (2, 7, 5), (1, 63, 64), (1, 64, 66), (1, 65, 128), (2, 200, 130), (5, 129, 33), (300, 3, 10),
          (40, 17, 200), (2, 300, 520), (1, 1500, 96), (1, 2049, 32)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,gate,state", [(F32, True, True), (BF, True, False), (HF, False, True), (F32, False, False)])
def test_padded(shape, dtype, gate, state):
    B, T, D = shape
    check(*make((B, T), B, D, dtype, gate, state))


@pytest.mark.parametrize("lengths", [[5], [0, 3, 0, 0, 70, 1, 1, 0], [64, 64, 64], [1] * 200, [16, 0, 16, 47, 1, 128, 300],
                                     [700, 0, 900, 3], [0, 0]])
@pytest.mark.parametrize("dtype,wide", [(F32, False), (BF, True)])
def test_packed(lengths, dtype, wide):
    """Rows before the first and behind the last sequence stay as they are."""
    ends = torch.tensor([0] + lengths).cumsum(0)
    rows = int(ends[-1]) + 10
    offsets = (ends + 4).to("cuda", torch.int64 if wide else torch.int32)
    m, table, dy, h0, dlast = make((rows,), len(lengths), 72, dtype)
    m.updateOutput(table, state=h0, offsets=offsets)
    m.backward(table, dy, state=h0, offsets=offsets, gradState=dlast)
    m.output.fill_(3)
    m.gradProjection.fill_(4)
    check(m, table, dy, h0, dlast, offsets)
    for t, mark in ((m.output, 3), (m.gradProjection, 4)):
        assert (t[:4] == mark).all() and (t[-6:] == mark).all()


def test_more_sequences_than_are_kept_on_the_chip():
    """The search goes to memory for more than 512 sequences."""
    lengths = [(7 * i) % 5 for i in range(700)]
    offsets = torch.tensor([0] + lengths).cumsum(0).to("cuda", torch.int32)
    check(*make((int(offsets[-1]),), 700, 48, BF), offsets=offsets)


def test_one_of_the_two_states():
    m, table, dy, h0, dlast = make((2, 90), 2, 32, F32)
    check(m, table, dy, h0, None)
    m.updateOutput(table)
    grads = [g.clone() for g in m.backward(table, dy, gradState=dlast)]
    want = reference(*[t.reshape(-1, 32) for t in table], m.bias, [0, 90, 180], torch.zeros_like(h0), dy.reshape(-1, 32), dlast)
    for k, t in zip(("dx", "dg", "dz"), grads):
        _near(t.reshape(-1, 32).cpu(), *want[k], k)
    _near(m.gradState.cpu(), *want["dstate"], "dstate")


def test_channels_off_their_pairs():
    check(*make((2, 100), 2, 66, BF, shift=1))
    check(*make((3, 50), 3, 31, HF, shift=3))
    m, table, dy, h0, dlast = make((90,), 4, 40, BF, shift=1, seed=3)
    check(m, table, dy, h0, dlast, torch.tensor([0, 30, 30, 77, 90], dtype=torch.int32, device="cuda"))


def test_extreme_gates():
    m, table, dy, h0, dlast = make((2, 150), 2, 16, F32)
    m.bias.zero_()
    g = torch.zeros(2, 150, 16, device="cuda")
    g[..., 0], g[..., 1], g[..., 2], g[..., 3] = 100.0, -100.0, float("inf"), float("-inf")
    g[..., 4], g[..., 5], g[:, ::2, 6], g[:, 1::2, 6] = 20.0, -20.0, 30.0, -30.0
    table[1] = g
    y = m.updateOutput(table, state=h0)
    s = table[2] * torch.sigmoid(table[2])
    assert torch.allclose(y[..., 2], h0[:, None, 2] * s[..., 2], rtol=1e-5) and torch.allclose(y[..., 3], table[0][..., 3] * s[..., 3], rtol=1e-5)
    g[..., 2:4] = 1.0  # the oracle's |g| eps has no infinities
    check(m, table, dy, h0, dlast)


def test_nothing_reaches_the_next_sequence():
    for bad in (float("nan"), float("inf")):
        m, table, dy, h0, dlast = make((200,), 3, 64, BF)
        offsets = torch.tensor([0, 70, 130, 200], dtype=torch.int32, device="cuda")
        clean = [t.clone() for t in [m.updateOutput(table, state=h0, offsets=offsets), m.state] +
                 m.backward(table, dy, state=h0, offsets=offsets, gradState=dlast) + [m.gradState]]
        table[0][75, 3] = bad
        dy[126, 5] = bad
        y = m.updateOutput(table, state=h0, offsets=offsets)
        grads = m.backward(table, dy, state=h0, offsets=offsets, gradState=dlast)
        for t, c in zip([y] + grads, [clean[0]] + clean[2:5]):
            assert torch.equal(t[:70], c[:70]) and torch.equal(t[130:], c[130:])
        assert not torch.isfinite(y[75:130, 3].float()).any() and torch.isfinite(y[70:75].float()).all()
        assert not torch.isfinite(grads[0][70:127, 5].float()).any()
        for t, c in ((m.state, clean[1]), (m.gradState, clean[5])):
            assert torch.equal(t[0], c[0]) and torch.equal(t[2], c[2])


def test_one_cluster_of_blocks_and_many_segments():
    """Long sequences of few channels go over clusters, many sequences over segments: a second shape of each, whose sums
    are those of rows one at a time."""
    m, table, dy, h0, dlast = make((1, 6000), 1, 64, BF, seed=5)
    check(m, table, dy, h0, dlast)
    m, table, dy, h0, dlast = make((600, 9), 600, 64, F32, seed=6)
    check(m, table, dy, h0, dlast)


def test_bad_offsets_stay_in_the_tensors():
    """Offsets that fall or point outside: every read is clamped (see the host's copy of the search), nothing hangs."""
    m, table, dy, h0, dlast = make((300,), 5, 64, F32)
    m.updateOutput(table, state=h0, offsets=torch.tensor([0, 60, 120, 180, 240, 300], dtype=torch.int32, device="cuda"))
    for bad in ([0, 200, 100, 150, 90, 300], [-5, 10, 20, 30, 40, 10 ** 6], [300, 200, 100, 50, 20, 0], [7, 7, 7, 7, 7, 7],
                [0, 10 ** 9, -10 ** 9, 64, 64, 200]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        m.updateOutput(table, state=h0, offsets=offsets)
        m.backward(table, dy, state=h0, offsets=offsets, gradState=dlast)
        torch.cuda.synchronize()


def test_no_rows_and_no_sequences():
    for B, T in ((3, 0), (0, 5), (0, 0)):
        m, table, dy, h0, dlast = make((B, T), B, 32, F32)
        y = m.updateOutput(table, state=h0)
        assert y.shape == (B, T, 32) and torch.equal(m.state, h0)
        m.gradBias.fill_(2)
        grads = m.backward(table, dy, state=h0, gradState=dlast)
        assert grads[0].shape == (B, T, 32) and torch.equal(m.gradState, dlast) and not m.gradBias.any()


@pytest.mark.parametrize("dtype,channels,shift", [(F32, 40, 0), (BF, 64, 0), (HF, 33, 1)])
def test_steps_follow_the_whole_sequence(dtype, channels, shift):
    """A prompt, then tokens one at a time, as serving runs it."""
    m, table, _, h0, _ = make((3, 20), 3, channels, dtype, shift=shift)
    m.evaluate()
    whole = m.updateOutput(table, state=h0).clone()
    final = m.state.clone()
    m.updateOutput([t[:, :12].contiguous() for t in table], state=h0)
    state = m.state.clone()
    want = reference(*[t.reshape(-1, channels) for t in table], m.bias, [0, 20, 40, 60], h0)
    for t in range(12, 20):
        y = m.step([p[:, t] for p in table], state)
        value, tol = (w.view(3, 20, -1)[:, t] for w in want["y"])
        _near(y.cpu(), value, tol, "y")
    _near(state.cpu(), *want["state"], "state")
    _near(final.cpu(), *want["state"], "state")
    assert torch.allclose(whole[:, -1].float(), y.float(), rtol=2e-2, atol=1e-2)


def test_the_state_goes_on_where_it_was_left():
    """The state that one call leaves is the next call's: also where it is the module's own tensor."""
    m, table, _, h0, _ = make((2, 60), 2, 32, F32)
    want = reference(*[t.reshape(-1, 32) for t in table], m.bias, [0, 60, 120], h0)
    m.evaluate()
    m.updateOutput([t[:, :30].contiguous() for t in table], state=h0)
    y = m.updateOutput([t[:, 30:].contiguous() for t in table], state=m.state)
    value, tol = (w.view(2, 60, -1)[:, 30:] for w in want["y"])
    _near(y.cpu(), value, tol, "y")
    _near(m.state.cpu(), *want["state"], "state")


def test_gradients_against_differences():
    m, table, dy, h0, dlast = make((2, 40), 2, 24, F32, seed=8)
    table = [t.contiguous() for t in table]
    def loss():
        return float((m.updateOutput(table, state=h0).double() * dy).sum() + (m.state.double() * dlast).sum())
    loss()
    grads = [g.clone() for g in m.backward(table, dy, state=h0, gradState=dlast)] + [m.gradBias.clone(), m.gradState.clone()]
    gen = torch.Generator(device="cuda").manual_seed(9)
    for t, g in zip(table + [m.bias, h0], grads):
        way, step, start = torch.empty_like(t).normal_(generator=gen), 2.0 ** -8, t.clone()
        t.copy_(start + step * way)
        up = loss()
        t.copy_(start - step * way)
        down = loss()
        t.copy_(start)
        # third derivatives of some ten times step^2 / 6, and 1e-6 of 2000 terms over the step: 1e-2 of the gradient's norm
        assert abs((up - down) / (2 * step) - float((g.double() * way).sum())) <= 1e-2 * max(1.0, float(g.norm()))


def test_separate_passes_and_accumulated_gradients():
    m, table, dy, h0, dlast = make((3, 70), 3, 48, BF)
    m.updateOutput(table, state=h0)
    whole = [g.clone() for g in m.backward(table, dy, 0.5, state=h0, gradState=dlast)]
    bias, dstate = m.gradBias.clone(), m.gradState.clone()
    m.gradBias.fill_(7)
    alone = m.updateGradInput(table, dy, state=h0, gradState=dlast)
    assert all(torch.equal(a, b) for a, b in zip(whole, alone)) and torch.equal(m.gradState, dstate) and (m.gradBias == 7).all()
    m.gradProjection.fill_(1)
    m.accGradParameters(table, dy, 0.5, state=h0, gradState=dlast)
    assert (m.gradProjection == 1).all() and torch.equal(m.gradBias, bias)
    m._accumulate = True
    m.accGradParameters(table, dy, 0.5, state=h0, gradState=dlast)
    assert torch.equal(m.gradBias, 2 * bias)
    plain = GatedLinearRecurrence(48, bias=False)
    plain.updateOutput(table)
    plain.backward(table, dy)
    assert plain.parameters() == ([], []) and plain.gradState is None


def test_the_same_bits_every_time_and_when_replayed():
    m, table, dy, h0, dlast = make((1, 3000), 1, 128, BF)
    def outputs():
        y = m.updateOutput(table, state=h0)
        grads = m.backward(table, dy, state=h0, gradState=dlast)
        return [t.clone() for t in [y, m.state, *grads, m.gradBias, m.gradState]]
    first = outputs()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, outputs()))
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        m.updateOutput(table, state=h0)
        m.backward(table, dy, state=h0, gradState=dlast)
    torch.cuda.synchronize()
    kept = [m.output, m.state, *m.gradInput, m.gradBias, m.gradState]
    for t in kept:
        t.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, kept))


def test_two_modules_on_two_streams():
    made = [make((2, 900), 2, 96, BF, seed=s) for s in (1, 2)]
    want = []
    for m, table, dy, h0, dlast in made:
        m.updateOutput(table, state=h0)
        want.append([t.clone() for t in m.backward(table, dy, state=h0, gradState=dlast)] + [m.gradBias.clone()])
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (m, table, dy, h0, dlast) in zip(streams, made):
            with torch.cuda.stream(s):
                m.updateOutput(table, state=h0)
                m.backward(table, dy, state=h0, gradState=dlast)
    torch.cuda.synchronize()
    for w, (m, *_) in zip(want, made):
        assert all(torch.equal(a, b) for a, b in zip(w, [*m.gradInput, m.gradBias]))


def test_refusals():
    m, table, dy, h0, dlast = make((2, 6), 2, 64, BF)
    with pytest.raises(AssertionError):
        m.backward(table, dy)
    with pytest.raises(AssertionError):
        m.updateOutput(table[:2])
    with pytest.raises(AssertionError):
        m.updateOutput([table[0], table[1], table[2].float()])
    with pytest.raises(AssertionError):
        m.updateOutput(table, state=h0.bfloat16())
    with pytest.raises(AssertionError):
        m.updateOutput([t[0] for t in table])  # two dimensions without offsets
    with pytest.raises(AssertionError):
        m.updateOutput(table, offsets=torch.tensor([0, 6, 12], device="cuda"))
    with pytest.raises(AssertionError):
        m.updateOutput([t[0] for t in table], offsets=torch.tensor([0, 6], device="cuda").float())
    with pytest.raises(AssertionError):
        m.updateOutput([t[0].cpu() for t in table], offsets=torch.tensor([0, 6]))
    with pytest.raises(AssertionError):
        m.step([t[:, 0] for t in table], h0[:1])
    m.evaluate()
    m.updateOutput(table, state=h0)
    with pytest.raises(AssertionError):
        m.backward(table, dy, state=h0)
    lib = capi.lib()
    launches = capi.kernel_launches()
    p = [t.data_ptr() for t in table]
    host = torch.zeros(2, 6, 64, dtype=BF)
    state = torch.empty_like(h0)
    assert lib.fbfftconv_recurrence(m._desc_ref, *p, None, None, host.data_ptr(), state.data_ptr(), None, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.fbfftconv_recurrence(m._desc_ref, *p, None, h0.data_ptr(), m.output.data_ptr(), h0.data_ptr(), None, None) == capi.ERR_INVALID_ARGUMENT
    assert capi.kernel_launches() == launches


def test_a_wait_that_nothing_ends_gives_up():
    """Clusters of blocks wait for one another's results; the limit of such a wait, on a barrier nothing completes."""
    lib = capi.lib()
    capi.check(lib.fbfftconv_recurrence_wait_selftest(torch.cuda.current_stream().cuda_stream))
    m, table, dy, h0, dlast = make((1, 3000), 1, 64, BF, seed=7)
    check(m, table, dy, h0, dlast)
    assert lib.fbfftconv_recurrence_status(0) == 0


def test_graphs_of_several_shapes():
    """A graph captured for one batch is replayed after other batches have run through the module, as a server with one
    graph for each batch size does it: nothing else may have taken the memory that the graph writes."""
    m = GatedLinearRecurrence(64)
    m.bias.normal_()
    made, graphs = {}, {}
    for n in (2, 5, 9):
        x = [torch.randn(n, 64, device="cuda") for _ in range(3)]
        long = [torch.randn(n, 20, 64, device="cuda") for _ in range(3)]
        state, dy = torch.randn(n, 64, device="cuda"), torch.randn(n, 20, 64, device="cuda")

        def work(x=x, long=long, state=state, dy=dy):
            y = m.step(x, state)
            return [y, m.updateOutput(long), *m.backward(long, dy), m.gradBias]

        work()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs[n] = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(graphs[n], stream=side):
            made[n] = (work(), state, work)
        torch.cuda.synchronize()
    fill = [torch.full((n, 20, 64), 7.0, device="cuda") for n in range(1, 40)]  # what freed memory would be given to
    for n, (outputs, state, work) in made.items():
        start = state.clone()
        graphs[n].replay()
        got = [t.clone() for t in outputs]
        state.copy_(start)
        m.gradBias.zero_()
        for a, b in zip(got, work()):
            assert torch.equal(a, b)
    assert all((t == 7).all() for t in fill)


def test_a_replaced_bias_is_looked_at():
    m, table, *_ = make((1, 4), 1, 32)
    m.updateOutput(table)
    m.bias = torch.zeros(16, device="cuda")
    with pytest.raises(AssertionError):
        m.updateOutput(table)
    with pytest.raises(AssertionError):
        m.step([t[:, 0] for t in table], torch.zeros(1, 32, device="cuda"))


def test_other_shapes_while_another_stream_still_works():
    """What the module lets go of for other shapes is not given away while the stream that used it last is at work."""
    m, table, dy, h0, dlast = make((2, 700), 2, 64, BF)
    small = make((1, 3), 1, 64, BF)
    m.updateOutput(table, state=h0)
    want = [t.clone() for t in m.backward(table, dy, state=h0, gradState=dlast)] + [m.gradBias.clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
        m.updateOutput(table, state=h0)
        grads = m.backward(table, dy, state=h0, gradState=dlast)
        got = [t.clone() for t in grads] + [m.gradBias.clone()]
    del grads
    m.evaluate()
    m.updateOutput(small[1])
    m.output = m.gradInput = m.gradProjection = m.state = m.gradState = m.checkpoints = None
    fill = [torch.full((n,), float("nan"), device="cuda") for n in (704, 1408, 2816, 22 * 64, 2 * 64, 32 * 64, 134400, 67200, 44800)
            for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.isnan(t).all() for t in fill)


def test_waits_that_run_out_in_the_middle_of_a_call():
    """With waits that nothing ends, the blocks of a cluster go their ways, and the call ends: its results are lost, the
    status says so, and the calls after it are as ever."""
    lib = capi.lib()
    made = [make((1, 3000), 1, 64, BF, seed=11), make((3000,), 2, 33, F32, seed=12)]
    offsets = [None, torch.tensor([0, 1100, 3000], dtype=torch.int32, device="cuda")]
    before = lib.fbfftconv_recurrence_wait_limit(0)
    try:
        for (m, table, dy, h0, dlast), at in zip(made, offsets):
            for _ in range(20):
                m.updateOutput(table, state=h0, offsets=at)
                assert lib.fbfftconv_recurrence_status(1) == 1
                m.backward(table, dy, state=h0, offsets=at, gradState=dlast)
                assert lib.fbfftconv_recurrence_status(1) == 1
    finally:
        lib.fbfftconv_recurrence_wait_limit(before)
    assert lib.fbfftconv_recurrence_status(0) == 0
    for (m, table, dy, h0, dlast), at in zip(made, offsets):
        check(m, table, dy, h0, dlast, at)
    assert lib.fbfftconv_recurrence_status(0) == 0


def test_a_lost_call_is_not_passed_over():
    """The calls after one whose waits ran out are refused until the status is reset, on a stream of its own too, and
    also where the first that lost its results was a replayed one."""
    lib = capi.lib()
    m, table, dy, h0, dlast = make((1, 3000), 1, 64, BF, seed=13)
    m.updateOutput(table, state=h0)
    m.backward(table, dy, state=h0)
    before = lib.fbfftconv_recurrence_wait_limit(0)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    try:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.updateOutput(table, state=h0)
        assert m.status() == 1  # waits for the device, whatever stream the call was on
        with pytest.raises(capi.FbfftconvError, match="gave up"):
            m.updateOutput(table, state=h0)
        with pytest.raises(capi.FbfftconvError, match="gave up"):
            m.backward(table, dy, state=h0)
        assert m.status(reset=True) == 1 and m.status() == 0
        with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
            m.updateOutput(table, state=h0)
    finally:
        lib.fbfftconv_recurrence_wait_limit(before)
    check(m, table, dy, h0, dlast)
    graph.replay()
    torch.cuda.synchronize()
    with pytest.raises(capi.FbfftconvError, match="gave up"):
        m.updateOutput(table, state=h0)
    assert m.status(reset=True) == 1
    check(m, table, dy, h0, dlast)


@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_output_gates_that_are_masked(dtype):
    """z at the type's lowest value is a gate of zero whatever the state is, and at its largest one that passes all on."""
    m = GatedLinearRecurrence(16)
    x = torch.full((1, 5, 16), 6.0, dtype=dtype, device="cuda")
    z = torch.full_like(x, torch.finfo(dtype).min)
    table, one = [x, torch.zeros_like(x), z], torch.ones_like(x)
    assert not m.updateOutput(table).any() and torch.isfinite(m.state).all()
    for grad in m.backward(table, one):
        assert not grad.any()
    state = torch.full((1, 16), 6.0, device="cuda")
    assert not m.step([t[:, 0] for t in table], state).any() and (state == 6).all()
    z.fill_(torch.finfo(dtype).max)
    x.fill_(2.0 ** -10)
    h = 2.0 ** -10 * (1 - 0.5 ** torch.arange(1, 6, device="cuda").double())
    y = m.updateOutput(table)[0, :, 0].double()
    assert ((y - h * z[0, 0, 0].double()).abs() <= torch.finfo(dtype).eps * y).all()
    dx, dg, dz = m.backward(table, one * 2.0 ** -20)
    assert all(torch.isfinite(g).all() for g in (dx, dg, dz))
    assert ((dz[0, :, 0].double() - h * 2.0 ** -20).abs() <= torch.finfo(dtype).eps * h * 2.0 ** -20 + 2.0 ** -25).all()


def test_one_module_in_several_layers():
    """A module that is shared by layers takes its own output in."""
    m, table, dy, h0, dlast = make((2, 50), 2, 32, F32, seed=14)
    y = m.updateOutput(table, state=h0)
    want = y.clone()
    check(m, [y, *table[1:]], dy, h0, dlast)
    assert torch.equal(y, want)


FIRST_CALL = """
import torch
from fbcunn_b200 import GatedLinearRecurrence
m = GatedLinearRecurrence(64)
table = [torch.randn(1, 3000, 64, device="cuda") for _ in range(3)]
dy = torch.randn(1, 3000, 64, device="cuda")
graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
    y = m.updateOutput(table)
    grads = m.backward(table, dy)
graph.replay()
got = [t.clone() for t in (y, m.state, *grads, m.gradBias)]
again = [m.updateOutput(table), m.state, *m.backward(table, dy), m.gradBias]
assert all(torch.equal(a, b) for a, b in zip(got, again)) and m.status() == 0
print("replayed")
"""


def test_the_first_call_of_a_process_may_be_captured():
    """What the library sets up at its first call is no part of a capture."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=240)
    assert run.returncode == 0 and "replayed" in run.stdout, run.stderr[-2000:]
