"""The sequence operators where an element's place passes 32 bits: what lies behind 2^31 elements is what the same rows give
by themselves.  Two launches may join their rows in other stretches, so recurrences are compared within the roundings of
fp32 and of the 16-bit output: a step of bf16, 2^-7, and 1e-5 for what cancels."""
import pytest
import torch

from fbcunn_b200 import AdamW, GatedLinearRecurrence, GatedResidualNorm

pytestmark = pytest.mark.gpu

D = 8192
ROWS = (1 << 31) // D + 1000
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def _need(gb):
    if torch.cuda.mem_get_info()[0] < gb << 30:
        pytest.skip(f"{gb} GB of device memory")


def _near(a, b):
    assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.float().abs().max())
    assert float((a.float() - b.float()).norm()) <= 2.0 ** -8 * float(b.float().norm())


def test_recurrence():
    """Forward and backward over packed rows; the last sequence begins behind 2^31 elements of x and ends at the end."""
    _need(60)
    wide = torch.empty(ROWS, 2 * D, dtype=BF, device="cuda").normal_()
    dy = torch.empty(ROWS, D, dtype=BF, device="cuda").normal_()
    first = (1 << 31) // D + 500
    offsets = torch.tensor([0, 70000, 70000, first, ROWS], dtype=torch.int64, device="cuda")
    m = GatedLinearRecurrence(D, outputGate=False)
    m.bias.copy_(torch.linspace(-1, 4, D))
    table = list(wide.split(D, -1))
    y = m.updateOutput(table, offsets=offsets)
    grads = m.backward(table, dy, offsets=offsets)
    got = [t[first:].clone() for t in [y, *grads]] + [m.state[3].clone()]
    small = GatedLinearRecurrence(D, outputGate=False)
    small.bias.copy_(m.bias)
    part = [t[first:].contiguous()[None] for t in table]
    want = [small.updateOutput(part)[0].clone()]
    want += [t[0].clone() for t in small.backward(part, dy[first:].contiguous()[None])] + [small.state[0]]
    for a, b in zip(got, want):
        _near(a, b)


def test_norms():
    _need(60)
    u, r, dr, dv = (torch.empty(ROWS, D, dtype=BF, device="cuda").normal_() for _ in range(4))
    m, small = (GatedResidualNorm(D, residualScale=0.5) for _ in range(2))
    out = m.updateOutput([u, r])
    grads = m.backward([u, r], [dr, dv])
    last = slice(ROWS - 300, ROWS)
    part = [t[last].clone() for t in (u, r)]
    want = [*small.updateOutput(part), *small.backward(part, [dr[last].clone(), dv[last].clone()])]
    for a, b in zip([*out, *grads], want):
        assert torch.equal(a[last], b)  # a row's sums do not depend on the others


def test_adamw():
    _need(40)
    n, keep = (1 << 31) + 1000, 2000
    p, g = torch.empty(n, dtype=BF, device="cuda").normal_(), torch.empty(n, dtype=BF, device="cuda").normal_()
    start = p[-keep:].float()
    opt = AdamW([p], [g], lr=1e-2, weightDecay=0.0, stateBits=8)
    opt.step()
    # the first step moves every parameter by lr against its gradient's sign
    want = start - 1e-2 * torch.sign(g[-keep:].float())
    half = torch.finfo(BF).eps / 2 * 1.01
    assert bool(((p[-keep:].float() - want).abs() <= half * want.abs() + 1e-6).all())
    blocks = opt.moments["m8_scale"]
    last = g[-(n % 256 or 256):].float().abs().max()
    assert abs(float(blocks[-1]) * 448 - 0.1 * float(last)) <= 1e-5 * float(last)
