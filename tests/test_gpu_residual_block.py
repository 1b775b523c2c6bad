"""The sequence-model operators together, as a residual block uses them: the norm that enters it, a projection, the
recurrence, a projection back, and the border to the next block with its gate, residual sum and norms; its gradients
against automatic differentiation in 64 bits, a training step with AdamW, that step captured and replayed, and a prompt
continued token by token.

Every stage is within 64 u = 4e-6 of the magnitudes that enter it; there are seven, and sums over 64 channels or 100 rows
between them: 1e-4 of a gradient's norm leaves room for cancellation."""
import pytest
import torch

from fbcunn_b200 import AdamW, GatedLinearRecurrence, GatedResidualNorm

pytestmark = pytest.mark.gpu

B, T, D = 2, 50, 64


class Block:
    def __init__(self, dtype=torch.float32, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        def normal(*shape, scale=1.0):
            return torch.empty(shape, device="cuda").normal_(generator=gen) * scale
        self.entry = GatedResidualNorm(D, post=None, pre="rms")
        self.mixer = GatedLinearRecurrence(D)
        self.border = GatedResidualNorm(D, post="rms", pre="layer", gate="sigmoid", residualScale=0.9, normBias=True)
        self.W1, self.W2 = normal(4 * D, D, scale=D ** -0.5).to(dtype), normal(D, D, scale=D ** -0.5).to(dtype)
        self.gradW1, self.gradW2 = torch.zeros_like(self.W1), torch.zeros_like(self.W2)
        self.mixer.bias.copy_(torch.linspace(-1, 4, D))
        for m in (self.entry, self.border):
            for w in m.parameters()[0]:
                w.add_(normal(D, scale=0.1))

    def parameters(self):
        p, g = [self.W1, self.W2], [self.gradW1, self.gradW2]
        for m in (self.entry, self.mixer, self.border):
            p += m.parameters()[0]
            g += m.parameters()[1]
        return p, g

    def updateOutput(self, r):
        self.v = self.entry.updateOutput(r)
        self.p = (self.v @ self.W1.t()).split(D, -1)
        self.y = self.mixer.updateOutput(list(self.p[:3]))
        self.u = self.y @ self.W2.t()
        return self.border.updateOutput([self.u, r, self.p[3]])

    def backward(self, r, grads):
        du, dr, dgate = self.border.backward([self.u, r, self.p[3]], grads)
        self.gradW2.copy_(du.flatten(0, 1).t() @ self.y.flatten(0, 1))
        self.mixer.backward(list(self.p[:3]), du @ self.W2)
        dp = torch.cat([self.mixer.gradProjection, dgate], -1)
        self.gradW1.copy_(dp.flatten(0, 1).t() @ self.v.flatten(0, 1))
        return dr + self.entry.backward(r, dp @ self.W1)


def exact(block, r, grads):
    """Outputs and gradients of the block in 64 bits."""
    leaves = [t.double().requires_grad_() for t in block.parameters()[0]] + [r.double().requires_grad_()]
    W1, W2, w0, bias, w1, b1, w2, b2, x0 = leaves
    rms = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    v = rms(x0, w0)
    x, g, z, gate = (v @ W1.t()).split(D, -1)
    a = torch.sigmoid(g + bias)
    h, rows = torch.zeros(r.shape[0], D, dtype=torch.float64, device="cuda"), []
    for t in range(r.shape[1]):
        h = a[:, t] * h + (1 - a[:, t]) * x[:, t]
        rows.append(h)
    y = torch.stack(rows, 1) * torch.nn.functional.silu(z)
    out = 0.9 * x0 + torch.sigmoid(gate) * (rms(y @ W2.t(), w1) + b1)
    last = torch.nn.functional.layer_norm(out, (D,), w2, b2, 1e-6)
    ((out * grads[0].double()).sum() + (last * grads[1].double()).sum()).backward()
    return [out.detach(), last.detach()], [t.grad for t in leaves]


def inputs(seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.empty(B, T, D, device="cuda").normal_(generator=gen) for _ in range(3)]


def test_gradients_of_a_block():
    block = Block()
    r, *grads = inputs()
    out = block.updateOutput(r)
    dr = block.backward(r, grads)
    want_out, want = exact(block, r, grads)
    for a, b in zip(out + block.parameters()[1] + [dr], want_out + want):
        assert float((a - b).norm()) <= 1e-4 * float(b.norm())


def test_training_steps():
    """Three steps, and the same with the last two captured and replayed.  The library's products may differ in their last
    places between the two, which moves few 8-bit codes: 1e-4 of a parameter's norm, of which a step of 1e-2 is some
    hundred times more."""
    r, *grads = inputs()
    blocks = [Block() for _ in range(2)]
    opts = [AdamW([b], lr=1e-2, stateBits=8, min8bitSize=D) for b in blocks]
    start = [p.clone() for p in blocks[0].parameters()[0]]

    def train(k):
        blocks[k].updateOutput(r)
        blocks[k].backward(r, grads)
        opts[k].step()

    for _ in range(3):
        train(0)
    train(1)  # what is kept for these shapes is made before the capture
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda.current_blas_handle()
        blocks[1].v @ blocks[1].W1.t()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            train(1)
    torch.cuda.synchronize()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert opts[0].steps == opts[1].steps == 3
    for a, b, s in zip(blocks[0].parameters()[0], blocks[1].parameters()[0], start):
        assert float((a - b).norm()) <= 1e-4 * float(a.norm())
        assert float((a - s).norm()) > 3e-3 * float(s.norm())


def test_a_prompt_and_its_tokens():
    block = Block()
    r, *_ = inputs()
    for m in (block.entry, block.mixer, block.border):
        m.evaluate()
    whole = [t.clone() for t in block.updateOutput(r)]
    n = T - 8
    block.updateOutput(r[:, :n].contiguous())
    state = block.mixer.state.clone()
    for t in range(n, T):
        now = r[:, t].contiguous()
        p = (block.entry.updateOutput(now) @ block.W1.t()).split(D, -1)
        y = block.mixer.step(list(p[:3]), state)
        out = block.border.updateOutput([y @ block.W2.t(), now, p[3]])
        for a, b in zip(out, whole):
            assert float((a - b[:, t]).norm()) <= 1e-4 * float(b[:, t].norm())
