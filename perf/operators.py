"""The sequence-model operators whose speed is measured: the gated linear recurrence, the norms around a block with
its gate and residual scale, and the AdamW step, each in its plain form (elementary tensor operations in 32 bits) and,
where `own` is true, as a user's program calls this package's modules.

A case is a dict of plain values; `op` says which operator it is:

    "recurrence"  h_t = a_t h_{t-1} + (1 - a_t) x_t, a_t = sigmoid(g_t + bias), y_t = h_t silu(z_t) (y_t = h_t without
                  the output gate): padded (batch, length, channels) or packed rows with offsets, forward alone or with
                  backward
    "token"       the same for one token of every sequence, the state updated in place
    "norms"       r' = residual_scale r + branch_scale act(gate) post(u), v = pre(r'), forward alone or with backward
    "adamw"       one step over many tensors, moments in 32 bits or in 8 (e4m3, each block of 256 with its scale, which is
                  an output of its own beside them)
"""
import math
import random

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _recurrence(name, batch, length, channels, dtype, gate=True, train=True, packed=False, state=False):
    """packed: `batch` sequences of ragged lengths, an empty one and one of a single row among them, in batch * length
    rows."""
    c = dict(op="recurrence", batch=batch, length=length, channels=channels, dtype=dtype, gate=gate, train=train,
             packed=packed, state=state)
    return dict(c, name=name) if name else c


def _token(name, batch, channels, dtype, gate=True):
    c = dict(op="token", batch=batch, channels=channels, dtype=dtype, gate=gate)
    return dict(c, name=name) if name else c


def _norms(name, batch, length, channels, dtype, residual, post="rms", pre="rms", gate="none", per="token", bias=False,
           train=True):
    """gate: "none", "linear" or "sigmoid"; per: a gate row for each "token", "sequence", or one for "all" rows."""
    c = dict(op="norms", batch=batch, length=length, channels=channels, dtype=dtype, residual=residual, post=post,
             pre=pre, gate=gate, per=per, bias=bias, train=train)
    return dict(c, name=name) if name else c


def _adamw(name, tensors, dtype, grads, bits, masters=False, width=0, layers=0):
    """tensors: "conv" = the convolution layers of the benchmark; "blocks" = `layers` blocks of `width` channels (three
    inputs, one output, norms and biases); "ragged" = `layers` tensors of odd sizes up to width * width."""
    c = dict(op="adamw", tensors=tensors, dtype=dtype, grads=grads, bits=bits, masters=masters, width=width,
             layers=layers)
    return dict(c, name=name) if name else c


def listed():
    return [
        # serving: one token of each of 16 sequences, where the call itself is what counts
        _token("recurrence one token", 16, 1024, "bf16"),
        # serving: a long prompt, one sequence, its state kept for the tokens that follow
        _recurrence("recurrence long prompt", 1, 131072, 1024, "f16", train=False, state=True),
        # training: a batch of ordinary lengths, forward and backward
        _recurrence("recurrence training", 8, 4096, 2048, "bf16"),
        # training in 32 bits on packed documents of ragged lengths, odd width, no output gate
        _recurrence("recurrence packed", 23, 331, 515, "f32", gate=False, packed=True, state=True),
        # serving: the boundary between two blocks for a few tokens
        _norms("norms few tokens", 16, 1, 2048, "bf16", "bf16", train=False),
        # serving: a prompt, residual stream in 32 bits
        _norms("norms prompt", 1, 8192, 5120, "bf16", "f32", train=False),
        # training: both norms, a gate computed from every token
        _norms("norms training", 8, 2048, 4096, "bf16", "bf16", gate="sigmoid"),
        # training in 32 bits: layer norms with biases, a gate for each sequence, nothing a power of two
        _norms("norms gate per sequence", 24, 513, 1000, "f32", "f32", post="layer", pre="layer", gate="linear",
               per="sequence", bias=True),
        # the convolution layers of the benchmark: few tensors, some of them tiny
        _adamw("adamw conv layers", "conv", "f32", "f32", 32),
        # a model's parameters in 32 bits
        _adamw("adamw 32-bit states", "blocks", "f32", "f32", 32, width=2048, layers=8),
        # 16-bit parameters with 32-bit masters, moments in 8 bits
        _adamw("adamw 8-bit masters", "blocks", "bf16", "bf16", 8, masters=True, width=2048, layers=8),
        # 16-bit parameters alone, moments in 8 bits, tensors of odd sizes
        _adamw("adamw 8-bit ragged", "ragged", "bf16", "f32", 8, width=1500, layers=60),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {"recurrence": 1.4e9, "norms": 1.0e9, "adamw": 3.0e9}
    while True:
        kind = rng.choice(["token", "recurrence", "recurrence", "norms", "norms", "adamw", "adamw"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        odd = rng.random() < 0.3
        if kind == "token":
            return _token(None, _log_int(rng, 1, 512), _log_int(rng, 64, 8192) if odd else 64 * _log_int(rng, 1, 128),
                          dtype, rng.random() < 0.7)
        if kind == "recurrence":
            c = _recurrence(None, _log_int(rng, 1, 64), _log_int(rng, 1, 65536),
                            _log_int(rng, 100, 4096) if odd else 64 * _log_int(rng, 4, 64), dtype,
                            gate=rng.random() < 0.7, train=rng.random() < 0.7, packed=rng.random() < 0.4,
                            state=rng.random() < 0.5)
        elif kind == "norms":
            gate = rng.choice(["none", "linear", "sigmoid"])
            post, pre = rng.choice([("rms", "rms"), ("rms", "rms"), ("layer", "layer"), ("none", "rms"),
                                    ("none", "layer"), ("rms", "none"), ("layer", "rms")])
            c = _norms(None, _log_int(rng, 1, 64), _log_int(rng, 1, 16384),
                       _log_int(rng, 33, 8192) if odd else 64 * _log_int(rng, 1, 128), dtype,
                       rng.choice([dtype, "f32"]), post=post, pre=pre, gate=gate,
                       per=rng.choice(["token", "sequence", "all"]) if gate != "none" else "token",
                       bias=rng.random() < 0.3, train=rng.random() < 0.7)
        else:
            bits = rng.choice([8, 32])
            masters = dtype != "f32" and rng.random() < 0.5
            tensors = rng.choice(["blocks", "ragged"])
            c = _adamw(None, tensors, dtype, rng.choice([dtype, "f32"]), bits, masters,
                       width=_log_int(rng, 100, 2048) if odd else 64 * _log_int(rng, 2, 32),
                       layers=_log_int(rng, 1, 12) if tensors == "blocks" else _log_int(rng, 1, 200))
        if 1e4 <= work(c)["bytes"] <= most[kind]:
            return c


# -- sizes -------------------------------------------------------------------------------------------
def _shapes(c):
    if c["tensors"] == "conv":
        layers = [(16, 16, 5, 5), (96, 3, 11, 11), (128, 64, 9, 9), (128, 128, 9, 9), (128, 128, 7, 7), (384, 384, 3, 3)]
        return [s for w in layers for s in (w, (w[0],))]
    d = c["width"]
    if c["tensors"] == "blocks":
        return [s for _ in range(c["layers"]) for s in ((3 * d, d), (d,), (d, d), (d,), (d,))]
    rng = random.Random(c["layers"] * 10007 + d)  # sizes belong to the case, not to the seed
    return [(_log_int(rng, 3, d * d),) for _ in range(c["layers"])]


_BLOCK = 256  # elements that share a scale
_SMALL = 4096  # tensors below keep moments in 32 bits


def _states(c):
    """Per tensor (elements, bits of its moments, first element in the flat buffer of that kind): every tensor starts
    on a block of its own."""
    at, out = {8: 0, 32: 0}, []
    for s in _shapes(c):
        n = math.prod(s)
        bits = c["bits"] if n >= _SMALL else 32
        out.append((n, bits, at[bits]))
        at[bits] += -(-n // _BLOCK) * _BLOCK
    return out, at


def work(case):
    c = case
    if c["op"] == "adamw":
        total = flops = 0
        e, eg = _BYTES[c["dtype"]], _BYTES[c["grads"]]
        for n, bits, _ in _states(c)[0]:
            total += n * (eg + (8 + e if c["masters"] else 2 * e))
            total += n * 16 if bits == 32 else n * 4 + -(-n // _BLOCK) * 16
            flops += n * (14 if bits == 32 else 40)
        return {"bytes": total, "flops": flops}
    e, d = _BYTES[c["dtype"]], c["channels"]
    if c["op"] == "token":
        n = c["batch"] * d
        return {"bytes": n * (e * (4 if c["gate"] else 3) + 8) + 4 * d, "flops": 14 * n}
    rows = c["batch"] * c["length"]
    n = rows * d
    if c["op"] == "recurrence":
        z = 1 if c["gate"] else 0
        total = n * e * (3 + z) + 4 * d + c["batch"] * d * 4 * (2 if c["state"] else 1) + 8 * c["batch"] * c["packed"]
        flops = n * (10 + 4 * z)
        if c["train"]:
            total += n * e * (5 + 2 * z) + 4 * d + c["batch"] * d * 4 * (3 if c["state"] else 0)
            flops += n * (24 + 10 * z)
        return {"bytes": total, "flops": flops}
    er, gates = _BYTES[c["residual"]], _gate_rows(c)
    post, pre = c["post"] != "none", c["pre"] != "none"
    weights = 4 * d * (post + pre) * (2 if c["bias"] else 1)
    total = n * (e + 2 * er + e * pre) + gates * d * e + weights
    flops = n * (2 + 6 * post + 6 * pre + 2 * (gates > 0))
    if c["train"]:
        # u where its norm or the gate needs it, r' where the second norm does, and the incoming and outgoing gradients
        total += n * (e * (post or gates > 0) + er * pre + er + e * pre + e + er) + 2 * gates * d * e + 2 * weights
        flops += n * (2 + 10 * post + 10 * pre + 4 * (gates > 0))
    return {"bytes": total, "flops": flops}


def _gate_rows(c):
    if c["gate"] == "none":
        return 0
    return {"token": c["batch"] * c["length"], "sequence": c["batch"], "all": 1}[c["per"]]


# -- a case ------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "adamw":
        return _prepare_adamw(c, s, gen)

    def normal(*shape, dtype=c["dtype"]):
        t = torch.empty(shape, dtype=_DT[dtype], device="cuda")
        return t.normal_(generator=gen)

    d = c["channels"]
    if c["op"] == "norms":
        return _prepare_norms(c, s, normal)
    # gates whose memory reaches from one row to some hundreds, as a trained layer's do
    s["bias"] = torch.linspace(-1, 6, d, device="cuda") + 0.1 * normal(d, dtype="f32")
    parts = 3 if c["gate"] else 2
    if c["op"] == "token":
        s["input"] = list(normal(c["batch"], parts * d).split(d, -1))
        s["state"] = normal(c["batch"], d, dtype="f32")
    else:
        shape = (c["batch"] * c["length"],) if c["packed"] else (c["batch"], c["length"])
        s["input"] = list(normal(*shape, parts * d).split(d, -1))  # one projection's output, in parts
        s["offsets"] = _offsets(c, seed).cuda() if c["packed"] else None
        s["state"] = normal(c["batch"], d, dtype="f32") if c["state"] else None
        if c["train"]:
            s["grad"] = normal(*shape, d)
            s["grad_state"] = normal(c["batch"], d, dtype="f32") if c["state"] else None
    if own:
        from fbcunn_b200 import GatedLinearRecurrence
        s["module"] = m = GatedLinearRecurrence(d, outputGate=c["gate"])
        m.bias.copy_(s["bias"])
        m.training() if c.get("train") else m.evaluate()
    return s


def _offsets(c, seed):
    rng = random.Random(seed)
    rows, n = c["batch"] * c["length"], c["batch"]
    cuts = sorted(rng.randint(0, rows) for _ in range(n - 1))
    if n > 3:
        cuts[0] = 0  # an empty sequence
        cuts[-1] = rows - 1  # and one of a single row
    return torch.tensor([0] + sorted(cuts) + [rows], dtype=torch.int32)


def _prepare_norms(c, s, normal):
    d, shape = c["channels"], (c["batch"], c["length"])
    s["u"] = normal(*shape, d)
    s["r"] = normal(*shape, d, dtype=c["residual"]) * 3
    s["gate"] = None
    if c["gate"] != "none":
        s["gate"] = normal(*{"token": shape, "sequence": (shape[0], 1), "all": (1, 1)}[c["per"]], d)
    for part in ("post", "pre"):
        there = c[part] != "none"
        s[part + "_weight"] = 1 + 0.1 * normal(d, dtype="f32") if there else None
        s[part + "_bias"] = 0.1 * normal(d, dtype="f32") if there and c["bias"] else None
    s["scales"] = (0.9, 0.5)  # residual, branch
    if c["train"]:
        s["grad_r"] = normal(*shape, d, dtype=c["residual"])
        s["grad_v"] = normal(*shape, d) if c["pre"] != "none" else None
    if own:
        from fbcunn_b200 import GatedResidualNorm
        s["module"] = m = GatedResidualNorm(
            d, post=_none(c["post"]), pre=_none(c["pre"]), gate=_none(c["gate"]), residualScale=0.9, branchScale=0.5,
            normBias=c["bias"], eps=1e-6)
        for part in ("post", "pre"):
            for what in ("Weight", "Bias"):
                if s[f"{part}_{what.lower()}"] is not None:
                    getattr(m, part + what).copy_(s[f"{part}_{what.lower()}"])
        m.training() if c["train"] else m.evaluate()
    return s


def _none(text):
    return None if text == "none" else text


_HYPER = dict(lr=3e-4, betas=(0.9, 0.999), eps=1e-8, weightDecay=0.1)


def _prepare_adamw(c, s, gen):
    def flat(n, scale, dtype="f32"):
        return torch.empty(n, dtype=torch.float32, device="cuda").normal_(generator=gen).mul_(scale).to(_DT[dtype])

    shapes, (states, size) = _shapes(c), _states(c)
    # parameters and gradients lie in one flat tensor each, as a program that flattens its model has them
    total = sum(-(-n // 64) * 64 for n, _, _ in states)
    master = flat(total, 0.02)
    s["flat"] = master.to(_DT[c["dtype"]]).clone()
    s["flat_grad"] = flat(total, 1e-3, c["grads"])
    s["flat_master"] = s["flat"].float() + flat(total, 1e-6) if c["masters"] else None
    s["p"], s["g"], s["w"], at = [], [], [], 0
    for shape, (n, _, _) in zip(shapes, states):
        s["p"].append(s["flat"][at: at + n].view(shape))
        s["g"].append(s["flat_grad"][at: at + n].view(shape))
        s["w"].append(s["flat_master"][at: at + n].view(shape) if c["masters"] else None)
        at += -(-n // 64) * 64
    s["step"] = 1000
    s["seed"] = 1234
    mom = s["moments"] = {}
    if size[32]:
        mom["m"], mom["v"] = flat(size[32], 3e-4), flat(size[32], 1e-3).square_()
    if size[8]:
        m, r = flat(size[8], 3e-4), flat(size[8], 1e-3).abs_()
        for n, bits, first in states:  # nothing behind a tensor's last element
            if bits == 8:
                end = first + -(-n // _BLOCK) * _BLOCK
                m[first + n: end], r[first + n: end] = 0, 0
        for key, x in (("m8", m), ("r8", r)):
            x = x.view(-1, _BLOCK)
            scale = x.abs().amax(1) / 448
            codes = (x / scale.clamp(min=1e-30)[:, None]).clamp(-448, 448)
            if key == "r8":
                codes = codes.clamp(min=2.0 ** -9) * (x > 0)
            mom[key], mom[key + "_scale"] = codes.to(torch.float8_e4m3fn).view(-1), scale
    if own:
        from fbcunn_b200 import AdamW
        s["optimizer"] = opt = AdamW(s["p"], s["g"], masters=s["w"] if c["masters"] else None, stateBits=c["bits"],
                                     min8bitSize=_SMALL, seed=s["seed"], **_HYPER)
        opt.loadState(dict(mom, steps=s["step"]))
    return s


def run(state):
    return _RUN[state["case"]["op"]](state)


# -- the recurrence ----------------------------------------------------------------------------------
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along the first dimension, h_{-1} = 0: every round doubles the rows that are joined."""
    reach, a, b = 1, a.clone(), b.clone()
    while reach < a.shape[0]:
        b[reach:] += a[reach:] * b[:-reach]
        a[reach:] = a[reach:] * a[:-reach]
        reach *= 2
    return b


def _rows(c, t):
    """(batch, length, d) or packed rows as (rows, sequences side by side, d) in 32 bits."""
    t = t.float()
    return t[:, None] if c["packed"] else t.transpose(0, 1)


def _ends(s):
    """First and last row of each sequence that has rows, and which ones those are."""
    off = s["offsets"].long()
    keep = (off[1:] > off[:-1]).nonzero()[:, 0]
    return off[:-1][keep], off[1:][keep] - 1, keep


def _run_recurrence(s):
    c = s["case"]
    if own:
        m = s["module"]
        y = m.updateOutput(s["input"], state=s["state"], offsets=s["offsets"])
        out = {"y": y, "state": m.state}
        if c["train"]:
            grads = m.backward(s["input"], s["grad"], state=s["state"], offsets=s["offsets"], gradState=s["grad_state"])
            out |= dict(zip(("dx", "dg", "dz"), grads), dbias=m.gradBias)
            if c["state"]:
                out["dstate"] = m.gradState
        return out
    dtype, d, packed = _DT[c["dtype"]], c["channels"], c["packed"]
    x, g = (_rows(c, t) for t in s["input"][:2])
    g = g + s["bias"]
    a, b = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    h0 = s["state"] if c["state"] else torch.zeros(c["batch"], d, device=x.device)
    ax, bx = a.clone(), b * x  # what a row takes from the row before, and what it adds
    if packed:
        first, last, keep = _ends(s)
        bx[first, 0] += a[first, 0] * h0[keep]
        ax[first, 0] = 0
    else:
        bx[0] += a[0] * h0
        ax[0] = 0
    h = _scan(ax, bx)
    y = h
    if c["gate"]:
        z = _rows(c, s["input"][2])
        sz = 1 / (1 + torch.exp(-z))
        y = h * z * sz
    back = (lambda t: t[:, 0].to(dtype)) if packed else (lambda t: t.transpose(0, 1).to(dtype))
    final = h0.clone()
    if packed:
        final[keep] = h[last, 0]
    else:
        final = h[-1].clone()
    out = {"y": back(y), "state": final}
    if not c["train"]:
        return out
    dy = _rows(c, s["grad"])
    e = dy * z * sz if c["gate"] else dy.clone()
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    if packed:
        before[first, 0] = h0[keep]
        if c["state"]:
            e[last, 0] += s["grad_state"][keep]
    else:
        before[0] = h0
        if c["state"]:
            e[-1] += s["grad_state"]
    after = torch.cat([ax[1:], torch.zeros_like(ax[:1])])
    D = _scan(after.flip(0), e.flip(0)).flip(0)
    dg = D * (before - x) * a * b
    out |= {"dx": back(b * D), "dg": back(dg), "dbias": dg.sum((0, 1))}
    if c["gate"]:
        out["dz"] = back(dy * h * sz * (1 + z * (1 - sz)))
    if c["state"]:
        if packed:
            dstate = s["grad_state"].clone()  # an empty sequence hands its state on
            dstate[keep] = a[first, 0] * D[first, 0]
        else:
            dstate = a[0] * D[0]
        out["dstate"] = dstate
    return out


def _run_token(s):
    c = s["case"]
    if own:
        return {"y": s["module"].step(s["input"], s["state"]), "state": s["state"]}
    x, g = (t.float() for t in s["input"][:2])
    g = g + s["bias"]
    h = s["state"] / (1 + torch.exp(-g)) + x / (1 + torch.exp(g))
    s["state"].copy_(h)
    y = h
    if c["gate"]:
        z = s["input"][2].float()
        y = h * z / (1 + torch.exp(-z))
    return {"y": y.to(_DT[c["dtype"]]), "state": s["state"]}


# -- the norms ---------------------------------------------------------------------------------------
def _norm(kind, x, weight, bias):
    """Norm(x) and what its gradient needs: the normalised rows and the reciprocal deviation."""
    if kind == "none":
        return x, x, None
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    hat = x * rstd
    out = hat * weight
    return (out if bias is None else out + bias), hat, rstd


def _norm_grad(kind, grad, hat, rstd, weight):
    """Gradients of _norm: by its input, its weight and its bias."""
    if kind == "none":
        return grad, None, None
    rows = tuple(range(grad.dim() - 1))
    dw, db = (grad * hat).sum(rows), grad.sum(rows)
    gw = grad * weight
    dx = gw - hat * (gw * hat).mean(-1, keepdim=True)
    if kind == "layer":
        dx = dx - gw.mean(-1, keepdim=True)
    return dx * rstd, dw, db


def _run_norms(s):
    c = s["case"]
    post, pre, gated = c["post"], c["pre"], c["gate"] != "none"
    if own:
        m = s["module"]
        inputs = [s["u"], s["r"]] + ([s["gate"]] if gated else [])
        out = m.updateOutput(inputs)
        out = {"r": out[0], "v": out[1]} if pre != "none" else {"r": out}
        if c["train"]:
            grads = m.backward(inputs, [s["grad_r"], s["grad_v"]] if pre != "none" else s["grad_r"])
            out |= dict(zip(("du", "dr", "dgate"), grads))
            for part in ("post", "pre"):
                if c[part] != "none":
                    out["d%s_weight" % part] = m.gradPostWeight if part == "post" else m.gradPreWeight
                    if c["bias"]:
                        out["d%s_bias" % part] = m.gradPostBias if part == "post" else m.gradPreBias
        return out
    alpha, beta = s["scales"]
    dtype, residual = _DT[c["dtype"]], _DT[c["residual"]]
    n, hat1, rstd1 = _norm(post, s["u"].float(), s["post_weight"], s["post_bias"])
    act = 1
    if gated:
        w = s["gate"].float()
        act = 1 / (1 + torch.exp(-w)) if c["gate"] == "sigmoid" else w
    r = alpha * s["r"].float() + beta * (act * n)
    v, hat2, rstd2 = _norm(pre, r, s["pre_weight"], s["pre_bias"])
    out = {"r": r.to(residual)}
    if pre != "none":
        out["v"] = v.to(dtype)
    if not c["train"]:
        return out
    dr = s["grad_r"].float()
    if pre != "none":
        dx, dw, db = _norm_grad(pre, s["grad_v"].float(), hat2, rstd2, s["pre_weight"])
        dr = dr + dx
        out["dpre_weight"] = dw
        if c["bias"]:
            out["dpre_bias"] = db
    out["dr"] = (alpha * dr).to(residual)
    dn = beta * dr * act
    if gated:
        da = beta * dr * n
        if c["gate"] == "sigmoid":
            da = da * act * (1 - act)
        if c["per"] != "token":
            da = da.sum((0, 1) if c["per"] == "all" else 1, keepdim=True)
        out["dgate"] = da.to(dtype)
    du, dw, db = _norm_grad(post, dn, hat1, rstd1, s["post_weight"])
    out["du"] = du.to(dtype)
    if post != "none":
        out["dpost_weight"] = dw
        if c["bias"]:
            out["dpost_bias"] = db
    return out


# -- the optimizer -----------------------------------------------------------------------------------
_M32 = 0xFFFFFFFF


def _mix(x):
    """A 32-bit counter made random: xor-shifts and products with the fractions of sqrt(2) and sqrt(3)."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & _M32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & _M32
    return x ^ (x >> 16)


def _key(seed, step, tensor):
    return _mix((_mix((seed + step * 0x9E3779B9) & _M32) + tensor) & _M32)


def _round8(x, low, uniform):
    """x in e4m3 with a scale for each block, rounded up with the probability of what is cut off (uniform in [0, 1));
    positive values that must stay positive keep at least the type's lowest."""
    top = x.abs().amax(1, keepdim=True)
    none = top < 2.0 ** -100
    y = x * torch.where(none, 0.0, 448 / top)
    size = y.abs()
    quantum = torch.ldexp(torch.ones_like(y), (torch.frexp(size)[1] - 1).clamp(min=-6) - 3)
    size = (torch.floor(size / quantum + uniform) * quantum).clamp(max=448)
    if low:
        size = torch.where(y > 0, size.clamp(min=2.0 ** -9), size)
    return torch.copysign(size, y).to(torch.float8_e4m3fn), torch.where(none, 0.0, top / 448)[:, 0]


def _run_adamw(s):
    c, mom = s["case"], s["moments"]
    names = [k for k in ("m", "v", "m8", "m8_scale", "r8", "r8_scale") if k in mom]
    out = {"p": s["flat"]} | ({"master": s["flat_master"]} if c["masters"] else {})
    if own:
        opt = s["optimizer"]
        opt.step()
        return out | {k: opt.moments[k] for k in names}
    s["step"] += 1
    (b1, b2), lr = _HYPER["betas"], _HYPER["lr"]
    c1, c2 = 1 - b1 ** s["step"], 1 - b2 ** s["step"]
    for k, (p, g, w, (n, bits, at)) in enumerate(zip(s["p"], s["g"], s["w"], _states(c)[0])):
        w = p if w is None else w
        g = g.reshape(-1).float()
        if bits == 32:
            m, v = mom["m"][at: at + n], mom["v"][at: at + n]
            m.mul_(b1).add_(g * (1 - b1))
            v.mul_(b2).add_(g * g * (1 - b2))
        else:
            end = at + -(-n // _BLOCK) * _BLOCK
            blocks = slice(at // _BLOCK, end // _BLOCK)
            pad = torch.zeros(end - at, device=g.device)
            pad[:n] = g
            g = pad.view(-1, _BLOCK)
            m = mom["m8"][at:end].float().view(-1, _BLOCK) * mom["m8_scale"][blocks, None]
            root = mom["r8"][at:end].float().view(-1, _BLOCK) * mom["r8_scale"][blocks, None]
            m = m * b1 + g * (1 - b1)
            v = root * root * b2 + g * g * (1 - b2)
            bitsets = _mix(torch.arange(end - at, device=g.device) ^ _key(s["seed"], s["step"], k)).view(-1, _BLOCK)
            codes, scale = _round8(m, False, (bitsets & 0xFFFF) / 65536.0)
            mom["m8"][at:end], mom["m8_scale"][blocks] = codes.view(-1), scale
            codes, scale = _round8(torch.sqrt(v), True, (bitsets >> 16) / 65536.0)
            mom["r8"][at:end], mom["r8_scale"][blocks] = codes.view(-1), scale
            m, v = m.view(-1)[:n], v.view(-1)[:n]
        new = w.reshape(-1).float() * (1 - lr * _HYPER["weightDecay"])
        new -= lr * (m / c1) / (torch.sqrt(v / c2) + _HYPER["eps"])
        w.copy_(new.view(w.shape))
        if w is not p:
            p.copy_(w)
    return out | {k: mom[k] for k in names}


_RUN = {"recurrence": _run_recurrence, "token": _run_token, "norms": _run_norms, "adamw": _run_adamw}


# -- the definitions in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"recurrence": _exact_recurrence, "token": _exact_token, "norms": _exact_norms, "adamw": _exact_adamw}[
        case["op"]](s)


def _exact_token(s):
    x, g = s["input"][0].double(), torch.sigmoid(s["input"][1].double() + s["bias"].double())
    h = g * s["state"].double() + (1 - g) * x
    y = torch.nn.functional.silu(s["input"][2].double()) * h if s["case"]["gate"] else h
    return {"y": y, "state": h}


def _exact_recurrence(s):
    """Row by row, every sequence by itself in time; sequences of one length side by side."""
    c = s["case"]
    d, n = c["channels"], c["batch"]
    if c["packed"]:
        off = s["offsets"].tolist()
        order = [list(range(off[i], off[i + 1])) for i in range(n)]
    else:
        order = [list(range(i * c["length"], (i + 1) * c["length"])) for i in range(n)]
    if max(len(o) for o in order) > 200000:
        return None
    flat = [t.double().reshape(-1, d) for t in s["input"]]
    a = torch.sigmoid(flat[1] + s["bias"].double())
    add = torch.sigmoid(-(flat[1] + s["bias"].double())) * flat[0]
    rows = flat[0].shape[0]
    h, prev = torch.zeros(rows, d, dtype=torch.float64, device="cuda"), None
    h0 = s["state"].double() if c["state"] else torch.zeros(n, d, dtype=torch.float64, device="cuda")
    final = h0.clone()
    groups = [[i] for i in range(n)] if c["packed"] else [list(range(n))]
    lanes = [(g, torch.tensor([order[i] for i in g], dtype=torch.long, device="cuda").t().contiguous()) for g in groups]
    before = torch.zeros_like(h)
    for members, index in lanes:
        cur = h0[members]
        al, bl = a[index], add[index]
        keep = torch.empty(index.shape[0] + 1, len(members), d, dtype=torch.float64, device="cuda")
        keep[0] = cur
        ks, as_, bs = keep.unbind(0), al.unbind(0), bl.unbind(0)
        for t in range(index.shape[0]):
            torch.addcmul(bs[t], as_[t], ks[t], out=ks[t + 1])
        final[members] = keep[-1]
        h[index], before[index] = keep[1:], keep[:-1]
        del al, bl, keep, ks, as_, bs
    y, shape = h, s["input"][0].shape
    if c["gate"]:
        sz = torch.sigmoid(flat[2])
        y = h * flat[2] * sz
    out = {"y": y.view(shape), "state": final}
    if not c["train"]:
        return out
    dy = s["grad"].double().reshape(-1, d)
    dh = dy * flat[2] * sz if c["gate"] else dy
    total = torch.zeros_like(h)
    d0 = torch.zeros_like(h0)
    for members, index in lanes:
        flow = s["grad_state"].double()[members] if c["state"] else torch.zeros(len(members), d, dtype=torch.float64,
                                                                              device="cuda")
        al, bl = a[index], dh[index]
        keep = torch.empty_like(al)
        ks, as_, bs = keep.unbind(0), al.unbind(0), bl.unbind(0)
        for t in reversed(range(index.shape[0])):
            torch.add(flow, bs[t], out=ks[t])
            flow = ks[t] * as_[t]
        d0[members] = flow
        total[index] = keep
        del al, bl, keep, ks, as_, bs
    dg = total * (before - flat[0]) * a * (1 - a)
    out |= {"dx": ((1 - a) * total).view(shape), "dg": dg.view(shape), "dbias": dg.sum(0)}
    if c["gate"]:
        out["dz"] = (dy * h * (sz + flat[2] * sz * (1 - sz))).view(shape)
    if c["state"]:
        out["dstate"] = d0
    return out


def _exact_norms(s):
    """The forward formula in 64 bits; its gradients by automatic differentiation."""
    c = s["case"]
    leaf = {k: s[k].double().requires_grad_(c["train"]) for k in
            ("u", "r", "gate", "post_weight", "post_bias", "pre_weight", "pre_bias") if s[k] is not None}

    def norm(x, part):
        kind, d = c[part], (c["channels"],)
        if kind == "none":
            return x
        w, b = leaf[part + "_weight"], leaf.get(part + "_bias")
        if kind == "layer":
            return torch.nn.functional.layer_norm(x, d, w, b, 1e-6)
        y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * w
        return y if b is None else y + b

    with torch.enable_grad():
        n = norm(leaf["u"], "post")
        if c["gate"] != "none":
            n = n * (torch.sigmoid(leaf["gate"]) if c["gate"] == "sigmoid" else leaf["gate"])
        r = s["scales"][0] * leaf["r"] + s["scales"][1] * n
        v = norm(r, "pre")
        out = {"r": r.detach()} | ({"v": v.detach()} if c["pre"] != "none" else {})
        if c["train"]:
            loss = (r * s["grad_r"].double()).sum()
            if c["pre"] != "none":
                loss = loss + (v * s["grad_v"].double()).sum()
            loss.backward()
    if c["train"]:
        out |= {"d" + k: t.grad for k, t in leaf.items()}
    return out


def _exact_adamw(s):
    c, mom, h = s["case"], s["moments"], _HYPER
    t = s["step"] + 1
    p, master = s["flat"].double(), s["flat_master"].double() if c["masters"] else None
    now = {k: v.double() for k, v in mom.items()}
    out = {"p": p} | ({"master": master} if c["masters"] else {}) | now
    at = 0
    for k, (n, bits, first) in enumerate(_states(c)[0]):
        g = s["flat_grad"][at: at + n].double()
        if bits == 32:
            part = slice(first, first + n)
            m = now["m"][part] = h["betas"][0] * now["m"][part] + (1 - h["betas"][0]) * g
            v = now["v"][part] = h["betas"][1] * now["v"][part] + (1 - h["betas"][1]) * g ** 2
        else:
            i = torch.arange(n, device="cuda")
            block = first // _BLOCK + i // _BLOCK
            m = h["betas"][0] * now["m8"][first: first + n] * now["m8_scale"][block] + (1 - h["betas"][0]) * g
            v = h["betas"][1] * (now["r8"][first: first + n] * now["r8_scale"][block]) ** 2
            v = v + (1 - h["betas"][1]) * g ** 2
            x = s["seed"] + t * 0x9E3779B9 & _M32
            for more in (k, None):  # the counter's two keys
                x ^= x >> 16
                x = x * 0x6A09E667 & _M32
                x ^= x >> 15
                x = x * 0xBB67AE85 & _M32
                x ^= x >> 16
                x = x + (more or 0) & _M32
            r = i ^ x
            for shift, odd in ((16, 0x6A09E667), (15, 0xBB67AE85), (16, 1)):
                r = (r ^ (r >> shift)) * odd & _M32
            for key, value, u in (("m8", m, r & 65535), ("r8", v.sqrt(), r >> 16)):
                top = torch.zeros(-(-n // _BLOCK), dtype=torch.float64, device="cuda")
                top.index_reduce_(0, i // _BLOCK, value.abs(), "amax")
                scaled = value / (top[i // _BLOCK] / 448).clamp(min=1e-300)
                grid = 2.0 ** (torch.log2(scaled.abs().clamp(min=2.0 ** -6)).floor() - 3)
                code = torch.floor(scaled.abs() / grid + u.double() / 65536) * grid
                if key == "r8":
                    code = torch.where(value > 0, code.clamp(min=2.0 ** -9), code)
                now[key][first: first + n] = code * torch.sign(value)
                now[key + "_scale"][first // _BLOCK: first // _BLOCK + top.numel()] = top / 448
        w = (master if c["masters"] else p)[at: at + n]
        w *= 1 - h["lr"] * h["weightDecay"]
        w -= h["lr"] * (m / (1 - h["betas"][0] ** t)) / ((v / (1 - h["betas"][1] ** t)).sqrt() + h["eps"])
        if c["masters"]:
            p[at: at + n] = w
        at += -(-n // 64) * 64
    return out
