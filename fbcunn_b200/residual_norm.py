"""The norms before and after a residual block, fused with the block's gate and the residual's scale.

One module stands at the border between two blocks: the norm after the block that ends, its gate, the residual sum,
and the norm before the block that begins (fbfftconv_residual_norm in include/fbfftconv.h):

    n = post(u),  r' = residualScale r + branchScale act(gate) n,  v = pre(r')

It is an nn-style module: updateOutput takes the table [u, r] or [u, r, gate] and returns [r', v]; backward takes the
same table and the gradients [dr', dv] and returns the table of gradients, with the weights' in gradPostWeight,
gradPreWeight (and gradPostBias, gradPreBias).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import capi
from .module import _capturing, _check_parameter, _device_index, _layout, _place, _ptr, _raw_stream, _stream, _used_here

_NORMS = {None: capi.NORM_NONE, "rms": capi.NORM_RMS, "layer": capi.NORM_LAYER}
_GATES = {None: capi.GATE_NONE, "linear": capi.GATE_LINEAR, "sigmoid": capi.GATE_SIGMOID}


class GatedResidualNorm:
    """GatedResidualNorm(channels): post and pre are "rms", "layer" or None (not both None), gate is "linear",
    "sigmoid" or None.

    u, r and the gate are (..., channels); r has u's type or fp32, the others u's.  The gate has u's shape, or one that
    is shared by consecutive rows: (batch, 1, channels) for a gate of each sequence, (1, ..., channels) or (channels)
    for one of all rows.  Without post-norm and gate the table may be [r] (or r itself): v = pre(r), the entry to the
    first block, which no scale touches.  Without pre-norm the output is r'.  Weights are fp32; in training() mode, the default, updateOutput
    leaves in `stats` what backward needs besides its inputs, and backward must follow the updateOutput of the same
    inputs.  An output that is given back as an input is the caller's from then on: the call makes another.  Gradients of weights are overwritten, or added to with accumulate=True."""

    def __init__(self, channels, *, post="rms", pre="rms", gate=None, residualScale=1.0, branchScale=1.0, normBias=False,
                 eps=1e-6, device="cuda", accumulate=False):
        assert post in _NORMS and pre in _NORMS, "norms are 'rms', 'layer' or None"
        assert post is not None or pre is not None, "neither norm is there"
        assert gate in _GATES, "gates are 'linear', 'sigmoid' or None"
        assert 0 < int(channels) <= 16384, "1 to 16384 channels"
        self.channels, self.post, self.pre, self.gate = int(channels), post, pre, gate
        self.residualScale, self.branchScale, self.eps = float(residualScale), float(branchScale), float(eps)
        self.device = torch.device(device)
        self._accumulate = bool(accumulate)
        self.train = True

        def vector(there, value):
            return torch.full((self.channels,), value, dtype=torch.float32, device=self.device) if there else None

        for name, norm in (("Post", post), ("Pre", pre)):
            there = norm is not None
            setattr(self, name.lower() + "Weight", vector(there, 1.0))
            setattr(self, name.lower() + "Bias", vector(there and normBias, 0.0))
            setattr(self, f"grad{name}Weight", vector(there, 0.0))
            setattr(self, f"grad{name}Bias", vector(there and normBias, 0.0))
        self.output = None
        self.gradInput = None
        self.stats = None
        self._key = None
        self._workspace = None
        self._places = self._grad_places = self._weights = None  # of the weights and gradients when they were looked at
        self._captured = False  # whether a captured graph uses the tensors that are kept for the present shapes
        self._graphs = []       # such tensors of earlier shapes: a graph may be replayed after other shapes have run

    # -- nn.Module surface -------------------------------------------------------
    def training(self):
        self.train = True

    def evaluate(self):
        self.train = False

    def parameters(self):
        pairs = [(p, g) for p, g in ((self.postWeight, self.gradPostWeight), (self.postBias, self.gradPostBias),
                                     (self.preWeight, self.gradPreWeight), (self.preBias, self.gradPreBias)) if p is not None]
        return [p for p, _ in pairs], [g for _, g in pairs]

    def zeroGradParameters(self):
        for g in self.parameters()[1]:
            g.zero_()

    def updateOutput(self, input):
        u, r, gate = self._prepare(input)
        stats = self._stats if self.train else None
        inputs = _ptr(u), r.data_ptr(), _ptr(gate)
        if self._r_at in inputs or self._v_at in inputs:
            self._give_away(inputs)
        status = self._forward(
            self._desc_ref, *inputs, *self._weights, self._r_at if self._r_at > 0 else None,
            self._v_at if self._v_at > 0 else None, _ptr(stats), _raw_stream(self._index))
        if status:
            capi.check(status)
        self.stats = stats
        self.output = self._v if u is None else self._r_out if self._v is None else [self._r_out, self._v]
        return self.output

    def forward(self, input):
        return self.updateOutput(input)

    def backward(self, input, gradOutput, scale=None):
        """Gradients by the inputs (returned, and in gradInput) and by the weights."""
        return self._backward(input, gradOutput, 1.0 if scale is None else float(scale), True)

    def updateGradInput(self, input, gradOutput):
        return self._backward(input, gradOutput, 1.0, False)

    def accGradParameters(self, input, gradOutput, scale=None):
        """The weights' gradients alone; gradInput is left as it is."""
        kept = self.gradInput
        self._backward(input, gradOutput, 1.0 if scale is None else float(scale), True, scratch=True)
        self.gradInput = kept

    # -- internals -----------------------------------------------------------------
    def _table(self, input):
        if isinstance(input, torch.Tensor):
            input = [input]
        if len(input) == 1:
            assert self.post is None and self.gate is None, "a post-norm or a gate needs the block's output: [u, r]"
            return None, input[0], None
        assert len(input) == (2 if self.gate is None else 3), "the table is [u, r], with the gate [u, r, gate]"
        return input[0], input[1], input[2] if self.gate is not None else None

    def _prepare(self, input):
        """Checks the table; descriptor and outputs are kept for one set of shapes."""
        u, r, gate = self._table(input)
        key = (_layout(u), _layout(r), _layout(gate), self.residualScale, self.branchScale, self.eps)
        w1, b1, w2, b2 = self.postWeight, self.postBias, self.preWeight, self.preBias
        # _place of each, written out: small calls are bound by what the host does
        places = (w1 if w1 is None else (w1.data_ptr(), w1.nbytes), b1 if b1 is None else (b1.data_ptr(), b1.nbytes),
                  w2 if w2 is None else (w2.data_ptr(), w2.nbytes), b2 if b2 is None else (b2.data_ptr(), b2.nbytes))
        if places != self._places:
            self._check_weights(r)
            self._places, self._weights = places, tuple(_ptr(w) for w in (w1, b1, w2, b2))
        if key == self._key:
            if not self._captured:
                self._captured = _capturing()
            if _raw_stream(self._index) != self._made:
                _used_here(self._index, self._made, (self._r_out, self._v, self._stats, self._workspace, *(self._grads or ())))
            return u, r, gate
        for t in (u, r, gate):
            if t is None:
                continue
            assert isinstance(t, torch.Tensor) and t.is_cuda, "CUDA support only!"
            assert t.device == r.device, "tensors of two devices"
            assert t.dtype in capi.element_types(), "fp32, bf16 or fp16"
            assert t.dim() >= 1 and t.shape[-1] == self.channels, "channels mismatch"
        self._check_weights(r)
        kind = r.dtype if u is None else u.dtype
        rows = math.prod(r.shape[:-1])
        gate_rows = 0
        if u is not None:
            assert u.shape == r.shape, "u and r differ in shape"
            assert r.dtype in (kind, torch.float32), "the residual stream has the block's type or fp32"
        if gate is not None:
            assert gate.dtype == kind, "the gate has the block's type"
            gate_rows = self._gate_rows(gate.shape[:-1], r.shape[:-1])
        types = capi.element_types()
        desc = capi.NormDesc(
            rows, gate_rows, _row_stride(u), _row_stride(r), _row_stride(gate), self.channels, types[kind],
            types[r.dtype], _NORMS[self.post], _NORMS[self.pre], _GATES[self.gate], self.eps, self.residualScale,
            self.branchScale, _device_index(r.device))
        self._key, self._desc = None, desc  # no key until all that belongs to it is there
        self._desc_ref = ctypes.byref(self._desc)
        self._where, self._index, self._forward = r.device, _device_index(r.device), capi.lib().fbfftconv_residual_norm
        self._made = _raw_stream(self._index)
        if self._captured:
            self._graphs.append((self._r_out, self._v, self._stats, self._grads, self._workspace))
        self._captured = _capturing()
        self._r_out = self._v = self._stats = None
        self._r_out = torch.empty(r.shape, dtype=r.dtype, device=r.device) if u is not None else None
        self._v = torch.empty(r.shape, dtype=kind, device=r.device) if self.pre is not None else None
        self._stats = torch.empty((rows, 4), dtype=torch.float32, device=r.device)
        self._grads = self._workspace = None
        self._set_outputs()
        self._key = key
        self.stats = None
        return u, r, gate

    def _give_away(self, inputs):
        """Other outputs in the place of those that were returned before and are inputs now."""
        if self._captured:
            self._graphs.append((self._r_out, self._v))
        if self._r_at in inputs:
            self._r_out = torch.empty_like(self._r_out)
        if self._v_at in inputs:
            self._v = torch.empty_like(self._v)
        self._made = self._made if _raw_stream(self._index) == self._made else -1  # of two streams: recorded on any
        self._set_outputs()

    def _set_outputs(self):
        """Where the outputs lie; -1 for those that are not there or have no elements."""
        self._r_at, self._v_at = _ptr(self._r_out) or -1, _ptr(self._v) or -1

    def _check_weights(self, r):
        for w in (self.postWeight, self.postBias, self.preWeight, self.preBias):
            _check_parameter(w, self.channels, r.device)

    @staticmethod
    def _gate_rows(gate, rows):
        """Rows of a gate whose leading dimensions are those of the rows up to some place and 1 from there on."""
        gate = (1,) * (len(rows) - len(gate)) + tuple(gate)
        assert len(gate) == len(rows), "the gate has more dimensions than the rows"
        n, shared = 1, False
        for g, r in zip(gate, rows):
            assert g == r or g == 1, "the gate's rows are neither the rows nor shared by them"
            if g == r and r != 1:
                assert not shared, "rows that share a gate must be consecutive"
                n *= g
            elif r != 1:
                shared = True
        return n

    def _backward(self, input, gradOutput, scale, parameters, scratch=False):
        kept = self.stats
        u, r, gate = self._prepare(input)
        assert kept is not None and self.stats is kept, "updateOutput of the same inputs runs first, in training() mode"
        grad_r, grad_v = self._grad_outputs(gradOutput, u, r)
        if self._grads is None:
            n = int(capi.lib().fbfftconv_residual_norm_workspace_bytes(self._desc_ref))
            self._workspace = torch.empty(max(n, 16), dtype=torch.uint8, device=r.device)
            self._grads = self._new_grads(u, r, gate)
            self._made = self._made if _raw_stream(self._index) == self._made else -1  # of two streams: recorded on any
        du, dr, dgate = self._new_grads(u, r, gate) if scratch else self._grads
        weights = [None] * 4
        if parameters:
            gradients = (self.gradPostWeight, self.gradPostBias, self.gradPreWeight, self.gradPreBias)
            places = [_place(g) for g in gradients]
            if places != self._grad_places:
                for g in gradients:
                    _check_parameter(g, self.channels, r.device)
                self._grad_places = places
            weights = [_ptr(g) for g in gradients]
        capi.check(capi.lib().fbfftconv_residual_norm_backward(
            self._desc_ref, _ptr(u), r.data_ptr(), _ptr(gate), kept.data_ptr(),
            *self._weights[:3], _ptr(grad_r), _ptr(grad_v), _ptr(du),
            dr.data_ptr(), _ptr(dgate), *weights, scale, int(self._accumulate), self._workspace.data_ptr(),
            self._workspace.numel(), _stream(self._where)))
        self.gradInput = dr if u is None else [du, dr] + ([dgate] if gate is not None else [])
        return self.gradInput

    def _new_grads(self, u, r, gate):
        return tuple(None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (u, r, gate))

    def _grad_outputs(self, gradOutput, u, r):
        if u is None:  # v alone
            grad_v = gradOutput[-1] if isinstance(gradOutput, (list, tuple)) else gradOutput
            grad_r = None
        elif self.pre is None:
            grad_r, grad_v = gradOutput[0] if isinstance(gradOutput, (list, tuple)) else gradOutput, None
        else:
            grad_r, grad_v = gradOutput
        for g, like in ((grad_r, r), (grad_v, self._v)):
            if like is None or (g is None and u is None):
                continue
            assert isinstance(g, torch.Tensor) and g.is_cuda and g.device == r.device, "CUDA support only!"
            assert g.shape == like.shape and g.dtype == like.dtype and g.is_contiguous(), "gradOutput size or type mismatch"
        return grad_r, grad_v


def _row_stride(t):
    """The one distance between consecutive rows of (..., channels)."""
    if t is None or t.numel() == 0:
        return 0
    assert t.shape[-1] == 1 or t.stride(-1) == 1, "channels must be neighbours"
    stride, below = None, 1
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if stride is None:
            stride = s
        assert s == stride * below, "rows must lie one stride apart"
        below *= n
    stride = t.shape[-1] if stride is None else stride
    assert stride >= t.shape[-1], "rows overlap"
    return stride
