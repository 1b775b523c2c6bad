"""A gated linear recurrence along sequences, forward, backward and one token at a time.

``GatedLinearRecurrence`` is an nn-style module over fbfftconv_recurrence* (include/fbfftconv.h):

    a_t = sigmoid(g_t + bias),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t silu(z_t)

updateOutput takes the table [x, g, z] ([x, g] without the output gate: y_t = h_t), padded (batch, length, channels)
or packed (rows, channels) with offsets; backward the same table and the gradient by y; step one token of every
sequence with the states in place.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import capi
from .module import _capturing, _check_parameter, _device_index, _layout, _place, _ptr, _raw_stream, _stream, _used_here
from .residual_norm import _row_stride


class GatedLinearRecurrence:
    """GatedLinearRecurrence(channels): outputGate says whether the table has z, bias whether the gates have a learned
    one (fp32, zero at first).

    x, g and z are of one type, fp32, bf16 or fp16, and may be parts of one projection's output (rows a common distance
    apart); gradInput is laid out like that, as parts of one tensor, `gradProjection`.  states are fp32 (sequences,
    channels): the one after the last row of each sequence is left in `state`, the gradient by the initial one in
    gradState.  In training() mode, the default, updateOutput leaves in `checkpoints` what backward needs besides its
    inputs, and backward must follow the updateOutput of the same inputs.  An output or state that is given back as an
    input is the caller's from then on: the call makes others.  gradBias is overwritten, or added to with
    accumulate=True."""

    def __init__(self, channels, *, outputGate=True, bias=True, device="cuda", accumulate=False):
        assert int(channels) > 0, "channels must be positive"
        self.channels, self.outputGate = int(channels), bool(outputGate)
        self.device = torch.device(device)
        self._accumulate = bool(accumulate)
        self.bias = torch.zeros(self.channels, dtype=torch.float32, device=self.device) if bias else None
        self.gradBias = torch.zeros_like(self.bias) if bias else None
        self.train = True
        self.output = self.state = self.gradInput = self.gradProjection = self.gradState = self.checkpoints = None
        self._key = None
        self._step_key = None
        self._bias_place = self._grad_place = None  # of the bias and its gradient when they were looked at
        # whether a captured graph uses the tensors that are kept for the present shapes, and such tensors of earlier
        # shapes: a graph may be replayed after other shapes have run
        self._captured = self._step_captured = False
        self._graphs = []

    # -- nn.Module surface -------------------------------------------------------
    def training(self):
        self.train = True

    def evaluate(self):
        self.train = False

    def parameters(self):
        return ([self.bias], [self.gradBias]) if self.bias is not None else ([], [])

    def zeroGradParameters(self):
        if self.gradBias is not None:
            self.gradBias.zero_()

    def status(self, reset=False):
        """0, or 1 when blocks of a call that wait for one another gave up doing so since the last reset (waits for the
        device): that call's results are lost, and later calls raise until the status is reset."""
        with torch.cuda.device(self.device):
            return int(capi.lib().fbfftconv_recurrence_status(int(reset)))

    def updateOutput(self, input, state=None, offsets=None):
        """state: the initial states, or None for zeros; offsets: int32 or int64, sequences + 1 on the device, for packed
        rows, of which those outside of all sequences stay as they are in `output` and the gradients: zero, or what an
        earlier call of the same shapes left there."""
        x, g, z = self._prepare(input, offsets)
        self._check_state(state, "initial state")
        # what was returned before is an input now
        if state is not None and state.data_ptr() == self._state.data_ptr():
            self._state = self._another(self._state)
        output = self._output.data_ptr()
        if x.data_ptr() == output or g.data_ptr() == output or _ptr(z) == output:
            self._output = self._another(self._output)
        checkpoints = None
        if self.train:
            if self._checkpoints is None:
                n = int(capi.lib().fbfftconv_recurrence_checkpoint_bytes(self._desc_ref))
                self._checkpoints = torch.empty(max(n // 4, 1), dtype=torch.float32, device=x.device)
                self._made = self._made if _raw_stream(self._index) == self._made else -1  # of two streams: recorded on any
            checkpoints = self._checkpoints
        capi.check(capi.lib().fbfftconv_recurrence(
            self._desc_ref, x.data_ptr(), g.data_ptr(), _ptr(z), _ptr(self.bias), _ptr(state), self._output.data_ptr(),
            self._state.data_ptr(), _ptr(checkpoints), _stream(self._where)))
        self.output, self.state, self.checkpoints = self._output, self._state, checkpoints
        return self.output

    def forward(self, input, state=None, offsets=None):
        return self.updateOutput(input, state, offsets)

    def step(self, input, state):
        """One token: x, g and z are (sequences, channels), the states are updated in place."""
        x, g, z = self._table(input)
        key = (_layout(x), _layout(g), _layout(z))
        bias = self.bias
        if bias is not None and (bias.data_ptr(), bias.nbytes) != self._bias_place:  # _place, written out
            self._check_bias(x)
        if key != self._step_key:
            assert x.dim() == 2, "a step takes (sequences, channels)"
            self._check_table(x, g, z)
            desc = self._new_desc(x, g, z, None, x.shape[0], 1)
            self._step_key, self._step_desc = None, desc  # no key until all that belongs to it is there
            self._step_ref = ctypes.byref(self._step_desc)
            if self._step_captured:
                self._graphs.append(self._step_output)
            self._step_captured = False
            self._step_output = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            self._step_index, self._step_call = _device_index(x.device), capi.lib().fbfftconv_recurrence_step
            self._step_key, self._step_made = key, _raw_stream(self._step_index)
        if not self._step_captured:
            self._step_captured = _capturing()
        stream = _raw_stream(self._step_index)
        if stream != self._step_made:
            _used_here(self._step_index, self._step_made, (self._step_output,))
        assert state.shape == x.shape and state.dtype == torch.float32 and state.is_contiguous() and state.is_cuda
        status = self._step_call(
            self._step_ref, x.data_ptr(), g.data_ptr(), _ptr(z), None if bias is None else self._bias_place[0], state.data_ptr(),
            self._step_output.data_ptr(), stream)
        if status:
            capi.check(status)
        return self._step_output

    def backward(self, input, gradOutput, scale=None, *, state=None, offsets=None, gradState=None):
        """The table of gradients; `state` and `offsets` as updateOutput had them, gradState: the gradient by the final
        states, or None.  With either of the two states, gradState of the module is the one by the initial states."""
        return self._backward(input, gradOutput, 1.0 if scale is None else float(scale), state, offsets, gradState, True, True)

    def updateGradInput(self, input, gradOutput, *, state=None, offsets=None, gradState=None):
        return self._backward(input, gradOutput, 1.0, state, offsets, gradState, True, False)

    def accGradParameters(self, input, gradOutput, scale=None, *, state=None, offsets=None, gradState=None):
        self._backward(input, gradOutput, 1.0 if scale is None else float(scale), state, offsets, gradState, False, True)

    # -- internals -----------------------------------------------------------------
    def _table(self, input):
        assert len(input) == (3 if self.outputGate else 2), "the table is [x, g], with the output gate [x, g, z]"
        return input[0], input[1], input[2] if self.outputGate else None

    def _check_table(self, x, g, z):
        for t in (x, g, z):
            if t is None:
                continue
            assert isinstance(t, torch.Tensor) and t.is_cuda and t.device == x.device, "CUDA support only!"
            assert t.dtype in capi.element_types() and t.dtype == x.dtype, "x, g and z have one type: fp32, bf16 or fp16"
            assert t.shape == x.shape and t.shape[-1] == self.channels, "size mismatch"
        self._check_bias(x)

    def _check_bias(self, x):
        _check_parameter(self.bias, self.channels, x.device)
        self._bias_place = _place(self.bias)

    def _new_desc(self, x, g, z, offsets, sequences, length):
        rows = math.prod(x.shape[:-1])
        return capi.RecurrenceDesc(
            rows, sequences, length, _ptr(offsets), _row_stride(x), _row_stride(g), _row_stride(z), 0, 0, 0, 0, 0,
            int(offsets is not None and offsets.dtype == torch.int64), self.channels, capi.element_types()[x.dtype],
            _device_index(x.device))

    def _prepare(self, input, offsets):
        """Checks the table; descriptor and outputs are kept for one set of shapes."""
        x, g, z = self._table(input)
        key = (_layout(x), _layout(g), _layout(z), _layout(offsets))
        if _place(self.bias) != self._bias_place:
            self._check_bias(x)
        if key == self._key:
            if not self._captured:
                self._captured = _capturing()
            _used_here(self._index, self._made, (self._output, self._state, self._checkpoints, self._workspace, self._grad_state,
                                                 self._projection if self._grads else None))
        else:
            self._check_table(x, g, z)
            if offsets is None:
                assert x.dim() == 3, "(batch, length, channels), or packed (rows, channels) with offsets"
                sequences, length = x.shape[:2]
            else:
                assert x.dim() == 2, "packed rows are (rows, channels)"
                assert offsets.dim() == 1 and offsets.numel() >= 1 and offsets.device == x.device and offsets.is_contiguous()
                assert offsets.dtype in (torch.int32, torch.int64), "offsets are int32 or int64"
                sequences, length = offsets.numel() - 1, 0
            desc = self._new_desc(x, g, z, offsets, sequences, length)
            self._key, self._desc = None, desc  # no key until all that belongs to it is there
            self._desc_ref = ctypes.byref(self._desc)
            self._where, self._index = x.device, _device_index(x.device)
            self._made = _raw_stream(self._index)
            if self._captured:
                self._graphs.append((self._output, self._state, self._checkpoints, self._grads, self._workspace, self._grad_state))
            self._captured = _capturing()
            self._workspace = self._grad_state = self._output = self._state = None
            self._packed = offsets is not None
            self._output = self._rows(x, self.channels)
            self._state = torch.empty((sequences, self.channels), dtype=torch.float32, device=x.device)
            self._checkpoints = self._grads = None
            self.checkpoints = None
            self._key = key
        if offsets is not None:
            self._desc.offsets = offsets.data_ptr()
        return x, g, z

    def _check_state(self, state, what):
        if state is not None:
            assert state.shape == self._state.shape and state.dtype == torch.float32 and state.is_contiguous(), \
                f"the {what} is fp32 (sequences, channels)"
            assert state.device == self._where, "CUDA support only!"

    def _rows(self, x, channels):
        """A tensor of x's rows.  Packed ones outside of all sequences are never written: zeros, not what was in memory."""
        make = torch.zeros if self._packed else torch.empty
        return make(x.shape[:-1] + (channels,), dtype=x.dtype, device=x.device)

    def _another(self, t):
        """A tensor in the place of one that the module has given away."""
        if self._captured:
            self._graphs.append(t)
        self._made = self._made if _raw_stream(self._index) == self._made else -1  # of two streams: recorded on any
        return self._rows(t, self.channels) if t is self._output else torch.empty_like(t)

    def _backward(self, input, gradOutput, scale, state, offsets, gradState, inputs, parameters):
        kept = self.checkpoints
        x, g, z = self._prepare(input, offsets)
        assert kept is not None and self.checkpoints is kept, "updateOutput of the same inputs runs first, in training() mode"
        self._check_state(state, "initial state")
        self._check_state(gradState, "gradient by the final state")
        assert isinstance(gradOutput, torch.Tensor) and gradOutput.is_cuda and gradOutput.device == x.device, "CUDA support only!"
        assert gradOutput.shape == x.shape and gradOutput.dtype == x.dtype, "gradOutput size mismatch"
        parts = 3 if self.outputGate else 2
        if self._grads is None:
            self._projection = self._rows(x, parts * self.channels)
            n = int(capi.lib().fbfftconv_recurrence_workspace_bytes(self._desc_ref))
            self._workspace = torch.empty(max(n, 16), dtype=torch.uint8, device=x.device)
            self._grad_state = torch.empty_like(self._state)
            self._grads = list(self._projection.split(self.channels, -1))
            self._made = self._made if _raw_stream(self._index) == self._made else -1  # of two streams: recorded on any
            self._desc.grad_x_stride = self._desc.grad_g_stride = self._desc.grad_z_stride = parts * self.channels
        self._desc.grad_y_stride = _row_stride(gradOutput)
        states = inputs and (state is not None or gradState is not None)
        if states and gradState is not None and gradState.data_ptr() == self._grad_state.data_ptr():
            self._grad_state = self._another(self._grad_state)
        grads = [_ptr(t) if inputs else None for t in self._grads] + [None] * (3 - parts)
        with_bias = parameters and self.gradBias is not None
        if with_bias and _place(self.gradBias) != self._grad_place:
            _check_parameter(self.gradBias, self.channels, x.device)
            self._grad_place = _place(self.gradBias)
        capi.check(capi.lib().fbfftconv_recurrence_backward(
            self._desc_ref, x.data_ptr(), g.data_ptr(), _ptr(z), _ptr(self.bias), _ptr(state), kept.data_ptr(),
            gradOutput.data_ptr(), _ptr(gradState), *grads, self._grad_state.data_ptr() if states else None,
            self.gradBias.data_ptr() if with_bias else None, scale, int(self._accumulate), self._workspace.data_ptr(),
            self._workspace.numel(), _stream(self._where)))
        if inputs:
            self.gradInput, self.gradProjection = self._grads, self._projection
            self.gradState = self._grad_state if states else None
        return self.gradInput
