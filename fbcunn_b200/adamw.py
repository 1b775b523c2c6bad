"""One AdamW step over many tensors: what consumes the gradients that accGradParameters leaves.

``AdamW`` holds the moments of a list of parameters, in 32 bits or in 8, and steps them all in one launch
(fbfftconv_adamw_* in include/fbfftconv.h, which has the formulas).  The step count lives on the device, so a step
can be captured into a CUDA graph and replayed.
"""
from __future__ import annotations

import ctypes
import operator

import torch

from . import capi
from .module import _device_index, _stream

_BLOCK = 256  # elements that share a scale

# of every tensor at every step: what has another address or size is looked at anew
_address, _nbytes = torch.Tensor.data_ptr, operator.attrgetter("nbytes")


class AdamW:
    """AdamW(params, grads): two lists of tensors, or AdamW(modules) for the parameters of modules.

    stateBits      32, or 8: e4m3 moments with a scale for every 256 elements, for tensors of at least
                   `min8bitSize` elements (smaller ones keep 32 bits: their codes would save nothing)
    masters        for 16-bit parameters: a list of fp32 tensors that are the weights themselves (adopted, not
                   copied; None for fp32 parameters), or True to make them from the parameters; those are part of
                   state(), adopted ones are the caller's to save
    seed           of the random rounding of 8-bit moments

    lr, betas, eps, weightDecay and seed may be set anew between steps; they are those of all tensors: parameters that are
    not to be decayed belong to an optimizer of their own, which is one launch more.
    Tensors are contiguous and on one GPU; gradients have their parameter's shape and any of the three types.
    A tensor whose storage has been replaced since the last step is noticed and used from then on, if it is still such
    a tensor of as many elements."""

    def __init__(self, params, grads=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weightDecay=1e-2, *, stateBits=32,
                 min8bitSize=4096, masters=None, seed=0):
        params = list(params)
        if grads is None:
            modules, params, grads = params, [], []
            for m in modules:
                p, g = m.parameters()
                params += p
                grads += g
        self.params, self.grads = params, list(grads)
        assert len(self.params) == len(self.grads), "one gradient for each parameter"
        assert self.params, "no parameters"
        assert stateBits in (8, 32), "moments are held in 8 or 32 bits"
        self.lr, self.betas, self.eps, self.weightDecay = float(lr), tuple(map(float, betas)), float(eps), float(weightDecay)
        self.stateBits, self.min8bitSize, self.seed = int(stateBits), int(min8bitSize), int(seed)
        assert len(self.betas) == 2 and 0 <= self.seed < 1 << 32
        for t in self.params + self.grads:
            assert isinstance(t, torch.Tensor) and t.is_cuda, "CUDA support only!"
        self.device = self.params[0].device
        self._own_masters = masters is True
        if masters is True:
            masters = [None if p.dtype == torch.float32 else p.detach().float().contiguous() for p in self.params]
        self.masters = list(masters) if masters is not None else [None] * len(self.params)
        assert len(self.masters) == len(self.params), "one master for each parameter"
        self._counts = [p.numel() for p in self.params]
        self._check()
        # where each tensor's moments lie: (bits, first element) in the flat tensors, a tensor starts on a block
        size, self.layout = {8: 0, 32: 0}, []
        for p in self.params:
            bits = 8 if self.stateBits == 8 and p.numel() >= self.min8bitSize else 32
            self.layout.append((bits, size[bits]))
            size[bits] += -(-p.numel() // _BLOCK) * _BLOCK

        def zeros(n, dtype=torch.float32):
            return torch.zeros(n, dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype, device=self.device).view(dtype)

        self.moments = {}
        if size[32]:
            self.moments |= {"m": zeros(size[32]), "v": zeros(size[32])}
        if size[8]:
            for key in ("m8", "r8"):  # m and sqrt(v)
                self.moments[key] = zeros(size[8], torch.float8_e4m3fn)
                self.moments[key + "_scale"] = zeros(size[8] // _BLOCK)
        self._counter = zeros(2, torch.int64)
        self._handle = None
        self._watched = None
        self._rebuild()

    @property
    def steps(self) -> int:
        """Steps done so far (waits for the device)."""
        return int(self._counter[0])

    def setGradients(self, grads):
        """Other gradient tensors of the same sizes and types from the next step on."""
        grads = list(grads)
        assert len(grads) == len(self.params), "one gradient for each parameter"
        for p, g, old in zip(self.params, grads, self.grads):
            assert isinstance(g, torch.Tensor) and g.device == self.device and g.is_contiguous()
            assert g.shape == p.shape and g.dtype == old.dtype, "gradient size or type mismatch"
        before, self.grads = self.grads, grads
        try:
            self._rebuild()
        except capi.FbfftconvError:
            self.grads = before
            raise

    def step(self, lr=None, gradScale=1.0, scalars=None):
        """One step on the current stream.  gradScale multiplies the gradients; scalars, a tensor of two floats on the
        device, stands for (lr, gradScale) and is read there, for captured steps."""
        if scalars is not None:
            assert scalars.device == self.device and scalars.dtype == torch.float32 and scalars.numel() == 2
            assert scalars.is_contiguous()
            scalars = scalars.data_ptr()
        if list(map(_address, self._watched)) != self._addresses or list(map(_nbytes, self._watched)) != self._sizes:
            self._check()
            self._rebuild()
        elif self._built != (self.betas, self.eps, self.weightDecay, self.seed):
            self._rebuild()
        capi.check(capi.lib().fbfftconv_adamw_step(
            self._handle, self.lr if lr is None else lr, gradScale, scalars, _stream(self.device)))

    def state(self) -> dict:
        """The moments, the step count and the masters that were made here, as loadState takes them."""
        state = dict({k: v.clone() for k, v in self.moments.items()}, steps=self.steps)
        if self._own_masters:
            state["masters"] = [None if w is None else w.clone() for w in self.masters]
        return state

    def loadState(self, state):
        """Takes up where state() was asked for.  Parameters with masters of the state become their rounded copies."""
        masters = state.get("masters", []) if self._own_masters else []
        assert set(state) == set(self.moments) | {"steps"} | ({"masters"} if self._own_masters else set()), \
            "the state of other parameters, or of masters that are kept elsewhere"
        assert not self._own_masters or len(masters) == len(self.masters), "the state of other parameters"
        kept = [(self.moments[k], state[k]) for k in self.moments]
        for w, saved in zip(self.masters, masters):
            assert (w is None) == (saved is None), "the state of other parameters"
            if w is not None:
                kept.append((w, saved))
        for t, saved in kept:
            assert saved.shape == t.shape and saved.dtype == t.dtype, "the state of other parameters"
        for t, saved in kept:
            t.copy_(saved)
        for p, w in zip(self.params, self.masters):
            if self._own_masters and w is not None:
                p.detach().copy_(w)
        self._counter[0] = int(state["steps"])

    # -- internals -----------------------------------------------------------------
    def _check(self):
        for p, g, w, n in zip(self.params, self.grads, self.masters, self._counts):
            assert p.numel() == n, "a parameter has another size than its moments"
            assert g.shape == p.shape, "gradient size mismatch"
            assert w is None or (w.device == self.device and w.shape == p.shape and w.dtype == torch.float32 and w.is_contiguous())
            assert all(t.is_contiguous() and t.device == self.device and t.dtype in capi.element_types() for t in (p, g))

    def _rebuild(self):
        """The native handle for the tensors as they are now."""
        tensors = (capi.AdamwTensor * len(self.params))()
        types = capi.element_types()
        for t, p, g, w, (bits, at) in zip(tensors, self.params, self.grads, self.masters, self.layout):
            first, second = (("m8", "r8") if bits == 8 else ("m", "v"))
            t.param, t.grad, t.master = p.data_ptr(), g.data_ptr(), None if w is None else w.data_ptr()
            t.count, t.param_type, t.grad_type = p.numel(), types[p.dtype], types[g.dtype]
            if p.numel() == 0:
                continue
            width = 1 if bits == 8 else 4
            t.moment1 = self.moments[first].data_ptr() + width * at
            t.moment2 = self.moments[second].data_ptr() + width * at
            if bits == 8:
                t.scale1 = self.moments["m8_scale"].data_ptr() + 4 * (at // _BLOCK)
                t.scale2 = self.moments["r8_scale"].data_ptr() + 4 * (at // _BLOCK)
        options = capi.AdamwOptions(*self.betas, self.eps, self.weightDecay, self._counter.data_ptr(), self.seed,
                                    _device_index(self.device))
        handle = ctypes.c_void_p()
        capi.check(capi.lib().fbfftconv_adamw_create(tensors, len(self.params), ctypes.byref(options),
                                                     ctypes.byref(handle)))
        self._destroy()
        self._handle = handle
        self._built = (self.betas, self.eps, self.weightDecay, self.seed)
        self._watched = self.params + self.grads + [w for w in self.masters if w is not None]
        self._addresses, self._sizes = list(map(_address, self._watched)), list(map(_nbytes, self._watched))

    def _destroy(self):
        if self._handle is not None:
            capi.lib().fbfftconv_adamw_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self._destroy()
        except Exception:
            pass
