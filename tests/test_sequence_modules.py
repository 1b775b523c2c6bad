"""What the modules of the sequence operators keep from call to call, on the host: their native calls are recorded, not
made, and tensors of the host stand for the device's."""
import ctypes

import pytest
import torch

from fbcunn_b200 import AdamW, GatedLinearRecurrence, GatedResidualNorm, adamw, capi, module, recurrence, residual_norm


class OnDevice(torch.Tensor):
    """A tensor of the host that says it lies on the device."""
    is_cuda = property(lambda self: True)


class Host:
    """Stands for the library and the stream: calls are (name, arguments), with descriptors and tables copied."""

    def __init__(self):
        self.calls, self.stream, self.capturing, self.recorded, self.refused = [], 0, False, [], ""

    def __getattr__(self, name):
        if not name.startswith("fbfftconv_"):
            raise AttributeError(name)

        def call(*args):
            self.calls.append((name, [self._copy(a) for a in args]))
            if name.endswith("_bytes"):
                return 64
            if name == "fbfftconv_last_error":
                return b"refused"
            if name == self.refused:
                return capi.ERR_INVALID_ARGUMENT
            if name == "fbfftconv_adamw_create":
                args[3]._obj.value = 1
            return 0
        return call

    @staticmethod
    def _copy(a):
        value = getattr(a, "_obj", a)
        if isinstance(value, ctypes.Structure):
            return type(value).from_buffer_copy(value)
        if isinstance(value, ctypes.Array):
            return [type(t).from_buffer_copy(t) for t in value]
        return value

    def last(self, name):
        return next(args for n, args in reversed(self.calls) if n == name)


@pytest.fixture
def host(monkeypatch):
    h = Host()
    monkeypatch.setattr(capi, "lib", lambda: h)
    for m in (module, recurrence, residual_norm, adamw):
        for name, value in (("_raw_stream", lambda index: h.stream), ("_stream", lambda device: h.stream),
                            ("_capturing", lambda: h.capturing), ("_device_index", lambda device: 0)):
            if hasattr(m, name):
                monkeypatch.setattr(m, name, value)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index=None: h.stream)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, stream: h.recorded.append((t.data_ptr(), stream)))
    return h


def made(*shape, dtype=torch.float32):
    return torch.ones(shape, dtype=dtype).as_subclass(OnDevice)


def recurrent(channels=8, **kw):
    return GatedLinearRecurrence(channels, device="cpu", **kw)


def norm(channels=8, **kw):
    return GatedResidualNorm(channels, device="cpu", **kw)


def recurrence_table(n, length=3, channels=8):
    return [made(n, length, channels) for _ in range(3)]


def norm_table(n, channels=8):
    return [made(n, channels) for _ in range(2)]


CALLS = [  # (module, table of n rows or sequences, the call, the native entry, the descriptor's field that has n)
    (recurrent, recurrence_table, lambda m, t: m.updateOutput(t), "fbfftconv_recurrence", "sequences"),
    (recurrent, lambda n: [made(n, 8) for _ in range(3)], lambda m, t: m.step(t, made(t[0].shape[0], 8)),
     "fbfftconv_recurrence_step", "sequences"),
    (norm, norm_table, lambda m, t: m.updateOutput(t), "fbfftconv_residual_norm", "rows")]


def _no_memory(monkeypatch, after):
    """Allocations fail from the `after`-th on."""
    left = [after]

    def failing(make):
        def call(*args, **kw):
            left[0] -= 1
            if left[0] < 0:
                raise torch.OutOfMemoryError("no memory")
            return make(*args, **kw)
        return call
    for name in ("empty", "empty_like"):
        monkeypatch.setattr(torch, name, failing(getattr(torch, name)))


@pytest.mark.parametrize("which", range(len(CALLS)))
@pytest.mark.parametrize("after", [0, 1, 2])
def test_a_call_that_found_no_memory_leaves_nothing_behind(host, monkeypatch, which, after):
    """What a call of the first shape launches after a larger one has failed is described as it is, with tensors of its
    size."""
    build, table, call, entry, field = CALLS[which]
    m, small, large = build(), table(2), table(500)
    call(m, small)
    with monkeypatch.context() as patch:
        _no_memory(patch, after)
        try:
            call(m, large)
        except torch.OutOfMemoryError:
            pass
    for t in (small, large, small):
        out = call(m, t)
        assert getattr(host.last(entry)[0], field) == t[0].shape[0]
        out = out[0] if isinstance(out, list) else out
        assert out.shape == t[0].shape
        tensors = [v for v in vars(m).values() if isinstance(v, torch.Tensor)]
        assert out.data_ptr() in host.last(entry) and any(v.data_ptr() == out.data_ptr() for v in tensors)


@pytest.mark.parametrize("build,table,grads", [
    (recurrent, recurrence_table, lambda t: t[0]), (norm, norm_table, lambda t: t)])
def test_a_refused_call_or_one_without_memory_leaves_the_backward_pass(host, monkeypatch, build, table, grads):
    m, t = build(), table(2)
    m.updateOutput(t)
    with pytest.raises(AssertionError):
        m.updateOutput([x[..., :4] for x in t])
    for after in (0, 1, 2):
        with monkeypatch.context() as patch:
            _no_memory(patch, after)
            with pytest.raises(torch.OutOfMemoryError):
                m.backward(t, grads(t))
        assert not any(name.endswith("_backward") for name, _ in host.calls)
    got = m.backward(t, grads(t))
    assert all(g.shape == x.shape for g, x in zip(got, t))
    name, args = host.calls[-1]
    assert name.endswith("_backward") and all(g.data_ptr() in args for g in got)
    if build is recurrent:
        assert args[0].grad_x_stride == args[0].grad_z_stride == 24


STEPS = [lambda m, t: m.updateOutput(t), lambda m, t: m.step([x[:, 0] for x in t], made(2, 8))]
REPLACED = {  # what may become of a parameter between two calls, and whether the call can still be made
    "fewer": (lambda p: p[:3].clone(), False), "half": (lambda p: p.half(), False),
    "apart": (lambda p: torch.zeros(16).as_subclass(OnDevice)[::2], False),
    "other": (lambda p: torch.full_like(p, 2.0), True)}


@pytest.mark.parametrize("as_data", [False, True])
@pytest.mark.parametrize("how", REPLACED)
def test_replaced_parameters_are_looked_at(host, how, as_data):
    """As another tensor or in the same one; a sound one is used from then on, with the outputs that are there."""
    make, sound = REPLACED[how]

    def replace(m, name):
        p = getattr(m, name)
        new = make(p)
        if as_data:
            try:
                p.data = new
            except RuntimeError:  # of another type: not every version of the library allows that
                pytest.skip("such a replacement is refused before it reaches the module")
        else:
            setattr(m, name, new)
        return new

    def used(call, address):
        if not sound:
            with pytest.raises(AssertionError):
                call()
            return
        out = call()
        assert address in host.calls[-1][1]
        return out

    for step in STEPS:
        m, t = recurrent(), recurrence_table(2)
        step(m, t)
        new = replace(m, "bias")
        used(lambda: step(m, t), new.data_ptr())
    for name in ("postWeight", "preBias"):
        m, t = norm(normBias=True), norm_table(2)
        before = m.updateOutput(t)[0].data_ptr()
        new = replace(m, name)
        out = used(lambda: m.updateOutput(t), new.data_ptr())
        assert not sound or out[0].data_ptr() == before
    for name, m, t, dy in (("gradBias", recurrent(), recurrence_table(2), made(2, 3, 8)),
                           ("gradPostWeight", norm(), norm_table(2), norm_table(2)),
                           ("gradPreBias", norm(normBias=True), norm_table(2), norm_table(2))):
        for again in (False, True):
            m.updateOutput(t)
            if again:
                m.backward(t, dy)
            new = replace(m, name)
            used(lambda: m.backward(t, dy), new.data_ptr())
            m.updateGradInput(t, dy)  # which does not touch it
            setattr(m, name, made(8))


def test_outputs_that_are_given_back_stay_what_they_are(host):
    """A module that is applied again to what it returned writes to other tensors."""
    m, t = recurrent(), recurrence_table(2)
    for place in range(3):
        t[place] = m.updateOutput(t).as_subclass(OnDevice)
        again = m.updateOutput(t)
        assert again.data_ptr() != t[place].data_ptr() and again.data_ptr() in host.calls[-1][1]
        assert m.output is again and again.shape == t[place].shape
    m, t = norm(gate="linear"), norm_table(2) + [made(2, 8)]
    for place in range(3):
        for which in range(2):
            t[place] = m.updateOutput(t)[which].as_subclass(OnDevice)
            again = m.updateOutput(t)
            assert all(a.data_ptr() in host.calls[-1][1] for a in again)
            assert not {a.data_ptr() for a in again} & {x.data_ptr() for x in t}
    kept = [a.data_ptr() for a in m.updateOutput([x.clone() for x in t])]
    assert kept == [a.data_ptr() for a in m.updateOutput([x.clone() for x in t])]  # else the same ones are used again
    entry = norm(post=None)
    v = entry.updateOutput(made(2, 8)).as_subclass(OnDevice)
    assert entry.updateOutput(v).data_ptr() != v.data_ptr()
    for m, t in ((entry, [made(0, 8)]), (norm(), norm_table(0)), (norm(pre=None), norm_table(0)), (recurrent(), recurrence_table(0))):
        out = m.updateOutput(t)
        assert (out[-1] if isinstance(out, list) else out).numel() == 0 and m.updateOutput(t) is not None


def test_outputs_of_a_captured_graph_that_are_given_back_are_kept(host):
    host.capturing = True
    for m, t, at in ((recurrent(), recurrence_table(2), 0), (norm(), norm_table(2), 1)):
        out = m.updateOutput(t)
        out = out[0] if isinstance(out, list) else out
        t[at] = out.as_subclass(OnDevice)
        m.updateOutput(t)
        assert any(k is out for kept in m._graphs for k in (kept if isinstance(kept, tuple) else (kept,)))


def test_what_was_made_on_another_stream_in_between_is_recorded(host):
    """Tensors that were made anew on stream 2, in the place of some of stream 1, are recorded when stream 1 uses them."""
    def swap_state(m, t):
        m.updateOutput(t, state=m.state)

    def swap_output(m, t):
        m.updateOutput([m.output] + t[1:])

    def swap_grad_state(m, t):
        m.updateOutput(t)
        m.backward(t, t[0], gradState=m.gradState)

    cases = [(recurrent, recurrence_table, swap_state, lambda m: m.state),
             (recurrent, recurrence_table, swap_output, lambda m: m.output),
             (recurrent, recurrence_table, swap_grad_state, lambda m: m.gradState),
             (norm, norm_table, lambda m, t: m.updateOutput([t[0], m.output[0]]), lambda m: m.output[0])]
    for build, table, swap, what in cases:
        host.stream = 1
        m, t = build(), table(2)
        m.updateOutput(t)
        if build is recurrent:
            m.backward(t, t[0], state=made(2, 8), gradState=made(2, 8))
        host.stream = 2
        swap(m, t)
        new = what(m).data_ptr()
        host.stream, host.recorded = 1, []
        m.updateOutput(t)
        assert (new, 1) in host.recorded


def optimizer(sizes=(4, 600, 30), **kw):
    params = [made(n) for n in sizes]
    grads = [made(n) for n in sizes]
    return AdamW(params, grads, **kw), params, grads


def test_replaced_storage_of_optimized_tensors_is_looked_at(host):
    """As long as a tensor fits its moments it may lie elsewhere; what does not is refused before anything is launched."""
    opt, params, grads = optimizer(masters=[None] * 3)
    params[1].data = made(600)
    opt.step()
    assert host.last("fbfftconv_adamw_create")[0][1].param == params[1].data_ptr()
    fits, steps = {"param": params, "grad": grads}, sum(n == "fbfftconv_adamw_step" for n, _ in host.calls)
    for which, tensors in fits.items():
        for bad in (made(700), made(500), torch.zeros(1200).as_subclass(OnDevice)[::2], made(600).half().int(), made(20, 30)):
            kept = tensors[1].data
            try:
                tensors[1].data = bad
            except RuntimeError:
                continue
            if bad.shape == (20, 30) and which == "param":
                grads[1].data = bad  # a shape of as many elements is no other size
                opt.step()
                steps += 1
                grads[1].data = made(600)
            else:
                with pytest.raises(AssertionError):
                    opt.step()
                with pytest.raises(AssertionError):
                    opt.step()  # it stays refused
            tensors[1].data = kept
            opt.step()
            steps += 1
            assert sum(n == "fbfftconv_adamw_step" for n, _ in host.calls) == steps


def test_a_tensor_of_another_size_at_the_same_address_is_looked_at(host):
    opt, params, grads = optimizer()
    opt.step()
    for tensors in (params, grads):
        kept = tensors[2].data
        tensors[2].data = kept[:10]
        assert tensors[2].data_ptr() == kept.data_ptr()
        with pytest.raises(AssertionError):
            opt.step()
        tensors[2].data = kept


def test_masters_are_looked_at(host):
    params, grads = [made(64, dtype=torch.bfloat16)], [made(64)]
    opt = AdamW(params, grads, masters=[made(64)])
    opt.step()
    opt.masters[0].data = made(32)
    with pytest.raises(AssertionError):
        opt.step()


def test_the_state_has_the_masters_that_were_made_here(host):
    def build(**kw):
        params = [torch.full((40,), 1.0 + 2.0 ** -6, dtype=torch.bfloat16).as_subclass(OnDevice), made(8)]
        return AdamW(params, [made(40), made(8)], **kw), params

    opt, params = build(masters=True)
    opt.masters[0].add_(2.0 ** -12)  # what 16 bits do not hold
    state = opt.state()
    assert state["masters"][1] is None and state["masters"][0].data_ptr() != opt.masters[0].data_ptr()
    other, theirs = build(masters=True)
    theirs[0].zero_()
    other.loadState(state)
    assert torch.equal(other.masters[0], opt.masters[0]) and torch.equal(theirs[0], opt.masters[0].bfloat16())
    for bad in ({k: v for k, v in state.items() if k != "masters"}, dict(state, masters=state["masters"][:1]),
                dict(state, masters=[None, None]), dict(state, masters=[state["masters"][0][:7], None])):
        before = {k: v.clone() for k, v in other.moments.items()}
        with pytest.raises(AssertionError):
            other.loadState(bad)
        assert all(torch.equal(before[k], v) for k, v in other.moments.items())
    adopted, _ = build(masters=[made(40), None])
    assert "masters" not in adopted.state()
    adopted.loadState(adopted.state())
    with pytest.raises(AssertionError):
        adopted.loadState(state)


def test_hyperparameters_may_change_between_steps(host):
    opt, *_ = optimizer()
    opt.step()
    made_once = sum(n == "fbfftconv_adamw_create" for n, _ in host.calls)
    opt.step()
    assert sum(n == "fbfftconv_adamw_create" for n, _ in host.calls) == made_once
    for name, value, field in (("weightDecay", 0.5, "weight_decay"), ("eps", 1e-5, "eps"), ("seed", 9, "seed")):
        setattr(opt, name, value)
        opt.step()
        assert getattr(host.last("fbfftconv_adamw_create")[2], field) == value
    opt.betas = (0.5, 0.25)
    opt.lr = 0.125
    opt.step()
    assert host.last("fbfftconv_adamw_create")[2].beta2 == 0.25 and host.last("fbfftconv_adamw_step")[1] == 0.125


def test_packed_rows_that_no_sequence_has_are_zero(host, monkeypatch):
    """In new outputs and gradients, and in those that take the place of given-away ones."""
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: empty(*a, **kw).fill_(77))
    m, t = recurrent(), [made(9, 8) for _ in range(3)]
    offsets = torch.tensor([0, 2, 5])
    for _ in range(2):
        y = m.updateOutput(t, offsets=offsets)
        assert not y.any() and not any(g.any() for g in m.backward(t, t[0], offsets=offsets))
        t[0] = y.as_subclass(OnDevice)
    assert m.updateOutput(recurrence_table(2)).any()  # padded rows are all written


@pytest.mark.parametrize("build,table,entry", [(recurrent, recurrence_table, "fbfftconv_recurrence"),
                                               (norm, norm_table, "fbfftconv_residual_norm")])
def test_no_backward_pass_of_a_refused_forward_pass(host, build, table, entry):
    m, t = build(), table(2)
    host.refused = entry
    with pytest.raises(capi.FbfftconvError):
        m.updateOutput(t)
    with pytest.raises(AssertionError):
        m.backward(t, t[0] if build is recurrent else t)
    host.refused = ""
    m.updateOutput(t)
    m.backward(t, t[0] if build is recurrent else t)
