"""The recurrence's entry points refuse bad arguments before they touch a device, and its search over packed sequences
stays in bounds and ends for whatever the offsets hold (a host's copy of the kernel's index arithmetic)."""
import ctypes
import os
import random
import re

import pytest

from fbcunn_b200 import build as fb_build
from fbcunn_b200 import capi


@pytest.fixture(scope="module")
def lib():
    fb_build.build()
    return capi.lib()


def _desc(**kw):
    base = dict(rows=12, sequences=3, length=4, channels=64, type=capi.BFLOAT16, device=0)
    return capi.RecurrenceDesc(**{**base, **kw})


BAD = [dict(channels=0), dict(channels=-4), dict(channels=(1 << 22) + 1), dict(rows=-1), dict(sequences=-1), dict(length=-1),
       dict(type=5), dict(rows=13), dict(length=5), dict(length=0), dict(sequences=1 << 32, length=1 << 32, rows=0),
       dict(offsets=4098), dict(offsets=4100, wide_offsets=1), dict(rows=1 << 41, offsets=4096)]


@pytest.mark.parametrize("bad", range(len(BAD)))
def test_bad_descriptors(lib, bad):
    d = ctypes.byref(_desc(**BAD[bad]))
    refused = (capi.ERR_INVALID_ARGUMENT, capi.ERR_UNSUPPORTED_SIZE)
    assert lib.fbfftconv_recurrence(d, *[4096] * 8, None) in refused
    assert lib.fbfftconv_recurrence_backward(d, *[4096] * 13, 1.0, 0, 4096, 1 << 20, None) in refused
    assert lib.fbfftconv_recurrence_step(d, *[4096] * 6, None) in refused
    assert lib.fbfftconv_recurrence_checkpoint_bytes(d) == 0 and lib.fbfftconv_recurrence_workspace_bytes(d) == 0


def test_bad_pointers(lib):
    d = ctypes.byref(_desc())
    good = [4096, 8192, 12288, 16384, 20480, 24576, 28672, 32768]
    for i, value in [(0, None), (1, None), (5, None), (0, 4097), (2, 4097), (3, 4098), (4, 4098), (6, 20480), (7, 4098)]:
        args = list(good)
        args[i] = value
        assert lib.fbfftconv_recurrence(d, *args, None) == capi.ERR_INVALID_ARGUMENT
    overlap = ctypes.byref(_desc(x_stride=32))
    assert lib.fbfftconv_recurrence(overlap, *good, None) == capi.ERR_INVALID_ARGUMENT and "overlap" in capi.last_error()
    args = [4096 * (i + 1) for i in range(13)]
    assert lib.fbfftconv_recurrence_backward(d, *args, float("inf"), 0, 4096, 1 << 20, None) == capi.ERR_INVALID_ARGUMENT
    no_z = list(args)
    no_z[2] = None
    assert lib.fbfftconv_recurrence_backward(d, *no_z, 1.0, 0, 4096, 1 << 20, None) == capi.ERR_INVALID_ARGUMENT
    shared = list(args)
    shared[11] = shared[7]
    assert lib.fbfftconv_recurrence_backward(d, *shared, 1.0, 0, 4096, 1 << 20, None) == capi.ERR_INVALID_ARGUMENT
    assert lib.fbfftconv_recurrence_step(d, *good[:6], None) == capi.ERR_INVALID_ARGUMENT  # length 4


def test_search_over_any_offsets():
    rng = random.Random(1)
    for trial in range(3000):
        rows, n = rng.randint(1, 60), rng.randint(1, 9)
        offsets = [rng.choice([rng.randint(0, rows), rng.randint(-100, 100), 1 << 40]) for _ in range(n + 1)]
        if trial % 3 == 0:
            offsets = sorted(rng.randint(0, rows) for _ in range(n + 1))
        at = lambda i: min(max(offsets[i], 0), rows)
        def sequence_of(row):
            lo, hi = 0, n
            while hi - lo > 1:
                mid = (lo + hi) // 2
                lo, hi = (mid, hi) if at(mid) <= row else (lo, mid)
            assert 0 <= lo < n
            return at(lo), at(lo + 1)
        begin, end = at(0), at(n)
        for row in range(begin, end, 16):
            count, first, last, turns = min(16, end - row), 0, 0, 0
            lo, hi = sequence_of(row)
            first = int(row == lo)
            while hi > row and hi - row <= count:
                turns += 1
                assert turns <= 17, "no end"
                k = hi - row
                last |= 1 << (k - 1)
                if k == count:
                    break
                first |= 1 << k
                lo, more = sequence_of(hi)
                if more <= hi:
                    break
                hi = more
            assert first < 1 << count and last < 1 << count
            if trial % 3 == 0:  # sorted: exactly the rows that begin and end a sequence
                starts = {offsets[i] for i in range(n) if offsets[i] < offsets[i + 1]}
                ends = {offsets[i + 1] - 1 for i in range(n) if offsets[i] < offsets[i + 1]}
                assert [first >> i & 1 for i in range(count)] == [int(row + i in starts) for i in range(count)]
                assert [last >> i & 1 for i in range(count)] == [int(row + i in ends) for i in range(count)]


def _turns(name):
    """How many buffers the exchange between warps and blocks keeps of `name`: what the kernels' source says."""
    with open(os.path.join(fb_build.CSRC, "recurrence.cu")) as f:
        source = f.read()
    constant = int(re.search(r"constexpr int kTurns = (\d+);", source).group(1))
    fields = re.search(r"struct Exchange \{(.*?)\};", source, re.S).group(1)
    return constant if re.search(r"\b%s\[kTurns\]" % name, fields) else 1


def _unordered(blocks, backward, part, whole, warps=8, rounds=5):
    """Reads and writes of the same place of a cluster's exchange that nothing orders, at least one of them a write:
    barriers, the counted stores that a wait is for and each warp's program order are what orders them."""
    before, at = [], {}  # for each event the events that it follows, as bits; places -> [(event, is a write)]

    def event(*after, use=()):
        seen = 0
        for a in after:
            seen |= before[a] | 1 << a
        before.append(seen)
        for place, write in use:
            at.setdefault(place, []).append((len(before) - 1, write))
        return len(before) - 1

    last = {(b, w): event() for b in range(blocks) for w in range(warps)}
    everyone = [(b, w) for b in range(blocks) for w in range(warps)]

    def barrier():
        for b in range(blocks):
            met = event(*[last[b, w] for w in range(warps)])
            for w in range(warps):
                last[b, w] = event(last[b, w], met)

    for r in range(rounds):
        order = lambda w: warps - 1 - w if backward else w
        if backward:
            barrier()  # the one of the rows' states
        for b, w in everyone:
            last[b, w] = event(last[b, w], use=[(("part", b, r % part, order(w)), True)])
        barrier()
        for b, w in everyone:
            last[b, w] = event(last[b, w], use=[(("part", b, r % part, k), False) for k in range(warps) if k != order(w)])
        armed, sent = {}, {b: [] for b in range(blocks)}
        for b in range(blocks):
            if blocks > 1:
                last[b, 0] = armed[b] = event(last[b, 0])
        for b, w in everyone:
            for k in range(order(w), blocks if blocks > 1 else 0, warps):
                last[b, w] = event(last[b, w], use=[(("whole", k, r % whole, b), True)])
                sent[k].append(last[b, w])
        for b, w in everyone:
            if blocks > 1:
                last[b, w] = event(last[b, w], armed[b], *sent[b])
                last[b, w] = event(last[b, w], use=[(("whole", b, r % whole, k), False) for k in range(blocks)])
    return {place[0] for place, uses in at.items() for i, (x, wx) in enumerate(uses) for y, wy in uses[i + 1:]
            if (wx or wy) and not (before[y] >> x & 1 or before[x] >> y & 1)}


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("blocks", [1, 2, 3, 10])
def test_nothing_is_written_while_it_is_read(blocks, backward):
    assert not _unordered(blocks, backward, _turns("part"), _turns("whole"))
    # one buffer of the warps' stretches would be written early in the forward pass, one of the blocks' in both
    assert _unordered(blocks, backward, 1, 2) == (set() if backward else {"part"})
    if blocks > 1:
        assert "whole" in _unordered(blocks, backward, 2, 1)


def _run_cluster(rng, blocks, rounds, stays):
    """One run of a cluster whose waits may run out, in an order of steps that chance decides: the blocks that were sent
    to after they had left, and whether all ended.  A block waits for all stretches of a round, or until chance ends the
    wait; after that it goes on without sending, counting or waiting."""
    state = [dict(round=0, step="send", lost=False, got=[0] * (rounds + 2)) for _ in range(blocks)]
    arrived, sent_to_the_gone = 0, set()
    for _ in range(200 * blocks * rounds):
        alive = [b for b in state if b["step"] != "gone"]
        if not alive:
            break
        b = rng.choice(alive)
        if b["step"] == "send":
            if not b["lost"]:
                for k, other in enumerate(state):
                    if other["step"] == "gone":
                        sent_to_the_gone.add(k)
                    other["got"][b["round"]] += 1
            b["step"] = "wait"
        elif b["step"] == "wait":
            if not b["lost"] and b["got"][b["round"]] < blocks:
                if rng.random() > 0.02:
                    continue
                b["lost"] = True
            b["round"] += 1
            b["step"] = "send" if b["round"] < rounds else "end"
            if b["step"] == "end":
                arrived += 1
        elif not stays or arrived == blocks:
            b["step"] = "gone"
    return sent_to_the_gone, all(b["step"] == "gone" for b in state)


def test_a_block_whose_wait_ran_out_stays_until_no_other_can_send():
    with open(os.path.join(fb_build.CSRC, "recurrence.cu")) as f:
        kernels = [k.split("\ntemplate")[0] for k in f.read().split("__launch_bounds__(kThreads, 2)")[1:]]
    assert len(kernels) == 2
    stays = all(k.rfind("finish_exchange(") > k.rfind("exchange(shared, (uint32_t)round") > 0 for k in kernels)
    rng, too_early = random.Random(3), 0
    for trial in range(400):
        blocks, rounds = rng.randint(2, 16), rng.randint(1, 6)
        gone, ended = _run_cluster(rng, blocks, rounds, stays)
        assert not gone and ended
        too_early += bool(_run_cluster(rng, blocks, rounds, False)[0])
    assert too_early  # what the last barrier is for


def test_the_limit_of_waits(lib):
    before = lib.fbfftconv_recurrence_wait_limit(5)
    assert before >= 100000 and lib.fbfftconv_recurrence_wait_limit(before) == 5
    assert lib.fbfftconv_recurrence_wait_limit(before) == before


@pytest.mark.parametrize("field", ["x_stride", "g_stride", "z_stride", "y_stride", "grad_y_stride", "grad_x_stride", "grad_g_stride",
                                   "grad_z_stride"])
@pytest.mark.parametrize("stride", [-64, -(1 << 32) + 64, -(1 << 63)])
def test_negative_strides(lib, field, stride):
    """Also those that would be a sound one in 32 bits."""
    d = ctypes.byref(_desc(**{field: stride}))
    args = [4096 * (i + 1) for i in range(13)]
    for rc in (lib.fbfftconv_recurrence(d, *args[:8], None),
               lib.fbfftconv_recurrence_backward(d, *args, 1.0, 0, 4096, 1 << 20, None)):
        assert rc == capi.ERR_INVALID_ARGUMENT and "negative stride" in capi.last_error()


def test_every_kernel_has_a_place_in_the_table_of_cluster_counts():
    """On each device: a kernel without one would ask the driver at every call."""
    with open(os.path.join(fb_build.CSRC, "recurrence.cu")) as f:
        source = f.read()
    layouts = re.search(r"#define BY_TYPE\(call\)(.*?)\n\n", source, re.S).group(1).count("call(")
    kernels = len(re.findall(r"launch_divided\(\w+_kernel<T, V, \w+>", source)) * layouts
    assert kernels == int(re.search(r"kDividedKernels = (\d+);", source).group(1))
    assert re.search(r"known\[kMostDevices\]\[kDividedKernels\];", source)
