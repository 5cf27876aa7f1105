"""The operators' workspace on the hip device, without a GPU: one buffer for calls of every size, given back when a larger one
takes its place or memory runs out, and kept by the launch lists that name it. Plans of stub calls on a fake runtime."""

from __future__ import annotations

import collections
import ctypes

import pytest

from limn_amd.hip import replay
from limn_amd.hip.device import HipDevice
from limn_amd.seam import Call, Plan


class FakeHip:
    """hipMalloc and hipFree over made-up addresses, up to `room` bytes at a time."""

    def __init__(self, room=1 << 60):
        self.room, self.next_ptr, self.live, self.most = room, 0x10000, {}, 0

    def hipMalloc(self, ptr_ref, nbytes):
        if sum(self.live.values()) + nbytes > self.room:
            return 2
        ptr_ref._obj.value = self.next_ptr
        self.live[self.next_ptr] = nbytes
        self.next_ptr += (nbytes + 0xFFFF) // 0x10000 * 0x10000
        self.most = max(self.most, sum(self.live.values()))
        return 0

    def hipFree(self, ptr):
        del self.live[ptr.value]
        return 0

    def hipDeviceSynchronize(self):
        return 0


class Lib:
    """The library's replay entries: what each list was given as its workspace, and the graphs freed."""

    def __init__(self):
        self.named, self.freed = [], []

    def limn_hip_replay(self, steps, nsteps, args, nargs, slots, nslots, stream):
        self.named.append(ctypes.cast(args, ctypes.POINTER(ctypes.c_int64))[0])
        return 0

    def limn_hip_replay_graph_free(self, handle):
        self.freed.append(handle.value)
        return 0


def device(room=1 << 60):
    dev = HipDevice.__new__(HipDevice)
    dev.api, dev.lib, dev.pool = FakeHip(room), Lib(), {}
    dev._commits, dev._commit_targets, dev._committed = [], set(), []
    dev.replays, dev.replay_graphs, dev.issue_seconds, dev.tape = collections.OrderedDict(), False, 0.0, None
    return dev


def large(dev):
    """Allocations beside the one byte that a launch list without outputs has for them."""
    return [n for n in dev.api.live.values() if n > 1]


def plan(dev, need, out=()):
    """A plan of one call that takes a workspace of `need` bytes, and a launch that names it."""

    def fn(inputs, outs):
        ws, room = dev._scratch(need)
        assert room == need and (ws is None) == (need == 0)
        if need:
            base = max(p for p in dev.api.live if p <= ws)
            assert ws + need <= base + dev.api.live[base]  # inside what the runtime still has allocated
        if dev.tape is not None:
            dev.tape.append(replay.Launch(replay.STEP_KERNEL, (ws or 0,)))

    call = Call(fn=fn, inputs=(), outputs=tuple(None for _ in out), out_nbytes=tuple(out), zero_fill=False, assign_target=None)
    return Plan(calls=(call,), buffers=(), sinks=(), positions=0)


def test_calls_of_many_sizes_hold_what_the_largest_needs():
    dev = device()
    sizes = [(3 << 20) * n for n in [5, 1, 9, 2, 30, 17, 31, 29, 8, 64, 63]]
    plans = [plan(dev, n) for n in sizes]
    for _ in range(4):
        for p in plans:
            dev.run(p, {})
    assert dev.api.most <= max(sizes) * 9 // 8 + len(sizes)
    assert len(large(dev)) == 1


def test_sizes_that_creep_up_drop_few_lists():
    dev = device()
    plans = [plan(dev, (1 << 24) + 4096 * n) for n in range(64)]
    for _ in range(3):
        for p in plans:
            dev.run(p, {})
    assert sum(e[1] is not None for e in dev.replays.values()) == 64 and len(large(dev)) == 1
    assert len(set(dev.lib.named)) == 1


def test_a_list_names_a_workspace_that_stays_its_own_until_it_is_dropped():
    dev = device()
    small, large = plan(dev, 1 << 21), plan(dev, 1 << 25)
    for _ in range(3):
        dev.run(small, {})
    first = dev._workspace.ptr
    assert dev.lib.named == [first] and first in dev.api.live
    dev.replays[id(small)][1].graphs[b"k"] = ctypes.c_void_p(0x99)
    dev.run(large, {})  # a larger one: the list that names the first is dropped with its graphs, and the first given back
    assert dev.lib.freed == [0x99] and id(small) not in dev.replays and first not in dev.api.live
    for _ in range(3):
        dev.run(small, {})
    assert dev.lib.named == [first, dev._workspace.ptr] and dev._workspace.ptr in dev.api.live


def test_a_recording_that_outgrows_its_first_workspace_keeps_both():
    dev = device()
    calls = plan(dev, 1 << 21).calls + plan(dev, 1 << 25).calls
    both = Plan(calls=calls, buffers=(), sinks=(), positions=0)
    dev.run(both, {})
    dev._workspace = None  # let go between the first run and the one that records
    dev.run(both, {})
    prog = dev.replays[id(both)][1]
    assert len(prog.workspaces) == 2 and all(w.ptr in dev.api.live for w in prog.workspaces)
    dev.run(both, {})
    assert dev.lib.named == [prog.workspaces[0].ptr]


def test_trim_gives_back_a_workspace_that_no_list_names():
    dev = device()
    p = plan(dev, 1 << 22)
    dev.run(p, {})
    dev.trim()
    assert dev._workspace is None and not dev.api.live
    for _ in range(2):
        dev.run(p, {})
    dev.trim()  # recorded now: the list's launches name it
    assert dev._workspace.ptr in dev.api.live
    dev._drop_replay(id(p))
    dev.trim()
    assert dev._workspace is None and not dev.api.live


def test_an_allocation_that_fails_takes_the_workspace_back():
    dev = device(room=(1 << 25) + (1 << 20))
    p = plan(dev, 1 << 24)
    for _ in range(3):
        dev.run(p, {})
    buf = dev._alloc((1 << 25) - 1)  # fits only without the workspace
    assert dev._workspace is None and list(dev.api.live) == [buf.ptr] and id(p) not in dev.replays
    with pytest.raises(RuntimeError, match="allocating"):
        dev._alloc(1 << 25)
    del buf
    for _ in range(3):
        dev.run(p, {})
    assert dev.lib.named[-1] == dev._workspace.ptr


def test_a_list_that_is_being_replayed_is_not_dropped():
    """Its arena's allocation fails until the workspace is let go, which this list names: it keeps both itself and the bytes."""
    dev = device(room=(1 << 24) + (1 << 22))
    p, other = plan(dev, 1 << 24, out=(1 << 21,)), plan(dev, 1 << 24)
    for _ in range(2):
        dev.run(p, {})
        dev.run(other, {})
    prog, ws = dev.replays[id(p)][1], dev._workspace.ptr
    blocked = dev._alloc(3 << 20)
    with pytest.raises(RuntimeError, match="allocating"):
        dev.run(p, {})
    assert dev.replays[id(p)][1] is prog and prog.workspaces[0].ptr == ws and ws in dev.api.live
    assert id(other) not in dev.replays
    del blocked
    dev.run(p, {})
    assert dev.lib.named[-1] == ws


def test_no_bytes_take_no_buffer():
    dev = device()
    p = plan(dev, 0)
    for _ in range(3):
        dev.run(p, {})
    assert not large(dev) and dev._workspace is None
