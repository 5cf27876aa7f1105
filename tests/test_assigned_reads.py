"""Plans that read a tensor they have assigned: the readers of the new value launch behind the nest that makes it, those of the old
one read the buffer, which the executor changes at the end alone. Checked on the planner's own launch order, without a GPU."""

from __future__ import annotations

import numpy as np
import pytest

from limn_amd.paged import attend_paged
from limn_amd.seam import Op, Tensor, bfloat16, float32, lower_all, schedule, set_device, topological
from serving import paged_inputs
from test_emit_plan import emit, lowered
from test_serving import tensors

rng = np.random.default_rng(3)


@pytest.fixture(autouse=True)
def on_numpy():
    set_device("numpy")


def on(*shape, dtype=float32):
    return Tensor(rng.standard_normal(shape).astype(np.float32), dtype=dtype).realize()


def ordered(sinks) -> emit.Program:
    """The plan of these sinks: every nest's inputs are made in an earlier launch, or in an earlier member of its row program."""
    nests, kept = lowered(sinks)
    custom = {emit.realized(src) for n in topological([t.node for t in sinks]) if n.op is Op.CUSTOM for src in n.srcs}
    prog = emit.plan_program(nests, kept, custom)
    makers = {n.kernel.ast: k for k, n in enumerate(nests)}
    rows = {key for key, (run, launch) in prog.merged.items() if "_rows_" in launch.name}
    when, clock = {}, 0
    for k in range(len(nests)):
        role = prog.role(k)
        for members in ([prog.merged[key][0] for key in prog.launches_from(k)] if role == "merged" else [] if role in ("deferred", "inlined", "stash") else [[k]]):
            clock += 1
            when.update({c: clock for c in members})

    def made_at(node, reader, place):
        p = makers.get(node)
        if p is None:
            return
        if p in prog.inlined.producers:
            for src in nests[p].kernel.inputs:
                made_at(src, reader, place)
        elif p in prog.pairs:  # a contraction launched by its epilogue
            assert prog.pairs[p] == reader
            for src in nests[p].kernel.inputs:
                made_at(src, reader, place)
        else:
            together = any(p in prog.merged[key][0] and reader in prog.merged[key][0] and p < reader for key in rows)
            assert when[p] < place or together, f"{nests[reader].name} reads {nests[p].name} before it is there"

    for c, nest in enumerate(nests):
        assert not (nest.kernel.ast.op is Op.ASSIGN and c in prog.inlined.producers), f"{nest.name} is committed, but nothing stores it"
        if c in when:
            for node in nest.kernel.inputs:
                made_at(node, c, when[c])
    return prog


@pytest.mark.parametrize("dtype", ["float32", "float64", "bfloat16"])
@pytest.mark.parametrize("case", [dict(counts=(3, 1, 5), lengths=(7, 1, 5), heads=4, kv_heads=2, spare=2, rows_before=1), dict(counts=(2,), lengths=(5,), page=1)], ids=str)
def test_attend_paged_composed(case, dtype):
    x = paged_inputs(4, **{**case, "dtype": "float32" if dtype == "float64" else dtype})
    t = tensors(x, dtype)
    ordered([attend_paged(**t)])


def test_a_small_nest_and_its_readers():
    a, b = on(64, 48), on(64, 48)
    a.assign(a.detach() * 0.5 + b)
    ordered([a, a.detach().transpose() + 1.0, a.detach().sum(axis=0), (a.detach() * b).exp()])


def test_a_reader_of_the_old_value():
    a, b = on(16), on(16)
    old = Tensor.from_node(a.node)
    a.assign(b * 2.0 + 1.0)
    kept = ordered([old * 3.0 + on(5, 16), a.detach().reshape(16, 1).expand(16, 4).sum(axis=1)])
    assert kept is not None


def test_an_assign_that_is_no_sink_is_stored():
    a, b = on(8, 1), on(8, 32)
    old = Tensor.from_node(a.node)
    a.assign(b.sum(axis=1, keepdim=True) * 0.5)
    ordered([b - a.detach(), b * old])


def test_row_programs():
    x, mean = on(128, 256), on(128, 1)
    old = Tensor.from_node(mean.node)
    mean.assign(mean.detach() * 0.9 + x.sum(axis=1, keepdim=True) * (0.1 / 256))
    ordered([mean, x - mean.detach(), (x * old).sum(axis=1)])


def test_a_bias_that_is_assigned_from_float32():
    x, w, b, master = on(64, 64, dtype=bfloat16), on(64, 48, dtype=bfloat16), on(48, dtype=bfloat16), on(48)
    old = Tensor.from_node(b.node)
    b.assign(master.cast(bfloat16))
    prog = ordered([x @ w + old])
    assert all(terms[2] is None for terms in prog.addends.values())
