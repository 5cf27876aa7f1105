"""CUSTOM nodes that name one src twice, on the hip device without a GPU: a plan's call has each distinct src once, and the
runners take one buffer a src."""

from __future__ import annotations

import numpy as np
import pytest

from limn_amd.hip.device import SDPA, SDPA_BWD_KV, SDPA_BWD_Q, by_source
from limn_amd.seam import Node, Op, custom, float32, schedule


def buffers(n):
    return [Node(Op.BUFFER, (), float32, (4, 8), np.zeros(128, np.uint8)) for _ in range(n)]


@pytest.mark.parametrize("which", [(0, 1, 2), (0, 0, 0), (0, 1, 1), (0, 1, 0, 2), (0, 1, 2, 3, 3), (0, 1, 1, 2, 0, 3)])
def test_a_runner_gets_one_buffer_a_src(which):
    nodes = buffers(4)
    (node,) = custom("any", tuple(nodes[i] for i in which), (), ((float32, (4, 8)),))
    (kernel,) = schedule([node])
    seen = []
    run = by_source(lambda n: lambda inputs, outs: seen.append((inputs, outs)))(node)
    run([n.arg for n in kernel.inputs], ["out"])
    (inputs, outs), = seen
    assert outs == ["out"] and len(inputs) == len(which)
    assert all(b is nodes[i].arg for b, i in zip(inputs, which))


def test_paired_backwards_keep_their_repeats():
    def build(node):
        run = lambda inputs, outs: None  # noqa: E731
        run.sdpa_pair = (node.arg.name, "key", lambda: lambda inputs, outs: outs.append(inputs))
        return run

    nodes = buffers(5)
    srcs = tuple(nodes[i] for i in (0, 1, 1, 2, 3, 4))
    first, second = (by_source(build)(custom(name, srcs, (), ((float32, (4, 8)),))[0]).sdpa_pair for name in (SDPA_BWD_Q, SDPA_BWD_KV))
    assert first[1] == second[1]
    outs = []
    first[2]()([n.arg for n in nodes], outs)
    assert [any(b is n.arg for n in nodes) for b in outs[0]] == [True] * 6 and outs[0][1] is outs[0][2]
    plain = by_source(build)(custom(SDPA, tuple(nodes), (), ((float32, (4, 8)),))[0])
    assert plain.sdpa_pair[1] == "key"
