"""The head's cross entropy without a GPU: the form composed from limn's primitives against the definition in float64, its
gradients against differences, and every refusal."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from limn_amd.hip import runtime
from limn_amd.seam import Tensor, float32, float64, grad, int32, set_device
from limn_amd.xent import linear_cross_entropy
from oracle.attend import within, xent


@pytest.fixture(autouse=True)
def _numpy():
    set_device("numpy")


def draw(rows=6, width=5, vocab=11, seed=0):
    rng = np.random.default_rng(seed)
    targets = rng.integers(0, vocab, rows).astype(np.int32)
    return rng.standard_normal((rows, width)), rng.standard_normal((vocab, width)), targets


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("left_out", [(), (0, 3), (0, 1, 2, 3, 4, 5)])
def test_composed_matches_the_definition(reduction, left_out):
    x, w, targets = draw()
    targets[list(left_out)] = [-1, 11, -100, 2**31 - 1, -(2**31), 12][: len(left_out)]
    tx, tw = Tensor(x.reshape(2, 3, 5), dtype=float64, requires_grad=True), Tensor(w, dtype=float64, requires_grad=True)
    loss = linear_cross_entropy(tx, tw, Tensor(targets.reshape(2, 3), dtype=int32), reduction)
    live = max(1, 6 - len(left_out))
    weights = np.linspace(0.5, 1.5, 6) if reduction == "none" else np.full(6, 1.0 / live if reduction == "mean" else 1.0)
    want = xent(x, w, targets, weights)
    if reduction == "none":
        within(loss.numpy(), want["loss"][0].reshape(2, 3), 1e-12)
        loss = (loss * Tensor(weights.reshape(2, 3), dtype=float64)).sum()
    else:
        within(loss.numpy(), (want["loss"][0] * weights).sum(), 1e-12)
    dx, dw = grad(loss, [tx, tw])
    within(dx.numpy(), want["dx"][0].reshape(2, 3, 5), 1e-12)
    within(dw.numpy(), want["dw"][0], 1e-12)


def test_the_definitions_gradients_are_its_differences():
    x, w, targets = draw()
    targets[2] = -1
    g = np.linspace(0.5, 1.5, 6)
    want = xent(x, w, targets, g)
    step = 1e-5
    for name, k in (("dx", 0), ("dw", 1)):
        for at in np.ndindex(*(x, w)[k].shape):
            ends = []
            for way in (1, -1):
                moved = [x.copy(), w.copy()]
                moved[k][at] += way * step
                ends.append((xent(*moved, targets)["loss"][0] * g).sum())
            assert abs((ends[0] - ends[1]) / (2 * step) - want[name][0][at]) < 1e-8  # step^2 / 6 times a third derivative below 100


@pytest.mark.parametrize(
    "x,w,targets,reduction,message",
    [
        ((3, 4), (5, 6), (3,), "mean", "widths"),
        ((3, 4), (4,), (3,), "mean", "vocab, width"),
        ((3, 4), (5, 4), (4,), "mean", "targets"),
        ((2, 3, 4), (5, 4), (6,), "mean", "targets"),
        ((3, 4), (5, 4), (3,), "average", "reduction"),
    ],
)
def test_refusals(x, w, targets, reduction, message):
    with pytest.raises(ValueError, match=message):
        linear_cross_entropy(Tensor.zeros(x), Tensor.zeros(w), Tensor(np.zeros(targets), dtype=int32), reduction)


def test_types_are_refused():
    x, w = Tensor.zeros((3, 4)), Tensor.zeros((5, 4))
    with pytest.raises(ValueError, match="targets"):
        linear_cross_entropy(x, w, Tensor.zeros((3,), dtype=float32))
    with pytest.raises(ValueError, match="float"):
        linear_cross_entropy(x.int(), w, Tensor.zeros((3,), dtype=int32))


FAKE = ctypes.c_void_p(0x1000)  # never read: every call below fails its checks first


def call(backward=False, x=FAKE, targets=FAKE, workspace=FAKE, room=1 << 40, **kw):
    a = dict(dtype=1, rows=4, width=8, vocab=16)
    a.update(kw)
    lib = runtime.kernels()
    if backward:
        return lib.limn_hip_xent_bwd(x, FAKE, targets, FAKE, FAKE, FAKE, FAKE, a["dtype"], a["rows"], a["width"], a["vocab"], workspace, room, None)
    return lib.limn_hip_xent_fwd(x, FAKE, targets, FAKE, FAKE, a["dtype"], a["rows"], a["width"], a["vocab"], workspace, room, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize(
    "kw,code,message",
    [
        (dict(dtype=0), 2, "float32, float16 or bfloat16"),
        (dict(rows=0), 1, "positive"),
        (dict(vocab=-3), 1, "positive"),
        (dict(vocab=1 << 32), 2, "out of range"),
        (dict(rows=1 << 22, width=1 << 12), 2, "out of range"),
        (dict(x=None), 1, "null"),
        (dict(x=ctypes.c_void_p(0x1002)), 1, "aligned"),
        (dict(targets=ctypes.c_void_p(0x1002)), 1, "aligned"),
        (dict(room=16), 1, "workspace"),
        (dict(workspace=None), 1, "workspace"),
        (dict(workspace=ctypes.c_void_p(0x1004)), 1, "workspace"),
    ],
)
def test_the_abi_refuses_with_a_reason(backward, kw, code, message):
    assert call(backward, **kw) == code
    assert message in runtime.kernels().limn_hip_last_error().decode()
