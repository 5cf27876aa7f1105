"""The same tensor as several inputs of one operator on the MI355X, run call by call, recorded and replayed."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, storage_values
from limn_amd.attend import attend
from limn_amd.seam import Tensor, float32, grad, int32, realize, use_device
from limn_amd.xent import linear_cross_entropy
from oracle.attend import attend as definition
from oracle.attend import within, xent
from oracle.numpy_device import NumpyDevice

pytestmark = pytest.mark.gpu


def drawn(seed, *shapes, dtype="bfloat16"):
    rng = np.random.default_rng(seed)
    return [storage_values(rng.standard_normal(s).astype(np.float32), DTYPES[dtype]) for s in shapes]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hd", [24, 64, 128])
def test_attend(hipdev, dtype, hd):
    use_device(hipdev)
    x, y, do = drawn(hd, (2, 2, 150, hd), (2, 2, 150, hd), (2, 2, 150, hd), dtype=dtype)
    t = DTYPES[dtype]
    some = np.array([70, 150], np.int32)
    for _ in range(3):
        tx, ty, td = Tensor(x, dtype=t, requires_grad=True), Tensor(y, dtype=t, requires_grad=True), Tensor(do, dtype=t)
        out = attend(tx, tx, tx, causal=True)
        got = [out, *grad((out * td).sum(), [tx])]
        realize(*got)
        want = definition(x, x, x, dout=do, causal=True, dtype=dtype)
        within(got[0].numpy(), *want["out"])
        half = 2.0**-24 if dtype == "float32" else 2.0**-8
        total = sum(want[n][0] for n in ("dq", "dk", "dv"))
        # two additions round their results, of the shares or of two of them
        within(got[1].numpy(), total, sum(want[n][1] for n in ("dq", "dk", "dv")) + 2 * half * sum(np.abs(want[n][0]) for n in ("dq", "dk", "dv")))
        given = Tensor(some, dtype=int32)
        out = attend(ty, tx, tx, causal=True, prefix=given, lengths=given)
        got = [out, *grad((out * td).sum(), [ty])]
        realize(*got)
        want = definition(y, x, x, dout=do, causal=True, dtype=dtype, prefix=some, lengths=some)
        within(got[0].numpy(), *want["out"])
        within(got[1].numpy(), *want["dq"])


def test_a_cotangent_that_is_the_output(hipdev):
    """The gradient of out times itself held fast: the backward's dout is out's own buffer."""
    use_device(hipdev)
    q, k, v = drawn(3, *[(1, 2, 90, 64)] * 3)
    tq, tk, tv = (Tensor(a, dtype=DTYPES["bfloat16"], requires_grad=True) for a in (q, k, v))
    out = attend(tq, tk, tv, causal=True)
    got = [out, *grad((out * out.detach()).sum(), [tq, tk, tv])]
    realize(*got)
    do = got[0].numpy()
    want = definition(q, k, v, dout=do, causal=True, dtype="bfloat16")
    for name, x in zip(("dq", "dk", "dv"), got[1:]):
        within(x.numpy(), *want[name], name)


def test_a_head_that_is_its_rows(hipdev):
    use_device(hipdev)
    (x,) = drawn(4, (70, 64), dtype="float32")
    targets = np.arange(70, dtype=np.int32)[::-1].copy()
    tx = Tensor(x, dtype=float32, requires_grad=True)
    loss = linear_cross_entropy(tx, tx, Tensor(targets, dtype=int32), "sum")
    (g,) = grad(loss, [tx])
    realize(loss, g)
    want = xent(x, x, targets, np.ones(70))
    value = want["dx"][0] + want["dw"][0]
    within(g.numpy(), value, want["dx"][1] + want["dw"][1] + 2.0**-24 * np.abs(value))


@pytest.mark.parametrize("causal", [True, False])
def test_attention(hipdev, causal):
    """The framework's own attention, its paired backward among it."""
    x, y, do = drawn(5, *[(2, 3, 256, 128)] * 3)
    results = []
    for dev in (hipdev, NumpyDevice()):
        use_device(dev)
        for _ in range(3 if dev is hipdev else 1):
            tx, ty = (Tensor(a, dtype=DTYPES["bfloat16"], requires_grad=True) for a in (x, y))
            one, two = tx.attention(tx, tx, causal=causal), ty.attention(tx, tx, causal=causal)
            got = [one, two, *grad(((one + two) * Tensor(do, dtype=DTYPES["bfloat16"])).sum(), [tx, ty])]
            realize(*got)
        results.append([t.numpy() for t in got])
    for a, b in zip(*results):
        # as the attention tests compare the two devices: 2^-8 a rounding, a few of them in a row
        assert np.abs(a - b).max() <= 2e-2 * np.abs(b).max()
