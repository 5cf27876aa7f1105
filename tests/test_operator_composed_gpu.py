"""attend and linear_cross_entropy where the hip device runs the form composed of primitives: head dims past 256, float64, and
gradients of gradients."""

from __future__ import annotations

import numpy as np
import pytest

from limn_amd.attend import attend
from limn_amd.seam import Tensor, float32, float64, grad, int32, realize, set_device, use_device
from limn_amd.xent import linear_cross_entropy
from oracle.attend import attend as definition
from oracle.attend import within, xent
from test_operator_gradients import CALLS, orders

pytestmark = pytest.mark.gpu


def drawn(hd, seed):
    rng = np.random.default_rng(seed)
    q, k, v, do = (rng.standard_normal(s) for s in ((2, 4, 9, hd), (2, 2, 13, hd), (2, 2, 13, 7), (2, 4, 9, 7)))
    rules = dict(slopes=(0.5 ** np.arange(1, 5)).astype(np.float32), lengths=np.array([13, 9], np.int32), prefix=np.array([2, 0], np.int32),
                 documents=rng.integers(-1, 2, (2, 13)).astype(np.int32))
    return q, k, v, do, rules


@pytest.mark.parametrize("dtype,hd", [(float64, 6), (float32, 272)])
@pytest.mark.parametrize("softcap", [0.0, 1.0, 50.0, 1e6, 1e30])
def test_attend(hipdev, dtype, hd, softcap):
    use_device(hipdev)
    q, k, v, do, rules = drawn(hd, hd)
    if dtype == float32:
        q, k, v, do = (x.astype(np.float32) for x in (q, k, v, do))
    given = {n: Tensor(x, dtype=float32 if n == "slopes" else int32) for n, x in rules.items()}
    tq, tk, tv = (Tensor(x, dtype=dtype, requires_grad=True) for x in (q, k, v))
    out = attend(tq, tk, tv, causal=True, softcap=softcap, **given)
    got = [out, *grad((out * Tensor(do, dtype=dtype)).sum(), [tq, tk, tv])]
    realize(*got)
    want = definition(q, k, v, dout=do, causal=True, softcap=softcap, **rules)
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        value, bound = want[name]
        within(t.numpy(), value, bound if dtype == float32 else 1e-12, name)


def test_a_head_in_float64(hipdev):
    use_device(hipdev)
    rng = np.random.default_rng(3)
    x, w, targets = rng.standard_normal((6, 5)), rng.standard_normal((11, 5)), np.array([2, -1, 6, 11, 0, 3], np.int32)
    g = np.full(6, 0.25)
    want = xent(x, w, targets, g)
    x = x.copy()
    x[[1, 3]] = np.nan
    tx, tw = Tensor(x, dtype=float64, requires_grad=True), Tensor(w, dtype=float64, requires_grad=True)
    loss = linear_cross_entropy(tx, tw, Tensor(targets, dtype=int32))
    got = [loss, *grad(loss, [tx, tw])]
    realize(*got)
    within(got[0].numpy(), (want["loss"][0] * g).sum(), 1e-12)
    within(got[1].numpy(), want["dx"][0], 1e-12)
    within(got[2].numpy(), want["dw"][0], 1e-12)


@pytest.mark.parametrize("name", CALLS)
def test_gradients_of_gradients(hipdev, name):
    rng = np.random.default_rng(len(name))
    x, w = (rng.standard_normal((1, 2, 5, 4)).astype(np.float32) for _ in range(2))
    set_device("numpy")
    want = orders(CALLS[name], x, w, float64)
    use_device(hipdev)
    for i, (a, b) in enumerate(zip(orders(CALLS[name], x, w, float32), want)):
        assert np.abs(a - b).max() <= 2.0**-14 * np.abs(b).max(), (i, np.abs(a - b).max(), np.abs(b).max())
