"""Gradients through attend's and linear_cross_entropy's CUSTOM nodes where inputs share tensors, on the numpy device with the
definitions registered as its kernels: the same as through the form composed of primitives, to the second order."""

from __future__ import annotations

import numpy as np
import pytest

from limn_amd.attend import attend
from limn_amd.seam import Tensor, active_device, float32, float64, grad, int32, set_device
from limn_amd.xent import linear_cross_entropy
from oracle import attend as oracle


def _attend_kernel(name, srcs, node):
    causal, scale, softcap, given = node.arg.params
    rules = iter(srcs[3 : 3 + sum(given)])
    kw = {n: next(rules) for n, on in zip(("slopes", "documents", "prefix", "lengths"), given) if on}
    dout = srcs[-1] if name == "attend_bwd" else None
    got = oracle.attend(*srcs[:3], causal=causal, scale=scale, softcap=softcap, dout=dout, **kw)
    return tuple(got[n][0] for n in ("dq", "dk", "dv")) if dout is not None else (got["out"][0], got["lse"][0][..., None])


def _xent_kernel(name, srcs, node):
    x, w, targets = srcs[:3]
    got = oracle.xent(x, w, targets, g=srcs[4] if name == "xent_bwd" else None)
    return tuple(got[n][0] for n in (("dx", "dw") if name == "xent_bwd" else ("loss", "lse")))


KERNELS = dict(attend_fwd=_attend_kernel, attend_bwd=_attend_kernel, xent_fwd=_xent_kernel, xent_bwd=_xent_kernel)


def orders(call, x, w, dtype):
    """The value of `call`, the first gradients of its square's sum and the second of theirs, at x and w."""
    tx, tw = (Tensor(a, dtype=dtype, requires_grad=True) for a in (x, w))
    plain = grad((call(tx, tw) * call(tx, tw)).sum(), [tx, tw])
    out = call(tx, tw)
    first = grad((out * out).sum(), [tx, tw], create_graph=True)
    second = grad((first[0] * first[0]).sum() + (first[1] * first[1]).sum(), [tx, tw])
    return [t.numpy() for t in (out, *plain, *first, *second)]


def head(rows, weight, reduction="mean"):
    return linear_cross_entropy(rows, weight, Tensor(np.array([3, 0, -1, 4, 1], np.int32), dtype=int32), reduction=reduction)


CALLS = {
    "siblings": lambda x, w: attend(x * 1.5, x * 1.0 + w, w * 2.0, causal=True, softcap=3.0),
    "keys from both": lambda x, w: attend(x, x * 1.0 + w, w, causal=True, softcap=3.0),
    "one tensor thrice": lambda x, w: attend(x, x, x, causal=True) * w,
    "keys from the queries": lambda x, w: attend(x, x * w, (x * w) * 0.5, causal=True),
    "values from the keys": lambda x, w: attend(w, x, x + 1.0, scale=0.25),
    "a head from its rows": lambda x, w: head(x[0, 0], x[0, 0] * w[0, 0], reduction="none"),
    "a head that is its rows": lambda x, w: head(x[0, 0] * 2.0, w[0, 0]) + head(w[0, 0], w[0, 0]),
}


@pytest.mark.parametrize("name", CALLS)
def test_inputs_that_share_tensors(name):
    set_device("numpy")
    rng = np.random.default_rng(len(name))
    x, w = (rng.standard_normal((1, 2, 5, 4)).astype(np.float32) for _ in range(2))
    want = orders(CALLS[name], x, w, float64)  # float64 takes the composed form
    dev = active_device()
    dev.custom.update(KERNELS)
    got = orders(CALLS[name], x, w, float32)
    for i, (a, b) in enumerate(zip(got, want)):
        # chains of some hundred float32 roundings: a thousand half steps of the largest; a share counted twice is its own size
        assert np.abs(a - b).max() <= 2.0**-14 * np.abs(b).max(), (i, np.abs(a - b).max(), np.abs(b).max())


@pytest.mark.parametrize("name", ["keys from both", "a head from its rows"])
def test_a_device_with_the_forward_kernels_alone(name):
    set_device("numpy")
    rng = np.random.default_rng(7)
    x, w = (rng.standard_normal((1, 2, 5, 4)).astype(np.float32) for _ in range(2))
    want = orders(CALLS[name], x, w, float64)
    active_device().custom.update({n: f for n, f in KERNELS.items() if n.endswith("fwd")})
    for a, b in zip(orders(CALLS[name], x, w, float32), want):
        assert np.abs(a - b).max() <= 2.0**-14 * np.abs(b).max()
