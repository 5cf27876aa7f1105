"""Batches that read a tensor they have assigned, on the MI355X: the new value through the assigned tensor, the old one through the
buffer, again and again with other numbers (memory of an earlier run holds other ones), against the numpy oracle."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, download
from limn_amd.paged import attend_paged
from limn_amd.sampling import sample
from limn_amd.seam import Tensor, capture, realize, set_device, use_device
from oracle.attend import within
from oracle.serving import paged
from oracle.serving import sample as sample_oracle
from serving import paged_inputs
from test_paged_gpu import tensors

pytestmark = pytest.mark.gpu


def several(a, b):
    a.assign(a.detach() * 0.5 + b)
    return [a.detach().transpose() + 1.0, a.detach().sum(axis=0), (a.detach() * b).exp()]


def old_and_new(a, b):
    old = Tensor.from_node(a.node)
    a.assign(b * 2.0 + 1.0)
    return [old * 3.0 + b, a.detach().reshape(64, 48, 1).expand(64, 48, 4).sum(axis=2)]


def no_sink(a, b):
    old = Tensor.from_node(a.node)
    a.assign(b.sum(axis=1, keepdim=True) * (0.5 / 48) + b)
    return [b - a.detach(), b * old]


def running(a, b):
    old = Tensor.from_node(a.node)
    a.assign(a.detach() * 0.9 + b.sum(axis=1, keepdim=True) * (0.1 / 48))
    return [b - a.detach(), (b * old).sum(axis=1)]


@pytest.mark.parametrize("step", [several, old_and_new, no_sink, running])
@pytest.mark.parametrize("captured", [False, True])
def test_new_and_old_values(hipdev, step, captured):
    got = {}
    for name in ("numpy", "hip"):
        set_device("numpy") if name == "numpy" else use_device(hipdev)
        rng = np.random.default_rng(1)
        a = Tensor(rng.standard_normal((64, 48)).astype(np.float32)).realize()

        def run(b):
            out = step(a, b)
            realize(*out)
            return out

        call = capture(run) if captured and name == "hip" else run
        got[name] = []
        for _ in range(6):
            out = call(Tensor(rng.standard_normal((64, 48)).astype(np.float32)).realize())
            got[name] += [t.numpy().copy() for t in out] + [a.numpy().copy()]
            assert (Tensor(np.ones(1000)) * 3.0).sum().item() == 3000.0
    for k, (x, y) in enumerate(zip(got["hip"], got["numpy"])):
        # sums of 192 terms below 8 at most, in two orders; an exponential's argument below 8, by as much of it
        np.testing.assert_allclose(x, y, rtol=192 * 2.0**-24, atol=192 * 8 * 2.0**-24, err_msg=str(k))


@pytest.mark.parametrize("dtype,hd", [("float32", 260), ("bfloat16", 260), ("float64", 16)])
def test_attend_paged_composed(hipdev, dtype, hd):
    """Several steps over one cache, each with other new tokens: what is written is what the queries see."""
    use_device(hipdev)
    x = paged_inputs(4, dtype="float32" if dtype == "float64" else dtype, counts=(3, 1, 5), lengths=(7, 1, 5), heads=4, kv_heads=2, hd=hd, spare=2, rows_before=1)
    for turn in range(4):
        fresh = paged_inputs(5 + turn, dtype="float32" if dtype == "float64" else dtype, counts=(3, 1, 5), lengths=(7, 1, 5), heads=4, kv_heads=2, hd=hd, spare=2, rows_before=1)
        x.update({n: fresh[n] for n in "qkv"})
        t = tensors(hipdev, x, dtype)
        (out,) = realize(attend_paged(**t))
        (want, bound), keys, values = paged(**x, dtype="float32" if dtype == "float64" else dtype)
        within(download(hipdev, out, DTYPES[dtype], x["q"].shape), want, bound, f"turn {turn}")
        np.testing.assert_array_equal(t["key_pages"].numpy(), keys)
        np.testing.assert_array_equal(t["value_pages"].numpy(), values)
        x["key_pages"], x["value_pages"] = keys, values


@pytest.mark.parametrize("captured", [False, True])
def test_calls_of_kernels_read_what_was_assigned(hipdev, captured):
    """Lengths that a step moves on itself, and numbers that it halves, in one batch with the calls that take them."""
    use_device(hipdev)
    x = paged_inputs(6, dtype="bfloat16", counts=(1, 1, 1), lengths=(20, 3, 9), heads=4, kv_heads=2, hd=64, page=8, table_pages=4)
    x["table"][:] = np.arange(12).reshape(3, 4)
    t = tensors(hipdev, x, "bfloat16")
    logits = np.random.default_rng(7).standard_normal((3, 500)).astype(np.float32)
    u, z = Tensor(np.array([0.9, 0.7, 0.99], np.float32)).realize(), Tensor(logits).realize()

    def step():
        t["lengths"].assign(t["lengths"].detach() + 1)
        u.assign(u.detach() * 0.5)
        out = attend_paged(**t)
        tokens, logs = sample(z, u.detach())
        realize(out, tokens, logs)
        return out, tokens, logs

    run, share = capture(step) if captured else step, np.array([0.9, 0.7, 0.99], np.float32)
    for turn in range(6):
        out, tokens, logs = run()
        x["lengths"], share = x["lengths"] + 1, share * np.float32(0.5)
        (want, bound), x["key_pages"], x["value_pages"] = paged(**x, dtype="bfloat16")
        within(out.numpy(), want, bound, f"turn {turn}")
        drawn, (lp, b) = sample_oracle(logits, share)
        np.testing.assert_array_equal(tokens.numpy(), drawn)
        within(logs.numpy(), lp, b, "logprob")
        np.testing.assert_array_equal(t["lengths"].numpy(), x["lengths"])
        assert (Tensor(np.ones(1000)) * 3.0).sum().item() == 3000.0
