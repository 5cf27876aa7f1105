"""The head's cross entropy on the MI355X: limn_amd.xent on the hip device and the C ABI, against the definition in float64 within
the bounds on rounding that oracle/attend.py derives."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, storage_values, upload
from limn_amd.dtypes import ABI_CODE, from_storage
from limn_amd.hip import runtime
from limn_amd.seam import Tensor, capture, float32, grad, int32, realize, use_device
from limn_amd.xent import linear_cross_entropy
from oracle.attend import within, xent

pytestmark = pytest.mark.gpu


def draw(seed, dtype, rows, width, vocab, left_out=0.0, std=2.0):
    rng = np.random.default_rng(seed)
    x = storage_values(rng.standard_normal((rows, width)).astype(np.float32), DTYPES[dtype])
    w = storage_values((rng.standard_normal((vocab, width)) * std * width**-0.5).astype(np.float32), DTYPES[dtype])
    targets = rng.integers(0, vocab, rows).astype(np.int32)
    if left_out:
        out = rng.random(rows) < left_out
        targets[out] = rng.choice([-1, -100, vocab, 2**31 - 1, -(2**31)], out.sum())
    return rng, x, w, targets


def called(dev, x, w, targets, g, dtype, guard=256):
    """limn_hip_xent_fwd and limn_hip_xent_bwd on buffers of their own, with guard bytes behind every output that must stay."""
    t = DTYPES[dtype]
    (rows, width), vocab = x.shape, w.shape[0]
    code = ABI_CODE[t]
    ins = [upload(dev, x, t).arg, upload(dev, w, t).arg, upload(dev, targets, int32).arg]
    grads = upload(dev, g, float32).arg
    sizes = dict(loss=(rows * 4, float32, (rows,)), lse=(rows * 4, float32, (rows,)), dx=(x.size * t.itemsize, t, x.shape), dw=(w.size * t.itemsize, t, w.shape))
    outs = {n: dev._alloc(nb + guard) for n, (nb, _, _) in sizes.items()}
    for b in outs.values():
        dev.copyin(b, np.full(b.nbytes, 0xAB, np.uint8))
    for backward in (0, 1):
        need = dev.lib.limn_hip_xent_workspace(code, rows, width, vocab, backward)
        ws = dev._alloc(need)
        dev.copyin(ws, np.full(need, 0xFF, np.uint8))  # NaN, should any of it be read before it is written
        if backward:
            status = dev.lib.limn_hip_xent_bwd(*(b.ptr for b in ins), outs["lse"].ptr, grads.ptr, outs["dx"].ptr, outs["dw"].ptr, code, rows, width, vocab, ws.ptr, need, None)
        else:
            status = dev.lib.limn_hip_xent_fwd(*(b.ptr for b in ins), outs["loss"].ptr, outs["lse"].ptr, code, rows, width, vocab, ws.ptr, need, None)
        runtime.check_limn(status)
        dev.finish()
    got = {}
    for n, (nb, kind, shape) in sizes.items():
        raw = dev.copyout(outs[n])
        assert (raw[nb:] == 0xAB).all(), n
        got[n] = from_storage(raw[:nb], kind, shape)
    return got


def check(dev, x, w, targets, g, dtype):
    got = called(dev, x, w, targets, g, dtype)
    want = xent(x, w, targets, g, dtype)
    for n, y in got.items():
        within(y, *want[n], f"{n} {dtype}")
    return got


TYPES = ["float32", "bfloat16", "float16"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width,vocab", [(1, 1, 1), (1, 64, 2), (3, 8, 17), (33, 24, 100), (64, 64, 256), (130, 72, 257), (129, 100, 1000), (257, 128, 511), (48, 512, 5003), (300, 33, 129),
                                              (1030, 64, 640), (512, 768, 300), (5, 200, 9001)])
def test_sizes(hipdev, dtype, rows, width, vocab):
    rng, x, w, targets = draw(rows + width + vocab, dtype, rows, width, vocab, left_out=0.3)
    check(hipdev, x, w, targets, rng.standard_normal(rows).astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_several_pieces_of_the_vocabulary(hipdev, dtype):
    """More logits than one piece's buffer holds (128 MiB)."""
    rows, width, vocab = 4100, 40, 20011
    rng, x, w, targets = draw(1, dtype, rows, width, vocab, left_out=0.2)
    check(hipdev, x, w, targets, (rng.random(rows) / rows).astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [-130, -20, -12, 8, (-20, 4)])
def test_cotangents_of_every_size(hipdev, dtype, bits):
    """A mean over many rows, a loss multiplied up, and rows of very unlike weight."""
    rng, x, w, targets = draw(11, dtype, 150, 72, 1111, left_out=0.2)
    g = rng.standard_normal(150) * (2.0**bits if isinstance(bits, int) else np.exp2(rng.integers(*bits, 150)))
    check(hipdev, x, w, targets, g.astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_cotangents_of_rows_left_out(hipdev, dtype):
    """Whatever a row without a target gets as its cotangent, the others' gradients hold their bits."""
    rng, x, w, targets = draw(12, dtype, 70, 64, 300, left_out=0.3)
    g = rng.standard_normal(70).astype(np.float32) * np.float32(2.0**-14)
    want = check(hipdev, x, w, targets, g, dtype)
    g[targets < 0] = np.resize(np.float32([np.inf, np.nan, 1e38]), (targets < 0).sum())
    got = check(hipdev, x, w, targets, g, dtype)
    for name in want:
        np.testing.assert_array_equal(got[name], want[name])


def test_float32_numbers_of_every_size(hipdev):
    """Rows scaled from 2^-120 to 2^120 and back by the weight's columns: a float32 goes to its products in parts, each of which must hold its bits."""
    rng, x, w, targets = draw(9, "float32", 100, 64, 300)
    scale = np.exp2(rng.integers(-60, 61, 64)).astype(np.float32)
    x, w = x * scale, w / scale
    check(hipdev, x, w, targets, rng.standard_normal(100).astype(np.float32), "float32")
    big = np.zeros((4, 8), np.float32)
    big[0, 0] = np.finfo(np.float32).max  # past bfloat16's largest
    w = np.zeros((5, 8), np.float32)
    w[0, 0] = 1e-38
    w[1, 1] = 1.0
    got = check(hipdev, big, w, np.array([0, 1, 2, 4], np.int32), np.ones(4, np.float32), "float32")
    # float32's largest goes whole; 1e-38 (subnormal) goes to bfloat16's least step 2^-133, so their product 3.4028235
    # is off by up to 2^128 2^-134 = 2^-6, and lse, whose slope by a score is below 1, by no more (8 steps beside that)
    assert abs(got["lse"][0] - np.log(np.exp(3.4028235) + 4)) < 2.0**-6 + 2.0**-20


@pytest.mark.parametrize("dtype", TYPES)
def test_no_row_has_a_target(hipdev, dtype):
    rng, x, w, targets = draw(2, dtype, 70, 64, 130)
    targets[:] = -1
    got = check(hipdev, x, w, targets, np.ones(70, np.float32), dtype)
    assert not got["loss"].any() and not got["dx"].any() and not got["dw"].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("width", [64, 60])
def test_infinities_and_nan_in_rows_left_out(hipdev, dtype, bad, width):
    rng, x, w, targets = draw(3, dtype, 140, width, 300)
    targets[[0, 17, 139]] = [-1, 300, -7]
    x[[0, 17, 139]] = bad
    g = rng.standard_normal(140).astype(np.float32)
    g[17] = np.nan
    got = called(hipdev, x, w, targets, g, dtype)
    clean = np.where(np.isfinite(x), x, 0.0)
    want = xent(clean, w, targets, np.where(np.isfinite(g), g, 0.0), dtype)
    for n in ("loss", "dx", "dw"):
        within(got[n], *want[n], n)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_logits(hipdev, dtype):
    rng, x, w, targets = draw(4, dtype, 100, 64, 500, std=100.0)
    check(hipdev, x, w, targets, np.ones(100, np.float32), dtype)


def test_unaligned_operands(hipdev):
    """Rows of x and w that start on 2-byte boundaries, as a view into a larger buffer has them."""
    dev, t = hipdev, DTYPES["bfloat16"]
    rng, x, w, targets = draw(5, "bfloat16", 70, 64, 200)
    at = []
    for a in (x, w):
        host = np.concatenate([np.zeros(1, np.float32), a.reshape(-1)])
        at.append(upload(dev, host, t).arg)
    where = upload(dev, targets, int32).arg
    loss, lse = dev._alloc(280), dev._alloc(280)
    need = dev.lib.limn_hip_xent_workspace(3, 70, 64, 200, 0)
    ws = dev._alloc(need)
    runtime.check_limn(dev.lib.limn_hip_xent_fwd(at[0].ptr + 2, at[1].ptr + 2, where.ptr, loss.ptr, lse.ptr, 3, 70, 64, 200, ws.ptr, need, None))
    dev.finish()
    within(dev.copyout(loss).view(np.float32), *xent(x, w, targets, dtype="bfloat16")["loss"])
    g = np.ones(70, np.float32)
    need = dev.lib.limn_hip_xent_workspace(3, 70, 64, 200, 1)
    ws, dx, dw = dev._alloc(need), dev._alloc(70 * 64 * 2), dev._alloc(200 * 64 * 2 + 2)
    cot = upload(dev, g, float32).arg
    runtime.check_limn(dev.lib.limn_hip_xent_bwd(at[0].ptr + 2, at[1].ptr + 2, where.ptr, lse.ptr, cot.ptr, dx.ptr, dw.ptr + 2, 3, 70, 64, 200, ws.ptr, need, None))
    dev.finish()
    want = xent(x, w, targets, g, "bfloat16")
    within(from_storage(dev.copyout(dx), t, (70, 64)), *want["dx"])
    within(from_storage(dev.copyout(dw)[2:], t, (200, 64)), *want["dw"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_through_the_tensor_api(hipdev, dtype, reduction):
    use_device(hipdev)
    rng, x, w, targets = draw(6, dtype, 90, 64, 333, left_out=0.2)
    tx, tw = (Tensor(a, dtype=DTYPES[dtype], requires_grad=True) for a in (x.reshape(3, 30, 64), w))
    loss = linear_cross_entropy(tx, tw, Tensor(targets.reshape(3, 30), dtype=int32), reduction)
    live = ((targets >= 0) & (targets < 333)).sum()
    g = np.full(90, 1.0 / live if reduction == "mean" else 1.0, np.float32)
    total = loss if reduction != "none" else loss.sum()
    got = [loss, *grad(total, [tx, tw])]
    realize(*got)
    want = xent(x, w, targets, g, dtype)
    value, bound = want["loss"]
    if reduction == "none":
        within(got[0].numpy(), value.reshape(3, 30), bound.reshape(3, 30))
    else:  # 90 float32 additions, then a product by a reciprocal
        within(got[0].numpy(), (value * g).sum(), ((bound + 100 * 2.0**-24 * np.abs(value)) * g).sum())
    within(got[1].numpy(), want["dx"][0].reshape(3, 30, 64), want["dx"][1].reshape(3, 30, 64) + 2.0**-22 * np.abs(want["dx"][0]).reshape(3, 30, 64))
    within(got[2].numpy(), want["dw"][0], want["dw"][1] + 2.0**-22 * np.abs(want["dw"][0]))


@pytest.mark.parametrize("graphs", [True, False])
def test_captured_and_replayed(hipdev, graphs):
    use_device(hipdev)

    def step(x, w, targets):
        got = [linear_cross_entropy(x, w, targets)]
        got += grad(got[0], [x, w])
        realize(*got)
        return got

    def args(seed):
        rng, x, w, targets = draw(seed, "bfloat16", 200, 64, 700, left_out=0.1)
        return [Tensor(x, dtype=DTYPES["bfloat16"], requires_grad=True), Tensor(w, dtype=DTYPES["bfloat16"], requires_grad=True), Tensor(targets, dtype=int32)]

    saved, hipdev.replay_graphs = hipdev.replay_graphs, graphs
    try:
        program = capture(step)
        sets = [args(s) for s in range(3)]
        for a in sets[:2]:
            program(*a)
        for _ in range(2):
            for a in sets:
                got = [t.numpy() for t in program(*a)]
                fresh = [Tensor(t.numpy(), dtype=t.dtype, requires_grad=i < 2) for i, t in enumerate(a)]
                for y, z in zip(got, step(*fresh)):
                    np.testing.assert_array_equal(y, z.numpy())
    finally:
        hipdev.replay_graphs = saved
