"""The GPT's variants through the hip device: attention with every rule and the loss without logits in one training
step, against the numpy oracle, captured and replayed."""

from __future__ import annotations

from dataclasses import replace

import numpy as np
import pytest

from limn_amd.gpt import GPT, GPTConfig, make_trainer, packed_batch, synthetic_batch
from limn_amd.seam import CompiledDevice, Tensor, bfloat16, capture, float16, float32, grad, int32, nn, set_seed
from limn_amd.seam import device as limn_device
from limn_amd.attend import attend
from oracle import sdpa as ref
from oracle.numpy_device import NumpyDevice

pytestmark = pytest.mark.gpu

SMALL = GPTConfig(vocab=131, ctx=72, dim=128, layers=2, heads=2, batch=2, kv_heads=1, softcap=5.0, distance=True, fused_loss=True)


def step(dev, cfg, packed):
    limn_device.active_device = dev
    set_seed(7)
    model = GPT(cfg)
    batch = packed_batch(cfg, np.random.default_rng(7), mean=20) if packed else synthetic_batch(cfg, np.random.default_rng(7))
    loss = model.loss(*batch)
    return loss.item(), [g.numpy() for g in grad(loss, nn.parameters(model))]


@pytest.mark.parametrize("packed", [False, True], ids=["whole", "packed"])
@pytest.mark.parametrize("dtype", [float32, bfloat16], ids=["float32", "bfloat16"])
def test_training_step_matches_the_oracle(hipdev, dtype, packed):
    """Normalised max errors. bfloat16: the oracle rounds every node, 2^-8 of the value each time, some 8 in a row
    through a block's forward and as many back: 3e-2, as for the plain model. float32: rounding 2^-24 of sums of 1024
    terms at most, 16 of them in a row: 1024 * 16 * 2^-24 = 1e-3."""
    cfg = replace(SMALL, dtype=dtype)
    got_loss, got = step(hipdev, cfg, packed)
    want_loss, want = step(NumpyDevice(), cfg, packed)
    assert abs(got_loss - want_loss) <= (1e-5 if dtype == float32 else 2e-2) * want_loss
    for g, w in zip(got, want):
        assert np.isfinite(g).all()
        assert ref.worst(g, w) <= (1e-3 if dtype == float32 else 3e-2)


def test_training_captured_equals_uncaptured(hipdev):
    from limn_amd.hip.device import HipDevice

    plain = HipDevice()
    plain.run = lambda plan, sources: CompiledDevice.run(plain, plan, sources)

    def run(captured):
        limn_device.active_device = hipdev if captured else plain
        set_seed(8)
        model, _, train = make_trainer(SMALL, lr=1e-3)
        fn = capture(train) if captured else train
        r = np.random.default_rng(8)
        losses = [fn(*packed_batch(SMALL, r, mean=20)).item() for _ in range(6)]
        return losses, [p.numpy() for p in nn.parameters(model)]

    want_losses, want = run(False)
    losses, params = run(True)
    assert losses == want_losses
    for a, b in zip(params, want):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("dtype", [float32, float16, bfloat16], ids=["float32", "float16", "bfloat16"])
def test_answering_token_by_token_is_the_whole_sequence_at_once(hipdev, dtype):
    """A cache with room to spare, read one query at a time by its length, against one causal call. The two kernels
    round weights (half types: u = half a step each) and results apart from each other; both lie within
    (2^-24 (hd + t) + 2 u) max |v| of the exact result (scores below 4 in magnitude), and then one more u."""
    limn_device.active_device = hipdev
    r = np.random.default_rng(9)
    b, heads, kv, t, room, hd = 2, 4, 2, 37, 64, 64
    rows = r.standard_normal((b, heads, t, hd)).astype(np.float32) * 0.5
    q = Tensor(rows).cast(dtype).realize()
    k, v = (Tensor(r.standard_normal((b, kv, room, hd)).astype(np.float32) * 0.5).cast(dtype).realize() for _ in range(2))
    slopes = Tensor(np.array([0.5, 0.25, 0.125, 0.0625], np.float32))
    whole = attend(q, k[:, :, :t], v[:, :, :t], causal=True, softcap=4.0, slopes=slopes).cast(float32).numpy()
    u = {float32: 2.0**-24, float16: 2.0**-11, bfloat16: 2.0**-8}[dtype]
    bound = 2 * (2.0**-24 * (hd + t) * 8 + 3 * u) * np.abs(v.cast(float32).numpy()).max()
    for i in range(t):
        lengths = Tensor(np.full(b, i + 1, np.int32), dtype=int32)
        one = attend(Tensor(rows[:, :, i : i + 1]).cast(dtype).realize(), k, v, causal=True, softcap=4.0, slopes=slopes, lengths=lengths).cast(float32).numpy()
        assert np.abs(one[:, :, 0] - whole[:, :, i]).max() <= bound, i
