"""The GPT's variants on the numpy oracle: shared key heads, capped scores, a distance penalty, packed documents and the
loss without logits, together and one at a time, against the same model in torch's float64."""

from __future__ import annotations

from dataclasses import replace

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from limn_amd.gpt import GPT, GPTConfig, cross_entropy, make_trainer, packed_batch, synthetic_batch
from limn_amd.seam import device as limn_device
from limn_amd.seam import float32, grad, nn, set_seed

PLAIN = GPTConfig(vocab=37, ctx=24, dim=16, layers=2, heads=4, batch=3, dtype=float32)
EVERY = replace(PLAIN, kv_heads=2, softcap=3.0, distance=True, fused_loss=True)


@pytest.fixture(autouse=True)
def numpy_oracle():
    from oracle.numpy_device import NumpyDevice

    limn_device.active_device = NumpyDevice()


def torch_step(model: GPT, tokens: np.ndarray, targets: np.ndarray, documents: np.ndarray | None):
    """Loss and gradients, in float64."""
    W = {id(p): torch.tensor(p.numpy().astype(np.float64), requires_grad=True) for p in nn.parameters(model)}
    w = lambda p: W[id(p)]  # noqa: E731
    cfg, t = model.cfg, tokens.shape[1]
    hd, kv, at = cfg.dim // cfg.heads, cfg.key_heads, torch.arange(t)
    x = w(model.tok.weight)[torch.tensor(tokens, dtype=torch.long)]
    if not cfg.distance:
        x = x + w(model.pos.weight)[at]
    see = (at[:, None] >= at[None, :]).expand(len(tokens), 1, t, t)
    if documents is not None:
        d = torch.tensor(documents)
        see = see & (d[:, None, :, None] == d[:, None, None, :])
    for blk in model.blocks:
        b, _, c = x.shape
        h = F.linear(F.layer_norm(x, (c,), w(blk.ln1.weight), w(blk.ln1.bias), 1e-5), w(blk.qkv.weight), w(blk.qkv.bias))
        q, k, v = (p.reshape(b, t, -1, hd).transpose(1, 2) for p in h.split([c, kv * hd, kv * hd], -1))
        k, v = (p.repeat_interleave(cfg.heads // kv, 1) for p in (k, v))
        s = q @ k.transpose(-1, -2) * hd**-0.5
        if cfg.softcap:
            s = cfg.softcap * torch.tanh(s / cfg.softcap)
        if cfg.distance:
            slope = 2.0 ** (-8.0 * torch.arange(1, cfg.heads + 1, dtype=torch.float64) / cfg.heads)
            s = s - slope[:, None, None] * (at[:, None] - at[None, :]).abs()
        att = s.masked_fill(~see, float("-inf")).softmax(-1) @ v
        x = x + F.linear(att.transpose(1, 2).reshape(b, t, c), w(blk.proj.weight), w(blk.proj.bias))
        h = F.layer_norm(x, (c,), w(blk.ln2.weight), w(blk.ln2.bias), 1e-5)
        x = x + F.linear(F.gelu(F.linear(h, w(blk.up.weight), w(blk.up.bias)), approximate="tanh"), w(blk.down.weight), w(blk.down.bias))
    logits = F.linear(F.layer_norm(x, (cfg.dim,), w(model.ln.weight), w(model.ln.bias), 1e-5), w(model.head.weight))
    loss = F.cross_entropy(logits.reshape(-1, cfg.vocab), torch.tensor(targets, dtype=torch.long).reshape(-1), ignore_index=-1)
    loss.backward()
    return loss.item(), [W[id(p)].grad.numpy() for p in nn.parameters(model)]


def close(model, loss, grads, want_loss, want):
    """float32 against float64. Some 100 roundings follow one another through the two blocks and back, sums of up to
    64 terms among them, each off by at most 64 2^-24 of its largest term; a layer norm over 16 columns can raise a
    relative error some 10 times: 100 * 64 * 2^-24 * 10 = 4e-3 of the gradient's largest element at the very worst,
    and 1e-3 where no more than a quarter of them line up."""
    assert abs(loss - want_loss) <= 1e-5 * want_loss
    for p, g, w in zip(nn.parameters(model), grads, want):
        assert g.shape == w.shape == p.shape
        assert np.abs(g.numpy() - w).max() <= 1e-3 * np.abs(w).max() + 1e-7


@pytest.mark.parametrize("change", [{}, {"kv_heads": 1}, {"kv_heads": 2}, {"softcap": 3.0}, {"distance": True}, {"fused_loss": True}], ids=str)
def test_each_variant(change):
    cfg = replace(PLAIN, **change)
    set_seed(1)
    model = GPT(cfg)
    x, y = synthetic_batch(cfg, np.random.default_rng(1))
    loss = model.loss(x, y)
    close(model, loss.item(), grad(loss, nn.parameters(model)), *torch_step(model, x.numpy(), y.numpy(), None))
    if not cfg.fused_loss:
        assert loss.item() == cross_entropy(model(x), y).item()


def test_every_variant_together_on_packed_documents():
    set_seed(2)
    model = GPT(EVERY)
    x, y, documents = packed_batch(EVERY, np.random.default_rng(2), mean=6)
    assert (y.numpy()[:, -1] == -1).all() and 0 < (y.numpy() < 0).sum() < y.numel // 2 and documents.numpy().max() > 1
    loss = model.loss(x, y, documents)
    close(model, loss.item(), grad(loss, nn.parameters(model)), *torch_step(model, x.numpy(), y.numpy(), documents.numpy()))


def test_a_document_sees_none_of_its_neighbours():
    set_seed(3)
    model = GPT(EVERY)
    r = np.random.default_rng(3)
    x, _, documents = packed_batch(EVERY, r, mean=6)
    d, tokens = documents.numpy(), x.numpy().copy()
    before = model(x, documents).numpy()
    other = d != d[:, -1:]
    tokens[other] = r.integers(0, EVERY.vocab, other.sum())
    after = model(type(x)(tokens, dtype=x.dtype), documents).numpy()
    np.testing.assert_array_equal(after[~other], before[~other])
    assert (after[other] != before[other]).any()


def test_a_training_step_runs_and_moves_every_weight():
    set_seed(4)
    model, _, step = make_trainer(EVERY)
    before = [p.numpy().copy() for p in nn.parameters(model)]
    assert np.isfinite(step(*packed_batch(EVERY, np.random.default_rng(4), mean=6)).item())
    for a, p in zip(before, nn.parameters(model)):
        assert (a != p.numpy()).any() and np.isfinite(p.numpy()).all()


def test_sizes():
    assert EVERY.matmul_params() == PLAIN.matmul_params() - 2 * 16 * 16
    assert GPT(EVERY).blocks[0].qkv.weight.shape == (32, 16)


def test_refusals():
    for kv_heads in (3, 8, -1):
        with pytest.raises(ValueError, match="key heads evenly"):
            replace(PLAIN, kv_heads=kv_heads)
    x, y, documents = packed_batch(PLAIN, np.random.default_rng(0))
    with pytest.raises(ValueError, match="only the fused loss"):
        GPT(PLAIN).loss(x, y, documents)
