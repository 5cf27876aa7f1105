"""Answering with the GPT on the numpy oracle: prompts in parts over a paged cache, then one token a step, against the
whole model on whole sequences."""

from __future__ import annotations

from dataclasses import replace

import numpy as np
import pytest

from limn_amd.gpt import GPT, GPTConfig, Held
from limn_amd.seam import Tensor, bfloat16, float32, int8, int32, no_grad, set_seed
from limn_amd.seam import device as limn_device
from limn_amd.serve import Cache, generate, held, prefill
from serving import PROMPTS, whole_logits

PLAIN = GPTConfig(vocab=37, ctx=24, dim=16, layers=2, heads=4, batch=3, dtype=float32)
EVERY = replace(PLAIN, kv_heads=2, softcap=3.0, distance=True)

# float32, computed in two orders: some 60 roundings follow one another through the two blocks, sums of up to 64 terms among
# them, each off by at most 64 2^-24 of its largest term, and a layer norm over 16 columns can raise a relative error
# some 10 times: 60 * 64 * 2^-24 * 10 = 2.3e-3 of the largest logit at the very worst
WORST = 2.3e-3
# 8-bit inputs: an input at the border of two whole numbers may go the other way, by 1 of the 127 of the largest, and in
# each of the 8 layers that follow one another
WORST_INT8 = 8 / 127


@pytest.fixture(autouse=True)
def numpy_oracle():
    from oracle.numpy_device import NumpyDevice

    limn_device.active_device = NumpyDevice()


def model_of(cfg: GPTConfig) -> GPT:
    set_seed(5)
    return GPT(cfg)


@pytest.mark.parametrize("part", [1, 3, 7, 100])
@pytest.mark.parametrize("cfg", [PLAIN, EVERY], ids=["plain", "every"])
@pytest.mark.parametrize("small", [False, True], ids=["held", "int8"])
def test_prompts_in_parts_are_the_whole_model(cfg, part, small):
    with no_grad():
        model = held(model_of(cfg), small)
        cache = Cache(model, 12, 4)
        for s, p in enumerate(PROMPTS):
            cache.reserve(s, len(p))
        got = prefill(model, cache, range(len(PROMPTS)), PROMPTS, cache.table(range(len(PROMPTS))), part).numpy()
        want = np.stack([whole_logits(model, p)[-1] for p in PROMPTS])
    assert np.abs(got - want).max() <= (WORST_INT8 if small else WORST) * np.abs(want).max()


def test_a_cache_of_a_wider_type():
    """bfloat16 rows over float32 pages: queries, keys and values are cast to the pages' type, the stream stays the model's."""
    cfg = replace(EVERY, dtype=bfloat16)
    with no_grad():
        model = held(model_of(cfg))
        cache = Cache(model, 3, 8, dtype=float32)
        cache.reserve(0, 11)
        got = prefill(model, cache, [0], [PROMPTS[2]], cache.table([0]), 5)
        assert got.dtype == bfloat16 and cache.layers[0][0].dtype == float32
        want = whole_logits(model, PROMPTS[2])[-1]
    # bfloat16 nodes on the oracle: some 30 roundings of up to 2^-8 between the two, 6 2^-8 as they go both ways
    assert np.abs(got.numpy()[0] - want).max() <= 3e-2 * np.abs(want).max()


@pytest.mark.parametrize("cfg", [PLAIN, EVERY], ids=["plain", "every"])
@pytest.mark.parametrize("small", [False, True], ids=["held", "int8"])
@pytest.mark.parametrize("rules", [dict(temperature=0.0), dict(temperature=0.7), dict(top_k=5, top_p=0.8)], ids=["largest", "warm", "few"])
def test_answers_are_the_whole_models(cfg, small, rules):
    model = model_of(cfg)
    answers, shares = generate(model, PROMPTS, 9, seed=3, int8=small, page=4, part=8, **rules)
    assert answers.shape == shares.shape == (len(PROMPTS), 9) and answers.dtype == np.int32
    worst = WORST_INT8 if small else WORST
    with no_grad():
        kept = held(model, small)
        for p, answer, share in zip(PROMPTS, answers, shares):
            logits = whole_logits(kept, [*p, *answer])[len(p) - 1 : -1].astype(np.float64)
            off = worst * np.abs(logits).max()
            picked = np.take_along_axis(logits, answer[:, None], 1)[:, 0]
            order = np.sort(logits, 1)[:, ::-1]
            if rules.get("temperature") == 0.0:
                assert (picked >= order[:, 0] - 2 * off).all() and (share == 0).all()
            elif "top_k" in rules:  # one of the 5 largest, with a share between the whole row's and all
                assert (picked >= order[:, 4] - 2 * off).all()
                assert (share <= 0).all() and (share >= picked - np.log(np.exp(order[:, :5]).sum(1)) - 2 * off).all()
            else:
                warm = logits / 0.7
                want = picked / 0.7 - np.log(np.exp(warm).sum(1))
                assert np.abs(share - want).max() <= 2 * off / 0.7 + 1e-6


def test_a_seed_gives_its_answer_again():
    model = model_of(EVERY)
    first = generate(model, PROMPTS, 6, seed=1)[0]
    assert (first == generate(model, PROMPTS, 6, seed=1, page=3, part=2, captured=False)[0]).mean() > 0.9  # a border may move with the sums' order
    assert (first != generate(model, PROMPTS, 6, seed=2)[0]).any()


def test_a_context_is_used_to_its_end():
    model = model_of(PLAIN)
    answers, _ = generate(model, [list(range(20))], 5, temperature=0.0)  # 24 positions are read, the last token is drawn behind them
    assert answers.shape == (1, 5)
    with pytest.raises(ValueError, match="do not fit"):
        generate(model, [list(range(20))], 6)
    assert generate(model_of(EVERY), [list(range(20))], 30)[0].shape == (1, 30)  # no learned positions: no end


@pytest.mark.parametrize("prompts, count, match", [([], 3, "at least"), ([[1], []], 3, "at least"), ([[1]], 0, "at least"), ([[37]], 2, "must lie"), ([[-1]], 2, "must lie")])
def test_refusals(prompts, count, match):
    with pytest.raises(ValueError, match=match):
        generate(model_of(PLAIN), prompts, count)


def test_pages_are_given_out_and_come_back():
    cache = Cache(model_of(PLAIN), 6, 4)
    cache.reserve(7, 9)
    cache.reserve(8, 4)
    assert [len(cache.tables[s]) for s in (7, 8)] == [3, 1] and len(cache.free) == 2
    own = list(cache.tables[7])
    cache.reserve(7, 12)
    assert cache.tables[7] == own
    with pytest.raises(ValueError, match="free"):
        cache.reserve(8, 13)
    assert len(cache.tables[8]) == 1 and len(cache.free) == 2
    table = cache.table([8, 7]).numpy()
    assert table.tolist() == [[*cache.tables[8], -1, -1], own]
    cache.drop(7)
    assert len(cache.free) == 5 and 7 not in cache.tables


def test_held_leaves_the_model_as_it_was():
    model = model_of(PLAIN)
    before = [id(block.qkv) for block in model.blocks]
    kept = held(model, int8=True)
    assert [id(block.qkv) for block in model.blocks] == before and not isinstance(model.head, Held)
    assert all(block.down.weight.dtype == int8 and block.down.scales.shape == (16,) for block in kept.blocks)
    assert kept.head.weight.dtype == float32 and kept.head.scales is None
    x = Tensor(np.zeros((2, 3), dtype=np.int32), dtype=int32)
    assert model.tok(x).requires_grad and model.blocks[0].qkv.weight.requires_grad


def test_a_model_that_records_is_refused():
    model = model_of(PLAIN)
    cache = Cache(model, 1)
    cache.reserve(0, 2)
    with pytest.raises(ValueError, match="no gradient"):
        prefill(model, cache, [0], [[1, 2]], cache.table([0]))


@pytest.mark.parametrize(
    "change, match",
    [
        (dict(part=0), "part"),
        (dict(prompts=[[1, 2], []]), "at least one"),
        (dict(prompts=[]), "at least one"),
        (dict(sequences=[0]), "at least one"),
        (dict(prompts=[[1, 2], [37]]), "must lie"),
        (dict(prompts=[[1, 2], [-1]]), "must lie"),
        (dict(prompts=[[1, 2], [3] * 9]), "reserved"),
        (dict(sequences=[0, 5]), "reserved"),
        (dict(prompts=[list(range(25)), [1]]), "positions end"),
        (dict(table=[[0, 1]]), "table"),
        (dict(table=[[0], [1]]), "table"),
    ],
    ids=str,
)
def test_prefill_refuses(change, match):
    """A part of nothing would never end; tokens and positions outside the model's tables would be read there."""
    with no_grad():
        model = held(model_of(PLAIN))
        cache = Cache(model, 12, 4)
        cache.reserve(0, 25)
        cache.reserve(1, 8)
        a = {**dict(sequences=[0, 1], prompts=[[1, 2, 3, 4, 5], [3]], part=3), **change}
        table = Tensor(np.array(a["table"], dtype=np.int32), dtype=int32) if "table" in a else cache.table([0, 1])
        with pytest.raises(ValueError, match=match):
            prefill(model, cache, a["sequences"], a["prompts"], table, a["part"])


def test_a_table_of_no_sequences_and_a_reservation_that_fails():
    cache = Cache(model_of(PLAIN), 3, 4)
    with pytest.raises(ValueError, match="at least one"):
        cache.table([])
    with pytest.raises(ValueError, match="free"):
        cache.reserve(2, 13)
    assert cache.tables == {} and len(cache.free) == 3


def test_prompts_in_an_array():
    model = model_of(EVERY)
    prompts = np.array([[1, 2, 3], [4, 5, 6]])
    for a, b in zip(generate(model, prompts, 3, seed=1), generate(model, prompts.tolist(), 3, seed=1)):
        np.testing.assert_array_equal(a, b)
