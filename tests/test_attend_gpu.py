"""Attention with score rules on the MI355X: limn_amd.attend on the hip device and the C ABI, against the definition in
float64 within the bounds on rounding that oracle/attend.py derives."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import DTYPES, storage_values, upload
from limn_amd.attend import attend
from limn_amd.dtypes import ABI_CODE, from_storage
from limn_amd.hip import runtime
from limn_amd.seam import Tensor, capture, float32, grad, int32, realize, use_device
from oracle.attend import attend as definition
from oracle.attend import within

pytestmark = pytest.mark.gpu


def packed(rng, batch, t, mean, padded=True):
    docs = np.cumsum(rng.random((batch, t)) < 1.0 / mean, axis=1).astype(np.int32)
    if padded:
        for b in range(batch):
            docs[b, t - rng.integers(0, t // 3 + 1):] = -1
    return docs


def draw(seed, dtype, batch, heads, kv_heads, t_q, t_k, hd, hd_v, std=1.0):
    rng = np.random.default_rng(seed)
    shapes = ((batch, heads, t_q, hd), (batch, kv_heads, t_k, hd), (batch, kv_heads, t_k, hd_v), (batch, heads, t_q, hd_v))
    stds = (std, 1.0, 1.0, 1.0)
    return rng, [storage_values((rng.standard_normal(s) * f).astype(np.float32), DTYPES[dtype]) for s, f in zip(shapes, stds)]


def tensors(rules):
    return {n: Tensor(x, dtype=float32 if n == "slopes" else int32) for n, x in rules.items()}


def trained(dev, q, k, v, do, dtype, rules, flags):
    use_device(dev)
    tq, tk, tv = (Tensor(x, dtype=DTYPES[dtype], requires_grad=True) for x in (q, k, v))
    out = attend(tq, tk, tv, **flags, **tensors(rules))
    got = [out, *grad((out * Tensor(do, dtype=DTYPES[dtype])).sum(), [tq, tk, tv])]
    realize(*got)
    return dict(zip(("out", "dq", "dk", "dv"), (t.numpy() for t in got)))


def check(dev, q, k, v, do, dtype, rules, flags):
    got = trained(dev, q, k, v, do, dtype, rules, flags)
    want = definition(q, k, v, dout=do, dtype=dtype, **flags, **rules)
    for name, x in got.items():
        within(x, *want[name], f"{name} {dtype}")
    return got


HALVES = ["bfloat16", "float16"]
TYPES = ["float32", *HALVES]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t_q,t_k", [(1, 1), (1, 65), (2, 2), (31, 33), (64, 64), (129, 129), (70, 200), (300, 300)])
def test_lengths(hipdev, dtype, t_q, t_k):
    rng, (q, k, v, do) = draw(t_q * 1000 + t_k, dtype, 2, 2, 2, t_q, t_k, 64, 64)
    check(hipdev, q, k, v, do, dtype, {}, dict(causal=True))
    check(hipdev, q, k, v, do, dtype, {}, dict())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("bits", [-12, 10])
def test_cotangents_of_every_size(hipdev, dtype, hd, bits):
    """A mean's cotangents, and a loss multiplied up: float16's numbers reach neither products of small ones nor,
    past 2^16, of large ones."""
    rng, (q, k, v, do) = draw(hd + bits, dtype, 1, 2, 1, 190, 190, hd, hd)
    do = storage_values(do * np.float32(2.0**bits), DTYPES[dtype])
    check(hipdev, q, k, v, do, dtype, {}, dict(causal=True))
    check(hipdev, q, k, v, do, dtype, dict(slopes=np.array([0.25, 0.0625], np.float32)), dict(causal=True, softcap=5.0))


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_large_cotangents_of_a_call_that_sees_everything(hipdev, hd):
    """Score gradients past float16's range (they go multiplied by 2^8) in a call without masks, whose gradients are finite."""
    _, (q, k, v, do) = draw(hd, "float16", 1, 2, 1, 130, 130, hd, hd)
    got = check(hipdev, q, k, v, storage_values(do * np.float32(2.0**11), DTYPES["float16"]), "float16", {}, dict(scale=0.25))
    assert np.abs(got["dq"]).max() > 256


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,hd_v", [(1, 1), (8, 8), (16, 16), (32, 32), (33, 33), (40, 40), (64, 64), (64, 80), (72, 72), (80, 80), (96, 96), (100, 100), (128, 128), (128, 64), (160, 200), (256, 256)])
def test_head_dims(hipdev, dtype, hd, hd_v):
    rng, (q, k, v, do) = draw(hd * 7 + hd_v, dtype, 1, 2, 1, 150, 150, hd, hd_v)
    check(hipdev, q, k, v, do, dtype, dict(slopes=np.array([0.25, 0.0625], np.float32)), dict(causal=True, softcap=5.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (6, 2), (5, 5), (8, 1)])
def test_shared_heads(hipdev, dtype, heads, kv_heads):
    rng, (q, k, v, do) = draw(heads * 10 + kv_heads, dtype, 2, heads, kv_heads, 100, 100, 64, 64)
    rules = dict(slopes=(0.5 ** np.arange(1, heads + 1)).astype(np.float32), documents=packed(rng, 2, 100, 40))
    check(hipdev, q, k, v, do, dtype, rules, dict(causal=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("softcap,alibi,documents,prefix,ragged", [
    (4.0, False, False, False, False), (0.0, True, False, False, False), (0.0, False, True, False, False), (0.0, False, False, True, False),
    (0.0, False, False, False, True), (4.0, True, True, True, True), (0.0, True, True, False, True)])
def test_rules(hipdev, dtype, dim, causal, softcap, alibi, documents, prefix, ragged):
    t_q, t_k = (230, 290) if ragged else (290, 290)
    rng, (q, k, v, do) = draw(dim + 2 * causal, dtype, 3, 4, 2, t_q, t_k, dim, dim, std=3.0 if softcap else 1.0)
    rules = {}
    if alibi:
        rules["slopes"] = np.array([0.5, 0.1, 0.02, 0.0], np.float32)
    if documents:
        rules["documents"] = packed(rng, 3, t_k, 60)
    if prefix and causal:
        rules["prefix"] = np.array([0, 77, 250], np.int32)
    if ragged:
        rules["lengths"] = np.array([290, 131, 3], np.int32)  # one shorter than its queries
    check(hipdev, q, k, v, do, dtype, rules, dict(causal=causal, softcap=softcap))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,t_q,t_k", [(2, 2, 600, 600), (6, 2, 700, 700), (5, 1, 1000, 1000), (4, 1, 65, 700)])
def test_few_key_heads_cut_into_parts(hipdev, dtype, hd, heads, kv_heads, t_q, t_k):
    """Too few key blocks for the GPU: the queries' heads, then their tiles, are spread over workgroups."""
    rng, (q, k, v, do) = draw(heads + t_q + hd, dtype, 1, heads, kv_heads, t_q, t_k, hd, hd)
    check(hipdev, q, k, v, do, dtype, {}, dict(causal=True))
    check(hipdev, q, k, v, do, dtype, dict(documents=packed(rng, 1, t_k, 150), prefix=np.array([130], np.int32)), dict(causal=True, softcap=5.0))
    check(hipdev, q, k, v, do, dtype, dict(lengths=np.array([t_k - 90], np.int32)), dict())
    v[0, 0, t_k - 5] = np.inf  # the last rows alone see it
    check(hipdev, q, k, v, do, dtype, {}, dict(causal=True))


@pytest.mark.parametrize("dtype,hd,softcap", [("bfloat16", 128, 0.0), ("float16", 72, 4.0)])
def test_score_gradients_past_the_workspace_limit(hipdev, dtype, hd, softcap):
    """Calls whose score gradients would take more than 2.5 GiB compute the scores again in the dQ pass: two heads, repeated
    until they do, each repeat bit for bit the first."""
    rng, (q, k, v, do) = draw(hd, dtype, 1, 2, 2, 2048, 2048, hd, hd)
    reps = (5 << 29) // (2 * 16 * 32 * 16384) + 1
    docs = packed(rng, 1, 2048, 400)
    rules = dict(documents=docs, prefix=np.array([300], np.int32)) if softcap else {}
    flags = dict(causal=True, softcap=softcap)
    many = lambda x: np.tile(x, (reps, *[1] * (x.ndim - 1)))  # noqa: E731
    got = trained(hipdev, *(many(x) for x in (q, k, v, do)), dtype, {n: many(x) for n, x in rules.items()}, flags)
    want = definition(q, k, v, dout=do, dtype=dtype, **flags, **rules)
    for name, x in got.items():
        within(x[:1], *want[name], f"{name} {dtype}")
        assert all(np.array_equal(x[r], x[0]) for r in range(1, reps)), name


@pytest.mark.parametrize("dtype", TYPES)
def test_documents_in_any_order_and_rows_that_see_nothing(hipdev, dtype):
    rng, (q, k, v, do) = draw(5, dtype, 3, 2, 2, 200, 200, 64, 64)
    docs = rng.integers(-1, 4, (3, 200)).astype(np.int32)
    docs[1] = -1
    docs[2, :150] = -(2**31)
    docs[2, 150:] = 2**31 - 1
    for causal in (False, True):
        got = check(hipdev, q, k, v, do, dtype, dict(documents=docs), dict(causal=causal))
        assert not got["out"][1].any() and not got["dk"][1].any() and not got["dq"][1].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_infinities_and_nan_in_hidden_places(hipdev, dtype, dim, bad):
    """A padded token's rows (q, k, v and dout), another document's values, and keys past the live ones hold `bad`."""
    rng, (q, k, v, do) = draw(dim, dtype, 2, 4, 2, 170, 170, dim, dim)
    docs = np.repeat(np.arange(4), 50)[None, :170].repeat(2, 0).astype(np.int32)
    docs[:, 160:] = -1
    for x in (q, k, v, do):
        x[:, :, 160:] = bad
    v[0, 0, 77, 5] = bad  # document 1's rows alone see it (from row 77 on, if causal)
    do[0, 1, 120, 7] = bad  # a row of document 2: its dq, and the gradients of the keys it sees
    check(hipdev, q, k, v, do, dtype, dict(documents=docs), dict(causal=True))
    check(hipdev, q, k, v, do, dtype, dict(documents=docs), dict())
    rng, (q, k, v, do) = draw(dim + 1, dtype, 2, 4, 2, 40, 170, dim, dim)
    k[:, :, 150:] = bad
    v[:, :, 150:] = bad
    check(hipdev, q, k, v, do, dtype, dict(lengths=np.array([150, 64], np.int32)), dict(causal=True, softcap=5.0))
    rng, (q, k, v, do) = draw(dim + 2, dtype, 1, 2, 1, 100, 100, dim, dim)
    v[0, 0, 90, 3] = bad  # rows 90 to 99 see it
    k[0, 0, 99, 3] = bad if np.isnan(bad) else 0.0  # the last row alone sees it, which is NaN then
    check(hipdev, q, k, v, do, dtype, {}, dict(causal=True))


@pytest.mark.parametrize("dtype", TYPES)
def test_far_and_near_scores(hipdev, dtype):
    """Scores of some hundreds, where one key takes all the weight, and all equal ones."""
    rng, (q, k, v, do) = draw(11, dtype, 1, 2, 1, 130, 130, 64, 64, std=60.0)
    check(hipdev, q, k, v, do, dtype, {}, dict(causal=True))
    check(hipdev, np.zeros_like(q), k, v, do, dtype, {}, dict(causal=True))
    check(hipdev, q, k, v, do, dtype, dict(slopes=np.array([100.0, 1e-6], np.float32)), dict(causal=True, softcap=50.0, scale=0.01))
    check(hipdev, q, k, v, do, dtype, {}, dict(causal=True, scale=-0.02))
    check(hipdev, q, k, v, do, dtype, {}, dict(scale=0.0))


# ---- the C ABI -------------------------------------------------------------------------------------------------


def served(dev, q, k, v, dtype, rules, causal=False, softcap=0.0, scale=None, guard=256):
    """limn_hip_attend_fwd on buffers of its own, with guard bytes behind out and lse that must stay."""
    t = DTYPES[dtype]
    batch, heads, t_q, hd = q.shape
    kv_heads, t_k, hd_v = v.shape[1:]
    sizes = (batch, heads, kv_heads, t_q, t_k, hd, hd_v)
    ins = [upload(dev, x, t).arg for x in (q, k, v)]
    given = [upload(dev, rules[n], float32 if n == "slopes" else int32).arg if n in rules else None for n in ("slopes", "documents", "prefix", "lengths")]
    need = dev.lib.limn_hip_attend_workspace(ABI_CODE[t], *sizes, 0)
    ws = dev._alloc(max(1, need))
    out_bytes, lse_bytes = batch * heads * t_q * hd_v * t.itemsize, batch * heads * t_q * 4
    out, lse = dev._alloc(out_bytes + guard), dev._alloc(lse_bytes + guard)
    for b in (out, lse):
        dev.copyin(b, np.full(b.nbytes, 0xAB, np.uint8))
    scale = hd**-0.5 if scale is None else scale
    runtime.check_limn(dev.lib.limn_hip_attend_fwd(*(b.ptr for b in ins), *(b.ptr if b else None for b in given), out.ptr, lse.ptr, ABI_CODE[t], *sizes,
                                                   int(causal), scale, softcap, ws.ptr, need, None))
    dev.finish()
    raw_out, raw_lse = dev.copyout(out), dev.copyout(lse)
    assert (raw_out[out_bytes:] == 0xAB).all() and (raw_lse[lse_bytes:] == 0xAB).all()
    return from_storage(raw_out[:out_bytes], t, (batch, heads, t_q, hd_v)), raw_lse[:lse_bytes].view(np.float32).reshape(batch, heads, t_q)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,t_q,t_k,dim,lengths", [
    (8, 8, 1, 1000, 64, [777]), (8, 2, 1, 2049, 128, [2049, 1, 513, 0]), (4, 1, 5, 700, 80, [700, 5]), (40, 1, 1, 300, 64, [299, 31, 32]), (3, 3, 16, 16, 32, [16]),
    (6, 2, 70, 4100, 128, [4100]), (2, 1, 1, 1, 16, [1, 0]), (2, 2, 1, 640, 100, [555, 640])])
def test_tokens_against_a_cache(hipdev, dtype, heads, kv_heads, t_q, t_k, dim, lengths):
    rng, (q, k, v, _) = draw(t_k + dim, dtype, len(lengths), heads, kv_heads, t_q, t_k, dim, dim, std=2.0)
    for b, n in enumerate(lengths):  # what lies behind the live keys is never read
        k[b, :, n:] = np.nan
        v[b, :, n:] = np.nan
    rules = dict(lengths=np.array(lengths, np.int32), slopes=(0.9 ** np.arange(1, heads + 1) * 0.05).astype(np.float32))
    for softcap, given in ((0.0, dict(lengths=rules["lengths"])), (20.0, rules)):
        out, lse = served(hipdev, q, k, v, dtype, given, causal=True, softcap=softcap)
        want = definition(q, k, v, dtype=dtype, causal=True, softcap=softcap, **given)
        within(out, *want["out"], "out")
        within(lse, *want["lse"], "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,t_q,t_k,dim,lengths", [
    (2, 2, 64, 1024, 64, [1024]), (4, 2, 200, 1500, 128, [1500, 333]), (3, 1, 256, 1024, 80, [1000]), (2, 1, 333, 4097, 64, [4097]), (6, 3, 65, 2000, 40, [64, 0, 1999])])
def test_part_of_a_sequence_against_its_cache(hipdev, dtype, heads, kv_heads, t_q, t_k, dim, lengths):
    rng, (q, k, v, _) = draw(t_k + dim, dtype, len(lengths), heads, kv_heads, t_q, t_k, dim, dim, std=2.0)
    for b, n in enumerate(lengths):
        k[b, :, n:] = np.nan
        v[b, :, n:] = np.nan
    rules = dict(lengths=np.array(lengths, np.int32), slopes=(0.9 ** np.arange(1, heads + 1) * 0.05).astype(np.float32), prefix=np.full(len(lengths), 300, np.int32))
    if min(lengths) > 100:
        v[0, 0, min(lengths) - 50, 3] = np.inf  # seen by the last rows alone
    for softcap, given in ((0.0, dict(lengths=rules["lengths"])), (20.0, rules)):
        out, lse = served(hipdev, q, k, v, dtype, given, causal=True, softcap=softcap)
        want = definition(q, k, v, dtype=dtype, causal=True, softcap=softcap, **given)
        within(out, *want["out"], "out")
        within(lse, *want["lse"], "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads,t_q,t_k,dim", [(4, 2, 130, 1111, 64), (2, 2, 256, 1024, 128)])
def test_other_keys_than_the_queries_own(hipdev, dtype, heads, kv_heads, t_q, t_k, dim):
    """Queries that see every live key, the distance taken from the end of them."""
    rng, (q, k, v, _) = draw(t_k + dim, dtype, 2, heads, kv_heads, t_q, t_k, dim, dim)
    k[1, :, 700:] = np.nan
    v[1, :, 700:] = np.inf
    given = dict(lengths=np.array([t_k, 700], np.int32), slopes=(0.02 * 0.9 ** np.arange(heads)).astype(np.float32))
    out, lse = served(hipdev, q, k, v, dtype, given, softcap=10.0)
    want = definition(q, k, v, dtype=dtype, softcap=10.0, **given)
    within(out, *want["out"], "out")
    within(lse, *want["lse"], "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_key_some_queries_do_not_see(hipdev, dtype, bad):
    """The newest keys of several queries hold `bad`: the queries before them stay as they are, in a short cache and a long one."""
    for t_k, length in ((90, 80), (3000, 2999)):
        rng, (q, k, v, _) = draw(t_k, dtype, 1, 4, 2, 5, t_k, 64, 64)
        v[0, 0, length - 2, 3] = bad  # seen by the last two queries
        v[0, 1, length - 1, 60] = -bad  # by the last
        out, lse = served(hipdev, q, k, v, dtype, dict(lengths=np.array([length], np.int32)), causal=True)
        want = definition(q, k, v, dtype=dtype, causal=True, lengths=np.array([length], np.int32))
        within(out, *want["out"], "out")
        within(lse, *want["lse"], "lse")


def test_a_call_gives_the_same_bits_again(hipdev):
    rng, (q, k, v, do) = draw(3, "bfloat16", 2, 8, 2, 333, 333, 128, 128)
    rules = dict(documents=packed(rng, 2, 333, 80))
    first = trained(hipdev, q, k, v, do, "bfloat16", rules, dict(causal=True, softcap=30.0))
    again = trained(hipdev, q, k, v, do, "bfloat16", rules, dict(causal=True, softcap=30.0))
    for name in first:
        np.testing.assert_array_equal(first[name], again[name])


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_captured_and_replayed(hipdev, dtype, graphs):
    """Two layers (so a list long enough for a graph), captured and replayed on other inputs, with eager work of the same shapes between."""
    use_device(hipdev)

    def step(q, k, v, do, docs):
        x = attend(q, k, v, causal=True, documents=docs, softcap=9.0)
        out = attend(x, k, v, causal=True, documents=docs)
        got = [out, *grad((out * do).sum(), [q, k, v])]
        realize(*got)
        return got

    def args(seed):
        rng, (q, k, v, do) = draw(seed, dtype, 2, 4, 4, 90, 90, 64, 64)
        docs = packed(rng, 2, 90, 30)
        t = DTYPES[dtype]
        return [*(Tensor(x, dtype=t, requires_grad=True) for x in (q, k, v)), Tensor(do, dtype=t), Tensor(docs, dtype=int32)]

    saved, hipdev.replay_graphs = hipdev.replay_graphs, graphs
    try:
        program = capture(step)
        sets = [args(s) for s in range(3)]
        for a in sets[:2]:
            program(*a)
        for _ in range(2):
            for a in sets:
                got = [t.numpy() for t in program(*a)]
                fresh = [Tensor(x.numpy(), dtype=x.dtype, requires_grad=i < 3) for i, x in enumerate(a)]
                for x, y in zip(got, step(*fresh)):
                    np.testing.assert_array_equal(x, y.numpy())
    finally:
        hipdev.replay_graphs = saved


@pytest.mark.parametrize("dtype", TYPES)
def test_two_captured_programs_in_turn(hipdev, dtype):
    """Two programs of the same sizes, whose workspaces (parts, score gradients between the passes) are one, replayed in turn."""
    use_device(hipdev)
    t = DTYPES[dtype]

    def program(softcap):
        def step(q, k, v, do, docs):
            out = attend(q, k, v, causal=True, documents=docs, softcap=softcap)
            out = attend(out, k, v, causal=True, softcap=softcap)
            got = [out, *grad((out * do).sum(), [q, k, v])]
            realize(*got)
            return got

        return step, capture(step)

    def args(seed):
        rng, (q, k, v, do) = draw(seed, dtype, 4, 4, 1, 300, 300, 128, 128)
        return [*(Tensor(x, dtype=t, requires_grad=True) for x in (q, k, v)), Tensor(do, dtype=t), Tensor(packed(rng, 4, 300, 90), dtype=int32)]

    programs, sets = [program(0.0), program(6.0)], [args(s) for s in range(2)]
    for _, captured in programs:
        for a in sets:
            captured(*a)
    for _ in range(3):
        for a in sets:
            results = [(step, captured(*a)) for step, captured in programs]
            for step, got in results:
                got = [x.numpy() for x in got]
                fresh = [Tensor(x.numpy(), dtype=x.dtype, requires_grad=i < 3) for i, x in enumerate(a)]
                for x, y in zip(got, step(*fresh)):
                    np.testing.assert_array_equal(x, y.numpy())
