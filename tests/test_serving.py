"""attend_paged, sample, quantize_rows and int8_linear without a GPU: composed from limn's primitives against the definitions in
float64, their refusals, and the C ABI's."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from conftest import DTYPES, storage_values
from limn_amd.dtypes import to_storage
from limn_amd.hip import runtime
from limn_amd.int8 import int8_linear, quantize_rows
from limn_amd.paged import attend_paged
from limn_amd.sampling import sample
from limn_amd.seam import Tensor, float32, int8, int32, realize, set_device
from oracle.attend import within
from oracle.serving import int8_linear as int8_oracle
from oracle.serving import paged, quantized
from oracle.serving import sample as sample_oracle
from serving import logit_rows, paged_inputs


@pytest.fixture(autouse=True)
def numpy_device():
    set_device("numpy")


def tensors(x, dtype):
    t = DTYPES[dtype]
    kinds = dict(starts=int32, lengths=int32, table=int32, slopes=float32)
    return {n: None if a is None else Tensor(to_storage(a, kinds.get(n, t)), dtype=kinds.get(n, t)) for n, a in x.items()}


PAGED = [
    dict(),
    dict(counts=(3, 1, 5), lengths=(7, 1, 5), heads=4, kv_heads=2, spare=2, rows_before=1),
    dict(counts=(0, 2, 0, 1), lengths=(6, 9, 0, 3), page=3, slopes=True),
    dict(counts=(4, 2), lengths=(2, 9), page=1),  # more rows than positions
    dict(counts=(2, 2), lengths=(100, 6), page=4, table_pages=2),  # past the table
]


@pytest.mark.parametrize("dtype", ["float32", "float64", "bfloat16"])
@pytest.mark.parametrize("case", PAGED, ids=str)
def test_paged_composed(case, dtype):
    x = paged_inputs(1, **{**case, "dtype": "float32" if dtype == "float64" else dtype})
    t = tensors(x, dtype)
    out = attend_paged(**t, softcap=3.0)
    realize(out)
    (want, bound), keys, values = paged(**x, softcap=3.0, dtype="float32" if dtype == "float64" else dtype)
    within(out.numpy(), want, bound, "out")
    np.testing.assert_array_equal(t["key_pages"].numpy(), keys)
    np.testing.assert_array_equal(t["value_pages"].numpy(), values)


def test_paged_composed_bad_pages_and_no_new_keys():
    x = paged_inputs(2, counts=(3, 2), lengths=(9, 6), page=2)
    x["table"][0, 1], x["table"][1, 2] = 99, -5  # a hole, and the new tokens' own page
    t = tensors(x, "float32")
    out = attend_paged(**t)
    realize(out)
    (want, bound), keys, _ = paged(**x)
    within(out.numpy(), want, bound, "out")
    np.testing.assert_array_equal(t["key_pages"].numpy(), keys)
    t = tensors(x, "float32")
    out = attend_paged(**{**t, "k": None, "v": None})
    (want, bound), _, _ = paged(**{**x, "k": None, "v": None})
    within(out.numpy(), want, bound, "out")
    np.testing.assert_array_equal(t["key_pages"].numpy(), x["key_pages"])


SETTINGS = [
    dict(),
    dict(top_k=3),
    dict(top_p=0.6),
    dict(min_p=0.2),
    dict(temperature=0.4, top_k=5, top_p=0.9, min_p=0.01),
    dict(temperature=0.0),
    dict(top_k=1000, top_p=1.5, min_p=-1.0, temperature=2.0),
    dict(top_p=0.0),
]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
def test_sample_composed(kw):
    logits, u, _ = logit_rows(3, 40, 17)
    logits[3:9] = np.round(logits[3:9])  # equal ones
    logits[9] = 1.0
    logits[10, 4:] = -np.inf
    logits[11, ::2] = np.nan
    logits[12] = -np.inf
    logits[13, [2, 5]] = np.inf
    tokens, logs = sample(Tensor(logits), Tensor(u), **kw)
    got = realize(tokens, logs) and (tokens.numpy(), logs.numpy())
    rows = {n: None if n not in kw else np.full(40, kw[n]) for n in ("temperature", "top_k", "top_p", "min_p")}
    want, (lp, bound) = sample_oracle(logits, u, **rows)
    keep = np.arange(40) != 11  # a NaN among the rest is the kernels' to leave out
    np.testing.assert_array_equal(got[0][keep], want[keep])
    within(got[1][keep], lp[keep], bound[keep] + 1e-6, "logprob")


def test_sample_draws_by_the_shares():
    """Every share of the unit interval goes to its token."""
    logits = np.log(np.array([[0.5, 0.25, 0.125, 0.125]]))
    u = np.array([0.0, 0.49, 0.51, 0.74, 0.76, 0.87, 0.88, 0.999], np.float32)
    got, _ = sample(Tensor(np.repeat(logits, 8, 0)), Tensor(u))
    np.testing.assert_array_equal(got.numpy(), [0, 0, 1, 1, 2, 2, 3, 3])


@pytest.mark.parametrize("bias", [False, True])
def test_int8_composed(bias):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((2, 3, 19)).astype(np.float32)
    x[0, 0] = 0
    w = rng.standard_normal((7, 19)).astype(np.float32)
    b = rng.standard_normal(7).astype(np.float32) if bias else None
    values, scales = quantize_rows(Tensor(w))
    want, s = quantized(w)
    assert (np.abs(values.numpy().astype(int) - want) <= 1).all() and np.allclose(scales.numpy(), s, rtol=1e-6)
    y = int8_linear(Tensor(x), Tensor(want, dtype=int8), Tensor(s), None if b is None else Tensor(b))
    out, bound = int8_oracle(x.reshape(6, 19), want, s, b)
    # a number at the border of two whole ones may go the other way: one step of x times the largest weight
    step = (np.abs(x).max(-1).reshape(6, 1) / 127) * (np.abs(want).max() * s.max())
    within(y.numpy().reshape(6, 7), out, bound + step, "y")


def test_gradients_are_refused():
    x = paged_inputs(5)
    t = tensors(x, "float32")
    t["q"].requires_grad = True
    with pytest.raises(ValueError, match="no gradient"):
        attend_paged(**t)
    w = Tensor(np.ones((3, 4)), dtype=int8)
    with pytest.raises(ValueError, match="no gradient"):
        int8_linear(Tensor(np.ones((2, 4)), requires_grad=True, dtype=float32), w, Tensor(np.ones(3), dtype=float32))


@pytest.mark.parametrize(
    "change,message",
    [
        (dict(q=(3, 8)), "needs"),
        (dict(q=(3, 3, 8)), "evenly"),
        (dict(q=(3, 4, 7)), "mismatch"),
        (dict(value_pages=(9, 2, 4, 8)), "mismatch"),
        (dict(k=(3, 4, 8)), "new keys and values"),
        (dict(k=None), "go together"),
        (dict(starts=(2,)), "starts"),
        (dict(lengths=(3,)), "lengths"),
        (dict(table=(4,)), "table"),
        (dict(slopes=(3,)), "slopes"),
    ],
    ids=str,
)
def test_paged_refusals(change, message):
    shapes = dict(q=(3, 4, 8), k=(3, 2, 8), v=(3, 2, 8), key_pages=(8, 2, 4, 8), value_pages=(8, 2, 4, 8), starts=(3,), lengths=(2,), table=(2, 3), slopes=(4,))
    shapes.update(change)
    t = {n: None if s is None else Tensor(np.zeros(s), dtype=int32 if n in ("starts", "lengths", "table") else float32) for n, s in shapes.items()}
    with pytest.raises(ValueError, match=message):
        attend_paged(**t)


def test_paged_refuses_numbers_and_pages_that_are_no_buffers():
    t = tensors(paged_inputs(6), "float32")
    for kw, message in ((dict(softcap=-1.0), "softcap"), (dict(softcap=float("nan")), "softcap"), (dict(scale=float("inf")), "scale")):
        with pytest.raises(ValueError, match=message):
            attend_paged(**t, **kw)
    with pytest.raises(ValueError, match="in place"):
        attend_paged(**{**t, "key_pages": t["key_pages"] + 1.0})
    with pytest.raises(ValueError, match="in place"):
        attend_paged(**{**t, "value_pages": t["key_pages"]})
    with pytest.raises(ValueError, match="pages are"):
        attend_paged(**{**t, "q": t["q"].double()})


def test_sample_and_int8_refusals():
    x, u = Tensor(np.zeros((3, 5)), dtype=float32), Tensor(np.zeros(3), dtype=float32)
    for args, kw, message in (((x.int(), u), {}, "float logits"), ((x, x), {}, "uniforms"), ((x, u), dict(top_k=1.5), "whole"), ((x, u), dict(top_p=float("nan")), "finite"),
                              ((x, u), dict(temperature=Tensor(np.zeros(2), dtype=float32)), "temperature"), ((x, u), dict(top_k=u), "top_k")):
        with pytest.raises(ValueError, match=message):
            sample(*args, **kw)
    w, s = Tensor(np.zeros((4, 5)), dtype=int8), Tensor(np.zeros(4), dtype=float32)
    for args, message in (((x, x, s), "int8 weight"), ((u, w, s), "widths"), ((x, w, u), "scales"), ((x, w, s, u), "bias"), ((x.int(), w, s), "float rows")):
        with pytest.raises(ValueError, match=message):
            int8_linear(*args)
    with pytest.raises(ValueError, match="float"):
        quantize_rows(w)


# ---- the C ABI: every call below fails its checks before anything is launched; the pointers are never read ----

FAKE, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1001)


def call(entry, workspace=FAKE, room=1 << 40, **kw):
    lib = runtime.kernels()
    if entry == "paged":
        a = dict(q=FAKE, k=FAKE, v=FAKE, table=FAKE, dtype=1, tokens=4, sequences=2, heads=4, kv_heads=2, hd=16, pages=9, page=4, table_pages=3, q_row=64, k_row=32, v_row=32,
                 scale=0.25, softcap=0.0)
        a.update(kw)
        return lib.limn_hip_attend_paged(a["q"], a["k"], a["v"], FAKE, FAKE, FAKE, FAKE, a["table"], None, FAKE, *list(a.values())[4:], workspace, room, None)
    if entry == "sample":
        a = dict(logits=FAKE, uniforms=FAKE, dtype=1, rows=2, vocab=9, stride=9)
        a.update(kw)
        return lib.limn_hip_sample(a["logits"], a["uniforms"], None, None, None, None, FAKE, None, a["dtype"], a["rows"], a["vocab"], a["stride"], workspace, room, None)
    a = dict(x=FAKE, w=FAKE, s=FAKE, bias=None, dtype=1, rows=2, width=9, outputs=5)
    a.update(kw)
    if entry == "quantize":
        return lib.limn_hip_quantize_rows(a["x"], a["w"], a["s"], a["dtype"], a["rows"], a["width"], None)
    return lib.limn_hip_int8_linear(a["x"], a["w"], a["s"], a["bias"], FAKE, a["dtype"], a["rows"], a["width"], a["outputs"], workspace, room, None)


@pytest.mark.parametrize(
    "entry,kw,code,message",
    [
        ("paged", dict(dtype=0), 2, "float32, float16 or bfloat16"),
        ("paged", dict(tokens=0), 1, "positive"),
        ("paged", dict(page=0), 1, "positive"),
        ("paged", dict(kv_heads=3), 1, "evenly"),
        ("paged", dict(q_row=63), 1, "overlap"),
        ("paged", dict(v_row=31), 1, "overlap"),
        ("paged", dict(scale=float("nan")), 1, "scale"),
        ("paged", dict(softcap=-2.0), 1, "softcap"),
        ("paged", dict(hd=257, q_row=2000, k_row=2000, v_row=2000), 2, "head dim"),
        ("paged", dict(table_pages=1 << 30), 2, "out of range"),
        ("paged", dict(tokens=1 << 29), 2, "out of range"),
        ("paged", dict(q=None), 1, "null"),
        ("paged", dict(k=None), 1, "together"),
        ("paged", dict(q=ODD), 1, "aligned"),
        ("paged", dict(table=ctypes.c_void_p(0x1002)), 1, "aligned"),
        ("paged", dict(room=-1), 1, "workspace"),
        ("sample", dict(dtype=0), 2, "float32, float16 or bfloat16"),
        ("sample", dict(rows=0), 1, "positive"),
        ("sample", dict(stride=8), 1, "overlap"),
        ("sample", dict(vocab=(1 << 24) + 1, stride=1 << 25), 2, "out of range"),
        ("sample", dict(uniforms=None), 1, "null"),
        ("sample", dict(logits=ODD), 1, "aligned"),
        ("sample", dict(room=-1), 1, "workspace"),
        ("sample", dict(vocab=1 << 16, stride=1 << 16, workspace=None), 1, "workspace"),
        ("sample", dict(vocab=1 << 16, stride=1 << 16, room=1000), 1, "workspace"),
        ("quantize", dict(dtype=5), 2, "float32, float16 or bfloat16"),
        ("quantize", dict(width=0), 1, "positive"),
        ("quantize", dict(s=None), 1, "null"),
        ("quantize", dict(x=ODD), 1, "aligned"),
        ("quantize", dict(rows=1 << 31), 2, "out of range"),
        ("int8", dict(dtype=0), 2, "float32, float16 or bfloat16"),
        ("int8", dict(outputs=0), 1, "positive"),
        ("int8", dict(width=(1 << 17) + 1), 2, "2^17"),
        ("int8", dict(w=None), 1, "null"),
        ("int8", dict(bias=ODD), 1, "aligned"),
        ("int8", dict(workspace=None), 1, "workspace"),
        ("int8", dict(room=8), 1, "workspace"),
    ],
)
def test_the_abi_refuses_with_a_reason(entry, kw, code, message):
    assert call(entry, **kw) == code
    assert message in runtime.kernels().limn_hip_last_error().decode()


def test_paged_queries_keys_and_values_in_one():
    x = paged_inputs(5, counts=(2, 1), lengths=(7, 3), heads=4, kv_heads=2, hd=8, spare=1)
    tokens = len(x["q"])
    on = lambda n: Tensor(x[n])  # noqa: E731
    where = lambda: [Tensor(x[n], dtype=int32) for n in ("starts", "lengths", "table")]  # noqa: E731
    apart, one = ([on("key_pages"), on("value_pages")] for _ in range(2))
    want = attend_paged(on("q"), on("k"), on("v"), *apart, *where()).numpy()
    qkv = np.concatenate([x[n].reshape(tokens, -1) for n in ("q", "k", "v")], 1)
    np.testing.assert_array_equal(attend_paged(Tensor(qkv), None, None, *one, *where(), heads=4).numpy(), want)
    for a, b in zip(one, apart):
        np.testing.assert_array_equal(a.numpy(), b.numpy())
    for bad, heads, match in ((qkv, 3, "mismatch"), (qkv[:, :-1], 4, "mismatch"), (x["q"], 4, "all in one"), (qkv, -1, "all in one"), (qkv, 0, "all in one")):
        with pytest.raises(ValueError, match=match):
            attend_paged(Tensor(bad), None, None, *one, *where(), heads=heads)
    with pytest.raises(ValueError, match="beside"):
        attend_paged(Tensor(qkv), on("k"), on("v"), *one, *where(), heads=4)


def test_a_vocabulary_past_the_kernels_is_refused():
    logits = Tensor(np.zeros(1), dtype=float32).expand((1 << 24) + 1)
    with pytest.raises(ValueError, match="vocabulary"):
        sample(logits, Tensor(np.float32(0.5), dtype=float32))


def test_an_aligned_weight_asks_for_no_copy_of_its_size():
    """Of a width whose rows are aligned, the copy for a start that is not goes in slabs; other widths are copied whole."""
    lib = runtime.kernels()
    need = lambda width, outputs: lib.limn_hip_int8_linear_workspace(3, 16, width, outputs) - 16 * -(-width // 256) * 256 - 256  # noqa: E731
    assert need(4096, 131072) <= 1 << 26 and need(1 << 17, 1 << 16) <= 1 << 26
    assert need(512, 1000) == 512 * 1000 and need(4097, 8192) == 4352 * 8192


@pytest.mark.parametrize("dtype", ["float32", "float64"])
def test_rows_with_infinities_and_nan_in_8_bits(dtype):
    """Composed of primitives as in the kernels: zeros and the scale NaN, results of NaN, and no other row's."""
    x = np.random.default_rng(6).standard_normal((6, 20)).astype(dtype)
    x[1, 3], x[2, 19], x[4, 0] = np.inf, np.nan, -np.inf
    kind = DTYPES[dtype]
    with np.errstate(invalid="ignore"):
        values, scales = quantize_rows(Tensor(x, dtype=kind))
        y = int8_linear(Tensor(x, dtype=kind), Tensor(np.eye(5, 20), dtype=int8), Tensor(np.ones(5), dtype=float32)).numpy()
        values, scales = values.numpy(), scales.numpy()
    odd = np.isin(np.arange(6), [1, 2, 4])
    assert (values[odd] == 0).all() and np.isnan(scales[odd]).all() and np.isnan(y[odd]).all()
    assert np.isfinite(scales[~odd]).all() and np.isfinite(y[~odd]).all()
