"""Attention with score rules without a GPU: the form composed from limn's primitives against the definition in
float64, its gradients against the definition's and against differences, and every refusal."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from limn_amd.attend import attend
from limn_amd.hip import runtime
from limn_amd.seam import Tensor, float32, float64, grad, int32, set_device
from oracle.attend import attend as definition
from oracle.attend import within


@pytest.fixture(autouse=True)
def _numpy():
    set_device("numpy")


CASES = [
    dict(),
    dict(causal=True),
    dict(causal=True, softcap=3.0),
    dict(slopes=True, softcap=2.0),
    dict(causal=True, slopes=True, documents=[[0, 0, 0, 1, 1, 2, -1], [-1, -1, 4, 4, 4, 2, 2]]),
    dict(documents=[[0, 0, 0, 1, 1, 2, -1], [-1] * 7]),
    dict(causal=True, prefix=[3, 0]),
    dict(causal=True, prefix=[9, -1], documents=[[0] * 7, [0, 0, 0, 0, 1, 1, 1]]),
    dict(causal=True, t_q=3),
    dict(causal=True, t_q=3, lengths=[7, 4]),
    dict(causal=True, t_q=3, lengths=[2, 0], slopes=True),
    dict(t_q=1, lengths=[1, 6], softcap=4.0),
    dict(t_q=2, lengths=[-5, 99], causal=True),
]


def inputs(case, heads=4, kv_heads=2, t_k=7, hd=6, hd_v=5, seed=0):
    rng = np.random.default_rng(seed)
    case = dict(case)
    t_q = case.pop("t_q", t_k)
    rules = {n: np.array(case.pop(n), dtype=np.int32) for n in ("documents", "prefix", "lengths") if n in case}
    if case.pop("slopes", False):
        rules["slopes"] = (0.5 ** np.arange(1, heads + 1)).astype(np.float32)
    q, k, v, do = (rng.standard_normal(s) for s in ((2, heads, t_q, hd), (2, kv_heads, t_k, hd), (2, kv_heads, t_k, hd_v), (2, heads, t_q, hd_v)))
    return q, k, v, do, rules, case


def tensors(rules):
    return {n: Tensor(x, dtype=float32 if n == "slopes" else int32) for n, x in rules.items()}


@pytest.mark.parametrize("case", CASES, ids=str)
def test_composed_matches_the_definition(case):
    q, k, v, do, rules, flags = inputs(case)
    tq, tk, tv = (Tensor(x, dtype=float64, requires_grad=True) for x in (q, k, v))
    out = attend(tq, tk, tv, **flags, **tensors(rules))
    got = [out, *grad((out * Tensor(do, dtype=float64)).sum(), [tq, tk, tv])]
    want = definition(q, k, v, dout=do, **flags, **rules)
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        within(t.numpy(), want[name][0], 1e-12, name)


@pytest.mark.parametrize("case", [CASES[2], CASES[4], CASES[7], CASES[9]], ids=str)
def test_the_definitions_gradients_are_its_differences(case):
    q, k, v, do, rules, flags = inputs(case, heads=2, kv_heads=1, hd=3, hd_v=2)
    want = definition(q, k, v, dout=do, **flags, **rules)
    step = 1e-5
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        for at in list(np.ndindex(*x.shape))[:: max(1, x.size // 25)]:
            ends = []
            for way in (1, -1):
                moved = [y.copy() for y in (q, k, v)]
                moved[("dq", "dk", "dv").index(name)][at] += way * step
                ends.append((definition(*moved, **flags, **rules)["out"][0] * do).sum())
            # a central difference is off by step^2 / 6 times the third derivative (tens here) and 1e-16 / step
            assert abs((ends[0] - ends[1]) / (2 * step) - want[name][0][at]) < 1e-7


def test_second_order_gradients_go_through_the_composed_form():
    q, k, v, do, rules, flags = inputs(dict(causal=True, softcap=3.0), heads=2, kv_heads=1, hd=3, hd_v=2)
    tq, tk, tv = (Tensor(x, dtype=float64, requires_grad=True) for x in (q, k, v))
    out = attend(tq, tk, tv, **flags)
    (dq,) = grad((out * out).sum(), [tq], create_graph=True)
    (dd,) = grad((dq * dq).sum(), [tk])
    assert np.isfinite(dd.numpy()).all() and np.abs(dd.numpy()).max() > 0


def make(*shape, dtype=float32):
    return Tensor(np.zeros(shape), dtype=dtype)


@pytest.mark.parametrize(
    "shapes,kw,message",
    [
        (((4, 5), (4, 5), (4, 5)), {}, "heads, t, dim"),
        (((2, 4, 5), (2, 4, 6), (2, 4, 5)), {}, "mismatch"),
        (((2, 4, 5), (2, 4, 5), (2, 3, 5)), {}, "mismatch"),
        (((1, 2, 4, 5), (2, 2, 4, 5), (2, 2, 4, 5)), {}, "mismatch"),
        (((3, 4, 5), (2, 4, 5), (2, 4, 5)), {}, "evenly"),
        (((2, 5, 5), (2, 4, 5), (2, 4, 5)), dict(causal=True), "last of the keys"),
        (((2, 4, 5),) * 3, dict(prefix="scalar"), "not causal"),
        (((2, 4, 5),) * 3, dict(softcap=-1.0), "softcap"),
        (((2, 4, 5),) * 3, dict(softcap=float("nan")), "softcap"),
        (((2, 4, 5),) * 3, dict(scale=float("inf")), "scale"),
        (((2, 4, 5),) * 3, dict(slopes="short"), "slopes"),
        (((2, 4, 5),) * 3, dict(documents="float"), "documents"),
        (((3, 2, 4, 5),) * 3, dict(lengths="short"), "lengths"),
    ],
)
def test_refusals(shapes, kw, message):
    kw = dict(kw)
    for name, value in list(kw.items()):
        if value == "short":
            kw[name] = make(1, dtype=float32 if name == "slopes" else int32)
        elif value == "float":
            kw[name] = make(4)
        elif value == "scalar":
            kw[name] = make(dtype=int32)
    with pytest.raises(ValueError, match=message):
        attend(*(make(*s) for s in shapes), **kw)


def test_int_inputs_are_refused():
    x = make(2, 4, 5, dtype=int32)
    with pytest.raises(ValueError, match="float"):
        attend(x, x, x)


# ---- the C ABI: every call below fails its checks before anything is launched; the pointers are never read ----

FAKE = ctypes.c_void_p(0x1000)


def call(backward=False, workspace=FAKE, room=1 << 40, at=FAKE, **kw):
    a = dict(dtype=1, batch=2, heads=4, kv_heads=2, t_q=8, t_k=8, hd=16, hd_v=16, causal=0, scale=0.25, softcap=0.0, prefix=None, lengths=None)
    a.update(kw)
    lib = runtime.kernels()
    rules = [None, None, a["prefix"], a["lengths"]]
    sizes = [a[n] for n in ("dtype", "batch", "heads", "kv_heads", "t_q", "t_k", "hd", "hd_v", "causal", "scale", "softcap")]
    if backward:
        return lib.limn_hip_attend_bwd(at, FAKE, FAKE, *rules, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, *sizes, workspace, room, None)
    return lib.limn_hip_attend_fwd(at, FAKE, FAKE, *rules, FAKE, FAKE, *sizes, workspace, room, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize(
    "kw,code,message",
    [
        (dict(dtype=0), 2, "float32, float16 or bfloat16"),
        (dict(batch=0), 1, "positive"),
        (dict(t_k=0), 1, "positive"),
        (dict(kv_heads=3), 1, "evenly"),
        (dict(t_q=9, causal=1), 1, "last of the keys"),
        (dict(t_q=9, lengths=FAKE), 1, "last of the keys"),
        (dict(scale=float("nan")), 1, "scale"),
        (dict(softcap=-2.0), 1, "softcap"),
        (dict(softcap=float("inf")), 1, "softcap"),
        (dict(prefix=FAKE), 1, "not causal"),
        (dict(hd=257), 2, "head dims"),
        (dict(t_k=1 << 31, t_q=1), 2, "out of range"),
        (dict(at=None), 1, "null"),
        (dict(at=ctypes.c_void_p(0x1001)), 1, "aligned"),
        (dict(lengths=ctypes.c_void_p(0x1002)), 1, "aligned"),
        (dict(room=-1), 1, "workspace"),
    ],
)
def test_the_abi_refuses_with_a_reason(backward, kw, code, message):
    assert call(backward, **kw) == code
    assert message in runtime.kernels().limn_hip_last_error().decode()


def test_the_abi_asks_for_its_workspace():
    lib = runtime.kernels()
    need = lib.limn_hip_attend_workspace(1, 2, 4, 2, 8, 8, 16, 16, 1)
    assert need >= 2 * 4 * 8 * 4
    for ws, room in ((None, need), (FAKE, need - 1), (ctypes.c_void_p(0x1008), need)):
        assert call(True, workspace=ws, room=room) == 1
        assert "workspace" in lib.limn_hip_last_error().decode()
    assert lib.limn_hip_attend_workspace(0, 2, 4, 2, 8, 8, 16, 16, 1) == 0  # no kernel
