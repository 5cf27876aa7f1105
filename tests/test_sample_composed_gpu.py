"""sample's composed form on the hip device (float64 logits): rows of NaN and infinities, every kind of setting, against the oracle."""

from __future__ import annotations

import numpy as np
import pytest

from conftest import upload
from limn_amd.sampling import sample
from limn_amd.seam import Tensor, float32, float64, int32, realize, use_device
from oracle.attend import within
from oracle.serving import sample as oracle

pytestmark = pytest.mark.gpu
KINDS = dict(temperature=float32, top_k=int32, top_p=float32, min_p=float32)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=0.4, top_k=5, top_p=0.9, min_p=0.01), dict(temperature=0.0)], ids=str)
def test_float64_logits(hipdev, kw):
    use_device(hipdev)
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((14, 23)) * 2.5
    logits[0], logits[1], logits[2, 5:], logits[4] = -np.inf, np.nan, -np.inf, np.finfo(np.float64).min
    logits[5, [3, 20]], logits[6, ::2], logits[10, ::3], logits[10, 7] = np.inf, np.nan, np.nan, np.inf
    u = np.concatenate([rng.random(11), [1.0, np.nan, -2.0]]).astype(np.float32)
    on = lambda a, kind: Tensor.from_node(upload(hipdev, a, kind))  # noqa: E731
    rules = {n: np.full(14, r, np.int32 if n == "top_k" else np.float32) for n, r in kw.items()}
    got = sample(on(logits, float64), on(u, float32), **{n: on(r, KINDS[n]) for n, r in rules.items()})
    realize(*got)
    want, (lp, bound) = oracle(logits, u, **rules)
    np.testing.assert_array_equal(got[0].numpy(), want)
    within(got[1].numpy(), lp, bound, "logprob")
