"""Calls of attend_paged, sample, quantize_rows and int8_linear whose launches HIP would not take (2^32 threads and more) are refused by
their sizes, before anything is launched: the pointers are never read."""

from __future__ import annotations

import pytest

from limn_amd.hip import runtime
from test_serving import call

GENERAL = dict(hd=33, heads=1, kv_heads=1, q_row=33, k_row=33, v_row=33)  # a head dim of the general kernels
FAST = dict(heads=64, kv_heads=64, q_row=1024, k_row=1024, v_row=1024, table_pages=1)


@pytest.mark.parametrize(
    "entry,kw",
    [
        ("paged", dict(GENERAL, tokens=1 << 24)),  # a workgroup a token writes the cache first
        ("paged", dict(GENERAL, tokens=1 << 20, heads=64, q_row=64 * 33)),
        ("paged", dict(FAST, tokens=1 << 20, sequences=1 << 20)),  # a token a sequence
        ("paged", dict(FAST, dtype=3, tokens=(1 << 20) + 64, sequences=1 << 20)),  # more of them: tiles of 128 rows
        ("sample", dict(rows=1 << 24, vocab=256, stride=256)),
        ("sample", dict(rows=1 << 22, vocab=257, stride=257)),
        ("quantize", dict(rows=1 << 24)),
        ("int8", dict(rows=1 << 24)),
        ("int8", dict(rows=(1 << 24) - 3, width=9, outputs=5)),  # with the copy of the weight's rows beside them
        ("int8", dict(rows=3, width=16, outputs=1 << 28)),
        ("int8", dict(rows=1 << 21, width=16, outputs=1 << 19)),
    ],
    ids=str,
)
def test_launches_past_32_bits_of_threads(entry, kw):
    assert call(entry, room=1 << 60, **kw) == 2
    assert "out of range" in runtime.kernels().limn_hip_last_error().decode()
