"""The 4-bit KV cache where its arguments, lengths and values are extreme, in both attention kernels (a call whose
rows x group pass 255 goes to the one for prompts).  Bars as in test_kvcache_gpu.py.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kvcache as ok
from tests.test_kvcache_gpu import Case, bits, ctx, torch, value  # noqa: F401

pytestmark = pytest.mark.gpu

INT_MAX = 2**31 - 1


# --------------------------------------------------- windows, empty rows --
@pytest.mark.parametrize("window", [INT_MAX, INT_MAX - 1, 2**30, 301])
@pytest.mark.parametrize("sinks", [0, 3, INT_MAX])
@pytest.mark.parametrize("qs", [None, [3, 8, 2, 40, 5], [3, 100, 2, 40, 200]])
def test_windows_past_every_length(torch, ctx, window, sinks, qs):  # noqa: F811
    """The largest windows hide nothing, also beside idle slots and sequences with more rows than tokens."""
    c = Case(torch, ctx, 64, 2, 16, [0, 5, 0, 300, 150], qs, seed=21)
    c.check(8, window=window, sinks=sinks)


# ------------------------------------------------------------ magnitudes --
DECODE, PROMPT = [None, [50, 5]], [[100, 5]]       # with four heads a kv head


def values_up_to_the_largest(torch, ctx, qs):  # noqa: F811
    """Scales of values past 2^122, which append stores as finite groups."""
    c = Case(torch, ctx, 64, 2, 32, [150, 105], qs, seed=22, v_scale=5e37)
    assert (c.pool.part("v")[1][c.layer, c.table[0, 0], :, :, :, 0] >> 7).max() >= 127 + 122
    c.check(8)


@pytest.mark.parametrize("qs", DECODE)
def test_values_up_to_the_largest(torch, ctx, qs):  # noqa: F811
    values_up_to_the_largest(torch, ctx, qs)


def test_large_values_over_many_partial_results(torch, ctx):  # noqa: F811
    """As many chunks of a row as are joined in two steps."""
    c = Case(torch, ctx, 64, 1, 128, [9001], seed=30, v_scale=5e37, layers=1)
    c.layer = 0
    c.check(4)
