"""The paged KV cache at its edges: many heads a group, extreme values, lengths
that fall, destroyed streams.  Formulas and tolerances as in
tests/test_gpu_paged.py.
"""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.test_gpu_paged import BF16, F16, F32, handle, near, reported, run, sess  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads", [71, 128, 130])
@pytest.mark.parametrize("new,past,window,shared", [
    ([1], [200], 0, 0), ([40, 1, 3], [5, 300, 0], 0, 0), ([7, 1], [300, 400], 0, 257),
    ([90], [30], 50, 0)])
def test_more_heads_than_a_tile_has_rows(sess, heads, new, past, window, shared, dtype):
    """All query heads on one KV head: a token's heads lie in several tiles of 16 rows."""
    s = ref.make(30, dtype, new, past, heads, 1, 64, 16, shared)
    want = ref.attention(s, new, past, heads, window=window)
    near(want, run(sess, s, heads, new, local_window_size=window, shared_len=shared))
