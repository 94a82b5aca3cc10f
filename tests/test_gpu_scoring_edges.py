"""The scoring operators at the ends of what their documentation allows: labels that are no class, gradients and scores of extreme
size, several errors at once, arrays without cells, other libraries' captures."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from snekmer_amd import _hip, apply, engine
from test_gpu_scoring import HALF_STEP, SMALLEST, U, block, check_logp, plain_logp, rounded, values, whole_numbers

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = _hip.Context(0)
    yield c
    c.close()


# ---------------------------------------------------------------------------- labels that are no class
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("a", [1, 50, 1023, 1025, 2500])
def test_gradient_of_rows_with_wrong_labels(ctx, a, masked, dt):
    """Labels from the row's end to the end of its last tile and far behind it, in every row and the last one: NaN for the row's classes,
    0 where a class is not allowed, the other rows as without them."""
    rng = np.random.default_rng(a)
    end = -(-a // 1024) * 1024
    wrong = [a, a + 1, end - 1, end, end + 7, -2, 2 ** 31 - 1, 2 ** 32 + 3, 2 ** 62]
    labels = np.concatenate([[v, i % a] for i, v in enumerate(wrong)] + [[a]]).astype(np.int64)
    n = labels.size
    words, s = rounded(block("normal", n, a, a), dt)
    mask = (rng.random((n, a)) < 0.7).astype(np.uint8) if masked else None
    right = np.where((labels >= 0) & (labels < a), labels, -1)
    d, dm = ctx.to_device(words), None if mask is None else ctx.to_device(mask)
    ones = ctx.to_device(np.ones(n, np.float32))
    fwd = apply.log_probabilities(ctx, d, right, mask=dm)
    want = values(apply.log_probabilities_backward(ctx, d, right, fwd, d_logp=ones, mask=dm).download(), dt)
    got = apply.log_probabilities_backward(ctx, d, ctx.to_device(labels), fwd, d_logp=ones, mask=dm)
    with pytest.raises(_hip.HipError, match="label outside"):
        ctx.sync()
    got = values(got.download(), dt)
    allowed = np.ones((n, a), bool) if mask is None else mask != 0
    bad = right != labels
    assert np.isnan(got[bad][allowed[bad]]).all() and (got[bad][~allowed[bad]] == 0).all()
    assert np.array_equal(got[~bad], want[~bad])
