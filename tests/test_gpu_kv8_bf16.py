"""bf16 rows over the paged 8-bit cache: the rotated queries, which need more bits than bf16 or
f16 have, are not rounded to either."""
import numpy as np
import pytest

import serving_oracle as S
from test_gpu_kv8 import Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,d,page", [(8, 2, 128, 64), (16, 1, 128, 32), (8, 2, 64, 64), (32, 2, 64, 16)])
@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [1, 5, 3, 2], [150, 60, 1, 200]])
def test_attend_sharp_bf16_rows(llmrs, ctx, be, heads, kv, d, page, rows):
    """Scores of some tens, where a query rounded to 11 bits moves the probabilities by 1 %.  What is
    rounded: the probabilities to f16 (2^-11 of each, so 2^-11 sum p|v| at the most) and the result
    (2^-8); everything else has the f32 rows' tolerance."""
    t = Setup(llmrs, ctx, 130, [300, 1000, 37, 5], rows, heads, kv, d, page, "bf16", sharp=10.0)
    got, (ref, *pieces) = t.attend(be)
    tol = S.attend_tolerance("f32", ref, *pieces, d) + 2.0 ** -11 * pieces[0] + 2.0 ** -8 * np.abs(ref)
    off = np.abs(got - ref)
    assert np.all(off <= tol), (float((off / tol).max()), float((off > tol).mean()))
    # in 2-norm the result's own rounding is nearly all of it
    rounded = np.linalg.norm(S.bf16_value(S.bf16_bits(ref)) - ref)
    assert np.linalg.norm(got - ref) <= 1.02 * rounded


@pytest.mark.parametrize("heads,kv,d,page", [(8, 2, 128, 64), (16, 1, 64, 16)])
@pytest.mark.parametrize("rows", [1, 90])
def test_a_row_that_sees_one_token_gives_its_value(llmrs, ctx, be, heads, kv, d, page, rows):
    """The first row of a prompt has one probability, of 1: the result is the token's value, rounded
    to bf16 once.  What is on the way in f32 (a few roundings of 2^-24) can move it to the other side
    of a tie, which lies that near for one value in 2^13 or less."""
    t = Setup(llmrs, ctx, 131, [0] * 8, [rows] * 8, heads, kv, d, page, "bf16")
    got, (ref, *_) = t.attend(be)
    first = np.arange(8) * rows
    assert (got[first] != S.bf16_value(S.bf16_bits(ref[first]))).mean() < 1e-3


@pytest.mark.parametrize("rows", [1, 5, 150])
@pytest.mark.parametrize("low,high", [(-6, 4), (-37, 32)])
def test_attend_bf16_value_scales_far_apart(llmrs, ctx, be, rows, low, high):
    """Zero scales among them.  As for f32 rows (a probability with its scale, or without it, is held in
    steps of 2^-24 where the row's largest is 2^12 at the least: off by 2^-37 of that largest, which
    the row's largest sum p|v| is not below, and times codes of at most 127), with the probabilities'
    2^-11 and the result's 2^-8."""
    t = Setup(llmrs, ctx, 132, [500, 77], [rows, rows], 8, 2, 128, 16, "bf16", sharp=4.0)
    rng = np.random.default_rng(133)
    vs = (np.float64(10.0) ** rng.integers(low, high + 1, t.pool["vs"].shape) * rng.uniform(1, 2, t.pool["vs"].shape))
    t.pool["vs"] = np.where(rng.random(vs.shape) < 0.2, 0, vs).astype(np.float32)
    t.upload()
    got, (ref, *pieces) = t.attend(be)
    tol = S.attend_tolerance("f32", ref, *pieces, 128) + 2.0 ** -11 * pieces[0] + 2.0 ** -8 * np.abs(ref)
    tol += 127 * pieces[4][:, None, None] * 2.0 ** -37 * pieces[0].max(axis=2, keepdims=True)
    off = np.abs(got - ref)
    assert np.all(off <= tol), float((off / tol).max())
