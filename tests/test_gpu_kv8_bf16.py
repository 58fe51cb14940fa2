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
