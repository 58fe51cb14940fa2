"""The paged 8-bit cache over batches whose numbers lead outside: every sequence whose own
numbers fit gets its result, whatever stands in front of it, and nothing else is written."""
import numpy as np
import pytest

import serving_oracle as S
from test_gpu_kv8 import NP, Setup, same

pytestmark = pytest.mark.gpu


def _reported(llmrs, ctx, word):
    with pytest.raises(llmrs.LlmrsError) as e:
        ctx.sync()
    assert e.value.code == llmrs.EDEVICE and "word %d" % word in str(e.value)
    ctx.sync()  # reported once


def _fits(t, s):
    """Whether sequence s's rows lie inside the packed rows and its positions inside the tables."""
    a, b, length = int(t.row_start[s]), int(t.row_start[s + 1]), int(t.lens[s])
    reach = min(t.table.shape[1] * t.page, t.cos.shape[0])
    return 0 <= a < b <= t.n_rows and length >= 0 and length + b - a <= reach


def _check_all(llmrs, ctx, be, t, word):
    """Append, then attend, against the numpy forms of the sequences that fit."""
    (k, kx), (v, vx), (q, qx) = t.rows("k"), t.rows("v"), t.rows("q")
    be.kv8_append(t.cache, t.batch, k, v, t.g_cos, t.g_sin)
    _reported(llmrs, ctx, word)
    fit = [s for s in range(len(t.lens)) if _fits(t, s)]
    for s in fit:
        S.append(t.pool, t.row_start[s:s + 2], t.lens[s:s + 1], t.table[s:s + 1], kx, vx, t.cos, t.sin)
    same(t.download(), t.pool)
    out = llmrs.DeviceTensor.from_numpy(ctx, np.full((t.n_rows, t.heads * t.d), 77, NP[t.dtype]))
    ws = be.kv8_attention_workspace(t.cache, t.batch, t.heads, t.n_rows)
    be.kv8_attention(t.cache, t.batch, q, out, t.g_cos, t.g_sin, workspace=ws)
    _reported(llmrs, ctx, word)
    got, mine = out.numpy(), np.zeros(t.n_rows, bool)
    for s in fit:
        a, b = int(t.row_start[s]), int(t.row_start[s + 1])
        mine[a:b] = True
        ref, *pieces = [x[a:b] for x in S.attend(t.pool, t.row_start[s:s + 2], t.lens[s:s + 1], t.table[s:s + 1], qx,
                                                 t.n_rows, t.cos, t.sin)]
        off = np.abs(S.from_type(got)[a:b].reshape(ref.shape) - ref)
        assert np.all(off <= S.attend_tolerance(t.dtype, ref, *pieces, t.d)), s
    assert np.all(got[~mine] == 77)  # nobody's rows stay as they were


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [[2, 2, 1], [150, 60, 40]])  # both kernels' kinds of sequences
@pytest.mark.parametrize("change", [dict(lens=(0, -1)), dict(lens=(0, 10 ** 6)), dict(lens=(1, 2 ** 31 - 1)),
                                    dict(rows=(3, 10 ** 6)), dict(rows=(1, -5)), dict(rows=(1, 10 ** 6))])
def test_the_others_of_a_bad_batch(llmrs, ctx, be, change, rows, dtype):
    t = Setup(llmrs, ctx, 90, [20, 5, 9], rows, 4, 1, 64, 16, dtype)
    for name, (i, value) in change.items():
        {"lens": t.lens, "rows": t.row_start}[name][i] = value
    t.upload()
    _check_all(llmrs, ctx, be, t, 5)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_row_starts_that_fall(llmrs, ctx, be, dtype):
    """The first two sequences lead outside, the third one's many rows lie at [4, 300): its queries
    are its own, not those that an earlier call left in the workspace."""
    t = Setup(llmrs, ctx, 91, [5, 9, 20], [4, 0, 296], 8, 2, 64, 32, dtype)
    t.row_start = np.int32([0, 100000, 4, 300])
    t.upload()
    _check_all(llmrs, ctx, be, t, 5)
    q, _ = t.rows("q")
    ws = be.kv8_attention_workspace(t.cache, t.batch, t.heads, t.n_rows)
    first = be.kv8_attention(t.cache, t.batch, q, rope_cos=t.g_cos, rope_sin=t.g_sin, workspace=ws).numpy()[4:300]
    _reported(llmrs, ctx, 5)
    for fill in (0, 0x3C):  # whatever the workspace held
        old = np.full(ws.shape, fill, np.uint8)
        ws = llmrs.DeviceTensor.from_numpy(ctx, old)
        again = be.kv8_attention(t.cache, t.batch, q, rope_cos=t.g_cos, rope_sin=t.g_sin, workspace=ws).numpy()[4:300]
        _reported(llmrs, ctx, 5)
        assert np.array_equal(first.view(np.uint8), again.view(np.uint8))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gone", [[1], [0, 4], None])  # pages of sequence 0 (None: all)
def test_many_rows_without_some_pages(llmrs, ctx, be, gone, dtype):
    t = Setup(llmrs, ctx, 92, [200, 5], [150, 150], 8, 2, 128, 64, dtype)
    t.table[0, slice(None) if gone is None else gone] = -1
    t.upload()
    got, (ref, *pieces) = t.attend(be)
    _reported(llmrs, ctx, 6)
    assert np.all(np.abs(got - ref) <= S.attend_tolerance(dtype, ref, *pieces, t.d))
    if gone is None:
        assert np.all(got[:150] == 0) and np.all(ref[:150] == 0)
