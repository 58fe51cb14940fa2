"""The paged 8-bit cache in batches of more sequences than a CTA has threads, batches that a warp
or four to a page append, and pages whose scale grows in a decode step."""
import numpy as np
import pytest

import serving_oracle as S
from test_gpu_kv8 import Setup, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("seqs", [300, 1700])  # past 256 threads, and past twice 768
def test_attend_many_rows_in_many_sequences(llmrs, ctx, be, seqs, dtype):
    """Sequences of no, few and many rows side by side, many rows first and last."""
    rng = np.random.default_rng(100 + seqs)
    lens = rng.integers(0, 60, seqs).tolist()
    rows = np.where(rng.random(seqs) < 0.04, rng.integers(13, 80, seqs), rng.integers(0, 3, seqs))
    rows[[0, -1]] = 40
    Setup(llmrs, ctx, 101, lens, rows.tolist(), 4, 1, 64, 16, dtype).check_attend(be)


@pytest.mark.parametrize("page,d", [(128, 128), (128, 64), (64, 128), (16, 64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_grows_the_scale_of_full_pages(llmrs, ctx, be, page, d, dtype):
    """One new row to a sequence, behind up to a page's other tokens: their codes are rounded again."""
    lens = [page - 1, page - 2, 1, 3 * page - 1, page // 2, 2 * page - 1, page, 0]
    t = Setup(llmrs, ctx, 102, lens, [1] * len(lens), 3, 3, d, page, dtype)
    (_, kx), (_, vx) = t.rows("k"), t.rows("v")
    old = {n: t.pool[n].copy() for n in ("ks", "vs")}
    for gain in (8.0, 64.0, 0.5):  # it grows, grows again, and stays
        (k, kg), (v, vg) = ((llmrs.DeviceTensor.from_numpy(ctx, a.reshape(t.n_rows, -1)), S.from_type(a)) for a, _ in
                            (S.to_type(x * np.float32(gain), dtype) for x in (kx, vx)))
        be.kv8_append(t.cache, t.batch, k, v, t.g_cos, t.g_sin)
        S.append(t.pool, t.row_start, t.lens, t.table, kg, vg, t.cos, t.sin)
        same(t.download(), t.pool)
    ctx.sync()
    held = [t.table[s, n // page] for s, n in enumerate(lens) if n % page]
    assert all(np.all(t.pool[n][held] > 4 * old[n][held]) for n in old)


@pytest.mark.parametrize("seqs,most,kv,d,page,dtype", [
    (150, 60, 8, 128, 64, "f32"), (150, 60, 8, 64, 16, "bf16"), (60, 12, 8, 128, 128, "f16"), (20, 12, 2, 128, 32, "f32")])
def test_append_a_few_rows_to_many_sequences(llmrs, ctx, be, seqs, most, kv, d, page, dtype):
    """Up to `most` rows each, on both sides of where four warps take over from one."""
    rng = np.random.default_rng(103)
    lens, rows = rng.integers(0, 90, seqs).tolist(), rng.integers(0, most + 1, seqs).tolist()
    t = Setup(llmrs, ctx, 103, lens, rows, kv, kv, d, page, dtype)
    (k, kx), (v, vx) = t.rows("k"), t.rows("v")
    be.kv8_append(t.cache, t.batch, k, v, t.g_cos, t.g_sin)
    ctx.sync()
    S.append(t.pool, t.row_start, t.lens, t.table, kx, vx, t.cos, t.sin)
    same(t.download(), t.pool)
