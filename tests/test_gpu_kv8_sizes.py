"""The serving operators at the ends of their sizes: nothing to do, many query heads to a KV
head, pools past 4 GB."""
import numpy as np
import pytest

import serving_oracle as S
from test_gpu_kv8 import Setup, same

pytestmark = pytest.mark.gpu


def test_nothing_to_do(llmrs, ctx, be):
    """No sequences, sequences without rows, no rows at all: nothing is written but the counts."""
    t = Setup(llmrs, ctx, 120, [20, 5, 0], [0, 0, 0], 4, 2, 64, 16, "f32", spare_rows=3)
    before = t.download()
    (k, _), (v, _) = t.rows("k"), t.rows("v")
    t.attend(be)  # the rows are all spare ones, and stay as they were
    be.kv8_append(t.cache, t.batch, k, v, t.g_cos, t.g_sin)
    D = llmrs.DeviceTensor
    none = llmrs.SeqBatch(D.from_numpy(ctx, np.zeros(1, np.int32)), D(ctx, (0,), np.int32), D(ctx, (0, 4), np.int32))
    q, out = t.rows("q")[0], D.from_numpy(ctx, np.full((t.n_rows, 256), 77, np.float32))
    for batch, rows in ((none, slice(None)), (t.batch, slice(0, 0)), (none, slice(0, 0))):
        n = len(range(t.n_rows)[rows])
        cut = lambda x, w: x if n else D(ctx, (0, w))  # noqa: E731
        be.kv8_append(t.cache, batch, cut(k, 128), cut(v, 128), t.g_cos, t.g_sin)
        ws = be.kv8_attention_workspace(t.cache, batch, 4, n)
        be.kv8_attention(t.cache, batch, cut(q, 256), cut(out, 256), t.g_cos, t.g_sin, workspace=ws)
    be.kv8_read(t.cache, D(ctx, (0,), np.int32), D(ctx, (0, 2, 16, 64)), D(ctx, (0, 2, 16, 64)))
    ctx.sync()
    same(t.download(), before)
    assert np.all(out.numpy() == 77)
    accepted = D.from_numpy(ctx, np.full(2, 777, np.int32))
    be.verify_draft(D(ctx, (0, 50)), D.from_numpy(ctx, np.zeros(3, np.int32)), None, None, D(ctx, (0,)), D(ctx, (0,), np.int32),
                    accepted, workspace=be.verify_draft_workspace(0, 50))
    be.verify_draft(D(ctx, (0, 50)), D.from_numpy(ctx, np.zeros(1, np.int32)), None, None, D(ctx, (0,)), D(ctx, (0,), np.int32),
                    D(ctx, (0,), np.int32))
    ctx.sync()
    assert np.all(accepted.numpy() == 0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv", [(128, 1), (130, 1), (300, 2)])  # a row fills a tile of 128 vectors, or does not fit it
@pytest.mark.parametrize("rows", [[1, 1, 1], [2, 0, 5], [40, 3, 1]])
def test_attend_many_query_heads_to_a_kv_head(llmrs, ctx, be, heads, kv, rows, dtype):
    Setup(llmrs, ctx, 121, [100, 0, 333], rows, heads, kv, 64, 32, dtype).check_attend(be)


@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 200, 90]])
def test_pages_past_four_gigabytes(llmrs, ctx, be, rows):
    """The same pages at the start of a pool and behind its first 4.6 GB."""
    import torch
    t = Setup(llmrs, ctx, 122, [100, 0, 700], rows, 8, 1, 128, 64, "f32")
    first = 560_000  # 8192 bytes a page and pool
    n = first + t.pages
    big = {k: torch.zeros((n,) + v.shape[1:], dtype=torch.int8 if v.dtype == np.int8 else torch.float32, device="cuda")
           for k, v in t.pool.items()}
    for k, v in t.pool.items():
        big[k][first:] = torch.from_numpy(v).cuda()
    torch.cuda.synchronize()
    t.cache = llmrs.Kv8Cache(ctx, n, 64, 1, 128, k_codes=big["kq"], v_codes=big["vq"], k_scales=big["ks"], v_scales=big["vs"])
    t.batch = llmrs.SeqBatch(t.g_rs, t.g_lens, llmrs.DeviceTensor.from_numpy(ctx, np.where(t.table >= 0, t.table + first, -1).astype(np.int32)))
    (k, kx), (v, vx) = t.rows("k"), t.rows("v")
    be.kv8_append(t.cache, t.batch, k, v, t.g_cos, t.g_sin)
    S.append(t.pool, t.row_start, t.lens, t.table, kx, vx, t.cos, t.sin)
    t.check_attend(be)
    ids = t.table[2, :3]
    pages = llmrs.DeviceTensor.from_numpy(ctx, (ids + first).astype(np.int32))
    k_out, v_out = (llmrs.DeviceTensor(ctx, (3, 1, 64, 128)) for _ in range(2))
    be.kv8_read(t.cache, pages, k_out, v_out)
    for got, codes, scales in ((k_out, "kq", "ks"), (v_out, "vq", "vs")):
        assert np.array_equal(got.numpy(), t.pool[codes][ids].astype(np.float32) * t.pool[scales][ids][:, :, None, None])
    ctx.sync()
    same({k: x[first:].cpu().numpy() for k, x in big.items()}, t.pool)
    assert all(not x[:first].any() for x in big.values())  # nothing at the places that 32 bits would have reached
