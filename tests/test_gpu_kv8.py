"""The paged 8-bit cache on the GPU: codes and scales bit for bit against the numpy
form, attention against 64 bits (tolerances: serving_oracle.attend_tolerance)."""
import numpy as np
import pytest

import serving_oracle as S

pytestmark = pytest.mark.gpu

NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


class Setup:
    """A ragged batch over a pool with pages in no order; pages that no sequence uses hold
    NaN scales, and rows behind the last sequence NaN."""

    def __init__(self, llmrs, ctx, seed, lens, rows, heads, kv, d, page, dtype, spare_rows=2, sharp=1.0):
        rng = np.random.default_rng(seed)
        self.llmrs, self.ctx, self.dtype = llmrs, ctx, dtype
        self.heads, self.kv, self.d, self.page = heads, kv, d, page
        need = [max(1, -(-(l + r) // page)) for l, r in zip(lens, rows)]
        self.pages = sum(need) + 3
        order = rng.permutation(self.pages)
        self.table = np.full((len(lens), max(need) + 1), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.lens = np.int32(lens)
        self.row_start = np.int32(np.concatenate([[0], np.cumsum(rows)]))
        self.n_rows = int(self.row_start[-1]) + spare_rows
        shape = (self.pages, kv, page, d)
        self.pool = {"kq": np.clip(np.rint(rng.normal(0, 36, shape)), -127, 127).astype(np.int8),
                     "vq": np.clip(np.rint(rng.normal(0, 36, shape)), -127, 127).astype(np.int8),
                     "ks": (0.028 * np.exp(0.4 * rng.normal(0, 1, shape[:2]))).astype(np.float32),
                     "vs": (0.028 * np.exp(0.4 * rng.normal(0, 1, shape[:2]))).astype(np.float32)}
        for x in ("ks", "vs"):
            self.pool[x][order[at:]] = np.nan
        qkv = rng.normal(0, 1, (self.n_rows, (heads + 2 * kv) * d)).astype(np.float32)
        qkv[:, :heads * d] *= sharp
        qkv[int(self.row_start[-1]):] = np.nan
        self.raw, self.qkv = S.to_type(qkv, dtype)
        self.cos, self.sin = llmrs.rope_table(d, max(1, int(max(l + r for l, r in zip(lens, rows)))))
        self.upload()

    def upload(self):
        T = self.llmrs.DeviceTensor.from_numpy
        self.g = {k: T(self.ctx, v) for k, v in self.pool.items()}
        self.cache = self.llmrs.Kv8Cache(self.ctx, self.pages, self.page, self.kv, self.d, k_codes=self.g["kq"],
                                         v_codes=self.g["vq"], k_scales=self.g["ks"], v_scales=self.g["vs"])
        self.g_rs, self.g_lens, self.g_table = T(self.ctx, self.row_start), T(self.ctx, self.lens), T(self.ctx, self.table)
        self.batch = self.llmrs.SeqBatch(self.g_rs, self.g_lens, self.g_table)
        self.g_cos, self.g_sin = T(self.ctx, self.cos), T(self.ctx, self.sin)

    def rows(self, name):
        h, k = self.heads * self.d, self.kv * self.d
        a, b = {"q": (0, h), "k": (h, h + k), "v": (h + k, h + 2 * k)}[name]
        return self.llmrs.DeviceTensor.from_numpy(self.ctx, np.ascontiguousarray(self.raw[:, a:b])), \
            np.ascontiguousarray(self.qkv[:, a:b]).reshape(self.n_rows, -1, self.d)

    def download(self):
        return {k: v.numpy() for k, v in self.g.items()}

    def attend(self, be, scale=None, rope=True):
        q, qv = self.rows("q")
        out = self.llmrs.DeviceTensor.from_numpy(self.ctx, np.full((self.n_rows, self.heads * self.d), 77, NP[self.dtype]))
        ws = be.kv8_attention_workspace(self.cache, self.batch, self.heads, self.n_rows)
        tables = (self.g_cos, self.g_sin) if rope else (None, None)
        be.kv8_attention(self.cache, self.batch, q, out, *tables, scale=scale, workspace=ws)
        got = out.numpy()
        used = int(self.row_start[-1])
        assert np.all(got[used:] == 77)  # rows behind the last sequence stay as they were
        ref = S.attend(self.pool, self.row_start, self.lens, self.table, qv, self.n_rows,
                       *((self.cos, self.sin) if rope else (None, None)), scale=scale)
        return S.from_type(got)[:used].reshape(used, self.heads, self.d), [x[:used] for x in ref]

    def check_attend(self, be, **kw):
        got, (ref, *pieces) = self.attend(be, **kw)
        tol = S.attend_tolerance(self.dtype, ref, *pieces, self.d)
        off = np.abs(got - ref)
        assert np.all(off <= tol), (float((off / tol).max()), np.argwhere(~(off <= tol))[:4].tolist())


def same(got, want):
    for k in want:
        assert np.array_equal(got[k], want[k], equal_nan=got[k].dtype == np.float32), k


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("page,d,kv,dtype", [(16, 64, 1, "f32"), (32, 128, 3, "bf16"), (64, 128, 8, "f32"),
                                             (64, 64, 2, "f16"), (128, 128, 2, "bf16"), (128, 64, 4, "f32")])
def test_append_bit_exact(llmrs, ctx, be, page, d, kv, dtype):
    lens = [0, 5, page - 1, page, 3 * page + 7, 2, 300]
    rows = [1, 0, 2, 1, 2 * page + 3, page, 1]
    t = Setup(llmrs, ctx, 1, lens, rows, kv, kv, d, page, dtype)
    (k, kx), (v, vx) = t.rows("k"), t.rows("v")
    be.kv8_append(t.cache, t.batch, k, v, t.g_cos, t.g_sin)
    ctx.sync()  # the NaN rows behind the last sequence are not read
    S.append(t.pool, t.row_start, t.lens, t.table, kx, vx, t.cos, t.sin)
    same(t.download(), t.pool)


def test_append_many_sequences_and_growing_scale(llmrs, ctx, be):
    """600 sequences (several rounds of the batch search), row by row with magnitudes that grow
    and shrink; twice the same rows at the same places changes nothing."""
    rng = np.random.default_rng(9)
    lens, rows = rng.integers(0, 40, 600).tolist(), rng.integers(0, 3, 600).tolist()
    t = Setup(llmrs, ctx, 2, lens, rows, 1, 1, 64, 16, "f32")
    (k, kx), (v, vx) = t.rows("k"), t.rows("v")
    gain = np.float32(4.0) ** rng.integers(-3, 4, (t.n_rows, 1, 1)).astype(np.float32)
    kx, vx = kx * gain, vx * gain
    k = llmrs.DeviceTensor.from_numpy(ctx, kx.reshape(t.n_rows, -1))
    v = llmrs.DeviceTensor.from_numpy(ctx, vx.reshape(t.n_rows, -1))
    S.append(t.pool, t.row_start, t.lens, t.table, kx, vx, t.cos, t.sin)
    for _ in range(2):
        be.kv8_append(t.cache, t.batch, k, v, t.g_cos, t.g_sin)
        same(t.download(), t.pool)


def test_append_without_rotation_zero_and_tiny_rows(llmrs, ctx, be):
    t = Setup(llmrs, ctx, 3, [0, 10, 20], [5, 3, 40], 2, 2, 64, 32, "f32")
    (_, kx), (_, vx) = t.rows("k"), t.rows("v")
    kx, vx = kx.copy(), vx.copy()
    kx[:5] = 0.0           # an all-zero page: scale 0
    vx[:5] = 1e-41         # below the smallest normal scale: zero
    kx[8:] *= np.float32(1e30)
    k = llmrs.DeviceTensor.from_numpy(ctx, kx.reshape(t.n_rows, -1))
    v = llmrs.DeviceTensor.from_numpy(ctx, vx.reshape(t.n_rows, -1))
    be.kv8_append(t.cache, t.batch, k, v)
    ctx.sync()
    S.append(t.pool, t.row_start, t.lens, t.table, kx, vx)
    same(t.download(), t.pool)
    at = t.table[0, 0]
    assert np.all(t.pool["ks"][at] == 0) and np.all(t.pool["vs"][at] == 0)


def _reported(llmrs, ctx, word):
    with pytest.raises(llmrs.LlmrsError) as e:
        ctx.sync()
    assert e.value.code == llmrs.EDEVICE and "word %d" % word in str(e.value)
    ctx.sync()  # reported once


def test_append_reports_what_it_cannot_store(llmrs, ctx, be):
    t = Setup(llmrs, ctx, 4, [3, 0], [2, 2], 1, 1, 64, 16, "f32")
    (_, kx), (v, vx) = t.rows("k"), t.rows("v")
    kx = kx.copy()
    kx[1, 0, 5], kx[2, 0, 40] = np.inf, np.nan
    k = llmrs.DeviceTensor.from_numpy(ctx, kx.reshape(t.n_rows, -1))
    be.kv8_append(t.cache, t.batch, k, v)
    _reported(llmrs, ctx, 7)
    S.append(t.pool, t.row_start, t.lens, t.table, kx, vx)
    same(t.download(), t.pool)


def test_bad_pages_and_batches_are_skipped_and_reported(llmrs, ctx, be):
    t = Setup(llmrs, ctx, 5, [40, 5, 9], [2, 2, 1], 4, 1, 64, 16, "f32")
    good = t.table.copy()
    for bad in (-1, t.pages, 2 ** 31 - 1):
        t.table = good.copy()
        t.table[0, 2] = bad  # positions 32..47 of sequence 0: its new rows' page
        t.upload()
        (k, kx), (v, vx) = t.rows("k"), t.rows("v")
        be.kv8_append(t.cache, t.batch, k, v, t.g_cos, t.g_sin)
        _reported(llmrs, ctx, 6)
        want = {n: x.copy() for n, x in t.pool.items()}
        S.append(want, [0, 2, 3], [5, 9], good[1:], kx[2:], vx[2:], t.cos, t.sin)  # the others' rows are stored
        same(t.download(), want)
        t.pool = want
        t.check_attend(be)  # its tokens are left out
        _reported(llmrs, ctx, 6)
    t.table = np.full_like(good, -1)
    t.table[1:] = good[1:]
    t.upload()
    got, (ref, *_) = t.attend(be)
    assert np.all(got[:2] == 0) and np.all(ref[:2] == 0)  # a row that sees nothing
    _reported(llmrs, ctx, 6)


@pytest.mark.parametrize("change", [dict(lens=(0, -1)), dict(lens=(0, 10 ** 6)), dict(lens=(1, 2 ** 31 - 1)),
                                    dict(rows=(3, 10 ** 6)), dict(rows=(1, -5))])
def test_sequences_that_lead_outside_count_as_empty(llmrs, ctx, be, change):
    t = Setup(llmrs, ctx, 6, [20, 5, 9], [2, 2, 1], 2, 2, 64, 16, "f32")
    for name, (i, value) in change.items():
        {"lens": t.lens, "rows": t.row_start}[name][i] = value
    t.upload()
    before = t.download()
    (k, _), (v, _), (q, _) = t.rows("k"), t.rows("v"), t.rows("q")
    be.kv8_append(t.cache, t.batch, k, v, t.g_cos, t.g_sin)
    _reported(llmrs, ctx, 5)
    assert np.array_equal(t.download()["kq"][t.table[0, 0]], before["kq"][t.table[0, 0]])
    out = llmrs.DeviceTensor.from_numpy(ctx, np.full((t.n_rows, 128), 77, np.float32))
    be.kv8_attention(t.cache, t.batch, q, out, t.g_cos, t.g_sin)
    _reported(llmrs, ctx, 5)


def test_read_gives_the_values(llmrs, ctx, be):
    t = Setup(llmrs, ctx, 7, [100], [1], 3, 3, 128, 64, "f32")
    ids = t.table[0, :2][[1, 0, 1]].copy()  # an id twice
    pages = llmrs.DeviceTensor.from_numpy(ctx, ids)
    for dtype in (np.float32, np.float16, np.uint16):
        k = llmrs.DeviceTensor(ctx, (3, 3, 64, 128), dtype)
        v = llmrs.DeviceTensor(ctx, (3, 3, 64, 128), dtype)
        be.kv8_read(t.cache, pages, k, v)
        for got, codes, scales in ((k, "kq", "ks"), (v, "vq", "vs")):
            want = t.pool[codes][ids].astype(np.float32) * t.pool[scales][ids][:, :, None, None]
            want = {np.float32: lambda x: x, np.float16: lambda x: x.astype(np.float16),
                    np.uint16: S.bf16_bits}[dtype](want)
            assert np.array_equal(got.numpy(), want)
    be.kv8_read(t.cache, llmrs.DeviceTensor.from_numpy(ctx, np.int32([t.pages])),
                llmrs.DeviceTensor(ctx, (1, 3, 64, 128)), llmrs.DeviceTensor(ctx, (1, 3, 64, 128)))
    _reported(llmrs, ctx, 6)


# ------------------------------------------------------------------ attention
LENS = {"tiny": ([0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65], 1), "long": ([1000, 4097, 127, 128, 2049], 1),
        "drafts": ([0, 700, 33, 64, 1500], 5)}


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", list(LENS))
@pytest.mark.parametrize("heads,kv,d,page", [(8, 2, 128, 64), (8, 2, 64, 64), (8, 1, 128, 16), (3, 3, 64, 32),
                                             (14, 2, 128, 128), (6, 3, 128, 32), (20, 1, 64, 128)])
def test_attend_few_rows(llmrs, ctx, be, dtype, kind, heads, kv, d, page):
    lens, most = LENS[kind]
    rows = [1 + i % most for i in range(len(lens))]
    rows[len(rows) // 2] = most
    Setup(llmrs, ctx, 11, lens, rows, heads, kv, d, page, dtype).check_attend(be)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,d,page,lens,rows", [
    (8, 2, 128, 64, [0], [300]), (8, 2, 64, 32, [0, 130, 7], [129, 1, 200]), (4, 4, 128, 16, [513, 0, 0], [257, 0, 33]),
    (7, 1, 64, 128, [1000, 3], [65, 128]), (16, 2, 128, 128, [100, 0, 250, 64], [64, 77, 1, 190]),
    (40, 1, 128, 64, [60], [50])])
def test_attend_many_rows(llmrs, ctx, be, dtype, heads, kv, d, page, lens, rows):
    Setup(llmrs, ctx, 12, lens, rows, heads, kv, d, page, dtype).check_attend(be)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_many_sequences(llmrs, ctx, be, dtype):
    rng = np.random.default_rng(13)
    lens, rows = rng.integers(0, 90, 700).tolist(), rng.integers(0, 3, 700).tolist()
    Setup(llmrs, ctx, 13, lens, rows, 4, 1, 64, 16, dtype).check_attend(be)


@pytest.mark.parametrize("rows", [1, 150])
def test_attend_sharp_scaled_and_unrotated(llmrs, ctx, be, rows):
    t = Setup(llmrs, ctx, 14, [900, 20], [rows, rows], 8, 2, 128, 64, "f32", sharp=12.0)
    t.check_attend(be)
    t.check_attend(be, scale=0.01, rope=False)
    t.check_attend(be, scale=1.0, rope=False)


@pytest.mark.parametrize("rows", [1, 140])
@pytest.mark.parametrize("page", [16, 64])
def test_attend_scales_far_apart(llmrs, ctx, be, rows, page):
    """Value scales over ten orders of magnitude, zero scales among them, key scales over two."""
    t = Setup(llmrs, ctx, 15, [700, 40], [rows, rows], 8, 2, 128, page, "f32")
    rng = np.random.default_rng(16)
    t.pool["vs"] = np.where(rng.random(t.pool["vs"].shape) < 0.3, 0,
                            t.pool["vs"] * np.float32(10.0) ** rng.integers(-6, 5, t.pool["vs"].shape)).astype(np.float32)
    t.pool["ks"] = (t.pool["ks"] * np.float32(10.0) ** rng.integers(-2, 1, t.pool["ks"].shape)).astype(np.float32)
    t.upload()
    t.check_attend(be)


def test_attend_shared_prefix_pages(llmrs, ctx, be):
    t = Setup(llmrs, ctx, 17, [130, 130, 64], [1, 3, 1], 8, 2, 128, 64, "f32")
    t.table[1, :2] = t.table[0, :2]  # the first 128 positions are the same pages
    t.table[2, 0] = t.table[0, 0]
    t.upload()
    t.check_attend(be)


def test_attend_propagates_nan_queries_to_their_rows_alone(llmrs, ctx, be):
    for rows in (1, 150):
        t = Setup(llmrs, ctx, 18, [100, 100], [rows, rows], 4, 2, 64, 32, "f32")
        t.raw[rows] = np.nan  # the first row of sequence 1
        got, (ref, *pieces) = t.attend(be)
        tol = S.attend_tolerance("f32", ref, *pieces, 64)
        others = np.arange(2 * rows) != rows
        assert np.isnan(got[rows]).all()
        assert np.all(np.abs(got - ref)[others] <= tol[others])


def test_attend_strided_torch_rows_on_a_side_stream(llmrs, ctx, be):
    """q as a view of packed q|k|v rows, output into wider rows, on torch's side stream."""
    import torch
    t = Setup(llmrs, ctx, 19, [90, 1000], [1, 3], 8, 2, 128, 64, "f32")
    stream = torch.cuda.Stream()
    qkv = torch.from_numpy(t.raw).cuda()
    out = torch.full((t.n_rows, 1500), 77.0, device="cuda")
    torch.cuda.synchronize()
    ctx.sync()
    ws = be.kv8_attention_workspace(t.cache, t.batch, 8, t.n_rows)
    try:
        ctx.set_stream(stream.cuda_stream)
        be.kv8_append(t.cache, t.batch, qkv[:, 1024:1280], qkv[:, 1280:], t.g_cos, t.g_sin)
        be.kv8_attention(t.cache, t.batch, qkv[:, :1024], out[:, 100:1124], t.g_cos, t.g_sin, workspace=ws)
        stream.synchronize()
    finally:
        ctx.set_stream(None)
    x = t.qkv.reshape(t.n_rows, -1, 128)
    S.append(t.pool, t.row_start, t.lens, t.table, x[:, 8:10], x[:, 10:], t.cos, t.sin)
    same(t.download(), t.pool)
    ref, *pieces = S.attend(t.pool, t.row_start, t.lens, t.table, x[:, :8], t.n_rows, t.cos, t.sin)
    got, used = out.cpu().numpy(), 4
    assert np.all(got[used:] == 77) and np.all(got[:, :100] == 77) and np.all(got[:, 1124:] == 77)
    tol = S.attend_tolerance("f32", ref[:used], *[p[:used] for p in pieces], 128)
    assert np.all(np.abs(got[:used, 100:1124].reshape(used, 8, 128) - ref[:used]) <= tol)


def test_small_workspace_is_refused(llmrs, ctx, be):
    t = Setup(llmrs, ctx, 20, [90], [1], 8, 2, 128, 64, "f32")
    q, _ = t.rows("q")
    with pytest.raises(llmrs.LlmrsError) as e:
        be.kv8_attention(t.cache, t.batch, q, workspace=llmrs.DeviceTensor(ctx, (16,), np.uint8))
    assert e.value.code == llmrs.EINVAL and "workspace" in str(e.value)
