"""The paged 8-bit cache where its kernels change their way of working: sequences with few
and many rows in one call, query heads that do not fill a tile, scales at the ends of f32,
calls captured into graphs that run at the same time, pages filled by one call."""
import numpy as np
import pytest

import serving_oracle as S
from test_gpu_kv8 import NP, Setup, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,d", [(10, 2, 128), (24, 2, 64), (9, 3, 128), (8, 8, 64)])
def test_attend_few_and_many_rows_together(llmrs, ctx, be, dtype, heads, kv, d):
    """Vectors per KV head on both sides of where a sequence changes kernels, and none."""
    lens, rows = [0, 333, 129, 1, 64, 700, 0, 90], [1, 9, 0, 26, 5, 49, 3, 200]
    Setup(llmrs, ctx, 60, lens, rows, heads, kv, d, 64, dtype).check_attend(be)


@pytest.mark.parametrize("rows", [1, 5, 150])
def test_attend_value_scales_to_the_ends_of_f32(llmrs, ctx, be, rows):
    """From 10^-37 to 10^32 (a sum of 500 such values is still finite): no infinity or NaN on the
    way.  With many rows a tile's p * vs are two f16 pieces, shifted by a power of two that brings
    the row's largest, M, to 2^12 at the least (both roundings up of its logarithm cost one bit):
    their smallest step is 2^-24, so each is off by 2^-25 there, by 2^-37 M, and times codes of
    at most 127 the T of them by 127 T 2^-37 M.  M is at most the row's largest sum p|v|, since the
    token that has it has some code of 1 or more."""
    t = Setup(llmrs, ctx, 61, [500, 77], [rows, rows], 8, 2, 128, 16, "f32", sharp=6.0)
    rng = np.random.default_rng(62)
    t.pool["vs"] = (np.float32(10.0) ** rng.integers(-37, 33, t.pool["vs"].shape)).astype(np.float32)
    t.upload()
    got, (ref, mass, floor, s2, xs, ts) = t.attend(be)
    tol = S.attend_tolerance("f32", ref, mass, floor, s2, xs, ts, t.d)
    if rows == 150:
        tol += 127 * ts[:, None, None] * 2.0 ** -37 * mass.max(axis=2, keepdims=True)
    assert np.all(np.abs(got - ref) <= tol)


@pytest.mark.parametrize("rows", [2, 140])
def test_attend_gives_the_same_bits_again(llmrs, ctx, be, rows):
    t = Setup(llmrs, ctx, 63, [900, 20, 4000], [rows, rows, 1], 8, 2, 128, 64, "f32")
    q, _ = t.rows("q")
    ws = be.kv8_attention_workspace(t.cache, t.batch, 8, t.n_rows)
    first = be.kv8_attention(t.cache, t.batch, q, rope_cos=t.g_cos, rope_sin=t.g_sin, workspace=ws).numpy()
    for _ in range(5):
        again = be.kv8_attention(t.cache, t.batch, q, rope_cos=t.g_cos, rope_sin=t.g_sin, workspace=ws).numpy()
        used = int(t.row_start[-1])
        assert np.array_equal(first[:used].view(np.uint32), again[:used].view(np.uint32))


def test_graphs_with_a_workspace_each_run_at_the_same_time(llmrs, ctx, be):
    import torch
    made = []
    for i, rows in enumerate((1, 150, 6)):
        t = Setup(llmrs, ctx, 64 + i, [1500, 300], [rows, rows], 8, 2, 128, 64, "f32")
        q, qv = t.rows("q")
        out = torch.zeros(t.n_rows, 8 * 128, device="cuda")
        ws = be.kv8_attention_workspace(t.cache, t.batch, 8, t.n_rows)
        made.append((t, q, qv, out, ws, torch.cuda.Stream(), torch.cuda.CUDAGraph()))
    torch.cuda.synchronize()
    ctx.sync()
    try:
        for t, q, _, out, ws, stream, graph in made:
            ctx.set_stream(stream.cuda_stream)
            with torch.cuda.graph(graph, stream=stream):
                be.kv8_attention(t.cache, t.batch, q, out, t.g_cos, t.g_sin, workspace=ws)
        for _ in range(4):
            for *_, out, _, stream, graph in made:
                with torch.cuda.stream(stream):
                    out.zero_()
                    graph.replay()
        torch.cuda.synchronize()
    finally:
        ctx.set_stream(None)
    for t, _, qv, out, *_ in made:
        used = int(t.row_start[-1])
        ref, *pieces = [x[:used] for x in S.attend(t.pool, t.row_start, t.lens, t.table, qv, t.n_rows, t.cos, t.sin)]
        got = out.cpu().numpy()[:used].reshape(used, 8, 128)
        assert np.all(np.abs(got - ref) <= S.attend_tolerance("f32", ref, *pieces, 128))
    ctx.sync()


def _append(be, t, rope=True):
    (k, kv), (v, vv) = t.rows("k"), t.rows("v")
    be.kv8_append(t.cache, t.batch, k, v, *((t.g_cos, t.g_sin) if rope else ()))
    S.append(t.pool, t.row_start, t.lens, t.table, kv, vv, *((t.cos, t.sin) if rope else (None, None)))


@pytest.mark.parametrize("rows", [[1, 2, 1], [70, 300, 1]])
@pytest.mark.parametrize("page,d", [(16, 64), (128, 128)])
def test_append_over_codes_of_another_program(llmrs, ctx, be, rows, page, d):
    """Held codes of -128, which append itself never writes, rounded again as the scale grows."""
    t = Setup(llmrs, ctx, 67, [5, 130, 3], rows, 4, 2, d, page, "f32")
    for x in ("kq", "vq"):
        t.pool[x][np.random.default_rng(68).random(t.pool[x].shape) < 0.3] = -128
    for x in ("ks", "vs"):
        t.pool[x][:] = np.float32(2.0 ** -9)
    t.upload()
    _append(be, t)
    same(t.download(), t.pool)
    ctx.sync()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_full_pages_with_values_that_are_not_finite(llmrs, ctx, be, dtype):
    """They are stored as zero, in pages that one call fills, and their pages' scales do not know them."""
    t = Setup(llmrs, ctx, 69, [0, 17], [260, 150], 4, 2, 128, 128, dtype, spare_rows=0)
    hit = np.random.default_rng(70).random(t.raw.shape) < 0.001
    value = np.where(np.arange(t.raw.shape[1]) % 3 == 0, np.nan, np.where(np.arange(t.raw.shape[1]) % 3 == 1, np.inf, -np.inf))
    bits = np.broadcast_to(value.astype(np.float32), t.raw.shape)
    t.raw = np.where(hit, bits if dtype == "f32" else S.bf16_bits(bits), t.raw).astype(NP[dtype])
    t.qkv = np.where(hit, bits, t.qkv).astype(np.float32)
    with np.errstate(invalid="ignore"):
        _append(be, t)
    same(t.download(), t.pool)
    with pytest.raises(llmrs.LlmrsError) as e:
        ctx.sync()
    assert e.value.code == llmrs.EDEVICE
