"""Torch tensors on another stream than the context's: each call comes behind what torch's
current stream has been given, and what torch is given next comes behind the call."""
import numpy as np
import pytest

import serving_oracle as S
import test_gpu_verify as V
from test_gpu_kv8 import Setup, same

pytestmark = pytest.mark.gpu


def _busy(torch):
    """Some milliseconds of work on torch's current stream."""
    x = torch.ones(4096, 4096, device="cuda")
    for _ in range(20):
        x = (x @ x) * (1.0 / 4096)
    return x


def _attention(t, out):
    used = int(t.row_start[-1])
    qv = np.ascontiguousarray(t.qkv[:, :t.heads * t.d]).reshape(t.n_rows, -1, t.d)
    ref, *pieces = [x[:used] for x in S.attend(t.pool, t.row_start, t.lens, t.table, qv, t.n_rows, t.cos, t.sin)]
    got = out.cpu().numpy()[:used].reshape(ref.shape)
    assert np.all(np.abs(got - ref) <= S.attend_tolerance("f32", ref, *pieces, t.d))


@pytest.mark.parametrize("side", [False, True])
def test_inputs_are_waited_for(llmrs, ctx, be, side):
    """Rows, batch arrays and pages that torch's stream writes late; the context on its own stream."""
    import torch
    t = Setup(llmrs, ctx, 95, [90, 300, 1000], [1, 70, 3], 8, 2, 128, 64, "f32")
    ws = be.kv8_attention_workspace(t.cache, t.batch, 8, t.n_rows)
    c = V.make(96, 500, [2, 0, 3])
    ctx.sync()
    late = {n: torch.from_numpy(np.ascontiguousarray(a)).cuda() for n, a in
            dict(qkv=t.raw, rs=t.row_start, lens=t.lens, x=c["raw"], u=c["u"], draft=c["draft"], q=c["q"]).items()}
    now = {n: torch.zeros_like(a) for n, a in late.items()}
    out = torch.zeros(t.n_rows, 1024, device="cuda")
    late["pages"] = torch.from_numpy(t.table[1, :2].copy()).cuda()
    now["pages"] = pages = torch.full((2,), int(t.table[0, 0]), dtype=torch.int32, device="cuda")
    k_out, v_out = (torch.zeros(2, 2, 64, 128, device="cuda") for _ in range(2))
    tokens = torch.zeros(c["raw"].shape[0], dtype=torch.int32, device="cuda")
    accepted = torch.zeros(3, dtype=torch.int32, device="cuda")
    rs = torch.from_numpy(c["row_start"]).cuda()
    batch = llmrs.SeqBatch(now["rs"], now["lens"], torch.from_numpy(t.table).cuda())
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream() if side else torch.cuda.default_stream()):
        _busy(torch)  # the library's handles and memory are there
        torch.cuda.synchronize()
        _busy(torch)
        for n in late:
            now[n].copy_(late[n])
        qkv = now["qkv"]
        be.kv8_append(t.cache, batch, qkv[:, 1024:1280], qkv[:, 1280:], t.g_cos, t.g_sin)
        be.kv8_attention(t.cache, batch, qkv[:, :1024], out, t.g_cos, t.g_sin, workspace=ws)
        be.kv8_read(t.cache, pages, k_out, v_out)
        be.verify_draft(now["x"], rs, now["draft"], now["q"], now["u"], tokens, accepted)
        seen = [x.clone() for x in (out, k_out, v_out, tokens, accepted)]
        torch.cuda.current_stream().synchronize()
    x = t.qkv.reshape(t.n_rows, -1, 128)
    S.append(t.pool, t.row_start, t.lens, t.table, x[:, 8:10], x[:, 10:], t.cos, t.sin)
    _attention(t, seen[0])
    for got, codes, scales in ((seen[1], "kq", "ks"), (seen[2], "vq", "vs")):
        ids = t.table[1, :2]
        assert np.array_equal(got.cpu().numpy(), t.pool[codes][ids].astype(np.float32) * t.pool[scales][ids][:, :, None, None])
    want, count, _, margin = S.verify(c["logits"], c["row_start"], c["draft"], c["q"], c["u"], None)
    assert margin.min() > 1e-4
    assert np.array_equal(seen[3].cpu().numpy(), want) and np.array_equal(seen[4].cpu().numpy(), count)
    ctx.sync()
    same(t.download(), t.pool)


def test_results_are_waited_for(llmrs, ctx, be):
    """Torch reads the rows right behind a call that the context's stream has not come to yet."""
    import torch
    t = Setup(llmrs, ctx, 97, [4000, 300], [300, 3], 8, 2, 128, 64, "f32")
    q, _ = t.rows("q")
    ws = be.kv8_attention_workspace(t.cache, t.batch, 8, t.n_rows)
    tq = torch.from_numpy(np.ascontiguousarray(t.raw[:, :1024])).cuda()
    out = torch.zeros(t.n_rows, 1024, device="cuda")
    torch.cuda.synchronize()
    ctx.sync()
    own = llmrs.DeviceTensor(ctx, (t.n_rows, 1024))
    for _ in range(60):  # on the context's stream alone
        be.kv8_attention(t.cache, t.batch, q, own, t.g_cos, t.g_sin, workspace=ws)
    be.kv8_attention(t.cache, t.batch, tq, out, t.g_cos, t.g_sin, workspace=ws)
    seen = out.clone()
    torch.cuda.synchronize()
    _attention(t, seen)


def test_a_capture_on_torch_s_stream_takes_the_calls_in(llmrs, ctx, be):
    """The context on a stream of its own, torch capturing another: the calls become part of the graph."""
    import torch
    t = Setup(llmrs, ctx, 98, [90, 300], [1, 70], 8, 2, 128, 64, "f32")
    ws = be.kv8_attention_workspace(t.cache, t.batch, 8, t.n_rows)
    tq = torch.from_numpy(np.ascontiguousarray(t.raw[:, :1024])).cuda()
    q, out = torch.zeros_like(tq), torch.zeros(t.n_rows, 1024, device="cuda")
    torch.cuda.synchronize()
    ctx.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q.copy_(tq)
        be.kv8_attention(t.cache, t.batch, q, out, t.g_cos, t.g_sin, workspace=ws)
        seen = out + 0.0
    ctx.sync()
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        _attention(t, seen)


def test_a_captured_context_refuses_tensors_of_another_stream(llmrs, ctx, be):
    import torch
    t = Setup(llmrs, ctx, 99, [90], [1], 8, 2, 128, 64, "f32")
    ws = be.kv8_attention_workspace(t.cache, t.batch, 8, t.n_rows)
    q, out = torch.zeros(t.n_rows, 1024, device="cuda"), torch.zeros(t.n_rows, 1024, device="cuda")
    own, mine = t.rows("q")[0], llmrs.DeviceTensor(ctx, (t.n_rows, 1024))
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.sync()
    said = []
    try:
        ctx.set_stream(stream.cuda_stream)
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            be.kv8_attention(t.cache, t.batch, own, mine, t.g_cos, t.g_sin, workspace=ws)  # its own tensors: no order to keep
            with torch.cuda.stream(other):
                try:
                    be.kv8_attention(t.cache, t.batch, q, out, t.g_cos, t.g_sin, workspace=ws)
                except llmrs.LlmrsError as e:
                    said.append(str(e))
            be.kv8_attention(t.cache, t.batch, q, out, t.g_cos, t.g_sin, workspace=ws)  # and the capture goes on
    finally:
        ctx.set_stream(None)
    assert said and "captur" in said[0]
