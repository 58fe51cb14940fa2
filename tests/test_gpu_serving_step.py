"""The serving operators together, as a server runs them: drafted rows are appended and
attended, a projection of the result gives logits, the drafts are verified, and the
sequences' lengths move on by what was accepted -- eagerly and as one captured graph."""
import numpy as np
import pytest

import serving_oracle as S

pytestmark = pytest.mark.gpu

H, KV, D, PAGE, V, K, N = 8, 2, 64, 16, 211, 3, 5


class Server:
    """N sequences, K drafts each step; q|k|v rows come from an embedding, logits from a projection."""

    def __init__(self, llmrs, be, seed):
        import torch
        self.torch, self.llmrs, self.be = torch, llmrs, be
        rng = np.random.default_rng(seed)
        self.embed = rng.normal(0, 1, (V, (H + 2 * KV) * D)).astype(np.float32)
        self.head = (rng.normal(0, 1, (H * D, V)) * 0.3).astype(np.float32)
        pages = N * 12
        self.table = rng.permutation(pages).reshape(N, 12).astype(np.int32)
        self.pool = {"kq": np.zeros((pages, KV, PAGE, D), np.int8), "vq": np.zeros((pages, KV, PAGE, D), np.int8),
                     "ks": np.zeros((pages, KV), np.float32), "vs": np.zeros((pages, KV), np.float32)}
        self.lens = np.zeros(N, np.int32)
        self.cos, self.sin = llmrs.rope_table(D, 12 * PAGE)
        self.rs = (np.arange(N + 1) * (K + 1)).astype(np.int32)
        cuda = lambda a: torch.from_numpy(a.copy()).cuda()  # noqa: E731
        self.g = {k: cuda(v) for k, v in self.pool.items()}
        self.g_lens, self.g_head, self.g_cos, self.g_sin = (cuda(x) for x in (self.lens, self.head, self.cos, self.sin))
        self.cache = llmrs.Kv8Cache(be.ctx, pages, PAGE, KV, D, k_codes=self.g["kq"], v_codes=self.g["vq"],
                                    k_scales=self.g["ks"], v_scales=self.g["vs"])
        self.g_rs, self.g_table = cuda(self.rs), cuda(self.table)
        self.batch = llmrs.SeqBatch(self.g_rs, self.g_lens, self.g_table)
        n = N * (K + 1)
        self.g_qkv = torch.zeros(n, (H + 2 * KV) * D, device="cuda")
        self.g_out = torch.zeros(n, H * D, device="cuda")
        self.g_draft = torch.zeros(N * K, dtype=torch.int32, device="cuda")
        self.g_u = torch.zeros(n, device="cuda")
        self.g_tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.g_accepted = torch.zeros(N, dtype=torch.int32, device="cuda")
        self.g_logits = torch.zeros(n, V, device="cuda")
        self.ws = be.kv8_attention_workspace(self.cache, self.batch, H, n)
        self.ws2 = be.verify_draft_workspace(n, V)

    def step(self):
        q, k, v = self.g_qkv[:, :H * D], self.g_qkv[:, H * D:(H + KV) * D], self.g_qkv[:, (H + KV) * D:]
        self.be.kv8_append(self.cache, self.batch, k, v, self.g_cos, self.g_sin)
        self.be.kv8_attention(self.cache, self.batch, q, self.g_out, self.g_cos, self.g_sin, workspace=self.ws)
        self.torch.matmul(self.g_out, self.g_head, out=self.g_logits)
        self.be.verify_draft(self.g_logits, self.g_rs, self.g_draft, None, self.g_u, self.g_tokens, self.g_accepted,
                             workspace=self.ws2)
        self.g_lens.add_(self.g_accepted).add_(1)

    def feed(self, rng, last):
        """Rows: the last token of each sequence, then its drafts."""
        draft = rng.integers(0, V, (N, K)).astype(np.int32)
        ids = np.concatenate([last[:, None], draft], axis=1).reshape(-1)
        u = rng.random(N * (K + 1)).astype(np.float32) * np.float32(0.05)  # small draws, so that drafts are accepted
        for g, a in ((self.g_qkv, self.embed[ids]), (self.g_draft, draft.reshape(-1)), (self.g_u, u)):
            g.copy_(self.torch.from_numpy(np.ascontiguousarray(a)))
        return ids, draft, u

    def expect(self, ids, draft, u, gpu_logits):
        x = self.embed[ids].reshape(len(ids), -1, D)
        S.append(self.pool, self.rs, self.lens, self.table, x[:, H:H + KV], x[:, H + KV:], self.cos, self.sin)
        ref, *pieces = S.attend(self.pool, self.rs, self.lens, self.table, x[:, :H], len(ids), self.cos, self.sin)
        tol = S.attend_tolerance("f32", ref, *pieces, D)
        # each logit: the attention's error through the projection, and a 32-bit sum of H*D products
        off = tol.reshape(len(ids), -1) @ np.abs(self.head) \
            + 2.0 ** -24 * H * D * (np.abs(ref).reshape(len(ids), -1) @ np.abs(self.head))
        assert np.all(np.abs(gpu_logits - ref.reshape(len(ids), -1) @ self.head) <= off)
        tokens, accepted, _, _ = S.verify(gpu_logits, self.rs, draft.reshape(-1), None, u, None)
        return tokens, accepted


@pytest.mark.parametrize("captured", [False, True])
def test_serving_steps(llmrs, ctx, be, captured):
    import torch
    rng = np.random.default_rng(50)
    sv = Server(llmrs, be, 51)
    stream = torch.cuda.Stream()
    last = rng.integers(0, V, N).astype(np.int32)
    try:
        ctx.set_stream(stream.cuda_stream)
        graph = None
        if captured:
            with torch.cuda.stream(stream):
                sv.feed(rng, last)
                sv.step()  # library handles are made outside the capture
                sv.g_lens.zero_()
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    sv.step()
            for k in sv.g:
                sv.g[k].zero_()
            sv.g_lens.zero_()
            torch.cuda.synchronize()
        moved = 0
        for _ in range(12):
            with torch.cuda.stream(stream):
                ids, draft, u = sv.feed(rng, last)
                graph.replay() if captured else sv.step()
                stream.synchronize()
            logits = sv.g_logits.cpu().numpy()
            tokens, accepted = sv.expect(ids, draft, u, logits)
            got = sv.g_tokens.cpu().numpy()
            assert np.array_equal(sv.g_accepted.cpu().numpy(), accepted)
            assert np.array_equal(got, tokens)
            for k in sv.pool:
                assert np.array_equal(sv.g[k].cpu().numpy(), sv.pool[k]), k
            last = tokens[sv.rs[:-1] + accepted].astype(np.int32)
            sv.lens = (sv.lens + accepted + 1).astype(np.int32)
            moved += int(accepted.sum())
            assert np.array_equal(sv.g_lens.cpu().numpy(), sv.lens)
        assert moved > 0  # some drafts were accepted
        ctx.sync()
    finally:
        ctx.set_stream(None)


def test_two_graphs_with_a_workspace_each(llmrs, ctx, be):
    """Two captured steps replayed on two streams at the same time, a workspace each."""
    import torch
    servers, graphs, streams, fed = [], [], [torch.cuda.Stream(), torch.cuda.Stream()], []
    try:
        for i, stream in enumerate(streams):
            sv = Server(llmrs, be, 60 + i)
            ctx.set_stream(stream.cuda_stream)
            with torch.cuda.stream(stream):
                rng = np.random.default_rng(70 + i)
                fed.append(sv.feed(rng, rng.integers(0, V, N).astype(np.int32)))
                sv.step()
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    sv.step()
            for k in sv.g:
                sv.g[k].zero_()
            sv.g_lens.zero_()
            torch.cuda.synchronize()
            servers.append(sv)
            graphs.append(graph)
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for sv, (ids, draft, u) in zip(servers, fed):
            tokens, accepted = sv.expect(ids, draft, u, sv.g_logits.cpu().numpy())
            assert np.array_equal(sv.g_tokens.cpu().numpy(), tokens)
            assert np.array_equal(sv.g_accepted.cpu().numpy(), accepted)
            for k in sv.pool:
                assert np.array_equal(sv.g[k].cpu().numpy(), sv.pool[k]), k
    finally:
        ctx.set_stream(None)


def test_capture_without_a_workspace_is_refused(llmrs, ctx, be):
    import torch
    sv = Server(llmrs, be, 80)
    stream = torch.cuda.Stream()
    refused = []
    try:
        ctx.set_stream(stream.cuda_stream)
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            sv.g_u.mul_(1.0)
            try:
                be.kv8_attention(sv.cache, sv.batch, sv.g_qkv[:, :H * D], sv.g_out)
            except llmrs.LlmrsError as e:
                refused.append(str(e))
    finally:
        ctx.set_stream(None)
    assert refused and "workspace" in refused[0]
