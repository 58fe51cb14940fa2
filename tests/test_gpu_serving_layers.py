"""Batched layers put together from this library's own operators: RMSNorm, quantised
projections of all requests' rows, the paged cache and its attention, the gated FFN, and the
head's logits verified -- a prompt, a step with drafts and a plain one."""
import numpy as np
import pytest

import serving_oracle as S

pytestmark = pytest.mark.gpu

HID, H, KV, D, FFN, V, PAGE, LAYERS, EPS = 256, 8, 2, 64, 512, 480, 32, 2, 1e-5


def _weight(llmrs, ctx, be, rng, n, k):
    codes, scales = be.quantize_q4(llmrs.DeviceTensor.from_numpy(ctx, rng.normal(0, k ** -0.5, n * k).astype(np.float32)))
    return llmrs.QuantWeight(ctx, codes.numpy(), scales.numpy(), n, k)


def test_layers_of_several_requests(llmrs, ctx, be):
    rng = np.random.default_rng(110)
    T = llmrs.DeviceTensor.from_numpy
    embed = rng.normal(0, 1, (V, HID)).astype(np.float32)
    layers = [{n: _weight(llmrs, ctx, be, rng, *s) for n, s in
               dict(q=(H * D, HID), k=(KV * D, HID), v=(KV * D, HID), o=(HID, H * D), gate=(FFN, HID), up=(FFN, HID),
                    down=(HID, FFN)).items()} for _ in range(LAYERS)]
    head = _weight(llmrs, ctx, be, rng, V, HID)
    norm = T(ctx, rng.uniform(0.8, 1.2, HID).astype(np.float32))
    pages = 24
    table = rng.permutation(pages).reshape(3, 8).astype(np.int32)
    cos, sin = llmrs.rope_table(D, 8 * PAGE)
    g_cos, g_sin, g_table = T(ctx, cos), T(ctx, sin), T(ctx, table)
    caches = [llmrs.Kv8Cache(ctx, pages, PAGE, KV, D) for _ in range(LAYERS)]
    pools = [{n: x.numpy() for n, x in dict(kq=c.k_codes, vq=c.v_codes, ks=c.k_scales, vs=c.v_scales).items()} for c in caches]
    lens = np.zeros(3, np.int32)
    for rows in ([40, 9, 70], [4, 1, 3], [1, 1, 1]):  # whole prompts; drafts of two requests; one token each
        rs = np.int32(np.concatenate([[0], np.cumsum(rows)]))
        n = int(rs[-1])
        ids = rng.integers(0, V, n)
        x = T(ctx, embed[ids])
        batch = llmrs.SeqBatch(T(ctx, rs), T(ctx, lens), g_table)
        for w, cache, pool in zip(layers, caches, pools):
            y = be.rms_norm(x, norm, EPS)
            q, k, v = (be.matmul_transposed(y, w[i]) for i in "qkv")
            be.kv8_append(cache, batch, k, v, g_cos, g_sin)
            out = be.kv8_attention(cache, batch, q, rope_cos=g_cos, rope_sin=g_sin)
            heads = lambda a: a.numpy().reshape(n, -1, D)  # noqa: E731
            S.append(pool, rs, lens, table, heads(k), heads(v), cos, sin)
            for name, got in dict(kq=cache.k_codes, vq=cache.v_codes, ks=cache.k_scales, vs=cache.v_scales).items():
                used = np.concatenate([table[s, :-(-(lens[s] + rows[s]) // PAGE)] for s in range(3)])
                new, want = got.numpy()[used], pool[name][used]
                assert np.array_equal(new, want), name
            ref, *pieces = S.attend(pool, rs, lens, table, heads(q), n, cos, sin)
            assert np.all(np.abs(out.numpy().reshape(ref.shape) - ref) <= S.attend_tolerance("f32", ref, *pieces, D))
            be.add_assign(x, be.matmul_transposed(out, w["o"]))
            y = be.rms_norm(x, norm, EPS)
            gate = be.matmul_transposed(y, w["gate"])
            be.silu_mul(gate, be.matmul_transposed(y, w["up"]))
            be.add_assign(x, be.matmul_transposed(gate, w["down"]))
        if rows[0] == 40:
            lens += np.int32(rows)
            continue
        logits = be.matmul_transposed(be.rms_norm(x, norm, EPS), head)
        drafts = np.concatenate([ids[a + 1:b] for a, b in zip(rs, rs[1:])]).astype(np.int32)  # what the rows were made of
        u = (rng.random(n) * 0.02).astype(np.float32)
        tokens, accepted = llmrs.DeviceTensor(ctx, (n,), np.int32), llmrs.DeviceTensor(ctx, (3,), np.int32)
        be.verify_draft(logits, batch.row_start, T(ctx, drafts) if drafts.size else None, None, T(ctx, u), tokens, accepted)
        want, count, _, margin = S.verify(logits.numpy(), rs, drafts, None, u, None)
        assert margin[:, 0].min() > 2.0 ** -18 and margin[:, 1].min() > 1e-12
        assert np.array_equal(tokens.numpy(), want) and np.array_equal(accepted.numpy(), count)
        lens += count.astype(np.int32) + 1
    ctx.sync()
