"""The serving operators' numpy forms on the CPU, and the refusals of their C entries
(host checks, in front of any GPU work)."""
import ctypes

import numpy as np
import pytest

import serving_oracle as S


def test_bf16_rounding():
    x = np.float32([1.0, 1.00390625, 1.01171875, -3.14159, 0.0, 65504.0])
    v = S.bf16_value(S.bf16_bits(x))
    assert np.all(np.abs(v - x) <= 2.0 ** -8 * np.abs(x))
    assert v[1] == 1.0 and v[2] == np.float32(1.015625)  # ties to even


def test_append_holds_values_to_half_a_step():
    rng = np.random.default_rng(3)
    pool = {"kq": np.full((4, 2, 16, 64), 99, np.int8), "vq": np.full((4, 2, 16, 64), -99, np.int8),
            "ks": np.full((4, 2), 1e9, np.float32), "vs": np.full((4, 2), 1e9, np.float32)}  # what a page held before
    k = rng.normal(0, 1, (21, 2, 64)).astype(np.float32)
    v = rng.normal(0, 1, (21, 2, 64)).astype(np.float32) * 3
    S.append(pool, [0, 21], [0], [[2, 1]], k, v)
    for codes, scales, x in (("kq", "ks", k), ("vq", "vs", v)):
        got = pool[codes][[2, 1]] * pool[scales][[2, 1]][:, :, None, None]  # [2 pages, KV, 16, D]
        got = got.transpose(0, 2, 1, 3).reshape(32, 2, 64)[:21]
        step = np.repeat(pool[scales][[2, 1]], 16, axis=0)[:21, :, None]
        assert np.all(np.abs(got - x) <= 0.5001 * step)
    # a larger row later: the scale grows, older tokens are rounded again
    before = pool["kq"][1].copy() * pool["ks"][1][:, None, None]
    S.append(pool, [0, 1], [21], [[2, 1]], 10 * k[:1], v[:1])
    after = pool["kq"][1] * pool["ks"][1][:, None, None]
    assert np.all(np.abs(after[:, :5] - before[:, :5]) <= 0.5001 * pool["ks"][1][:, None, None])


def test_verify_keeps_the_target_distribution():
    """Over a fine grid of draws the first token out is distributed as p, whatever q is."""
    rng = np.random.default_rng(5)
    logits = rng.normal(0, 1.5, (2, 5)).astype(np.float32)
    p = np.exp(logits[0].astype(np.float64))
    p /= p.sum()
    q = rng.random(5).astype(np.float32)
    q /= q.sum()
    grid = (np.arange(200) + 0.5) / 200
    share = np.zeros(5)
    for d in range(5):
        for ua in grid:
            for ub in grid[::10]:
                tokens, _, _, _ = S.verify(logits, [0, 2], [d], q[None], np.float64([ua, ub]), None)
                share[tokens[0]] += q[d]
    share /= share.sum()
    assert np.abs(share - p).max() < 0.02  # the grid's steps: 1/200 in u_a, 1/20 in u_b


# ------------------------------------------------------------------ refusals
def _structs(llmrs, **kw):
    c = dict(d_k_codes=4096, d_v_codes=4096, d_k_scales=4096, d_v_scales=4096, n_pages=8, page_size=64, n_kv_heads=2,
             head_dim=128)
    b = dict(n_seqs=1, d_row_start=4096, d_lens=4096, d_page_table=4096, max_pages=4)
    for name, value in kw.items():
        (c if name in c else b)[name] = value
    return llmrs.Kv8Struct(**c), llmrs.Kv8BatchStruct(**b)


BAD_CACHE = [dict(page_size=48), dict(page_size=256), dict(page_size=0), dict(head_dim=96), dict(head_dim=0),
             dict(n_kv_heads=0), dict(n_pages=0), dict(d_k_codes=0), dict(d_v_scales=0), dict(d_v_codes=4104),
             dict(n_pages=1 << 28)]
BAD_BATCH = [dict(n_seqs=-1), dict(n_seqs=70000), dict(d_lens=0), dict(d_page_table=0), dict(max_pages=0),
             dict(max_pages=1 << 27)]


def _refused(llmrs, rc, words):
    assert rc == llmrs.EINVAL
    text = llmrs.lib().llmrs_last_error().decode()
    assert words in text, text


@pytest.mark.parametrize("change", BAD_CACHE + BAD_BATCH, ids=str)
def test_cache_and_batch_are_checked(llmrs, change):
    c, b = _structs(llmrs, **change)
    L, r = llmrs.lib(), ctypes.byref
    _refused(llmrs, L.llmrs_kv8_append(None, r(c), r(b), 4096, 4096, llmrs.F32, 256, 3, None, None, 0), "kv8:")
    _refused(llmrs, L.llmrs_kv8_attention(None, r(c), r(b), 4096, 1024, 4096, 1024, llmrs.F32, 3, 8, None, None, 0,
                                          0.0, None, 0), "kv8:")
    n = ctypes.c_size_t(0)
    _refused(llmrs, L.llmrs_kv8_attention_workspace(r(c), r(b), 8, 3, r(n)), "kv8:")


def test_call_arguments_are_checked(llmrs):
    c, b = _structs(llmrs)
    L, r = llmrs.lib(), ctypes.byref

    def append(k=4096, v=4096, dtype=llmrs.F32, ld=256, n=3, cos=None, sin=None, n_pos=0):
        return L.llmrs_kv8_append(None, r(c), r(b), k, v, dtype, ld, n, cos, sin, n_pos)

    _refused(llmrs, append(), "ctx is NULL")
    _refused(llmrs, append(dtype=7), "dtype")
    _refused(llmrs, append(k=None), "NULL rows")
    _refused(llmrs, append(v=4100), "16-byte")
    _refused(llmrs, append(ld=255), "stride")
    _refused(llmrs, append(ld=257), "16-byte")
    _refused(llmrs, append(ld=260, dtype=llmrs.BF16), "16-byte")
    _refused(llmrs, append(n=-1), "n_rows")
    _refused(llmrs, append(cos=4096), "both or neither")
    _refused(llmrs, append(cos=4096, sin=4096, n_pos=0), "n_pos")

    def attend(q=4096, ldq=1024, out=4096, ldo=1024, dtype=llmrs.F32, n=3, heads=8, scale=0.0):
        return L.llmrs_kv8_attention(None, r(c), r(b), q, ldq, out, ldo, dtype, n, heads, None, None, 0, scale, None, 0)

    _refused(llmrs, attend(), "ctx is NULL")
    _refused(llmrs, attend(heads=7), "head counts")
    _refused(llmrs, attend(heads=0), "head counts")
    _refused(llmrs, attend(ldq=1000), "stride")
    _refused(llmrs, attend(out=None), "NULL rows")
    _refused(llmrs, attend(scale=-1.0), "scale")
    _refused(llmrs, attend(scale=float("nan")), "scale")
    _refused(llmrs, attend(scale=float("inf")), "scale")

    _refused(llmrs, L.llmrs_kv8_read(None, r(c), None, 2, 4096, 4096, llmrs.F32), "kv8_read")
    _refused(llmrs, L.llmrs_kv8_read(None, r(c), 4096, 2, 4100, 4096, llmrs.F32), "16-byte")
    _refused(llmrs, L.llmrs_kv8_read(None, r(c), 4096, 2, 4096, 4096, 9), "dtype")

    def verify(logits=4096, ld=100, dtype=llmrs.F32, vocab=100, n=3, seqs=1, rs=4096, draft=4096, q=4096, ldq=100,
               u=4096, tokens=4096, accepted=4096):
        return L.llmrs_verify_draft(None, logits, ld, dtype, vocab, n, seqs, rs, draft, q, ldq, u, None, tokens,
                                    accepted, None, None, 0)

    _refused(llmrs, verify(), "ctx is NULL")
    _refused(llmrs, verify(dtype=3), "dtype")
    _refused(llmrs, verify(vocab=0), "vocab")
    _refused(llmrs, verify(n=70000), "n_rows")
    _refused(llmrs, verify(ld=99), "strides")
    _refused(llmrs, verify(ldq=99), "strides")
    _refused(llmrs, verify(draft=None), "no drafted tokens")
    _refused(llmrs, verify(u=None), "NULL")
    _refused(llmrs, verify(accepted=None), "NULL")
    n = ctypes.c_size_t(0)
    assert L.llmrs_verify_draft_workspace(5, 128256, r(n)) == llmrs.OK and n.value > 0
    _refused(llmrs, L.llmrs_verify_draft_workspace(5, 0, r(n)), "bad arguments")
    assert L.llmrs_kv8_attention_workspace(r(c), r(b), 8, 3, r(n)) == llmrs.OK and n.value > 0
