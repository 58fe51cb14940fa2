"""Verification of drafted tokens on the GPU against the 64-bit numpy form.  Acceptances use
row sums of 32-bit exponentials: an exponential is off by 2 units in the last place (2^-22),
32 of them are summed in 32 bits (2^-19 at most), the rest in 64, so p is off by less than
2^-18 of itself.  The draw itself is made in 64 bits."""
import numpy as np
import pytest

import serving_oracle as S

pytestmark = pytest.mark.gpu

P_OFF = 2.0 ** -18


def make(seed, vocab, drafts, dtype="f32", heat=1.0, probs=True, spread=2.0):
    rng = np.random.default_rng(seed)
    rows = [k + 1 for k in drafts]
    rs = np.int32(np.concatenate([[0], np.cumsum(rows)]))
    n = int(rs[-1])
    logits = spread * rng.normal(0, 1, (n, vocab)).astype(np.float32)
    for r in range(n):
        logits[r, rng.integers(0, vocab, 3)] += 5.0
    raw, logits = S.to_type(logits, dtype)
    mine = np.concatenate([np.arange(a, b - 1) for a, b in zip(rs, rs[1:])]).astype(int) if n else np.zeros(0, int)
    x = logits[mine].astype(np.float64) + 0.7 * rng.normal(0, 1, (mine.size, vocab))
    q = np.exp(x - x.max(axis=1, keepdims=True)) if mine.size else np.zeros((0, vocab))
    q = (q / q.sum(axis=1, keepdims=True)).astype(np.float32) if mine.size else q.astype(np.float32)
    if probs:
        draft = np.int32([rng.choice(vocab, p=r.astype(np.float64) / r.astype(np.float64).sum()) for r in q])
    else:
        draft = q.argmax(axis=1).astype(np.int32) if mine.size else np.zeros(0, np.int32)
    u = rng.random(n).astype(np.float32)
    heats = np.full(len(rows), heat, np.float32)
    return dict(raw=raw, logits=logits, row_start=rs, draft=draft.reshape(-1), q=q if probs else None, u=u, heats=heats)


def run(llmrs, ctx, be, c, spare=0, temperature=True, workspace=True):
    T = llmrs.DeviceTensor.from_numpy
    n, vocab = c["raw"].shape
    m = len(c["row_start"]) - 1
    tokens, probs = T(ctx, np.full(n, 777, np.int32)), T(ctx, np.full(n, 777, np.float32))
    accepted = T(ctx, np.full(m, 777, np.int32))
    ws = be.verify_draft_workspace(n, vocab) if workspace else None
    be.verify_draft(T(ctx, c["raw"]), T(ctx, c["row_start"]), T(ctx, c["draft"]) if c["draft"].size else
                    llmrs.DeviceTensor(ctx, (0,), np.int32), None if c["q"] is None else T(ctx, c["q"]), T(ctx, c["u"]),
                    tokens, accepted, probs, temperature=T(ctx, c["heats"]) if temperature else None, workspace=ws)
    return tokens.numpy(), accepted.numpy(), probs.numpy()


def check(llmrs, ctx, be, c, **kw):
    tokens, accepted, probs = run(llmrs, ctx, be, c, **kw)
    want, count, p, margin = S.verify(c["logits"], c["row_start"], c["draft"], c["q"], c["u"],
                                      c["heats"] if kw.get("temperature", True) else None)
    decided = 0
    for s in range(len(count)):
        a, b = c["row_start"][s], c["row_start"][s + 1]
        if margin[s, 0] < P_OFF or margin[s, 1] < 1e-12:
            continue  # a draw on a border
        decided += 1
        assert accepted[s] == count[s], s
        assert np.array_equal(tokens[a:b], want[a:b]), (s, tokens[a:b], want[a:b])
        assert np.all(np.abs(probs[a:b] - p[a:b]) <= P_OFF * p[a:b] + 1e-37), s
    used = c["row_start"][-1]
    assert np.all(tokens[used:] == 777) and np.all(probs[used:] == 777)
    return decided


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab,drafts", [(5, [1, 3]), (1000, [4, 0, 2, 7, 1]), (8192, [3] * 9), (8193, [2, 0]),
                                          (32003, [5, 1, 0, 3]), (128256, [4, 2])])
@pytest.mark.parametrize("probs", [True, False])
def test_verify(llmrs, ctx, be, dtype, vocab, drafts, probs):
    c = make(vocab + len(drafts), vocab, drafts, dtype, probs=probs)
    assert check(llmrs, ctx, be, c) >= len(drafts) - 1
    ctx.sync()


@pytest.mark.parametrize("heat", [0.0, 0.3, 1.7, 1e-6, 100.0])
def test_verify_temperatures(llmrs, ctx, be, heat):
    check(llmrs, ctx, be, make(31, 3001, [4, 0, 6, 2, 1, 3], heat=heat))
    check(llmrs, ctx, be, make(32, 3001, [4, 0, 6, 2, 1, 3], heat=heat, probs=False))


def test_verify_mixed_temperatures_none_and_no_workspace(llmrs, ctx, be):
    c = make(33, 2000, [3, 3, 3, 3])
    c["heats"] = np.float32([0.0, 0.5, 1.0, 2.0])
    check(llmrs, ctx, be, c)
    c["heats"] = np.full(4, 9.0, np.float32)
    check(llmrs, ctx, be, c, temperature=False, workspace=False)


def test_verify_many_sequences_some_without_rows(llmrs, ctx, be):
    rng = np.random.default_rng(34)
    drafts = rng.integers(-1, 4, 900).tolist()  # -1: no rows
    drafts[0] = -1
    c = make(34, 40, drafts)
    assert check(llmrs, ctx, be, c) > 850
    ctx.sync()


def test_verify_leaves_rows_behind_the_last_sequence(llmrs, ctx, be):
    c = make(35, 500, [2, 3])
    n = c["raw"].shape[0]
    for name, value in (("raw", np.nan), ("logits", np.nan), ("u", 0.5)):
        c[name] = np.concatenate([c[name], np.full((3,) + c[name].shape[1:], value, np.float32)])
    check(llmrs, ctx, be, c)
    assert c["raw"].shape[0] == n + 3


def test_verify_masked_logits(llmrs, ctx, be):
    """-inf and NaN have no weight, +inf takes it all, a row without any weight ends the sequence."""
    c = make(36, 300, [2, 2, 2, 0, 0, 1])
    rs, x = c["row_start"], c["logits"]
    x[rs[0]:rs[1], ::2] = -np.inf
    x[rs[1]:rs[2], 5:290] = np.nan
    x[rs[2] + 1] = -np.inf                        # nothing is left of the second row
    x[rs[3], [7, 100]] = np.inf
    x[rs[4]] = np.nan
    x[rs[5], :] = -np.inf
    x[rs[5], 42] = 0.0                            # one token alone
    c["raw"] = x.copy()
    tokens, accepted, probs = run(llmrs, ctx, be, c)
    check(llmrs, ctx, be, c)
    assert tokens[rs[4]] == -1 and accepted[4] == 0 and probs[rs[4]] == 0
    assert tokens[rs[3]] in (7, 100)


def test_verify_equal_distributions_and_extreme_draws(llmrs, ctx, be):
    """u = 0 accepts every possible draft; q far above p rejects; p == q in a rejected row
    (a draw of 1 or more, outside the documented range) draws from p."""
    c = make(37, 64, [3, 3, 1])
    c["u"][:4] = 0.0
    c["q"][3:6] = 0.0
    c["q"][np.arange(3, 6), c["draft"][3:6]] = 1.0
    check(llmrs, ctx, be, c)
    r = c["row_start"][2]
    c["logits"][r] = 0.0
    c["raw"] = c["logits"].copy()
    c["q"][6] = np.float32(1 / 64)
    c["u"][r] = 1.0
    check(llmrs, ctx, be, c)
    c["u"][r + 1] = 2.0
    tokens, _, _ = run(llmrs, ctx, be, c)
    assert tokens[r] == 63  # behind the sum: the last token with weight
    c["u"][r + 1] = np.nan
    assert 0 <= run(llmrs, ctx, be, c)[0][r] < 64


def test_verify_ties_take_the_lowest_token(llmrs, ctx, be):
    c = make(38, 9000, [1, 0], heat=0.0)
    c["logits"][:] = 0.0
    c["logits"][:, [8500, 4000, 4001]] = 3.0
    c["raw"] = c["logits"].copy()
    c["draft"][0] = 4000
    check(llmrs, ctx, be, c)
    assert np.array_equal(run(llmrs, ctx, be, c)[0], [4000, 4000, 4000])


def test_verify_reports_drafts_and_batches_outside(llmrs, ctx, be):
    c = make(39, 100, [2, 1])
    c["draft"][1] = 100
    check(llmrs, ctx, be, c)
    with pytest.raises(llmrs.LlmrsError) as e:
        ctx.sync()
    assert e.value.code == llmrs.EDEVICE
    for bad in ([0, 3, 9], [0, 7, 5], [-1, 3, 5], [0, -2, 5]):
        c = make(39, 100, [2, 1])
        c["row_start"] = np.int32(bad)
        run(llmrs, ctx, be, c)
        with pytest.raises(llmrs.LlmrsError) as e:
            ctx.sync()
        assert e.value.code == llmrs.EDEVICE and "word 5" in str(e.value)


def test_verify_strided_rows(llmrs, ctx, be):
    import torch
    c = make(40, 1001, [3, 2])
    n, v = c["raw"].shape
    wide = torch.zeros(n, 1100, device="cuda")
    wide[:, 7:7 + v] = torch.from_numpy(c["raw"]).cuda()
    q = torch.zeros(c["q"].shape[0], 1050, device="cuda")
    q[:, 1:1 + v] = torch.from_numpy(c["q"]).cuda()
    put = {k: torch.from_numpy(c[k]).cuda() for k in ("row_start", "draft", "u")}
    tokens = torch.empty(n, dtype=torch.int32, device="cuda")
    accepted = torch.empty(2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    be.verify_draft(wide[:, 7:7 + v], put["row_start"], put["draft"], q[:, 1:1 + v], put["u"], tokens, accepted)
    ctx.sync()
    want, count, _, _ = S.verify(c["logits"], c["row_start"], c["draft"], c["q"], c["u"], None)
    assert np.array_equal(tokens.cpu().numpy(), want) and np.array_equal(accepted.cpu().numpy(), count)
