"""Verification of drafted tokens where its inputs are at their ends: fewer drafts than the
row starts ask for, none at all, row starts that fall, the smallest temperatures."""
import numpy as np
import pytest

import serving_oracle as S
from test_gpu_verify import P_OFF, check, make, run

pytestmark = pytest.mark.gpu


def _reported(llmrs, ctx, word):
    with pytest.raises(llmrs.LlmrsError) as e:
        ctx.sync()
    assert e.value.code == llmrs.EDEVICE and "word %d" % word in str(e.value)
    ctx.sync()  # reported once


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("row_start,have,short", [
    ([0, 10, 10, 10, 10, 10], 5, [0]),     # nine drafts in one sequence, room for one of each of five
    ([0, 3, 3, 6, 10], 3, [2, 3]),         # the first two sequences' drafts are there
    ([0, 0, 0, 0, 3], 0, [3]),             # none at all
    ([0, 4, 5, 6], 2, [0])])               # what is behind a short sequence without drafts is drawn
def test_verify_drafts_that_are_not_there(llmrs, ctx, be, row_start, have, short, probs):
    c = make(50, 700, [k - 1 for k in np.diff(row_start)], probs=probs)
    assert c["row_start"].tolist() == row_start
    c["draft"] = c["draft"][:have].copy()
    if probs:
        c["q"] = c["q"][:have].copy()
        if have == 0:
            c["q"] = None
    tokens, accepted, out = run(llmrs, ctx, be, c)
    _reported(llmrs, ctx, 5)
    for s, (a, b) in enumerate(zip(row_start, row_start[1:])):
        if s in short:
            assert accepted[s] == 0 and np.all(tokens[a:b] == 777) and np.all(out[a:b] == 777)
    # the others as if the short ones had no rows
    whole = make(50, 700, [k - 1 for k in np.diff(row_start)], probs=probs)
    want, count, p, margin = S.verify(whole["logits"], whole["row_start"], whole["draft"], whole["q"], whole["u"], whole["heats"])
    for s, (a, b) in enumerate(zip(row_start, row_start[1:])):
        if s not in short:
            assert margin[s].min() > 1e-4  # no draw of this input lies on a border
            assert accepted[s] == count[s] and np.array_equal(tokens[a:b], want[a:b])
            assert np.all(np.abs(out[a:b] - p[a:b]) <= P_OFF * p[a:b])


def test_verify_plain_sampling_with_rows_behind_the_last_sequence(llmrs, ctx, be):
    """More rows than sequences and no drafts: the spare rows belong to nobody."""
    c = make(51, 900, [0, 0, -1, 0])
    for name, value in (("raw", np.nan), ("logits", np.nan), ("u", 0.5)):
        c[name] = np.concatenate([c[name], np.full((4,) + c[name].shape[1:], value, np.float32)])
    c["q"] = None
    assert check(llmrs, ctx, be, c) == 4
    ctx.sync()
    T = llmrs.DeviceTensor.from_numpy
    tokens, accepted = T(ctx, np.full(7, 777, np.int32)), T(ctx, np.full(4, 777, np.int32))
    be.verify_draft(T(ctx, c["raw"]), T(ctx, c["row_start"]), None, None, T(ctx, c["u"]), tokens, accepted)
    ctx.sync()
    want = S.verify(c["logits"], c["row_start"], c["draft"], None, c["u"], None)[0]
    assert np.array_equal(tokens.numpy()[:3], want[:3]) and np.all(tokens.numpy()[3:] == 777)
    assert np.all(accepted.numpy() == 0)


def test_verify_temperatures_behind_row_starts_that_fall(llmrs, ctx, be):
    """Row starts [0, 4, 1]: the second sequence does not fit, the first one's rows have its temperature."""
    c = make(52, 800, [3, 0])
    c["heats"] = np.float32([2.0, 0.3])
    c["u"][:3] = 0.0  # the drafts are accepted, and their probabilities go out
    want, count, p, margin = S.verify(c["logits"][:4], [0, 4], c["draft"], c["q"], c["u"], c["heats"])
    assert count[0] == 3 and margin[0, 1] > 1e-4
    c["row_start"] = np.int32([0, 4, 1])
    tokens, accepted, out = run(llmrs, ctx, be, c)
    _reported(llmrs, ctx, 5)
    assert accepted.tolist() == [3, 0] and np.array_equal(tokens[:4], want)
    assert np.all(np.abs(out[:4] - p) <= P_OFF * p)
    assert tokens[4] == 777 and out[4] == 777


@pytest.mark.parametrize("heat", [1.1e-38, 4.4e-39, 4e-39, 1e-39, 1e-42, 1e-45])
@pytest.mark.parametrize("probs", [True, False])
def test_verify_smallest_temperatures(llmrs, ctx, be, heat, probs):
    """Below 2^-126 / log2(e) the reciprocal of the temperature is past f32: p is still one at the
    likeliest token, which several share here."""
    c = make(53, 3001, [4, 0, 2, 3], heat=heat, probs=probs)
    c["logits"][:, [17, 2500]] = 60.0
    c["draft"][:] = 17
    c["raw"] = c["logits"].copy()
    if probs:
        c["q"][:] = np.float32(1 / 3001)
    assert check(llmrs, ctx, be, c) == 4
    assert run(llmrs, ctx, be, c)[1].sum() > 0  # u * q < 1/2: some are accepted


def test_verify_draws_next_to_a_border(llmrs, ctx, be):
    """Two tokens, exp(-t) and 1, and a draw u that lies beside the border of the first one, p0 =
    exp(-t) / (1 + exp(-t)), by a share of 1.3e-12 to 1e-11 of it: the 64-bit exponential, off by
    r^5 / 120 < 1.25e-12 of itself for |r| <= ln(2) / 64 (the likelier token's is exactly 1), still
    decides each one, and sums with a few roundings of 2^-53 do not matter."""
    rng = np.random.default_rng(54)
    t = rng.uniform(0.02, 80.0, 4_000_000).astype(np.float32)
    w = np.exp(-t.astype(np.float64))
    p0 = w / (1 + w)
    u = p0.astype(np.float32)
    off = (w * (1 - u.astype(np.float64)) - u) / w  # above 0: the first token is drawn
    some = (np.abs(off) > 1.3e-12) & (np.abs(off) < 1e-11)
    t, u, off = t[some], u[some], off[some]
    assert 300 < t.size < 4000 and 0.3 < (off > 0).mean() < 0.7 and t.min() < 2 and t.max() > 60
    logits = np.stack([-t, np.zeros_like(t)], axis=1)
    T = llmrs.DeviceTensor.from_numpy
    n = t.size
    tokens, accepted = llmrs.DeviceTensor(ctx, (n,), np.int32), llmrs.DeviceTensor(ctx, (n,), np.int32)
    be.verify_draft(T(ctx, logits), T(ctx, np.arange(n + 1, dtype=np.int32)), None, None, T(ctx, u), tokens, accepted)
    ctx.sync()
    assert np.array_equal(tokens.numpy(), np.where(off > 0, 0, 1))
