"""Plain numpy forms of the serving operators: the paged 8-bit cache's append
(the same f32 roundings, so codes and scales agree bit for bit), its attention
and the verification of drafted tokens in 64 bits."""
import numpy as np

FLT_MIN = np.float32(2.0 ** -126)


def bf16_bits(x):
    """float32 -> bfloat16 bits (round to nearest even), as uint16."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def to_type(x, dtype):
    """float32 values -> (array as a DeviceTensor takes it, the values it holds)."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x, x
    if dtype == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float32)
    b = bf16_bits(x)
    return b, bf16_value(b)


def from_type(a):
    return bf16_value(a) if a.dtype == np.uint16 else a.astype(np.float32)


def rotate32(x, cos, sin):
    """x [rows, heads, D], tables [rows, D/2]: each operation rounded to f32."""
    h = x.shape[-1] // 2
    lo, hi, c, s = x[..., :h], x[..., h:], cos[:, None], sin[:, None]
    return np.concatenate([lo * c - hi * s, lo * s + hi * c], axis=-1).astype(np.float32)


def append(pool, row_start, lens, table, k, v, cos=None, sin=None):
    """pool: dict of kq, vq (int8), ks, vs (f32), changed in place; k, v f32 [rows, KV, D]."""
    page = pool["kq"].shape[2]
    for s, length in enumerate(lens):
        a, n = row_start[s], row_start[s + 1] - row_start[s]
        if n == 0:
            continue
        pos = np.arange(length, length + n)
        for codes, scales, x in ((pool["kq"], pool["ks"], k), (pool["vq"], pool["vs"], v)):
            x = x[a:a + n]
            if codes is pool["kq"] and cos is not None:
                x = rotate32(x, cos[pos], sin[pos])
            x = np.where(np.isfinite(x), x, np.float32(0))
            for p in range(length // page, (length + n - 1) // page + 1):
                t0, t1 = max(length, p * page), min(length + n, (p + 1) * page)
                held, at = t0 - p * page, table[s][p]
                for g in range(codes.shape[1]):
                    part = x[t0 - length:t1 - length, g]
                    old = scales[at, g] if held else np.float32(0)
                    new = max(old, np.float32(np.abs(part).max()) / np.float32(127))
                    if new < FLT_MIN:
                        new = np.float32(0)
                    inv = np.float32(1) / new if new > 0 else np.float32(0)
                    if new > old and held:
                        codes[at, g, :held] = np.rint(codes[at, g, :held].astype(np.float32) * (old / new))
                    codes[at, g, held:held + t1 - t0] = np.clip(np.rint(part * inv), -127, 127)
                    scales[at, g] = new


def attend(pool, row_start, lens, table, q, n_rows, cos=None, sin=None, scale=None):
    """out [n_rows, H, D] f64 (NaN where no row is) for q f32 [rows, H, D], and per row and head
    the pieces a tolerance is made of: sum p|v| and sum |v| [rows, H, D],
    S2 = max_t scale*sqrt(sum_d (q_d k_td)^2), X = max_t |score| and T."""
    n_pages, kv, page, d = pool["kq"].shape
    heads = q.shape[1]
    rep = heads // kv
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out = np.full((n_rows, heads, d), np.nan)
    mass, floor, s2, xs, ts = np.zeros_like(out), np.zeros_like(out), np.zeros((n_rows, heads)), np.zeros((n_rows, heads)), np.zeros(n_rows)
    for s, length in enumerate(lens):
        a, n = row_start[s], row_start[s + 1] - row_start[s]
        if n == 0:
            continue
        total = length + n
        ids = np.asarray(table[s][:-(-total // page)])
        there = np.repeat((ids >= 0) & (ids < n_pages), page)[:total]
        ids = np.where((ids >= 0) & (ids < n_pages), ids, 0)
        pos = np.arange(length, total)
        x = q[a:a + n].astype(np.float64)
        if cos is not None:
            h, c, sn = d // 2, cos[pos].astype(np.float64)[:, None], sin[pos].astype(np.float64)[:, None]
            x = np.concatenate([x[..., :h] * c - x[..., h:] * sn, x[..., :h] * sn + x[..., h:] * c], axis=-1)
        for g in range(kv):
            k = (pool["kq"][ids, g].astype(np.float64) * pool["ks"][ids, g].astype(np.float64)[:, None, None])
            v = (pool["vq"][ids, g].astype(np.float64) * pool["vs"][ids, g].astype(np.float64)[:, None, None])
            k, v = k.reshape(-1, d)[:total], v.reshape(-1, d)[:total]
            k, v = np.where(there[:, None], k, 0), np.where(there[:, None], v, 0)
            for hh in range(g * rep, (g + 1) * rep):
                w = scale * x[:, hh] @ k.T
                ok = (np.arange(total)[None, :] <= pos[:, None]) & there[None, :]
                xs[a:a + n, hh] = np.where(ok, np.abs(w), 0).max(axis=1)
                s2[a:a + n, hh] = np.where(ok, scale * np.sqrt((x[:, hh] ** 2) @ (k ** 2).T), 0).max(axis=1)
                w = np.where(ok, w, -np.inf)
                m = np.where(ok.any(axis=1), w.max(axis=1), 0)
                p = np.where(ok, np.exp(w - m[:, None]), 0)
                l = p.sum(axis=1, keepdims=True)
                p = np.where(l > 0, p / np.where(l > 0, l, 1), 0)
                out[a:a + n, hh] = p @ v
                mass[a:a + n, hh] = p @ np.abs(v)
                floor[a:a + n, hh] = ok @ np.abs(v)
        ts[a:a + n] = pos + 1
    return out, mass, floor, s2, xs, ts


def attend_tolerance(dtype, ref, mass, floor, s2, xs, ts, d):
    """How far a row may be off, roundings counted as independent (four standard deviations
    or more): u = 2^-24 for each f32 operation of the sums over T positions and over D
    products and of the exponent; for 16-bit rows also the rounding of q and of the
    probabilities to f16 (2^-11 each) and of the result to its type.  A probability far below
    the row's largest is held by f16 pieces at a scale of 2^14: their smallest step is 2^-24,
    so it is off by half of that, 2^-39 of the largest, however small it is itself; with the
    sum of the probabilities at least the largest, that adds 2^-39 sum |v|."""
    ts, s2, xs = ts[:, None, None], s2[..., None], xs[..., None]
    tol = 2.0 ** -24 * (32 + 2 * np.sqrt(ts) + 8 * np.sqrt(d) * s2 + 4 * xs) * mass + 2.0 ** -39 * floor + 1e-30
    if dtype == "f32":
        return tol
    half_step = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    return tol + 2.0 ** -11 * (1 + 4 * s2) * mass + half_step * np.abs(ref) + (2.0 ** -25 if dtype == "f16" else 0)


def verify(logits, row_start, draft, draft_probs, u, temperature):
    """(tokens [rows] with -1, accepted [seqs], probs [rows] f64, margins [seqs, 2]): the smallest
    distance of a sequence's acceptances from their borders, as a share of p (an error of p is a
    share of it), and of its draw from its token's borders, as a share of the total."""
    n, vocab = logits.shape
    tokens, probs = np.full(n, -1, np.int64), np.zeros(n)
    accepted = np.zeros(len(row_start) - 1, np.int64)
    at, margin = 0, np.ones((len(accepted), 2))
    for s in range(len(row_start) - 1):
        a, b = row_start[s], row_start[s + 1]
        for r in range(a, b):
            x = logits[r].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
            heat = 1.0 if temperature is None else float(temperature[s])
            if not (x > -np.inf).any():
                p = np.zeros(vocab)
            elif not heat > 0:
                p = np.zeros(vocab)
                p[int(np.argmax(x))] = 1.0
            else:
                p = np.exp((x - x.max()) / heat)
                p /= p.sum()
            w = p
            if r < b - 1:
                i = at + r - a
                d = int(draft[i])
                inside = 0 <= d < vocab
                if draft_probs is None:
                    q = np.zeros(vocab)
                    if inside:
                        q[d] = 1.0
                else:
                    q = draft_probs[i].astype(np.float64)
                pd, qd = (p[d], q[d]) if inside else (0.0, 1.0)
                if heat > 0 and pd > 0:
                    margin[s, 0] = min(margin[s, 0], abs(float(u[r]) * qd - pd) / pd)
                if float(u[r]) * qd < pd:
                    tokens[r], probs[r] = d, pd
                    accepted[s] += 1
                    continue
                rest = np.maximum(p - q, 0)
                w = rest if rest.sum() > 0 else p
            if p.any():
                cum = np.cumsum(w)
                target = float(u[b - 1]) * cum[-1]
                hit = np.flatnonzero((cum > target) & (w > 0))
                t = int(hit[0]) if hit.size else int(np.flatnonzero(w > 0)[-1])
                if heat > 0:
                    margin[s, 1] = min(abs(cum[t] - target), abs(target - (cum[t] - w[t]))) / cum[-1]
                tokens[r], probs[r] = t, p[t]
            break
        at += max(0, b - a - 1)
    return tokens, accepted, probs, margin
