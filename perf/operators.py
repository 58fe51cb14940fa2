"""What the batched serving operators compute, in plain torch operations, and the cases they are timed on.

Three operators over a paged cache whose keys and values are held as int8 codes with one f32 scale for each
(page of tokens, KV head):

  append   rotate the new keys, round keys and values to the pages' codes and store them
  attend   causal attention of each sequence's newest rows over its pages (one row: a decode step; a few: drafted
           tokens to be verified; many: a prompt or a chunk of one)
  verify   accept or reject drafted tokens against the target's probabilities, and draw the next token

Pools: codes [pages][KV heads][page size][D] int8, scales [pages][KV heads] f32.  A batch packs the new rows of all
sequences: sequence s has rows row_start[s] .. row_start[s+1]-1, lens[s] tokens already in the cache, and its row i
stands at position lens[s] + i.  page_table[s] names its pages in order.

`own` selects what run() calls: the plain form below, or this framework's operators.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
GOLDEN = 0.6180339887498949
FLT_MIN = 2.0 ** -126


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one request of the 8B shape decoding: a single new token into a half-full page; latency is all
        _c("append one token 8B", "append", "f32", 32, 8, 128, 64, 1, (1000, 1000), (1, 1)),
        # a decode step of a full serving batch, odd batch size, 16-bit activations
        _c("append 191 decode rows", "append", "bf16", 32, 8, 128, 64, 191, (1, 2000), (1, 1)),
        # prompts of mixed length arriving at once, small pages: thousands of rows to rotate and round
        _c("append prompts 4x2k p32", "append", "f32", 32, 8, 128, 32, 4, (0, 150), (900, 2048)),
        # one request of the 1B shape (D = 64) early in its answer: the smallest attention call
        _c("attend one short 1B", "attend", "f32", 32, 8, 64, 64, 1, (250, 250), (1, 1)),
        # one request of the 8B shape at the benchmark's cache length
        _c("attend one at 4096 8B", "attend", "f32", 32, 8, 128, 64, 1, (4096, 4096), (1, 1)),
        # a decode step of a ragged serving batch: bound by reading the cache
        _c("attend 64 ragged 8B", "attend", "f32", 32, 8, 128, 64, 64, (37, 8192), (1, 1)),
        # one very long context, 70B head layout, large pages
        _c("attend one at 131k 70B", "attend", "bf16", 64, 8, 128, 128, 1, (131000, 131000), (1, 1)),
        # drafted tokens of 16 requests, up to six rows each, checked in one pass
        _c("attend drafts 16x6 8B", "attend", "f32", 32, 8, 128, 64, 16, (300, 4000), (1, 6)),
        # chunks of three prompts behind cached tokens, f32 activations (the framework's own), ragged
        _c("attend chunks 3x1k 8B f32", "attend", "f32", 32, 8, 128, 64, 3, (0, 3000), (333, 1024)),
        # two long prompts from their start, 16-bit activations: bound by the products
        _c("attend prompts 2x4k 8B bf16", "attend", "bf16", 32, 8, 128, 64, 2, (0, 0), (3500, 4096)),
        # one request, four drafted tokens, the full vocabulary
        _v("verify one x4", "f32", 128256, 1, (4, 4), 1.0, True),
        # a serving batch with up to seven drafts each, ragged, at a temperature
        _v("verify 64 x7", "f32", 128256, 64, (0, 7), 0.8, True),
    ]


def _c(name, op, dtype, heads, kv, d, page, seqs, lens, rows):
    c = {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv, "head_dim": d, "page": page, "seqs": seqs,
         "len_min": lens[0], "len_max": lens[1], "rows_min": rows[0], "rows_max": rows[1]}
    return dict(c, name=name) if name else c


def _v(name, dtype, vocab, seqs, drafts, temperature, probs):
    c = {"op": "verify", "dtype": dtype, "vocab": vocab, "seqs": seqs, "drafts_min": drafts[0],
         "drafts_max": drafts[1], "temperature": temperature, "draft_probs": probs}
    return dict(c, name=name) if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "verify"])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    if op == "verify":
        vocab = _log(rng, 1000, 160000)
        k = rng.randint(1, 8)
        seqs = _log(rng, 1, max(1, min(96, 64 * 4 * 128256 // (vocab * (k + 1)))))
        return _v(None, dtype, vocab, seqs, (rng.randint(0, k), k), rng.choice([1.0, 0.7, 1.3, 0.0]),
                  rng.random() < 0.7)
    d = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8, 8, 8])
    heads = kv * rng.choice([1, 2, 4, 4, 7, 8])
    page = rng.choice([16, 32, 64, 64, 128])
    kind = rng.choice(["decode", "drafts", "prompt"])
    if kind == "prompt":
        seqs = rng.randint(1, 4)
        rows_max = _log(rng, 40, 8000 // seqs if op == "append" else 2500 // seqs)
        len_max = rng.choice([0, _log(rng, 1, 1500)])
        rows = (rng.randint(0, rows_max), rows_max)
    else:
        seqs = _log(rng, 1, 128)
        k = 1 if kind == "decode" else rng.randint(2, 9)
        rows = (rng.randint(0 if seqs > 1 else 1, k), k)
        len_max = _log(rng, 1, 2000 if op == "append" else max(2, min(120000, 240000 // seqs)))
    return _c(None, op, dtype, heads, kv, d, page, seqs, (rng.randint(0, len_max), len_max), rows)


def _spread(n, lo, hi, phase):
    """n whole numbers over [lo, hi], the first of them hi."""
    return [hi - int((hi - lo + 1) * (((i + (phase if i else 0)) * GOLDEN) % 1.0)) for i in range(n)]


def _lens(case):
    return _spread(case["seqs"], case["len_min"], case["len_max"], 0.0)


def _rows(case):
    if case["op"] == "verify":
        return [k + 1 for k in _spread(case["seqs"], case["drafts_min"], case["drafts_max"], 0.3)]
    return _spread(case["seqs"], case["rows_min"], case["rows_max"], 0.3)


def work(case):
    rows = _rows(case)
    n, es = sum(rows), 4 if case["dtype"] == "f32" else 2
    if case["op"] == "verify":
        drafts = n - len(rows)
        byts = n * case["vocab"] * es + 12 * n + 4 * drafts + 8 * len(rows)
        if case["draft_probs"]:  # the row of the first rejected draft, and the drafted tokens' own probabilities
            byts += sum(1 for r in rows if r > 1) * case["vocab"] * 4
        return {"bytes": byts, "flops": 4 * n * case["vocab"]}
    lens, kv, d, page = _lens(case), case["kv_heads"], case["head_dim"], case["page"]
    new = n * kv * d
    if case["op"] == "append":  # rows read, codes written; the written pages' values are read back as well
        back = sum(_touched(l, r, page) for l, r in zip(lens, rows)) * page * kv * d
        return {"bytes": 2 * new * (es + 1) + n * d * 4 + 2 * back * 3, "flops": 2 * new * 8}
    live = [(l, r) for l, r in zip(lens, rows) if r]
    cached = sum(l + r for l, r in live)
    pairs = sum(l * r + r * (r + 1) // 2 for l, r in live)
    return {"bytes": 2 * cached * kv * d + 8 * (cached // page) * kv + 2 * n * case["heads"] * d * es + n * d * 4,
            "flops": 4 * d * case["heads"] * pairs}


def _touched(length, rows, page):
    return (length + rows - 1) // page - length // page + 1 if rows else 0


# ------------------------------------------------------------------ inputs
def _package():
    if "llmrs_b200" not in sys.modules:
        pkg = os.path.join(os.getcwd(), "llm.rs_b200")
        spec = importlib.util.spec_from_file_location("llmrs_b200", os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["llmrs_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["llmrs_b200"]


_backend = []


def _be():
    """The framework's backend: made once, as a program does at its start, and put on torch's stream."""
    if not _backend:
        pkg = _package()
        _backend.extend((pkg.CudaBackend(pkg.Context(0)), None))
    stream = torch.cuda.current_stream().cuda_stream
    if stream != _backend[1]:
        _backend[0].ctx.set_stream(stream)
        _backend[1] = stream
    return _backend[0]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = _prepare_verify(case, g) if case["op"] == "verify" else _prepare_cache(case, g)
    st["case"] = case
    return st


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _prepare_cache(case, g):
    kv, d, page, heads = case["kv_heads"], case["head_dim"], case["page"], case["heads"]
    lens, rows = _lens(case), _rows(case)
    need = [max(1, -(-(l + r) // page)) for l, r in zip(lens, rows)]
    width, pages = max(need), sum(need) + 3
    # pages are handed out in no order; entries behind a sequence's last page name no page
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    starts = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    col = torch.arange(width, device="cuda")
    at = starts[:, None] + col[None, :]
    inside = col[None, :] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(inside, order[at.clamp(max=pages - 1)], torch.full_like(order[:1], -1)).contiguous()
    st = {"lens": _ints(lens), "row_start": _ints([sum(rows[:i]) for i in range(len(rows) + 1)]), "table": table,
          "max_rows": max(1, max(rows)), "n_rows": sum(rows)}
    for x in ("k", "v"):  # codes as rounding normal values leaves them; scales of values of a few units
        st[x + "_codes"] = (_randn(g, pages, kv, page, d) * 36).round_().clamp_(-127, 127).to(torch.int8)
        st[x + "_scales"] = 0.028 * torch.exp(0.3 * _randn(g, pages, kv))
    # the packed rows of the fused projection: queries, keys, values; some heads attend sharply
    qkv = _randn(g, st["n_rows"], (heads + 2 * kv) * d)
    sharp = 0.5 + 2.0 * _rand(g, heads)
    qkv[:, : heads * d].view(-1, heads, d).mul_(sharp[None, :, None])
    st["qkv"] = qkv.to(DTYPES[case["dtype"]])
    n_pos = width * page
    freq = 500000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * freq[None, :]
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    # the pages this call writes, as the program that handed them out knows them
    units = [(s, p) for s in range(len(rows)) if rows[s]
             for p in range(lens[s] // page, (lens[s] + rows[s] - 1) // page + 1)]
    st["unit_seq"] = torch.tensor([u[0] for u in units], device="cuda")
    st["unit_page"] = torch.tensor([u[1] for u in units], device="cuda")
    st["touched"] = table[st["unit_seq"], st["unit_page"]].contiguous()
    if own:
        pkg, be = _package(), _be()
        st["cache"] = pkg.Kv8Cache(be.ctx, pages, page, kv, d, k_codes=st["k_codes"], v_codes=st["v_codes"],
                                   k_scales=st["k_scales"], v_scales=st["v_scales"])
        st["batch"] = pkg.SeqBatch(st["row_start"], st["lens"], st["table"])
        st["ws"] = be.kv8_attention_workspace(st["cache"], st["batch"], heads, st["n_rows"])
    return st


def _prepare_verify(case, g):
    rows, v = _rows(case), case["vocab"]
    n, drafts = sum(rows), sum(rows) - len(rows)
    st = {"row_start": _ints([sum(rows[:i]) for i in range(len(rows) + 1)]), "n_rows": n, "n_drafts": drafts}
    # a model's logits: a broad floor and a few likely tokens in each row
    logits = 2.2 * _randn(g, n, v)
    likely = torch.randint(0, v, (n, 6), generator=g, device="cuda")
    logits.scatter_add_(1, likely, 7.0 + 4.0 * _rand(g, n, 6))
    seq = torch.repeat_interleave(torch.arange(len(rows), device="cuda"), torch.tensor(rows, device="cuda"))
    last = torch.zeros(n, dtype=torch.bool, device="cuda")
    last[st["row_start"][1:].long() - 1] = True
    # the drafting model is near the target; its tokens are drawn from its own probabilities
    q = torch.softmax(logits[~last] + 0.8 * _randn(g, drafts, v), dim=1)
    if case["draft_probs"]:
        st["q"] = q
        noise = -torch.log(-torch.log(_rand(g, drafts, v).clamp_(1e-12, 1 - 1e-7)))
        st["draft"] = (torch.log(q) + noise).argmax(1).to(torch.int32) if drafts else _ints([])
    else:
        st["q"] = None
        st["draft"] = q.argmax(1).to(torch.int32) if drafts else _ints([])
    st["logits"] = logits.to(DTYPES[case["dtype"]])
    st["u"] = _rand(g, n)
    st["temperature"] = torch.full((len(rows),), case["temperature"], device="cuda")
    st["seq"] = seq
    if own:
        be = _be()
        st["ws"] = be.verify_draft_workspace(n, v)
    return st


# ------------------------------------------------------------------ one pass
def run(st):
    op = st["case"]["op"]
    if op == "append":
        return _append_own(st) if own else _append_plain(st)
    if op == "attend":
        return _attend_own(st) if own else _attend_plain(st)
    return _verify_own(st) if own else _verify_plain(st)


def _split(st):
    """Views of the packed rows: q [n, H*D], k and v [n, KV*D]."""
    c = st["case"]
    h, k = c["heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
    return st["qkv"][:, :h], st["qkv"][:, h:h + k], st["qkv"][:, h + k:]


def _append_own(st):
    be, (_, k, v) = _be(), _split(st)
    be.kv8_append(st["cache"], st["batch"], k, v, rope_cos=st["cos"], rope_sin=st["sin"])
    c = st["case"]
    shape = (st["touched"].numel(), c["kv_heads"], c["page"], c["head_dim"])
    k_now = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    v_now = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    be.kv8_read(st["cache"], st["touched"], k_now, v_now)
    return {"k": k_now, "v": v_now, "k_scales": st["k_scales"], "v_scales": st["v_scales"]}


def _attend_own(st):
    q, _, _ = _split(st)
    out = torch.empty(q.shape, dtype=q.dtype, device="cuda")
    _be().kv8_attention(st["cache"], st["batch"], q, out, rope_cos=st["cos"], rope_sin=st["sin"], workspace=st["ws"])
    return out


def _verify_own(st):
    tokens = torch.empty(st["n_rows"], dtype=torch.int32, device="cuda")
    accepted = torch.empty(st["case"]["seqs"], dtype=torch.int32, device="cuda")
    probs = torch.empty(st["n_rows"], dtype=torch.float32, device="cuda")
    _be().verify_draft(st["logits"], st["row_start"], st["draft"], st["q"], st["u"], tokens, accepted, probs,
                       temperature=st["temperature"], workspace=st["ws"])
    return {"tokens": tokens, "accepted": accepted, "probs": probs}


# ------------------------------------------------------------------ plain form
def _rotate(x, cos, sin):
    """Rotate-half of x [n, heads, D] by the rows cos, sin [n, D/2], each operation rounded to 32 bits."""
    half = x.shape[-1] // 2
    lo, hi, c, s = x[..., :half], x[..., half:], cos[:, None, :], sin[:, None, :]
    return torch.cat((lo * c - hi * s, lo * s + hi * c), dim=-1)


def _places(st):
    """Sequence, index within it and position of each packed row."""
    row = torch.arange(st["n_rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(st["row_start"][1:].contiguous(), row, right=True)
    i = row - st["row_start"][seq]
    return seq, i.long(), (st["lens"][seq] + i).long()


def _append_plain(st):
    c = st["case"]
    kv, d, page = c["kv_heads"], c["head_dim"], c["page"]
    _, k, v = _split(st)
    _, _, pos = _places(st)
    k = _rotate(k.float().view(-1, kv, d), st["cos"][pos], st["sin"][pos])
    v = v.float().view(-1, kv, d)
    first = st["unit_page"][:, None] * page + torch.arange(page, device="cuda")[None, :]  # positions [U, page]
    length = st["lens"][st["unit_seq"]].long()[:, None]
    start = st["row_start"][st["unit_seq"]].long()[:, None]
    count = st["row_start"][st["unit_seq"] + 1].long()[:, None] - start
    new = (first >= length) & (first < length + count)
    row = (start + first - length).clamp(0, st["n_rows"] - 1)
    new, before = new[:, None, :, None], (first < length)[:, None, :, None]
    kept = (st["unit_page"] * page < length[:, 0])[:, None]  # the page held tokens before
    ids = st["touched"].long()
    out = {}
    for name, x in (("k", k), ("v", v)):
        codes, scales = st[name + "_codes"], st[name + "_scales"]
        x = torch.where(new, x[row].permute(0, 2, 1, 3), torch.zeros((), device="cuda"))  # [U, KV, page, D]
        old_codes = codes[ids]
        old = torch.where(kept, scales[ids], torch.zeros((), device="cuda"))
        # the scale covers the page's largest magnitude and never shrinks while the page is in use
        now = torch.maximum(old, x.abs().amax(dim=(2, 3)) / 127.0)
        now = torch.where(now < FLT_MIN, torch.zeros_like(now), now)
        some = now > 0
        inv = torch.where(some, 1.0 / now, torch.zeros_like(now))[:, :, None, None]
        ratio = torch.where(some, old / now, torch.ones_like(now))[:, :, None, None]
        fresh = torch.round(x * inv).clamp(-127, 127)
        again = torch.round(old_codes.float() * ratio)
        stored = torch.where(new, fresh, torch.where(before, again, old_codes.float()))
        codes[ids] = stored.to(torch.int8)
        scales[ids] = now
        out[name] = (stored * now[:, :, None, None]).to(torch.bfloat16)
    return {"k": out["k"], "v": out["v"], "k_scales": st["k_scales"], "v_scales": st["v_scales"]}


def _paged(codes, scales, table):
    """The tokens that the page tables name, as 32-bit floats [n, KV, T, D]."""
    ids = table.clamp(min=0).long()
    x = codes[ids].float() * scales[ids][..., None, None]  # [n, P, KV, page, D]
    n, p, kv, page, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(n, kv, p * page, d)


def _attend_plain(st):
    c = st["case"]
    n, kv, d, heads = c["seqs"], c["kv_heads"], c["head_dim"], c["heads"]
    rep, m = heads // kv, st["max_rows"]
    q, _, _ = _split(st)
    seq, i, pos = _places(st)
    q = _rotate(q.float().view(-1, heads, d), st["cos"][pos], st["sin"][pos])
    qs = torch.zeros(n, m, kv, rep, d, device="cuda")
    qs[seq, i] = q.view(-1, kv, rep, d)
    qs = qs.permute(0, 2, 1, 3, 4).reshape(n, kv, m * rep, d)
    keys = _paged(st["k_codes"], st["k_scales"], st["table"])
    s = torch.matmul(qs, keys.transpose(2, 3)) * (1.0 / math.sqrt(d))
    del keys
    t = torch.arange(s.shape[3], device="cuda")
    last = st["lens"].long()[:, None] + torch.arange(m, device="cuda")[None, :]  # [n, m]
    masked = t[None, None, :] > last[:, :, None]
    s = s.view(n, kv, m, rep, -1).masked_fill(masked[:, None, :, None, :], -math.inf)
    s = torch.exp(s - s.amax(dim=-1, keepdim=True))
    total = s.sum(dim=-1, keepdim=True)
    values = _paged(st["v_codes"], st["v_scales"], st["table"])
    o = torch.matmul(s.view(n, kv, m * rep, -1), values).view(n, kv, m, rep, d) / total
    return o.permute(0, 2, 1, 3, 4)[seq, i].reshape(-1, heads * d).to(DTYPES[c["dtype"]])


def _verify_plain(st):
    c = st["case"]
    n, vocab, rs = st["n_rows"], c["vocab"], st["row_start"].long()
    row = torch.arange(n, device="cuda")
    seq = st["seq"]
    i = row - rs[seq]
    k = rs[1:] - rs[:-1] - 1  # drafts of each sequence
    is_last = i == k[seq]
    # probabilities in 64 bits: a draw can fall next to a border
    x = st["logits"].double()
    t = st["temperature"].double()[seq][:, None]
    e = torch.exp((x - x.amax(dim=1, keepdim=True)) / torch.where(t > 0, t, torch.ones_like(t)))
    p = e / e.sum(dim=1, keepdim=True)
    place = torch.arange(vocab, device="cuda")[None, :]
    likeliest = torch.where(e == 1, place, torch.full_like(place, vocab)).amin(dim=1, keepdim=True)
    p = torch.where(t > 0, p, (place == likeliest).double())  # temperature 0: the first of the likeliest tokens
    drafted = (row - seq).clamp(max=max(0, st["n_drafts"] - 1))  # rows of the drafts lie packed without the last rows
    u = st["u"].double()
    ok = torch.zeros(n, dtype=torch.bool, device="cuda")
    if st["n_drafts"]:
        token = st["draft"].long()[drafted]
        pd = p[row, token]
        qd = st["q"][drafted, token].double() if st["q"] is not None else torch.ones_like(pd)
        ok = (u * qd < pd) & ~is_last
    grid = torch.zeros(c["seqs"], c["drafts_max"] + 1, dtype=torch.int64, device="cuda")
    grid[seq, i] = ok.long()
    accepted = grid.cumprod(dim=1).sum(dim=1)
    chosen = rs[:-1] + accepted
    w = p[chosen]
    if st["n_drafts"]:
        at = drafted[chosen]
        if st["q"] is not None:
            rest = (w - st["q"][at].double()).clamp(min=0)
        else:
            rest = w.scatter(1, st["draft"].long()[at][:, None], 0.0)
        rejected = (accepted < k)[:, None] & (rest.sum(dim=1, keepdim=True) > 0)
        w = torch.where(rejected, rest, w)
    cum = w.cumsum(dim=1)
    over = cum > (u[rs[1:] - 1] * cum[:, -1])[:, None]
    first = torch.where(over & (w > 0), place, torch.full_like(place, vocab)).amin(dim=1)
    final = torch.where(w > 0, place, torch.full_like(place, -1)).amax(dim=1)
    nxt = torch.where(first < vocab, first, final)
    tokens = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    if st["n_drafts"]:
        tokens = torch.where(i < accepted[seq], token, tokens)
    tokens = torch.where(i == accepted[seq], nxt[seq], tokens)
    # the target's probability of each token that goes out
    probs = torch.where(tokens >= 0, p[row, tokens.clamp(min=0)], torch.zeros_like(u))
    return {"tokens": tokens.to(torch.int32), "accepted": accepted.to(torch.int32), "probs": probs.float()}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "verify":
        return _verify_exact(st)
    return _append_exact(st) if case["op"] == "append" else _attend_exact(st)


def _turn64(x, pos, table_cos, table_sin):
    """x [n, heads, D] in 64 bits as complex pairs (j, j + D/2), turned by the tables' angles."""
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:])
    w = torch.complex(table_cos[pos].double(), table_sin[pos].double())
    z = z * w[:, None, :]
    return torch.cat((z.real, z.imag), dim=-1)


def _append_exact(st):
    c = st["case"]
    kv, d, page, h = c["kv_heads"], c["head_dim"], c["page"], c["heads"] * c["head_dim"]
    lens, rs = st["lens"].tolist(), st["row_start"].tolist()
    table = st["table"].tolist()
    x = st["qkv"].double()
    out = {}
    for name, off in (("k", h), ("v", h + kv * d)):
        codes, scales = st[name + "_codes"].double(), st[name + "_scales"].double()
        rows = x[:, off:off + kv * d].reshape(-1, kv, d)
        ids = []
        for s, length in enumerate(lens):
            n = rs[s + 1] - rs[s]
            if not n:
                continue
            mine = rows[rs[s]:rs[s + 1]]
            if name == "k":
                mine = _turn64(mine, torch.arange(length, length + n, device="cuda"), st["cos"], st["sin"])
            for p in range(length // page, (length + n - 1) // page + 1):
                a, b = max(length, p * page), min(length + n, (p + 1) * page)
                part = mine[a - length:b - length].transpose(0, 1)  # [KV, tokens, D]
                at, lo, hi = table[s][p], a - p * page, b - p * page
                ids.append(at)
                now = part.abs().amax(dim=(1, 2)) / 127
                if lo:
                    now = torch.maximum(now, scales[at])
                    codes[at, :, :lo] = torch.round(codes[at, :, :lo] * (scales[at] / now)[:, None, None])
                codes[at, :, lo:hi] = torch.round(part / now[:, None, None])
                scales[at] = now
        at = torch.tensor(ids, device="cuda", dtype=torch.long)
        out[name], out[name + "_scales"] = codes[at] * scales[at][:, :, None, None], scales
    return out


def _attend_exact(st):
    c = st["case"]
    kv, d, heads, page = c["kv_heads"], c["head_dim"], c["heads"], c["page"]
    lens, rs = st["lens"].tolist(), st["row_start"].tolist()
    out = torch.zeros(st["n_rows"], heads, d, dtype=torch.float64, device="cuda")
    for s, length in enumerate(lens):
        n = rs[s + 1] - rs[s]
        if not n:
            continue
        total = length + n
        ids = st["table"][s, :-(-total // page)].long()
        pos = torch.arange(length, total, device="cuda")
        q = _turn64(st["qkv"][rs[s]:rs[s + 1], :heads * d].double().view(n, heads, d), pos, st["cos"], st["sin"])
        for g in range(kv):
            k = (st["k_codes"][ids, g].double() * st["k_scales"][ids, g].double()[:, None, None]).view(-1, d)[:total]
            v = (st["v_codes"][ids, g].double() * st["v_scales"][ids, g].double()[:, None, None]).view(-1, d)[:total]
            hs = slice(g * (heads // kv), (g + 1) * (heads // kv))
            w = torch.einsum("nhd,td->hnt", q[:, hs], k) / d ** 0.5
            w.masked_fill_(torch.arange(total, device="cuda")[None, :] > pos[:, None], -math.inf)
            out[rs[s]:rs[s + 1], hs] = torch.einsum("hnt,td->nhd", torch.softmax(w, dim=-1), v)
    return out.view(st["n_rows"], heads * d)


def _verify_exact(st):
    vocab, heat = st["case"]["vocab"], st["case"]["temperature"]
    rs, draft, u = st["row_start"].tolist(), st["draft"].tolist(), st["u"].tolist()
    probs, at = torch.zeros(st["n_rows"], dtype=torch.float64), 0
    for a, b in zip(rs, rs[1:]):
        for r in range(a, b):
            x = st["logits"][r].double()
            if heat:
                p = torch.exp(torch.log_softmax(x / heat, dim=0))
            else:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1
            w = p
            if r < b - 1:
                d = draft[at + r - a]
                q = st["q"][at + r - a].double() if st["q"] is not None else torch.zeros_like(p)
                q[d] = q[d] if st["q"] is not None else 1
                if u[r] * float(q[d]) < float(p[d]):
                    probs[r] = p[d]
                    continue
                rest = (p - q).clamp(min=0)
                w = rest if float(rest.sum()) > 0 else p
            cum = torch.cumsum(w, 0)
            hit = (cum > u[b - 1] * cum[-1]).nonzero()
            probs[r] = p[int(hit[0]) if len(hit) else int(w.nonzero()[-1])]
            break
        at += b - a - 1
    return {"tokens": None, "accepted": None, "probs": probs.cuda()}
