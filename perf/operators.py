"""The operators of one batched verify / prefill step on device data, in plain
torch and through the framework:

  append   per-head norms of q and k, the position rotation, and K / V written
           to a paged cache (paged.rope_append);
  attend   attention of each sequence's new rows over its paged cache
           (paged.attn_paged);
  verify   acceptance of drafted tokens against the target's distribution and
           the residual draw, from given uniform numbers (paged.verify).

A batch is ragged: sequence s owns rows row_start[s] .. row_start[s + 1] - 1 of
the packed tensors and they are the last rows of its kv_len[s] positions.
`own` chooses the framework's calls; otherwise `run` computes the plain form.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _append(name, dtype, heads, kv_heads, dim, n_seq, rows_lo, rows_hi, past_lo, past_hi, page, norm, rot,
            inter, table):
    return {"name": name, "op": "append", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "n_seq": n_seq, "rows_lo": rows_lo, "rows_hi": rows_hi, "past_lo": past_lo, "past_hi": past_hi,
            "page": page, "norm": norm, "rot": rot, "interleaved": inter, "table": table}


def _attend(name, dtype, heads, kv_heads, dim, n_seq, rows_lo, rows_hi, past_lo, past_hi, page, window, lse):
    return {"name": name, "op": "attend", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "n_seq": n_seq, "rows_lo": rows_lo, "rows_hi": rows_hi, "past_lo": past_lo, "past_hi": past_hi,
            "page": page, "window": window, "lse": lse}


def _verify(name, dtype, n_seq, k_lo, k_hi, vocab, q, mixed):
    return {"name": name, "op": "verify", "dtype": dtype, "n_seq": n_seq, "k_lo": k_lo, "k_hi": k_hi,
            "vocab": vocab, "draft_probs": q, "mixed": mixed}


def listed():
    return [
        # one session's verify pass of the 1.5B-shaped target (k = 4): 5 rows, latency
        _append("append verify 1x5", "f16", 12, 2, 128, 1, 5, 5, 639, 639, 16, False, 128, False, "f16"),
        # 64 sessions' verify pass of the 7B shape, head norms on, adjacent-pair rotation of half the head
        _append("append verify 64x1-7", "bf16", 28, 4, 128, 64, 1, 7, 0, 2050, 16, True, 64, True, "f32"),
        # prompts of four sequences written in one pass, 7B shape, head norms on
        _append("append prefill 4x2047", "f16", 28, 4, 128, 4, 2047, 2047, 0, 1000, 16, True, 128, False, "f32"),
        # a decode step of one session of the 1.5B-shaped target
        _attend("attend decode 1x700", "f16", 12, 2, 128, 1, 1, 1, 699, 699, 16, 0, False),
        # the batched bench: 8 sessions' verify passes, k = 4, contexts of 128 to 1536
        _attend("attend verify 8x5", "f16", 12, 2, 128, 8, 5, 5, 123, 1531, 16, 0, False),
        # a full server's decode step, 7B shape, contexts from one token to long ones
        _attend("attend decode 64 ragged", "bf16", 28, 4, 128, 64, 1, 1, 0, 8190, 16, 0, False),
        # a verify pass (k = 6) at a very long context, 7B shape
        _attend("attend verify 1x7 long", "f16", 28, 4, 128, 1, 7, 7, 131000, 131000, 64, 0, True),
        # chunks and single rows together, 0.5B-shaped draft, sliding window, odd sizes
        _attend("attend mixed window", "bf16", 14, 2, 64, 9, 1, 701, 0, 1500, 32, 500, True),
        # prefill chunks of four long prompts, 7B shape: the compute-bound end
        _attend("attend prefill 4x2047", "f16", 28, 4, 128, 4, 2047, 2047, 1, 4097, 16, 0, False),
        # one session's acceptance, k = 4, 151,936 tokens
        _verify("verify 1x4", "f16", 1, 4, 4, 151936, True, False),
        # a full server's acceptance: 0 to 4 drafts, greedy and sampled sessions mixed, min-p
        _verify("verify 64x0-4", "f16", 64, 0, 4, 151936, True, True),
        # drafts without a distribution (n-gram lookups), 32,000 tokens, odd count
        _verify("verify 13x1-7 lookup", "f32", 13, 1, 7, 32000, False, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads, kv_heads, dim = rng.choice([(12, 2, 128), (14, 2, 64), (28, 4, 128), (8, 8, 128), (16, 1, 64)])
    dtype = rng.choice(["f16", "bf16"])
    page = rng.choice([8, 16, 16, 32, 64])
    op = rng.choice(["append", "attend", "attend", "verify"])
    if op == "append":
        rows = _log(rng, 1, 2000)
        n_seq = _log(rng, 1, max(1, min(64, 8000 // rows)))
        rot = rng.choice([dim, dim, dim // 2])
        c = _append("", dtype, heads, kv_heads, dim, n_seq, max(1, rows // rng.choice([1, 2, 5])), rows, 0,
                    _log(rng, 1, 3001), page, rng.choice([True, False]), rot, rng.choice([True, False]),
                    rng.choice(["f16", "f32"]))
    elif op == "attend":
        rows = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 1500)])
        past = _log(rng, 1, 20000 if rows < 9 else 4000)
        n_seq = _log(rng, 1, max(1, min(64, 120000 // past, 4500 // rows)))
        c = _attend("", dtype, heads, kv_heads, dim, n_seq, max(1, rows // rng.choice([1, 3])), rows,
                    past // rng.choice([1, 2, 10]), past, page, rng.choice([0, 0, _log(rng, 1, 2000)]),
                    rng.choice([True, False]))
    else:
        k = rng.randint(1, 8)
        vocab = _log(rng, 1000, 151936)
        c = _verify("", rng.choice(["f16", "bf16", "f32"]), _log(rng, 1, 32), rng.randint(0, k), k, vocab,
                    rng.choice([True, True, False]), rng.choice([True, False]))
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly over their logarithm, in a fixed mixed order."""
    if n == 1:
        return [hi]
    a = [int(round(math.exp(math.log(lo + 1) + (math.log(hi + 1) - math.log(lo + 1)) * i / (n - 1)))) - 1
         for i in range(n)]
    step = next(p for p in (7, 11, 13, 17, 19, 23) if n % p)
    return [a[(i * step + n // 2) % n] for i in range(n)]


def _rows(case):
    rows = _spread(case["rows_lo"], case["rows_hi"], case["n_seq"])
    past = _spread(case["past_lo"], case["past_hi"], case["n_seq"])[::-1]
    return rows, past


def _visible(rows, past, window):
    """(visible pairs, positions read) of one sequence."""
    pairs = 0
    if window:
        pairs = sum(min(past + i + 1, window) for i in range(rows))
        return pairs, past + rows - max(0, past + 1 - window)
    return rows * past + rows * (rows + 1) // 2, past + rows


def work(case):
    if case["op"] == "verify":
        ks = _spread(case["k_lo"], case["k_hi"], case["n_seq"])
        item = 4 if case["dtype"] == "f32" else 2
        # every row of logits once; one draft row a sequence that drafted (where the draw is made)
        q = sum(1 for k in ks if k) * case["vocab"] * 4 if case["draft_probs"] else 0
        n = sum(k + 1 for k in ks) * case["vocab"]
        return {"bytes": n * item + q, "flops": 4 * n}
    rows, past = _rows(case)
    n, h, hk, d = sum(rows), case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        table = 4 if case["table"] == "f32" else 2
        return {"bytes": 4 * n * (h + 2 * hk) * d + n * case["rot"] * table, "flops": 6 * n * (h + hk) * d}
    seen = [_visible(r, p, case["window"]) for r, p in zip(rows, past)]
    return {"bytes": 4 * n * h * d + sum(s[1] for s in seen) * 4 * hk * d + (4 * n * h if case["lse"] else 0),
            "flops": 4 * d * h * sum(s[0] for s in seen)}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _batch(case, gen):
    rows, past = _rows(case)
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    lens = [r + p for r, p in zip(rows, past)]
    page = case["page"]
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    width = max(need) + 2
    table = torch.zeros(case["n_seq"], width, dtype=torch.int32, device=DEV)
    at = torch.arange(width, device=DEV)[None]
    need_t, first = _ints(need)[:, None], _ints([sum(need[:i]) for i in range(len(need))])[:, None]
    table = torch.where(at < need_t, order[(first + at).clamp(max=n_pages - 1).long()], table)
    return {"row_start": _ints(start), "kv_len": _ints(lens), "page_table": table.contiguous(),
            "n_rows": start[-1], "max_rows": max(rows), "max_len": max(lens), "n_pages": n_pages}


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    s = {"case": case}
    dt = DTYPES[case["dtype"]]
    if case["op"] == "verify":
        _prepare_verify(case, s, gen, dt)
    else:
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        s.update(_batch(case, gen))
        n, pool = s["n_rows"], (s["n_pages"], hk, case["page"], d)
        s["k_pool"] = _normal(gen, *pool).mul_(1.5).to(dt)
        s["v_pool"] = _normal(gen, *pool).to(dt)
        if case["op"] == "append":
            # the projection's output rows: q | k | v side by side
            s["qkv"] = (_normal(gen, n, (h + 2 * hk) * d) * 1.7).to(dt)
            half = case["rot"] // 2
            inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
            ang = torch.arange(s["max_len"], dtype=torch.float64, device=DEV)[:, None] * inv[None]
            s["rope"] = torch.cat([ang.cos(), ang.sin()], 1).to(DTYPES[case["table"]])
            s["q_norm"] = (1 + 0.2 * _normal(gen, d)).to(dt) if case["norm"] else None
            s["k_norm"] = (1 + 0.2 * _normal(gen, d)).to(dt) if case["norm"] else None
            s["q_out"] = torch.zeros(n, h, d, dtype=dt, device=DEV)
        else:
            s["q"] = _normal(gen, n, h, d).to(dt)
            s["out"] = torch.zeros(n, h, d, dtype=dt, device=DEV)
            s["lse"] = torch.zeros(n, h, dtype=torch.float32, device=DEV) if case["lse"] else None
    if own:
        # what a server keeps from step to step: its context on the current stream, views of the cache
        # and of the step's batch, the attention's workspace
        from androidllm_b200 import ops, paged
        s["ctx"] = ops.default_context(0, torch.cuda.current_stream().cuda_stream)
        if case["op"] != "verify":
            s["kv"] = paged.PagedKV(s["k_pool"], s["v_pool"])
            s["seqs"] = paged.SeqBatch(s["row_start"], s["kv_len"], s["page_table"], n_rows=s["n_rows"],
                                       max_rows=s["max_rows"])
        if case["op"] == "attend":
            s["work"] = paged.AttnWorkspace(s["ctx"], case["heads"], case["kv_heads"], case["dim"])
    return s


def _prepare_verify(case, s, gen, dt):
    ks = _spread(case["k_lo"], case["k_hi"], case["n_seq"])
    n_seq, k, vocab = case["n_seq"], max(case["k_hi"], 1), case["vocab"]
    start = [0]
    for v in ks:
        start.append(start[-1] + v + 1)
    n = start[-1]
    s["row_start"], s["k_max"] = _ints(start), k
    # a few likely tokens over a long tail, as a language model's logits have
    logits = _normal(gen, n, vocab) * 2.0
    peaks = torch.randint(0, vocab, (n, 40), generator=gen, device=DEV)
    logits.scatter_add_(1, peaks, 4.0 + 5.0 * torch.rand(n, 40, generator=gen, device=DEV))
    s["logits"] = logits.to(dt)
    i = torch.arange(k, device=DEV)[None]
    row = (s["row_start"][:-1, None] + i).clamp(max=n - 1).long()
    temp = torch.full((n_seq,), 0.8, device=DEV)
    min_p = torch.zeros(n_seq, device=DEV)
    if case["mixed"]:
        at = torch.arange(n_seq, device=DEV)
        temp = torch.where(at % 5 == 3, torch.zeros_like(temp), temp + 0.1 * (at % 3))
        min_p = torch.where(at % 4 == 1, torch.full_like(min_p, 0.05), min_p)
    s["temperature"], s["min_p"] = temp, min_p
    # the draft model: the target's logits with noise; its candidates drawn from its own distribution
    t = torch.where(temp > 0, temp, torch.full_like(temp, 0.1))[:, None, None]
    dl = (logits[row] + 0.6 * _normal(gen, n_seq, k, vocab)) / t
    q = torch.softmax(dl, -1)
    noise = -torch.log(-torch.log(torch.rand(n_seq, k, vocab, generator=gen, device=DEV).clamp(1e-9, 1 - 1e-7)))
    s["draft_tokens"] = (dl + noise).argmax(-1).to(torch.int32)
    s["draft_probs"] = q if case["draft_probs"] else None
    s["uniforms"] = torch.rand(n_seq, k + 1, generator=gen, device=DEV, dtype=torch.float64)
    s["tokens"] = torch.zeros(n_seq, k + 1, dtype=torch.int32, device=DEV)
    s["n_accepted"] = torch.zeros(n_seq, dtype=torch.int32, device=DEV)
    s["p_draft"] = torch.zeros(n_seq, k, device=DEV)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["op"] == "append":
        return _own_append(s) if own else _plain_append(s)
    if case["op"] == "attend":
        return _own_attend(s) if own else _plain_attend(s)
    return _own_verify(s) if own else _plain_verify(s)


def _own_append(s):
    from androidllm_b200 import paged
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].view(s["n_rows"], h + 2 * hk, d)
    paged.rope_append(s["ctx"], s["kv"], s["seqs"], x[:, :h], x[:, h:h + hk], x[:, h + hk:], s["rope"], s["q_out"],
                      q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, interleaved=c["interleaved"])
    return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _own_attend(s):
    from androidllm_b200 import paged
    paged.attn_paged(s["ctx"], s["kv"], s["seqs"], s["q"], s["out"], s["work"], window=s["case"]["window"],
                     lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _own_verify(s):
    from androidllm_b200 import paged
    paged.verify(s["ctx"], s["row_start"], s["logits"], s["draft_tokens"], s["draft_probs"], s["uniforms"],
                 s["temperature"], s["tokens"], s["n_accepted"], min_p=s["min_p"], p_draft=s["p_draft"])
    return {"tokens": s["tokens"], "n_accepted": s["n_accepted"], "p_draft": s["p_draft"]}


def _places(s):
    """Sequence and position of every row."""
    row = torch.arange(s["n_rows"], device=DEV)
    start = s["row_start"].long()
    seq = torch.searchsorted(start[1:].contiguous(), row, right=True)
    pos = s["kv_len"].long()[seq] - (start[seq + 1] - row)
    return seq, pos


def _plain_append(s):
    c = s["case"]
    h, hk, d, rot, page = c["heads"], c["kv_heads"], c["dim"], c["rot"], c["page"]
    dt = s["qkv"].dtype
    x = s["qkv"].view(s["n_rows"], h + 2 * hk, d)
    qk = x[:, :h + hk].float()
    if c["norm"]:
        w = torch.cat([s["q_norm"].float().expand(h, d), s["k_norm"].float().expand(hk, d)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + 1e-6) * w
    seq, pos = _places(s)
    cs = s["rope"].float()[pos]
    cos, sin = cs[:, None, :rot // 2], cs[:, None, rot // 2:]
    if c["interleaved"]:
        a, b = qk[..., 0:rot:2], qk[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    qk = torch.cat([turned, qk[..., rot:]], -1).to(dt)
    where = s["page_table"].long()[seq, pos // page]
    s["k_pool"][where, :, pos % page] = qk[:, h:]
    s["v_pool"][where, :, pos % page] = x[:, h + hk:]
    return {"q": qk[:, :h].contiguous(), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_attend(s):
    c = s["case"]
    h, hk, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    n_seq, rows, length = c["n_seq"], s["max_rows"], s["max_len"]
    start, lens = s["row_start"].long(), s["kv_len"].long()
    at = torch.arange(length, device=DEV)
    where = s["page_table"].long()[:, at // page]                      # (n_seq, length)
    k = s["k_pool"][where, :, at % page].float()                       # (n_seq, length, hk, d)
    v = s["v_pool"][where, :, at % page].float()
    i = torch.arange(rows, device=DEV)[None]
    n_new = (start[1:] - start[:-1])[:, None]
    q = s["q"][(start[:-1, None] + i).clamp(max=s["n_rows"] - 1)].float()
    q = q.view(n_seq, rows, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(n_seq, hk, -1, d)
    score = (q @ k.permute(0, 2, 3, 1)).view(n_seq, h, rows, length) * (1.0 / math.sqrt(d))
    pos = (lens[:, None] - n_new + i)[:, :, None]                      # (n_seq, rows, 1)
    seen = (at <= pos) & (at < lens[:, None, None])
    if c["window"]:
        seen &= at > pos - c["window"]
    score = score.masked_fill(~seen[:, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill((at >= lens[:, None])[:, :, None, None], 0.0)
    o = (p.view(n_seq, hk, -1, length) @ v.permute(0, 2, 1, 3)).view(n_seq, h, rows, d)
    o = o / total.clamp(min=1e-30)
    seq, _ = _places(s)
    inside = torch.arange(s["n_rows"], device=DEV) - start[seq]
    out = o.permute(0, 2, 1, 3)[seq, inside].to(s["q"].dtype)
    lse = (top + torch.log(total))[..., 0].permute(0, 2, 1)[seq, inside] if c["lse"] else None
    return {"out": out, "lse": lse}


def _plain_verify(s):
    n_seq, k = s["draft_tokens"].shape
    start = s["row_start"].long()
    k_seq = start[1:] - start[:-1] - 1                                  # drafted tokens of each sequence
    n, vocab = s["logits"].shape
    lg = s["logits"].double()
    seq = torch.searchsorted(start[1:].contiguous(), torch.arange(n, device=DEV), right=True)
    temp = s["temperature"].double()[seq, None]
    top = lg.amax(-1, keepdim=True)
    e = torch.exp((lg - top) / torch.where(temp > 0, temp, torch.ones_like(temp)))
    e = torch.where(e < s["min_p"].double()[seq, None], torch.zeros_like(e), e)
    p = e / e.sum(-1, keepdim=True)
    # greedy: all of the mass on the first largest logit
    first = lg.argmax(-1, keepdim=True)
    p = torch.where(temp > 0, p, torch.zeros_like(p).scatter_(-1, first, 1.0))
    i = torch.arange(k, device=DEV)[None]
    drafted = i < k_seq[:, None]
    row = torch.where(drafted, start[:-1, None] + i, 0)
    x = s["draft_tokens"].long()
    p_x = p[row].gather(-1, x[..., None])[..., 0]
    greedy = ~(s["temperature"] > 0)[:, None]
    if s["draft_probs"] is None:
        q_x = torch.ones_like(p_x)
    else:
        q_x = s["draft_probs"].gather(-1, x[..., None])[..., 0].double()
    q_x = torch.where(greedy, torch.ones_like(q_x), q_x)
    ok = drafted & (s["uniforms"][:, :k] * q_x < p_x)
    acc = ok.to(torch.int64).cumprod(1).sum(1)
    stop = start[:-1] + acc
    r = p[stop]
    tried = acc.clamp(max=k - 1)
    if s["draft_probs"] is None:
        q = torch.zeros_like(r).scatter_(-1, x.gather(1, tried[:, None]), 1.0)
    else:
        q = s["draft_probs"][torch.arange(n_seq, device=DEV), tried].double()
    q = torch.where((acc < k_seq)[:, None] & ~greedy, q, torch.zeros_like(q))
    left = (r - q).clamp(min=0.0)
    r = torch.where((left.sum(-1) > 0)[:, None], left, r)
    cum = r.cumsum(-1)
    goal = s["uniforms"].gather(1, k_seq[:, None]) * cum[:, -1:]
    hit = (cum > goal) & (r > 0)
    last = vocab - 1 - (r > 0).flip(-1).to(torch.int8).argmax(-1)
    new = torch.where(hit.any(-1), hit.to(torch.int8).argmax(-1), last)
    j = torch.arange(k + 1, device=DEV)[None]
    pad = torch.cat([x, torch.full((n_seq, 1), -1, dtype=torch.int64, device=DEV)], 1)
    tokens = torch.where(j < acc[:, None], pad, torch.where(j == acc[:, None], new[:, None], -1))
    return {"tokens": tokens.to(torch.int32), "n_accepted": acc.to(torch.int32),
            "p_draft": torch.where(drafted, p_x, 0.0).float()}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    start, f64 = s["row_start"].tolist(), torch.float64
    if case["op"] == "verify":
        x, temps, mins = s["draft_tokens"].tolist(), s["temperature"].tolist(), s["min_p"].tolist()
        p_draft = torch.zeros(len(x), s["k_max"], dtype=f64, device=DEV)
        for b in range(case["n_seq"]):
            for i in range(start[b + 1] - start[b] - 1):
                l = s["logits"][start[b] + i].to(f64)
                if temps[b] > 0:
                    w = torch.softmax(l / temps[b], 0)
                    w[w < mins[b] * w.max()] = 0
                    p_draft[b, i] = w[x[b][i]] / w.sum()
                else:
                    p_draft[b, i] = float(int((l == l.max()).nonzero()[0, 0]) == x[b][i])
        return {"tokens": None, "n_accepted": None, "p_draft": p_draft}
    lens, table = s["kv_len"].tolist(), s["page_table"].tolist()
    h, hk, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "append":
        q = torch.empty(s["n_rows"], h, d, dtype=f64, device=DEV)
        k_pool, v_pool = s["k_pool"].to(f64), s["v_pool"].to(f64)
        x = s["qkv"].to(f64).view(s["n_rows"], h + 2 * hk, d)
        half = case["rot"] // 2
        first = torch.arange(half, device=DEV) * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        for b in range(case["n_seq"]):
            lo, hi = start[b], start[b + 1]
            pos = torch.arange(lens[b] - (hi - lo), lens[b], device=DEV)
            ang = s["rope"].to(f64)[pos][:, None]
            turn = torch.complex(ang[..., :half], ang[..., half:])
            got = []
            for y, w in ((x[lo:hi, :h], s["q_norm"]), (x[lo:hi, h:h + hk], s["k_norm"])):
                if w is not None:
                    y = w.to(f64) * y / ((y * y).sum(-1, keepdim=True) / d + 1e-6).sqrt()
                z = torch.complex(y[..., first], y[..., second]) * turn
                y = y.clone()
                y[..., first], y[..., second] = z.real, z.imag
                got.append(y)
            q[lo:hi] = got[0]
            pages = torch.tensor(table[b], device=DEV)[pos // page]
            k_pool[pages, :, pos % page] = got[1]
            v_pool[pages, :, pos % page] = x[lo:hi, h + hk:]
        return {"q": q, "k_pool": k_pool, "v_pool": v_pool}
    out = torch.zeros(s["n_rows"], h, d, dtype=f64, device=DEV)
    lse = torch.zeros(s["n_rows"], h, dtype=f64, device=DEV)
    for b in range(case["n_seq"]):
        lo, hi, n = start[b], start[b + 1], lens[b]
        pages = torch.tensor(table[b][:-(-n // page)], device=DEV)
        k = s["k_pool"][pages].transpose(0, 1).reshape(hk, -1, d)[:, :n].to(f64)
        v = s["v_pool"][pages].transpose(0, 1).reshape(hk, -1, d)[:, :n].to(f64)
        i = n - (hi - lo) + torch.arange(hi - lo, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None]
        hidden = (j > i) | ((j <= i - case["window"]) if case["window"] else (j < 0))
        for g in range(h):
            a = s["q"][lo:hi, g].to(f64) @ k[g * hk // h].T / math.sqrt(d)
            a[hidden] = -math.inf
            lse[lo:hi, g] = torch.logsumexp(a, 1)
            out[lo:hi, g] = torch.softmax(a, 1) @ v[g * hk // h]
    return {"out": out, "lse": lse if case["lse"] else None}
