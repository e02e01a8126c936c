"""Performance cases of the paged cache: head preparation into pages, decode
attention of one new token a sequence, prompt attention over a ragged batch
(both with an optional sliding window and sinks), and eviction by accumulated
attention weight. Each in its plain form (elementary torch operations in 32
bits) and, where `own` is set, through the framework's calls.

A case is a dict of plain values:
  op      prep | decode | prompt | evict
  heads, kv, hd, page, seqs
  lo, hi  the shortest and longest sequence's entries (prep, prompt: entries
          before the batch's rows), spread over their logarithm
  rows_lo, rows_hi  rows a sequence brings (prompt; prep, 0: one row each)
  window, sinks     (window 0: everything before a row)
  norm, ahead       prep: heads normalised; positions ahead of the entries
  weigh             decode: accumulates the attention weights
  keep, recent      evict
"""
import math

import torch

own = False

DEV = "cuda"
THETA, EPS = 1.0e6, 1.0e-5
# query heads, KV heads, head size of the framework's own model shapes
HEADS = {"qwen2-0.5b": (14, 2, 64), "llama8b": (32, 8, 128), "lfm2-1.2b": (32, 8, 64)}


def _case(name, op, heads, page, seqs, lo, hi, **more):
    H, KV, hd = HEADS[heads]
    c = {"op": op, "heads": H, "kv": KV, "hd": hd, "page": page, "seqs": seqs, "lo": lo, "hi": hi,
         "rows_lo": 0, "rows_hi": 0, "window": 0, "sinks": 0, "norm": False, "ahead": 0,
         "weigh": False, "keep": 0, "recent": 0, **more}
    return {"name": name, **c} if name else c


def listed():
    return [
        # A token of each of 64 conversations served together.
        _case("prep-step", "prep", "llama8b", 16, 64, 40, 8000),
        # Five prompts of one batch behind earlier turns, heads normalised;
        # entries were evicted before, so positions run ahead of them.
        _case("prep-prompts", "prep", "lfm2-1.2b", 64, 5, 30, 6000, rows_lo=131, rows_hi=1900,
              norm=True, ahead=700),
        # The first tokens of one short chat: latency alone.
        _case("decode-short", "decode", "qwen2-0.5b", 64, 1, 45, 45),
        # A token of each of 64 conversations under a window of 1024 with the
        # first 4 entries kept visible.
        _case("decode-window", "decode", "llama8b", 16, 64, 40, 30000, window=1024, sinks=4),
        # One conversation near the longest context, nothing hidden.
        _case("decode-long", "decode", "llama8b", 64, 1, 131000, 131000),
        # 24 conversations whose caches are held at a budget: the step also
        # adds up the weights that the eviction ranks by.
        _case("decode-weights", "decode", "lfm2-1.2b", 32, 24, 500, 6000, weigh=True),
        # A token and its four drafts behind a long prompt.
        _case("prompt-drafts", "prompt", "lfm2-1.2b", 64, 1, 6000, 6000, rows_lo=5, rows_hi=5),
        # Seven fresh or continued prompts in one batch, odd lengths.
        _case("prompt-batch", "prompt", "qwen2-0.5b", 16, 7, 1, 900, rows_lo=33, rows_hi=1500),
        # A chunk of a long prompt under a window of 4096 with 4 sinks.
        _case("prompt-window", "prompt", "llama8b", 64, 1, 18000, 18000, rows_lo=2048,
              rows_hi=2048, window=4096, sinks=4),
        # One short cache cut to its budget.
        _case("evict-one", "evict", "qwen2-0.5b", 64, 1, 577, 577, keep=512, recent=64, sinks=4),
        # Sixteen caches cut to 2048 entries, the shorter ones copied whole.
        _case("evict-batch", "evict", "lfm2-1.2b", 32, 16, 700, 6000, keep=2048, recent=512,
              sinks=4),
        # Two caches of the longest context cut to 4096 entries.
        _case("evict-long", "evict", "llama8b", 64, 2, 100000, 131000, keep=4096, recent=1024,
              sinks=4),
    ]


def draw(rng):
    def log(a, b):
        return max(a, min(b, round(math.exp(rng.uniform(math.log(a), math.log(b))))))

    op, heads = rng.choice(["prep", "decode", "prompt", "evict"]), rng.choice(sorted(HEADS))
    page = rng.choice([16, 32, 64, 128])
    if op == "prep":
        hi = log(1, 20000)
        prompts = rng.random() < 0.5
        return _case(None, op, heads, page, log(1, 8) if prompts else log(1, 64), log(1, hi), hi,
                     rows_lo=log(1, 100) if prompts else 0, rows_hi=log(100, 700) if prompts else 0,
                     norm=rng.random() < 0.5, ahead=rng.choice([0, log(1, 90000)]))
    window = rng.choice([0, log(16, 4096)])
    sinks = rng.choice([0, log(1, 64)]) if window else 0
    if op == "decode":
        seqs = log(1, 64)
        hi = log(1, 131000 // seqs)
        return _case(None, op, heads, page, seqs, log(1, hi), hi, window=window, sinks=sinks,
                     weigh=rng.random() < 0.5)
    if op == "prompt":
        seqs = log(1, 8)
        rows = log(1, 2048 // seqs)
        hi = log(1, 16000 // seqs)
        return _case(None, op, heads, page, seqs, log(1, hi), hi, rows_lo=log(1, rows),
                     rows_hi=rows, window=window, sinks=sinks)
    seqs = log(1, 24)
    hi = log(200, 131000 // seqs)
    keep = log(128, 4096)
    return _case(None, op, heads, page, seqs, log(100, hi), hi, keep=keep,
                 recent=log(1, keep // 2), sinks=rng.choice([0, log(1, 64)]))


# ------------------------------------------------------------------ inputs

def _spread(lo, hi, n, by):
    """n whole numbers from lo to hi, even in their logarithm, out of order."""
    if n == 1:
        return [hi]
    while math.gcd(by, n) > 1:
        by += 1
    return [round(lo * (hi / lo) ** (i * by % n / (n - 1))) for i in range(n)]


def _sizes(c):
    """(entries, rows) of each sequence, the rows among the entries."""
    n = c["seqs"]
    lens = _spread(c["lo"], c["hi"], n, 5)
    if c["rows_hi"]:
        rows = _spread(c["rows_lo"], c["rows_hi"], n, 3)
        return [p + r for p, r in zip(lens, rows)], rows
    return lens, [1] * n


def _seen(c, i):
    """Entries that entry i's row sees."""
    w = c["window"]
    return i + 1 if not w or w >= i + 1 else w + min(c["sinks"], i + 1 - w)


def _rope_table(hd, positions):
    """Cosines and sines: rows 0..1023 of those positions, row 1024 + i of
    position 1024 i, as the head preparation takes them."""
    r = torch.arange(1024 + (positions + 1023) // 1024, dtype=torch.float64, device=DEV)
    pos = torch.where(r < 1024, r, (r - 1024) * 1024)
    freq = THETA ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEV) / hd)
    a = pos[:, None] * freq
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    H, KV, hd, ps, n = c["heads"], c["kv"], c["hd"], c["page"], c["seqs"]
    lens, rows = _sizes(c)
    M = sum(rows)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=DEV, dtype=dtype)

    def i32(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    wide = -(-max(lens) // ps)
    counts = i32([-(-x // ps) for x in lens])
    new = -(-c["keep"] // ps) if c["op"] == "evict" else 0
    used = int(counts.sum())
    pages = used + n * new + 3
    order = torch.randperm(pages, generator=g, device=DEV).int()
    # a sequence's pages in its table row, -1 behind them
    at = torch.arange(wide, device=DEV)
    first = counts.cumsum(0) - counts
    table = torch.where(at < counts[:, None], order[(first[:, None] + at).clamp(max=pages - 1)],
                        -1).int().contiguous()
    s = {"c": c, "k": randn(pages, ps, KV * hd, dtype=torch.float16),
         "v": randn(pages, ps, KV * hd, dtype=torch.float16), "table": table, "lens": i32(lens),
         "wide": max(lens)}
    if c["op"] == "prep":
        s["qkv"] = randn(M, (H + 2 * KV) * hd)
        s["rope"] = _rope_table(hd, 131072)
        s["q_norm"], s["k_norm"] = (1 + 0.1 * randn(hd), 1 + 0.1 * randn(hd))
    elif c["op"] == "evict":
        s["weights"] = randn(n, wide * ps).square_()  # a few heavy entries, many light ones
        s["new_table"] = order[used:used + n * new].reshape(n, new).contiguous()
    else:
        s["q"] = randn(M, H * hd) * (1.5 / math.sqrt(hd))
        if c["weigh"]:
            s["weights"] = randn(n, wide * ps).abs_()
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    s["row_start"] = i32(starts) if c["rows_hi"] else None
    if c["op"] == "prep":
        s["pos"] = i32([x - r + t + c["ahead"] for x, r in zip(lens, rows) for t in range(r)])
    s["rows_wide"] = max(rows)
    if own:
        from webgllm_amd import ops
        s["shape"] = ops.attn_shape(H, KV, hd, eps=EPS, use_norm=c["norm"])
        s["cache"] = ops.PagedCache(s["k"], s["v"], table, s["lens"])
        if c["op"] == "decode":
            s["scratch"] = ops.paged_decode_scratch(s["cache"], s["shape"], weights=c["weigh"])
        elif c["op"] == "prompt":
            s["scratch"] = ops.paged_prefill_scratch(s["cache"], s["shape"], M)
        elif c["op"] == "evict":
            s["scratch"] = ops.paged_evict_scratch(s["cache"])
    return s


# ------------------------------------------------------------------- a pass

def run(state):
    return {"prep": _prep, "decode": _decode, "prompt": _prompt, "evict": _evict}[
        state["c"]["op"]](state)


def _rows(s, M):
    """Sequence and entry of each row."""
    m = torch.arange(M, device=DEV)
    if s["row_start"] is None:
        return m, s["lens"].long() - 1
    start = s["row_start"].long()
    b = torch.searchsorted(start, m, right=True) - 1
    return b, s["lens"].long()[b] - start[b + 1] + m


def _gather(pages, table, wide, KV, hd):
    """The first `wide` entries of every sequence: [sequences, KV, wide, hd]
    floats (whatever page 0 holds behind a sequence's own)."""
    i = torch.arange(wide, device=DEV)
    at = table[:, i // pages.shape[1]].clamp(min=0).long()
    x = pages[at, i % pages.shape[1]].float()
    return x.view(x.shape[0], wide, KV, hd).permute(0, 2, 1, 3).contiguous()


def _softmax(x):
    """Softmax over the last dim; zeros where nothing is visible."""
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    t = e.sum(-1, keepdim=True)
    return e / torch.where(t == 0, 1.0, t)


def _prep(s):
    c, qkv = s["c"], s["qkv"]
    H, KV, hd = c["heads"], c["kv"], c["hd"]
    if own:
        from webgllm_amd import ops
        q = ops.paged_head_prep(qkv, s["shape"], s["rope"], s["cache"], pos=s["pos"],
                                row_start=s["row_start"], q_norm=s["q_norm"] if c["norm"] else None,
                                k_norm=s["k_norm"] if c["norm"] else None)
        return q, s["k"], s["v"]
    M = qkv.shape[0]
    b, i = _rows(s, M)
    ps = c["page"]
    page = s["table"][b, i // ps].long()
    x = qkv.view(M, H + 2 * KV, hd)
    qk, v = x[:, :H + KV], x[:, H + KV:]
    if c["norm"]:
        w = torch.cat([s["q_norm"].expand(H, hd), s["k_norm"].expand(KV, hd)])
        qk = qk * w * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS)
    freq = THETA ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEV) / hd)
    a = s["pos"].double()[:, None] * freq
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    x1, x2 = qk[..., :hd // 2], qk[..., hd // 2:]
    r = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
    s["k"][page, i % ps] = r[:, H:].reshape(M, KV * hd).half()
    s["v"][page, i % ps] = v.reshape(M, KV * hd).half()
    return (r[:, :H] * (1.0 / math.sqrt(hd))).reshape(M, H * hd), s["k"], s["v"]


def _decode(s):
    c, q, lens = s["c"], s["q"], s["lens"]
    H, KV, hd, n = c["heads"], c["kv"], c["hd"], c["seqs"]
    if own:
        from webgllm_amd import ops
        out = ops.paged_attn_decode(q, s["shape"], s["cache"], window=c["window"],
                                    sinks=c["sinks"], weights=s.get("weights"),
                                    scratch=s["scratch"])
        return (out, s["weights"]) if c["weigh"] else out
    wide = s["wide"]
    k, v = _gather(s["k"], s["table"], wide, KV, hd), _gather(s["v"], s["table"], wide, KV, hd)
    j = torch.arange(wide, device=DEV)
    n_keys = lens[:, None].long()
    see = j < n_keys
    if c["window"]:
        see = see & ((j >= n_keys - c["window"]) | (j < c["sinks"]))
    x = q.view(n, KV, H // KV, hd) @ k.transpose(-1, -2)
    p = _softmax(torch.where(see[:, None, None], x, -math.inf))
    out = (p @ torch.where(see[:, None, :, None], v, 0.0)).reshape(n, H * hd).half()
    if not c["weigh"]:
        return out
    s["weights"][:, :wide] += p.sum((1, 2))
    return out, s["weights"]


def _prompt(s):
    c, q = s["c"], s["q"]
    H, KV, hd, n = c["heads"], c["kv"], c["hd"], c["seqs"]
    if own:
        from webgllm_amd import ops
        return ops.paged_attn_prefill(q, s["shape"], s["cache"], s["row_start"],
                                      window=c["window"], sinks=c["sinks"], scratch=s["scratch"])
    M, R, wide = q.shape[0], s["rows_wide"], s["wide"]
    start = s["row_start"].long()
    count = start[1:] - start[:-1]
    k, v = _gather(s["k"], s["table"], wide, KV, hd), _gather(s["v"], s["table"], wide, KV, hd)
    r = torch.arange(R, device=DEV)
    qp = q[(start[:-1, None] + r).clamp(max=M - 1)].view(n, R, KV, H // KV, hd)
    qp = qp.permute(0, 2, 3, 1, 4).reshape(n, KV, H // KV * R, hd)
    i = (s["lens"].long() - count)[:, None] + r  # the rows' entries
    j = torch.arange(wide, device=DEV)
    see = (j <= i[..., None]) & (r < count[:, None])[..., None]
    if c["window"]:
        see = see & ((j > i[..., None] - c["window"]) | (j < c["sinks"]))
    x = (qp @ k.transpose(-1, -2)).view(n, KV, H // KV, R, wide)
    p = _softmax(torch.where(see[:, None, None], x, -math.inf))
    live = (j < s["lens"].long()[:, None])[:, None, :, None]
    o = p.view(n, KV, H // KV * R, wide) @ torch.where(live, v, 0.0)
    o = o.view(n, KV, H // KV, R, hd).permute(0, 3, 1, 2, 4).reshape(n, R, H * hd)
    b, _ = _rows(s, M)
    return o[b, torch.arange(M, device=DEV) - start[b]].half()


def _evict(s):
    c, lens, w = s["c"], s["lens"], s["weights"]
    ps, keep, n = c["page"], c["keep"], c["seqs"]
    if own:
        from webgllm_amd import ops
        new, kept, kw = ops.paged_evict(s["cache"], w, keep, s["new_table"], sinks=c["sinks"],
                                        recent=c["recent"], scratch=s["scratch"])
        return new.lens, kept, kw, s["k"], s["v"]
    j = torch.arange(w.shape[1], device=DEV)
    n_keys = lens[:, None].long()
    rank = torch.where((j < c["sinks"]) | (j >= n_keys - c["recent"]), 0, 1)
    rank = torch.where(j >= n_keys, 2, rank)
    by_weight = torch.argsort(torch.where(torch.isnan(w), -math.inf, w), dim=-1, descending=True,
                              stable=True)
    order = by_weight.gather(1, torch.argsort(rank.gather(1, by_weight), dim=-1, stable=True))
    # the kept entries in order; those that a shorter cache has not got, last
    best = torch.where(rank.gather(1, order[:, :keep]) < 2, order[:, :keep], w.shape[1])
    idx = best.sort(-1).values
    idx = torch.cat([idx, idx.new_full((n, keep - idx.shape[1]), w.shape[1])], 1)
    live = idx < w.shape[1]
    at = idx.clamp(max=w.shape[1] - 1)
    src = s["table"].gather(1, at // ps).long() * ps + at % ps
    i = torch.arange(keep, device=DEV).expand(n, keep)
    dst = s["new_table"].gather(1, i // ps).long() * ps + i % ps
    # (a shorter cache's missing entries write its first one's place with itself)
    src, dst = torch.where(live, src, src[:, :1]), torch.where(live, dst, dst[:, :1])
    flat = (-1, s["k"].shape[2])
    for pool in (s["k"].view(flat), s["v"].view(flat)):
        pool[dst.reshape(-1)] = pool[src.reshape(-1)]
    kept = torch.where(live, idx, -1).int()
    return (lens.clamp(max=keep), kept, torch.where(live, w.gather(1, at), 0.0), s["k"], s["v"])


# -------------------------------------------------------------- what it takes

def work(case):
    c = case
    H, KV, hd = c["heads"], c["kv"], c["hd"]
    lens, rows = _sizes(c)
    M, entry = sum(rows), KV * hd * 2 * 2  # bytes of an entry's key and value
    if c["op"] == "prep":
        return {"bytes": M * ((H + 2 * KV) * hd * 4 + H * hd * 4 + entry + 4 + hd * 4),
                "flops": M * (H + KV) * hd * 8}
    if c["op"] == "evict":
        kept = [min(n, c["keep"]) for n in lens]
        return {"bytes": sum(n * 4 for n in lens) + sum(kept) * (2 * entry + 8), "flops": 0}
    pairs = read = 0
    for n, r in zip(lens, rows):
        seen = [_seen(c, i) for i in range(n - r, n)]
        pairs += sum(seen)
        first = 0 if not c["window"] else max(0, n - r + 1 - c["window"])
        read += n - first + min(c["sinks"] if c["window"] else 0, first)
    weights = 2 * 4 * read if c["weigh"] else 0
    return {"bytes": read * entry + M * H * hd * (4 + 2) + weights, "flops": 4 * pairs * H * hd}


# ------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    H, KV, hd, ps = c["heads"], c["kv"], c["hd"], c["page"]
    lens, rows = _sizes(c)
    D = KV * hd

    def slots(b, n):
        """Places in the pool of sequence b's first n entries."""
        pages = s["table"][b, :-(-n // ps)].long()
        return (pages[:, None] * ps + torch.arange(ps, device=DEV)).reshape(-1)[:n]

    K, V = s["k"].view(-1, D), s["v"].view(-1, D)
    if c["op"] == "evict":
        new_k, new_v = s["k"].clone(), s["v"].clone()
        keep, wide = c["keep"], s["weights"].shape[1]
        kept_w = torch.zeros(len(lens), keep, dtype=torch.float64, device=DEV)
        kept = torch.full((len(lens), keep), -1, dtype=torch.int32, device=DEV)
        for b, n in enumerate(lens):
            w = s["weights"][b, :n].double()
            must = torch.zeros(n, dtype=torch.bool, device=DEV)
            if n > keep:
                must[:c["sinks"]] = True
                must[n - c["recent"]:] = True
                room = keep - int(must.sum())
                rest = (~must).nonzero()[:, 0]
                must[rest[torch.argsort(-w[rest], stable=True)[:room]]] = True
                idx = must.nonzero()[:, 0]
            else:
                idx = torch.arange(n, device=DEV)
            m = idx.numel()
            to = (s["new_table"][b].long()[:, None] * ps +
                  torch.arange(ps, device=DEV)).reshape(-1)[:m]
            new_k.view(-1, D)[to] = K[slots(b, n)[idx]]
            new_v.view(-1, D)[to] = V[slots(b, n)[idx]]
            kept[b, :m], kept_w[b, :m] = idx.int(), w[idx]
        return s["lens"].clamp(max=keep), kept, kept_w, new_k.double(), new_v.double()
    if c["op"] == "prep":
        x = s["qkv"].double().view(-1, H + 2 * KV, hd)
        q, k, v = x.split([H, KV, KV], 1)
        if c["norm"]:
            q = q / (q.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["q_norm"].double()
            k = k / (k.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["k_norm"].double()
        step = torch.arange(hd // 2, dtype=torch.float64, device=DEV)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                           s["pos"].double()[:, None] * torch.pow(THETA, -2.0 * step / hd))

        def rotate(y):
            z = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous())
            z = z * turn[:, None]
            return torch.cat([z.real, z.imag], -1)

        q, k = rotate(q) / math.sqrt(hd), rotate(k)
        new_k, new_v = K.double(), V.double()
        m = 0
        for b, (n, r) in enumerate(zip(lens, rows)):
            to = slots(b, n)[n - r:]
            new_k[to], new_v[to] = k[m:m + r].reshape(r, D), v[m:m + r].reshape(r, D)
            m += r
        return q.reshape(-1, H * hd), new_k.view(s["k"].shape), new_v.view(s["v"].shape)
    out, w_out = [], s["weights"].double() if c["weigh"] else None
    m = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        at = slots(b, n)
        qb = s["q"][m:m + r].double().view(r, H, hd)
        m += r
        i = torch.arange(n - r, n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)
        hide = j > i
        if c["window"]:
            hide = hide | ((j <= i - c["window"]) & (j >= c["sinks"]))
        heads = []
        for h in range(H):
            g = h // (H // KV)
            kb, vb = (t[at, g * hd:(g + 1) * hd].double() for t in (K, V))
            x = (qb[:, h] @ kb.T).masked_fill(hide, -math.inf)
            p = torch.softmax(x, -1)
            heads.append(p @ vb)
            if c["weigh"]:
                w_out[b, :n] += p.sum(0)
        out.append(torch.cat(heads, -1))
    out = torch.cat(out)
    return (out, w_out) if c["weigh"] else out
