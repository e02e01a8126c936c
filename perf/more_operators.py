"""Performance cases of serving many requests together: attention of sequences
that share a long prefix of the paged cache, low-rank adapters of many
requests beside a shared projection, and head preparation into pages with
rotary positions of several axes. Each in its plain form (elementary torch
operations in 32 bits) and, where `own` is set, through the framework's calls.

A case is a dict of plain values:
  op      axes | shared | adapter
  seqs    sequences of the batch
  rows_lo, rows_hi  rows a sequence brings (0: one each), spread over their logarithm
axes and shared:
  heads, page       a key of HEADS; entries a page
  lo, hi            a sequence's entries before the batch's rows (shared: those
                    behind the prefix, the rows among them)
axes:
  sections          frequencies of each axis, "16,24,24"
  interleaved, norm
shared:
  groups            of neighbouring sequences; the last has what is left
  pre_lo, pre_hi    entries that a group shares, in whole pages
adapter:
  proj              a key of PROJ
  slots, rank_lo, rank_hi  adapters and their ranks
  bare              every bare-th sequence has no adapter (0: none of them)
"""
import math

import torch

own = False

DEV = "cuda"
THETA, EPS = 1.0e6, 1.0e-5
# query heads, KV heads, head size of the framework's own model shapes
HEADS = {"qwen2-0.5b": (14, 2, 64), "llama8b": (32, 8, 128), "lfm2-1.2b": (32, 8, 64)}
# inputs and outputs (of the parts that have a first factor of their own) of their projections
PROJ = {"qwen2-0.5b-qkv": (896, (896, 128, 128)), "qwen2-0.5b-o": (896, (896,)),
        "qwen2-0.5b-gate-up": (896, (4864, 4864)), "qwen2-0.5b-down": (4864, (896,)),
        "lfm2-1.2b-o": (2048, (2048,)), "lfm2-1.2b-gate-up": (2048, (8192, 8192)),
        "lfm2-1.2b-down": (8192, (2048,)), "llama8b-qkv": (4096, (4096, 1024, 1024)),
        "llama8b-o": (4096, (4096,)), "llama8b-gate-up": (4096, (14336, 14336)),
        "llama8b-down": (14336, (4096,))}
SECTIONS = {64: ["8,12,12", "12,10,10", "16,16", "32"], 128: ["16,24,24", "24,20,20", "32,32"]}


def _axes(name, heads, page, seqs, lo, hi, **more):
    c = {"op": "axes", "heads": heads, "page": page, "seqs": seqs, "lo": lo, "hi": hi,
         "rows_lo": 0, "rows_hi": 0, "sections": "16,24,24", "interleaved": False, "norm": False,
         **more}
    return {"name": name, **c} if name else c


def _shared(name, heads, page, seqs, groups, pre_lo, pre_hi, lo, hi, **more):
    c = {"op": "shared", "heads": heads, "page": page, "seqs": seqs, "groups": groups,
         "pre_lo": pre_lo, "pre_hi": pre_hi, "lo": lo, "hi": hi, "rows_lo": 0, "rows_hi": 0, **more}
    return {"name": name, **c} if name else c


def _adapter(name, proj, seqs, slots, rank_lo, rank_hi, **more):
    c = {"op": "adapter", "proj": proj, "seqs": seqs, "slots": slots, "rank_lo": rank_lo,
         "rank_hi": rank_hi, "rows_lo": 0, "rows_hi": 0, "bare": 0, **more}
    return {"name": name, **c} if name else c


def listed():
    return [
        # A token of each of 64 conversations about images served together.
        _axes("axes-step", "llama8b", 16, 64, 40, 8000),
        # Five prompts with an image each behind earlier turns, heads normalised.
        _axes("axes-images", "llama8b", 64, 5, 30, 6000, rows_lo=131, rows_hi=900,
              sections="24,20,20", interleaved=True, norm=True),
        # Three short chats behind one short system prompt: latency alone.
        _shared("shared-short", "qwen2-0.5b", 64, 3, 1, 64, 64, 7, 40),
        # A token of each of 64 conversations behind one system prompt with tools.
        _shared("shared-chat", "llama8b", 16, 64, 1, 6000, 6000, 40, 2000),
        # Five such prompts at once, each with its own conversations.
        _shared("shared-groups", "lfm2-1.2b", 32, 45, 5, 500, 5000, 20, 1500),
        # 32 questions about one long document.
        _shared("shared-long", "llama8b", 64, 32, 1, 100000, 100000, 10, 400),
        # A token and its drafts (3 to 8) of 16 conversations behind one prompt.
        _shared("shared-drafts", "llama8b", 64, 16, 1, 8000, 8000, 20, 900, rows_lo=4, rows_hi=9),
        # One request's token: latency alone.
        _adapter("adapter-one", "qwen2-0.5b-o", 1, 1, 8, 8),
        # A token of each of 64 requests of 40 adapters, every seventh without one.
        _adapter("adapter-step", "llama8b-qkv", 64, 40, 8, 64, bare=7),
        # A token of each of 24 requests, an adapter each, on a wide projection.
        _adapter("adapter-wide", "lfm2-1.2b-gate-up", 24, 24, 16, 16),
        # Five prompts of different adapters in one batch, odd lengths and ranks.
        _adapter("adapter-prompts", "llama8b-qkv", 5, 5, 11, 64, rows_lo=131, rows_hi=900),
        # A prompt of one adapter on the widest projection.
        _adapter("adapter-prompt-wide", "llama8b-gate-up", 1, 1, 32, 32, rows_lo=2048,
                 rows_hi=2048),
    ]


def draw(rng):
    def log(a, b):
        return max(a, min(b, round(math.exp(rng.uniform(math.log(a), math.log(b))))))

    op = rng.choice(["axes", "shared", "shared", "adapter", "adapter"])
    if op == "adapter":
        proj = rng.choice(sorted(PROJ))
        rank = log(4, 64)
        ranks = {"rank_lo": log(1, rank), "rank_hi": rank}
        if rng.random() < 0.5:
            seqs = log(1, 64)
            return _adapter(None, proj, seqs, log(1, seqs), bare=rng.choice([0, 0, 3, 10]), **ranks)
        seqs = log(1, 8)
        rows = log(8, 2048 // seqs)
        return _adapter(None, proj, seqs, log(1, seqs), rows_lo=log(1, rows), rows_hi=rows,
                        bare=rng.choice([0, 0, 3]), **ranks)
    heads, page = rng.choice(sorted(HEADS)), rng.choice([16, 32, 64, 128])
    if op == "axes":
        hi = log(1, 20000)
        prompts = rng.random() < 0.5
        return _axes(None, heads, page, log(1, 8) if prompts else log(1, 64), log(1, hi), hi,
                     rows_lo=log(1, 100) if prompts else 0, rows_hi=log(100, 400) if prompts else 0,
                     sections=rng.choice(SECTIONS[HEADS[heads][2]]),
                     interleaved=rng.random() < 0.5, norm=rng.random() < 0.5)
    seqs = log(2, 64)
    groups = log(1, max(1, seqs // 2))
    pre = log(page, 100000 // max(8, seqs))
    if rng.random() < 0.3:  # drafts
        seqs = min(seqs, 16)
        rows = log(2, 9)
        hi = log(rows + 1, 1000)
        return _shared(None, heads, page, seqs, min(groups, seqs), log(page, pre), pre,
                       log(rows, hi), hi, rows_lo=log(1, rows), rows_hi=rows)
    hi = log(2, 64000 // seqs)
    return _shared(None, heads, page, seqs, groups, log(page, pre), pre, log(1, hi), hi)


# ------------------------------------------------------------------ inputs

def _spread(lo, hi, n, by):
    """n whole numbers from lo to hi, even in their logarithm, out of order."""
    if n == 1:
        return [hi]
    while math.gcd(by, n) > 1:
        by += 1
    return [round(lo * (hi / lo) ** (i * by % n / (n - 1))) for i in range(n)]


def _rows(c):
    """Rows of each sequence."""
    return _spread(c["rows_lo"], c["rows_hi"], c["seqs"], 3) if c["rows_hi"] else [1] * c["seqs"]


def _groups(c):
    """(first sequence, one past the last, shared entries) of each group."""
    n, k, page = c["seqs"], c["groups"], c["page"]
    size = _spread(1, max(1, 2 * n // k - 1), k, 2)  # a few large ones and small ones
    edges, pre = [0], _spread(c["pre_lo"], c["pre_hi"], k, 2)
    for g in range(k):
        left = k - 1 - g  # (a sequence at least for each group to come)
        edges.append(n if left == 0 else min(edges[-1] + max(size[g], 1), n - left))
    return [(edges[g], edges[g + 1], max(1, pre[g] // page) * page) for g in range(k)]


def _lens(c):
    """Entries of each sequence, the batch's rows among them."""
    rows, lens = _rows(c), _spread(c["lo"], c["hi"], c["seqs"], 5)
    if c["op"] == "axes":
        return [n + r for n, r in zip(lens, rows)]
    pre = [p for a, b, p in _groups(c) for _ in range(a, b)]
    return [p + max(n, r) for p, n, r in zip(pre, lens, rows)]


def _slots(c):
    """Adapter of each sequence (-1: none)."""
    return [-1 if c["bare"] and i % c["bare"] == c["bare"] - 1 else (i * 7 + 3) % c["slots"]
            for i in range(c["seqs"])]


def _ranks(c):
    return _spread(c["rank_lo"], c["rank_hi"], c["slots"], 3)


def _axis_of(c, pairs):
    """Axis of each frequency."""
    s = [int(x) for x in c["sections"].split(",")]
    if not c["interleaved"]:
        return [a for a, n in enumerate(s) for _ in range(n)]
    n = len(s)  # frequency f is axis f % n's while that has frequencies left, then the first's
    return [f % n if f < n * s[f % n] else 0 for f in range(pairs)]


def _rope_table(hd, positions):
    """Cosines and sines: rows 0..1023 of those positions, row 1024 + i of
    position 1024 i, as the head preparation takes them."""
    r = torch.arange(1024 + (positions + 1023) // 1024, dtype=torch.float64, device=DEV)
    pos = torch.where(r < 1024, r, (r - 1024) * 1024)
    freq = THETA ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEV) / hd)
    a = pos[:, None] * freq
    return torch.cat([a.cos(), a.sin()], 1).float()


def _image_positions(at, rows, axes, seed):
    """Positions of `rows` rows from `at` on: text, an image of a few rows and
    columns of patches (time stands still), text behind its largest position."""
    out, p = [], at
    text = rows // 4
    side = max(1, int(math.sqrt(rows // 2))) + seed % 3
    for t in range(rows):
        if t < text or t >= text + side * side:
            out.append([p] * axes)
            p += 1
        else:
            i = t - text
            out.append([p, p + i // side, p + i % side][:axes] + [p] * (axes - 3))
            if i == side * side - 1 or t == rows - 1:
                p += side
    return out


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(rows):
    out = [0]
    for r in rows:
        out.append(out[-1] + r)
    return out


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows = _rows(c)
    s = {"c": c, "rows": rows, "row_start": _i32(_starts(rows)) if c["rows_hi"] else None}
    if c["op"] == "adapter":
        return _prepare_adapter(s, g)
    H, KV, hd = HEADS[c["heads"]]
    ps, n, M, lens = c["page"], c["seqs"], sum(rows), _lens(c)
    wide = -(-max(lens) // ps)
    groups = _groups(c) if c["op"] == "shared" else [(b, b + 1, 0) for b in range(n)]
    used = sum(p // ps + sum(-(-(x - p) // ps) for x in lens[a:b]) for a, b, p in groups)
    order = torch.randperm(used + 3, generator=g, device=DEV).tolist()
    table, at = [], 0
    for a, b, p in groups:
        first, at = order[at:at + p // ps], at + p // ps
        for x in lens[a:b]:
            mine = -(-(x - p) // ps)
            table.append(first + order[at:at + mine] + [-1] * (wide - p // ps - mine))
            at += mine
    s.update(lens=lens, groups=groups, table=_i32(table), lens_dev=_i32(lens),
             k=_randn(g, used + 3, ps, KV * hd, dtype=torch.float16),
             v=_randn(g, used + 3, ps, KV * hd, dtype=torch.float16))
    if c["op"] == "axes":
        axes = len(c["sections"].split(","))
        pos = [p for b, (x, r) in enumerate(zip(lens, rows))
               for p in _image_positions(x - r, r, axes, seed + b)]
        if not c["rows_hi"]:  # tokens behind an image: its patches took fewer positions
            shift = torch.randint(0, 40, (M, axes), generator=g, device=DEV).tolist()
            pos = [[max(0, x - d) for x, d in zip(p, e)] for p, e in zip(pos, shift)]
        s.update(pos=_i32(pos), qkv=_randn(g, M, (H + 2 * KV) * hd), rope=_rope_table(hd, 131072),
                 q_norm=1 + 0.1 * _randn(g, hd), k_norm=1 + 0.1 * _randn(g, hd),
                 axis_of=torch.tensor(_axis_of(c, hd // 2), device=DEV))
    else:
        s.update(q=_randn(g, M, H * hd) * (1.5 / math.sqrt(hd)),
                 group_start=_i32([a for a, _, _ in groups] + [n]),
                 shared=_i32([p for _, _, p in groups]))
    if own:
        from webgllm_amd import ops
        s["shape"] = ops.attn_shape(H, KV, hd, eps=EPS, use_norm=c.get("norm", False))
        s["cache"] = ops.PagedCache(s["k"], s["v"], s["table"], s["lens_dev"])
        if c["op"] == "axes":
            s["axes"] = ops.rope_axes([int(x) for x in c["sections"].split(",")],
                                      interleaved=c["interleaved"])
        else:
            s["scratch"] = ops.paged_shared_scratch(s["cache"], s["shape"], M, c["groups"])
    return s


def _prepare_adapter(s, g):
    c = s["c"]
    K, cols = PROJ[c["proj"]]
    M, N, parts = sum(s["rows"]), sum(cols), len(cols)
    ranks, slots = _ranks(c), _slots(c)
    most = -(-max(ranks) // 8) * 8
    s.update(K=K, cols=cols, ranks=ranks, slots=slots, slot=_i32(slots), rank=_i32(ranks),
             a=_randn(g, c["slots"], parts, most, K, dtype=torch.float16) / math.sqrt(K),
             b=_randn(g, c["slots"], N, most, dtype=torch.float16) * 0.05,
             scale=torch.tensor([16.0 / r for r in ranks], device=DEV),
             x=(_randn(g, M, K) / 32).half(), row_scale=32 * (1 + 0.1 * _randn(g, M)),
             y=_randn(g, M, N))
    if own:
        from webgllm_amd import ops
        s["adapters"] = ops.Adapters(s["a"], s["b"], s["rank"], s["scale"], cols)
        s["scratch"] = ops.adapter_scratch(s["adapters"], M)
    return s


# ------------------------------------------------------------------- a pass

def run(state):
    return {"axes": _run_axes, "shared": _run_shared, "adapter": _run_adapter}[
        state["c"]["op"]](state)


def _softmax(x):
    """Softmax over the last dim; zeros where nothing is visible."""
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    t = e.sum(-1, keepdim=True)
    return e / torch.where(t == 0, 1.0, t)


def _run_axes(s):
    c, qkv = s["c"], s["qkv"]
    H, KV, hd = HEADS[c["heads"]]
    if own:
        from webgllm_amd import ops
        q = ops.paged_head_prep(qkv, s["shape"], s["rope"], s["cache"], pos=s["pos"],
                                row_start=s["row_start"], q_norm=s["q_norm"] if c["norm"] else None,
                                k_norm=s["k_norm"] if c["norm"] else None, axes=s["axes"])
        return q, s["k"], s["v"]
    M, ps, lens = qkv.shape[0], c["page"], s["lens_dev"].long()
    b = m = torch.arange(M, device=DEV)
    if s["row_start"] is None:
        i = lens - 1
    else:
        start = s["row_start"].long()
        b = torch.searchsorted(start, m, right=True) - 1
        i = lens[b] - start[b + 1] + m
    page = s["table"][b, i // ps].long()
    x = qkv.view(M, H + 2 * KV, hd)
    qk, v = x[:, :H + KV], x[:, H + KV:]
    if c["norm"]:
        w = torch.cat([s["q_norm"].expand(H, hd), s["k_norm"].expand(KV, hd)])
        qk = qk * w * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS)
    freq = THETA ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64, device=DEV) / hd)
    a = s["pos"][:, s["axis_of"]].double() * freq
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    x1, x2 = qk[..., :hd // 2], qk[..., hd // 2:]
    r = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
    s["k"][page, i % ps] = r[:, H:].reshape(M, KV * hd).half()
    s["v"][page, i % ps] = v.reshape(M, KV * hd).half()
    return (r[:, :H] * (1.0 / math.sqrt(hd))).reshape(M, H * hd), s["k"], s["v"]


def _run_shared(s):
    c, q = s["c"], s["q"]
    H, KV, hd = HEADS[c["heads"]]
    if own:
        from webgllm_amd import ops
        return ops.paged_attn_shared(q, s["shape"], s["cache"], s["group_start"], s["shared"],
                                     row_start=s["row_start"], scratch=s["scratch"])
    G, ps, rows, lens = H // KV, c["page"], s["rows"], s["lens"]
    out, m0 = [], 0

    def entries(pool, table, first, count):
        """Entries first .. first + count - 1 of each table row: [rows, KV, count, hd]."""
        i = torch.arange(first, first + count, device=DEV)
        x = pool[table[:, i // ps].clamp(min=0).long(), i % ps].float()
        return x.view(x.shape[0], count, KV, hd).transpose(1, 2).contiguous()

    for a, b, p in s["groups"]:  # the prefix's keys and values once a group
        n, R, wide = b - a, max(rows[a:b]), max(x - p for x in lens[a:b])
        take = torch.tensor([[min(t, r - 1) for t in range(R)] for r in rows[a:b]], device=DEV)
        start = torch.tensor(_starts(rows[a:b]), device=DEV)
        count = start[1:] - start[:-1]
        qg = q[m0 + start[:-1, None] + take].view(n, R, KV, G, hd).permute(0, 2, 3, 1, 4)
        kp, vp = (entries(x, s["table"][a:a + 1], 0, p)[0] for x in (s["k"], s["v"]))
        ks, vs = (entries(x, s["table"][a:b], p, wide) for x in (s["k"], s["v"]))
        flat = qg.permute(1, 0, 2, 3, 4).reshape(KV, n * G * R, hd)
        x1 = (flat @ kp.transpose(1, 2)).view(KV, n, G * R, p).transpose(0, 1)
        x2 = qg.reshape(n, KV, G * R, hd) @ ks.transpose(2, 3)
        last = (s["lens_dev"][a:b].long() - count)[:, None] + take - p  # the rows' entries
        see = torch.arange(wide, device=DEV) <= last[..., None]
        x2 = torch.where(see[:, None, None], x2.view(n, KV, G, R, wide), -math.inf)
        w = _softmax(torch.cat([x1, x2.view(n, KV, G * R, wide)], -1))
        o = (w[..., :p].transpose(0, 1).reshape(KV, n * G * R, p) @ vp).view(KV, n, G * R, hd)
        live = torch.arange(wide, device=DEV) < (s["lens_dev"][a:b, None].long() - p)
        o = o.transpose(0, 1) + w[..., p:] @ torch.where(live[:, None, :, None], vs, 0.0)
        o = o.view(n, KV, G, R, hd).permute(0, 3, 1, 2, 4).reshape(n, R, H * hd)
        out.append(o[torch.arange(R, device=DEV) < count[:, None]])
        m0 += sum(rows[a:b])
    return torch.cat(out).half()


def _run_adapter(s):
    x, y, cols = s["x"], s["y"], s["cols"]
    if own:
        from webgllm_amd import ops
        return ops.adapter_add(y, x, s["adapters"], s["slot"], row_start=s["row_start"],
                               row_scale=s["row_scale"], scratch=s["scratch"])
    most, edges = s["a"].shape[2], _starts(cols)
    if s["row_start"] is None:  # a row a sequence: all their adapters in one product
        on = s["slot"].clamp(min=0).long()
        has = (s["slot"] >= 0)[:, None, None]
        f = torch.where(has[:, 0], (s["scale"][on] * s["row_scale"])[:, None], 0.0)
        t = (s["a"][on].float() @ x.float()[:, None, :, None])[..., 0]
        t = torch.where((torch.arange(most, device=DEV) < s["rank"][on, None])[:, None] & has, t,
                        0.0)
        for j in range(len(cols)):
            b = s["b"][on, edges[j]:edges[j + 1]].float()
            y[:, edges[j]:edges[j + 1]] += f * (b @ t[:, j, :, None])[..., 0]
        return y
    m = 0
    for r, at in zip(s["rows"], s["slots"]):
        if at >= 0:
            rank = s["ranks"][at]
            f = (s["scale"][at] * s["row_scale"][m:m + r])[:, None]
            for j in range(len(cols)):
                t = x[m:m + r].float() @ s["a"][at, j, :rank].float().T
                b = s["b"][at, edges[j]:edges[j + 1], :rank].float()
                y[m:m + r, edges[j]:edges[j + 1]] += f * (t @ b.T)
        m += r
    return y


# -------------------------------------------------------------- what it takes

def work(case):
    c = case
    rows = _rows(c)
    M = sum(rows)
    if c["op"] == "adapter":
        K, cols = PROJ[c["proj"]]
        N, parts, ranks, slots = sum(cols), len(cols), _ranks(c), _slots(c)
        on = [(r, ranks[a]) for r, a in zip(rows, slots) if a >= 0]
        return {"bytes": sum(r for r, _ in on) * (K * 2 + 4 + N * 8) +
                sum(ranks[a] for a in set(slots) if a >= 0) * (parts * K + N) * 2,
                "flops": sum(2 * r * k * (parts * K + N) for r, k in on)}
    H, KV, hd = HEADS[c["heads"]]
    entry = KV * hd * 2 * 2  # bytes of an entry's key and value
    if c["op"] == "axes":
        axes = len(c["sections"].split(","))
        return {"bytes": M * ((H + 2 * KV) * hd * 4 + H * hd * 4 + entry + 4 * axes + hd * 4),
                "flops": M * (H + KV) * hd * 8}
    read = pairs = 0
    lens = _lens(c)
    for a, b, p in _groups(c):
        read += p + sum(x - p for x in lens[a:b])
        pairs += sum(r * x - r * (r - 1) // 2 for r, x in zip(rows[a:b], lens[a:b]))
    return {"bytes": read * entry + M * H * hd * (4 + 2), "flops": 4 * pairs * H * hd}


# ------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c, rows = s["c"], s["rows"]
    if c["op"] == "adapter":
        y, m = s["y"].double(), 0
        part = [j for j, n in enumerate(s["cols"]) for _ in range(n)]
        part = torch.tensor(part, device=DEV)
        for r, at in zip(rows, s["slots"]):
            for t in range(m, m + r, 512) if at >= 0 else ():
                rank, end = s["ranks"][at], min(t + 512, m + r)
                xs = s["x"][t:end].double() * s["row_scale"][t:end, None].double()
                low = torch.stack([xs @ a.double().T for a in s["a"][at, :, :rank]])
                for j in range(low.shape[0]):
                    cut = part == j
                    y[t:end, cut] += s["scale"][at].double() * (
                        low[j] @ s["b"][at, cut, :rank].double().T)
            m += r
        return y
    H, KV, hd = HEADS[c["heads"]]
    ps, D = c["page"], KV * hd
    K, V = s["k"].view(-1, D), s["v"].view(-1, D)

    def places(b, n):
        """Rows of the pool that hold sequence b's first n entries."""
        pages = s["table"][b, :-(-n // ps)].long()
        return (pages[:, None] * ps + torch.arange(ps, device=DEV)).reshape(-1)[:n]

    m = 0
    if c["op"] == "axes":
        x = s["qkv"].double().view(-1, H + 2 * KV, hd)
        q, k, v = x.split([H, KV, KV], 1)
        if c["norm"]:
            q = q / (q.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["q_norm"].double()
            k = k / (k.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["k_norm"].double()
        turn = torch.empty(x.shape[0], hd // 2, dtype=torch.complex128, device=DEV)
        for f, axis in enumerate(_axis_of(c, hd // 2)):
            angle = s["pos"][:, axis].double() * THETA ** (-2.0 * f / hd)
            turn[:, f] = torch.complex(angle.cos(), angle.sin())

        def rotate(y):
            z = torch.complex(y[..., :hd // 2].contiguous(), y[..., hd // 2:].contiguous())
            z = z * turn[:, None]
            return torch.cat([z.real, z.imag], -1)

        q, k = rotate(q) / math.sqrt(hd), rotate(k)
        new_k, new_v = K.double(), V.double()
        for b, (n, r) in enumerate(zip(s["lens"], rows)):
            to = places(b, n)[n - r:]
            new_k[to], new_v[to] = k[m:m + r].reshape(r, D), v[m:m + r].reshape(r, D)
            m += r
        return q.reshape(-1, H * hd), new_k.view(s["k"].shape), new_v.view(s["v"].shape)
    out = []
    for b, (n, r) in enumerate(zip(s["lens"], rows)):
        at = places(b, n)
        hide = torch.arange(n, device=DEV) > torch.arange(n - r, n, device=DEV)[:, None]
        heads = []
        for h in range(KV):
            kb, vb = (t[at, h * hd:(h + 1) * hd].double() for t in (K, V))
            for e in range(H // KV):
                j = (h * (H // KV) + e) * hd
                w = s["q"][m:m + r, j:j + hd].double() @ kb.T
                heads.append(torch.softmax(w.masked_fill(hide, -math.inf), -1) @ vb)
        out.append(torch.cat(heads, -1))
        m += r
    return torch.cat(out)
