"""The paged cache on the GPU where rounding, values that are not finite and
work split between workgroups meet, against plain formulas in 64 bits."""
import pytest
import torch

from tests.test_paged_gpu import DEV, Case, _attend, _i32, _near, _sees

pytestmark = pytest.mark.gpu


def _starts(rows):
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    return start


@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (32, 8, 64), (32, 8, 128)])
@pytest.mark.parametrize("n", [1, 12, 60])
def test_prompt_weights_keep_their_bits(hip, H, KV, hd, n):
    """Rows of up to 40 entries whose values, 1 and -1 in turn, all but cancel:
    what rounding a weight to 11 bits would lose (some 2^-13 of the weights' sum
    at a few entries) is 2^-3 and more of the result. In blocks of each shape (by
    the batch's rows).
    Bound: half a step of the half output (2^-11, or 2^-25 below the normal
    halves); scores off by (2^-22 + hd 2^-24) S, S = sum |q_d k_d|, twice (a
    weight and the sum); an exponent, between 12 and 15 at most, rounded to
    2^-21 and its power to 2^-23, weights split at 2^-22, i + 1 additions of 2^-24
    in either sum: all under (i + 9) 2^-22 of sum w |v| = 1."""
    from webgllm_amd import ops
    R = 40
    c = Case([R] * n, KV, hd, 16, seed=21)
    sign = 1 - 2 * ((torch.arange(R, device=DEV)[:, None] + torch.arange(KV * hd, device=DEV)) % 2)
    for b in range(n):
        c.v.view(-1, KV * hd)[c.rows[b]] = sign.half()
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((n * R, H * hd), generator=c.g, device=DEV) * 0.1 / hd ** 0.5
    got = ops.paged_attn_prefill(q, shape, c.cache, _i32(_starts([R] * n)))
    hide = torch.ones((R, R), dtype=torch.bool, device=DEV).triu(1)
    for b in {0, n // 2, n - 1}:
        k, v = (x.repeat_interleave(H // KV, 1).transpose(0, 1).contiguous() for x in c.kv(b))
        qb = q[b * R:(b + 1) * R].double().view(R, H, hd).transpose(0, 1).contiguous()
        kt = k.transpose(1, 2).contiguous()
        p = torch.softmax((qb @ kt).masked_fill(hide, -torch.inf), -1)
        S = (qb.abs() @ kt.abs()).masked_fill(hide, 0).amax(-1)
        want = p @ v
        E = 2 * (2 ** -22 + hd * 2 ** -24) * S + (torch.arange(R, device=DEV) + 10) * 2 ** -22
        off = (got[b * R:(b + 1) * R].double().view(R, H, hd).transpose(0, 1) - want).abs()
        tol = 2 ** -11 * want.abs() + 2 ** -25 + E[..., None]
        assert (off <= tol).all(), (b, float((off - tol).max()))


def _bad_dim(rows, past, window, sinks, H, KV, hd, entry, dim, bad):
    """Prompts whose one value, of one KV head's dim, is not finite: that dim of
    the rows and query heads that see it is no number, everything else the sums
    in 64 bits (with 0 in that value's place)."""
    from webgllm_amd import ops
    lens = [p + r for p, r in zip(past, rows)]
    c = Case(lens, KV, hd, 64, seed=22)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((sum(rows), H * hd), generator=c.g, device=DEV) * 1.5 / hd ** 0.5
    at = (c.rows[0][entry], KV // 2 * hd + dim)
    v = c.v.view(-1, KV * hd)
    v[at] = 0.0
    kv = [c.kv(b) for b in range(len(rows))]
    v[at] = bad
    got = ops.paged_attn_prefill(q, shape, c.cache, _i32(_starts(rows)), window, sinks)
    first, G = 0, H // KV
    for b, (n, r) in enumerate(zip(lens, rows)):
        edge = [entry, entry + window] if b == 0 else []
        some = {0, 1, r // 3, r - 2, r - 1} | {i - past[b] + d for i in edge for d in (-1, 0, 1)}
        for t in sorted(some & set(range(r))):
            i = n - r + t
            hit = torch.zeros((H, hd), dtype=torch.bool, device=DEV)
            if b == 0 and entry in _sees(i, n, window, sinks):
                hit[KV // 2 * G:(KV // 2 + 1) * G, dim] = True
            hit, row = hit.view(-1), got[first + t]
            want, tol, _ = _attend(q[first + t].view(H, hd), kv[b][0][:i + 1], kv[b][1][:i + 1],
                                   i, window, sinks)
            assert not torch.isfinite(row[hit]).any(), (b, t)
            _near(row[~hit], want[~hit], tol[~hit], (b, t))
        first += r


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 64), (8, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("dim", [2, 5, 63])  # (in either lane of a query)
@pytest.mark.parametrize("entry,bad", [(40, float("nan")), (3500, float("inf")),
                                       (6002, float("nan")), (6004, float("-inf"))])
def test_prompt_one_dim_not_finite_in_shares(hip, H, KV, hd, dim, entry, bad):
    """Five rows behind 6000 entries, which several workgroups share: one value
    of one dim that is not finite leaves the other dims, and the rows that do not
    see it, their results."""
    _bad_dim([5], [6000], 0, 0, H, KV, hd, entry, dim, bad)


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 64), (32, 8, 128)])
@pytest.mark.parametrize("rows", [[300, 40], [1000, 77], [2600, 900]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (150, 7)])
@pytest.mark.parametrize("entry,bad", [(3, float("inf")), (9, float("nan")),
                                       (290, float("-inf"))])
def test_prompt_one_dim_not_finite_in_blocks(hip, H, KV, hd, rows, window, sinks, entry, bad):
    """The same in blocks of every shape (by the batch's rows), at both ends of
    the window and among the sinks."""
    _bad_dim(rows, [100, 0], window, sinks, H, KV, hd, entry, 37, bad)


def _ms(call):
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    times = []
    for _ in range(5):
        a.record()
        call()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return sorted(times)[2]


@pytest.mark.parametrize("what", ["value", "late value", "key", "query"])
def test_prompt_not_finite_costs_little(hip, what):
    """A chunk of 1024 rows behind 9000 entries takes about the same time where
    a value, a key or the queries are not finite (three times is far past what
    one such step or the clock's changes add, far under a second pass by row)."""
    from webgllm_amd import ops
    H, KV, hd = 32, 8, 128
    c = Case([10024], KV, hd, 64, seed=23)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((1024, H * hd), generator=c.g, device=DEV) * 1.5 / hd ** 0.5
    scratch = ops.paged_prefill_scratch(c.cache, shape, 1024)

    def call():
        ops.paged_attn_prefill(q, shape, c.cache, _i32([0, 1024]), scratch=scratch)

    call()
    clean = _ms(call)
    nan = float("nan")
    if what == "query":
        q.view(1024, H, hd)[::2, :, 5] = nan
    elif what == "key":
        c.k.view(-1, KV * hd)[c.rows[0][100]] = nan
    else:
        c.v.view(-1, KV * hd)[c.rows[0][100 if what == "value" else 9500]] = nan
    bad = _ms(call)
    assert bad <= 3 * clean, (bad, clean)


# ------------------------------------------------------------- decode attention

def test_decode_groups_in_any_order(hip):
    """Groups of 16, 4 and 16 query heads a KV head, whose workgroups take more,
    less and more LDS again."""
    from webgllm_amd import ops
    KV, hd = 2, 128
    c = Case([70, 9], KV, hd, 16, seed=25)
    for G in (16, 4, 16, 1, 9, 16):
        shape = ops.attn_shape(G * KV, KV, hd)
        q = torch.randn((2, G * KV * hd), generator=c.g, device=DEV) / hd ** 0.5
        got = ops.paged_attn_decode(q, shape, c.cache)
        for b, n in enumerate(c.lens):
            want, tol, _ = _attend(q[b].view(-1, hd), *c.kv(b), n - 1, 0, 0)
            _near(got[b], want, tol, (G, b))


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (40, 2, 128), (64, 4, 64)])
@pytest.mark.parametrize("weigh", [False, True])
def test_decode_joins_of_many_units(hip, H, KV, hd, weigh):
    """300 sequences of some hundred entries: most units are cut by a run's end,
    and a workgroup of the join takes several query heads in turn."""
    from webgllm_amd import ops
    n, page = 300, 32
    lens = [301 + 37 * b % 211 for b in range(n)]
    c = Case(lens, KV, hd, page, seed=26)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((n, H * hd), generator=c.g, device=DEV) * 1.5 / hd ** 0.5
    old = torch.rand((n, c.cache.max_entries), generator=c.g, device=DEV) if weigh else None
    w = old.clone() if weigh else None
    got = ops.paged_attn_decode(q, shape, c.cache, weights=w)
    for b in range(0, n, 3):
        k, v = c.kv(b)
        want, tol, p = _attend(q[b].view(H, hd), k, v, lens[b] - 1, 0, 0)
        _near(got[b], want, tol, b)
        if weigh:
            # a weight's relative error as _attend bounds it, and the sum's rounding
            kh = k.repeat_interleave(H // KV, 1)
            S = (kh.abs() * q[b].double().view(H, hd).abs()).sum(-1).amax()
            E = 2 * (2 ** -22 + hd * 2 ** -24) * S + 2 ** -12
            total = old[b, :lens[b]].double() + p.sum(0)
            off = (w[b, :lens[b]].double() - total).abs()
            assert (off <= E * p.sum(0) + 2 ** -24 * total).all(), (b, float(off.max()))
            assert torch.equal(w[b, lens[b]:], old[b, lens[b]:])
    assert torch.equal(got, ops.paged_attn_decode(q, shape, c.cache, weights=w))


@pytest.mark.parametrize("what", ["query", "key"])
def test_decode_weights_of_entries_without_a_page(hip, what):
    """Weights of entries that have no page stay as they are, bit for bit, where
    the row's own are not finite too."""
    from webgllm_amd import ops
    H, KV, hd, page = 8, 2, 64, 16
    c = Case([70, 50], KV, hd, page, seed=27)
    c.table[0, 1], c.table[1, 2] = -1, 10 ** 6
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((2, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    if what == "query":
        q[0, 3] = float("nan")
    else:
        c.k.view(-1, KV * hd)[c.rows[0][60], 5] = float("inf")
    w = torch.rand((2, c.cache.max_entries), generator=c.g, device=DEV)
    old = w.clone()
    ops.paged_attn_decode(q, shape, c.cache, weights=w)
    dead = torch.zeros_like(w, dtype=torch.bool)
    dead[0, 16:32] = dead[0, 70:] = dead[1, 32:48] = dead[1, 50:] = True
    assert torch.equal(w[dead], old[dead])
    assert not torch.isfinite(w[0, 60]) and torch.isfinite(w[1]).all()
    assert (w[1][~dead[1]] > old[1][~dead[1]]).any()


# ---------------------------------------------------------------------- eviction

@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("held", [float("nan"), 7.0])
def test_evicted_entries_without_a_page_are_zeros(hip, long, held):
    """What a new page held before, in the place of a kept entry that has no page,
    is not seen by the rows that follow: the entry is zeros there."""
    from webgllm_amd import ops
    H, KV, hd, page, keep = 8, 2, 64, 16, 48
    n = 20000 if long else 300  # (chunks, one workgroup)
    c = Case([n, 40], KV, hd, page, seed=24)
    c.table[0, 1], c.table[0, n // page] = -1, 2 ** 31 - 1
    c.table[1, 0] = 10 ** 6
    pool = [torch.full((7, page, KV * hd), held, dtype=torch.float16, device=DEV) for _ in range(2)]
    w = torch.zeros((2, c.cache.max_entries), device=DEV)  # (all equal: the first ones stay)
    new = _i32([[4, 0, 5], [1, 2, 6]])
    to, kept, _ = ops.paged_evict(c.cache, w, keep, new, sinks=4, recent=20, pool=tuple(pool))
    want = [list(range(keep - 20)) + list(range(n - 20, n)), list(range(40))]
    assert to.lens.tolist() == [keep, 40]
    assert [r[:m] for r, m in zip(kept.tolist(), (keep, 40))] == want
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((2, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    got = ops.paged_attn_decode(q, shape, to)
    dead = [set(range(16, 32)) | set(range(n // page * page, n)), set(range(16))]
    for b, (m, old) in enumerate(zip((keep, 40), (c.kv(0), c.kv(1)))):
        k, v = (x[want[b]].clone() for x in old)
        gone = torch.tensor([j in dead[b] for j in want[b]], device=DEV)
        k[gone], v[gone] = 0, 0
        at = new[b].long().repeat_interleave(page)[:m] * page + torch.arange(m, device=DEV) % page
        for x, y in zip((k, v), pool):
            assert torch.equal(y.view(-1, KV, hd)[at].double(), x), b
        out, tol, _ = _attend(q[b].view(H, hd), k, v, m - 1, 0, 0)
        _near(got[b], out, tol, b)


# ------------------------------------------------------------------ Python's checks

def test_numbers_past_32_bits_are_refused(hip):
    """Arguments that the library would take for another number."""
    from webgllm_amd import ops
    c = Case([20, 30], 2, 64, 16, seed=28)
    shape, big = ops.attn_shape(4, 2, 64), 2 ** 32
    q, w = torch.zeros((2, 256), device=DEV), torch.zeros((2, 99), device=DEV)
    start = _i32([0, 1, 2])
    far = torch.empty(big + 512, dtype=torch.float16, device=DEV).as_strided((2, 256), (big + 256, 1))
    for call in (lambda: ops.paged_attn_decode(q, shape, c.cache, window=big + 5),
                 lambda: ops.paged_attn_decode(q, shape, c.cache, window=9, sinks=big),
                 lambda: ops.paged_attn_prefill(q, shape, c.cache, start, window=big + 1),
                 lambda: ops.paged_attn_prefill(q, shape, c.cache, start, 9, sinks=-big),
                 lambda: ops.paged_evict(c.cache, w, big + 4, c.table),
                 lambda: ops.paged_evict(c.cache, w, 4, c.table, sinks=big),
                 lambda: ops.paged_evict(c.cache, w, 4, c.table, recent=big),
                 lambda: ops.PagedCache(c.k, c.v, c.table, c.cache.lens, max_entries=big + 9),
                 lambda: ops.paged_attn_decode(q, shape, c.cache, out=far)):
        with pytest.raises(ValueError, match="32 bits"):
            call()


def test_a_caches_tensors_change_in_place(hip):
    """Calls see lengths and tables changed in place; setting another tensor,
    which the calls would not see, is refused."""
    from webgllm_amd import ops
    H, KV, hd, page = 4, 2, 64, 16
    c = Case([40, 30], KV, hd, page, seed=29)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((2, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    for name in ("k", "v", "table", "lens", "max_entries"):
        with pytest.raises(AttributeError):
            setattr(c.cache, name, getattr(c.cache, name) + 1)
    c.cache.lens.sub_(7)
    c.cache.table[0, 0] = -1
    got = ops.paged_attn_decode(q, shape, c.cache)
    for b, n in enumerate((33, 23)):
        k, v = c.kv(b)
        want, tol, _ = _attend(q[b].view(H, hd), k[:n], v[:n], n - 1, 0, 0,
                               set(range(16)) if b == 0 else ())
        _near(got[b], want, tol, b)


# ------------------------------------------------------------------ what calls leave

def test_calls_leave_table_and_lengths(hip):
    """No call writes to the table or the lengths, with entries out of range among
    them, nor attention to the pages."""
    from webgllm_amd import ops
    H, KV, hd, page = 8, 2, 64, 16
    c = Case([100, 64, 48, 40], KV, hd, page, seed=30)
    c.table[0, 0], c.table[1, 1], c.table[3] = -1, 2 ** 31 - 1, -1
    c.cache.lens[2] = 2 ** 31 - 1
    shape = ops.attn_shape(H, KV, hd)
    held = [t.clone() for t in (c.table, c.cache.lens, c.k, c.v)]

    def same(n):
        return all(torch.equal(a.view(torch.int16) if a.dtype == torch.float16 else a,
                               b.view(torch.int16) if b.dtype == torch.float16 else b)
                   for a, b in list(zip((c.table, c.cache.lens, c.k, c.v), held))[:n])

    q = torch.randn((4, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    w = torch.zeros((4, c.cache.max_entries), device=DEV)
    ops.paged_attn_decode(q, shape, c.cache, 30, 4, weights=w)
    assert same(4)
    ops.paged_attn_prefill(q, shape, c.cache, _i32([0, 1, 2, 3, 4]))
    assert same(4)
    pool = torch.empty((8, page, KV * hd), dtype=torch.float16, device=DEV)
    ops.paged_evict(c.cache, w, 20, _i32(list(range(8))).view(4, 2), 2, 5, pool=(pool, pool.clone()))
    assert same(4)
    rope = torch.zeros((1030, hd), device=DEV)
    ops.paged_head_prep(torch.randn((4, (H + 2 * KV) * hd), device=DEV), shape, rope, c.cache)
    assert same(2)


@pytest.mark.parametrize("H,KV,hd,rows,splits", [
    (14, 2, 64, [3, 5, 1, 2], 42), (32, 8, 128, [3, 5, 1, 2], 8), (4, 4, 64, [3, 5, 1, 2], 42),
    (14, 2, 64, [40, 9, 130, 0], 5), (32, 8, 128, [40, 9, 130, 0], 1),
    (4, 4, 64, [40, 9, 130, 0], 16)])
def test_prompt_rows_are_shared_out(hip, H, KV, hd, rows, splits):
    """Few rows in a cache of up to 25,600 entries a sequence: the scratch holds
    `splits` parts a row and head (512 workgroups, or 256 where four waves of keys
    of 128 dims fill a compute unit, over the blocks of 32 queries of all KV heads);
    the row of 9000 entries leaves some, the row of 300 only their number."""
    from webgllm_amd import ops
    lens, page = [9000, 767, 5100, 300], 64
    c = Case(lens, KV, hd, page, seed=31)
    wide = torch.full((4, 400), -1, dtype=torch.int32, device=DEV)
    wide[:, :c.table.shape[1]] = c.table
    cache = ops.PagedCache(c.k, c.v, wide, _i32(lens))
    shape, M = ops.attn_shape(H, KV, hd), sum(rows) + 4
    scratch = ops.paged_prefill_scratch(cache, shape, M)
    assert scratch.numel() == (M * H * splits * (hd + 4) * 4 if splits > 1 else 16)
    start = _i32([2 + x for x in _starts(rows)])
    q = torch.randn((M, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    scratch.fill_(255)
    ops.paged_attn_prefill(q, shape, cache, start, scratch=scratch)
    if splits > 1:
        parts = scratch.view(torch.int32).view(M, H, splits, hd + 4)
        assert (parts[2, :, :2, :hd] != -1).all()  # (the first sequence's first row)
        assert int(parts[2, 0, 0, hd + 2]) > 1
        if rows[3]:
            assert (parts[M - 3, :, :, :hd] == -1).all() and int(parts[M - 3, 0, 0, hd + 2]) == 1
