"""Attention of sequences that share long prefixes (wg_paged_attn_shared) on the
GPU, against plain formulas in 64 bits and the calls that read every sequence
by itself. Every place of the pool that no row of a call sees holds NaN."""
import pytest
import torch

from tests.test_paged_gpu import DEV, GARBAGE, _attend, _gen, _i32, _near

pytestmark = pytest.mark.gpu


def _starts(rows):
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    return start


class Shared:
    """Groups [(shared entries, [entries behind them of each sequence])] in a
    pool of NaN, the shared ones in the same pages (whole ones of them). `room`
    entries a sequence at least (None: where nothing is run as a call that shares
    nothing): under 2048, rows of several tokens run as prompts, and up to 32 MiB
    of keys and values in all a row a sequence as tokens."""

    def __init__(self, groups, KV, hd, page, seed=0, room=None):
        from webgllm_amd import ops
        g = self.g = _gen(seed)
        self.KV, self.hd, self.page = KV, hd, page
        self.lens = [p + n for p, own in groups for n in own]
        if room is None:
            room = max(2100, (32 << 20) // (4 * KV * hd * len(self.lens)) + 1)
        wide = max(max(self.lens) // page + 2, -(-room // page))
        used = sum(p // page + sum(-(-(p % page + n) // page) for n in own) for p, own in groups)
        order = torch.randperm(used + 2, generator=g, device=DEV).tolist()
        table, at, D = [], 0, KV * hd
        for p, own in groups:
            first, at = order[at:at + p // page], at + p // page
            for n in own:
                mine = -(-(p % page + n) // page)
                row = first + order[at:at + mine]
                at += mine
                table.append(row + [GARBAGE[i % 4] for i in range(wide - len(row))])
        self.k = torch.full((used + 2, page, D), float("nan"), dtype=torch.float16, device=DEV)
        self.v = self.k.clone()
        self.table = _i32(table)
        self.rows = [torch.tensor([row[i // page] * page + i % page for i in range(n)],
                                  dtype=torch.long, device=DEV)
                     for row, n in zip(table, self.lens)]
        b = 0
        self.group_start, self.shared = [0], []
        for p, own in groups:
            for i, _ in enumerate(own):
                for pool in (self.k, self.v):
                    live = self.rows[b + i] if i == 0 else self.rows[b + i][p // page * page:]
                    pool.view(-1, D)[live] = torch.randn((live.numel(), D), generator=g,
                                                         device=DEV).half()
                    # (a page's entries before the first own one are copies)
                    tail = slice(p // page * page, p)
                    pool.view(-1, D)[self.rows[b + i][tail]] = pool.view(-1, D)[self.rows[b][tail]]
            b += len(own)
            self.group_start.append(b)
            self.shared.append(p)
        self.cache = ops.PagedCache(self.k, self.v, self.table, _i32(self.lens))

    def kv(self, b):
        D = self.KV * self.hd
        return tuple(p.view(-1, D)[self.rows[b]].double().view(-1, self.KV, self.hd)
                     for p in (self.k, self.v))

    def queries(self, H, M, scale=1.5):
        return torch.randn((M, H * self.hd + 8), generator=self.g, device=DEV)[
            :, :H * self.hd] * scale / self.hd ** 0.5

    def run(self, q, H, rows=None, **more):
        from webgllm_amd import ops
        start = None if rows is None else _i32(_starts(rows))
        return ops.paged_attn_shared(q, ops.attn_shape(H, self.KV, self.hd), self.cache,
                                     _i32(self.group_start), _i32(self.shared), start, **more)

    def check(self, got, q, H, rows=None, dead=(), only=None):
        m = 0
        for b, n in enumerate(self.lens):
            r = 1 if rows is None else rows[b]
            k, v = self.kv(b) if only is None or b in only else (None, None)
            for t in range(r):
                if k is not None:
                    want, tol, _ = _attend(q[m].reshape(H, self.hd), k, v, n - r + t, 0, 0, dead)
                    _near(got[m], want, tol, (b, t))
                m += 1


HEADS = [(14, 2, 64), (32, 8, 128), (32, 8, 64), (3, 3, 128), (32, 1, 64), (40, 2, 128), (20, 4, 64)]
GROUPS = [(64, [1, 2, 17, 33, 300]), (5, [1, 40]), (129, [1]), (1000, [7, 1, 64, 65, 31, 500, 2])]


@pytest.mark.parametrize("H,KV,hd", HEADS)
@pytest.mark.parametrize("page", [1, 16, 128])
@pytest.mark.parametrize("room", [None, 0])
def test_tokens(hip, H, KV, hd, page, room):
    """A token of each sequence, prefixes that end inside a page too."""
    c = Shared(GROUPS, KV, hd, page, seed=H, room=room)
    n = len(c.lens)
    q = c.queries(H, n)
    out = torch.full((n, H * hd + 2), 3.0, dtype=torch.float16, device=DEV)
    got = c.run(q, H, out=out[:, :H * hd])
    assert (out[:, H * hd:] == 3).all()
    c.check(got, q, H)
    assert torch.equal(got, c.run(q, H))


@pytest.mark.parametrize("H,KV,hd", HEADS)
@pytest.mark.parametrize("rows", [[1] * 15, [1, 5, 3, 0, 2, 1, 9, 1, 2, 1, 4, 4, 1, 7, 1],
                                  [1, 2, 1, 1, 60, 1, 2, 1, 7, 1, 1, 35, 0, 1, 2],
                                  [1, 2, 17, 33, 60, 1, 40, 1, 7, 1, 33, 65, 0, 100, 2]])
@pytest.mark.parametrize("room", [2100, 0])
def test_rows(hip, H, KV, hd, rows, room):
    """Several rows a sequence, up to all entries behind the prefix; rows behind
    the last sequence stay."""
    c = Shared(GROUPS, KV, hd, 16, seed=H + 1, room=room)
    q = c.queries(H, sum(rows) + 2)
    out = torch.full((sum(rows) + 2, H * hd), 3.0, dtype=torch.float16, device=DEV)
    got = c.run(q, H, rows, out=out)
    assert (got[sum(rows):] == 3).all()
    c.check(got, q, H, rows)
    out.fill_(3)
    assert torch.equal(got, c.run(q, H, rows, out=out))


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (14, 2, 64)])
@pytest.mark.parametrize("more", [0, 60])
def test_rows_before_the_first_sequence(hip, H, KV, hd, more):
    """Rows before the first sequence and behind the last stay, whatever scratch
    holds for them, and those between are as without."""
    from webgllm_amd import ops
    c = Shared(GROUPS, KV, hd, 16, seed=H + 7)
    rows = [1 + i % 3 for i in range(len(c.lens))]
    rows[1], rows[4] = 2, 0
    M, sh = sum(rows), ops.attn_shape(H, KV, hd)
    q = c.queries(H, 5 + M + more)
    starts, groups = _i32([5 + s for s in _starts(rows)]), (_i32(c.group_start), _i32(c.shared))
    want = c.run(q[5:5 + M], H, rows)
    c.check(want, q[5:5 + M], H, rows)
    sc = ops.paged_shared_scratch(c.cache, sh, len(q), len(c.shared))
    for fill in (0, 1, 127, 255):
        sc.fill_(fill)
        out = torch.full((len(q), H * hd), 3.0, dtype=torch.float16, device=DEV)
        ops.paged_attn_shared(q, sh, c.cache, *groups, starts, sc, out)
        assert (out[:5] == 3).all() and (out[5 + M:] == 3).all()
        c.check(out[5:5 + M], q[5:5 + M], H, rows)


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 128), (14, 2, 64)])
@pytest.mark.parametrize("rows", [None, 3])
def test_long_prefix(hip, H, KV, hd, rows):
    """Prefixes and ends of their own that are shared out over workgroups."""
    c = Shared([(20000, [1000, 5, 3, 9000]), (6016, [40] * 12), (7000, [3000])], KV, hd, 64, seed=3)
    rows = None if rows is None else [rows] * len(c.lens)
    q = c.queries(H, sum(rows) if rows else len(c.lens))
    got = c.run(q, H, rows)
    c.check(got, q, H, rows, only={0, 1, 3, 5, 15, 16})
    for _ in range(3):
        assert torch.equal(got, c.run(q, H, rows))


@pytest.mark.parametrize("rows", [None, 2])
def test_one_large_group_and_many_small_ones(hip, rows):
    """More sequences than a wave looks at once, in one group and in many."""
    H, KV, hd = 8, 2, 64
    for groups in ([(200, [1 + i % 37 for i in range(700)])],
                   [(64 + i % 100, [2 + (i + j) % 30 for j in range(1 + i % 4)]) for i in range(300)]):
        c = Shared([(p, [x + 1 for x in own]) for p, own in groups], KV, hd, 16, seed=4)
        r = None if rows is None else [rows] * len(c.lens)
        q = c.queries(H, sum(r) if r else len(c.lens))
        got = c.run(q, H, r)
        c.check(got, q, H, r, only=set(range(0, len(c.lens), 61)))


@pytest.mark.parametrize("rows", [None, 3])
def test_pools_past_32_bits(hip, rows):
    """Pages whose values lie past 2^32 bytes and 2^31 values of the pool."""
    from webgllm_amd import ops
    H, KV, hd, page = 32, 8, 128, 16
    c = Shared([(2000, [40, 5, 90]), (96, [300, 8])], KV, hd, page, seed=16, room=14000)
    n, most = c.k.shape[0], (2 ** 31 + 2 ** 27) // (page * KV * hd)
    pools = [torch.empty((most, page, KV * hd), dtype=torch.float16, device=DEV) for _ in range(2)]
    for pool, small in zip(pools, (c.k, c.v)):
        pool[most - n:] = small
    r = None if rows is None else [rows] * 5
    q = c.queries(H, 5 * (rows or 1))
    want = c.run(q, H, r)
    c.check(want, q, H, r)
    moved = torch.where((c.table >= 0) & (c.table < n), c.table + most - n, c.table)
    c.cache = ops.PagedCache(*pools, moved, c.cache.lens)
    assert torch.equal(c.run(q, H, r), want)


@pytest.mark.parametrize("rows", [None, 1])
@pytest.mark.parametrize("groups", [1, 32767, 65535])
@pytest.mark.parametrize("wide", [8, 600])
def test_the_most_sequences(hip, rows, groups, wide):
    """65,535 sequences behind 16 entries, in one group, in pairs, alone. The bound:
    scores off by 2^-20 of sum |q k|, so weights by as much, a weight's 21 bits and
    some 32 sums, and the result's half step."""
    from webgllm_amd import ops
    H, KV, hd, n = 2, 1, 64, 65535
    g = _gen(15)
    k = torch.randn((n + 4, 4, KV * hd), generator=g, device=DEV).half()
    v = torch.randn((n + 4, 4, KV * hd), generator=g, device=DEV).half()
    i = torch.arange(n, dtype=torch.int32, device=DEV)
    table = torch.full((n, wide), -1, dtype=torch.int32, device=DEV)
    table[:, :4], table[:, 4] = torch.arange(4, dtype=torch.int32, device=DEV), i + 4
    cache = ops.PagedCache(k, v, table, 17 + i % 4)
    starts = torch.linspace(0, n, groups + 1, device=DEV, dtype=torch.float64).int()
    shared = torch.full((groups,), 16, dtype=torch.int32, device=DEV)
    q = torch.randn((n, H * hd), generator=g, device=DEV) / 8
    row_start = None if rows is None else torch.arange(n + 1, dtype=torch.int32, device=DEV)
    got = ops.paged_attn_shared(q, ops.attn_shape(H, KV, hd), cache, starts, shared, row_start)
    for a in range(0, n, 8192):
        b = slice(a, min(a + 8192, n))
        at = table[b, :5].long()
        kk, vv = (t[at].view(-1, 20, hd).double() for t in (k, v))
        qq = q[b].double().view(-1, H, hd)
        hide = torch.arange(20, device=DEV) >= cache.lens[b, None]
        s = torch.matmul(qq, kk.transpose(1, 2).contiguous()).masked_fill(hide[:, None], -float("inf"))
        mag = torch.matmul(qq.abs(), kk.abs().transpose(1, 2).contiguous()).amax(2, keepdim=True)
        p = s.softmax(2)
        want, size = torch.matmul(p, vv), torch.matmul(p, vv.abs())
        tol = (2 ** -19 * mag + 2 ** -18) * size + 2 ** -11 * want.abs() + 2 ** -25
        off = (got[b].double().view(-1, H, hd) - want).abs()
        assert (off <= tol).all(), float((off - tol).max())


@pytest.mark.parametrize("rows", [False, True])
def test_sequences_that_end_in_the_prefix(hip, rows):
    """Empty sequences of a padded batch, ones whose rows begin inside the prefix,
    lengths out of range: their own pages throughout; the others as ever."""
    H, KV, hd = 8, 2, 64
    c = Shared([(160, [3, 9, 20, 1, 5, 30, 2])], KV, hd, 16, seed=5)
    lens = list(c.lens)
    lens[1], lens[3], lens[4], lens[6] = 0, 100, 160, -7
    c.cache.lens.copy_(_i32(lens))
    r = [2, 1, 9, 3, 2, 1, 1] if rows else None
    q = c.queries(H, sum(r) if rows else 7)
    got = c.run(q, H, r)
    c.lens = lens
    m = 0
    for b, n in enumerate(lens):
        for t in range(r[b] if rows else 1):
            i = n - (r[b] if rows else 1) + t
            if n <= 0 or i < 0:
                assert (got[m] == 0).all(), b
            else:
                k, v = (x[:n] for x in c.kv(b))
                want, tol, _ = _attend(q[m].reshape(H, hd), k, v, i, 0, 0)
                _near(got[m], want, tol, (b, t))
            m += 1


@pytest.mark.parametrize("rows", [None, 2])
@pytest.mark.parametrize("first", [1, 70, 75])
def test_groups_that_begin_with_empty_sequences(hip, rows, first):
    """The prefix is found where a group's first sequences are empty and their table
    rows name no pages; where all but one are, or all."""
    H, KV, hd = 8, 2, 64
    c = Shared([(96, [3 + i % 5 for i in range(75)]), (64, [9, 20])], KV, hd, 16, seed=13)
    lens = list(c.lens)
    lens[:first] = [0] * first
    c.cache.lens.copy_(_i32(lens))
    c.table[:first] = -1
    r = None if rows is None else [0] * first + [rows] * (77 - first)
    q = c.queries(H, 77 if r is None else sum(r))
    got = c.run(q, H, r)
    if r is None:
        assert (got[:first] == 0).all()
    for b in (first, 74, 75, 76):
        for t in range(rows or 1) if lens[b] else ():
            m = b if r is None else (b - first) * rows + t
            want, tol, _ = _attend(q[m].reshape(H, hd), *c.kv(b), lens[b] - (rows or 1) + t, 0, 0)
            _near(got[m], want, tol, (b, t))


@pytest.mark.parametrize("rows", [None, 4])
@pytest.mark.parametrize("starts,shared", [([0, 3, 3, 6], [320, 64, 100]), ([2, 5], [320]),
                                           ([0, 1, 2, 3, 4, 5, 6], [320] * 6),
                                           ([0, 6], [0]), ([0, 6], [-5]), ([0, 6], [2 ** 31 - 1]),
                                           ([0, 2, 6], [33, 319]), ([0, 6], [1])])
def test_groups_are_only_where_entries_are_read(hip, rows, starts, shared):
    """The same results whatever the groups: empty ones, sequences of no group,
    parts of what is shared, more than there is."""
    H, KV, hd = 14, 2, 64
    c = Shared([(320, [40, 5, 9, 300, 17, 64])], KV, hd, 16, seed=6)
    c.group_start, c.shared = starts, shared
    r = None if rows is None else [rows] * 6
    q = c.queries(H, 6 * (rows or 1))
    c.check(c.run(q, H, r), q, H, r)


@pytest.mark.parametrize("rows", [None, 3])
def test_missing_pages(hip, rows):
    """Shared entries and own ones without a page are not seen; a sequence of none
    gives zeros."""
    H, KV, hd, page = 8, 2, 64, 16
    c = Shared([(160, [40, 70, 33]), (64, [20, 9])], KV, hd, page, seed=7)
    c.table[:3, 2] = -1
    c.table[:3, 9] = 10 ** 6
    c.table[1, 11] = -2 ** 31
    c.table[3:] = -1
    r = None if rows is None else [rows] * 5
    q = c.queries(H, 5 * (rows or 1))
    got = c.run(q, H, r)
    gone = set(range(32, 48)) | set(range(144, 160))
    m = 0
    for b in range(5):
        for t in range(rows or 1):
            if b >= 3:
                assert (got[m] == 0).all()
            else:
                k, v = c.kv(b)
                dead = gone | (set(range(176, 192)) if b == 1 else set())
                want, tol, _ = _attend(q[m].reshape(H, hd), k, v, c.lens[b] - (rows or 1) + t, 0, 0, dead)
                _near(got[m], want, tol, (b, t))
            m += 1


@pytest.mark.parametrize("rows", [None, 3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite(hip, rows, bad):
    """In an own entry they reach that sequence alone, in a shared one its group
    alone; of an entry that a row does not see, nothing."""
    H, KV, hd = 8, 2, 64
    c = Shared([(96, [40, 70, 33]), (64, [20, 9, 50])], KV, hd, 16, seed=8)
    n, D = 6, KV * hd
    r = None if rows is None else [rows] * n
    per = rows or 1
    q = c.queries(H, n * per)
    want = c.run(q, H, r).clone()
    c.v.view(-1, D)[c.rows[1][120], :hd] = bad
    got = c.run(q, H, r)
    for b in range(n):
        sl = slice(b * per, b * per + per)
        if b == 1:
            assert not torch.isfinite(got[sl, :4 * hd]).any()
            assert torch.equal(got[sl, 4 * hd:], want[sl, 4 * hd:])
        else:
            assert torch.equal(got[sl], want[sl]), b
    c.v.view(-1, D)[c.rows[1][120], :hd] = 1
    c.v.view(-1, D)[c.rows[3][7], hd:] = bad
    if rows:  # the newest entry: the rows before it do not see it
        c.v.view(-1, D)[c.rows[5][113], :] = bad
    got = c.run(q, H, r)
    assert torch.isfinite(got[:3 * per]).all()
    assert not torch.isfinite(got[3 * per:, 4 * hd:]).any()
    if rows:
        assert torch.isfinite(got[3 * per:-1, :4 * hd]).all()
        assert not torch.isfinite(got[-1]).any()
    q[0, 5] = float("nan")
    got2 = c.run(q, H, r)
    assert not torch.isfinite(got2[0, :hd]).any() and torch.equal(got2[0, hd:], got[0, hd:])
    assert torch.equal(got2[1:3 * per], got[1:3 * per])


def test_large_queries_and_strong_entries(hip):
    """Queries far past the largest half; a strong entry in the prefix, and one
    behind it, over many weak ones."""
    H, KV, hd = 4, 2, 64
    c = Shared([(3000, [50, 90, 1])], KV, hd, 64, seed=9)
    q = c.queries(H, 3)
    q[0] *= 1e7
    q[1] *= 1e-9
    got = c.run(q, H)
    for b in range(3):
        k, v = c.kv(b)
        want, tol, p = _attend(q[b].reshape(H, hd), k, v, c.lens[b] - 1, 0, 0)
        if b == 0:  # scores near 1e8: one entry takes all the weight
            assert (p.amax(1) > 0.999999).all()
            tol = 2 ** -10 * want.abs() + 2 ** -24
        _near(got[b], want, tol, b)
    for at in (17, 3030):
        k0 = c.k.clone()
        q = c.queries(H, 3, 0.01)
        for h in range(KV):  # score 14 for the head's first query head
            d = q[0].view(H, hd)[h * 2].double()
            c.k.view(-1, KV, hd)[c.rows[0][at], h] = (14 * d / (d * d).sum()).clamp(-60000, 60000).half()
        c.check(c.run(q, H), q, H)
        c.k.copy_(k0)


@pytest.mark.parametrize("H,KV,hd", HEADS)
@pytest.mark.parametrize("page", [1, 8, 64])
@pytest.mark.parametrize("longer", [0, 1])
def test_short_sequences(hip, H, KV, hd, page, longer):
    """Caches as long as a workgroup takes a sequence whole, and longer: lengths of
    one, of all there is, none, out of range; pages that are missing; values that are
    not finite. A sequence's bits do not depend on the others'."""
    step = 128 // (4 if KV % 4 == 0 else 2 if KV % 2 == 0 else 1)
    most = step * (7 if hd == 64 else 5) // page * page
    own = [1, 2, step, step + 1, most - 40, 33, most // 2, 7, 9, 12, 5]
    c = Shared([(8, [n for n in own[:4]]), (40, [own[4]]), (0, own[5:])], KV, hd, page, seed=17, room=0)
    table = torch.full((len(own), most // page + longer), -1, dtype=torch.int32, device=DEV)
    n = min(table.shape[1], c.table.shape[1])
    table[:, :n] = c.table[:, :n]
    from webgllm_amd import ops
    c.cache = ops.PagedCache(c.k, c.v, table, c.cache.lens)
    lens = list(c.lens)
    lens[7], lens[8] = 0, -3
    c.cache.lens.copy_(_i32(lens))
    table[9] = -1
    D = KV * hd
    c.v.view(-1, D)[c.rows[10][2], :hd] = float("nan")
    q = c.queries(H, len(own))
    out = torch.full((len(own), H * hd + 4), 3.0, dtype=torch.float16, device=DEV)
    got = c.run(q, H, out=out[:, :H * hd])
    assert (out[:, H * hd:] == 3).all() and (got[7:10] == 0).all()
    for b in range(7):
        want, tol, _ = _attend(q[b].reshape(H, hd), *c.kv(b), lens[b] - 1, 0, 0)
        _near(got[b], want, tol, b)
    G = H // KV
    assert not torch.isfinite(got[10, :G * hd]).any() and torch.isfinite(got[10, G * hd:]).all()
    again = c.run(q, H)
    assert torch.equal(got[:10], again[:10])
    if not longer:
        lens[1], lens[2] = 0, 1
        c.cache.lens.copy_(_i32(lens))
        assert torch.equal(c.run(q, H)[3:7], got[3:7])


@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (32, 8, 128)])
def test_few_bytes_run_as_decode(hip, H, KV, hd):
    """Up to 32 MiB of keys and values a row a sequence has paged_attn_decode's
    bits, and its scratch is enough."""
    from webgllm_amd import ops
    most = (32 << 20) // (4 * KV * hd)
    for room in (most // 8, most // 8 + 1):
        c = Shared([(640, [30, 9, 1]), (96, [40, 8, 3, 2, 70])], KV, hd, 1, seed=14, room=room)
        shape, n = ops.attn_shape(H, KV, hd), 8
        assert c.cache.max_entries == room
        q = c.queries(H, n)
        got, want = c.run(q, H), ops.paged_attn_decode(q, shape, c.cache)
        need = [ops.paged_shared_scratch(c.cache, shape, n, 2), ops.paged_decode_scratch(c.cache, shape)]
        assert torch.equal(got, want) or room > most // 8
        assert (need[0].numel() <= need[1].numel()) == (room == most // 8)
        c.check(got, q, H)


@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("rows", [None, 5])
def test_as_the_calls_that_share_nothing(hip, H, KV, hd, rows):
    """Within two halves' steps of paged_attn_decode and paged_attn_prefill: each
    is within half a step, and 2^-12 of sum w |v| (under 2^-10 in all, for values of
    this size), of the sums in 64 bits."""
    from webgllm_amd import ops
    c = Shared([(1500, [30 + 9 * i for i in range(9)]), (96, [300, 8])], KV, hd, 32, seed=10)
    n, shape = len(c.lens), ops.attn_shape(H, KV, hd)
    r = None if rows is None else [rows] * n
    q = c.queries(H, n * (rows or 1))
    got = c.run(q, H, r).float()
    want = (ops.paged_attn_decode(q, shape, c.cache) if rows is None else
            ops.paged_attn_prefill(q, shape, c.cache, _i32(_starts(r)))).float()
    assert ((got - want).abs() <= 2 ** -10 * want.abs() + 2 ** -9).all()


def test_captured_step_follows_lengths_groups_and_pages(hip):
    """A step captured once and replayed as sequences grow, leave a group and the
    prefix changes; each replay as an eager call."""
    from webgllm_amd import ops
    H, KV, hd, page = 32, 8, 64, 16
    c = Shared([(640, [40, 5, 9]), (320, [100, 17, 64])], KV, hd, page, seed=11)
    shape = ops.attn_shape(H, KV, hd)
    q, starts, shared = c.queries(H, 6), _i32(c.group_start), _i32(c.shared)
    rows = _i32([0, 2, 3, 3, 6, 8, 9])
    q9 = c.queries(H, 9)
    sc = [ops.paged_shared_scratch(c.cache, shape, m, 2) for m in (6, 9)]
    got = [torch.zeros((m, H * hd), dtype=torch.float16, device=DEV) for m in (6, 9)]

    def step(out, scratch):
        ops.paged_attn_shared(q, shape, c.cache, starts, shared, scratch=scratch[0], out=out[0])
        ops.paged_attn_shared(q9, shape, c.cache, starts, shared, rows, scratch[1], out[1])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        step(got, sc)
    lens0 = c.cache.lens.clone()
    changes = [lambda: None, lambda: c.cache.lens.sub_(_i32([1, 2, 5, 40, 3, 60])),
               lambda: shared.copy_(_i32([100, 320])), lambda: starts.copy_(_i32([0, 5, 6])),
               lambda: (shared.copy_(_i32([0, 0])), c.cache.lens.copy_(lens0)),
               lambda: (starts.copy_(_i32([1, 3, 6])), shared.copy_(_i32([640, 320])))]
    for change in changes:
        change()
        for t in got:
            t.fill_(9)
        gr.replay()
        want = [torch.zeros_like(t) for t in got]
        step(want, [torch.full_like(x, 255) for x in sc])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.isfinite(a).all() and torch.equal(a, b)


def test_scratch_and_streams(hip):
    """What a scratch holds before does not matter; two streams with a scratch
    each at once."""
    from webgllm_amd import ops
    H, KV, hd = 32, 8, 128
    c = Shared([(2000, [40, 5, 9, 300])], KV, hd, 32, seed=12)
    shape = ops.attn_shape(H, KV, hd)
    q = c.queries(H, 4)
    want = c.run(q, H).clone()
    need = ops.paged_shared_scratch(c.cache, shape, 4, 1)
    for fill in (0, 255, 127):
        assert torch.equal(want, c.run(q, H, scratch=need.fill_(fill)))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for s in (a, b):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append([c.run(q, H) for _ in range(5)])
    a.synchronize(), b.synchronize()
    for out in outs[0] + outs[1]:
        assert torch.equal(out, want)


def test_python_checks(hip):
    from webgllm_amd import lib as L
    from webgllm_amd import ops
    c = Shared([(32, [3, 5])], 2, 64, 16)
    shape = ops.attn_shape(4, 2, 64)
    q, one, two = torch.zeros((2, 256), device=DEV), _i32([0, 2]), _i32([32])

    def call(q=q, starts=one, shared=two, **more):
        return ops.paged_attn_shared(q, shape, c.cache, starts, shared, **more)

    for more, msg in ((dict(starts=_i32([0])), "2 sequences"), (dict(q=q[:1]), "1 rows"),
                      (dict(q=q.half()), "float32"), (dict(shared=two.float()), "int32"),
                      (dict(q=q[:, :200]), "shorter"), (dict(shared=two.cpu()), "device"),
                      (dict(row_start=_i32([0, 1])), "row_start"),
                      (dict(out=torch.zeros((3, 256), dtype=torch.float16, device=DEV)), "out")):
        with pytest.raises(ValueError, match=msg):
            call(**more)
    with pytest.raises(L.WgError, match="scratch"):
        call(scratch=torch.empty(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(L.WgError, match="3 groups"):
        call(starts=_i32([0, 1, 1, 2]), shared=_i32([1, 1, 1]))
