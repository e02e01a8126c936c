"""The paged cache on the GPU (wg_paged_*) against plain formulas in 64 bits:
head preparation into pages, decode and prompt attention under windows with
sinks, the summed attention weights, and eviction. Every place of the pool
that no row of a call sees holds NaN."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
GARBAGE = (-1, 2 ** 31 - 1, -2 ** 31, 10 ** 6)  # table entries that name no page


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Case:
    """Sequences of `lens` entries in a pool of NaN: seen(b) of each filled."""

    def __init__(self, lens, KV, hd, page, seed=0, seen=None, spare=3):
        from webgllm_amd import ops
        g = self.g = _gen(seed)
        self.lens, self.KV, self.hd, self.page = lens, KV, hd, page
        counts = [-(-max(n, 0) // page) for n in lens]
        total = sum(counts) + spare
        self.wide = max(max(counts), 1) + 1
        order = torch.randperm(total, generator=g, device=DEV).tolist()
        table, at = [], 0
        for c in counts:
            table.append(order[at:at + c] + [GARBAGE[i % 4] for i in range(self.wide - c)])
            at += c
        self.spare = order[at:]
        D = KV * hd
        self.k = torch.full((total, page, D), float("nan"), dtype=torch.float16, device=DEV)
        self.v = self.k.clone()
        self.table, self.rows = _i32(table), []
        for b, n in enumerate(lens):
            r = [table[b][i // page] * page + i % page for i in range(n)]
            self.rows.append(torch.tensor(r, dtype=torch.long, device=DEV))
            live = self.rows[b] if seen is None else self.rows[b][
                torch.tensor(sorted(seen(b)), dtype=torch.long, device=DEV)]
            for pool in (self.k, self.v):
                pool.view(-1, D)[live] = torch.randn((live.numel(), D), generator=g,
                                                     device=DEV).half()
        self.cache = ops.PagedCache(self.k, self.v, self.table, _i32(lens))

    def kv(self, b):
        D = self.KV * self.hd
        return tuple(p.view(-1, D)[self.rows[b]].double().view(-1, self.KV, self.hd)
                     for p in (self.k, self.v))


def _sees(i, n, window, sinks):
    return [j for j in range(n) if j <= i and (not window or j < sinks or j > i - window)]


def _attend(q, k, v, i, window, sinks, dead=(), half_weights=False):
    """(output, error bound, weights [H, n]) of one row [H, hd] at entry i, in
    64 bits. The bound: half a step of the half output (2^-11, or 2^-25 below
    the normal halves), and what float32 scores and sums allow. A score's
    error is at most (2^-22 + hd 2^-24) S, S = sum |q_d k_d| (its query holds
    22 bits; hd additions); a weight's relative error twice that; the sums of
    weights and of weighted values add at most 2^-12 (some 2^12 additions of
    half a 2^-23 step), all of sum w |v|. half_weights (prompts): each weight
    is rounded to a half once, which is off by at most 2^-11 of it, or by 2^-25
    below the normal halves; the largest so far is 2^12 at least, and so is the
    sum: that adds 2^-11 sum w |v| + 2^-37 sum |v|."""
    H, hd = q.shape
    n, KV = k.shape[0], k.shape[1]
    see = torch.tensor([j for j in _sees(i, n, window, sinks) if j not in dead],
                       dtype=torch.long, device=DEV)
    w = torch.zeros((H, n), dtype=torch.float64, device=DEV)
    if not see.numel():
        return torch.zeros(H * hd, device=DEV).double(), torch.zeros(H * hd, device=DEV).double(), w
    kh, vh = (x[see].repeat_interleave(H // KV, 1).transpose(0, 1) for x in (k, v))
    q = q.double()
    p = torch.softmax((kh @ q[:, :, None])[..., 0], -1)
    S = (kh.abs() @ q.abs()[:, :, None]).amax((1, 2))
    E = 2 * (2 ** -22 + hd * 2 ** -24) * S + 2 ** -12
    out, mag = (p[:, None] @ vh)[:, 0], (p[:, None] @ vh.abs())[:, 0]
    w[:, see] = p
    tol = 2 ** -11 * out.abs() + 2 ** -25 + E[:, None] * mag
    if half_weights:
        tol = tol + 2 ** -11 * mag + 2 ** -37 * vh.abs().sum(1)
    return out.reshape(-1), tol.reshape(-1), w


def _near(got, want, tol, what=""):
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    assert (off <= tol).all(), (what, float((off - tol).max()), float(off.max()))


# ------------------------------------------------------------ head preparation

def _rope(theta, hd, ctx):
    from webgllm_amd.engine import _rope_table
    return _rope_table(theta, hd, ctx).to(DEV)


@pytest.mark.parametrize("H,KV,hd,rot,norm", [(14, 2, 64, 64, False), (32, 8, 128, 128, True),
                                              (32, 8, 64, 64, True), (6, 3, 64, 32, True),
                                              (4, 2, 96, 96, False), (2, 1, 128, 0, True),
                                              (4, 4, 256, 256, True), (3, 1, 8, 8, False)])
@pytest.mark.parametrize("page", [1, 16, 128])
def test_head_prep_bits(hip, H, KV, hd, rot, norm, page):
    """Every row as wg_head_prep writes it into a contiguous cache, bit for
    bit; nothing else of the pool changes."""
    from webgllm_amd import ops
    g = _gen(1)
    rows = [5, 0, 1, 40, 0, 2, 0]
    past = [0, 7, 1100, 3, 0, 64, 0]
    lens = [p + r for p, r in zip(past, rows)]
    c = Case(lens, KV, hd, page, seen=lambda b: ())
    M = sum(rows) + 3  # rows behind the last sequence
    shape = ops.attn_shape(H, KV, hd, rot, 1e-5, norm)
    wide = (H + 2 * KV) * hd
    qkv = torch.randn((M, wide + 16), generator=g, device=DEV)[:, :wide]
    rope = _rope(1e6, hd, 4096)
    qn, kn = (1 + 0.1 * torch.randn(hd, generator=g, device=DEV) for _ in range(2))
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    pos = _i32([p + i + 700 for p, r in zip(past, rows) for i in range(r)] + [1, 2, 3])
    for ahead in (False, True):
        c.k.fill_(float("nan")), c.v.fill_(float("nan"))
        q_out = torch.full((M, H * hd + 4), 7.0, device=DEV)[:, :H * hd]
        ops.paged_head_prep(qkv, shape, rope, c.cache, pos=pos if ahead else None,
                            row_start=_i32(start), q_norm=qn, k_norm=kn, q_out=q_out)
        assert (q_out[start[-1]:] == 7).all()
        left = torch.ones(c.k.shape[0] * page, dtype=torch.bool, device=DEV)
        for b, r in enumerate(rows):
            if not r:
                continue
            ck = torch.full((4096, KV * hd), float("nan"), dtype=torch.float16, device=DEV)
            cv = ck.clone()
            p0 = past[b] + (700 if ahead else 0)
            sl = slice(start[b], start[b] + r)
            want = ops.head_prep(qkv[sl].contiguous(), shape, rope, _i32([p0]), ck, cv, qn, kn)
            assert torch.equal(q_out[sl], want), b
            at = c.rows[b][past[b]:]
            left[at] = False
            for pool, cc in ((c.k, ck), (c.v, cv)):
                assert torch.equal(pool.view(-1, KV * hd)[at], cc[p0:p0 + r]), b
        for pool in (c.k, c.v):
            assert torch.isnan(pool.view(-1, KV * hd)[left]).all()


@pytest.mark.parametrize("hd", [64, 96])
def test_head_prep_rows_without_an_entry(hip, hd):
    """A padded decode batch (an empty sequence), a missing page, positions
    that the rope table does not hold: zero queries, nothing stored."""
    from webgllm_amd import ops
    H, KV, page = 4, 2, 16
    c = Case([3, 0, 20, 33, 5], KV, hd, page, seen=lambda b: ())
    c.table[2, 1] = -1
    shape = ops.attn_shape(H, KV, hd)
    qkv = torch.randn((5, (H + 2 * KV) * hd), generator=_gen(2), device=DEV)
    pos = _i32([2, 0, 19, 1 << 20, -1])
    q = ops.paged_head_prep(qkv, shape, _rope(1e4, hd, 2048), c.cache, pos=pos)
    assert (q[1:] == 0).all() and (q[0] != 0).any()
    for pool in (c.k, c.v):
        wrote = ~torch.isnan(pool).all(-1).view(-1)
        assert wrote.nonzero()[:, 0].tolist() == [int(c.rows[0][2])]


def test_head_prep_more_rows_than_entries(hip):
    """Rows before a sequence's first entry (a length cut short) get zero
    queries; the others keep their entries."""
    from webgllm_amd import ops
    H, KV, hd, page = 4, 2, 64, 16
    c = Case([3, 9], KV, hd, page, seen=lambda b: ())
    shape = ops.attn_shape(H, KV, hd)
    qkv = torch.randn((9, (H + 2 * KV) * hd), generator=_gen(3), device=DEV)
    q = ops.paged_head_prep(qkv, shape, _rope(1e4, hd, 2048), c.cache, row_start=_i32([0, 5, 9]))
    assert (q[:2] == 0).all() and (q[2:] != 0).any(1).all()
    wrote = ~torch.isnan(c.v).all(-1).view(-1)
    assert sorted(wrote.nonzero()[:, 0].tolist()) == sorted(
        c.rows[0].tolist() + c.rows[1][5:].tolist())


# ------------------------------------------------------------- decode attention

LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 1025]


@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (32, 8, 128), (32, 8, 64), (3, 3, 128),
                                     (64, 1, 64), (40, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (16, 4), (33, 40), (100, 0),
                                          (2 ** 31 - 1, 5)])
def test_decode(hip, H, KV, hd, window, sinks):
    from webgllm_amd import ops
    page = {14: 16, 32: 64, 3: 8, 64: 1, 40: 256}[H]
    c = Case(LENS, KV, hd, page, seed=window % 97 + sinks,
             seen=lambda b: _sees(LENS[b] - 1, LENS[b], window, sinks))
    n = len(LENS)
    shape = ops.attn_shape(H, KV, hd)
    q = (torch.randn((n, H * hd + 8), generator=c.g, device=DEV) * 1.5 / hd ** 0.5)[:, :H * hd]
    out = torch.full((n, H * hd + 2), 3.0, dtype=torch.float16, device=DEV)
    w = torch.randn((n, c.cache.max_entries + 5), generator=c.g, device=DEV)
    w0 = w.clone()
    got = ops.paged_attn_decode(q, shape, c.cache, window, sinks, out=out[:, :H * hd])
    again = ops.paged_attn_decode(q, shape, c.cache, window, sinks, weights=w)
    assert torch.equal(got, again) and (out[:, H * hd:] == 3).all()
    for b, x in enumerate(LENS):
        want, tol, p = _attend(q[b].view(H, hd), *c.kv(b), x - 1, window, sinks)
        _near(got[b], want, tol, b)
        add = (w[b].double() - w0[b].double())
        seen = _sees(x - 1, x, window, sinks)
        unseen = torch.ones(w.shape[1], dtype=torch.bool, device=DEV)
        unseen[seen] = False
        assert (add[unseen] == 0).all(), b
        if seen:
            # weights: relative error as _attend derives it (S below 40: at
            # most 2^-11), half a step of the sum per addition
            ref = p.sum(0)[seen]
            off = (add[seen] - ref).abs()
            assert (off <= 2 ** -11 * ref + 2 ** -23 * (w[b, seen].abs() + ref)).all(), b


def test_decode_long_splits(hip):
    """Entries of one long and some short sequences, all split and joined:
    against 64 bits, the same bits at every call."""
    from webgllm_amd import ops
    H, KV, hd = 32, 8, 128
    lens = [40001, 1, 3000, 17]
    c = Case(lens, KV, hd, 32, seed=5)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((4, H * hd), generator=c.g, device=DEV) * 1.5 / hd ** 0.5
    for window, sinks in ((0, 0), (20000, 7)):
        got = ops.paged_attn_decode(q, shape, c.cache, window, sinks)
        for _ in range(3):
            assert torch.equal(got, ops.paged_attn_decode(q, shape, c.cache, window, sinks))
        for b, x in enumerate(lens):
            k, v = c.kv(b)
            i = torch.arange(x, device=DEV)
            see = (i >= x - window) | (i < sinks) if window else i >= 0
            want, tol, _ = _attend(q[b].view(H, hd), k[see], v[see], int(see.sum()) - 1, 0, 0)
            _near(got[b], want, tol, b)


def test_decode_many_sequences(hip):
    """More sequences than workgroups, most of them empty."""
    from webgllm_amd import ops
    H, KV, hd, n = 4, 2, 64, 3000
    lens = [(i * 7 % 50 if i % 9 == 0 else 0) for i in range(n)]
    c = Case(lens, KV, hd, 16, seed=6)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((n, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    got = ops.paged_attn_decode(q, shape, c.cache)
    for b in (0, 9, 18, 2997, 1, 2, 2999, 1503):
        want, tol, _ = _attend(q[b].view(H, hd), *c.kv(b), lens[b] - 1, 0, 0)
        _near(got[b], want, tol, b)
    empty = torch.tensor([x == 0 for x in lens], device=DEV)
    assert (got[empty] == 0).all()


def test_decode_missing_pages_and_lengths_out_of_range(hip):
    """A table entry that names no page hides its entries, a length past
    max_entries or below 0 is cut."""
    from webgllm_amd import ops
    H, KV, hd, page = 8, 2, 64, 16
    c = Case([100, 64, 48, 40], KV, hd, page, seed=7)
    full = c.table.clone()
    for row, col, bad in ((0, 0, -1), (0, 3, 10 ** 6), (0, 6, -2 ** 31), (1, 1, 2 ** 31 - 1)):
        c.table[row, col] = bad
    c.table[3] = -1
    cache = ops.PagedCache(c.k, c.v, c.table, _i32([100, 64, 2 ** 31 - 1, 40]),
                           max_entries=100)
    c.table[2, 3:] = -1
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((4, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    w = torch.zeros((4, 100), device=DEV)
    got = ops.paged_attn_decode(q, shape, cache, weights=w)
    dead = [set(range(16)) | set(range(48, 64)) | set(range(96, 100)), set(range(16, 32)), (), ()]
    for b, n in enumerate((100, 64, 48)):
        want, tol, p = _attend(q[b].view(H, hd), *c.kv(b), n - 1, 0, 0, dead[b])
        _near(got[b], want, tol, b)
        assert (w[b, :n].double() - p.sum(0)).abs().max() <= 2 ** -11 * H
        assert all(float(w[b, j]) == 0 for j in dead[b])
    assert (got[3] == 0).all() and (w[3] == 0).all()
    cache.lens[0] = -5
    assert (ops.paged_attn_decode(q, shape, cache)[0] == 0).all()
    assert full.shape == c.table.shape


def test_decode_values_that_are_not_finite(hip):
    """A sequence that sees a value that is not finite gives no number there;
    the others keep their bits."""
    from webgllm_amd import ops
    H, KV, hd = 8, 2, 64
    c = Case([70, 90, 33], KV, hd, 16, seed=8)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((3, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    want = ops.paged_attn_decode(q, shape, c.cache)
    c.v.view(-1, KV * hd)[c.rows[1][50], :hd] = float("inf")
    c.k.view(-1, KV * hd)[c.rows[1][20], hd:] = float("nan")
    got = ops.paged_attn_decode(q, shape, c.cache)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert not torch.isfinite(got[1]).any()
    q[0, 5] = float("nan")
    got = ops.paged_attn_decode(q, shape, c.cache)
    assert not torch.isfinite(got[0, :hd]).any() and torch.equal(got[0, hd:], want[0, hd:])


def test_decode_large_queries_and_scores(hip):
    """Queries far past the largest half, and far below the smallest: the
    softmax of their scores all the same."""
    from webgllm_amd import ops
    H, KV, hd = 4, 2, 64
    c = Case([50, 50, 50], KV, hd, 16, seed=9)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((3, H * hd), generator=c.g, device=DEV)
    q[0] *= 1e7
    q[1] *= 1e-9
    q[2] = 0
    got = ops.paged_attn_decode(q, shape, c.cache)
    for b in range(3):
        k, v = c.kv(b)
        want, tol, p = _attend(q[b].view(H, hd), k, v, 49, 0, 0)
        if b == 0:  # scores near 1e8: one entry takes all the weight
            assert (p.amax(1) > 0.999999).all()
            tol = 2 ** -10 * want.abs() + 2 ** -24
        _near(got[b], want, tol, b)


def test_pool_past_32_bits(hip):
    """Pages past 4 GiB of a pool: preparation, both attentions, eviction."""
    from webgllm_amd import ops
    H, KV, hd, page = 8, 8, 128, 64
    pages = (5 << 30) // (page * KV * hd * 2)
    k = torch.zeros((pages, page, KV * hd), dtype=torch.float16, device=DEV)
    v = torch.zeros_like(k)
    table = _i32([[pages - 1, 1, pages - 2]])
    cache = ops.PagedCache(k, v, table, _i32([150]))
    shape = ops.attn_shape(H, KV, hd)
    g = _gen(10)
    qkv = torch.randn((150, 3 * H * hd), generator=g, device=DEV)
    q = ops.paged_head_prep(qkv, shape, _rope(1e4, hd, 1024), cache, row_start=_i32([0, 150]))
    flat = torch.cat([torch.arange(page, device=DEV) + p * page for p in (pages - 1, 1, pages - 2)])
    kk, vv = (t.view(-1, KV * hd)[flat[:150]].double().view(150, KV, hd) for t in (k, v))
    assert torch.equal(vv.view(150, -1).half(), qkv[:, 2 * H * hd:].half())
    dec = ops.paged_attn_decode(q[149:].contiguous(), shape, cache)
    pre = ops.paged_attn_prefill(q, shape, cache, _i32([0, 150]))
    for i in (0, 70, 149):
        want, tol, _ = _attend(q[i].view(H, hd), kk, vv, i, 0, 0, half_weights=True)
        _near(pre[i], want, tol, i)
    _near(dec[0], want, tol)
    w = torch.rand((1, cache.max_entries), generator=g, device=DEV)
    to, kept, _ = ops.paged_evict(cache, w, 100, _i32([[5, pages - 9]]), 4, 20)
    src = flat[kept[0].long()]
    dst = torch.cat([torch.arange(page, device=DEV) + p * page for p in (5, pages - 9)])[:100]
    for t in (k, v):
        assert torch.equal(t.view(-1, KV * hd)[src], t.view(-1, KV * hd)[dst])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("strong", [0, 17, 69_000])
def test_many_weak_entries_behind_a_strong_one(hip, hd, strong):
    """70,000 entries whose weights are e^-18 of one entry's, so each under the
    halves' smallest step beside it: their sum, 1e-3, counts."""
    from webgllm_amd import ops
    H, KV, page, n = 8, 2, 64, 70_000
    c = Case([n], KV, hd, page, seed=strong)
    D = KV * hd
    k, v = (torch.zeros((n, KV, hd), device=DEV) for _ in range(2))
    k[strong, :, 0] = 18.0
    v[:] = torch.rand((KV, hd), generator=c.g, device=DEV) + 0.5
    v[strong] = 0.0
    c.k.view(-1, D)[c.rows[0]] = k.view(n, D).half()
    c.v.view(-1, D)[c.rows[0]] = v.view(n, D).half()
    kk, vv = c.kv(0)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.zeros((3, H, hd), device=DEV)
    q[:, :, 0] = torch.linspace(0.9, 1.0, 3, device=DEV)[:, None]
    q = q.view(3, H * hd)
    pre = ops.paged_attn_prefill(q, shape, c.cache, _i32([0, 3]))
    for i in range(3):
        want, tol, _ = _attend(q[i].view(H, hd), kk, vv, n - 3 + i, 0, 0, half_weights=True)
        assert (want > 1e-4).all()
        _near(pre[i], want, tol, i)
    want, tol, _ = _attend(q[2].view(H, hd), kk, vv, n - 1, 0, 0)
    _near(ops.paged_attn_decode(q[2:], shape, c.cache)[0], want, tol)


# ------------------------------------------------------------- prompt attention

def _check_prompt(c, q, got, rows, H, window, sinks, every=1):
    m = 0
    for b, (n, r) in enumerate(zip(c.lens, rows)):
        k, v = c.kv(b)
        for t in range(r):
            if t % every == 0 or t == r - 1:
                want, tol, _ = _attend(q[m + t].view(H, -1), k, v, n - r + t, window, sinks,
                                       half_weights=True)
                _near(got[m + t], want, tol, (b, t))
        m += r


@pytest.mark.parametrize("window", [0, 100, 4096, 2**31 - 1])
def test_more_rows_than_entries(hip, window):
    """A batch of more rows than its sequence has entries: the rows before the
    first entry get zeros, the others see what is there, under any window."""
    from webgllm_amd import ops
    H, KV, hd, n, M = 8, 2, 64, 70, 100
    c = Case([n], KV, hd, 16, seed=window % 97)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((M, H * hd), generator=c.g, device=DEV) * 1.5 / hd ** 0.5
    got = ops.paged_attn_prefill(q, shape, c.cache, _i32([0, M]), window, 2)
    assert (got[:M - n] == 0).all()
    k, v = c.kv(0)
    for i in range(0, n, 7):
        want, tol, _ = _attend(q[M - n + i].view(H, hd), k, v, i, window, 2, half_weights=True)
        _near(got[M - n + i], want, tol, i)
    want, tol, _ = _attend(q[-1].view(H, hd), k, v, n - 1, window, 2)
    _near(ops.paged_attn_decode(q[-1:], shape, c.cache, window, 2)[0], want, tol)


@pytest.mark.parametrize("H,KV,hd", [(14, 2, 64), (32, 8, 128), (4, 4, 64)])
@pytest.mark.parametrize("rows", [[3, 5, 1, 2], [40, 9, 130, 0]])
def test_prompt_shares_by_length(hip, H, KV, hd, rows):
    """Few rows in a cache that could hold much more: long sequences are split
    over workgroups, short ones are not, in one call, whatever the scratch held."""
    from webgllm_amd import ops
    page, lens = 64, [9000, 767, 5100, 300]
    c = Case(lens, KV, hd, page, seed=3)
    wide = torch.full((4, 400), -1, dtype=torch.int32, device=DEV)
    wide[:, :c.table.shape[1]] = c.table
    cache = ops.PagedCache(c.k, c.v, wide, _i32(lens))
    shape, M = ops.attn_shape(H, KV, hd), sum(rows) + 4
    start = [2]
    for r in rows:
        start.append(start[-1] + r)
    q = torch.randn((M, H * hd), generator=c.g, device=DEV) * 1.5 / hd ** 0.5
    scratch = ops.paged_prefill_scratch(cache, shape, M)
    assert scratch.numel() > 16 or M > 100
    outs = []
    for fill in (0, 127, 255):  # (as counts of shares: none, huge ones, NaN)
        scratch.fill_(fill)
        out = torch.full((M, H * hd), 3.0, dtype=torch.float16, device=DEV)
        ops.paged_attn_prefill(q, shape, cache, _i32(start), scratch=scratch, out=out)
        assert (out[:2] == 3).all() and (out[-2:] == 3).all()
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    _check_prompt(c, q[2:], outs[0][2:], rows, H, 0, 0, 11)


@pytest.mark.parametrize("H,KV,hd,page", [(14, 2, 64, 16), (32, 8, 128, 64), (32, 8, 64, 8),
                                          (3, 3, 128, 1), (32, 1, 64, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 2), (16, 4), (70, 33), (50, 0)])
def test_prompt(hip, H, KV, hd, page, window, sinks):
    from webgllm_amd import ops
    rows = [1, 0, 33, 5, 64, 0, 1, 131]
    past = [0, 9, 0, 100, 3, 0, 250, 40]
    lens = [p + r for p, r in zip(past, rows)]

    def seen(b):
        return {j for i in range(past[b], lens[b]) for j in _sees(i, lens[b], window, sinks)}

    c = Case(lens, KV, hd, page, seed=window + sinks, seen=seen)
    M = sum(rows) + 2
    shape = ops.attn_shape(H, KV, hd)
    q = (torch.randn((M, H * hd + 4), generator=c.g, device=DEV) * 1.5 / hd ** 0.5)[:, :H * hd]
    out = torch.full((M, H * hd), 3.0, dtype=torch.float16, device=DEV)
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    got = ops.paged_attn_prefill(q, shape, c.cache, _i32(start), window, sinks, out=out)
    assert got is out and (out[-2:] == 3).all()
    _check_prompt(c, q, got, rows, H, window, sinks, 3)
    assert torch.equal(out, ops.paged_attn_prefill(q, shape, c.cache, _i32(start), window, sinks,
                                                   out=torch.full_like(out, 3.0)))


@pytest.mark.parametrize("rows,past,window,sinks", [([5], [6000], 0, 0), ([5, 2], [9000, 1], 0, 0),
                                                    ([1], [5000], 0, 0), ([3], [7000], 4000, 9),
                                                    ([700], [2000], 600, 4), ([600], [900], 0, 0)])
@pytest.mark.parametrize("H,KV,hd", [(32, 8, 64), (8, 2, 128)])
def test_prompt_long(hip, rows, past, window, sinks, H, KV, hd):
    """Few rows over many entries (split and joined), and many."""
    from webgllm_amd import ops
    lens = [p + r for p, r in zip(past, rows)]
    c = Case(lens, KV, hd, 64, seed=11)
    shape = ops.attn_shape(H, KV, hd)
    M = sum(rows)
    q = torch.randn((M, H * hd), generator=c.g, device=DEV) * 1.5 / hd ** 0.5
    start = _i32([0] + [sum(rows[:i + 1]) for i in range(len(rows))])
    got = ops.paged_attn_prefill(q, shape, c.cache, start, window, sinks)
    m = 0
    for b, (n, r) in enumerate(zip(lens, rows)):
        k, v = c.kv(b)
        for t in sorted({0, r // 3, r - 1}):
            i = n - r + t
            j = torch.arange(i + 1, device=DEV)
            see = (j > i - window) | (j < sinks) if window else j >= 0
            want, tol, _ = _attend(q[m + t].view(H, hd), k[:i + 1][see], v[:i + 1][see],
                                   int(see.sum()) - 1, 0, 0, half_weights=True)
            _near(got[m + t], want, tol, (b, t))
        m += r


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 64), (32, 8, 128), (14, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (333, 5)])
def test_prompt_many_rows(hip, H, KV, hd, window, sinks):
    """A batch of some thousands of rows: blocks of the most queries."""
    from webgllm_amd import ops
    rows, past = [2701, 3, 1999, 700], [0, 900, 77, 1200]
    if KV == 2:
        rows = [3 * r for r in rows]
    lens = [p + r for p, r in zip(past, rows)]
    c = Case(lens, KV, hd, 32, seed=12)
    shape, M = ops.attn_shape(H, KV, hd), sum(rows)
    q = torch.randn((M, H * hd), generator=c.g, device=DEV) * 1.5 / hd ** 0.5
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    got = ops.paged_attn_prefill(q, shape, c.cache, _i32(start), window, sinks)
    for b, (n, r) in enumerate(zip(lens, rows)):
        k, v = c.kv(b)
        for t in sorted({0, 1, r // 2, r - 2, r - 1}):
            i = n - r + t
            want, tol, _ = _attend(q[start[b] + t].view(H, hd), k[:i + 1], v[:i + 1], i, window,
                                   sinks, half_weights=True)
            _near(got[start[b] + t], want, tol, (b, t))
    # every row of the first sequence, against a batch of it alone
    alone = ops.paged_attn_prefill(q[:rows[0]], shape, c.cache, _i32([0] + [rows[0]] * 4), window,
                                   sinks)
    off = (alone.double() - got[:rows[0]].double()).abs()
    assert (off <= 2 ** -8 * c.v.nan_to_num().abs().amax()).all()


def test_prompt_rows_without_entries_and_missing_pages(hip):
    from webgllm_amd import ops
    H, KV, hd, page = 8, 2, 64, 16
    c = Case([3, 60, 0], KV, hd, page, seed=12)
    c.table[1, 0] = -1
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((5 + 60 + 2, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    got = ops.paged_attn_prefill(q, shape, c.cache, _i32([0, 5, 65, 67]))
    assert (got[:2] == 0).all() and (got[65:] == 0).all() and (got[5:5 + 16] == 0).all()
    _check_prompt(c, q[2:], got[2:], [3], H, 0, 0)
    k, v = c.kv(1)
    for t in (16, 17, 40, 59):
        want, tol, _ = _attend(q[5 + t].view(H, hd), k, v, t, 0, 0, set(range(16)), True)
        _near(got[5 + t], want, tol, t)


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_prompt_values_that_are_not_finite(hip, window, sinks, bad):
    """Rows that see such a value give no number; every other row keeps its
    result, of the same block too."""
    from webgllm_amd import ops
    H, KV, hd = 8, 2, 64
    c = Case([90, 40], KV, hd, 16, seed=13)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((130, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    want = ops.paged_attn_prefill(q, shape, c.cache, _i32([0, 90, 130]), window, sinks)
    for key, pool in ((50, c.v), (70, c.k)):
        pool.view(-1, KV * hd)[c.rows[0][key]] = bad
    got = ops.paged_attn_prefill(q, shape, c.cache, _i32([0, 90, 130]), window, sinks)
    for i in range(90):
        hit = any(j in _sees(i, 90, window, sinks) for j in (50, 70))
        if hit:
            assert not torch.isfinite(got[i]).all(), i
        else:
            assert torch.isfinite(got[i]).all(), i
            assert (got[i].double() - want[i].double()).abs().max() <= 2 ** -10 * 4, i
    assert torch.equal(got[90:], want[90:])


def test_prompt_large_queries(hip):
    from webgllm_amd import ops
    H, KV, hd = 4, 2, 64
    c = Case([40], KV, hd, 16, seed=14)
    shape = ops.attn_shape(H, KV, hd)
    q = torch.randn((40, H * hd), generator=c.g, device=DEV) / hd ** 0.5
    q[7] *= 1e7
    q[20] *= 1e-8
    got = ops.paged_attn_prefill(q, shape, c.cache, _i32([0, 40]))
    k, v = c.kv(0)
    for i in (6, 7, 8, 20, 39):
        want, tol, _ = _attend(q[i].view(H, hd), k, v, i, 0, 0, half_weights=True)
        _near(got[i], want, 2 ** -10 * want.abs() + 2 ** -24 if i == 7 else tol, i)


# ---------------------------------------------------------------------- eviction

def _kept(w, n, keep, sinks, recent):
    if n <= keep:
        return list(range(n))
    w = [-math.inf if math.isnan(x) else x for x in w[:n].tolist()]
    mid = sorted(range(sinks, n - recent), key=lambda j: (-w[j], j))[:keep - sinks - recent]
    return list(range(sinks)) + sorted(mid) + list(range(n - recent, n))


EVICT_LENS = [0, 1, 63, 64, 65, 100, 129, 1000, 2500]


@pytest.mark.parametrize("keep,sinks,recent", [(64, 4, 16), (1, 0, 0), (1, 1, 0), (1, 0, 1),
                                               (64, 0, 0), (40, 8, 32), (999, 3, 500)])
@pytest.mark.parametrize("kind", ["random", "few", "special"])
def test_evict(hip, keep, sinks, recent, kind):
    from webgllm_amd import ops
    KV, hd, page, page2 = 2, 64, 16, 64
    c = Case(EVICT_LENS, KV, hd, page, seed=keep)
    n, D = len(EVICT_LENS), KV * hd
    w = torch.rand((n, c.cache.max_entries + 3), generator=c.g, device=DEV)
    if kind == "few":  # many equal ones, zeros of both signs
        w = torch.randint(-1, 3, w.shape, generator=c.g, device=DEV).float()
        w[:, ::5] = -0.0
    elif kind == "special":
        pick = torch.randint(0, 6, w.shape, generator=c.g, device=DEV)
        for i, x in enumerate((float("nan"), math.inf, -math.inf, 1e-42, -3.4e38)):
            w[pick == i] = x
    per = -(-keep // page2)
    pk = torch.full((n * per + 2, page2, D), 5.0, dtype=torch.float16, device=DEV)
    pv = pk.clone()
    perm = torch.randperm(n * per + 2, generator=c.g, device=DEV)[:n * per].view(n, per)
    old = c.k.clone(), c.v.clone()
    to, kept, kw = ops.paged_evict(c.cache, w, keep, perm.int().contiguous(), sinks, recent,
                                   pool=(pk, pv))
    for a, b in ((c.k, old[0]), (c.v, old[1])):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    left = torch.ones(pk.shape[0] * page2, dtype=torch.bool, device=DEV)
    for b, x in enumerate(EVICT_LENS):
        want = _kept(w[b].cpu(), x, keep, sinks, recent)
        m = len(want)
        assert int(to.lens[b]) == m
        assert kept[b].tolist() == want + [-1] * (keep - m), (b, x)
        assert torch.equal(kw[b, :m].view(torch.int32), w[b, want].view(torch.int32))
        assert (kw[b, m:] == 0).all()
        dst = (perm[b][:, None] * page2 + torch.arange(page2, device=DEV)).reshape(-1)[:m]
        left[dst] = False
        for new, src in ((pk, c.k), (pv, c.v)):
            assert torch.equal(new.view(-1, D)[dst].view(torch.int16),
                               src.view(-1, D)[c.rows[b][want]].view(torch.int16)), b
    for new in (pk, pv):
        assert (new.view(-1, D)[left] == 5).all()


@pytest.mark.parametrize("n", [16385, 24577, 40000, 131071])
@pytest.mark.parametrize("kind", ["random", "few", "special", "one"])
@pytest.mark.parametrize("keep,sinks,recent", [(4097, 4, 1000), (4097, 1000, 3097),
                                               (100, 0, 0), (4000, 0, 3999)])
def test_evict_long(hip, n, kind, keep, sinks, recent):
    """Sequences that several workgroups share."""
    from webgllm_amd import ops
    c = Case([n, 500], 1, 64, 256, seed=15, spare=40)
    w = torch.rand((2, c.cache.max_entries), generator=c.g, device=DEV).square_()
    w[0, 1000:2000] = 0.5
    if kind == "few":
        w = torch.randint(-1, 3, w.shape, generator=c.g, device=DEV).float()
        w[:, ::5] = -0.0
    elif kind == "special":
        pick = torch.randint(0, 6, w.shape, generator=c.g, device=DEV)
        for i, x in enumerate((float("nan"), math.inf, -math.inf, 1e-42, -3.4e38)):
            w[pick == i] = x
    elif kind == "one":
        w.fill_(0.25)
    table = _i32(c.spare[:34]).view(2, 17)
    to, kept, kw = ops.paged_evict(c.cache, w, keep, table, sinks, recent)
    assert to.lens.tolist() == [keep, min(keep, 500)]
    for b, x in enumerate((n, 500)):
        want = _kept(w[b].cpu(), x, keep, sinks, recent)
        assert kept[b].tolist() == want + [-1] * (keep - len(want))
        got, pick = kw[b, :len(want)], w[b, torch.tensor(want, device=DEV)]
        assert torch.equal(got.view(torch.int32), pick.view(torch.int32))
        assert (kw[b, len(want):] == 0).all()
    dst = (table[0].long()[:, None] * 256 + torch.arange(256, device=DEV)).reshape(-1)[:keep]
    for p in (c.k, c.v):
        assert torch.equal(p.view(-1, 64)[dst], p.view(-1, 64)[c.rows[0][kept[0].long()]])


@pytest.mark.parametrize("long", [False, True])
def test_evict_missing_pages_and_lens_in_place(hip, long):
    """Entries without a page, old or new, are not moved; the new lengths may
    take the old ones' place."""
    import ctypes as C

    from webgllm_amd import lib as L
    from webgllm_amd import ops
    KV, hd, page = 1, 64, 16
    c = Case([60, 20] + [30000] * long, KV, hd, page, seed=16, spare=11)
    c.table[0, 1] = -1
    n = len(c.lens)
    new = _i32([c.spare[3 * i:3 * i + 3] for i in range(n)])
    new[0, 1] = 10 ** 6
    w = torch.zeros((n, c.cache.max_entries), device=DEV)  # all equal: the first ones stay
    kept = torch.empty((n, 40), dtype=torch.int32, device=DEV)
    to = ops.PagedCache(c.k, c.v, new, c.cache.lens)
    s = torch.cuda.current_stream().cuda_stream
    scratch = ops.paged_evict_scratch(c.cache)
    L.check(hip.wg_paged_evict(C.byref(c.cache.desc), KV * hd, w.data_ptr(), w.stride(0), 40, 0, 0,
                               C.byref(to.desc), c.cache.lens.data_ptr(), None, 0, kept.data_ptr(),
                               40, scratch.data_ptr(), scratch.numel(), s))
    assert c.cache.lens.tolist() == [40, 20] + [40] * long
    assert all(kept[b].tolist() == list(range(40)) for b in range(n) if b != 1)
    D = KV * hd
    flat = c.k.view(-1, D)
    for i in range(40):
        p = int(new[0, i // page])
        if p >= c.k.shape[0]:
            continue
        row = flat[p * page + i % page]
        if 16 <= i < 32:
            assert torch.isnan(row).all()  # its page is missing: left as it was
        else:
            assert torch.equal(row, flat[c.rows[0][i]])
    dst = (new[1].long()[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:20]
    assert torch.equal(flat[dst], flat[c.rows[1]])


# ------------------------------------------------------------------ run together

def _served(steps, graph):
    """Prompts, decode steps with summed weights under a budget, an eviction
    in between, more steps, as a program serves them: every output."""
    from webgllm_amd import ops
    H, KV, hd, page, n = 8, 2, 64, 16, 3
    g = _gen(17)
    shape = ops.attn_shape(H, KV, hd)
    rope = _rope(1e4, hd, 4096)
    k = torch.zeros((64, page, KV * hd), dtype=torch.float16, device=DEV)
    v = torch.zeros_like(k)
    table = torch.randperm(64, generator=g, device=DEV).int()[:60].view(6, 10).contiguous()
    rows = [50, 90, 7]
    lens = _i32(rows)
    cache = ops.PagedCache(k, v, table[:3], lens)
    wide = (H + 2 * KV) * hd
    start = _i32([0, 50, 140, 147])
    qkv = torch.randn((147, wide), generator=g, device=DEV)
    outs = []
    q = ops.paged_head_prep(qkv, shape, rope, cache, row_start=start)
    outs.append(ops.paged_attn_prefill(q, shape, cache, start))
    weights = torch.zeros((n, cache.max_entries), device=DEV)
    pos = lens.clone()  # the next token's position
    step_in = torch.empty((n, wide), device=DEV)
    step_out = torch.empty((n, H * hd), dtype=torch.float16, device=DEV)

    def body(cache, weights, scratch):
        cache.lens.add_(1)
        q = ops.paged_head_prep(step_in, shape, rope, cache, pos=pos)
        ops.paged_attn_decode(q, shape, cache, window=64, sinks=4, weights=weights,
                              scratch=scratch, out=step_out)
        pos.add_(1)

    def run(cache, weights, inputs):
        scratch = ops.paged_decode_scratch(cache, shape, True)
        graphed = None
        if graph:
            keep = [t.clone() for t in (cache.lens, pos, weights, k, v)]
            step_in.copy_(inputs[0])
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                body(cache, weights, scratch)
                torch.cuda.synchronize()
                graphed = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graphed, stream=s):
                    body(cache, weights, scratch)
            torch.cuda.current_stream().wait_stream(s)
            for t, old in zip((cache.lens, pos, weights, k, v), keep):
                t.copy_(old)
        for x in inputs:
            step_in.copy_(x)
            graphed.replay() if graph else body(cache, weights, scratch)
            outs.append(step_out.clone())

    inputs = torch.randn((2 * steps, n, wide), generator=g, device=DEV)
    run(cache, weights, inputs[:steps])
    to, kept, kw = ops.paged_evict(cache, weights, 48, table[3:], sinks=4, recent=16)
    outs += [kept, kw.clone()]
    w2 = torch.zeros((n, to.max_entries), device=DEV)
    w2[:, :48] = kw
    run(to, w2, inputs[steps:])
    return outs + [w2, to.lens.clone(), pos.clone()], (qkv, inputs, rope, shape, start)


def test_served_together(hip):
    """The same run with every step eager and as replays of a captured graph
    gives the same bits; and each attention output is what 64 bits give for
    keys and values prepared as rows of a plain list."""
    steps = 12
    eager, (qkv, inputs, rope, shape, start) = _served(steps, False)
    graphed, _ = _served(steps, True)
    for a, b in zip(eager, graphed):
        assert torch.equal(a, b)
    from webgllm_amd import ops
    H, KV, hd = 8, 2, 64
    rows = [50, 90, 7]
    outs = iter(eager)
    prompt = next(outs)
    entries = []  # (k, v) rows of each sequence
    D = KV * hd

    def prep(x, p0):
        ck = torch.zeros((4096, D), dtype=torch.float16, device=DEV)
        cv = ck.clone()
        q = ops.head_prep(x.contiguous(), shape, rope, _i32([p0]), ck, cv)
        return q, ck[p0:p0 + len(x)], cv[p0:p0 + len(x)]

    for b, r in enumerate(rows):
        s0 = int(start[b])
        q, kk, vv = prep(qkv[s0:s0 + r], 0)
        entries.append([kk, vv])
        for t in range(r):
            want, tol, _ = _attend(q[t].view(H, hd), kk.double().view(-1, KV, hd),
                                   vv.double().view(-1, KV, hd), t, 0, 0, half_weights=True)
            _near(prompt[s0 + t], want, tol, (b, t))
    sums = [torch.zeros(200, dtype=torch.float64, device=DEV) for _ in rows]
    for half in range(2):
        for x in range(steps):
            got = next(outs)
            for b, r in enumerate(rows):
                q, kk, vv = prep(inputs[half * steps + x][b:b + 1], r + half * steps + x)
                e = entries[b]
                e[0], e[1] = torch.cat([e[0], kk]), torch.cat([e[1], vv])
                n = len(e[0])
                want, tol, p = _attend(q[0].view(H, hd), e[0].double().view(n, KV, hd),
                                       e[1].double().view(n, KV, hd), n - 1, 64, 4)
                _near(got[b], want, tol, (half, x, b))
                sums[b][:n] += p.sum(0)
        if half == 0:
            kept, kw = next(outs), next(outs)
            for b in range(3):
                n = len(entries[b][0])
                idx = [j for j in kept[b].tolist() if j >= 0]
                assert len(idx) == min(48, n)
                # the sums of 12 steps: 2^-11 relative each, as test_decode
                assert (kw[b, :len(idx)].double() - sums[b][idx]).abs().max() <= 2 ** -10 * 12
                mid = range(4, n - 16)  # behind the sinks, before the recent ones
                least = min((float(sums[b][j]) for j in idx if j in mid), default=0.0)
                gone = [j for j in range(n) if j not in idx]
                assert all(j in mid and float(sums[b][j]) <= least + 12 * 2 ** -10 for j in gone)
                entries[b] = [t[idx] for t in entries[b]]
                s = torch.zeros_like(sums[b])
                s[:len(idx)] = sums[b][idx]
                sums[b] = s
    w2, lens, pos = next(outs), next(outs), next(outs)
    for b, r in enumerate(rows):
        assert int(lens[b]) == len(entries[b][0]) and int(pos[b]) == r + 2 * steps
        assert (w2[b, :60].double() - sums[b][:60]).abs().max() <= 2 ** -10 * 24


def test_two_graphs_and_eager_calls(hip):
    """Two captured graphs with a scratch each, replayed in turn and with an
    eager call on a third, give their eager results every time; a call on
    another stream too."""
    from webgllm_amd import ops
    H, KV, hd = 32, 8, 64
    lens = [700, 31, 4000]
    cs = [Case(lens, KV, hd, 32, seed=s) for s in (18, 19)]
    shape = ops.attn_shape(H, KV, hd)
    qs = [torch.randn((3, H * hd), generator=c.g, device=DEV) / 8 for c in cs]
    rows = _i32([0, 1, 1, 3])
    graphs = []
    for c, q in zip(cs, qs):
        want = [ops.paged_attn_decode(q, shape, c.cache),
                ops.paged_attn_prefill(q, shape, c.cache, rows)]
        sc = ops.paged_decode_scratch(c.cache, shape), ops.paged_prefill_scratch(c.cache, shape, 3)
        got = [torch.empty_like(want[0]), torch.zeros_like(want[1])]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            ops.paged_attn_decode(q, shape, c.cache, scratch=sc[0], out=got[0])
            ops.paged_attn_prefill(q, shape, c.cache, rows, scratch=sc[1], out=got[1])
        graphs.append((gr, got, want, sc))
    for _ in range(4):
        for gr, got, want, _sc in graphs:
            for t in got:
                t.fill_(9)
            gr.replay()
            assert torch.equal(ops.paged_attn_decode(qs[0], shape, cs[0].cache), graphs[0][2][0])
        torch.cuda.synchronize()
        for gr, got, want, _sc in graphs:
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.paged_attn_decode(qs[1], shape, cs[1].cache)
        b = ops.paged_attn_prefill(qs[1], shape, cs[1].cache, rows)
    side.synchronize()
    assert torch.equal(a, graphs[1][2][0]) and torch.equal(b, graphs[1][2][1])


@pytest.mark.parametrize("wide", [5, 280])
def test_captured_step_follows_table_and_lengths(hip, wide):
    """A step and an eviction captured once, replayed after lengths, pages,
    positions and the rows' ends changed on the device: each time what eager
    calls give. wide 280: a cache that could hold more than one workgroup
    selects from."""
    from webgllm_amd import ops
    H, KV, hd, page, n = 8, 2, 64, 64, 3
    pages = n * wide + 12
    g = _gen(21)
    k = torch.randn((pages, page, KV * hd), generator=g, device=DEV).half()
    v = torch.randn_like(k)
    table = torch.empty((n, wide), dtype=torch.int32, device=DEV)
    lens, starts = _i32([1] * n), _i32([0, 1, 2, 3])
    cache = ops.PagedCache(k, v, table, lens)
    shape = ops.attn_shape(H, KV, hd)
    rope = _rope(1e4, hd, 20480)
    qkv = torch.randn((7, (H + 2 * KV) * hd), generator=g, device=DEV)
    weights = torch.zeros((n, wide * page), device=DEV)
    new_table = torch.empty((n, 3), dtype=torch.int32, device=DEV)
    scratch = (ops.paged_prefill_scratch(cache, shape, 7), ops.paged_decode_scratch(cache, shape, True),
               ops.paged_evict_scratch(cache))

    def step():
        q = ops.paged_head_prep(qkv, shape, rope, cache, row_start=starts)
        pre = ops.paged_attn_prefill(q, shape, cache, starts, 200, 2, scratch=scratch[0])
        dec = ops.paged_attn_decode(q[:n], shape, cache, weights=weights, scratch=scratch[1])
        to, kept, kw = ops.paged_evict(cache, weights, 150, new_table, 2, 20, scratch=scratch[2])
        return q, pre, dec, to.lens, kept, kw

    def place(seed, lengths, ends):
        h = _gen(seed)
        order = torch.randperm(pages, generator=h, device=DEV).int()
        table.copy_(order[:n * wide].view(n, wide))
        new_table.copy_(order[n * wide:n * wide + 9].view(n, 3))
        lens.copy_(_i32(lengths))
        starts.copy_(_i32(ends))
        weights.copy_(torch.rand(weights.shape, generator=h, device=DEV))
        k.copy_(torch.randn(k.shape, generator=h, device=DEV))
        v.copy_(torch.randn(v.shape, generator=h, device=DEV))
        qkv.copy_(torch.randn(qkv.shape, generator=h, device=DEV))

    top = wide * page
    cases = [(1, [9, 170, 300], [0, 3, 5, 7]), (2, [top, 5, 64], [0, 5, 6, 7]),
             (3, [151, 150, top - 1], [0, 1, 4, 7]), (4, [7, top, 128], [0, 7, 7, 7])]
    place(*cases[0])
    step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = step()
    for case in cases + cases[:1]:
        place(*case)
        want = [t.clone() for t in step()] + [weights.clone(), k.clone(), v.clone()]
        place(*case)
        graph.replay()
        for i, (a, b) in enumerate(zip([*got, weights, k, v], want)):
            assert torch.equal(a, b), (case, i)


def test_most_sequences(hip):
    """65,535 sequences of up to three entries, one of 300, through every
    operator; several sequences share a first page."""
    from webgllm_amd import ops
    H, KV, hd, n = 2, 1, 64, 65535
    g = _gen(24)
    lens = torch.randint(0, 4, (n,), generator=g, device=DEV, dtype=torch.int32)
    lens[4097], lens[-1] = 300, 3
    wide, page = 300, 1
    table = torch.full((n, wide), -1, dtype=torch.int32, device=DEV)
    table[:, 0] = torch.arange(n, device=DEV) // 3  # (three share each first page)
    table[:, 1:3] = (n + torch.arange(2 * n, device=DEV).view(n, 2)).int()
    table[4097, 3:] = 3 * n + torch.arange(297, device=DEV, dtype=torch.int32)
    pages = 3 * n + 300 + 2 * n
    k = torch.randn((pages, page, hd), generator=g, device=DEV).half()
    v = torch.randn_like(k)
    cache = ops.PagedCache(k, v, table, lens)
    shape = ops.attn_shape(H, KV, hd)
    ends = torch.cat([torch.zeros(1, device=DEV), (lens > 0).cumsum(0)]).int()
    M = int(ends[-1])
    before = k.clone()
    qkv = torch.randn((M, (H + 2) * hd), generator=g, device=DEV)
    rows = torch.nonzero(lens > 0)[:, 0]
    shared = lens[rows] == 1  # (their only entry lies on the shared page: not written)
    fresh = ops.PagedCache(k, v, torch.where(table < n, -1, table), lens)
    q = ops.paged_head_prep(qkv, shape, _rope(1e4, hd, 1024), fresh, row_start=ends)
    assert (q[shared] == 0).all() and not (q[~shared] == 0).all(-1).any()
    assert torch.equal(k[:n], before[:n]) and not torch.equal(k[n:3 * n], before[n:3 * n])
    weights = torch.zeros((n, wide), device=DEV)
    full = torch.randn((n, H * hd), generator=g, device=DEV) / 8
    dec = ops.paged_attn_decode(full, shape, cache, weights=weights)
    pre = ops.paged_attn_prefill(full[rows].contiguous(), shape, cache, ends)
    assert (dec[lens == 0] == 0).all()
    assert (weights.sum(1) - H * (lens > 0)).abs().max() < 1e-3
    at = dict(zip(rows.tolist(), range(M)))
    for b in [4097, n - 1, *torch.randint(0, n, (40,), generator=g, device=DEV).tolist()]:
        m = int(lens[b])
        if m == 0:
            continue
        e = table[b, :m].long()
        kk, vv = (t[e].double().view(m, 1, hd) for t in (k, v))
        want, tol, _ = _attend(full[b].view(H, hd), kk, vv, m - 1, 0, 0, half_weights=True)
        _near(dec[b], want, tol, b)
        _near(pre[at[b]], want, tol, b)
    new = (3 * n + 300 + torch.arange(2 * n, device=DEV).view(n, 2)).int()
    to, kept, _ = ops.paged_evict(cache, weights, 2, new, 0, 1)
    assert torch.equal(to.lens, lens.clamp(max=2))
    for b in (4097, n - 1):
        m = int(lens[b])
        best = int(weights[b, :m - 1].argmax())
        assert kept[b].tolist() == [best, m - 1]
        assert torch.equal(k[new[b].long()], k[table[b, [best, m - 1]].long()])


def test_two_streams_at_once(hip):
    """Calls under way on two streams, each with its own tensors and scratch,
    give what they give alone."""
    from webgllm_amd import ops
    H, KV, hd = 32, 8, 128
    jobs = []
    for seed, lens in ((22, [3000, 17, 5000]), (23, [40, 9000])):
        c = Case(lens, KV, hd, 64, seed=seed)
        M = 6 * len(lens)
        q = torch.randn((M, H * hd), generator=c.g, device=DEV) / 12
        jobs.append((c, q, _i32(range(0, M + 1, 6)), torch.cuda.Stream()))
    shape = ops.attn_shape(H, KV, hd)

    def run(c, q, rows):
        n = len(c.lens)
        w = torch.zeros((n, c.cache.max_entries), device=DEV)
        a = ops.paged_attn_prefill(q, shape, c.cache, rows, 700, 4)
        b = ops.paged_attn_decode(q[:n], shape, c.cache, weights=w)
        return a, b, w

    want = [run(*j[:3]) for j in jobs]
    torch.cuda.synchronize()
    got = [[] for _ in jobs]
    for j in jobs:
        j[3].wait_stream(torch.cuda.current_stream())
    for _ in range(12):
        for i, j in enumerate(jobs):
            with torch.cuda.stream(j[3]):
                got[i].append(run(*j[:3]))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, w)), i


def test_python_checks(hip):
    from webgllm_amd import ops
    c = Case([20, 30], 2, 64, 16, seed=20)
    shape = ops.attn_shape(4, 2, 64)
    q = torch.zeros((2, 256), device=DEV)
    bad = [lambda: ops.PagedCache(c.k, c.v[:1], c.table, c.cache.lens),
           lambda: ops.PagedCache(c.k.float(), c.v.float(), c.table, c.cache.lens),
           lambda: ops.PagedCache(c.k, c.v, c.table[:1], c.cache.lens),
           lambda: ops.PagedCache(c.k, c.v, c.table.long(), c.cache.lens),
           lambda: ops.paged_attn_decode(q[:1], shape, c.cache),
           lambda: ops.paged_attn_decode(q, ops.attn_shape(4, 4, 64), c.cache),
           lambda: ops.paged_attn_decode(q.half(), shape, c.cache),
           lambda: ops.paged_attn_decode(q[:, :200], shape, c.cache),
           lambda: ops.paged_attn_decode(q, shape, c.cache, weights=torch.zeros(2, 5, device=DEV)),
           lambda: ops.paged_attn_decode(q, shape, c.cache, out=q),
           lambda: ops.paged_attn_prefill(q, shape, c.cache, _i32([0, 2])),
           lambda: ops.paged_attn_prefill(q, shape, c.cache, None),
           lambda: ops.paged_evict(c.cache, torch.zeros(2, 5, device=DEV), 4, c.table),
           lambda: ops.paged_evict(c.cache, torch.zeros(2, 99, device=DEV), 0, c.table),
           lambda: ops.paged_evict(c.cache, torch.zeros(2, 99, device=DEV), 4, c.table[:1]),
           lambda: ops.paged_evict(c.cache, torch.zeros(2, 99, device=DEV), 4, c.table,
                                   pool=(c.k[..., :64].contiguous(), c.v[..., :64].contiguous())),
           lambda: ops.paged_head_prep(torch.zeros((2, 512), device=DEV), shape,
                                       torch.zeros((1100, 32), device=DEV), c.cache),
           lambda: ops.paged_head_prep(torch.zeros((2, 512), device=DEV), shape,
                                       torch.zeros((1100, 64), device=DEV), c.cache,
                                       pos=_i32([1]))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
