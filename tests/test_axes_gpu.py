"""Head preparation into pages under rotary positions of several axes
(wg_paged_head_prep_axes), on the GPU: bit for bit the single-position calls',
frequency by frequency, and the formula in 64 bits."""
import pytest
import torch

from tests.test_paged_gpu import DEV, Case, _gen, _i32, _rope

pytestmark = pytest.mark.gpu

SHAPES = [(14, 2, 64, 64, False), (32, 8, 128, 128, True), (32, 8, 64, 64, True),
          (6, 3, 64, 32, True), (4, 2, 96, 96, False), (4, 4, 256, 256, True), (3, 1, 8, 8, False),
          (60, 30, 128, 128, False)]


def _sections(pairs, axes):
    n = [pairs // axes] * axes
    n[0] += pairs - sum(n)
    return n


def _axis_of(n, interleaved):
    if not interleaved:
        return [a for a, k in enumerate(n) for _ in range(k)]
    return [f % len(n) if f < len(n) * n[f % len(n)] else 0 for f in range(sum(n))]


@pytest.mark.parametrize("H,KV,hd,rot,norm", SHAPES)
@pytest.mark.parametrize("axes,interleaved", [(1, False), (2, True), (3, False), (3, True),
                                              (4, False), (4, True)])
def test_frequency_by_frequency(hip, H, KV, hd, rot, norm, axes, interleaved):
    """Each dim of a query or key is that of a call in which all frequencies turn
    by its axis; values and everything else of the pool alike."""
    from webgllm_amd import ops
    if rot // 2 < axes:
        pytest.skip("more axes than frequencies")
    rows, past, page = [5, 0, 1, 40], [0, 7, 1100, 3], 16
    lens = [p + r for p, r in zip(past, rows)]
    c = Case(lens, KV, hd, page, seen=lambda b: ())
    M, wide = sum(rows) + 2, (H + 2 * KV) * hd  # two rows behind the last sequence
    g = _gen(axes)
    shape = ops.attn_shape(H, KV, hd, rot, 1e-5, norm)
    qkv = torch.randn((M, wide + 16), generator=g, device=DEV)[:, :wide]
    qn, kn = (1 + 0.1 * torch.randn(hd, generator=g, device=DEV) for _ in range(2))
    rope, start = _rope(1e6, hd, 8192), _i32([0, 5, 5, 6, 46])
    pos = torch.randint(0, 8192, (M, axes + 2), generator=g, device=DEV, dtype=torch.int32)
    n = _sections(rot // 2, axes)
    if interleaved and axes == 3:  # (more than every third frequency for the last)
        n = [n[0] - n[0] // 2, n[1], n[2] + n[0] // 2]

    def prep(p, ax):
        c.k.fill_(float("nan")), c.v.fill_(float("nan"))
        q_out = torch.full((M, H * hd + 4), 7.0, device=DEV)[:, :H * hd]
        got = ops.paged_head_prep(qkv, shape, rope, c.cache, pos=p, row_start=start, q_norm=qn,
                                  k_norm=kn, q_out=q_out, axes=ax)
        return got.clone(), c.k.clone(), c.v.clone()

    q, k, v = prep(pos[:, :axes], ops.rope_axes(n, interleaved))
    of = _axis_of(n, interleaved)
    dim_axis = torch.tensor(of + of + [0] * (hd - rot), device=DEV)
    want = [prep(pos[:, a].contiguous(), None) for a in range(axes)]
    assert (q[sum(rows):] == 7).all()
    for a, (wq, wk, wv) in enumerate(want):
        at = dim_axis == a
        for got, ref, heads in ((q, wq, H), (k, wk, KV)):
            x, y = (t.reshape(-1, heads, hd)[..., at] for t in (got, ref))
            assert torch.equal(x.nan_to_num(99.0), y.nan_to_num(99.0)), a
        assert torch.equal(v.nan_to_num(99.0), wv.nan_to_num(99.0))


@pytest.mark.parametrize("hd,interleaved", [(64, False), (128, True), (96, True)])
def test_formula(hip, hd, interleaved):
    """Against 64 bits. Bound: the table's cos and sin are off by 2^-24 each, an
    angle's by 2^-22 (two products and a sum of such), a rotation by 2^-22 more of
    |x1| + |x2|, the query's scale by 2^-23 of it; a key's half by half a step
    (2^-11, or 2^-25 below the normal halves)."""
    from webgllm_amd import ops
    H, KV, page, M = 4, 2, 16, 9
    c = Case([40] * M, KV, hd, page, seen=lambda b: ())
    g = _gen(hd)
    qkv = torch.randn((M, (H + 2 * KV) * hd), generator=g, device=DEV)
    pos = torch.randint(0, 30000, (M, 3), generator=g, device=DEV, dtype=torch.int32)
    n = _sections(hd // 2, 3)
    got = ops.paged_head_prep(qkv, ops.attn_shape(H, KV, hd), _rope(1e6, hd, 32768), c.cache,
                              pos=pos, axes=ops.rope_axes(n, interleaved))
    x = qkv.double().view(M, -1, hd)[:, :H + KV]
    p = pos[:, _axis_of(n, interleaved)].double()
    a = p * 1e6 ** (-2.0 * torch.arange(hd // 2, device=DEV).double() / hd)
    cos, sin = a.cos()[:, None], a.sin()[:, None]
    x1, x2 = x[..., :hd // 2], x[..., hd // 2:]
    want = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
    tol = (2 ** -21) * (x1.abs() + x2.abs()).repeat(1, 1, 2)
    s = hd ** -0.5
    off = (got.double().view(M, H, hd) - want[:, :H] * s).abs()
    assert (off <= s * (tol[:, :H] + 2 ** -22 * want[:, :H].abs())).all()
    for b in range(M):
        k = c.k.view(-1, KV, hd)[c.rows[b][39]].double()
        w, t = want[b, H:], tol[b, H:]
        assert ((k - w).abs() <= t + 2 ** -11 * w.abs() + 2 ** -25).all(), b


@pytest.mark.parametrize("hd", [64, 96])
def test_positions_that_the_table_does_not_hold(hip, hd):
    """One such position among a row's, of an axis without a frequency too: a zero
    query and nothing stored; so without an entry or a page."""
    from webgllm_amd import ops
    H, KV, page = 4, 2, 16
    c = Case([3, 5, 20, 33, 5, 0, 7], KV, hd, page, seen=lambda b: ())
    c.table[2, 1] = -1
    shape = ops.attn_shape(H, KV, hd)
    qkv = torch.randn((7, (H + 2 * KV) * hd), generator=_gen(2), device=DEV)
    pos = _i32([[2, 5, 9], [0, 2048, 1], [4, 4, 4], [1, 1, -1], [7, -2 ** 31, 7], [0, 0, 0],
                [2047, 0, 2 ** 31 - 1]])
    q = ops.paged_head_prep(qkv, shape, _rope(1e4, hd, 2048), c.cache, pos=pos,
                            axes=ops.rope_axes([hd // 2 - 4, 4, 0]))
    assert (q[1:] == 0).all() and (q[0] != 0).any()
    for pool in (c.k, c.v):
        wrote = ~torch.isnan(pool).all(-1).view(-1)
        assert wrote.nonzero()[:, 0].tolist() == [int(c.rows[0][2])]


def test_python_checks(hip):
    from webgllm_amd import lib as L
    from webgllm_amd import ops
    c = Case([3, 5], 2, 64, 16)
    shape, rope = ops.attn_shape(4, 2, 64), _rope(1e4, 64, 2048)
    qkv = torch.zeros((2, 8 * 64), device=DEV)
    ax = ops.rope_axes([8, 12, 12])

    def call(pos, axes=ax):
        return ops.paged_head_prep(qkv, shape, rope, c.cache, pos=pos, axes=axes)

    for pos, msg in ((None, "need positions"), (_i32([[0, 0]] * 2), "3 axes"),
                     (_i32([[0, 0, 0]]), "3 axes"), (torch.zeros((2, 3), device=DEV), "int32"),
                     (torch.zeros((2, 3), dtype=torch.int32), "device"),
                     (_i32([0] * 6), "column stride")):
        with pytest.raises(ValueError, match=msg):
            call(pos)
    for n in ([], [1] * 5, [2 ** 40]):
        with pytest.raises(ValueError):
            ops.rope_axes(n)
    with pytest.raises(L.WgError, match="31 frequencies"):
        call(_i32([[0, 0, 0]] * 2), ops.rope_axes([8, 12, 11]))
