"""Low-rank adapters (wg_adapter_add) at the edges of their inputs, on the GPU:
values that are not finite against the formula in 64 bits, infinities and their
signs among them, scales far from 1, and results of any stride."""
import pytest
import torch

from tests.test_adapter_gpu import DEV, Set, _i32, _starts

pytestmark = pytest.mark.gpu

INF = float("inf")


def _formula(c, got, x, y, f, slots, rows=None):
    """got as the formula has it: infinities with their signs, NaN, and all else
    within Set.want's bound. Returns how many infinities there were."""
    m, seen = 0, 0
    for b, at in enumerate(slots):
        n = 1 if rows is None else rows[b]
        sl = slice(m, m + n)
        m += n
        if not n:
            continue
        want, tol = c.want(x[sl], y[sl], None if f is None else f[sl], at)
        g, finite, nan = got[sl].double(), torch.isfinite(want), torch.isnan(want)
        assert torch.equal(torch.isnan(g), nan), (b, at)
        inf = ~finite & ~nan
        assert torch.equal(g[inf], want[inf]), (b, at)
        assert ((g - want).abs()[finite] <= tol[finite]).all(), (b, at)
        seen += int(inf.sum())
    return seen


SHAPES = [(8, (4, 8)), (104, (20, 4, 36, 60)), (896, (896, 128, 128)), (4184, (64,))]
ROWS = [None, [3, 5, 40, 0, 2], [131, 17, 1, 200, 64]]


def _call(c, slots, rows, x, y, f):
    from webgllm_amd import ops
    start = None if rows is None else _i32(_starts(rows))
    return ops.adapter_add(y.clone(), x, c.set, _i32(slots), start, f)


@pytest.mark.parametrize("K,cols", SHAPES)
@pytest.mark.parametrize("rows", ROWS)
def test_infinite_inputs(hip, K, cols, rows):
    """Between the factors of rank 1 stands an infinity: outputs are infinities."""
    slots = [0, 1, 2, 0, -1]
    c = Set([1, 1, 9], K, cols, seed=K)
    x, y, f = c.rows(sum(rows) if rows else 5)
    x[0, K - 3], x[3, 0], x[-3, K // 2] = INF, -INF, INF
    assert _formula(c, _call(c, slots, rows, x, y, f), x, y, f, slots, rows) >= 2 * c.N


@pytest.mark.parametrize("K,cols", SHAPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("ranks", [[16, 5, 8], [40, 64, 3], [130, 256, 70]])
def test_infinities_in_a_first_factor(hip, K, cols, rows, ranks):
    """Also among the last inputs, where K ends inside a step."""
    slots = [0, 1, 2, 0, -1]
    c = Set(ranks, K, cols, seed=K + 1)
    c.a[0, 0, 3, K - 1], c.a[1, -1, ranks[1] - 1, K - 8], c.a[2, 0, 0, K - 2] = INF, -INF, INF
    x, y, f = c.rows(sum(rows) if rows else 5)
    assert _formula(c, _call(c, slots, rows, x, y, f), x, y, f, slots, rows) >= sum(
        (rows or [1] * 5)[b] * cols[j] for b, j in ((0, 0), (1, -1), (2, 0)))


@pytest.mark.parametrize("K,cols", SHAPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("ranks", [[16, 5, 8], [40, 64, 3], [130, 256, 70]])
def test_infinities_in_a_second_factor(hip, K, cols, rows, ranks):
    """An output's infinity has the sign of what stands between the factors."""
    slots = [0, 1, 2, 0, -1]
    c = Set(ranks, K, cols, seed=K + 2)
    N = c.N
    c.b[0, 1, 3], c.b[0, N - 1, ranks[0] - 1], c.b[1, N // 2, ranks[1] - 1], c.b[2, 0, 1] = \
        INF, -INF, -INF, INF
    x, y, f = c.rows(sum(rows) if rows else 5)
    n = rows or [1] * 5
    assert _formula(c, _call(c, slots, rows, x, y, f), x, y, f, slots, rows) == sum(
        n[b] * k for b, k in ((0, 2), (1, 1), (2, 1), (3, 2)))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("e,x_times,a_times", [(-120, 1.0, 1.0), (120, 2.0 ** 13, 2.0 ** 14)])
def test_scales_far_apart(hip, rows, e, x_times, a_times):
    """An adapter's and a row's scale whose product alone is an ordinary number."""
    slots = [0, 1, 0, 1, -1]
    c = Set([8, 40], 896, (64, 32), seed=e + 200)
    c.a *= a_times
    c.scale.fill_(1.7 * 2.0 ** e)
    x, y, _ = c.rows(sum(rows) if rows else 5)
    x *= x_times
    f = torch.full((len(y),), 2.0 ** -e, device=DEV)
    c.check(_call(c, slots, rows, x, y, f), x, y, f, slots, rows)


@pytest.mark.parametrize("extra,offset", [(0, 1), (1, 0), (4, 0), (4, 2), (7, 3), (64, 0), (6, 0)])
@pytest.mark.parametrize("rows", [[5, 0, 1, 40], [131, 200], [33, 64, 40], [700]])
@pytest.mark.parametrize("ranks", [[16, 5, 64], [256, 7, 130]])
def test_results_of_any_stride(hip, rows, extra, offset, ranks):
    """y of rows wider than its outputs, at any float of an allocation: what lies
    between its rows and around them stays."""
    from webgllm_amd import ops
    c = Set(ranks, 896, (896, 128, 124), seed=extra)
    M = sum(rows) + 3
    x, y0, f = c.rows(M)
    flat = torch.full((M * (c.N + extra) + 64,), 5.0, device=DEV)
    y = flat[offset:offset + M * (c.N + extra)].view(M, c.N + extra)[:, :c.N]
    y.copy_(y0)
    slots = [2, -1, 0, 1][:len(rows)]
    start = _i32([1 + s for s in _starts(rows)])
    got = ops.adapter_add(y, x, c.set, _i32(slots), start, f)
    assert got is y
    sl = slice(1, 1 + sum(rows))
    c.check(y[sl], x[sl], y0[sl], f[sl], slots, rows)
    assert torch.equal(y[:1], y0[:1]) and torch.equal(y[-2:], y0[-2:])
    y.fill_(5.0)
    assert (flat == 5).all()


@pytest.mark.parametrize("rows", [None, [1, 2]])
def test_the_most_inputs(hip, rows):
    """Rows of 2^30 inputs, 2^31 bytes: few of them not 0, up to the last."""
    from webgllm_amd import ops
    K, N, n = 2 ** 30, 8, 2 if rows is None else 3
    a = torch.zeros((1, 8, K), dtype=torch.float16, device=DEV)
    x = torch.zeros((n, K), dtype=torch.float16, device=DEV)
    at = torch.tensor([0, 4095, 4096, 2 ** 29 - 1, 2 ** 29, 2 ** 29 + 12345, K - 4097, K - 1], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    a[0][:, at] = torch.randn((8, 8), generator=g, device=DEV).half()
    x[:, at] = torch.randn((n, 8), generator=g, device=DEV).half()
    b = torch.randn((1, N, 8), generator=g, device=DEV).half()
    y = torch.randn((n, N), generator=g, device=DEV)
    c = ops.Adapters(a, b, _i32([8]), torch.ones(1, device=DEV))
    got = ops.adapter_add(y.clone(), x, c, _i32([0] * (n if rows is None else 2)),
                          None if rows is None else _i32(_starts(rows)))
    # (8 products a sum between the factors, 8 behind them, 22 bits between)
    t = x[:, at].double() @ a[0][:, at].double().T.contiguous()
    mag = x[:, at].double().abs() @ a[0][:, at].double().abs().T.contiguous()
    want = y.double() + t @ b[0].double().T.contiguous()
    et = 8 * 2 ** -24 * mag + 2 ** -22 * t.abs().amax(1, keepdim=True)
    B = b[0].double().abs().T.contiguous()
    tol = et @ B + 12 * 2 ** -24 * (t.abs() @ B) + 2 ** -24 * (y.double().abs() + want.abs())
    assert ((got.double() - want).abs() <= tol).all()
