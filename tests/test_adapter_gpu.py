"""Low-rank adapters of many requests (wg_adapter_add) on the GPU against the
formula in 64 bits. What no row may read (a slot's factors behind its rank,
slots that no row names) holds NaN."""
import pytest
import torch

from tests.test_paged_gpu import DEV, _gen, _i32

pytestmark = pytest.mark.gpu


def _starts(rows):
    start = [0]
    for r in rows:
        start.append(start[-1] + r)
    return start


class Set:
    """Adapters of these ranks over a projection K -> cols."""

    def __init__(self, ranks, K, cols, most=None, seed=0):
        from webgllm_amd import ops
        g = self.g = _gen(seed)
        self.ranks, self.K, self.cols, self.N = ranks, K, cols, sum(cols)
        n = len(ranks)
        self.most = most = most or -(-max(max(ranks), 1) // 8) * 8
        self.a = torch.full((n, len(cols), most, K), float("nan"), dtype=torch.float16, device=DEV)
        self.b = torch.full((n, self.N, most), float("nan"), dtype=torch.float16, device=DEV)
        for i, r in enumerate(ranks):
            self.a[i, :, :r] = (torch.randn((len(cols), r, K), generator=g, device=DEV) / K ** 0.5).half()
            self.b[i, :, :r] = (torch.randn((self.N, r), generator=g, device=DEV) * 0.05).half()
        self.scale = torch.rand(n, generator=g, device=DEV) + 0.5
        self.set = ops.Adapters(self.a, self.b, _i32(ranks), self.scale, cols)

    def rows(self, M, pad=0):
        x = (torch.randn((M, self.K + 8 * pad), generator=self.g, device=DEV) / 32).half()
        y = torch.randn((M, self.N + 4 * pad + (1 if pad else 0)), generator=self.g, device=DEV)
        f = 32 * (1 + 0.1 * torch.randn(M, generator=self.g, device=DEV))
        return x[:, :self.K], y[:, :self.N], f

    def want(self, x, y, f, at):
        """(result, bound) of rows whose adapter is `at`, in 64 bits. The bound:
        A x by sums of at most K / 32 + 64 additions in a row, each off by 2^-24 of
        sum |a x|; 22 bits of its largest value kept; `rank` additions, the product
        with the scales by 3 roundings, and the result's own half steps."""
        y, x = y.double(), x.double()
        if not 0 <= at < len(self.ranks) or not self.ranks[at]:
            return y, torch.zeros_like(y)
        r = self.ranks[at]
        s = float(self.scale[at]) * (1.0 if f is None else f.double()[:, None])
        out, tol, e = y.clone(), torch.zeros_like(y), 0
        for j, n in enumerate(self.cols):
            A, B = self.a[at, j, :r].double(), self.b[at, e:e + n, :r].double()
            t = x @ A.T.contiguous()
            et = (self.K / 32 + 64) * 2 ** -24 * (x.abs() @ A.abs().T.contiguous()) + \
                2 ** -22 * t.abs().amax(1, keepdim=True)
            add = s * (t @ B.T.contiguous())
            mag = abs(s) * (t.abs() @ B.abs().T.contiguous())
            out[:, e:e + n] += add
            tol[:, e:e + n] = abs(s) * (et @ B.abs().T.contiguous()) + (r + 4) * 2 ** -24 * mag
            e += n
        return out, tol + 2 ** -24 * (y.abs() + out.abs())

    def check(self, got, x, y, f, slots, rows=None):
        m = 0
        for b, at in enumerate(slots):
            n = 1 if rows is None else rows[b]
            sl = slice(m, m + n)
            m += n
            if not n:
                continue
            want, tol = self.want(x[sl], y[sl], None if f is None else f[sl], at)
            off = (got[sl].double() - want).abs()
            assert (off <= tol).all(), (b, at, float((off - tol).max()), float(off.max()))


SHAPES = [(896, (896, 128, 128)), (896, (896,)), (64, (96,)), (8, (4,)), (4096, (4096, 1024, 1024)),
          (2048, (8192, 8192)), (4864, (896,)), (104, (20, 4, 36, 60)), (14336, (4096,))]


@pytest.mark.parametrize("K,cols", SHAPES)
@pytest.mark.parametrize("ranks", [[8], [16, 3, 64, 0, 1, 33], [128, 130, 256]])
def test_tokens(hip, K, cols, ranks):
    """A row each: adapters named once, twice and not at all, rows without one."""
    from webgllm_amd import ops
    c = Set(ranks + [7], K, cols, seed=K)  # (the last slot is nobody's)
    c.a[-1], c.b[-1] = float("nan"), float("nan")
    n = len(ranks)
    slots = [i % n for i in range(11)] + [-1, n + 1, 2 ** 31 - 1, -2 ** 31, 0]
    x, y, f = c.rows(len(slots), pad=1)
    for scale in (f, None):
        got = y.clone()
        big = torch.full((len(slots), c.N + 3), 5.0, device=DEV)
        big[:, :c.N] = y
        ops.adapter_add(big[:, :c.N], x, c.set, _i32(slots), row_scale=scale)
        assert (big[:, c.N:] == 5).all()
        c.check(big[:, :c.N], x, y, scale, slots)
        again = ops.adapter_add(got, x, c.set, _i32(slots), row_scale=scale)
        assert again is got and torch.equal(got, big[:, :c.N])
        assert torch.equal(got[11:15], y[11:15])


@pytest.mark.parametrize("K,cols", SHAPES)
@pytest.mark.parametrize("rows", [[5, 0, 1, 40, 0, 2], [131, 17, 1, 64], [33], [700, 3, 129, 40]])
@pytest.mark.parametrize("ranks", [[16, 5, 64, 40], [256, 7, 130, 200]])
def test_prompts(hip, K, cols, rows, ranks):
    """Rows of several sequences, some without an adapter; rows before the first
    and behind the last stay."""
    from webgllm_amd import ops
    c = Set(ranks, K, cols, seed=len(rows))
    slots = [(3 * i + 1) % 5 - 1 for i in range(len(rows))]
    M = sum(rows)
    x, y, f = c.rows(M + 5, pad=2)
    start = _i32([2 + s for s in _starts(rows)])
    got = ops.adapter_add(y.clone(), x, c.set, _i32(slots), start, f)
    assert torch.equal(got[:2], y[:2]) and torch.equal(got[2 + M:], y[2 + M:])
    sl = slice(2, 2 + M)
    c.check(got[sl], x[sl], y[sl], f[sl], slots, rows)
    assert torch.equal(got, ops.adapter_add(y.clone(), x, c.set, _i32(slots), start, f))


@pytest.mark.parametrize("K,cols", [(896, (896, 128, 128)), (4096, (4096,)), (14336, (256,))])
@pytest.mark.parametrize("rank", [5, 16, 40])
def test_a_tokens_bits_do_not_depend_on_the_batch(hip, K, cols, rank):
    """A row alone (one launch), in a small and in a large batch (two) gives the same
    bits."""
    from webgllm_amd import ops
    c = Set([rank, rank], K, cols, seed=rank)
    x, y, f = c.rows(300)
    slots = _i32([i % 2 for i in range(300)])
    want = ops.adapter_add(y.clone(), x, c.set, slots, row_scale=f)
    c.check(want[:6], x[:6], y[:6], f[:6], [0, 1] * 3)
    for a, b in ((0, 1), (7, 8), (40, 57)):
        got = ops.adapter_add(y[a:b].clone(), x[a:b], c.set, slots[a:b], row_scale=f[a:b])
        assert torch.equal(got, want[a:b])


@pytest.mark.parametrize("ranks", [[16, 8], [64, 40], [128, 9], [256, 256]])
def test_scratch_of_more_rows(hip, ranks):
    """Scratch of a batch's most rows does for any fewer, however they lie in
    sequences; nothing is written behind it."""
    from webgllm_amd import ops
    c = Set(ranks, 2048, (64, 32, 32), seed=9)
    whole = torch.full((ops.adapter_scratch(c.set, 700).numel() + 4096,), 77, dtype=torch.uint8,
                       device=DEV)
    sc = whole[:-4096]
    for rows in ([1], [5, 11], [33] * 3, [128], [1] * 200, [129, 127], [64] * 4, [500], [700], [20] * 35):
        x, y, f = c.rows(sum(rows))
        slots = [i % 2 for i in range(len(rows))]
        got = ops.adapter_add(y.clone(), x, c.set, _i32(slots), _i32(_starts(rows)), f, sc)
        c.check(got, x, y, f, slots, rows)
        assert (whole[-4096:] == 77).all()


def test_many_sequences(hip):
    """More sequences than a wave looks at once, few rows each, many adapters."""
    from webgllm_amd import ops
    ranks = [1 + i % 24 for i in range(150)]
    c = Set(ranks, 896, (128, 64), seed=3)
    rows = [i * 7 % 4 for i in range(900)]
    slots = [(i * 11) % 170 - 10 for i in range(900)]
    x, y, f = c.rows(sum(rows))
    got = ops.adapter_add(y.clone(), x, c.set, _i32(slots), _i32(_starts(rows)), f)
    c.check(got, x, y, f, slots, rows)
    x, y, f = c.rows(900)
    got = ops.adapter_add(y.clone(), x, c.set, _i32(slots), row_scale=f)
    c.check(got, x, y, f, slots)


@pytest.mark.parametrize("rows", [None, 1])
def test_the_most_sequences(hip, rows):
    """65,535 sequences of one row, by both forms."""
    from webgllm_amd import ops
    c, n = Set([8, 0, 3], 64, (16, 4), seed=10), 65535
    x, y, f = c.rows(n)
    slots = [(i * 7) % 5 - 1 for i in range(n)]
    start = None if rows is None else _i32(range(n + 1))
    got = ops.adapter_add(y.clone(), x, c.set, _i32(slots), start, f)
    slot = _i32(slots)
    for at in range(-1, 4):
        m = slot == at
        want, tol = c.want(x[m], y[m], f[m], at)
        assert ((got[m].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("rows", [None, [5, 40, 1]])
def test_factors_past_32_bits(hip, rows):
    """Slots whose factors lie past 2^32 bytes and 2^31 values."""
    from webgllm_amd import ops
    c = Set([64, 16, 40], 4096, (8192, 8192), most=64, seed=11)
    slots, M = [2, 0, 1], sum(rows) if rows else 3
    x, y, f = c.rows(M)
    start = None if rows is None else _i32(_starts(rows))
    want = ops.adapter_add(y.clone(), x, c.set, _i32(slots), start, f)
    c.check(want, x, y, f, slots, rows)
    n = 4200  # (of 524,288 and 1,048,576 values)
    a = torch.empty((n, 2, 64, 4096), dtype=torch.float16, device=DEV)
    b = torch.empty((n, 16384, 64), dtype=torch.float16, device=DEV)
    rank, scale = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(n, device=DEV)
    for big, small in ((a, c.a), (b, c.b), (rank, c.set.rank), (scale, c.scale)):
        big[n - 3:] = small
    many = ops.Adapters(a, b, rank, scale, c.cols)
    got = ops.adapter_add(y.clone(), x, many, _i32([n - 3 + i for i in slots]), start, f)
    assert torch.equal(got, want)


def test_large_and_small_values(hip):
    """Rows far apart in size, factors near the largest and smallest halves."""
    from webgllm_amd import ops
    c = Set([16, 8], 896, (64, 32), seed=4)
    c.a[0, :, :16] *= 3000
    c.b[0, :, :16] *= 1e5
    c.a[1, 0, :8] = 2.0 ** -24
    c.b[1, :, :8] = 2.0 ** -20
    for rows in (None, [30, 34]):
        slots = [0, 1] * 32 if rows is None else [0, 1]
        x, y, f = c.rows(64)
        x *= torch.logspace(-4, 4, 64, base=10, device=DEV)[torch.randperm(64, generator=c.g, device=DEV)][
            :, None].half()
        x.clamp_(-60000, 60000)
        y *= 1e-6
        start = None if rows is None else _i32(_starts(rows))
        got = ops.adapter_add(y.clone(), x, c.set, _i32(slots), start, f)
        assert torch.isfinite(got).all()
        c.check(got, x, y, f, slots, rows)


@pytest.mark.parametrize("rows", [None, [3, 5, 40]])
def test_values_that_are_not_finite(hip, rows):
    """In a row they reach that row alone, in a second factor's row that output of
    the adapter's rows alone."""
    from webgllm_amd import ops
    c = Set([16, 12, 24], 256, (64, 32), seed=5)
    slots = [0, 1, 2]
    M = sum(rows) if rows else 3
    start = None if rows is None else _i32(_starts(rows))
    x, y, f = c.rows(M)
    want = ops.adapter_add(y.clone(), x, c.set, _i32(slots), start, f)
    x[1, 7] = float("inf")
    c.b[2, 50, 3] = float("nan")
    got = ops.adapter_add(y.clone(), x, c.set, _i32(slots), start, f)
    last = M - (rows[2] if rows else 1)
    assert not torch.isfinite(got[1]).any() and not torch.isfinite(got[last:, 50]).any()
    same = torch.ones_like(got, dtype=torch.bool)
    same[1], same[last:, 50] = False, False
    assert torch.equal(got[same], want[same])


@pytest.mark.parametrize("rows", [None, [9, 0, 150, 1]])
def test_captured_call_follows_slots(hip, rows):
    """A call captured once, replayed as sequences change adapters and a slot is
    loaded anew; each replay as an eager call."""
    from webgllm_amd import ops
    c = Set([16, 8, 32], 896, (896, 128, 128), most=32, seed=6)
    slots = _i32([0, 1, 2, -1])
    start = None if rows is None else _i32(_starts(rows))
    x, y, f = c.rows(sum(rows) if rows else 4)
    sc = ops.adapter_scratch(c.set, len(y))
    got = y.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=s):
        ops.adapter_add(got, x, c.set, slots, start, f, sc)

    def load():
        c.a[1] = (torch.randn(c.a[1].shape, generator=c.g, device=DEV) / 30).half()
        c.b[1] = (torch.randn(c.b[1].shape, generator=c.g, device=DEV) * 0.1).half()
        c.set.rank[1] = 21
        c.scale[1] = 3.0

    for change in (lambda: None, lambda: slots.copy_(_i32([2, 2, 1, 0])), load,
                   lambda: slots.fill_(-1), lambda: slots.copy_(_i32([1, 1, 1, 1])),
                   lambda: c.set.rank.copy_(_i32([2 ** 31 - 1, -3, 0]))):
        change()
        if int(c.set.rank[0]) > 32:
            c.a[0], c.b[0] = 0.5, 0.25  # (a rank past the slot's is cut to it)
        got.copy_(y)
        gr.replay()
        want = ops.adapter_add(y.clone(), x, c.set, slots, start, f, torch.full_like(sc, 255))
        torch.cuda.synchronize()
        assert torch.isfinite(got).all() and torch.equal(got, want)


def test_two_streams_at_once(hip):
    from webgllm_amd import ops
    c = Set([16, 8, 32], 2048, (2048,), seed=7)
    x, y, f = c.rows(40)
    slots = _i32([i % 3 for i in range(40)])
    want = ops.adapter_add(y.clone(), x, c.set, slots, row_scale=f)
    outs = []
    torch.cuda.synchronize()
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            outs += [ops.adapter_add(y.clone(), x, c.set, slots, row_scale=f) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_beside_a_projection(hip):
    """Behind the GEMV and the GEMM of a 4-bit matrix, from their half inputs: the
    sum of the projection's result and the adapter's."""
    import numpy as np

    from oracle import oracle as O
    from webgllm_amd import ops
    N, K = 256, 512
    w = (np.random.default_rng(8).standard_normal((N, K)) * 0.02).astype(np.float32)
    m = ops.Q4Matrix.from_q4_0(ops.to_device_bytes(O.quantize_q4_0(w)).to(DEV), N, K)
    c = Set([16, 24], K, (128, 64, 64), seed=8)
    for M, project in ((2, ops.gemv), (100, ops.gemm)):
        x, _, f = c.rows(M)
        x = x.contiguous()
        base = project(m, x, row_scale=f)
        rows = [1, 1] if M == 2 else [63, 37]
        got = ops.adapter_add(base.clone(), x, c.set, _i32([1, 0]), _i32(_starts(rows)), f)
        c.check(got, x, base, f, [1, 0], rows)


def test_python_checks(hip):
    from webgllm_amd import ops
    c = Set([8, 4], 64, (32, 16))
    x, y, f = c.rows(2)
    slot = _i32([0, 1])
    for call, msg in ((lambda: ops.adapter_add(y, x.float(), c.set, slot), "halves"),
                      (lambda: ops.adapter_add(y, x[:, :56], c.set, slot), "shorter"),
                      (lambda: ops.adapter_add(y[:1], x, c.set, slot), "fit"),
                      (lambda: ops.adapter_add(y[:, :40], x, c.set, slot), "fit"),
                      (lambda: ops.adapter_add(y, x, c.set, slot[:1]), "2 rows"),
                      (lambda: ops.adapter_add(y, x, c.set, slot.long()), "int32"),
                      (lambda: ops.adapter_add(y, x, c.set, slot, _i32([0, 2])), "row_start"),
                      (lambda: ops.adapter_add(y, x, c.set, slot, row_scale=f[:1]), "row scales"),
                      (lambda: ops.adapter_add(y, x.cpu(), c.set, slot), "device"),
                      (lambda: ops.Adapters(c.a, c.b, c.set.rank, c.scale, (48,)), "parts"),
                      (lambda: ops.Adapters(c.a, c.b[:1], c.set.rank, c.scale, (32, 16)), "slots"),
                      (lambda: ops.Adapters(c.a.float(), c.b, c.set.rank, c.scale, (32, 16)), "halves"),
                      (lambda: ops.Adapters(c.a, c.b, c.set.rank.float(), c.scale, (32, 16)), "int32")):
        with pytest.raises(ValueError, match=msg):
            call()
    with pytest.raises(AttributeError):
        c.set.a = c.a
