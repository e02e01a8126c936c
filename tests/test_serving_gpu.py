"""Adapters, head preparation under several axes and attention behind shared
prefixes as a server of many requests runs them, on the GPU: two adapters'
requests, each behind its own prefix with an image, prompts and then tokens."""
import pytest
import torch

from tests.test_adapter_gpu import Set
from tests.test_paged_gpu import DEV, _attend, _gen, _i32, _near, _rope

pytestmark = pytest.mark.gpu

D, H, KV, HD, PAGE = 512, 8, 2, 64, 16
QKV = (H * HD, KV * HD, KV * HD)
SECTIONS = [8, 12, 12]


def _matrix(N, K, seed):
    import numpy as np

    from oracle import oracle as O
    from webgllm_amd import ops
    w = (np.random.default_rng(seed).standard_normal((N, K)) * 0.02).astype(np.float32)
    return ops.Q4Matrix.from_q4_0(ops.to_device_bytes(O.quantize_q4_0(w)).to(DEV), N, K)


class Server:
    """Six sequences, 0 .. 3 of adapter 1 and 4, 5 of adapter 0, behind prefixes of
    96 and 48 entries, in one pool of NaN."""

    def __init__(self):
        from webgllm_amd import ops
        self.g = _gen(40)
        self.qkv, self.o = _matrix(sum(QKV), D, 1), _matrix(D, H * HD, 2)
        self.aq, self.ao = Set([16, 24], D, QKV, seed=41), Set([8, 5], H * HD, (D,), seed=42)
        self.shape = ops.attn_shape(H, KV, HD)
        self.rope = _rope(1e4, HD, 4096)
        self.axes = ops.rope_axes(SECTIONS)
        self.pre, self.starts = [96, 48], [0, 4, 6]
        self.slots = [1, 1, 1, 1, 0, 0]
        order = torch.randperm(60, generator=self.g, device=DEV).tolist()
        rows, at = [], 0
        for (a, b), p in zip(((0, 4), (4, 6)), self.pre):
            first, at = order[at:at + p // PAGE], at + p // PAGE
            for _ in range(a, b):
                rows.append(first + order[at:at + 4] + [-1] * (700 - p // PAGE - 4))
                at += 4
        self.k = torch.full((60, PAGE, KV * HD), float("nan"), dtype=torch.float16, device=DEV)
        self.v = self.k.clone()
        self.table = _i32(rows)
        self.cache = ops.PagedCache(self.k, self.v, self.table, _i32([0] * 6))

    def x(self, M):
        return (torch.randn((M, D), generator=self.g, device=DEV) / 32).half(), \
            32 * (1 + 0.1 * torch.randn(M, generator=self.g, device=DEV))

    def entries(self, b, n):
        i = torch.arange(n, device=DEV)
        at = self.table[b][i // PAGE].long() * PAGE + i % PAGE
        return tuple(t.view(-1, KV, HD)[at].double() for t in (self.k, self.v))


def _turn(x, pos):
    """Heads [n, HD] rotated by a row's positions, in 64 bits."""
    a = torch.tensor([pos[e] for e, n in enumerate(SECTIONS) for _ in range(n)],
                     dtype=torch.float64, device=DEV)
    a = a * 1e4 ** (-2.0 * torch.arange(HD // 2, device=DEV).double() / HD)
    x1, x2 = x[..., :HD // 2], x[..., HD // 2:]
    return torch.cat([x1 * a.cos() - x2 * a.sin(), x2 * a.cos() + x1 * a.sin()], -1)


def test_requests_of_two_adapters(hip):
    """Prefixes as prompts of the groups' first sequences, then rows of all of them:
    tokens and drafts. Every value within its operator's bound of 64 bits, from what
    the operators before it wrote."""
    from webgllm_amd import ops
    s = Server()
    group_start, shared, slot = _i32(s.starts), _i32(s.pre), _i32(s.slots)
    lens = [0] * 6

    def step(rows, pos):
        M, start = sum(rows), [0]
        for r in rows:
            start.append(start[-1] + r)
        one = rows == [1] * 6
        for b, r in enumerate(rows):
            lens[b] += r
        s.cache.lens.copy_(_i32(lens))
        x, f = s.x(M)
        project = ops.gemv if M <= 8 else ops.gemm
        base = project(s.qkv, x, row_scale=f)
        rs = None if one else _i32(start)
        y = ops.adapter_add(base.clone(), x, s.aq.set, slot, rs, f)
        s.aq.check(y, x, base, f, s.slots, rows)
        q = ops.paged_head_prep(y, s.shape, s.rope, s.cache, pos=_i32(pos), row_start=rs, axes=s.axes)
        att = ops.paged_attn_shared(q, s.shape, s.cache, group_start, shared, rs)
        base = project(s.o, att, row_scale=f)
        z = ops.adapter_add(base.clone(), att, s.ao.set, slot, rs, f)
        s.ao.check(z, att, base, f, s.slots, rows)
        m = 0
        for b, r in enumerate(rows):
            k, v = s.entries(b, lens[b])
            for t in range(r):
                i = lens[b] - r + t
                heads = y[m].double().view(-1, HD)
                want = _turn(heads[:H + KV], pos[m])
                # (cosines and sines off by 2^-22, two products and a sum; then the half)
                tol = 2 ** -20 * heads[:H + KV].abs().amax(-1, keepdim=True)
                assert ((q[m].double().view(H, HD) - want[:H] / 8).abs() <= tol[:H]).all()
                off = (k[i] - want[H:]).abs()
                assert (off <= tol[H:] + 2 ** -11 * want[H:].abs() + 2 ** -25).all()
                assert torch.equal(v[i], heads[H + KV:].half().double())
                out, bound, _ = _attend(q[m].view(H, HD), k, v, i, 0, 0)
                _near(att[m], out, bound, (b, t))
                m += 1
        return att

    # the prefixes: each by its group's first sequence, with an image of 4 x 4 patches
    def image(n):
        text = [[i] * 3 for i in range(8)]
        patches = [[8, 8 + i // 4, 8 + i % 4] for i in range(16)]
        return text + patches + [[12 + i] * 3 for i in range(n - 24)]

    step([96, 0, 0, 0, 48, 0], image(96) + image(48))
    for b in range(6):
        lens[b] = s.pre[0] if b < 4 else s.pre[1]
    at = [84, 84, 84, 84, 36, 36]  # positions run behind the entries
    for rows in ([5, 1, 9, 2, 3, 4], [1] * 6, [1] * 6, [2, 0, 1, 3, 0, 1], [1] * 6):
        pos = [[at[b] + t] * 3 for b, r in enumerate(rows) for t in range(r)]
        step(rows, pos)
        at = [a + r for a, r in zip(at, rows)]


def test_a_captured_token_step(hip):
    """A token of each sequence captured whole (projection, adapter, preparation,
    attention, projection, adapter), replayed as lengths, positions, adapters and
    groups change: each replay the eager step's bits."""
    from webgllm_amd import ops
    s = Server()
    s.k.copy_(torch.randn(s.k.shape, generator=s.g, device=DEV))
    s.v.copy_(torch.randn(s.v.shape, generator=s.g, device=DEV))
    group_start, shared, slot = _i32(s.starts), _i32(s.pre), _i32(s.slots)
    s.cache.lens.copy_(_i32([p + i for p, i in zip([96] * 4 + [48] * 2, (3, 20, 7, 31, 1, 40))]))
    pos = _i32([[50 + i, 60 + i, 70 + i] for i in range(6)])
    x, f = s.x(6)
    sq, so = ops.adapter_scratch(s.aq.set, 6), ops.adapter_scratch(s.ao.set, 6)
    sa = ops.paged_shared_scratch(s.cache, s.shape, 6, 2)
    y, z = torch.empty((6, sum(QKV)), device=DEV), torch.empty((6, D), device=DEV)
    q = torch.empty((6, H * HD), device=DEV)
    att = torch.empty((6, H * HD), dtype=torch.float16, device=DEV)

    def step():
        ops.gemv(s.qkv, x, out=y, row_scale=f)
        ops.adapter_add(y, x, s.aq.set, slot, row_scale=f, scratch=sq)
        ops.paged_head_prep(y, s.shape, s.rope, s.cache, pos=pos, q_out=q, axes=s.axes)
        ops.paged_attn_shared(q, s.shape, s.cache, group_start, shared, scratch=sa, out=att)
        ops.gemv(s.o, att, out=z, row_scale=f)
        ops.adapter_add(z, att, s.ao.set, slot, row_scale=f, scratch=so)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for change in (lambda: None, lambda: (s.cache.lens.add_(1), pos.add_(1)),
                   lambda: slot.copy_(_i32([0, -1, 1, 1, 1, 0])),
                   lambda: group_start.copy_(_i32([0, 3, 6])), lambda: shared.copy_(_i32([64, 0])),
                   lambda: (x.copy_(s.x(6)[0]), s.cache.lens.add_(1), pos.add_(1))):
        change()
        old = s.k.clone(), s.v.clone()
        graph.replay()
        got = [t.clone() for t in (y, q, att, z, s.k, s.v)]
        s.k.copy_(old[0]), s.v.copy_(old[1])
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (y, q, att, z, s.k, s.v)):
            assert torch.isfinite(b).all() and torch.equal(a, b)
