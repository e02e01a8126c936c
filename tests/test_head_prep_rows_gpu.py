"""Head preparation into pages of more rows than run at once, on the GPU: the bits of
a call for each sequence."""
import pytest
import torch

from tests.test_paged_gpu import DEV, Case, _gen, _i32, _rope

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,KV,hd", [(32, 8, 64), (32, 8, 128), (14, 2, 64), (16, 16, 128)])
@pytest.mark.parametrize("rows", [[900, 0, 1000, 1, 999], [1400, 131, 1900, 566], [5000, 3500]])
@pytest.mark.parametrize("axes", [0, 3])
def test_many_rows(hip, H, KV, hd, rows, axes):
    from webgllm_amd import ops
    past = [7 * b for b in range(len(rows))]
    lens = [p + r for p, r in zip(past, rows)]
    c = Case(lens, KV, hd, 64, seen=lambda b: ())
    M, g = sum(rows), _gen(hd + axes)
    shape = ops.attn_shape(H, KV, hd, hd, 1e-5, True)
    qkv = torch.randn((M, (H + 2 * KV) * hd), generator=g, device=DEV)
    qn, kn = (1 + 0.1 * torch.randn(hd, generator=g, device=DEV) for _ in range(2))
    pos = torch.randint(0, 8192, (M, 3) if axes else (M,), generator=g, device=DEV,
                        dtype=torch.int32)
    more = dict(q_norm=qn, k_norm=kn,
                axes=ops.rope_axes([hd // 2 - 20, 10, 10], True) if axes else None)
    rope, start = _rope(1e6, hd, 8192), [0]
    for r in rows:
        start.append(start[-1] + r)
    q = ops.paged_head_prep(qkv, shape, rope, c.cache, pos=pos, row_start=_i32(start), **more)
    k, v = c.k.clone(), c.v.clone()
    c.k.fill_(float("nan")), c.v.fill_(float("nan"))
    for b, r in enumerate(rows):
        for t in range(start[b], start[b + 1], 500):
            n = min(500, start[b + 1] - t)  # (the sequence as long as these rows leave it)
            c.cache.lens.copy_(_i32(lens))
            c.cache.lens[b] = past[b] + t - start[b] + n
            one = ops.paged_head_prep(qkv[t:t + n], shape, rope, c.cache, pos=pos[t:t + n],
                                      row_start=_i32([0] * (b + 1) + [n] * (len(rows) - b)), **more)
            assert torch.equal(one, q[t:t + n])
    assert torch.equal(k.view(torch.int16), c.k.view(torch.int16))
    assert torch.equal(v.view(torch.int16), c.v.view(torch.int16))
