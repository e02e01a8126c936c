"""The paged cache on the GPU where rounding, values that are not finite and
work split between workgroups meet, against plain formulas in 64 bits."""
import pytest
import torch

from tests.test_paged_gpu import DEV, Case, _i32

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
