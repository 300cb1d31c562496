"""Decode attention over a 4-bit pool where nearly all of the softmax's weight lies on one token with a zero value row: what is left of
the output is made of weights far below the largest."""

import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

from directkv_b200 import kernel  # noqa: E402
from directkv_b200._lib import get_context  # noqa: E402

DEV = "cuda:0"
N, NH_KV, PAGE = 1600, 8, 16
BATCH = 400                                               # requests over the same rows: enough that a warp has all tokens of one to itself


def _case(level, at, seed):
    """Codes of K and V; the weights of all tokens but `at` are about 2^level of the largest, their values are positive."""
    g = torch.Generator().manual_seed(seed)
    score = level * (1 + 0.05 * torch.randn(N, NH_KV, 1, generator=g))                   # log2 of the weight
    k = (score / (128 ** 0.5 * 1.4426950408889634)).expand(N, NH_KV, 128) * (1 + 0.02 * torch.randn(N, NH_KV, 128, generator=g))
    v = 0.5 + torch.rand(N, NH_KV, 128, generator=g)
    k[at], v[at] = 0.0, 0.0
    return [ref.quantise(x.to(torch.bfloat16)) for x in (k, v)]


def _want(q, parts, scale):
    """(out, bound) in 64 bits.  The bound counts: rounding of the result to bf16 (2^-8); of every weight to fp16 after a scaling that
    brings the largest to 2^12 at least (2^-11 of the weight, or 2^-25 where it is below the normal range: 2^-37 of the largest weight);
    scores of 128 products in fp32, in numerator and sum; sums of N terms in fp32."""
    n_q, nh_q, _ = q.shape
    k, v = ref.values(*parts[0]), ref.values(*parts[1])
    out, bound = torch.zeros(n_q, nh_q, 128, dtype=torch.float64), torch.zeros(n_q, nh_q, 128, dtype=torch.float64)
    for j in range(n_q):
        m = N - n_q + 1 + j
        for h in range(nh_q):
            kv = h // (nh_q // NH_KV)
            s = (k[:m, kv] @ q[j, h].double()) * scale
            p = torch.exp(s - s.max())
            size = float((k[:m, kv].abs() @ q[j, h].double().abs()).max()) * scale
            vv = v[:m, kv]
            o = p @ vv / p.sum()
            rel = 2 * size * 128 * 2.0 ** -23 + N * 2.0 ** -23 + 2.0 ** -20
            out[j, h] = o
            bound[j, h] = o * (2.0 ** -8 + rel) + torch.clamp(p * 2.0 ** -11, min=2.0 ** -37) @ vv / p.sum()
    return out, bound


@pytest.mark.parametrize("at", [0, 777, N - 20])
@pytest.mark.parametrize("level", [-20, -26, -30])
@pytest.mark.parametrize("batch,nh_q,n_q,columns", [(BATCH, 8, 1, 0), (BATCH, 16, 5, 3000), (1, 8, 1, 3000)])
def test_weights_far_below_the_largest_count(level, at, batch, nh_q, n_q, columns):
    parts = _case(level, at, 600 + at)
    pool = kernel.KV4Pool(*[t.to(DEV) for p in parts for t in p], page_size=PAGE)
    q = torch.ones(n_q, nh_q, 128, dtype=torch.bfloat16)
    table = torch.zeros(batch, N // PAGE + columns, dtype=torch.int32)
    table[:, :N // PAGE] = torch.arange(N // PAGE)
    lse = torch.zeros(batch, n_q, nh_q, device=DEV)
    out = kernel.decode_kv4(q.expand(batch, n_q, nh_q, 128).contiguous().to(DEV), pool, torch.full((batch,), N, dtype=torch.int32, device=DEV), 128 ** -0.5,
                            table.to(DEV), lse_out=lse)
    want, bound = _want(q, parts, 128 ** -0.5)
    assert (bound <= 0.05 * want).all(), "the bound must be small beside the output itself"
    error = (out.cpu().double() - want).abs()
    assert (error <= bound).all(), f"worst {(error / bound).max():.1f} times the bound, {(error / want).max():.3f} of the output"
    # the largest weight is 1 (a score of zero), the others add less than N * 2^-14
    assert (lse.abs() <= N * 2.0 ** -14).all()
    assert get_context(0).read_status() == 0
