"""Head norms with the position rotation on the GPU, against the plain 64-bit form."""

import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu

from directkv_b200 import kernel, workloads  # noqa: E402
from directkv_b200._lib import get_context  # noqa: E402

DEV = "cuda:0"
BAD_POSITION = 1 << 2


def _inputs(n, hq, hk, seed, fused=False):
    g = torch.Generator().manual_seed(seed)
    rows = (torch.randn(n, hq + 2 * hk, 128, generator=g) * 1.5).to(torch.bfloat16)
    if fused:
        dev = rows.to(DEV)
        return rows[:, :hq], rows[:, hq:hq + hk], dev[:, :hq], dev[:, hq:hq + hk], g
    q, k = rows[:, :hq].contiguous(), rows[:, hq:hq + hk].contiguous()
    return q, k, q.to(DEV), k.to(DEV), g


def _close(got, want, bound):
    got = got.cpu().double()
    assert got.shape == want.shape and torch.isfinite(got).all()
    worst = ((got - want).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{worst:.2f} times the bound"


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("n,hq,hk", [(1, 1, 1), (1, 32, 8), (3, 5, 1), (7, 4, 4), (130, 28, 4), (1000, 3, 2), (2, 56, 56), (5000, 32, 8), (6007, 9, 3), (12000, 5, 0)])
def test_norm_and_rotation(n, hq, hk, fused):
    q, k, qd, kd, g = _inputs(n, hq, hk, n + hq, fused)
    cs = workloads.build_cos_sin(2000, 10000.0)
    pos = torch.randint(0, 2000, (n,), generator=g).to(torch.int32 if n % 2 else torch.int64)
    wq = (1 + 0.3 * torch.randn(128, generator=g)).to(torch.bfloat16)
    wk = torch.randn(hk, 128, generator=g)                                  # per head, fp32
    per_head = torch.randn(hq, 128, generator=g).to(torch.bfloat16)
    for w_q, w_k, table in ((wq, wk, cs), (None, None, cs), (wq, None, None), (per_head, torch.randn(128, generator=g), cs)):
        dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
        got = kernel.qk_norm_rope(qd, kd, None if table is None else pos.to(DEV), dev(table), dev(w_q), dev(w_k), eps=1e-5)
        for y, x, w in zip(got, (q, k), (w_q, w_k)):
            _close(y, *ref.norm_rope(x, w, pos, table, 1e-5))
    assert get_context(0).read_status() == 0


def test_in_place_and_one_sided_calls():
    q, k, qd, kd, g = _inputs(33, 4, 2, 5, fused=True)
    cs = workloads.build_cos_sin(64, 500000.0)
    pos = torch.arange(33, dtype=torch.int32)
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    want_q, want_k = ref.norm_rope(q, w.cpu(), pos, cs, 1e-6), ref.norm_rope(k, w.cpu(), pos, cs, 1e-6)
    only_q = kernel.qk_norm_rope(qd, None, pos.to(DEV), cs.to(DEV), w)
    assert only_q[1] is None
    only_k = kernel.qk_norm_rope(None, kd, pos.to(DEV), cs.to(DEV), None, w)
    assert only_k[0] is None
    _close(only_q[0], *want_q), _close(only_k[1], *want_k)
    out = kernel.qk_norm_rope(qd, kd, pos.to(DEV), cs.to(DEV), w, w, q_out=qd, k_out=kd)
    assert out[0] is qd and torch.equal(qd, only_q[0]) and torch.equal(kd, only_k[1])


def test_zero_rows_and_bad_positions():
    q, k, qd, kd, g = _inputs(4, 2, 1, 6)
    qd[1] = 0
    q[1] = 0
    cs = workloads.build_cos_sin(10, 10000.0)
    pos = torch.tensor([9, 0, 10, -1], dtype=torch.int64)
    w = torch.ones(128, dtype=torch.bfloat16)
    got = kernel.qk_norm_rope(qd, kd, pos.to(DEV), cs.to(DEV), w.to(DEV), w.to(DEV))
    assert get_context(0).read_status() == BAD_POSITION
    _close(got[0], *ref.norm_rope(q, w, pos, cs, 1e-6)), _close(got[1], *ref.norm_rope(k, w, pos, cs, 1e-6))
    none = torch.empty(0, 2, 128, dtype=torch.bfloat16, device=DEV)
    assert kernel.qk_norm_rope(none, none, torch.empty(0, dtype=torch.int32, device=DEV), cs.to(DEV))[0].shape == (0, 2, 128)


def test_not_a_number_stays_in_its_row():
    q, k, qd, kd, g = _inputs(3, 2, 2, 7)
    qd[1, 0, 5] = float("nan")
    w = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    got = kernel.qk_norm_rope(qd, kd, None, None, w, w)[0].cpu()
    want, bound = ref.norm_rope(q, w.cpu(), None, None, 1e-6)
    assert torch.isnan(got[1, 0]).all()
    ok = torch.ones(3, 2, dtype=torch.bool)
    ok[1, 0] = False
    assert ((got.double() - want).abs() <= bound)[ok].all()
