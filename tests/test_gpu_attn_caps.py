"""Large scores under large caps.  The scores are whole numbers (sums of products below 2^24, exact in fp32), so the cap's
own error is all there is.  A capped score is held to 2^-21 of its value, or 2^-12 where that is more: the quotient is
rounded by 2^-24, the tanh is off by 2^-22 and the products with the cap and log2 e by 2^-24 each; where the prompt form
takes a polynomial instead, its error is below 2^-12.  With every score off by at most e, each way, a row changes by
sum p_j |v_j - o| (exp(e) - 1), at most (A + |o|)(exp(e) - 1) with A = sum p_j |v_j|.  Keys of nearly one score stand in steps
whose other scores are small, and in steps that hold one far beyond the cap."""
import math

import pytest
import torch

import b200q
from paged import Step, attend
from test_gpu_attn import BOTH, DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("hq", [2, 20])
@pytest.mark.parametrize("cap,score", [(4e5, 132096), (4e5, 80384), (1e5, 33024), (1e4, 3296), (3e4, 464), (1000, 336), (100, 36), (50, 17)])
def test_equal_scores_weigh_alike_whatever_stands_beside_them(f, hq, cap, score):
    step = Step([(1, 512), (2, 700)], hq, 1, 64, 16)
    g = torch.Generator().manual_seed(5)
    # q = (16, 1, 0 ..): score = 16 k0 + k1
    q = torch.zeros(step.rows, hq, 64)
    q[..., 0], q[..., 1] = 16.0, 1.0
    q = q.to(torch.bfloat16)
    top = torch.tensor(float(score // 16)).to(torch.bfloat16).float()   # k0: a bf16
    for b, n in ((0, 512), (1, 700)):
        pages, rows = step.slots(b, torch.arange(n))
        k = torch.zeros(n, 64)
        k[:, 0] = top
        k[:, 1] = torch.randint(-1, 2, (n,), generator=g)
        far = torch.arange(n) // 128 % 2 == 1   # every other 128 keys hold one whose score is far below
        k[far & (torch.arange(n) % 128 == 77), 0] = -3 * top
        step.k_pages[pages, 0, rows] = k.to(torch.bfloat16)
        v = torch.where(far, -1.0, 1.0)[:, None] + 0.25 * torch.randn(n, 64, generator=g)
        step.v_pages[pages, 0, rows] = v.to(torch.bfloat16)
    want = attend(step, q, scale=1.0, softcap=cap)
    values = step.v_pages
    step.v_pages = values.abs()
    a = attend(step, q, scale=1.0, softcap=cap)
    step.v_pages = values
    step.to(DEV)
    out = f(q.to(DEV), *step.args(), 2, scale=1.0, softcap=cap).cpu().double()
    slip = math.expm1(2.0 ** -21 * 1.01 * score + 2.0 ** -12)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10) * a + slip * (a + want.abs())
    worst = float(((out - want).abs() / tol).max())
    assert worst <= 1, worst
    assert b200q.device_error() == 0
