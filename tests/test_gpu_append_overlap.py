"""q_out where it may lie: on bf16 queries themselves, and between the rows of the buffer that holds q, k and v."""
import pytest
import torch

import b200q
from paged import Step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rows", [1, 3, 700])
@pytest.mark.parametrize("d,hq", [(64, 24), (128, 32)])
def test_in_place_gives_the_same_bits(rows, d, hq):
    step = Step([(rows, rows)], hq, 2, d, 16).to(DEV)
    y = torch.randn(rows, hq + 4, d, device=DEV).bfloat16()
    f, w = torch.full((d // 2,), 0.1, device=DEV), 1 + 0.1 * torch.randn(d, device=DEV)
    kw = dict(inv_freq=f, q_norm=w, k_norm=w)
    want = b200q.k_kv_append(y[:, :hq], y[:, hq:hq + 2], y[:, hq + 2:], *step.args(), **kw)
    got = b200q.k_kv_append(y[:, :hq], y[:, hq:hq + 2], y[:, hq + 2:], *step.args(), q_out=y[:, :hq], **kw)
    assert torch.equal(got, want) and got.data_ptr() == y.data_ptr()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_between_the_rows_of_one_buffer(dtype):
    hq, hkv, d = 4, 2, 64
    step = Step([(5, 9), (2, 40)], hq, hkv, d, 16).to(DEV)
    y = torch.randn(7, 2 * hq + 2 * hkv, d, device=DEV).to(dtype)   # q, k, v and room behind them
    old = y.clone()
    args = y[:, :hq], y[:, hq:hq + hkv], y[:, hq + hkv:hq + 2 * hkv], *step.args()
    want = b200q.k_kv_append(*args)
    flat = y.view(7, -1).view(torch.bfloat16)
    out = flat[:, flat.shape[1] - hq * d:].view(7, hq, d)
    assert torch.equal(b200q.k_kv_append(*args, q_out=out), want)
    assert torch.equal(y[:, :hq + 2 * hkv], old[:, :hq + 2 * hkv])


def test_fp32_queries_are_not_replaced_in_place():
    step = Step([(3, 9)], 4, 2, 64, 16).to(DEV)
    y = torch.randn(3, 8, 64, device=DEV)
    for out in (y.view(torch.bfloat16).view(3, 16, 64)[:, :4], y.view(-1).view(torch.bfloat16)[:3 * 256].view(3, 4, 64)):
        with pytest.raises(b200q.B200QError, match="invalid argument"):
            b200q.k_kv_append(y[:, :4], y[:, 4:6], y[:, 6:], *step.args(), q_out=out)
