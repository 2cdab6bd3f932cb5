"""Padding rows of an append, before the first sequence and behind the last: they may hold anything, count for nothing and
stay as they are, while the rows between them come out as they do alone."""
import math

import pytest
import torch

import b200q
from paged import Step

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,before,behind", [(64, 0, 9), (128, 3, 0), (128, 5, 600)])
def test_what_padding_rows_hold_is_of_no_matter(dtype, d, before, behind):
    hq, hkv = 6, 2
    step = Step([(4, 30), (0, 8), (7, 7)], hq, hkv, d, 16).to(DEV)
    n = step.rows
    g = torch.Generator().manual_seed(2)
    x = torch.randn(before + n + behind, hq + 2 * hkv, d, generator=g).to(dtype).to(DEV)
    x[:before], x[before + n:] = math.nan, math.inf
    f, w = torch.full((d // 2,), 0.3, device=DEV), 1 + 0.1 * torch.randn(d, generator=g).to(DEV)
    kw = dict(inv_freq=f, q_norm=w, k_norm=w)
    parts = lambda y: (y[:, :hq], y[:, hq:hq + hkv], y[:, hq + hkv:])
    want = b200q.k_kv_append(*parts(x[before:before + n]), *step.args(), **kw)
    pages = step.k_pages.clone(), step.v_pages.clone()
    step.k_pages.fill_(3.0), step.v_pages.fill_(3.0)
    out = torch.full((x.shape[0], hq, d), 7.0, dtype=torch.bfloat16, device=DEV)
    b200q.k_kv_append(*parts(x), step.k_pages, step.v_pages, step.table, step.lens, step.cu + before, q_out=out, **kw)
    assert b200q.device_error() == 0
    assert torch.equal(out[before:before + n], want)
    assert (out[:before] == 7).all() and (out[before + n:] == 7).all()
    for b, (r, m) in enumerate(step.sizes):
        at, rows = step.slots(b, torch.arange(m - r, m))
        for now, then in ((step.k_pages, pages[0]), (step.v_pages, pages[1])):
            assert torch.equal(now[at, :, rows], then[at, :, rows])
            now[at, :, rows] = 3.0
    assert (step.k_pages == 3).all() and (step.v_pages == 3).all()   # nothing else was stored
