"""Page-table entries that name no page, at places that rows see: zeros and bit 21, whatever the number is.

Expected is the definition over a table whose entry names a page of zeros; the tolerance is that of the attention's own
tests (test_gpu_attn.py)."""
import pytest
import torch

import b200q
from paged import Step
from test_gpu_attn import BOTH, DEV, check, queries

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("hq", [4, 40])   # up to 16 rows a kv head, and more
@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (64, 128), (128, 256)])
@pytest.mark.parametrize("entry", [-2 ** 31, -2 ** 31 + 1, -1, 10 ** 6, 2 ** 31 - 1])
def test_an_entry_outside_the_cache_reads_as_zeros(f, hq, d, page, entry):
    def step():
        return Step([(1, 700), (2, 3 * page), (1, 20)], hq, 2, d, page, spare=1)
    good, bad = step(), step()
    spare = (set(range(good.k_pages.shape[0])) - set(good.table.flatten().tolist())).pop()
    for b, i in ((0, 1), (1, 2)):
        good.table[b, i] = spare
        bad.table[b, i] = entry
    good.k_pages[spare] = 0
    good.v_pages[spare] = 0
    q = queries(good)
    bad.to(DEV)
    out = f(q.to(DEV), *bad.args(), 2)
    assert b200q.device_error() == 2 << 20 and b200q.device_error() == 0
    check(good, q, out)
