"""Values that some rows of a step see and others do not, infinite or NaN: the others are as if the key were not there.

The rows of one sequence see different keys (a later token's, and with a window an earlier one's), yet share the products
with a tile of values, where 0 times such a value would be NaN.  Expected: the fp64 definition over values with zeros in
the bad places, which is right for every row that does not see them, and for the others too but in the bad places
themselves, where the bad value is what comes back (a row sees one bad value a column here)."""
import math

import pytest
import torch

import b200q
from paged import Step, attend
from test_gpu_attn import BOTH, DEV, Abs, queries

pytestmark = pytest.mark.gpu


def spoil(step, places):
    """places: (sequence, position, kv head, columns, value) -> (the step's clean values, mask and values of the rows that
    see a bad one [rows][hq][d])"""
    clean = step.v_pages.clone()
    group = step.hq // step.hkv
    hit = torch.zeros(step.rows, step.hq, step.d, dtype=torch.float64)
    for b, at, h, cols, bad in places:
        pages, rows = step.slots(b, torch.tensor([at]))
        for c in cols:
            step.v_pages[pages, h, rows, c] = bad
            clean[pages, h, rows, c] = 0
        r, n = step.sizes[b]
        for i in range(r):
            pos = n - r + i
            if at <= pos and (not step.window or at > pos - step.window):
                hit[int(step.cu[b]) + i, h * group:(h + 1) * group, torch.tensor(cols)] += bad
    return clean, hit


def run(f, sizes, hq, hkv, d, page, places, window=0, softcap=0.0, most=None):
    step = Step(sizes, hq, hkv, d, page, pad=1, junk=math.nan)
    step.window = window
    q = queries(step)
    clean, hit = spoil(step, places(step))
    step.to(DEV)
    out = f(q.to(DEV), *step.args(), most or step.most, window=window, softcap=softcap)
    torch.cuda.synchronize()
    assert b200q.device_error() == 0
    step.v_pages = clean
    kw = dict(window=window, softcap=softcap)
    want, a = attend(step, q, **kw), attend(Abs(step), q, **kw)
    n = int(step.cu[-1])
    got, hit = out.cpu().double()[:n], hit[:n]
    longest = max(m for _, m in sizes)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10 + longest * 2.0 ** -24) * a + 1e-30   # test_gpu_attn.py's
    ok = (got - want[:n]).abs() <= tol[:n]
    sees = hit != 0
    assert ok[~sees].all(), (int((~ok[~sees]).sum()), "rows spoilt that do not see the value", torch.nonzero(~ok & ~sees)[:5])
    assert torch.equal(torch.isnan(got[sees]), torch.isnan(hit[sees]))
    assert torch.equal(got[sees].nan_to_num(nan=0.0), hit[sees].nan_to_num(nan=0.0))


BAD = [math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 2, 64, 16), (2, 2, 128, 64), (20, 1, 128, 32), (64, 2, 64, 128)])
def test_a_later_tokens_value_does_not_reach_earlier_rows(f, bad, hq, hkv, d, page):
    """verify windows: short ones that leave blocks whole, and long ones that shares cut"""
    def places(s):
        got = []
        for b, (r, n) in enumerate(s.sizes):
            for i in range(1, r):   # each row but the first: its own key spoils a column of its own
                got.append((b, n - r + i, i % s.hkv, [7 * i % d], bad))
        got.append((0, s.sizes[0][1] - 1, s.hkv - 1, list(range(40, 44)), bad))
        return got
    run(f, [(5, 300), (2, 2), (8, 9000), (1, 40), (3, 129)], hq, hkv, d, page, places)
    run(f, [(4, 60), (3, 17)], hq, hkv, d, page, places, softcap=20.0)


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (20, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("window", [5, 37, 200])
def test_a_value_that_left_the_window_does_not_reach_later_rows(f, hq, hkv, d, window):
    def places(s):
        # the oldest key that the first row sees, which the next no longer does, and one two rows on
        return [(b, n - r + i - window + 1, 0, [3 + i, 50 + i], math.nan) for b, (r, n) in enumerate(s.sizes) for i in (0, 2)
                if n - r - window + 1 >= 0]
    run(f, [(6, 400), (9, 6000), (4, 205)], hq, hkv, d, 16, places, window=window)


@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 64), (4, 1, 128), (12, 2, 64)])
@pytest.mark.parametrize("window", [0, 90])
def test_prompts_keep_a_spoilt_tokens_value_from_the_rows_before_it(hq, hkv, d, window):
    def places(s):
        got = [(0, 5, 0, [1], math.inf), (0, 140, 0, [2, 9], math.nan), (0, 299, 0, [4], -math.inf), (1, 77, s.hkv - 1, [d - 1], math.nan)]
        return got + [(2, 1200 + i, 0, [i], math.nan) for i in range(0, 60, 7)]
    run(b200q.attn_prompt, [(300, 300), (64, 80), (100, 1290)], hq, hkv, d, 32, places, window=window)


@pytest.mark.parametrize("f", BOTH)
def test_a_whole_cache_of_nan_gives_nan(f):
    """every value bad: every row sees one, and the call ends as soon as any other"""
    step = Step([(9, 3000), (4, 50), (1, 700)], 8, 1, 128, 64, junk=math.nan)
    step.v_pages[:] = math.nan
    q = queries(step)
    step.to(DEV)
    out = f(q.to(DEV), *step.args(), 9)
    assert torch.isnan(out.float()).all() and b200q.device_error() == 0


def test_a_row_that_sees_an_infinity_keeps_it_beside_one_it_does_not_see():
    """both in one column: the row between them gets the infinity, not 0 times the other"""
    for f in BOTH:
        for hq in (4, 40):
            step = Step([(3, 50)], hq, 1, 64, 16)
            for at, bad in ((47, math.inf), (49, -math.inf)):
                pages, rows = step.slots(0, torch.tensor([at]))
                step.v_pages[pages, 0, rows, 9] = bad
            q = queries(step)
            step.to(DEV)
            out = f(q.to(DEV), *step.args(), 3).cpu().float()
            assert (out[:2, :, 9] == math.inf).all() and torch.isnan(out[2, :, 9]).all()
            out[:, :, 9] = 0
            assert torch.isfinite(out).all()


def test_a_long_context_is_gone_over_without_another_warps_wait_running_out():
    """262144 keys, the last token's value bad in every head: the block that holds its row has 255 more, each added up again over
    all keys by a warp, which takes longer than the 2 s after which a wait of the block's other warps gives up"""
    n, r, heads, d, page = 262144, 1280, 32, 64, 256
    g = torch.Generator(device=DEV).manual_seed(0)
    kp = torch.empty(n // page, heads, page, d, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    vp = torch.empty_like(kp).normal_(generator=g)
    vp[-1, :, -1] = math.nan
    q = torch.randn(r, heads, d, generator=g, device=DEV).bfloat16()
    table = torch.arange(n // page, dtype=torch.int32, device=DEV)[None]
    lens, cu = torch.tensor([n], dtype=torch.int32, device=DEV), torch.tensor([0, r], dtype=torch.int32, device=DEV)
    out = b200q.attn_prompt(q, kp, vp, table, lens, cu, r)
    torch.cuda.synchronize()
    assert b200q.device_error() == 0
    bad = torch.isnan(out.float())
    assert bad[-1].all() and not bad[:-1].any()
    for h in (0, 31):
        k, v = kp[:, h].reshape(n, d).double(), vp[:, h].reshape(n, d).double()
        for i in (r - 2, r - 100, r - 256, r - 257):
            m = n - r + i + 1
            p = torch.softmax(q[i, h].double() @ k[:m].T / 8, -1)
            want, a = p @ v[:m], p @ v[:m].abs()
            # p's rounding is off by 2^-8 a term at most, signs independent: 2^-8 of the norm of p v, which is the output's own
            # for independent values; and the output's 2^-8.  A column with 1 / sqrt(n) of A is judged by the norm of all 64.
            assert (out[i, h].double() - want).norm() <= 2.0 ** -6 * want.norm() and (want.abs() < 2.0 ** -4 * a).all()
