"""attn_decode and attn_prompt on a B200 against the definition in fp64.

Tolerances.  The output is bf16: off by at most 2^-8 of its value.  Before it, each probability is rounded to bf16 once
(2^-8 relative), so a row is off by at most 2^-8 sum_j p_j |v_j| = 2^-8 A, A the same attention over |v|.  The scores are
fp32 sums of d exact products (each below |q|_2 |k|_2, order unknown): d 2^-24 sum |q_i k_i| scale, at most 2^-17 * 45 for
these inputs (|q| < 30, |k| < 20 at d = 128, scale 1 / sqrt(d)), and ex2.approx adds 2^-22: together under 2^-11 of each
probability.  fp32 accumulation over n keys: n 2^-24 A at worst, under 2^-8 A for n below 2^16.  Where rows are longer than
that the check is on the norm.  So: |got - want| <= 2^-8 |want| + (2^-8 + 2^-10 + n 2^-24) A."""
import math

import pytest
import torch

import b200q
from paged import Step, attend

pytestmark = pytest.mark.gpu
DEV = "cuda"


def queries(step, seed=3, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(step.rows, step.hq, step.d, generator=g)).to(torch.bfloat16)


class Abs:
    """the step with |v| for v"""

    def __init__(self, s):
        self.__dict__.update(s.__dict__)
        self.v_pages = s.v_pages.cpu().abs()
        self.slots = s.slots


def check(step, q, got, **kw):
    want, a = attend(step, q, **kw), attend(Abs(step), q, **kw)
    n = int(step.cu[-1])
    longest = max(m for _, m in step.sizes)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10 + longest * 2.0 ** -24) * a + 1e-30
    got = got.cpu().double()[:n]
    worst = ((got - want[:n]).abs() / tol[:n]).max()
    assert worst <= 1, float(worst)


def run(step, f, q=None, **kw):
    q = queries(step) if q is None else q
    step.to(DEV)
    out = torch.full((step.rows, step.hq, step.d), 7.0, dtype=torch.bfloat16, device=DEV)
    got = f(q.to(DEV), *step.args(), step.most, out=out, **kw)
    torch.cuda.synchronize()
    assert got is out and b200q.device_error() == 0
    check(step, q, out, **kw)
    assert (out[int(step.cu[-1]):] == 7).all()   # padding rows as they were
    return out


BOTH = [b200q.attn_decode, b200q.attn_prompt]
DECODE = {"one key": [(1, 1)], "one row": [(1, 100)], "many": [(1, 1), (1, 16), (1, 17), (1, 700), (1, 31)],
          "verify": [(5, 300), (16, 16), (0, 40), (1, 1), (7, 4100)]}


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("sizes", sorted(DECODE))
@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (64, 256), (128, 128)])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (3, 3), (7, 1)])
def test_few_rows(f, sizes, d, page, hq, hkv):
    run(Step(DECODE[sizes], hq, hkv, d, page, pad=3, junk=math.nan, interleave=True), f)


PROMPT = {"whole": [(130, 130)], "chunk": [(100, 1000)], "ragged": [(1, 1), (257, 300), (0, 5), (64, 64), (33, 700)]}


@pytest.mark.parametrize("sizes", sorted(PROMPT))
@pytest.mark.parametrize("d,page", [(64, 32), (128, 16), (128, 256), (128, 128)])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (2, 2), (10, 2)])
def test_prompts(sizes, d, page, hq, hkv):
    run(Step(PROMPT[sizes], hq, hkv, d, page, pad=1, junk=math.nan), b200q.attn_prompt)


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("window", [1, 15, 16, 17, 128, 129, 5000])
@pytest.mark.parametrize("softcap", [0.0, 5.0])
def test_windows_and_caps(f, window, softcap):
    sizes = [(9, 600), (1, 1), (16, 20), (4, 1300)] + ([(150, 400)] if f is b200q.attn_prompt else [])
    step = Step(sizes, 8, 2, 64 if window % 2 else 128, 16, junk=math.nan)
    # pages that fell out of every row's window are free: the table names no page there
    for b, (r, n) in enumerate(sizes):
        step.table[b, :max(0, n - r - window + 1) // 16] = -1
    out = run(step, f, window=window, softcap=softcap)
    assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("f", BOTH)
def test_sequences_without_a_visible_key_give_zeros(f):
    step = Step([(2, 0), (3, 2), (1, 5)], 4, 2, 128, 16, junk=math.inf)
    out = run(step, f)
    assert (out[:3] == 0).all() and (out[3:6] != 0).any()
    step = Step([(1, 0)], 4, 4, 64, 16)
    assert (run(step, f) == 0).all()


@pytest.mark.parametrize("f", BOTH)
def test_scale_and_large_scores(f):
    step = Step([(3, 90), (1, 40)], 4, 2, 64, 16)
    q = queries(step, scale=1.0)
    run(step, f, q=q, scale=0.01)
    # one key far above the others: its value alone comes back, and nothing overflows
    step = Step([(2, 200)], 2, 1, 64, 16)
    pages, rows = step.slots(0, torch.tensor([77]))
    step.k_pages[pages, 0, rows] = 30.0
    q = torch.full((2, 2, 64), 30.0).to(torch.bfloat16)
    out = run(step, f, q=q, scale=1.0)
    assert torch.equal(out.cpu(), step.v_pages[pages, 0, rows].cpu()[:, None].expand(2, 2, 64))


@pytest.mark.parametrize("f", BOTH)
def test_a_visible_nan_reaches_its_rows_alone(f):
    step = Step([(2, 50), (1, 60)], 4, 2, 64, 16)
    pages, rows = step.slots(0, torch.tensor([10]))
    step.v_pages[pages, 1, rows, 5] = math.nan
    q = queries(step)
    step.to(DEV)
    out = f(q.to(DEV), *step.args(), 2)
    bad = torch.isnan(out).cpu()
    want = torch.zeros(3, 4, 64, dtype=torch.bool)
    want[:2, 2:, 5] = True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("f", BOTH)
def test_strided_rows(f):
    step = Step([(3, 70), (2, 9)], 4, 2, 128, 32).to(DEV)
    y = torch.randn(5, 8, 128, device=DEV).to(torch.bfloat16)
    z = torch.zeros(5, 6, 128, device=DEV).to(torch.bfloat16)
    f(y[:, 2:6], *step.args(), 3, out=z[:, 1:5])
    check(step, y[:, 2:6].contiguous(), z[:, 1:5].contiguous())
    assert (z[:, 0] == 0).all() and (z[:, 5] == 0).all()


@pytest.mark.parametrize("f", BOTH)
def test_the_same_bits_again_and_on_another_stream(f):
    step = Step([(4, 3000), (2, 500), (1, 7000)], 8, 2, 128, 64).to(DEV)
    q = queries(step).to(DEV)
    one = f(q, *step.args(), 4)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:   # calls that may overlap: each has its own scratch
        with torch.cuda.stream(s):
            outs.append(f(q, *step.args(), 4))
    torch.cuda.synchronize()
    assert all(torch.equal(one, o) for o in outs)


@pytest.mark.parametrize("f", BOTH)
def test_captured_and_replayed_with_new_lengths(f):
    step = Step([(2, 300), (1, 40)], 4, 2, 64, 16)
    q = queries(step)
    step.to(DEV)
    qd = q.to(DEV)
    f(qd, *step.args(), 2)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):   # two graphs of the same call
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f(qd, *step.args(), 2))
        graphs.append(g)
    for sizes in ([(2, 300), (1, 40)], [(2, 17), (1, 1)], [(2, 290), (1, 33)]):
        step.lens.copy_(torch.tensor([n for _, n in sizes]))
        step.sizes = sizes
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            check(step, q, o)


@pytest.mark.parametrize("f", BOTH)
def test_bad_tables_lengths_and_row_counts_are_reported(f):
    step = Step([(1, 40), (1, 20)], 4, 2, 64, 16)
    q = queries(step)
    want = attend(step, q)
    step.table[0, 1] = 10 ** 6
    step.to(DEV)
    out = f(q.to(DEV), *step.args(), 1)
    assert b200q.device_error() == 2 << 20 and b200q.device_error() == 0
    assert torch.isfinite(out.float()).all()
    assert ((out[1].cpu().double() - want[1]).abs() <= 0.02 * want.abs().max()).all()
    step = Step([(1, 40), (1, 20)], 4, 2, 64, 16)
    step.lens[1] = 1000
    step.to(DEV)
    f(q.to(DEV), *step.args(), 1)
    assert b200q.device_error() & (2 << 20)
    step = Step([(40, 40), (1, 20)], 4, 2, 64, 16).to(DEV)
    f(torch.zeros(41, 4, 64, dtype=torch.bfloat16, device=DEV), *step.args(), 1)
    assert b200q.device_error() == 4 << 20


def test_a_long_cache_and_an_offset_past_32_bits():
    """one row over 40,000 keys, their pages at the end of a pool of more than 2^31 values"""
    n, page, d = 40000, 128, 128
    need = -(-n // page)
    pages = (1 << 31) // (page * d) + need + 8
    pool = torch.empty(pages, 1, page, d, dtype=torch.bfloat16, device=DEV)
    pool[-need:].normal_()
    step = Step([(1, 1)], 4, 1, d, page)
    step.sizes = [(1, n)]
    step.lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    step.cu = step.cu.to(DEV)
    step.table = torch.arange(pages - need, pages, dtype=torch.int32, device=DEV)[None]
    step.k_pages = step.v_pages = pool
    q = queries(step)
    for f in BOTH:
        got = f(q.to(DEV), *step.args(), 1)
        small = Step([(1, 1)], 4, 1, d, page)
        small.sizes, small.cu = [(1, n)], step.cu
        small.table = torch.arange(need, dtype=torch.int32)[None]
        small.k_pages = small.v_pages = pool[-need:].cpu()
        check(small, q, got)


def test_many_sequences():
    """more sequences than a block has threads, most of them short"""
    g = torch.Generator().manual_seed(0)
    sizes = [(1, int(torch.randint(1, 60, (), generator=g))) for _ in range(700)]
    sizes[300] = (1, 3000)
    sizes[5] = (0, 10)
    run(Step(sizes, 4, 2, 64, 16), b200q.attn_decode)
    run(Step(sizes, 4, 2, 64, 16), b200q.attn_prompt)


@pytest.mark.parametrize("d,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("hq,hkv,rows", [(8, 8, 1), (16, 8, 8), (32, 8, 16)])
def test_shares_longer_than_the_ring(d, page, hq, hkv, rows):
    """every CTA walks several sequences, with far more keys than its shared memory holds at once"""
    g = torch.Generator().manual_seed(1)
    sizes = [(rows, int(torch.randint(2000, 6000, (), generator=g))) for _ in range(9)] + [(rows, 16), (rows, 9000)]
    run(Step(sizes, hq, hkv, d, page, junk=math.nan), b200q.attn_decode)


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("hq,hkv,rows", [(17, 1, 1), (12, 2, 3), (8, 1, 16), (64, 2, 4), (40, 1, 16)])
@pytest.mark.parametrize("d,page,window", [(128, 64, 0), (64, 16, 0), (64, 128, 300), (128, 256, 129)])
def test_rows_of_one_tile_and_past_it(f, hq, hkv, rows, d, page, window):
    """17 to 128 rows a kv head, and 640: one to 47 steps, an odd one at the end, blocks that shares cut and whole ones"""
    sizes = [(rows, 128), (rows, 6000), (0, 9), (1, 129), (rows, rows), (rows, 257), (rows, 1500)]
    run(Step(sizes, hq, hkv, d, page, pad=2, junk=math.nan), f, window=window)


def test_more_row_blocks_than_a_warp_has_lanes():
    """600 rows of 16 query heads: 38 blocks of 256 rows, shares that begin and end inside them"""
    run(Step([(20, 20), (600, 700), (1, 3), (530, 530)], 16, 1, 64, 16, junk=math.nan), b200q.attn_prompt)
    run(Step([(600, 700), (9, 5)], 16, 1, 128, 64), b200q.attn_prompt, window=40)


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("hq", [2, 20])
@pytest.mark.parametrize("softcap", [0.5, 2.0, 30.0, 1e4, 1e7])
def test_scores_on_all_sides_of_the_cap(f, hq, softcap):
    """from scores far beyond the cap (there tanh's slope brings the scores' own errors to nothing) to caps far beyond the
    scores: tanh is right to 2^-16 of its value throughout, so a probability to 2^-16 times 30, below the 2^-11 above"""
    step = Step([(3, 500), (1, 129), (5, 40)], hq, 1, 64, 16)
    run(step, f, q=queries(step, scale=5.0), softcap=softcap)
    step = Step([(3, 500), (1, 129), (5, 40)], hq, 1, 128, 32)
    run(step, f, softcap=softcap, window=100)


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("hq", [2, 20])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_score_that_is_no_number_spoils_its_rows_alone(f, hq, bad):
    """query heads 0 and the last hold it; the others are as the definition has them"""
    step = Step([(2, 300), (1, 60)], hq, 1, 64, 16)
    q = queries(step)
    spoilt = q.clone()
    spoilt[0, 0, 3] = spoilt[1, hq - 1, 3] = bad
    for softcap in (0.0, 20.0):
        want = attend(step, q, softcap=softcap)
        step.to(DEV)
        out = f(spoilt.to(DEV), *step.args(), 2, softcap=softcap).cpu().double()
        left = torch.ones(3, hq, dtype=torch.bool)
        left[0, 0] = left[1, hq - 1] = False
        a = attend(Abs(step), q, softcap=softcap)
        assert ((out - want).abs()[left] <= (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10 + 300 * 2.0 ** -24) * a)[left]).all()
        if softcap == 0 or math.isnan(bad):
            assert torch.isnan(out[0, 0]).all() and torch.isnan(out[1, hq - 1]).all()


@pytest.mark.parametrize("f", BOTH)
@pytest.mark.parametrize("d,page,width", [(128, 64, 16), (128, 64, 17), (64, 16, 24), (64, 16, 25), (128, 128, 3)])
@pytest.mark.parametrize("batch", [1, 18, 40])
def test_tables_at_the_widths_that_leave_blocks_whole(f, d, page, width, batch):
    """384 and 1024 keys of table a sequence, and a page more; more blocks than CTAs; windows that empty none and some"""
    g = torch.Generator().manual_seed(2)
    top = width * page
    sizes = [(1, top)] + [(1, int(torch.randint(0, top + 1, (), generator=g))) for _ in range(batch - 1)]
    run(Step(sizes, 8, 4, d, page, junk=math.nan), f)
    run(Step([(3, n) for _, n in sizes], 8, 4, d, page, junk=math.nan), f, window=37)
