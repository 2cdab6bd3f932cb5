"""k_kv_append on a B200 against the definition in fp64: cache slots, rotation, norm, strides, padding, bad tables.

Tolerances.  Outputs are bf16: a rounding is off by at most half a step, eps / 2 = 2^-8 of the value.  Before it the
values are fp32: the norm's factor carries a sum of d squares, an rsqrt and two products (under 16 roundings of 2^-24),
the rotation two products, a sum and a cos / sin of an angle below pi rounded once to fp32 (absolute 2^-22 at most, times
the pair's size).  So an output is within 2^-8 of its own size plus 2^-18 of its pair's size of the definition, and a
head without norm and rotation is the exact rounding of its input."""
import pytest
import torch

import b200q
from paged import Step, norm, rotate

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bound(want, heads):
    """the per-value tolerance: want's own size and its head's largest (an upper bound of its pair's)"""
    return 2.0 ** -8 * want.abs() + 2.0 ** -17 * heads.abs().amax(-1, keepdim=True) + 1e-30


def inputs(step, dtype, seed=1, extra=0):
    """q, k, v as views of one row [hq + 2 hkv + extra heads]"""
    g = torch.Generator().manual_seed(seed)
    y = torch.randn(step.rows, step.hq + 2 * step.hkv + extra, step.d, generator=g).to(dtype)
    a, b = step.hq, step.hq + step.hkv
    return y, (y[:, :a], y[:, a:b], y[:, b:b + step.hkv])


def expected(step, parts, inv_freq=None, interleaved=False, weights=(None, None), eps=1e-6):
    q, k, v = (x.double() for x in parts)
    if weights[0] is not None:
        q = norm(q, weights[0], eps)
    if weights[1] is not None:
        k = norm(k, weights[1], eps)
    if inv_freq is not None:
        pos = torch.cat([torch.arange(n - r, n) for r, n in step.sizes] + [torch.zeros(step.pad)]).double()
        q, k = rotate(q, pos, inv_freq, interleaved), rotate(k, pos, inv_freq, interleaved)
    return q, k, v


def check(step, parts, before, q_out, sentinel, **kw):
    q, k, v = expected(step, parts, **kw)
    n = int(step.cu[-1])
    exact = kw.get("inv_freq") is None and kw.get("weights", (None, None)) == (None, None)
    got = q_out.cpu()
    if exact:
        assert torch.equal(got[:n], parts[0][:n].to(torch.bfloat16))
    assert ((got[:n].double() - q[:n]).abs() <= bound(q[:n], q[:n])).all()
    assert torch.equal(got[n:], sentinel[n:])   # padding rows as they were
    for cache, old, x in ((step.k_pages.cpu(), before[0], k), (step.v_pages.cpu(), before[1], v)):
        left = torch.ones(cache.shape[0], cache.shape[2], dtype=torch.bool)
        for b, (r, m) in enumerate(step.sizes):
            pages, rows = step.slots(b, torch.arange(m - r, m))
            left[pages, rows] = False
            want = x[int(step.cu[b]):int(step.cu[b]) + r]
            assert ((cache[pages, :, rows].double() - want).abs() <= bound(want, want)).all()
        same = (cache.view(torch.int16) == old.view(torch.int16)).all(-1).all(1)
        assert same[left].all()   # every other slot as it was


def run(step, dtype, extra=0, **kw):
    y, parts = inputs(step, dtype, extra=extra)
    before = step.k_pages.clone(), step.v_pages.clone()
    yd = y.to(DEV)
    step.to(DEV)
    a, b = step.hq, step.hq + step.hkv
    sentinel = torch.full((step.rows, step.hq, step.d), 7.0, dtype=torch.bfloat16)
    out = sentinel.to(DEV)
    w = kw.get("weights", (None, None))
    got = b200q.k_kv_append(yd[:, :a], yd[:, a:b], yd[:, b:b + step.hkv], *step.args(),
                            inv_freq=None if kw.get("inv_freq") is None else kw["inv_freq"].to(DEV),
                            interleaved=kw.get("interleaved", False), eps=kw.get("eps", 1e-6),
                            q_norm=None if w[0] is None else w[0].to(DEV), k_norm=None if w[1] is None else w[1].to(DEV),
                            q_out=out)
    assert got is out
    check(step, parts, before, out, sentinel, **kw)
    assert b200q.device_error() == 0


SIZES = {"one token": [(1, 1)], "one row far": [(1, 70000)], "a prompt": [(257, 257)],
         "ragged": [(3, 40), (1, 1), (0, 17), (65, 129), (1, 64)]}


@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (128, 256)])
def test_plain(sizes, dtype, d, page):
    run(Step(SIZES[sizes], 4, 2, d, page, pad=2), dtype, extra=1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rope", [(64, 16), (64, 64), (128, 48), (128, 96), (128, 128)])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (5, 1), (7, 7)])
def test_rotation_and_norm(interleaved, d, rope, hq, hkv):
    f = (500000.0 ** (-torch.arange(rope // 2, dtype=torch.float64) / (rope // 2))).float()
    g = torch.Generator().manual_seed(4)
    w = (1 + 0.2 * torch.randn(d, generator=g), 1 + 0.2 * torch.randn(d, generator=g))
    run(Step(SIZES["ragged"], hq, hkv, d, 32, pad=1, interleave=True), torch.float32, inv_freq=f, interleaved=interleaved,
        weights=w)


@pytest.mark.parametrize("which", [(True, False), (False, True)])
def test_one_norm_in_bf16(which):
    w = tuple(torch.linspace(0.5, 1.5, 128).to(torch.bfloat16) if x else None for x in which)
    run(Step(SIZES["ragged"], 6, 3, 128, 16), torch.bfloat16, weights=w, eps=1e-2)


def test_far_positions_keep_their_angles():
    """at position 2^20 the fastest pair has turned 166,886 times"""
    f = torch.tensor([1.0, 0.37, 1e-3, 5e-6] * 8)
    run(Step([(2, 1 << 20), (3, 262144)], 2, 1, 64, 256), torch.float32, inv_freq=f)


def test_keys_and_values_alone_and_queries_in_place():
    step = Step([(5, 9)], 4, 2, 128, 16)
    y, (q, k, v) = inputs(step, torch.bfloat16)
    step.to(DEV)
    yd = y.to(DEV)
    f = torch.full((32,), 0.1)
    assert b200q.k_kv_append(None, yd[:, 4:6], yd[:, 6:8], *step.args(), inv_freq=f.to(DEV)) is None
    alone = step.k_pages.clone()
    want = b200q.k_kv_append(yd[:, :4], yd[:, 4:6], yd[:, 6:8], *step.args(), inv_freq=f.to(DEV))
    assert torch.equal(alone, step.k_pages)
    got = b200q.k_kv_append(yd[:, :4], yd[:, 4:6], yd[:, 6:8], *step.args(), inv_freq=f.to(DEV), q_out=yd[:, :4])
    assert torch.equal(got, want) and got.data_ptr() == yd.data_ptr()
    assert torch.equal(yd[:, 4:].cpu(), y[:, 4:])


def test_no_rows():
    step = Step([(0, 3)], 4, 2, 128, 16).to(DEV)
    e = torch.empty(0, 4, 128, device=DEV)
    assert b200q.k_kv_append(e, e[:, :2], e[:, :2], *step.args()).shape == (0, 4, 128)


@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_a_bad_table_entry_stores_nothing_and_is_reported(entry):
    step = Step([(3, 20), (2, 5)], 4, 2, 64, 16)
    y, (q, k, v) = inputs(step, torch.float32)
    step.table[0, 1] = entry     # positions 17..19 of sequence 0
    old = step.k_pages.clone()
    step.to(DEV)
    yd = y.to(DEV)
    got = b200q.k_kv_append(yd[:, :4], yd[:, 4:6], yd[:, 6:8], *step.args())
    assert b200q.device_error() == 1 << 16 and b200q.device_error() == 0
    assert torch.equal(got.cpu(), q.to(torch.bfloat16))
    pages, rows = step.slots(1, torch.arange(3, 5))
    now = step.k_pages.cpu()
    assert torch.equal(now[pages, :, rows], k[3:5].to(torch.bfloat16))
    now[pages, :, rows] = old[pages, :, rows]
    assert torch.equal(now, old)


def test_a_position_past_the_table_is_reported_and_a_negative_one_left_alone():
    step = Step([(2, 16), (4, 2)], 4, 2, 64, 16)   # sequence 1: two rows more than tokens
    y, _ = inputs(step, torch.float32)
    step.lens[0] = 18                                # rows at 16 and 17, the table holds 0 .. 15
    old = step.k_pages.clone()
    step.to(DEV)
    yd = y.to(DEV)
    out = torch.full((6, 4, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    b200q.k_kv_append(yd[:, :4], yd[:, 4:6], yd[:, 6:8], *step.args(), q_out=out)
    assert b200q.device_error() == 1 << 16
    assert (out[2:4] == 7).all() and torch.equal(out[4:].cpu(), y[4:, :4].to(torch.bfloat16))
    pages, rows = step.slots(1, torch.arange(2))
    now = step.k_pages.cpu()
    now[pages, :, rows] = old[pages, :, rows]
    assert torch.equal(now, old)


def test_captured_and_replayed_with_new_lengths():
    """a decode step as a graph: the kernels read lens and the table when they run"""
    step = Step([(1, 30), (1, 1)], 4, 2, 128, 16).to(DEV)
    y, _ = inputs(step, torch.float32)
    yd = y.to(DEV)
    call = lambda: b200q.k_kv_append(yd[:, :4], yd[:, 4:6], yd[:, 6:8], *step.args())
    call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
        out = call()
    for a, b in ((17, 5), (31, 16)):
        step.k_pages.zero_()
        step.lens.copy_(torch.tensor([a, b]))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), y[:, :4].to(torch.bfloat16))
        for s, n in ((0, a), (1, b)):
            pages, rows = step.slots(s, torch.tensor([n - 1]))
            assert torch.equal(step.k_pages.cpu()[pages, :, rows], y[s:s + 1, 4:6].to(torch.bfloat16))
        assert int((step.k_pages != 0).any(-1).sum()) == 4
