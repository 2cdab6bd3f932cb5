"""The paged operators together, as a block of a model uses them: Q8_0 q/k/v projection, k_kv_append, attn_prompt for the
prompt and attn_decode for verify windows and single tokens (captured once and replayed over growing lengths), Q8_0 output
projection.

Each stage is checked on what the stage before gave it.  The projections: fp32 sums of exact fp16 products for up to 16 rows
of bf16 (relative L2 1e-5, as their own tests); the prompt's weights and rows are rounded to fp16 (2^-11 each): 1e-3.  The
cache and the queries: bf16 of fp32, 2^-8 of the value and 2^-17 of the head's largest.  The attention: as its own tests."""
import numpy as np
import pytest
import torch

import b200q
import oracle as O
from helpers import rel_l2
from paged import Step, attend, norm, rotate

pytestmark = pytest.mark.gpu
DEV = "cuda"
HQ, HKV, D, PAGE, H = 8, 2, 64, 16, 512
N = (HQ + 2 * HKV) * D


def q8_blocks(seed, n, k):
    rng = np.random.default_rng(seed)
    qv = rng.integers(-127, 128, (n, k // 32, 32), dtype=np.int8)
    d = rng.uniform(2e-4, 1e-3, (n, k // 32)).astype(np.float16)
    return np.concatenate([d.view(np.uint8).reshape(n, k // 32, 2), qv.view(np.uint8)], -1).reshape(n, -1)


class Block:
    def __init__(self):
        self.qkv_raw, self.o_raw = q8_blocks(1, N, H), q8_blocks(2, H, HQ * D)
        up = [torch.from_numpy(x).to(DEV) for x in (self.qkv_raw, self.o_raw)]
        self.qkv, self.o = b200q.tile_q8(up[0], N, H), b200q.tile_q8(up[1], H, HQ * D)
        self.qkv_tc, self.o_tc = b200q.tile_q8_tc(up[0], N, H), b200q.tile_q8_tc(up[1], H, HQ * D)
        g = torch.Generator().manual_seed(3)
        self.norms = [1 + 0.1 * torch.randn(D, generator=g) for _ in range(2)]
        self.inv = 10000.0 ** (-torch.arange(16).double() / 16)
        self.inv = self.inv.float()
        self.dev = [x.to(DEV) for x in (*self.norms, self.inv)]

    def __call__(self, x, step, most):
        """the block on a step's rows x [rows][H] bf16 -> y [rows][H] fp32 and what lay between"""
        few = x.shape[0] <= 16
        y = b200q.mma_q8(self.qkv, N, H, x) if few else b200q.mma_q8_prompt(self.qkv_tc, N, H, x)
        h = y.view(-1, HQ + 2 * HKV, D)
        q = b200q.k_kv_append(h[:, :HQ], h[:, HQ:HQ + HKV], h[:, HQ + HKV:], *step.args(), inv_freq=self.dev[2],
                              q_norm=self.dev[0], k_norm=self.dev[1])
        a = (b200q.attn_decode if most <= 16 else b200q.attn_prompt)(q, *step.args(), most)
        z = a.view(-1, HQ * D)
        return (b200q.mma_q8(self.o, H, HQ * D, z) if few else b200q.mma_q8_prompt(self.o_tc, H, HQ * D, z)), y, q, a

    def check(self, x, step, got):
        out, y, q, a = (t.cpu() for t in got)
        loose = 1e-5 if x.shape[0] <= 16 else 1e-3
        assert rel_l2(y.numpy(), O.q8_gemm_exact(self.qkv_raw, N, H, x.cpu().float().numpy())) < loose
        h = y.double().view(-1, HQ + 2 * HKV, D)
        pos = torch.cat([torch.arange(n - r, n) for r, n in step.sizes])
        parts = [rotate(norm(h[:, i:j], w, 1e-6), pos, self.inv, False)
                 for (i, j), w in zip(((0, HQ), (HQ, HQ + HKV)), self.norms)] + [h[:, HQ + HKV:]]
        close = lambda g, w: ((g.double() - w).abs() <= 2.0 ** -8 * w.abs() + 2.0 ** -17 * w.abs().amax(-1, keepdim=True)).all()
        assert close(q, parts[0])
        k, v = step.k_pages.cpu(), step.v_pages.cpu()
        for b, (r, n) in enumerate(step.sizes):
            pages, rows = step.slots(b, torch.arange(n - r, n))
            at = slice(int(step.cu[b]), int(step.cu[b]) + r)
            assert close(k[pages, :, rows], parts[1][at]) and close(v[pages, :, rows], parts[2][at])
        want = attend(step, q)
        pool = step.v_pages
        step.v_pages = step.v_pages.abs()
        bar = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -10 + 1000 * 2.0 ** -24) * attend(step, q)
        step.v_pages = pool
        assert ((a.double() - want).abs() <= bar).all()
        assert rel_l2(out.numpy(), O.q8_gemm_exact(self.o_raw, H, HQ * D, a.float().view(-1, HQ * D).numpy())) < loose


def resize(step, sizes):
    """the step's sequences at other sizes of the same rows"""
    step.sizes = sizes
    step.lens.copy_(torch.tensor([n for _, n in sizes], dtype=torch.int32))


def test_prompt_verify_and_single_tokens():
    block = Block()
    g = torch.Generator().manual_seed(5)
    rows = lambda n: torch.randn(n, H, generator=g).to(torch.bfloat16).to(DEV)
    ends = [150, 37, 400]
    whole = Step([(n, n) for n in ends], HQ, HKV, D, PAGE)   # the prompts; pages for 40 tokens more a sequence
    more = Step([(0, n + 40) for n in ends], HQ, HKV, D, PAGE)
    for t in ("table", "k_pages", "v_pages", "width"):
        setattr(whole, t, getattr(more, t))
    whole.to(DEV)
    x = rows(sum(ends))
    block.check(x, whole, block(x, whole, max(ends)))

    def follow(r):   # a step of r rows a sequence over the same cache
        s = Step([(r, r)] * 3, HQ, HKV, D, PAGE).to(DEV)
        for t in ("table", "k_pages", "v_pages", "width"):
            setattr(s, t, getattr(whole, t))
        resize(s, [(r, n + r) for n in ends])
        return s

    s = follow(5)   # a verify window of 5, of which 2 are kept
    x = rows(15)
    block.check(x, s, block(x, s, 5))
    ends = [n + 2 for n in ends]

    s, x = follow(1), rows(3)   # single tokens: one captured block, replayed
    block(x, s, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = block(x, s, 1)
    for i in range(20):
        resize(s, [(1, n + 1 + i) for n in ends])
        x.copy_(rows(3))
        graph.replay()
        torch.cuda.synchronize()
        if i % 6 == 0:
            block.check(x, s, got)
    assert b200q.device_error() == 0
