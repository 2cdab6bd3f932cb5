"""Paged-cache inputs and the fp64 definitions of the paged attention operators, shared by their tests.

A step: sequence b has sizes[b] = (rows, cached tokens), the step's rows included; its row i of r stands at position
n - r + i.  Everything is made on the CPU from a seed; `Step.to` moves it."""
import math

import torch


class Step:
    """A ragged step over a paged cache of [pages][hkv][page][d] bf16, pages handed out in a random order."""

    def __init__(self, sizes, hq, hkv, d, page, seed=0, pad=0, spare=3, junk=None, interleave=False, device="cpu"):
        g = torch.Generator().manual_seed(seed)
        self.sizes, self.hq, self.hkv, self.d, self.page, self.pad, self.device = sizes, hq, hkv, d, page, pad, device
        need = [-(-max(n, 0) // page) for _, n in sizes]
        self.width, total = max(1, max(need)), sum(need)
        pages = total + spare
        perm = torch.randperm(pages, generator=g)[:total].to(torch.int32)
        self.table = torch.full((len(sizes), self.width), -1, dtype=torch.int32)
        at = 0
        for b, w in enumerate(need):
            self.table[b, :w] = perm[at:at + w]
            at += w
        self.cu = torch.tensor([0] + [r for r, _ in sizes], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        self.lens = torch.tensor([n for _, n in sizes], dtype=torch.int32)
        self.rows = int(self.cu[-1]) + pad
        self.most = max(1, max(r for r, _ in sizes))
        # interleave: keys and values in one pool, a page of keys beside its page of values
        pool = torch.randn(pages, 2, hkv, page, d, generator=g).to(torch.bfloat16)
        if junk is not None:   # what no token of a sequence sits in
            used = torch.zeros(pages, page, dtype=torch.bool)
            for b, (_, n) in enumerate(sizes):
                for p in range(0, n, page):
                    used[int(self.table[b, p // page]), :min(page, n - p)] = True
            pool = torch.where(used[:, None, None, :, None], pool, torch.tensor(junk, dtype=torch.bfloat16))
        self.pool = pool
        self.k_pages, self.v_pages = pool[:, 0], pool[:, 1]
        if not interleave:
            self.k_pages, self.v_pages = self.k_pages.contiguous(), self.v_pages.contiguous()
        self.gen = g

    def to(self, device):
        """the tensors on `device`, strides kept"""
        for name in ("table", "cu", "lens"):
            setattr(self, name, getattr(self, name).to(device))
        if self.k_pages.is_contiguous():
            self.k_pages, self.v_pages = self.k_pages.to(device), self.v_pages.to(device)
        else:
            self.pool = self.pool.to(device)
            self.k_pages, self.v_pages = self.pool[:, 0], self.pool[:, 1]
        self.device = device
        return self

    def args(self):
        return self.k_pages, self.v_pages, self.table, self.lens, self.cu

    def slots(self, b, positions):
        """(page, row) of sequence b's positions"""
        p = torch.as_tensor(positions)
        return self.table[b].cpu().long()[p // self.page], p % self.page


def rotate(x, pos, inv_freq, interleaved):
    """x [rows][heads][d] fp64, pos [rows]: the first 2 * len(inv_freq) values of each head turned by pos * inv_freq"""
    h = inv_freq.numel()
    t = pos.double()[:, None, None] * inv_freq.double()
    c, s = t.cos(), t.sin()
    y = x.clone()
    i = torch.arange(h)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + h)
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    return y


def norm(x, w, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


def attend(step, q, scale=None, softcap=0.0, window=0):
    """fp64 attention of the step's rows over its cache (CPU): [rows][hq][d]; padding rows and rows that see no key: 0"""
    s, d = step, step.d
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(s.rows, s.hq, d, dtype=torch.float64)
    group = s.hq // s.hkv
    kp, vp, q = s.k_pages.cpu(), s.v_pages.cpu(), q.cpu().double()
    for b, (r, n) in enumerate(s.sizes):
        at = int(s.cu[b])
        if r == 0 or n <= 0:
            continue
        pages, rows = s.slots(b, torch.arange(n))
        pos = torch.arange(n - r, n)[:, None]
        j = torch.arange(n)[None]
        see = j <= pos
        if window:
            see = see & (j > pos - window)
        for h in range(s.hkv):
            k, v = kp[pages, h, rows].double(), vp[pages, h, rows].double()
            for e in range(h * group, (h + 1) * group):
                x = q[at:at + r, e] @ k.T * scale
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                x = x.masked_fill(~see, -math.inf)
                top = x.amax(-1, keepdim=True)
                p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total == 0, 1.0, total)
                # a key that no row of the sequence sees has no part in any sum, whatever its value holds
                p, u = p[:, see.any(0)], v[see.any(0)]
                out[at:at + r, e] = p @ u
    return out
