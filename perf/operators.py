"""What the paged attention operators are measured on: appending a step's keys and values to a paged cache (with the
per-head norm and the position rotation on the way), attention of a decode or verify step over that cache, and
attention of prompt chunks over it.

`run` computes an operator in elementary torch operations (fp32, angles in fp64, rounded once at the end), or, where
`own` is true, by the framework's calls.  `exact` restates the definitions in fp64.

All three share one description of a step: `cu` [B + 1] the row ranges of the sequences in the step's ragged rows,
`lens` [B] the cached tokens of each sequence with the step's own, `table` [B][W] its pages.  Row i of a sequence with
r rows stands at position lens - r + i; rows from cu[B] on are padding and stay as they are.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "nemotron-3.5-bolt-tensorfold-dgx-spark_b200")


def _case(name, op, batch, rows, length, ragged, hq, hkv, d, page, mix, softcap=0.0, window=0, dtype="bf16", rope=0,
          interleaved=False, norm=False, pad=0):
    """rows: the most rows of a sequence in the step; length: the most cached tokens; ragged: sequences of differing
    rows and lengths; pad: padding rows behind the last sequence; mix: which ragged lengths"""
    c = dict(name=name, op=op, batch=batch, rows=rows, length=length, ragged=ragged, hq=hq, hkv=hkv, d=d, page=page,
             mix=mix)
    if op == "append":
        c.update(dtype=dtype, rope=rope, interleaved=interleaved, norm=norm, pad=pad)
    else:
        c.update(softcap=softcap, window=window)
    return c


def listed():
    return [
        # one decode step of one sequence, q/k/v as the Q8_0 projection's fp32 rows: latency
        _case("append one token", "append", 1, 1, 700, False, 32, 8, 128, 64, 1, dtype="f32", rope=128),
        # several prompts at once, odd lengths, small heads without sharing, pairs rotated side by side, padded rows
        _case("append ragged prompts", "append", 7, 1501, 2500, True, 24, 24, 64, 32, 2, dtype="bf16", rope=64,
              interleaved=True, pad=37),
        # a whole prompt of the GQA projections' benchmark length, heads normed, half of each rotated
        _case("append 8192 tokens", "append", 1, 8192, 8192, False, 32, 8, 128, 128, 3, dtype="f32", rope=64, norm=True),
        # one decode step of one short chat: latency
        _case("decode one short", "decode", 1, 1, 1000, False, 32, 8, 128, 64, 4),
        # a serving batch of 16
        _case("decode 16 ragged", "decode", 16, 1, 4096, True, 32, 8, 128, 64, 5),
        # a serving batch of 64 with long contexts: the most keys and values together
        _case("decode 64 ragged", "decode", 64, 1, 6000, True, 32, 8, 128, 32, 6),
        # one sequence at the model's longest context: the cache's length is the only axis to split
        _case("decode 262144", "decode", 1, 1, 262144, False, 32, 8, 128, 128, 7),
        # verify windows of a drafter, small heads shared by 7, capped scores and a sliding window, small pages
        _case("verify window", "decode", 8, 16, 16384, True, 28, 4, 64, 16, 8, softcap=30.0, window=6000),
        # a short question
        _case("prompt 77", "prompt", 1, 77, 77, False, 32, 8, 128, 64, 9),
        # several prompts with small unshared heads, capped scores and a sliding window
        _case("prompt ragged", "prompt", 6, 1500, 1999, True, 12, 12, 64, 32, 10, softcap=50.0, window=700),
        # a chunk of a prompt behind a long cached prefix: few rows, many keys
        _case("prompt chunk", "prompt", 1, 512, 32768, False, 32, 8, 128, 128, 11),
        # a whole prompt of the GQA projections' benchmark length
        _case("prompt 8192", "prompt", 1, 8192, 8192, False, 32, 8, 128, 128, 12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt"])
    d = rng.choice([64, 128])
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    mix = rng.randrange(1 << 20)
    ragged = rng.random() < 0.7
    softcap = rng.choice([0.0, 0.0, 20.0, 50.0])
    if op == "append":
        rows = _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(128, 8192 // rows)))
        length = rows + _log(rng, 1, 8192)
        c = _case("", op, batch, rows, length, ragged, hkv * group, hkv, d, page, mix, dtype=rng.choice(["f32", "bf16"]),
                  rope=rng.choice([0, d // 2, d]), interleaved=rng.random() < 0.5, norm=rng.random() < 0.5,
                  pad=rng.choice([0, 5]))
    elif op == "decode":
        rows = rng.choice([1, 1, 1, rng.randint(2, 16)])
        length = rows + _log(rng, 1, 262144)
        batch = _log(rng, 1, max(1, min(64, 262144 * 8 * 128 // (length * hkv * d))))
        c = _case("", op, batch, rows, length, ragged, hkv * group, hkv, d, page, mix, softcap=softcap,
                  window=rng.choice([0, 0, _log(rng, 1, length + 1)]))
    else:
        rows = _log(rng, 1, min(8192, int(8192 * math.sqrt(32 / (hkv * group)))))
        most = 16 * 8192 * 8192 // (rows * hkv * group)
        length = rows + _log(rng, 1, max(1, min(32768, most - rows)))
        batch = _log(rng, 1, max(1, min(16, most // length)))
        c = _case("", op, batch, rows, length, ragged, hkv * group, hkv, d, page, mix, softcap=softcap,
                  window=rng.choice([0, 0, _log(rng, 1, length + 1)]))
    del c["name"]
    return c


def _sizes(case):
    """(rows, cached tokens) of every sequence: plain numbers that the case alone decides"""
    rng = random.Random(case["mix"])
    got = []
    for i in range(case["batch"]):
        r, n = case["rows"], case["length"]
        if case["ragged"] and i:
            r = rng.randint(max(1, r // 4), r)
            n = max(r, rng.randint(max(1, n // 4), n))
        got.append((r, n))
    return got


def work(case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    sizes = _sizes(case)
    rows = sum(r for r, _ in sizes)
    pages = sum(-(-n // case["page"]) for _, n in sizes)
    small = 4 * (3 * len(sizes) + 1)
    if case["op"] == "append":
        e = 4 if case["dtype"] == "f32" else 2
        # q, k, v in; q, k, v out in bf16; the rotation and the norms are a few operations a value
        return {"bytes": rows * (hq + 2 * hkv) * d * (e + 2) + small, "flops": rows * (hq + hkv) * d * 6}
    w = case["window"] or 1 << 60
    seen = keys = 0
    for r, n in sizes:
        first, last = n - r, n - 1
        keys += n - max(0, first - w + 1)
        full = min(max(first, w - 1), last + 1)   # rows from here on see w keys
        seen += (full - first) * (first + 1 + full) // 2 + (last + 1 - full) * w
    return {"bytes": keys * hkv * d * 4 + 2 * rows * hq * d * 2 + 4 * pages + small, "flops": 4 * seen * hq * d}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    sizes = _sizes(case)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    need = [-(-n // page) for _, n in sizes]
    width, total = max(need), sum(need)
    pages = total + 3                                       # a pool that is not quite full
    perm = torch.randperm(pages, generator=g, device=DEV)[:total].to(torch.int32)
    at = torch.arange(width, device=DEV)[None] < torch.tensor(need, device=DEV)[:, None]
    table = torch.full((len(sizes), width), -1, dtype=torch.int32, device=DEV)
    table[at] = perm
    cu = torch.tensor([0] + [r for r, _ in sizes], dtype=torch.int32, device=DEV).cumsum(0, dtype=torch.int32)
    lens = torch.tensor([n for _, n in sizes], dtype=torch.int32, device=DEV)
    n = sum(r for r, _ in sizes)
    s = dict(case=case, table=table, cu=cu, lens=lens, total=n, most=max(r for r, _ in sizes))
    shape = (pages, hkv, page, d)
    if case["op"] == "append":
        # one row holds q, k and v of a token side by side, as the fused projection leaves them
        dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        qkv = torch.randn(n + case["pad"], (hq + 2 * hkv) * d, generator=g, device=DEV).to(dt)
        s["q"], s["k"], s["v"] = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
        s["k_pages"] = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        s["v_pages"] = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        s["q_out"] = torch.zeros(n + case["pad"], hq, d, dtype=torch.bfloat16, device=DEV)
        half = case["rope"] // 2
        s["inv_freq"] = (500000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / max(half, 1))).float() if half else None
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device=DEV)
            s["k_norm"] = 1 + 0.1 * torch.randn(d, generator=g, device=DEV)
    else:
        s["k_pages"] = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
        s["v_pages"] = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
        s["q"] = (1.5 * torch.randn(n, hq, d, generator=g, device=DEV)).bfloat16()
    return s


EPS = 1e-5


def run(s):
    case = s["case"]
    if own:
        if PKG not in sys.path:
            sys.path.insert(0, PKG)
        import b200q
        if case["op"] == "append":
            q = b200q.k_kv_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"],
                                  inv_freq=s["inv_freq"], interleaved=case["interleaved"], q_norm=s["q_norm"],
                                  k_norm=s["k_norm"], eps=EPS, q_out=s["q_out"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        f = b200q.attn_decode if case["op"] == "decode" else b200q.attn_prompt
        return f(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["cu"], s["most"],
                 softcap=case["softcap"], window=case["window"])
    return _append(s) if case["op"] == "append" else _attend(s)


# ---------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------
def _rows(s):
    """sequence and position of every row that belongs to one"""
    t = torch.arange(s["total"], device=DEV)
    cu = s["cu"].long()
    b = torch.searchsorted(cu, t, right=True) - 1
    return b, s["lens"].long()[b] - cu[b + 1] + t


def _append(s):
    case = s["case"]
    b, pos = _rows(s)
    q, k, v = (s[x][:s["total"]].float() for x in "qkv")
    if case["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    rope = case["rope"]
    if rope:
        angle = pos[:, None].double() * s["inv_freq"].double()
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

        def turn(x):
            y = x[..., :rope]
            if case["interleaved"]:
                a, c = y[..., 0::2], y[..., 1::2]
                y = torch.stack((a * cos - c * sin, c * cos + a * sin), -1).flatten(-2)
            else:
                a, c = y[..., :rope // 2], y[..., rope // 2:]
                y = torch.cat((a * cos - c * sin, c * cos + a * sin), -1)
            return torch.cat((y, x[..., rope:]), -1)

        q, k = turn(q), turn(k)
    page = case["page"]
    at = s["table"].long()[b, pos // page]
    s["q_out"][:s["total"]] = q.bfloat16()
    s["k_pages"][at, :, pos % page] = k.bfloat16()
    s["v_pages"][at, :, pos % page] = v.bfloat16()
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    group, batch, most = hq // hkv, case["batch"], s["most"]
    b, pos = _rows(s)
    i = torch.arange(s["total"], device=DEV) - s["cu"].long()[b]
    q = torch.zeros(batch, most, hkv, group, d, device=DEV)
    q[b, i] = s["q"].float().view(-1, hkv, group, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * most, d)
    at = s["table"].long().clamp(min=0)
    k = s["k_pages"][at].transpose(1, 2).float().reshape(batch, hkv, -1, d)      # [B][heads][keys][d]
    v = s["v_pages"][at].transpose(1, 2).float().reshape(batch, hkv, -1, d)
    x = torch.matmul(q, k.transpose(2, 3)) * (1 / math.sqrt(d))
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    x = x.view(batch, hkv, group, most, -1)
    place = torch.full((batch, most), -1, device=DEV)
    place[b, i] = pos
    j = torch.arange(x.shape[-1], device=DEV)
    see = j <= place[..., None]
    if case["window"]:
        see &= j > place[..., None] - case["window"]
    x = x.masked_fill(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(batch, hkv, group * most, -1), v).view(batch, hkv, group, most, d)
    y = y / torch.where(total == 0, 1.0, total)
    return y.permute(0, 3, 1, 2, 4)[b, i].reshape(-1, hq, d).bfloat16()


# ---------------------------------------------------------------------------------------------------------------
# the definitions in fp64, sequence by sequence
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    sizes, page, d = _sizes(case), case["page"], case["d"]
    at = [0]
    for r, _ in sizes:
        at.append(at[-1] + r)
    if case["op"] == "append":
        qo = s["q_out"].double()
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        for b, (r, n) in enumerate(sizes):
            pos = torch.arange(n - r, n, device=DEV)
            slot = s["table"][b].long()[torch.div(pos, page, rounding_mode="floor")] * page + pos % page
            for name, weight in (("q", "q_norm"), ("k", "k_norm"), ("v", None)):
                x = s[name][at[b]:at[b + 1]].double()
                if weight and case["norm"]:
                    x = x / ((x * x).sum(-1, keepdim=True) / d + EPS).sqrt() * s[weight].double()
                if weight and case["rope"]:
                    half = case["rope"] // 2
                    # the pairs as complex numbers, turned by e^(i pos f)
                    z = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos[:, None] * s["inv_freq"].double()[None])[:, None]
                    if case["interleaved"]:
                        x[..., :case["rope"]] = torch.view_as_real(torch.view_as_complex(x[..., :case["rope"]].unflatten(-1, (half, 2)).contiguous()) * z).flatten(-2)
                    else:
                        y = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * z
                        x[..., :half], x[..., half:2 * half] = y.real, y.imag
                if name == "q":
                    qo[at[b]:at[b + 1]] = x
                else:
                    into = kp if name == "k" else vp
                    for h in range(case["hkv"]):
                        into[slot // page, h, slot % page] = x[:, h]
        return {"q": qo, "k_pages": kp, "v_pages": vp}
    group = case["hq"] // case["hkv"]
    out = torch.zeros(s["total"], case["hq"], d, dtype=torch.float64, device=DEV)
    for b, (r, n) in enumerate(sizes):
        used = s["table"][b, :-(-n // page)].long()
        for h in range(case["hkv"]):
            k = s["k_pages"][used, h].reshape(-1, d)[:n].double()
            v = s["v_pages"][used, h].reshape(-1, d)[:n].double()
            for lo in range(0, r, 1024):
                hi = min(lo + 1024, r)
                pos = torch.arange(n - r + lo, n - r + hi, device=DEV)[:, None]
                key = torch.arange(n, device=DEV)[None]
                hidden = key > pos
                if case["window"]:
                    hidden |= key <= pos - case["window"]
                for e in range(h * group, (h + 1) * group):
                    x = (s["q"][at[b] + lo:at[b] + hi, e].double() @ k.T) / d ** 0.5
                    if case["softcap"]:
                        x = (x / case["softcap"]).tanh() * case["softcap"]
                    x = x.masked_fill(hidden, float("-inf"))
                    out[at[b] + lo:at[b] + hi, e] = torch.softmax(x, -1) @ v
    return out
