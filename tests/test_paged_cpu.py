"""CPU tests of the paged attention operators: every refusal comes before a launch (the addresses below are never read),
and the fp64 definitions the GPU tests use are themselves checked."""
import math

import pytest
import torch

import b200q
from paged import Step, attend, rotate

A = 0x100000   # aligned addresses that nothing reads


CACHE = dict(kp=A, vp=A, ks=2 * 16 * 128, vs=2 * 16 * 128, table=A, lens=A, cu=A, ldt=4, pages=8, page=16, hkv=2, d=128, width=4,
             batch=2)
APPEND = dict(q=A, k=A, v=A, x_dtype=0, ldq=512, ldk=256, ldv=256, rows=4, hq=4, inv=A, rope=64, inter=0, qn=0, kn=0, nd=0,
              eps=1e-6, qo=A, ldo=512, stream=0)
ATTN = dict(q=A, ldq=512, rows=4, hq=4, max_rows=4, scale=0.1, softcap=0.0, window=0, out=A, ldo=512, ws=A, wsb=1 << 40, stream=0)


def call(name, base, kw):
    """the C entry point with a good call's arguments but for those in kw"""
    assert set(kw) <= set(CACHE) | set(base)
    kv = b200q._PAGED.pack(*(kw.get(n, x) for n, x in CACHE.items()))
    return getattr(b200q.lib(), name)(kv, *(kw.get(n, x) for n, x in base.items()))


def append(**kw):
    return call("b200q_kv_append", APPEND, kw)


CACHE_REFUSALS = [dict(kp=0), dict(vp=0), dict(kp=A + 8), dict(ks=2 * 16 * 128 - 8), dict(vs=2 * 16 * 128 + 4), dict(ks=1 << 39),
                  dict(pages=0), dict(page=8), dict(page=48), dict(page=512), dict(d=96), dict(hkv=0), dict(hkv=-2), dict(table=0),
                  dict(width=5), dict(width=0), dict(lens=0), dict(cu=0), dict(cu=A + 2), dict(batch=0), dict(batch=4097),
                  dict(width=1 << 27, ldt=1 << 27)]


@pytest.mark.parametrize("kw", CACHE_REFUSALS + [
    dict(k=0), dict(v=0), dict(q=0), dict(qo=0), dict(q=A + 4), dict(x_dtype=2), dict(ldq=511), dict(ldq=508), dict(ldk=128),
    dict(ldv=130), dict(ldo=504), dict(rope=8), dict(rope=144), dict(rope=-16), dict(inv=0), dict(rows=-1), dict(hq=-1),
    dict(hq=5000), dict(qn=A, nd=3), dict(qn=A + 8), dict(kn=A, eps=-1.0), dict(kn=A, eps=float("nan"))])
def test_append_refuses(kw):
    assert append(**kw) == b200q.EINVAL


def test_append_of_no_rows_is_nothing():
    assert append(rows=0) == b200q.OK
    assert b200q.lib().b200q_kv_append(None, *APPEND.values()) == b200q.EINVAL


@pytest.mark.parametrize("f", ["b200q_attn_decode", "b200q_attn_prompt"])
@pytest.mark.parametrize("kw", CACHE_REFUSALS + [
    dict(q=0), dict(out=0), dict(q=A + 8), dict(out=A + 4), dict(ldq=504), dict(ldo=516), dict(rows=-1), dict(hq=0), dict(hq=5),
    dict(max_rows=0), dict(max_rows=1 << 30), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=float("nan")), dict(window=-1), dict(ws=0), dict(ws=A + 8)])
def test_attention_refuses(f, kw):
    assert call(f, ATTN, kw) == b200q.EINVAL


@pytest.mark.parametrize("f", ["b200q_attn_decode", "b200q_attn_prompt"])
@pytest.mark.parametrize("kw", [dict(softcap=1e-45), dict(softcap=2e38), dict(softcap=float("inf"))])
def test_caps_out_of_range_are_refused(f, kw):
    assert call(f, ATTN, kw) == b200q.EINVAL


def test_workspace_follows_the_rows_a_kv_head():
    """up to 8 and 16 rows a kv head, up to a tile of 128, more"""
    w = b200q.lib().b200q_attn_decode_workspace_bytes
    sizes = [w(8, 1, 128, 1), w(16, 1, 128, 1), w(17, 1, 128, 1), w(8, 1, 128, 16), w(9, 1, 128, 16), w(512, 1, 128, 16)]
    assert sizes[0] < sizes[1] < sizes[2] == sizes[3] < sizes[4] == sizes[5]
    p = b200q.lib().b200q_attn_prompt_workspace_bytes
    assert p(8, 1, 128, 16, 16, 1) == sizes[3] and p(8, 1, 128, 17, 17, 1) == sizes[4]
    for f, rows in (("b200q_attn_decode", 16), ("b200q_attn_prompt", 100)):   # one byte short
        need = w(4, 2, 128, rows) if "decode" in f else p(4, 2, 128, rows, rows, 2)
        assert call(f, ATTN, dict(max_rows=rows, wsb=need - 1)) == b200q.ENOSPACE


def test_attention_of_no_rows_too_many_and_too_little_workspace():
    L = b200q.lib()
    for f in ("b200q_attn_decode", "b200q_attn_prompt"):
        assert call(f, ATTN, dict(rows=0)) == b200q.OK
        assert call(f, ATTN, dict(wsb=0)) == b200q.ENOSPACE
    assert call("b200q_attn_decode", ATTN, dict(max_rows=17)) == b200q.EINVAL
    assert L.b200q_attn_decode_workspace_bytes(4, 2, 128, 17) == 0
    assert 0 < L.b200q_attn_decode_workspace_bytes(32, 8, 128, 1) <= 8 << 20
    assert 0 < L.b200q_attn_prompt_workspace_bytes(32, 8, 128, 77, 77, 1) <= 64 << 20


def test_host_tensors_are_refused():
    step = Step([(1, 3)], 4, 2, 64, 16)
    x = torch.zeros(1, 4, 64)
    with pytest.raises(b200q.B200QError, match="CUDA tensor"):
        b200q.k_kv_append(x, x[:, :2], x[:, :2], *step.args())
    for f in (b200q.attn_decode, b200q.attn_prompt):
        with pytest.raises(b200q.B200QError, match="CUDA tensor"):
            f(x.bfloat16(), *step.args(), 1)


def test_the_rotation_is_a_complex_product():
    x = torch.randn(3, 2, 64, dtype=torch.float64)
    f, pos = torch.rand(16), torch.tensor([0, 5, 900])
    z = torch.polar(torch.ones(()).double(), pos[:, None, None] * f.double())
    y = rotate(x, pos, f, True)
    want = torch.view_as_real(torch.view_as_complex(x[..., :32].unflatten(-1, (16, 2))) * z).flatten(-2)
    assert torch.allclose(y[..., :32], want, atol=1e-12) and torch.equal(y[..., 32:], x[..., 32:])
    y = rotate(x, pos, f, False)
    w = torch.complex(x[..., :16], x[..., 16:32]) * z
    assert torch.allclose(y[..., :32], torch.cat((w.real, w.imag), -1), atol=1e-12)


def test_the_attention_definition_is_a_masked_softmax():
    step = Step([(3, 37), (2, 2), (1, 0), (4, 3)], 4, 2, 64, 16, pad=1)
    q = torch.randn(step.rows, 4, 64, dtype=torch.float64)
    got = attend(step, q)
    pages, rows = step.slots(0, torch.arange(37))
    k, v = step.k_pages[pages, 1, rows].double(), step.v_pages[pages, 1, rows].double()
    for i in range(3):   # row i sees keys 0 .. 34 + i
        want = torch.softmax(q[i, 3] @ k[:35 + i].T / 8, -1) @ v[:35 + i]
        assert torch.allclose(got[i, 3], want, atol=1e-12)
    one = attend(step, q, window=1)   # each row sees its own key alone
    assert torch.allclose(one[2, 2], v[36], atol=1e-12)
    assert (got[5] == 0).all()       # a sequence without keys
    assert (got[6] == 0).all() and (got[7] != 0).any()   # four rows, three tokens: the first has no place
    assert (got[10:] == 0).all()     # padding
    hot = attend(step, 100 * q, softcap=2.0)
    x = 2 * torch.tanh(100 * q[0, 3] @ k[:35].T / 8 / 2)
    assert torch.allclose(hot[0, 3], torch.softmax(x, -1) @ v[:35], atol=1e-12) and math.isfinite(float(hot.sum()))
