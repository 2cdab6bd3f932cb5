"""CPU tests of the paged attention operators: every refusal comes before a launch (the addresses below are never read),
and the fp64 definitions the GPU tests use are themselves checked."""
import ctypes
import math

import pytest
import torch

import b200q
from paged import Step, attend, rotate

vp = ctypes.c_void_p
A = 0x100000   # aligned addresses that nothing reads


def append_args(**kw):
    a = dict(q=vp(A), k=vp(A), v=vp(A), x_dtype=0, ldq=512, ldk=256, ldv=256, rows=4, hq=4, hkv=2, d=128, kp=vp(A), vp_=vp(A),
             ks=2 * 16 * 128, vs=2 * 16 * 128, pages=8, page=16, table=vp(A), ldt=4, width=4, lens=vp(A), cu=vp(A), batch=2,
             inv=vp(A), rope=64, inter=0, qn=None, kn=None, nd=0, eps=1e-6, qo=vp(A), ldo=512, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


CACHE_REFUSALS = [dict(kp=None), dict(vp_=None), dict(kp=vp(A + 8)), dict(ks=2 * 16 * 128 - 8), dict(vs=2 * 16 * 128 + 4),
                  dict(pages=0), dict(page=8), dict(page=48), dict(page=512), dict(d=96), dict(hkv=0), dict(table=None),
                  dict(width=5), dict(width=0), dict(lens=None), dict(cu=None), dict(cu=vp(A + 2)), dict(batch=0),
                  dict(batch=4097), dict(width=1 << 27, ldt=1 << 27)]


@pytest.mark.parametrize("kw", CACHE_REFUSALS + [
    dict(k=None), dict(v=None), dict(q=None), dict(qo=None), dict(q=vp(A + 4)), dict(x_dtype=2), dict(ldq=511), dict(ldq=508),
    dict(ldk=128), dict(ldv=130), dict(ldo=504), dict(rope=8), dict(rope=144), dict(rope=-16), dict(inv=None), dict(rows=-1),
    dict(hq=-1), dict(hq=5000), dict(qn=vp(A), nd=3), dict(qn=vp(A + 8)), dict(kn=vp(A), eps=-1.0),
    dict(kn=vp(A), eps=float("nan"))])
def test_append_refuses(kw):
    assert b200q.lib().b200q_kv_append(*append_args(**kw)) == b200q.EINVAL


def test_append_of_no_rows_is_nothing():
    assert b200q.lib().b200q_kv_append(*append_args(rows=0)) == b200q.OK


def attn_args(**kw):
    a = dict(q=vp(A), ldq=512, rows=4, hq=4, kp=vp(A), vp_=vp(A), ks=2 * 16 * 128, vs=2 * 16 * 128, pages=8, page=16, hkv=2, d=128,
             table=vp(A), ldt=4, width=4, lens=vp(A), cu=vp(A), batch=2, max_rows=4, scale=0.1, softcap=0.0, window=0, out=vp(A),
             ldo=512, ws=vp(A), wsb=1 << 40, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("f", ["b200q_attn_decode", "b200q_attn_prompt"])
@pytest.mark.parametrize("kw", CACHE_REFUSALS + [
    dict(q=None), dict(out=None), dict(q=vp(A + 8)), dict(out=vp(A + 4)), dict(ldq=504), dict(ldo=516), dict(rows=-1), dict(hq=0),
    dict(hq=5), dict(max_rows=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(softcap=-1.0), dict(softcap=float("nan")), dict(window=-1), dict(ws=None), dict(ws=vp(A + 8))])
def test_attention_refuses(f, kw):
    assert getattr(b200q.lib(), f)(*attn_args(**kw)) == b200q.EINVAL


def test_attention_of_no_rows_too_many_and_too_little_workspace():
    L = b200q.lib()
    for f in (L.b200q_attn_decode, L.b200q_attn_prompt):
        assert f(*attn_args(rows=0)) == b200q.OK
        assert f(*attn_args(wsb=16)) == b200q.ENOSPACE
    assert L.b200q_attn_decode(*attn_args(max_rows=17)) == b200q.EINVAL
    assert L.b200q_attn_decode_workspace_bytes(4, 2, 128, 17) == 0
    assert 0 < L.b200q_attn_decode_workspace_bytes(32, 8, 128, 1) <= 8 << 20


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
