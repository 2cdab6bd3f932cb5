"""b200q_kv_append refuses a q_out that lies on what the kernel has yet to read (before a launch: the addresses below are
never read).  fp32 rows cannot be replaced in place by bf16 ones: head h of the result would lie on the input's head h / 2."""
import pytest

import b200q
from test_paged_cpu import A, append

W, K = 4 * 128, 2 * 128   # a row's values of q, and of k or v
FUSED = W + 2 * K


@pytest.mark.parametrize("kw", [
    dict(),                                                          # fp32 on itself
    dict(ldo=2 * 512),                                               # at the same pitch in bytes
    dict(x_dtype=1, ldo=520),                                        # bf16 at another pitch
    dict(x_dtype=1, ldq=520),
    dict(x_dtype=1, qo=A + 16),                                      # a little off itself
    dict(x_dtype=1, qo=A + 2 * 128),
    dict(x_dtype=1, rows=1, qo=A + 2 * 128),
    dict(x_dtype=0, rows=1),
])
def test_q_out_on_q(kw):
    far = A + (1 << 24)
    assert append(**dict(dict(k=far, v=far + (1 << 20)), **kw)) == b200q.EINVAL


@pytest.mark.parametrize("x_dtype,e", [(0, 4), (1, 2)])
@pytest.mark.parametrize("at", [W, W + K - 8, W + K, FUSED - 8, -8])
def test_q_out_on_k_or_v_of_one_buffer(x_dtype, e, at):
    """a fused row [q | k | v]; q_out begins at value `at` of the row, in the rows' own pitch (-8: in the row before)"""
    ld = dict(ldq=FUSED, ldk=FUSED, ldv=FUSED, ldo=FUSED * e // 2)
    qo = A + (1 << 20) + at * e
    assert append(x_dtype=x_dtype, q=A + (1 << 20), k=A + (1 << 20) + W * e, v=A + (1 << 20) + (W + K) * e, qo=qo, **ld) == b200q.EINVAL
