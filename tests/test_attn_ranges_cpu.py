"""Scales and caps whose quotient or exponent factor fp32 cannot hold are refused (before a launch: the addresses below are
never read).  A quotient of 0 would stand for "no cap"."""
import pytest

import b200q
from test_paged_cpu import ATTN, call


@pytest.mark.parametrize("f", ["b200q_attn_decode", "b200q_attn_prompt"])
@pytest.mark.parametrize("scale,softcap", [(1e-10, 9e37), (1e-7, 5e37), (0.125, 0.125 * 2.0 ** 126.5), (1e-30, 1e10), (3e38, 0.0), (2.5e38, 1e37)])
def test_refused(f, scale, softcap):
    assert call(f, ATTN, dict(scale=scale, softcap=softcap)) == b200q.EINVAL


@pytest.mark.parametrize("f", ["b200q_attn_decode", "b200q_attn_prompt"])
@pytest.mark.parametrize("scale,softcap", [(1e-30, 0.0), (1.9e38, 0.0), (0.125, 1e36), (1e-6, 1e-6)])
def test_not_refused(f, scale, softcap):
    """without rows nothing is launched"""
    assert call(f, ATTN, dict(scale=scale, softcap=softcap, rows=0)) == b200q.OK
