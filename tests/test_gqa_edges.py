"""The paged cache of ordinary heads without a GPU, at its edges: what the entry points of include/gqa_attn.h refuse and accept beside tests/test_gqa.py."""
import ctypes as C

import pytest

import jittorinfer_amd as J
from tests.test_gqa import SHAPE, UNSUPPORTED, _attn, _cut, _latent, _pool, _rows


@pytest.mark.parametrize("cap,code", [(float("inf"), UNSUPPORTED), (float("nan"), UNSUPPORTED), (3.4e38, 0), (1e-45, 0)])
def test_softcaps_are_finite(cap, code):
    """c tanh(s / c) has no value at an infinite c."""
    for a in (_attn(logit_softcap=cap), _latent(logit_softcap=cap)):
        assert J.library().gqa_attn_check(C.byref(a)) == code
