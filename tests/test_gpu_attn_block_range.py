"""The attention-block operators at the ends of their types' range: large and small gradients and
scores in fp16, values that are not finite, element offsets past 32 bits, ReLU's kink.

Tolerances are those of test_gpu_attn_block.py's rounding model, unchanged.
"""
import ctypes

import numpy as np
import pytest

import attn_block_ref as ref
from attn_block_ref import np_type, rounded, to_bits
from test_gpu_attn_block import BF16, F16, F32, _Case, _dev, _get, _gn_ws, _new

pytestmark = pytest.mark.gpu


def _set(c, **values):
    """A case with other values in some of q, k, v, do."""
    for name, a in values.items():
        a = rounded(a, c.dtype)
        assert np.isfinite(a).all()
        setattr(c, name, a)
        setattr(c, {"q": "dq_", "k": "dk_", "v": "dv_", "do": "ddo"}[name], c._put(a))
    return c


# ---------------------------------------------------------------- the forward's lse
@pytest.mark.parametrize("scale", [None, 1.0, -0.125])
def test_attention_f16_lse_of_large_scores(gpu, scale):
    """Every score has a large common part, about 45,000 behind the scale: lse is that of the sums that
    the kernel took."""
    c = _Case(1, 2, 1, 140, 270, 64, F16, scale=scale)
    common = np.sqrt(45000 / abs(float(c.scale)))
    q, k = c.q.copy(), c.k.copy()
    q[..., 0] = common * np.sign(c.scale)
    k[..., 0] = common
    _, lse, _, _ = _set(c, q=q, k=k).check_forward()
    assert lse.min() > 40000
