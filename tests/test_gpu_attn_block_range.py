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


# ---------------------------------------------------------------- the backward's lse and delta in fp16
@pytest.mark.parametrize("d,scale", [(64, None), (64, 1.0), (80, None), (64, -0.125)])
def test_attention_f16_large_lse(gpu, d, scale):
    """Log-sum-exps of about 45,000: every score has a large common part."""
    c = _Case(1, 2, 1, 140, 270, d, F16, scale=scale)
    common = np.sqrt(45000 / abs(float(c.scale)))
    q, k = c.q.copy(), c.k.copy()
    q[..., 0] = common * np.sign(c.scale)
    k[..., 0] = common
    _set(c, q=q, k=k)
    o, lse, p, es = c.check_forward()
    assert lse.min() > 40000
    c.check_backward(o, lse, p, es)


def test_attention_f16_large_negative_lse(gpu):
    c = _Case(1, 2, 1, 140, 270, 64, F16)
    q, k = c.q.copy(), c.k.copy()
    q[..., 0], k[..., 0] = 600, -600
    _set(c, q=q, k=k).check()


@pytest.mark.parametrize("d,scale", [(64, None), (128, None), (40, 2.0 ** -19)])
def test_attention_f16_large_delta(gpu, d, scale):
    """sum(dO * out) of every query above 1.05e6 (16 times the type's range), as loss scaling can bring;
    the results stay in range. One head has small gradients beside it."""
    c = _Case(1, 2, 2, 140, 150, d, F16, scale=scale)
    do = (1.2e6 / d) * (1 + 0.1 * c.do)
    do[:, :, 1] = 0.01 * c.do[:, :, 1]
    _set(c, v=1.2 + 0.05 * c.v, do=do)
    o, lse, p, es = c.check_forward()
    assert (c.do[:, :, 0] * o[:, :, 0]).sum(-1).min() > 1.05e6
    c.check_backward(o, lse, p, es)


def test_attention_one_query_beyond_range_leaves_dv_alone(gpu):
    """delta of one query beyond 2^31: dV, which it is no part of, is what it is."""
    c = _Case(1, 1, 1, 130, 140, 128, F16)
    q, v, do = c.q.copy(), 300 + 0.1 * c.v, 0.01 * c.do
    do[0, 5] = 65000.0
    q[0, 5] = 0
    _set(c, q=q, v=v, do=do)
    o, lse, p = c.reference()
    assert (c.do[0, 5, 0] * o[0, 5, 0]).sum() > 2.0 ** 31
    _, _, dv = c.backward(rounded(o, F16), lse)
    want = p[0, 0].T @ c.do[0, :, 0]
    size = p[0, 0].T @ np.abs(c.do[0, :, 0])
    es = 8 * 2.0 ** -24 * (float(c.scale) * np.sqrt((c.q ** 2).sum(-1).max() * (c.k ** 2).sum(-1).max()) + 8)
    assert (np.abs(dv[0, :, 0] - want) <= (2.0 ** -11 + es + 32 * 2.0 ** -24) * size + 2.0 ** -11 * np.abs(want) + 2.0 ** -24).all()
