"""The attention block (GroupNorm + SiLU, projection, attention, projection, dropout + residual)
against the same formulas in 64 bits: output and every gradient."""
import numpy as np
import pytest

import attn_block_ref as ref
from attn_block_ref import U, from_bits, np_type, rounded, to_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(2, 7, 9, 64, 2, 8), (1, 14, 14, 128, 2, 32), (1, 1, 1, 64, 4, 4),
                                   (2, 5, 31, 192, 8, 12)])
@pytest.mark.parametrize("dtype,code,p", [("bf16", 1, 0.0), ("fp16", 2, 0.1)])
def test_attention_block(gpu, shape, dtype, code, p):
    from omnimatchdeeplearningtool_b200.attention_block import AttentionBlock
    from omnimatchdeeplearningtool_b200.backend import DeviceBuffer
    n, h, w, c, heads, groups = shape
    t, d = h * w, c // heads
    rng = np.random.Generator(np.random.PCG64(c + t))
    prm = {"gamma": 1 + 0.2 * rng.standard_normal(c), "beta": 0.2 * rng.standard_normal(c),
           "w_qkv": rng.standard_normal((3 * c, c)) / np.sqrt(c), "b_qkv": 0.1 * rng.standard_normal(3 * c),
           "w_out": rng.standard_normal((c, c)) / np.sqrt(c), "b_out": 0.1 * rng.standard_normal(c)}
    prm = {k: v.astype(np.float32) for k, v in prm.items()}
    x, do = (rounded(rng.standard_normal((n, t, c)), code) for _ in range(2))
    blk = AttentionBlock(n, h, w, c, heads, groups, prm, dtype, dropout=p, seed=77)
    xd, dod = DeviceBuffer.from_numpy(to_bits(x, code)), DeviceBuffer.from_numpy(to_bits(do, code))
    blk.forward(xd.ptr, step=3)
    got = {"out": from_bits(blk.out.to_numpy((n, t, c), np_type(code)), code)}
    grads = blk.backward(dod.ptr)
    got["x"] = from_bits(grads["x"].to_numpy((n, t, c), np_type(code)), code)
    for k, v in prm.items():
        got[k] = grads[k].to_numpy(v.shape).astype(np.float64)

    wq, wo = rounded(prm["w_qkv"], code), rounded(prm["w_out"], code)
    hid, _, rstd, z, xh = ref.group_norm(x, prm["gamma"].astype(float), prm["beta"].astype(float), groups, 1e-5, 3)
    qkv = (hid @ wq.T + prm["b_qkv"]).reshape(n, t, 3, heads, d)
    att, saved = np.zeros((n, t, heads, d)), {}
    mask, scale = np.ones((t, t), bool), 1 / np.sqrt(d)
    for i in range(n):
        for j in range(heads):
            o, _, pr = ref.attention(*(qkv[i, :, a, j] for a in range(3)), scale, mask)
            att[i, :, j], saved[i, j] = o, pr
    y = att.reshape(n, t, c) @ wo.T + prm["b_out"]
    keep, f = ref.keep_mask(n * t * c, p, 77, 3)
    drop = np.where(keep, f, 0.0).reshape(n, t, c)
    want = {"out": x + drop * y}
    dy = drop * do
    want["w_out"] = dy.reshape(-1, c).T @ att.reshape(-1, c)
    want["b_out"] = dy.sum((0, 1))
    datt = (dy @ wo).reshape(n, t, heads, d)
    dqkv = np.zeros_like(qkv)
    for i in range(n):
        for j in range(heads):
            g, _, _ = ref.attention_backward(*(qkv[i, :, a, j] for a in range(3)), att[i, :, j], datt[i, :, j],
                                             saved[i, j], scale, mask)
            for a in range(3):
                dqkv[i, :, a, j] = g[a]
    dqkv = dqkv.reshape(n, t, 3 * c)
    want["w_qkv"] = dqkv.reshape(-1, 3 * c).T @ hid.reshape(-1, c)
    want["b_qkv"] = dqkv.sum((0, 1))
    dx, want["gamma"], want["beta"], _, _ = ref.group_norm_backward(dqkv @ wq, z, xh, rstd, prm["gamma"].astype(float),
                                                                    groups, 3)
    want["x"] = dx + do
    # about eight 16-bit roundings between the input and the last gradient, each of half an ulp of
    # values of the tensor's size; twice that
    for k in want:
        err = np.abs(got[k] - want[k]).max() / max(np.abs(want[k]).max(), 1e-3)
        assert err <= 16 * U[code], (k, err)
    blk.close()


def test_attention_block_refuses_what_it_cannot_store():
    from omnimatchdeeplearningtool_b200.attention_block import AttentionBlock
    prm = {k: np.zeros(1, np.float32) for k in ("gamma", "beta", "w_qkv", "b_qkv", "w_out", "b_out")}
    for c, heads, groups in ((60, 4, 4), (64, 3, 4), (64, 4, 5), (320, 2, 4)):
        with pytest.raises(ValueError):
            AttentionBlock(1, 2, 2, c, heads, groups, prm)
    with pytest.raises(ValueError):
        AttentionBlock(1, 2, 2, 64, 4, 4, prm, dtype="fp32")
