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


# ---------------------------------------------------------------- score gradients in fp16
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-5])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_small_gradients(gpu, size, d, dtype):
    """Gradients of the size that long training has, over 4096 keys; the other operand is large enough
    for results in the type's normal range, so that the score gradients' rounding shows."""
    big = min(3000.0, 30 / size)
    c = _Case(1, 1, 1, 140, 4096, d, dtype)
    _set(c, k=c.k * big, q=c.q / big, do=c.do * size).check()
    c = _Case(1, 2, 1, 4096, 70, d, dtype)
    _set(c, q=c.q * big, k=c.k / big, do=c.do * size).check()


@pytest.mark.parametrize("scale", [2.0 ** -19, 2.0 ** -16, -2.0 ** -12])
def test_attention_small_scale(gpu, scale):
    c = _Case(1, 2, 1, 197, 197, 64, F16, scale=scale)
    _set(c, k=c.k * 2000).check()
    c = _Case(1, 2, 1, 197, 197, 64, F16, scale=scale)
    _set(c, q=c.q * 2000).check()


@pytest.mark.parametrize("scale", [1.0, 3.0, 5.5])
def test_attention_large_scale(gpu, scale):
    c = _Case(1, 2, 1, 150, 197, 64, F16, scale=scale)
    _set(c, q=0.2 * c.q, k=0.2 * c.k).check()


def test_attention_gradients_of_unlike_sizes(gpu):
    """Queries' gradients from 1e-4 to 1e4 side by side: each row of dQ at its own precision; heads and
    batch entries whose gradients are zero or whose queries are not in use among them."""
    c = _Case(2, 4, 2, 300, 500, 64, F16, qlens=[300, 129], klens=[500, 260])
    size = 10.0 ** np.linspace(-4, 4, 300)[None, :, None, None]
    do = c.do * size
    do[:, :, 1], do[1, :40, 2], do[0, 250:, 3] = 0, 0, 0
    _set(c, k=c.k / 8, q=c.q, v=c.v, do=do)
    o, lse, p, es = c.check_forward()
    dq, dk, dv = c.backward(rounded(o, F16), lse)
    assert np.isfinite(dq).all() and np.isfinite(dk).all() and np.isfinite(dv).all()
    assert (dq[:, :, 1] == 0).all() and (dq[1, 129:] == 0).all() and (dk[1, 260:] == 0).all()
    u = 2.0 ** -11
    for i in range(2):
        m = ref.visible(300, 500, c.ql[i], c.kl[i], False)
        for j in range(4):
            g, terms, sizes = ref.attention_backward(c.q[i, :, j], c.k[i, :, j // 2], c.v[i, :, j // 2],
                                                     rounded(o, F16)[i, :, j], c.do[i, :, j], p[i, j], float(c.scale), m)
            tol = u * terms[0] + (es + 32 * 2.0 ** -24) * sizes[0] + u * np.abs(g[0]) + 2.0 ** -24
            assert (np.abs(dq[i, :, j] - g[0]) <= tol).all()


@pytest.mark.parametrize("grad,qsize,ksize", [("dq", 100, 0.01), ("dk", 0.01, 100)])
def test_attention_large_gradients_stay_finite(gpu, grad, qsize, ksize):
    """Score gradients far beyond the type's range (sharp scores, sum(dO v) of 1e6) whose products with
    the small operand lie in it."""
    c = _Case(1, 2, 1, 197, 260, 64, F16, scale=1.0)
    _set(c, q=qsize * c.q, k=ksize * c.k, v=40 * c.v, do=5e3 * np.tanh(c.do))
    o, lse, p, es = c.check_forward()
    o = rounded(o, F16)
    got = dict(zip(("dq", "dk", "dv"), c.backward(o, lse)))[grad]
    want, tol, top, u = np.zeros_like(got), np.zeros_like(got), 0, 2.0 ** -11
    for j in range(2):
        g, terms, sizes = ref.attention_backward(c.q[0, :, j], c.k[0, :, 0], c.v[0, :, 0], o[0, :, j], c.do[0, :, j],
                                                 p[0, j], float(c.scale), np.ones((197, 260), bool))
        n, at = (0, j) if grad == "dq" else (1, 0)
        want[0, :, at] += g[n]
        tol[0, :, at] += u * terms[n] + (es + 32 * 2.0 ** -24) * sizes[n]
        delta = (c.do[0, :, j] * o[0, :, j]).sum(1, keepdims=True)
        top = max(top, np.abs(p[0, j] * (c.do[0, :, j] @ c.v[0, :, 0].T - delta)).max())
    assert top > 2e5 and (np.abs(want) + tol).max() < 65504
    assert (np.abs(got - want) <= tol + u * np.abs(want) + 2.0 ** -24).all()


# ---------------------------------------------------------------- probabilities in fp16
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_rarely_seen_keys(gpu, d, dtype):
    """Keys that every query gives a probability of about 1e-7: their dV at the same relative precision."""
    c = _Case(1, 2, 1, 300, 400, d, dtype)
    q, k = c.q.copy(), c.k.copy()
    q[..., 0] = 8
    k[:, ::2, :, 0] = -10 / (8 * float(c.scale))
    _set(c, q=q, k=k, do=500 * c.do)
    _, _, p = c.reference()
    assert p[0, 0][:, ::2].max() < 1e-5
    c.check()


# ---------------------------------------------------------------- GroupNorm's two passes at the kink
@pytest.mark.parametrize("shape", [(1, 49, 64, 64, 8), (2, 300, 48, 48, 12), (3, 130, 15, 16, 3), (1, 30011, 64, 64, 8),
                                   (1, 30011, 32, 32, 8), (2, 9, 40, 40, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_group_norm_passes_agree_at_the_kink(gpu, shape, dtype):
    """The backward lets a gradient through where the forward's output is above 0, and nowhere else:
    on constant maps (every pre-activation within rounding of 0), and where a map's values meet the
    kink. dY is 1, so the gradient of beta counts the elements that let it through."""
    from omnimatchdeeplearningtool_b200._lib import call
    n, hw, c, cs, g = shape
    elem, cpg = 4 if dtype == F32 else 2, c // g
    rng = np.random.Generator(np.random.PCG64(sum(shape) + dtype))
    for trial in range(6):
        if trial % 2 == 0:                  # constant maps
            x = np.repeat(rng.choice([-1, 1], (n, 1, g)) * 10.0 ** rng.uniform(0, 2, (n, 1, g)), cpg, 2) * np.ones((1, hw, 1))
            beta = np.zeros(c)
        elif dtype == F16:                  # (an output below 2^-25 would be 0 in f16)
            continue
        else:                               # a few values a map; beta puts one of them on the kink
            x = rng.integers(-3, 4, (n, hw, c)) * 0.37 + rng.standard_normal((1, 1, c))
            x = rounded(x, dtype)
            _, mean, rstd, _, xh = ref.group_norm(x, 1.0, 0.0, g, 1e-5, 0)
            beta = None
        x = rounded(x, dtype)
        gamma = rounded(rng.choice([-1, 1], c) * rng.uniform(0.5, 2, c), F32)
        if beta is None:
            beta = rounded(-xh[0, 0] * gamma, F32)
        full = np.zeros((n, hw, cs))
        full[..., :c] = x
        xd, gd, bd = _dev(full, dtype), _dev(gamma.astype(np.float32)), _dev(beta.astype(np.float32))
        y, m, r = _new(n * hw * cs * elem), _new(n * g * 4), _new(n * g * 4)
        dy = _dev(np.ones((n, hw, cs)), dtype)
        dx, dg, db = _new(n * hw * cs * elem), _new(c * 4), _new(c * 4)
        for kind in (1, 2) if dtype == F32 else (1,):
            call("omCudaGroupNormActNhwc", xd.ptr, y.ptr, gd.ptr, bd.ptr, m.ptr, r.ptr, _gn_ws(n, hw, c, cs, g, dtype, 0).ptr,
                 n, hw, c, cs, g, 1e-5, kind, dtype)
            call("omCudaGroupNormActNhwcBackward", dy.ptr, xd.ptr, m.ptr, r.ptr, gd.ptr, bd.ptr, dx.ptr, dg.ptr, db.ptr,
                 _gn_ws(n, hw, c, cs, g, dtype, 1).ptr, n, hw, c, cs, g, kind, dtype)
            out = _get(y, (n, hw, cs), dtype)[..., :c]
            through = (out > 0) & ((kind == 1) | (out < 6))
            assert (db.to_numpy((c,)) == through.sum((0, 1))).all(), (trial, kind)


# ---------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("dims", [(1, 2, 1, 5, 4096, 64), (1, 2, 2, 300, 200, 64), (2, 2, 1, 150, 300, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_nan_scores_are_not_an_empty_row(gpu, dims, dtype):
    """A query with a NaN has NaN as its output and its lse (minus infinity says that a query sees no
    key); a NaN in one key reaches every query that sees it. Other queries are as without it."""
    b, h, hkv, sq, sk, d = dims
    c = _Case(*dims, dtype)
    want, wl = c.forward()
    q = c.q.copy()
    q[0, 1, 0, 3] = np.nan
    c.q, c.dq_ = q, c._put(q)
    got, gl = c.forward()
    hit = np.zeros((b, sq, h), bool)
    hit[0, 1, 0] = True
    assert np.isnan(got[hit]).all() and np.isnan(gl.transpose(0, 2, 1)[hit]).all()
    assert (got[~hit] == want[~hit]).all() and (gl.transpose(0, 2, 1)[~hit] == wl.transpose(0, 2, 1)[~hit]).all()
    c = _Case(*dims, dtype)
    c.k[0, sk // 2, 0, 2] = np.nan
    c.dk_ = c._put(c.k)
    got, gl = c.forward()
    assert np.isnan(got[0, :, :h // hkv]).all() and np.isnan(gl[0, :h // hkv]).all()
    assert (got[1:] == want[1:]).all() and (gl[1:] == wl[1:]).all()


# ---------------------------------------------------------------- dropout in a captured step
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_dropout_replayed_with_another_step(gpu, dtype):
    """A captured call draws the mask of the step that device memory holds when it is replayed, the same
    as a call with that offset."""
    from omnimatchdeeplearningtool_b200._lib import call, lib
    n, seed, base = 5003, 9, (1 << 40) - 2
    rng = np.random.Generator(np.random.PCG64(dtype))
    x, r = _dev(rng.standard_normal(n), dtype), _dev(rng.standard_normal(n), dtype)
    step, out, one = _dev(np.zeros(1, np.uint64)), _new(n * 4), _new(n * 4)
    args = (x.ptr, r.ptr, out.ptr, n, 0.3, seed, base, step.ptr, dtype)
    call("omCudaDropoutAddStep", *args)
    call("omCudaSynchronize")
    call("omCudaGraphBeginCapture")
    st = lib.omCudaDropoutAddStep(*args)
    graph = ctypes.c_void_p()
    assert lib.omCudaGraphEndCapture(ctypes.byref(graph)) == 0 and st == 0
    seen = []
    for s in (0, 1, 2, 1 << 33, 1):
        step.upload(np.array([s], np.uint64))
        call("omCudaGraphLaunch", graph)
        call("omCudaSynchronize")
        got = out.to_numpy((n,), np_type(dtype))
        call("omCudaDropoutAdd", x.ptr, r.ptr, one.ptr, n, 0.3, seed, base + s, dtype)
        assert (got == one.to_numpy((n,), np_type(dtype))).all()
        seen.append(got)
    call("omCudaGraphDestroy", graph)
    assert (seen[1] == seen[4]).all() and all((a != b).any() for i, a in enumerate(seen[:4]) for b in seen[:i])


def test_dropout_step_refusals(gpu):
    from omnimatchdeeplearningtool_b200._lib import lib
    b, step = _new(4096), _new(16)

    def f(p=step.ptr, prob=0.1, n=8):
        return lib.omCudaDropoutAddStep(b.ptr, None, b.ptr, n, prob, 0, 0, p, BF16)

    assert f() == 0 and f(n=0) == 0
    assert f(p=None) == -2 and f(p=step.ptr + 4) == -2 and f(prob=1.5) == -2 and f(n=-1) == -2


# ---------------------------------------------------------------- dropout past 32 bits of elements and of groups
@pytest.mark.parametrize("shift", [32, 35])
def test_dropout_long_tensors(gpu, shift):
    """The last elements of an in-place call of 2^32 + 24 (2^35 + 24) elements are those of their own
    index: past 2^32 the element offset, past 2^35 the group index needs its high word."""
    import torch
    from omnimatchdeeplearningtool_b200._lib import call
    from omnimatchdeeplearningtool_b200.backend import DeviceBuffer
    n = (1 << shift) + 24
    if torch.cuda.mem_get_info(0)[0] < 2 * n + (8 << 30):
        pytest.skip("not enough free device memory")
    buf = DeviceBuffer(2 * n)
    try:
        call("omCudaMemset", buf.ptr, 0x3F, buf.nbytes)       # 0x3F3F, 0.74609375
        call("omCudaDropoutAdd", buf.ptr, None, buf.ptr, n, 0.5, 77, 5, BF16)
        last = np.zeros(4096 + 24, np.uint16)
        call("omCudaCopyD2H", last.ctypes.data, buf.ptr + 2 * (n - last.size), last.nbytes)
        first = np.zeros(4096, np.uint16)
        call("omCudaCopyD2H", first.ctypes.data, buf.ptr, first.nbytes)
    finally:
        buf.free()
    keep, _ = ref.keep_mask(last.size, 0.5, 77, 5, first=n - last.size)
    assert ((last != 0) == keep).all() and (last[keep] == 0x3FBF).all()
    keep, _ = ref.keep_mask(4096, 0.5, 77, 5)
    assert ((first != 0) == keep).all()


def test_attention_backward_scale_limits(gpu):
    from omnimatchdeeplearningtool_b200._lib import lib
    b, ws, g = _new(1 << 16), _new(1 << 20), _new(1 << 16)
    st = (ctypes.c_longlong * 24)(*[256, 64, 64] * 8)

    def f(scale):
        return lib.omCudaAttentionBackward(b.ptr, b.ptr, b.ptr, b.ptr, b.ptr, b.ptr, g.ptr, g.ptr + 8192, g.ptr + 16384, st,
                                           None, None, ws.ptr, 1, 1, 1, 4, 4, 64, scale, 0, BF16)

    assert f(2.0 ** -20) == 0 and f(-2.0 ** -20) == 0 and f(4.0) == 0
    assert f(2.0 ** -21) == -3 and f(0.0) == -3 and f(float("inf")) == -2 and f(float("nan")) == -2
