"""GroupNorm + activation, dropout and attention on the device against their 64-bit references.

Tolerances come from the rounding model, before any run: u = half an ulp of the type
(attn_block_ref.U), inputs exact (rounded before the reference sees them).
"""
import ctypes

import numpy as np
import pytest

import attn_block_ref as ref
from attn_block_ref import U, from_bits, np_type, rounded, to_bits

pytestmark = pytest.mark.gpu

F32, BF16, F16 = 0, 1, 2


def _dev(a, dtype=None):
    from omnimatchdeeplearningtool_b200.backend import DeviceBuffer
    return DeviceBuffer.from_numpy(a if dtype is None else to_bits(a, dtype))


def _new(nbytes):
    """A buffer of NaN patterns (0xFF bytes), so that what a call leaves unwritten shows."""
    from omnimatchdeeplearningtool_b200._lib import call
    from omnimatchdeeplearningtool_b200.backend import DeviceBuffer
    b = DeviceBuffer(max(int(nbytes), 16))
    call("omCudaMemset", b.ptr, 0xFF, b.nbytes)
    return b


def _get(buf, shape, dtype):
    return from_bits(buf.to_numpy(shape, np_type(dtype)), dtype)


# ---------------------------------------------------------------- GroupNorm
def _gn_ws(n, hw, c, cs, g, dtype, backward):
    from omnimatchdeeplearningtool_b200._lib import lib
    nbytes = lib.omCudaGroupNormNhwcWorkspaceBytes(n, hw, c, cs, g, dtype, backward)
    assert nbytes >= 0
    return _new(nbytes)


# one value a group; groups that end inside a vector; padded channels; one group; many channels;
# a sample of one pixel; tall maps; more channels than a block's threads cover at once
GN_SHAPES = [(1, 1, 8, 8, 8), (2, 3, 20, 24, 5), (1, 49, 512, 512, 32), (3, 130, 15, 16, 1), (2, 257, 96, 96, 32),
             (5, 1, 40, 40, 4), (1, 5000, 24, 24, 3), (2, 61, 2304, 2304, 16), (1, 9, 4099, 4104, 1),
             (40, 17, 30, 32, 10), (3, 3136, 64, 64, 32), (1, 30011, 64, 64, 8)]


@pytest.mark.parametrize("shape", GN_SHAPES)
@pytest.mark.parametrize("dtype,kind", [(F32, 3), (BF16, 1), (F16, 0), (BF16, 3), (F16, 2)])
def test_group_norm(gpu, shape, dtype, kind):
    from omnimatchdeeplearningtool_b200._lib import call
    n, hw, c, cs, g = shape
    rng = np.random.Generator(np.random.PCG64(sum(shape) + dtype * 7 + kind))
    x = np.zeros((n, hw, cs))
    x[..., :c] = rng.standard_normal((n, hw, c)) * rng.uniform(0.5, 2, c) + 3 * rng.standard_normal(c)
    x = rounded(x, dtype)
    x_dev = x.copy()
    x_dev[..., c:] = np.nan      # what the padding holds is not used
    dy = rounded(rng.standard_normal((n, hw, cs)), dtype)
    gamma = rounded(1 + 0.3 * rng.standard_normal(c), F32)
    beta = rounded(0.5 * rng.standard_normal(c), F32)
    y, mean, rstd, z, xh = ref.group_norm(x[..., :c], gamma, beta, g, 1e-5, kind)

    elem = {F32: 4}.get(dtype, 2)
    dx_, dg_, db_ = _dev(x_dev, dtype), _dev(gamma.astype(np.float32)), _dev(beta.astype(np.float32))
    out, m, r = _new(n * hw * cs * elem), _new(n * g * 4), _new(n * g * 4)
    call("omCudaGroupNormActNhwc", dx_.ptr, out.ptr, dg_.ptr, db_.ptr, m.ptr, r.ptr,
         _gn_ws(n, hw, c, cs, g, dtype, 0).ptr, n, hw, c, cs, g, 1e-5, kind, dtype)
    got = _get(out, (n, hw, cs), dtype)
    # fp32 statistics: the mean is off by a few ulps of the values' size, which the normalisation
    # multiplies by rstd, as it does the inverse deviation's relative error
    e = 16 * U[F32]
    size = np.abs(x[..., :c]).max()
    cpg = c // g
    rc = np.repeat(rstd, cpg, 1)[:, None, :]
    tol = U[dtype] * np.abs(y) + e * (np.abs(gamma) * (size * rc + np.abs(xh) * (1 + size ** 2 * rc ** 2)) + np.abs(z)) * 2
    assert (np.abs(got[..., :c] - y) <= tol + 2.0 ** -24).all()
    assert (got[..., c:] == 0).all()
    assert (np.abs(m.to_numpy((n, g)) - mean) <= e * size).all()
    assert (np.abs(r.to_numpy((n, g)) - rstd) <= e * rstd * (1 + size ** 2 * rstd ** 2)).all()

    # backward from the reference's statistics
    mean32, rstd32 = mean.astype(np.float32), rstd.astype(np.float32)
    xh = ((x[..., :c].reshape(n, hw, g, cpg) - mean32[:, None, :, None]) * rstd32[:, None, :, None].astype(np.float64)
          ).reshape(n, hw, c)
    z = xh * gamma + beta
    dx, dgam, dbet, dsize, dz = ref.group_norm_backward(dy[..., :c], z, xh, rstd32.astype(np.float64), gamma, g, kind)
    dyd, dm, dr = _dev(dy, dtype), _dev(mean32), _dev(rstd32)
    gx, gg, gb = _new(n * hw * cs * elem), _new(c * 4), _new(c * 4)
    call("omCudaGroupNormActNhwcBackward", dyd.ptr, dx_.ptr, dm.ptr, dr.ptr, dg_.ptr, db_.ptr, gx.ptr, gg.ptr, gb.ptr,
         _gn_ws(n, hw, c, cs, g, dtype, 1).ptr, n, hw, c, cs, g, kind, dtype)
    got = _get(gx, (n, hw, cs), dtype)
    assert (got[..., c:] == 0).all()
    # fp32 arithmetic moves z by a few ulps; next to a kink (ReLU, ReLU6) the derivative may then
    # fall on the other side, so those elements are judged by the size of their terms
    near = np.zeros(z.shape, bool)
    for kink in {1: (0.0,), 2: (0.0, 6.0)}.get(kind, ()):
        near |= np.abs(z - kink) <= e * (np.abs(xh * gamma) + np.abs(beta) + np.abs(gamma) * size * rc + 1)
    # xh is off by a few ulps of the values' size times rstd, and each mean by its terms' sizes
    noise = 2 * e * dsize * (1 + size * rc) * (1 + np.abs(xh))
    flip = np.abs(dy[..., :c]) * np.abs(gamma) * rc
    loose = near.reshape(n, hw, g, cpg).any((1, 3))      # one flipped element moves its group's means
    loose = np.repeat(loose, cpg, 1)[:, None, :] * flip.max() * (1 + np.abs(xh) * np.abs(xh).max())
    tol = U[dtype] * np.abs(dx) + noise + loose * near.sum() / max(1, hw * cpg) + near * flip
    assert (np.abs(got[..., :c] - dx) <= tol + 2.0 ** -24).all()
    lost = (near * np.abs(dy[..., :c])).sum((0, 1))
    # a sum of n * hw terms in a tree of fp32 partial sums
    sums = 2 * e * (np.abs(dz) * (1 + np.abs(xh) + size * rc)).sum((0, 1))
    assert (np.abs(gg.to_numpy((c,)) - dgam) <= sums + (lost * np.abs(xh).max() if near.any() else 0) + 1e-30).all()
    assert (np.abs(gb.to_numpy((c,)) - dbet) <= sums + lost + 1e-30).all()


@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_group_norm_backward_at_the_kink(gpu, dtype, kind):
    """((x - mean) * rstd) * gamma + beta is 0 in fp32 and below 0 without rounding (-2.7e-9): no gradient."""
    from omnimatchdeeplearningtool_b200._lib import call
    n, hw, c = 1, 300, 8
    mean, rstd, gamma, beta = (np.array([v], np.uint32).view(np.float32) for v in
                               (0xbe7efff0, 0x3f67b984, 0x3f47aba7, 0x3e1933e6))
    x = np.float32(-0.4609375)
    assert (x - mean) * rstd * gamma + beta == 0
    xd, dyd = _dev(np.full((n, hw, c), x), dtype), _dev(np.ones((n, hw, c)), dtype)
    md, rd, gd, bd = _dev(mean), _dev(rstd), _dev(np.repeat(gamma, c)), _dev(np.repeat(beta, c))
    dx, dg, db = _new(n * hw * c * 4), _new(c * 4), _new(c * 4)
    call("omCudaGroupNormActNhwcBackward", dyd.ptr, xd.ptr, md.ptr, rd.ptr, gd.ptr, bd.ptr, dx.ptr, dg.ptr, db.ptr,
         _gn_ws(n, hw, c, c, 1, dtype, 1).ptr, n, hw, c, c, 1, kind, dtype)
    assert (_get(dx, (n, hw, c), dtype) == 0).all()
    assert (dg.to_numpy((c,)) == 0).all() and (db.to_numpy((c,)) == 0).all()


def test_group_norm_optional_arguments_in_place_and_repeat(gpu):
    from omnimatchdeeplearningtool_b200._lib import call
    rng = np.random.Generator(np.random.PCG64(5))
    n, hw, c, g = 2, 333, 48, 6
    x = rounded(rng.standard_normal((n, hw, c)), BF16)
    y = ref.group_norm(x, 1.0, 0.0, g, 1e-3, 0)[0]
    buf, ws = _dev(x, BF16), _gn_ws(n, hw, c, c, g, BF16, 1)
    runs = []
    for _ in range(2):
        out = _new(n * hw * c * 2)
        call("omCudaGroupNormActNhwc", buf.ptr, out.ptr, None, None, None, None, ws.ptr, n, hw, c, c, g, 1e-3, 0, BF16)
        runs.append(out.to_numpy((n, hw, c), np.uint16))
    assert (runs[0] == runs[1]).all()
    call("omCudaGroupNormActNhwc", buf.ptr, buf.ptr, None, None, None, None, ws.ptr, n, hw, c, c, g, 1e-3, 0, BF16)
    assert (buf.to_numpy((n, hw, c), np.uint16) == runs[0]).all()
    assert np.abs(from_bits(runs[0], BF16) - y).max() <= U[BF16] * np.abs(y).max() + 1e-4
    # no parameter gradients asked for; dX over dY
    _, mean, rstd, _, _ = ref.group_norm(x, 1.0, 0.0, g, 1e-3, 0)
    dy = rounded(rng.standard_normal((n, hw, c)), BF16)
    xd, m, r = _dev(x, BF16), _dev(mean.astype(np.float32)), _dev(rstd.astype(np.float32))
    a, b, dg, db = _dev(dy, BF16), _new(n * hw * c * 2), _new(c * 4), _new(c * 4)
    call("omCudaGroupNormActNhwcBackward", a.ptr, xd.ptr, m.ptr, r.ptr, None, None, b.ptr, dg.ptr, db.ptr, ws.ptr, n,
         hw, c, c, g, 0, BF16)
    call("omCudaGroupNormActNhwcBackward", a.ptr, xd.ptr, m.ptr, r.ptr, None, None, a.ptr, None, None, ws.ptr, n, hw,
         c, c, g, 0, BF16)
    assert (a.to_numpy((n, hw, c), np.uint16) == b.to_numpy((n, hw, c), np.uint16)).all()
    # an empty batch: nothing to normalise, and zero parameter gradients
    call("omCudaGroupNormActNhwc", None, None, None, None, None, None, None, 0, hw, c, c, g, 1e-3, 0, BF16)
    call("omCudaGroupNormActNhwcBackward", None, None, None, None, None, None, None, dg.ptr, db.ptr, None, 0, hw, c, c,
         g, 0, BF16)
    assert (dg.to_numpy((c,)) == 0).all() and (db.to_numpy((c,)) == 0).all()


def test_group_norm_refusals(gpu):
    from omnimatchdeeplearningtool_b200._lib import lib
    b, ws = _new(4096), _new(1 << 20)

    def fwd(x=b.ptr, y=b.ptr, ws_=ws.ptr, n=1, hw=4, c=16, cs=16, g=2, eps=1e-5, act=0, dt=BF16):
        return lib.omCudaGroupNormActNhwc(x, y, None, None, None, None, ws_, n, hw, c, cs, g, eps, act, dt)

    assert fwd() == 0
    assert fwd(x=None) == -2 and fwd(y=None) == -2 and fwd(x=b.ptr + 2) == -2
    assert fwd(g=3) == -2 and fwd(cs=12) == -2 and fwd(cs=8) == -2 and fwd(hw=0) == -2 and fwd(n=-1) == -2
    assert fwd(eps=-1.0) == -2 and fwd(eps=float("nan")) == -2 and fwd(act=4) == -2 and fwd(act=-1) == -2
    assert fwd(dt=3) == -3
    assert lib.omCudaGroupNormActNhwcBackward(b.ptr, b.ptr, None, b.ptr, None, None, b.ptr, None, None, ws.ptr, 1, 4,
                                              16, 16, 2, 0, BF16) == -2


# ---------------------------------------------------------------- dropout
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2049, 100003])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("p,res", [(0.1, True), (0.5, False), (0.0, True), (1.0, True), (1.0, False)])
def test_dropout(gpu, n, dtype, p, res):
    from omnimatchdeeplearningtool_b200._lib import call
    rng = np.random.Generator(np.random.PCG64(n + dtype))
    x = rounded(rng.standard_normal(n), dtype)
    r = rounded(rng.standard_normal(n), dtype)
    seed, offset = 0xFEDCBA9876543210, 0x8000000100000002
    keep, scale = ref.keep_mask(n, p, seed, offset)
    want = np.where(keep, x * scale, 0) + (r if res else 0)
    xd, rd, out = _dev(x, dtype), _dev(r, dtype), _new(n * 4)
    call("omCudaDropoutAdd", xd.ptr, rd.ptr if res else None, out.ptr, n, p, seed, offset, dtype)
    got = _get(out, (n,), dtype)
    tol = U[dtype] * np.abs(want) + 2 * U[F32] * (np.abs(x * scale) + np.abs(r)) + 2.0 ** -25
    assert (np.abs(got - want) <= tol).all()
    if not res:
        assert ((got == 0) == (~keep | (x == 0))).all()
    # in place, and the same mask again
    call("omCudaDropoutAdd", xd.ptr, rd.ptr if res else None, xd.ptr, n, p, seed, offset, dtype)
    assert (xd.to_numpy((n,), np_type(dtype)) == out.to_numpy((n,), np_type(dtype))).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_dropout_off_alignment_and_non_finite(gpu, dtype):
    """Pointers off the 16-byte boundary give the same elements; a dropped NaN or infinity is 0."""
    from omnimatchdeeplearningtool_b200._lib import call
    n, size = 1000, 4 if dtype == F32 else 2
    rng = np.random.Generator(np.random.PCG64(dtype))
    x = rounded(rng.standard_normal(n + 3), dtype)
    x[::5], x[1::5] = np.nan, np.inf
    keep, scale = ref.keep_mask(n, 0.3, 11, 5)
    xd, a, b = _dev(x, dtype), _new((n + 3) * 4), _new((n + 3) * 4)
    call("omCudaDropoutAdd", xd.ptr + 3 * size, None, a.ptr + 3 * size, n, 0.3, 11, 5, dtype)
    x0 = _dev(x[3:], dtype)
    call("omCudaDropoutAdd", x0.ptr, None, b.ptr, n, 0.3, 11, 5, dtype)
    got = _get(a, (n + 3,), dtype)
    assert np.isnan(got[:3]).all()      # the 0xFF bytes in front are untouched
    one = _get(b, (n,), dtype)
    assert ((got[3:] == one) | (np.isnan(one) & np.isnan(got[3:]))).all()
    assert (one[~keep] == 0).all()
    assert (np.isnan(one) == (keep & np.isnan(x[3:]))).all() and (np.isinf(one) == (keep & np.isinf(x[3:]))).all()


def test_dropout_counter_past_32_bits_of_elements(gpu):
    """Element 2^32 + i is not element i: the group index is 64 bits wide (one byte-sized check of
    a 2^32-element call would need 16 GB, so the generator's high counter word is checked through
    the offset word that follows it, and the kept share over a large call)."""
    from omnimatchdeeplearningtool_b200._lib import call
    n = 1 << 22
    one, out = _dev(np.ones(n), BF16), _new(n * 2)
    call("omCudaDropoutAdd", one.ptr, None, out.ptr, n, 0.25, 1, 0, BF16)
    a = _get(out, (n,), BF16) != 0
    call("omCudaDropoutAdd", one.ptr, None, out.ptr, n, 0.25, 1, 1 << 32, BF16)
    b = _get(out, (n,), BF16) != 0
    sd = np.sqrt(0.25 * 0.75 / n)
    assert abs(a.mean() - 0.75) < 5 * sd and abs(b.mean() - 0.75) < 5 * sd
    assert abs((a == b).mean() - (0.75 ** 2 + 0.25 ** 2)) < 6 * sd      # independent streams
    keep, _ = ref.keep_mask(4096, 0.25, 1, 0, first=n - 4096)
    assert (a[-4096:] == keep).all()


def test_dropout_refusals(gpu):
    from omnimatchdeeplearningtool_b200._lib import lib
    b = _new(4096)

    def f(x=b.ptr, y=b.ptr, n=8, p=0.1, dt=BF16):
        return lib.omCudaDropoutAdd(x, None, y, n, p, 0, 0, dt)

    assert f() == 0 and f(n=0, x=None, y=None) == 0
    assert f(x=None) == -2 and f(y=None) == -2 and f(n=-1) == -2 and f(x=b.ptr + 1) == -2
    assert f(p=-0.1) == -2 and f(p=1.5) == -2 and f(p=float("nan")) == -2 and f(dt=3) == -3


# ---------------------------------------------------------------- attention
def _strides(layout, b, s, h, d, extra=1):
    """Strides (batch, token, head) and elements of a [b, s, h, d] tensor's allocation."""
    if layout == "bhsd":
        return (h * s * d, d, s * d)
    if layout == "packed":
        return (s * 3 * h * d, 3 * h * d, d)
    return (s * h * d * extra, h * d * extra, d)


def _place(a, layout):
    """The flat memory image of [b, s, h, d] values (bshd with a gap after each token's heads)."""
    if layout == "bhsd":
        return np.ascontiguousarray(a.transpose(0, 2, 1, 3))
    if layout == "gap":
        return np.ascontiguousarray(np.concatenate([a, np.full_like(a, 7.0)], 2))
    return np.ascontiguousarray(a)


class _Case:
    """One attention problem on the host in 64 bits and on the device."""

    def __init__(self, b, h, hkv, sq, sk, d, dtype, layout="bshd", causal=False, qlens=None, klens=None, scale=None,
                 garbage=False, seed=0, qscale=1.0):
        rng = np.random.Generator(np.random.PCG64(seed + b * 131 + h * 17 + sq * 3 + sk * 7 + d))
        self.dims, self.dtype, self.layout, self.causal = (b, h, hkv, sq, sk, d), dtype, layout, causal
        self.scale = np.float32(1 / np.sqrt(d) if scale is None else scale)
        self.q = rounded(rng.standard_normal((b, sq, h, d)) * qscale, dtype)
        self.k, self.v = (rounded(rng.standard_normal((b, sk, hkv, d)), dtype) for _ in range(2))
        self.do = rounded(rng.standard_normal((b, sq, h, d)), dtype)
        self.ql = [sq] * b if qlens is None else [min(max(x, 0), sq) for x in qlens]
        self.kl = [sk] * b if klens is None else [min(max(x, 0), sk) for x in klens]
        if garbage:     # tokens past the lengths hold NaN and infinities
            for i in range(b):
                self.q[i, self.ql[i]:], self.do[i, self.ql[i]:] = np.nan, np.inf
                self.k[i, self.kl[i]:], self.v[i, self.kl[i]:] = np.nan, -np.inf
        self.qlens = None if qlens is None else _dev(np.array(qlens, np.int32))
        self.klens = None if klens is None else _dev(np.array(klens, np.int32))
        self.dq_, self.dk_, self.dv_ = (self._put(x) for x in (self.q, self.k, self.v))
        self.ddo = self._put(self.do)

    def _put(self, a):
        return _dev(_place(a, self.layout), self.dtype)

    def st(self, s, h):
        b, d = self.dims[0], self.dims[5]
        return _strides("bshd" if self.layout == "gap" else self.layout, b, s, h, d, 2 if self.layout == "gap" else 1)

    def read(self, buf, s, h):
        b, d = self.dims[0], self.dims[5]
        if self.layout == "bhsd":
            return _get(buf, (b, h, s, d), self.dtype).transpose(0, 2, 1, 3)
        if self.layout == "gap":
            got = _get(buf, (b, s, 2 * h, d), self.dtype)
            assert np.isnan(got[:, :, h:]).all()        # the gaps are untouched
            return got[:, :, :h]
        return _get(buf, (b, s, h, d), self.dtype)

    def room(self, s, h):
        b, d = self.dims[0], self.dims[5]
        return _new(b * s * h * d * 2 * (2 if self.layout == "gap" else 1))

    def reference(self):
        b, h, hkv, sq, sk, d = self.dims
        o, lse = np.zeros((b, sq, h, d)), np.zeros((b, h, sq))
        p = {}
        for i in range(b):
            m = ref.visible(sq, sk, self.ql[i], self.kl[i], self.causal)
            for j in range(h):
                o[i, :, j], lse[i, j], p[i, j] = ref.attention(self.q[i, :, j], self.k[i, :, j * hkv // h],
                                                              self.v[i, :, j * hkv // h], float(self.scale), m)
        return o, lse, p

    def ws(self, backward):
        from omnimatchdeeplearningtool_b200._lib import lib
        b, h, hkv, sq, sk, d = self.dims
        nbytes = lib.omCudaAttentionWorkspaceBytes(b, h, hkv, sq, sk, d, backward)
        assert nbytes >= 0
        return _new(nbytes)

    def forward(self, lse=True):
        from omnimatchdeeplearningtool_b200._lib import call
        b, h, hkv, sq, sk, d = self.dims
        out, ls = self.room(sq, h), _new(b * h * sq * 4)
        st = (ctypes.c_longlong * 12)(*self.st(sq, h), *self.st(sk, hkv), *self.st(sk, hkv), *self.st(sq, h))
        call("omCudaAttention", self.dq_.ptr, self.dk_.ptr, self.dv_.ptr, out.ptr, ls.ptr if lse else None, st,
             self.qlens.ptr if self.qlens else None, self.klens.ptr if self.klens else None, self.ws(0).ptr, b, h, hkv,
             sq, sk, d, float(self.scale), int(self.causal), self.dtype)
        return self.read(out, sq, h), ls.to_numpy((b, h, sq)).astype(np.float64)

    def backward(self, o, lse):
        from omnimatchdeeplearningtool_b200._lib import call
        b, h, hkv, sq, sk, d = self.dims
        od, ld = self._put(o), _dev(lse.astype(np.float32))
        gq, gk, gv = self.room(sq, h), self.room(sk, hkv), self.room(sk, hkv)
        qs, ks = self.st(sq, h), self.st(sk, hkv)
        st = (ctypes.c_longlong * 24)(*qs, *ks, *ks, *qs, *qs, *qs, *ks, *ks)
        call("omCudaAttentionBackward", self.ddo.ptr, self.dq_.ptr, self.dk_.ptr, self.dv_.ptr, od.ptr, ld.ptr, gq.ptr,
             gk.ptr, gv.ptr, st, self.qlens.ptr if self.qlens else None, self.klens.ptr if self.klens else None,
             self.ws(1).ptr, b, h, hkv, sq, sk, d, float(self.scale), int(self.causal), self.dtype)
        return self.read(gq, sq, h), self.read(gk, sk, hkv), self.read(gv, sk, hkv)

    def check_forward(self):
        o, lse, p = self.reference()
        got, gl = self.forward()
        b, h, hkv, sq, sk, d = self.dims
        u = U[self.dtype]
        # scores: fp32 sums of d products; a score's error is a probability's relative error
        qn = np.sqrt(np.nansum(np.where(np.isinf(self.q), 0, self.q) ** 2, -1)).max(initial=0)
        kn = np.sqrt(np.nansum(np.where(np.isinf(self.k), 0, self.k) ** 2, -1)).max(initial=0)
        es = 8 * U[F32] * (abs(float(self.scale)) * qn * kn + 8)
        for i in range(b):
            for j in range(h):
                v = np.where(p[i, j].any(0)[:, None], self.v[i, :, j * hkv // h], 0)
                size = p[i, j] @ np.abs(v)
                # probabilities and the output are each rounded once to the type
                tol = (u + es) * size + u * np.abs(o[i, :, j]) + 2.0 ** -24
                assert (np.abs(got[i, :, j] - o[i, :, j]) <= tol).all(), (i, j)
        fin = np.isfinite(lse)
        assert (np.isneginf(gl) == ~fin).all()
        assert (np.abs(gl[fin] - lse[fin]) <= es + 2 * U[F32] * np.abs(lse[fin])).all()
        return o, lse, p, es

    def check_backward(self, o, lse, p, es):
        b, h, hkv, sq, sk, d = self.dims
        o = rounded(o, self.dtype)
        got = self.backward(o, lse)
        u = U[self.dtype]
        want = [np.zeros((b, n, m, d)) for n, m in ((sq, h), (sk, hkv), (sk, hkv))]
        tol = [np.zeros_like(w) for w in want]
        for i in range(b):
            m = ref.visible(sq, sk, self.ql[i], self.kl[i], self.causal)
            for j in range(h):
                c = j * hkv // h
                g, terms, sizes = ref.attention_backward(self.q[i, :, j], self.k[i, :, c], self.v[i, :, c], o[i, :, j],
                                                         self.do[i, :, j], p[i, j], float(self.scale), m)
                for w, t, x, y, z, at in zip(want, tol, g, terms, sizes, (j, c, c)):
                    w[i, :, at] += x
                    # each probability or score gradient is rounded once to the type; fp32 noise of
                    # the probability, of the two products and of their difference
                    t[i, :, at] += u * y + (es + 32 * U[F32]) * z
        for w, t, x, name in zip(want, tol, got, ("dq", "dk", "dv")):
            bad = np.abs(x - w) - (t + u * np.abs(w) + 2.0 ** -24)
            assert (bad <= 0).all(), (name, bad.max(), np.abs(x - w).max())

    def check(self):
        self.check_backward(*self.check_forward())


ATTN = [
    # b, h, hkv, sq, sk, d
    (1, 1, 1, 1, 1, 64), (2, 3, 3, 5, 7, 16), (1, 2, 1, 1, 300, 64), (1, 4, 2, 130, 129, 32), (2, 2, 2, 197, 197, 64),
    (1, 2, 2, 128, 128, 128), (1, 1, 1, 257, 383, 80), (1, 6, 2, 64, 64, 24), (1, 2, 2, 300, 1, 40),
    (1, 1, 1, 127, 256, 96), (3, 1, 1, 33, 65, 8), (1, 8, 8, 7, 1100, 32), (1, 1, 1, 900, 3, 128), (2, 2, 1, 1, 1, 120),
]


@pytest.mark.parametrize("dims", ATTN)
@pytest.mark.parametrize("dtype,causal", [(BF16, False), (F16, True)])
def test_attention(gpu, dims, dtype, causal):
    _Case(*dims, dtype, causal=causal).check()


@pytest.mark.parametrize("layout", ["bshd", "bhsd", "gap"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128, 72])
def test_attention_lengths_and_layouts(gpu, layout, causal, d):
    """Padded batches: full, partial, one-token and empty entries, more queries than keys (rows
    that see nothing under the causal mask), with NaN and infinities past the lengths."""
    _Case(5, 4, 2, 150, 200, d, BF16, layout, causal, qlens=[150, 77, 1, 0, 130], klens=[200, 0, 130, 64, 3],
          garbage=True).check()


def test_attention_lengths_are_clamped(gpu):
    _Case(3, 2, 2, 40, 50, 64, F16, qlens=[1000, -5, 40], klens=[50, 9, 2 ** 31 - 1], garbage=True).check()


def test_attention_only_key_lengths(gpu):
    _Case(4, 2, 1, 130, 260, 64, F16, klens=[260, 129, 0, 1], garbage=True).check()


@pytest.mark.parametrize("qscale", [0.0, 30.0, 300.0])
def test_attention_flat_and_sharp_scores(gpu, qscale):
    """Equal scores, and scores so far apart that one key takes all."""
    _Case(1, 2, 2, 140, 270, 64, BF16, qscale=qscale).check()
    _Case(1, 2, 2, 140, 270, 64, BF16, qscale=qscale, scale=-0.2).check()


def test_attention_rising_scores(gpu):
    """Keys whose scores grow along the sequence, so the running maximum moves in every block."""
    c = _Case(1, 1, 1, 130, 1000, 64, BF16)
    c.q[..., 0] = 8.0
    c.k[..., 0] = rounded(np.linspace(-60, 60, 1000), BF16)[None, :, None]
    c.dq_, c.dk_ = c._put(c.q), c._put(c.k)
    c.check()
    c.k = np.ascontiguousarray(c.k[:, ::-1])
    c.dk_ = c._put(c.k)
    c.check()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_more_tiles_than_the_gpu_holds(gpu, d, causal):
    """Many more (batch, head, tile) items than places on the GPU, runs of empty entries among them."""
    rng = np.random.Generator(np.random.PCG64(d))
    b = 70
    qlens = [int(x) for x in rng.integers(0, 161, b)]
    klens = [int(x) for x in rng.integers(0, 301, b)]
    for i in range(10, 40):
        klens[i] = 0
    for i in range(45, 60):
        qlens[i] = 0
    _Case(b, 9, 3, 160, 300, d, F16, causal=causal, qlens=qlens, klens=klens, garbage=True).check()


@pytest.mark.parametrize("b,h,s,causal,d", [(3, 4, 1100, True, 40), (1, 12, 900, False, 64), (2, 6, 1000, True, 128)])
def test_attention_parts_in_turns(gpu, b, h, s, causal, d):
    """Tiles split into parts, several turns a CTA, and parts without keys beside full ones; repeated,
    as what one warp does ahead of another differs from run to run."""
    kl = [s, s // 7, s // 3][:b]
    c = _Case(b, h, h, s, s, d, BF16, causal=causal, klens=kl, garbage=True)
    o, lse, p, es = c.check_forward()
    first = c.forward()
    for _ in range(20):
        got = c.forward()
        assert (got[0] == first[0]).all() and (got[1] == first[1]).all()


def test_attention_serving_batch(gpu):
    """A batch whose tiles take every CTA several turns: each entry repeats one of four (so that the
    device's results can be compared with each other bit for bit), the four against 64 bits."""
    from omnimatchdeeplearningtool_b200._lib import call
    b, h, s, d = 64, 12, 197, 64
    c = _Case(4, h, h, s, s, d, F16)
    o, lse = c.forward()
    c.check_forward()
    st = (ctypes.c_longlong * 12)(*(_strides("bshd", b, s, h, d) * 4))
    qd, kd, vd = (_dev(np.tile(x, (b // 4, 1, 1, 1)), F16) for x in (c.q, c.k, c.v))
    for _ in range(3):
        out, ls = _new(b * s * h * d * 2), _new(b * h * s * 4)
        call("omCudaAttention", qd.ptr, kd.ptr, vd.ptr, out.ptr, ls.ptr, st, None, None, None, b, h, h, s, s, d,
             float(c.scale), 0, F16)
        got = _get(out, (b, s, h, d), F16)
        assert (got == np.tile(o, (b // 4, 1, 1, 1))).all()
        assert (ls.to_numpy((b, h, s)) == np.tile(lse, (b // 4, 1, 1))).all()


def test_attention_packed_projection(gpu):
    """Q, K, V and their gradients as thirds of one [b, s, 3, h, d] tensor, in place."""
    from omnimatchdeeplearningtool_b200._lib import call
    b, s, h, d = 2, 197, 3, 64
    c = _Case(b, h, h, s, s, d, BF16)
    qkv = _dev(np.stack([c.q, c.k, c.v], 2), BF16)
    out, ls = _new(b * s * h * d * 2), _new(b * h * s * 4)
    pk = _strides("packed", b, s, h, d)
    st = (ctypes.c_longlong * 12)(*pk, *pk, *pk, *_strides("bshd", b, s, h, d))
    ptr = [qkv.ptr + i * h * d * 2 for i in range(3)]
    call("omCudaAttention", *ptr, out.ptr, ls.ptr, st, None, None, c.ws(0).ptr, b, h, h, s, s, d, float(c.scale), 0, BF16)
    o, lse = c.forward()
    assert (c.read(out, s, h) == o).all() and (ls.to_numpy((b, h, s)) == lse).all()
    gq, gk, gv = c.backward(o, lse)
    od, g = c._put(o), _new(b * s * 3 * h * d * 2)
    gp = [g.ptr + i * h * d * 2 for i in range(3)]
    one = _strides("bshd", b, s, h, d)
    st = (ctypes.c_longlong * 24)(*pk, *pk, *pk, *one, *one, *pk, *pk, *pk)
    call("omCudaAttentionBackward", c.ddo.ptr, *ptr, od.ptr, ls.ptr, *gp, st, None, None, c.ws(1).ptr, b, h, h, s, s, d,
         float(c.scale), 0, BF16)
    got = _get(g, (b, s, 3, h, d), BF16)
    assert (got[:, :, 0] == gq).all() and (got[:, :, 1] == gk).all() and (got[:, :, 2] == gv).all()


def test_attention_is_repeatable_and_needs_no_lse(gpu):
    for dims in ((2, 4, 2, 300, 700, 64), (1, 2, 2, 3, 2000, 128)):
        c = _Case(*dims, BF16, causal=True)
        o, lse = c.forward()
        o2, lse2 = c.forward()
        assert (o == o2).all() and (lse == lse2).all()
        assert (c.forward(lse=False)[0] == o).all()
        a, b = c.backward(o, lse), c.backward(o, lse)
        assert all((x == y).all() for x, y in zip(a, b))


def test_attention_gradient_against_differences(gpu):
    """The device's gradients along random directions against central differences of the 64-bit
    forward; the bound is the sum of the elements' rounding bounds along the direction."""
    c = _Case(1, 2, 1, 70, 90, 64, F16, causal=True)
    o, lse, p = c.reference()
    got = c.backward(rounded(o, F16), lse)
    rng = np.random.Generator(np.random.PCG64(9))
    base = [c.q.copy(), c.k.copy(), c.v.copy()]
    for n, (g, a) in enumerate(zip(got, base)):
        d = rng.standard_normal(a.shape)
        vals = []
        for sign in (1, -1):
            c.q, c.k, c.v = (x + sign * 1e-5 * d if i == n else x for i, x in enumerate(base))
            vals.append((c.reference()[0] * c.do).sum())
        num = (vals[0] - vals[1]) / 2e-5
        # each of the terms carries about three roundings of half an ulp (probability or score
        # gradient, the saved output, the result), independent, so they add in squares; 8 sigma
        sd = 3 * U[F16] * np.sqrt(((g * d) ** 2).sum() + (np.abs(g).mean() * d ** 2).sum())
        assert abs((g * d).sum() - num) <= 8 * sd + 1e-6 * abs(num), (n, num, sd)


def test_attention_zero_sizes(gpu):
    from omnimatchdeeplearningtool_b200._lib import call
    st12, st24 = (ctypes.c_longlong * 12)(*[64] * 12), (ctypes.c_longlong * 24)(*[64] * 24)
    # no batch, no queries: nothing to do
    call("omCudaAttention", None, None, None, None, None, st12, None, None, None, 0, 1, 1, 4, 4, 64, 1.0, 0, BF16)
    k = _dev(np.ones((1, 4, 1, 64)), BF16)
    call("omCudaAttention", None, k.ptr, k.ptr, None, None, st12, None, None, None, 1, 1, 1, 0, 4, 64, 1.0, 0, BF16)
    # no keys: zeros, minus infinity; and zero gradients on either side
    q, out, ls, ws = _dev(np.ones((1, 4, 1, 64)), BF16), _new(512), _new(16), _new(1 << 16)
    call("omCudaAttention", q.ptr, None, None, out.ptr, ls.ptr, st12, None, None, ws.ptr, 1, 1, 1, 4, 0, 64, 1.0, 0, BF16)
    assert (_get(out, (4, 64), BF16) == 0).all() and np.isneginf(ls.to_numpy((4,))).all()
    g = _new(512)
    call("omCudaAttentionBackward", q.ptr, q.ptr, None, None, out.ptr, ls.ptr, g.ptr, None, None, st24, None, None, ws.ptr,
         1, 1, 1, 4, 0, 64, 1.0, 0, BF16)
    assert (_get(g, (4, 64), BF16) == 0).all()
    g1, g2 = _new(512), _new(512)
    call("omCudaAttentionBackward", None, None, k.ptr, k.ptr, None, None, None, g1.ptr, g2.ptr, st24, None, None, ws.ptr,
         1, 1, 1, 0, 4, 64, 1.0, 0, BF16)
    assert (_get(g1, (4, 64), BF16) == 0).all() and (_get(g2, (4, 64), BF16) == 0).all()


def test_attention_refusals(gpu):
    from omnimatchdeeplearningtool_b200._lib import lib
    b, ws = _new(1 << 16), _new(1 << 20)
    good = [256, 64, 64] * 8

    def f(q=b.ptr, k=b.ptr, v=b.ptr, o=b.ptr, st=good, bt=1, h=1, hkv=1, sq=4, sk=4, d=64, dt=BF16):
        arr = (ctypes.c_longlong * 12)(*st[:12]) if st else None
        return lib.omCudaAttention(q, k, v, o, None, arr, None, None, ws.ptr, bt, h, hkv, sq, sk, d, 1.0, 0, dt)

    assert f() == 0
    assert f(q=None) == -2 and f(k=None) == -2 and f(v=None) == -2 and f(o=None) == -2 and f(st=None) == -2
    assert f(q=b.ptr + 8) == -2 and f(h=3, hkv=2) == -2 and f(hkv=0) == -2 and f(sq=-1) == -2 and f(d=0) == -2
    for at in (1, 4, 7, 10):          # token strides: not a multiple of 8, zero, negative
        for bad in (68, 0, -64):
            st = list(good)
            st[at] = bad
            assert f(st=st) == -2
    assert f(d=60) == -3 and f(d=136) == -3 and f(dt=F32) == -3

    def g(lse=b.ptr, w=ws.ptr, dq=b.ptr, dt=BF16, st=good):
        arr = (ctypes.c_longlong * 24)(*st)
        return lib.omCudaAttentionBackward(b.ptr, b.ptr, b.ptr, b.ptr, b.ptr, lse, dq, b.ptr + 4096, b.ptr + 8192, arr,
                                           None, None, w, 1, 1, 1, 4, 4, 64, 1.0, 0, dt)

    assert g(dq=b.ptr + 16384) == 0
    assert g(lse=None) == -2 and g(w=None) == -2 and g(w=ws.ptr + 4) == -2 and g(dq=None) == -2 and g(dt=F32) == -3
    assert g(st=good[:22] + [60] + good[23:]) == -2


def test_attention_long_offsets(gpu):
    """A token stride so long that the last tokens lie past 2^31 elements of the allocation."""
    from omnimatchdeeplearningtool_b200._lib import call
    from omnimatchdeeplearningtool_b200.backend import DeviceBuffer
    sq, sk, d, gap = 3, 200, 64, 11_000_000      # (sk - 1) * gap > 2^31
    c = _Case(1, 1, 1, sq, sk, d, BF16)
    big = DeviceBuffer(((sk - 1) * gap + d) * 2)
    host = to_bits(c.k[0, :, 0], BF16)
    for j in range(sk):
        call("omCudaCopyH2D", big.ptr + j * gap * 2, host[j].ctypes.data, d * 2)
    out, ls = _new(sq * d * 2), _new(sq * 4)
    st = (ctypes.c_longlong * 12)(sq * d, d, d, sk * gap, gap, d, sk * d, d, d, sq * d, d, d)
    call("omCudaAttention", c.dq_.ptr, big.ptr, c.dv_.ptr, out.ptr, ls.ptr, st, None, None, c.ws(0).ptr, 1, 1, 1, sq, sk, d,
         float(c.scale), 0, BF16)
    o, lse = c.forward()
    assert (c.read(out, sq, 1) == o).all() and (ls.to_numpy((1, 1, sq)) == lse).all()
    big.free()
