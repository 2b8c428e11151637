"""A self-attention block on channels-last maps, forward and backward.

The block that the engine's vision transformers and attention U-Nets put between their
convolutions, on the fused path's NHWC 16-bit storage, where an [N, H, W, C] map is the token
matrix [N, H*W, C]:

    h   = act(GroupNorm(x))            omCudaGroupNormActNhwc
    qkv = h Wqkv + bqkv                omCudaConv2dBnAct (1x1)          [N, H*W, 3, heads, C/heads]
    a   = attention(q, k, v)           omCudaAttention, on qkv in place
    y   = a Wo + bo                    omCudaConv2dBnAct (1x1)
    out = x + dropout(y)               omCudaDropoutAdd

and the same calls' backward in reverse. Nothing is stored for the backward but the activations,
the group statistics and one log-sum-exp a query: attention's probabilities and the dropout mask
are worked out again. Weight gradients take the fp32 weight-gradient kernel.

All calls go to the library's compute stream; results are device buffers.
"""
from __future__ import annotations

import ctypes
import itertools
from typing import Dict, List, Optional

import numpy as np

from ._lib import ACT_NONE, ACT_SILU, DTYPE_BF16, DTYPE_F16, call, lib
from .backend import DeviceBuffer

DTYPES = {"bf16": DTYPE_BF16, "fp16": DTYPE_F16}


class AttentionBlock:
    """``params``: host arrays gamma, beta [C], w_qkv [3C, C], b_qkv [3C], w_out [C, C], b_out [C]
    (rows are output channels, as conv weights [Cout, Cin, 1, 1]).

    The dropout mask is that of ``seed`` and the step that :meth:`forward` is given. A model's blocks
    need seeds of their own, since two blocks with one seed drop the same elements in a step; a block
    that is given none takes the next number of its process."""

    _seeds = itertools.count()

    def __init__(self, n: int, h: int, w: int, c: int, heads: int, groups: int,
                 params: Dict[str, np.ndarray], dtype: str = "bf16", dropout: float = 0.0,
                 seed: Optional[int] = None, eps: float = 1e-5, act: int = ACT_SILU):
        if dtype not in DTYPES:
            raise ValueError(f"dtype must be one of {sorted(DTYPES)}")
        if min(n, h, w, c, heads, groups) < 1:
            raise ValueError("sizes must be positive")
        if c % heads or (c // heads) % 8 or c // heads > 128 or c % groups:
            raise ValueError("channels must split into groups, and into heads of 8 .. 128 channels "
                             "(a multiple of 8)")
        if lib.omCudaStoredChannels(c) != c:
            raise ValueError("channels must be stored without padding (a multiple of 8)")
        for name, count in (("gamma", c), ("beta", c), ("w_qkv", 3 * c * c), ("b_qkv", 3 * c), ("w_out", c * c),
                            ("b_out", c)):
            if name not in params or np.size(params[name]) != count:
                raise ValueError(f"parameter {name} must be there, with {count} values")
        self.n, self.h, self.w, self.c = n, h, w, c
        self.heads, self.groups, self.d, self.tokens = heads, groups, c // heads, h * w
        self.dt, self.p, self.eps, self.act = DTYPES[dtype], dropout, eps, act
        self.seed = next(AttentionBlock._seeds) if seed is None else seed
        self.scale = 1.0 / float(np.sqrt(self.d))
        self._keep: List[DeviceBuffer] = []
        self.params = {k: self._dev(v) for k, v in params.items()}
        self._pack()
        m = n * self.tokens
        self.hid, self.att, self.out = (self._buf(m * c * 2) for _ in range(3))
        self.qkv = self._buf(m * 3 * c * 2)
        self.mean, self.rstd = (self._buf(n * groups * 4) for _ in range(2))
        self.lse = self._buf(n * heads * self.tokens * 4)
        dims = (n, heads, heads, self.tokens, self.tokens, self.d)
        self.dims = dims
        need = [lib.omCudaAttentionWorkspaceBytes(*dims, b) for b in (0, 1)]
        need += [lib.omCudaGroupNormNhwcWorkspaceBytes(n, self.tokens, c, c, groups, self.dt, b)
                 for b in (0, 1)]
        self.ws = self._buf(max(need + [16]))
        third, one = (self.tokens * 3 * c, 3 * c, self.d), (self.tokens * c, c, self.d)
        self._fwd_strides = (ctypes.c_longlong * 12)(*third, *third, *third, *one)
        self._bwd_strides = (ctypes.c_longlong * 24)(*third, *third, *third, *one, *one,
                                                     *third, *third, *third)
        self._grads: Dict[str, DeviceBuffer] = {}
        self.step, self.step_ptr = -1, None

    # ------------------------------------------------------------------ buffers
    def _dev(self, a: np.ndarray) -> DeviceBuffer:
        b = DeviceBuffer.from_numpy(np.ascontiguousarray(a, np.float32))
        self._keep.append(b)
        return b

    def _buf(self, nbytes: int) -> DeviceBuffer:
        b = DeviceBuffer(int(nbytes))
        self._keep.append(b)
        return b

    def close(self) -> None:
        for b in self._keep:
            b.free()
        self._keep.clear()

    def _pack_one(self, weight: DeviceBuffer, bias, cout: int, cin: int):
        packed = self._buf(int(lib.omCudaPackedConvWeightElems(cout, 1, 1, cin)) * 2)
        b = self._buf(cout * 4)
        call("omCudaPackConvWeight", weight.ptr, bias.ptr if bias else None, None, None, None, None,
             self.eps, packed.ptr, b.ptr, cout, cin, 1, 1, cin, self.dt)
        return packed, b

    def _pack(self) -> None:
        """The projections' weights for the forward, and transposed for the backward."""
        c, p = self.c, self.params
        self.pk_qkv = self._pack_one(p["w_qkv"], p["b_qkv"], 3 * c, c)
        self.pk_out = self._pack_one(p["w_out"], p["b_out"], c, c)
        t_qkv, t_out = self._buf(3 * c * c * 4), self._buf(c * c * 4)
        call("omCudaTranspose", p["w_qkv"].ptr, t_qkv.ptr, 3 * c, c)
        call("omCudaTranspose", p["w_out"].ptr, t_out.ptr, c, c)
        self.pk_qkv_t = self._pack_one(t_qkv, None, c, 3 * c)
        self.pk_out_t = self._pack_one(t_out, None, c, c)

    def _project(self, x: int, packed, y: int, cin: int, cout: int) -> None:
        call("omCudaConv2dBnAct", x, packed[0].ptr, packed[1].ptr, None, y, self.n, self.h, self.w,
             cin, cout, 1, 1, 1, 0, ACT_NONE, self.dt, self.dt)

    def _qkv_ptrs(self, base: int):
        return [base + i * self.c * 2 for i in range(3)]

    # ------------------------------------------------------------------ passes
    def forward(self, x: int, step: Optional[int] = None, step_ptr: Optional[int] = None) -> int:
        """``x``: device pointer of the [N, H, W, C] map, which stays until the backward; returns the
        output's. ``step`` selects the dropout mask: without one, the step after the last call's, the
        first call's being 0. ``step_ptr``: device pointer of a 64-bit number to be added to it (then 0
        without one), read when the pass and its backward run; a captured pass needs it to draw new
        masks on its replays."""
        n, t, c = self.n, self.tokens, self.c
        if step is None:
            step = 0 if step_ptr else self.step + 1
        self.x, self.step, self.step_ptr = x, step, step_ptr
        call("omCudaGroupNormActNhwc", x, self.hid.ptr, self.params["gamma"].ptr,
             self.params["beta"].ptr, self.mean.ptr, self.rstd.ptr, self.ws.ptr, n, t, c, c,
             self.groups, self.eps, self.act, self.dt)
        self._project(self.hid.ptr, self.pk_qkv, self.qkv.ptr, c, 3 * c)
        call("omCudaAttention", *self._qkv_ptrs(self.qkv.ptr), self.att.ptr, self.lse.ptr,
             self._fwd_strides, None, None, self.ws.ptr, *self.dims, self.scale, 0, self.dt)
        self._project(self.att.ptr, self.pk_out, self.out.ptr, c, c)
        self._dropout(self.out.ptr, x, self.out.ptr)
        return self.out.ptr

    def _dropout(self, x: int, residual: Optional[int], out: int) -> None:
        count = self.n * self.tokens * self.c
        if self.step_ptr:
            call("omCudaDropoutAddStep", x, residual, out, count, self.p, self.seed, self.step, self.step_ptr, self.dt)
        else:
            call("omCudaDropoutAdd", x, residual, out, count, self.p, self.seed, self.step, self.dt)

    def _weight_grad(self, x: DeviceBuffer, dy: DeviceBuffer, cin: int, cout: int, dw, db) -> None:
        """dW [cout, cin] and db from channels-last 16-bit tensors, in fp32."""
        n, h, w = self.n, self.h, self.w
        x32, dy32 = self._scratch("x32", n * h * w * cin * 4), self._scratch("dy32", n * h * w * cout * 4)
        call("omCudaNhwcToNchw", x.ptr, x32.ptr, n, cin, h, w, cin, self.dt)
        call("omCudaNhwcToNchw", dy.ptr, dy32.ptr, n, cout, h, w, cout, self.dt)
        call("omCudaConv2dBackwardWeight", x32.ptr, dy32.ptr, dw.ptr, db.ptr, n, cin, h, w, cout, 1,
             1, 1, 0)

    def _scratch(self, name: str, nbytes: int) -> DeviceBuffer:
        b = self._grads.get(name)
        if b is None or b.nbytes < nbytes:
            b = self._grads[name] = self._buf(nbytes)
        return b

    def backward(self, dout: int) -> Dict[str, DeviceBuffer]:
        """Gradients of the last forward pass from the output's: x (in the map's dtype), and gamma,
        beta, w_qkv, b_qkv, w_out, b_out in fp32."""
        n, t, c = self.n, self.tokens, self.c
        m, g = n * t, self._scratch
        dy, datt, dhid, dx = (g(k, m * c * 2) for k in ("dy", "datt", "dhid", "x"))
        dqkv = g("dqkv", m * 3 * c * 2)
        grads = {"x": dx, "gamma": g("gamma", c * 4), "beta": g("beta", c * 4),
                 "w_qkv": g("w_qkv", 3 * c * c * 4), "b_qkv": g("b_qkv", 3 * c * 4),
                 "w_out": g("w_out", c * c * 4), "b_out": g("b_out", c * 4)}
        self._dropout(dout, None, dy.ptr)
        self._weight_grad(self.att, dy, c, c, grads["w_out"], grads["b_out"])
        self._project(dy.ptr, self.pk_out_t, datt.ptr, c, c)
        call("omCudaAttentionBackward", datt.ptr, *self._qkv_ptrs(self.qkv.ptr), self.att.ptr,
             self.lse.ptr, *self._qkv_ptrs(dqkv.ptr), self._bwd_strides, None, None, self.ws.ptr,
             *self.dims, self.scale, 0, self.dt)
        self._weight_grad(self.hid, dqkv, c, 3 * c, grads["w_qkv"], grads["b_qkv"])
        self._project(dqkv.ptr, self.pk_qkv_t, dhid.ptr, 3 * c, c)
        call("omCudaGroupNormActNhwcBackward", dhid.ptr, self.x, self.mean.ptr, self.rstd.ptr,
             self.params["gamma"].ptr, self.params["beta"].ptr, dx.ptr, grads["gamma"].ptr,
             grads["beta"].ptr, self.ws.ptr, n, t, c, c, self.groups, self.act, self.dt)
        call("omCudaAddActNhwc", dx.ptr, dout, dx.ptr, m * c, ACT_NONE, self.dt)   # the residual's
        return grads
