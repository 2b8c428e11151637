"""The channels-last attention-block operators, as a user calls them and in their plain form.

Three operators, each with its backward: GroupNorm with an activation on NHWC maps, attention
whose backward recomputes the probabilities, and dropout (with the residual add) from a
counter-based generator. With ``own`` false, ``run`` computes them with elementary torch
operations in 32 bits; with ``own`` true it calls the library's entry points.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}          # OM_DTYPE_*
ACTS = {"none": 0, "relu": 1, "relu6": 2, "silu": 3}  # OM_ACT_*
EPS = 1e-5


def listed():
    return [
        # the last stage of an image classifier at batch 1: latency of one small call
        dict(name="gn_fwd_head", op="gn_fwd", n=1, hw=49, c=512, cs=512, groups=32, act="silu", dtype="bf16"),
        # a 56x56 stage at serving batch: bandwidth
        dict(name="gn_fwd_stage", op="gn_fwd", n=64, hw=3136, c=256, cs=256, groups=32, act="silu", dtype="bf16"),
        # a 37x53 crop with 180 channels stored as 184, groups of 15 channels
        dict(name="gn_bwd_odd", op="gn_bwd", n=5, hw=1961, c=180, cs=184, groups=12, act="relu", dtype="f16"),
        # fp32 training of a 112x112 stage
        dict(name="gn_bwd_stage", op="gn_bwd", n=16, hw=12544, c=64, cs=64, groups=16, act="silu", dtype="f32"),
        # the tokens of one image behind a projection, with the residual
        dict(name="drop_fwd_tokens", op="drop_fwd", n=197 * 768, p=0.1, residual=True, dtype="bf16"),
        # the gradient of a training batch of token maps, an odd count
        dict(name="drop_bwd_batch", op="drop_bwd", n=64 * 1025 * 768 + 3, p=0.2, residual=False, dtype="f16"),
        # a few prompt tokens reading the tokens of a 64x64 feature map
        dict(name="attn_fwd_prompts", op="attn_fwd", b=2, h=8, hkv=8, sq=7, sk=4096, d=32, causal=False, lens="none",
             layout="bshd", dtype="bf16"),
        # 14x14 patches and a class token, a serving batch, on the packed projection output
        dict(name="attn_fwd_patches", op="attn_fwd", b=64, h=12, hkv=12, sq=197, sk=197, d=64, causal=False,
             lens="none", layout="packed", dtype="f16"),
        # a long causal sequence with shared key/value heads
        dict(name="attn_fwd_long", op="attn_fwd", b=1, h=16, hkv=4, sq=8192, sk=8192, d=128, causal=True,
             lens="none", layout="bhsd", dtype="bf16"),
        # training on 14x14 patches and a class token
        dict(name="attn_bwd_patches", op="attn_bwd", b=32, h=12, hkv=12, sq=197, sk=197, d=64, causal=False,
             lens="none", layout="packed", dtype="bf16"),
        # a padded batch of sequences of different lengths, one of them empty, shared heads
        dict(name="attn_bwd_ragged", op="attn_bwd", b=6, h=8, hkv=2, sq=777, sk=777, d=80, causal=True, lens="both",
             layout="bshd", dtype="f16"),
        # training on all the tokens of a 64x64 feature map
        dict(name="attn_bwd_image", op="attn_bwd", b=2, h=12, hkv=12, sq=4096, sk=4096, d=64, causal=False,
             lens="none", layout="packed", dtype="bf16"),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gn_fwd", "gn_bwd", "drop_fwd", "drop_bwd", "attn_fwd", "attn_fwd", "attn_bwd", "attn_bwd"])
    if op.startswith("gn"):
        groups = rng.choice([1, 4, 8, 12, 16, 32])
        cpg = _logint(rng, 1, max(1, 640 // groups))
        c = groups * cpg
        cs = -(-c // 8) * 8
        # 16 values a group at least: the gradient of a smaller group is next to nothing but rounding
        hw = _logint(rng, -(-16 // cpg), 16384)
        n = _logint(rng, 1, 64)
        while n > 1 and n * hw * cs > 12 * 1000 * 1000:
            n = -(-n // 2)
        return dict(op=op, n=n, hw=hw, c=c, cs=cs, groups=groups, act=rng.choice(["none", "relu", "relu6", "silu"]),
                    dtype=rng.choice(["f32", "bf16", "f16"]))
    if op.startswith("drop"):
        return dict(op=op, n=_logint(rng, 1000, 48 * 1000 * 1000), p=rng.choice([0.05, 0.1, 0.2, 0.3, 0.5]),
                    residual=op == "drop_fwd" and rng.random() < 0.6, dtype=rng.choice(["f32", "bf16", "f16"]))
    hkv = rng.choice([1, 2, 3, 4, 8, 12])
    h = hkv * rng.choice([1, 1, 1, 2, 4])
    d = rng.choice([16, 24, 32, 40, 64, 64, 80, 96, 128])
    layout = rng.choice(["bshd", "bhsd", "packed"]) if h == hkv else rng.choice(["bshd", "bhsd"])
    sk = _logint(rng, 1, 6000)
    kind = rng.choice(["self", "self", "few", "cross"])
    sq = sk if layout == "packed" or kind == "self" else _logint(rng, 1, 16) if kind == "few" else _logint(rng, 1, 6000)
    lens = rng.choice(["none", "none", "kv", "both"])
    b = _logint(rng, 1, 32)
    # no more score entries than the largest listed case of the same direction has
    most = 250e6 if op == "attn_fwd" else 200e6
    while b > 1 and b * h * sq * sk > most:
        b = -(-b // 2)
    if b * h * sq * sk > most:
        sq = max(1, int(most / (b * h * sk)))
        layout = "bshd" if layout == "packed" else layout
    return dict(op=op, b=b, h=h, hkv=hkv, sq=sq, sk=sk, d=d, causal=rng.random() < 0.4, lens=lens, layout=layout,
                dtype=rng.choice(["bf16", "f16"]))


# ---------------------------------------------------------------- the cases' lengths and work
def _lengths(case):
    """Per batch entry: (query tokens, key tokens) in use, by a fixed pattern that has full,
    partial and empty entries."""
    share = [0.63, 1.0, 0.31, 0.0, 0.87, 0.52]
    got = []
    for i in range(case["b"]):
        f = share[i % 6]
        kl = int(math.ceil(case["sk"] * f)) if case["lens"] != "none" else case["sk"]
        ql = int(math.ceil(case["sq"] * f)) if case["lens"] == "both" else case["sq"]
        got.append((ql, kl))
    return got


def _pairs(case):
    """Visible (query, key) pairs of one head over the batch."""
    total = 0
    for ql, kl in _lengths(case):
        if not case["causal"]:
            total += ql * kl
        else:  # query i sees keys j <= i + kl - ql
            first = max(0, ql - kl)
            n = ql - first
            top = kl - n + 1  # keys that the first seeing query sees
            total += n * top + n * (n - 1) // 2 if n > 0 else 0
    return total


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    op = case["op"]
    if op.startswith("gn"):
        e = case["n"] * case["hw"] * case["cs"]
        small = case["n"] * case["groups"] * 8 + case["c"] * 8
        if op == "gn_fwd":
            return {"bytes": 2 * e * size + small, "flops": 12 * e}
        return {"bytes": 3 * e * size + small + case["c"] * 8, "flops": 25 * e}
    if op.startswith("drop"):
        return {"bytes": case["n"] * size * (3 if case["residual"] else 2), "flops": 2 * case["n"]}
    ql, kl = (sum(x) for x in zip(*_lengths(case)))
    h, hkv, d = case["h"], case["hkv"], case["d"]
    q_side, kv_side = case["b"] * case["sq"] * h * d * size, case["b"] * case["sk"] * hkv * d * size
    q_read, kv_read = ql * h * d * size, kl * hkv * d * size
    lse = case["b"] * case["sq"] * h * 4
    if op == "attn_fwd":
        return {"bytes": q_read + 2 * kv_read + q_side + lse, "flops": 4 * d * h * _pairs(case)}
    return {"bytes": 3 * q_read + 2 * kv_read + lse + q_side + 2 * kv_side, "flops": 10 * d * h * _pairs(case)}


# ---------------------------------------------------------------- inputs
def _heads(g, layout, b, s, h, d, dt):
    """A random [b, s, h, d] tensor in the layout's memory order."""
    if layout == "bhsd":
        return torch.randn((b, h, s, d), generator=g, device="cuda").to(dt).transpose(1, 2)
    return torch.randn((b, s, h, d), generator=g, device="cuda").to(dt)


def _empty_heads(layout, b, s, h, d, dt):
    if layout == "bhsd":
        return torch.empty((b, h, s, d), device="cuda", dtype=dt).transpose(1, 2)
    return torch.empty((b, s, h, d), device="cuda", dtype=dt)


def _strides(*tensors):
    """(batch, token, head) strides in elements, one triple per tensor, as the entry points take them."""
    import ctypes
    flat = [t.stride(i) for t in tensors for i in (0, 1, 2)]
    return (ctypes.c_longlong * len(flat))(*flat)


def _prepare_attention(case, g, dt):
    b, h, hkv, sq, sk, d = (case[k] for k in ("b", "h", "hkv", "sq", "sk", "d"))
    s = {}
    if case["layout"] == "packed":  # one projection's output [b, s, 3, h, d]
        qkv = torch.randn((b, sq, 3, h, d), generator=g, device="cuda").to(dt)
        s["q"], s["k"], s["v"] = qkv.unbind(2)
    else:
        s["q"] = _heads(g, case["layout"], b, sq, h, d, dt)
        s["k"] = _heads(g, case["layout"], b, sk, hkv, d, dt)
        s["v"] = _heads(g, case["layout"], b, sk, hkv, d, dt)
    s["scale"] = 1.5 / math.sqrt(d)  # trained heads are sharper than unit-variance scores
    lengths = _lengths(case)
    s["qlen"] = torch.tensor([x for x, _ in lengths], dtype=torch.int32, device="cuda") if case["lens"] == "both" else None
    s["klen"] = torch.tensor([y for _, y in lengths], dtype=torch.int32, device="cuda") if case["lens"] != "none" else None
    s["out"] = _empty_heads(case["layout"], b, sq, h, d, dt)
    if case["op"] == "attn_fwd":
        s["lse"] = torch.empty((b, h, sq), device="cuda")
        s["strides"] = _strides(s["q"], s["k"], s["v"], s["out"])
        return s
    # what a forward pass leaves for its backward, and the gradient that arrives
    o, s["lse"] = _plain_forward(dict(case=case, **s))
    s["out"].copy_(o)
    s["do"] = _heads(g, case["layout"], b, sq, h, d, dt)
    if case["layout"] == "packed":
        s["dq"], s["dk"], s["dv"] = torch.empty((b, sq, 3, h, d), device="cuda", dtype=dt).unbind(2)
    else:
        s["dq"] = _empty_heads(case["layout"], b, sq, h, d, dt)
        s["dk"] = _empty_heads(case["layout"], b, sk, hkv, d, dt)
        s["dv"] = _empty_heads(case["layout"], b, sk, hkv, d, dt)
    s["strides"] = _strides(*(s[k] for k in ("q", "k", "v", "out", "do", "dq", "dk", "dv")))
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"].startswith("attn"):
        return dict(case=case, **_prepare_attention(case, g, dt))
    if case["op"].startswith("drop"):
        n = case["n"]
        s = dict(case=case, x=torch.randn(n, generator=g, device="cuda").to(dt), out=torch.empty(n, device="cuda", dtype=dt))
        s["res"] = torch.randn(n, generator=g, device="cuda").to(dt) if case["residual"] else None
        # the run's random stream: a seed, and the training step's place in it
        s["rng"] = (0x9D2C5680_0000_0000 + seed * 0x10001, 3 + (seed << 20))
        return s
    n, hw, c, cs, groups = (case[k] for k in ("n", "hw", "c", "cs", "groups"))
    # a convolution's output: channels with their own offset and spread, stored padding zero
    x = torch.randn((n, hw, cs), generator=g, device="cuda")
    x = x * (0.5 + torch.rand(cs, generator=g, device="cuda")) + 0.5 * torch.randn(cs, generator=g, device="cuda") + 0.25
    x[:, :, c:] = 0
    s = dict(case=case, x=x.to(dt))
    s["gamma"] = 1 + 0.2 * torch.randn(c, generator=g, device="cuda")
    s["beta"] = 0.2 * torch.randn(c, generator=g, device="cuda")
    s["out"] = torch.empty((n, hw, cs), device="cuda", dtype=dt)
    s["mean"] = torch.empty((n, groups), device="cuda")
    s["rstd"] = torch.empty((n, groups), device="cuda")
    if case["op"] == "gn_bwd":
        xg = s["x"][:, :, :c].float().reshape(n, hw, groups, c // groups)
        s["mean"].copy_(xg.mean((1, 3)))
        s["rstd"].copy_((xg.var((1, 3), unbiased=False) + EPS).rsqrt())
        s["dy"] = torch.randn((n, hw, cs), generator=g, device="cuda").to(dt)
        s["dgamma"] = torch.empty(c, device="cuda")
        s["dbeta"] = torch.empty(c, device="cuda")
    return s


# ---------------------------------------------------------------- plain forms
def _plain_group_norm(s):
    case = s["case"]
    n, hw, c, cs, groups = (case[k] for k in ("n", "hw", "c", "cs", "groups"))
    x = s["x"][:, :, :c].float().reshape(n, hw, groups, c // groups)
    mean = x.mean((1, 3))
    rstd = (((x - mean[:, None, :, None]) ** 2).mean((1, 3)) + EPS).rsqrt()
    z = ((x - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(n, hw, c) * s["gamma"] + s["beta"]
    if case["act"] == "relu":
        z = torch.where(z > 0, z, torch.zeros_like(z))
    elif case["act"] == "relu6":
        z = torch.minimum(torch.where(z > 0, z, torch.zeros_like(z)), torch.full_like(z, 6.0))
    elif case["act"] == "silu":
        z = z / (1 + torch.exp(-z))
    out = torch.zeros((n, hw, cs), device="cuda", dtype=s["x"].dtype)
    out[:, :, :c] = z.to(out.dtype)
    return {"out": out, "mean": mean, "rstd": rstd}


def _plain_group_norm_backward(s):
    case = s["case"]
    n, hw, c, cs, groups = (case[k] for k in ("n", "hw", "c", "cs", "groups"))
    x = s["x"][:, :, :c].float().reshape(n, hw, groups, c // groups)
    rstd = s["rstd"][:, None, :, None]
    xh = ((x - s["mean"][:, None, :, None]) * rstd).reshape(n, hw, c)
    z = xh * s["gamma"] + s["beta"]
    dz = s["dy"][:, :, :c].float()
    if case["act"] == "relu":
        dz = torch.where(z > 0, dz, torch.zeros_like(dz))
    elif case["act"] == "relu6":
        dz = torch.where((z > 0) & (z < 6), dz, torch.zeros_like(dz))
    elif case["act"] == "silu":
        sig = 1 / (1 + torch.exp(-z))
        dz = dz * sig * (1 + z * (1 - sig))
    dbeta = dz.sum((0, 1))
    dgamma = (dz * xh).sum((0, 1))
    t = (dz * s["gamma"]).reshape(n, hw, groups, c // groups)
    xh = xh.reshape(n, hw, groups, c // groups)
    m1 = t.mean((1, 3), keepdim=True)
    m2 = (t * xh).mean((1, 3), keepdim=True)
    dx = torch.zeros((n, hw, cs), device="cuda", dtype=s["x"].dtype)
    dx[:, :, :c] = (rstd * (t - m1 - xh * m2)).reshape(n, hw, c).to(dx.dtype)
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _plain_dropout(s):
    """Element i takes 16 bits of Philox4x32-10 (Salmon et al., 2011) at counter (i // 8, offset)
    and key seed: bits 16 * (i % 2) up of word (i % 8) // 2. It is kept where they are at least
    T = round(65536 p), and multiplied by 65536 / (65536 - T)."""
    n = s["case"]["n"]
    seed, offset = s["rng"]
    low = 0xFFFFFFFF
    i = torch.arange(-(-n // 8), device="cuda", dtype=torch.int64)
    c0, c1 = i & low, i >> 32
    c2, c3 = torch.full_like(i, offset & low), torch.full_like(i, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], 1)
    bits = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]
    t = int(s["case"]["p"] * 65536 + 0.5)
    y = torch.where(bits >= t, s["x"].float() * (65536.0 / (65536 - t)), torch.zeros((), device="cuda"))
    if s["res"] is not None:
        y = y + s["res"].float()
    return {"out": y.to(s["x"].dtype)}


def _scores(s):
    """fp32 scores [b, h, sq, sk], minus infinity where a query does not see a key."""
    case = s["case"]
    rep = case["h"] // case["hkv"]
    q, k, v = (s[x].float().transpose(1, 2) for x in ("q", "k", "v"))
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    a = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    i = torch.arange(case["sq"], device="cuda")[None, None, :, None]
    j = torch.arange(case["sk"], device="cuda")[None, None, None, :]
    ql = s["qlen"].reshape(-1, 1, 1, 1) if s["qlen"] is not None else case["sq"]
    kl = s["klen"].reshape(-1, 1, 1, 1) if s["klen"] is not None else case["sk"]
    if case["causal"] or s["klen"] is not None:
        seen = (i < ql) & (j < kl)
        if case["causal"]:
            seen = seen & (j <= i + kl - ql)
        a = torch.where(seen, a, torch.full((), -math.inf, device="cuda"))
    return q, k, v, a


def _plain_forward(s):
    q, k, v, a = _scores(s)
    m = a.amax(3, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(a - m)
    del a
    total = p.sum(3, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return o.transpose(1, 2).to(s["q"].dtype), (m + torch.log(total)).squeeze(3)


def _plain_backward(s):
    case = s["case"]
    q, k, v, a = _scores(s)
    o, do = s["out"].float().transpose(1, 2), s["do"].float().transpose(1, 2)
    lse = torch.where(torch.isinf(s["lse"]), torch.zeros_like(s["lse"]), s["lse"])[..., None]
    p = torch.exp(a - lse)
    del a
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(3, keepdim=True)) * s["scale"]
    del p
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q)
    dk, dv = (t.reshape(case["b"], case["hkv"], -1, case["sk"], case["d"]).sum(2) for t in (dk, dv))
    dt = s["q"].dtype
    return {"dq": dq.transpose(1, 2).to(dt), "dk": dk.transpose(1, 2).to(dt), "dv": dv.transpose(1, 2).to(dt)}


# ---------------------------------------------------------------- the library's calls
def _ptr(t):
    return t.data_ptr() if t is not None else None


def _library(s):
    """The entry points, initialised for this thread, and this state's workspace."""
    from omnimatchdeeplearningtool_b200 import backend
    from omnimatchdeeplearningtool_b200._lib import call, lib
    if "ws" not in s:
        if lib.omCudaGetCurrentDevice() < 0:
            backend.init(torch.cuda.current_device())
        case = s["case"]
        backward = case["op"].endswith("bwd")
        if case["op"].startswith("gn"):
            nbytes = lib.omCudaGroupNormNhwcWorkspaceBytes(case["n"], case["hw"], case["c"], case["cs"], case["groups"],
                                                           CODES[case["dtype"]], backward)
        elif case["op"].startswith("attn"):
            nbytes = lib.omCudaAttentionWorkspaceBytes(case["b"], case["h"], case["hkv"], case["sq"], case["sk"],
                                                       case["d"], backward)
        else:
            nbytes = 0
        s["ws"] = torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device="cuda")
    return call


def _own(s):
    call, case = _library(s), s["case"]
    op, code = case["op"], CODES[case["dtype"]]
    if op == "gn_fwd":
        call("omCudaGroupNormActNhwc", _ptr(s["x"]), _ptr(s["out"]), _ptr(s["gamma"]), _ptr(s["beta"]), _ptr(s["mean"]),
             _ptr(s["rstd"]), _ptr(s["ws"]), case["n"], case["hw"], case["c"], case["cs"], case["groups"], EPS,
             ACTS[case["act"]], code)
        return {"out": s["out"], "mean": s["mean"], "rstd": s["rstd"]}
    if op == "gn_bwd":
        call("omCudaGroupNormActNhwcBackward", _ptr(s["dy"]), _ptr(s["x"]), _ptr(s["mean"]), _ptr(s["rstd"]),
             _ptr(s["gamma"]), _ptr(s["beta"]), _ptr(s["out"]), _ptr(s["dgamma"]), _ptr(s["dbeta"]), _ptr(s["ws"]),
             case["n"], case["hw"], case["c"], case["cs"], case["groups"], ACTS[case["act"]], code)
        return {"dx": s["out"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}
    if op.startswith("drop"):
        # the backward pass is the same call on the gradient
        call("omCudaDropoutAdd", _ptr(s["x"]), _ptr(s["res"]), _ptr(s["out"]), case["n"], case["p"], s["rng"][0],
             s["rng"][1], code)
        return {"out": s["out"]}
    sizes = (case["b"], case["h"], case["hkv"], case["sq"], case["sk"], case["d"], s["scale"], case["causal"], code)
    if op == "attn_fwd":
        call("omCudaAttention", _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["out"]), _ptr(s["lse"]), s["strides"],
             _ptr(s["qlen"]), _ptr(s["klen"]), _ptr(s["ws"]), *sizes)
        return {"out": s["out"], "lse": s["lse"]}
    call("omCudaAttentionBackward", _ptr(s["do"]), _ptr(s["q"]), _ptr(s["k"]), _ptr(s["v"]), _ptr(s["out"]),
         _ptr(s["lse"]), _ptr(s["dq"]), _ptr(s["dk"]), _ptr(s["dv"]), s["strides"], _ptr(s["qlen"]), _ptr(s["klen"]),
         _ptr(s["ws"]), *sizes)
    return {"dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "gn_fwd":
        return _plain_group_norm(state)
    if op == "gn_bwd":
        return _plain_group_norm_backward(state)
    if op.startswith("drop"):
        return _plain_dropout(state)
    if op == "attn_fwd":
        out, lse = _plain_forward(state)
        return {"out": out, "lse": lse}
    return _plain_backward(state)


# ---------------------------------------------------------------- 64 bits
def _exact_group_norm(case, s):
    c = case["c"]
    x = s["x"][:, :, :c].double().transpose(1, 2).requires_grad_()
    gamma, beta = s["gamma"].double().requires_grad_(), s["beta"].double().requires_grad_()
    z = torch.nn.functional.group_norm(x, case["groups"], gamma, beta, EPS)
    f = torch.nn.functional
    y = {"none": lambda t: t, "relu": f.relu, "relu6": f.relu6, "silu": f.silu}[case["act"]](z)
    pad = (0, case["cs"] - c)
    if case["op"] == "gn_fwd":
        xg = x.detach().reshape(case["n"], case["groups"], -1)
        return {"out": f.pad(y.detach().transpose(1, 2), pad), "mean": xg.mean(2),
                "rstd": 1 / torch.sqrt(xg.var(2, unbiased=False) + EPS)}
    dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), s["dy"][:, :, :c].double().transpose(1, 2))
    return {"dx": f.pad(dx.transpose(1, 2), pad), "dgamma": dgamma, "dbeta": dbeta}


def _exact_dropout(case, s):
    n, (seed, offset) = case["n"], s["rng"]
    u = np.uint64
    low, half = u(0xFFFFFFFF), u(32)
    i = np.arange((n + 7) // 8, dtype=u)
    c = [i & low, i >> half, np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ u(key[0]), b & low, (a >> half) ^ c[3] ^ u(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.stack(c, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    t = int(case["p"] * 65536 + 0.5)
    y = np.where(bits >= t, s["x"].double().cpu().numpy() * (65536.0 / (65536 - t)), 0.0)
    return {"out": y + s["res"].double().cpu().numpy() if s["res"] is not None else y}


def _exact_attention(case, s):
    """Head by head through autograd, on the queries that see a key."""
    b, h, hkv, sq, sk, d = (case[k] for k in ("b", "h", "hkv", "sq", "sk", "d"))
    backward = case["op"] == "attn_bwd"
    z = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out, lse = z(b, sq, h, d), torch.full((b, h, sq), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = z(b, sq, h, d), z(b, sk, hkv, d), z(b, sk, hkv, d)
    per = max(1, int(100e6 / max(1, sq * sk)))  # heads at a time
    for i, (ql, kl) in enumerate(_lengths(case)):
        first = max(0, ql - kl) if case["causal"] else 0
        if kl == 0 or first >= ql:
            continue
        for at in range(0, h, per):
            hs = torch.arange(at, min(h, at + per), device="cuda")
            ks = hs // (h // hkv)
            q = s["q"][i, first:ql][:, hs].double().transpose(0, 1).requires_grad_(backward)
            k = s["k"][i, :kl][:, ks].double().transpose(0, 1).requires_grad_(backward)
            v = s["v"][i, :kl][:, ks].double().transpose(0, 1).requires_grad_(backward)
            a = (q @ k.transpose(1, 2)) * s["scale"]
            if case["causal"]:
                hide = torch.ones(ql - first, kl, dtype=torch.bool, device="cuda").triu(kl - (ql - first) + 1)
                a = a.masked_fill(hide, -math.inf)
            o = torch.softmax(a, 2) @ v
            if not backward:
                out[i, first:ql, hs] = o.transpose(0, 1)
                lse[i, hs, first:ql] = torch.logsumexp(a, 2)
                continue
            g = torch.autograd.grad(o, (q, k, v), s["do"][i, first:ql][:, hs].double().transpose(0, 1))
            dq[i, first:ql, hs] = g[0].transpose(0, 1)
            dk[i, :kl].index_add_(1, ks, g[1].transpose(0, 1))
            dv[i, :kl].index_add_(1, ks, g[2].transpose(0, 1))
    return {"dq": dq, "dk": dk, "dv": dv} if backward else {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("gn"):
        return _exact_group_norm(case, s)
    if case["op"].startswith("drop"):
        return _exact_dropout(case, s)
    return _exact_attention(case, s)
