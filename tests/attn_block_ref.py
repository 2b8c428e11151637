"""64-bit references of the channels-last attention-block operators, and 16-bit helpers.

Every function works in float64 on the values the device holds (16-bit inputs are rounded
first), so a difference from the device is the device's own rounding.
"""
import numpy as np

U = {0: 2.0 ** -24, 1: 2.0 ** -8, 2: 2.0 ** -11}   # unit roundoff (half an ulp of 1): 24, 8, 11 significant bits


def to_bits(a, dtype):
    """Device representation of a float array: float32, bf16 bits (uint16) or float16."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == 0:
        return a
    if dtype == 2:
        return a.astype(np.float16)
    u = a.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def from_bits(a, dtype):
    if dtype == 1:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def rounded(a, dtype):
    return from_bits(to_bits(a, dtype), dtype)


def np_type(dtype):
    return {0: np.float32, 1: np.uint16, 2: np.float16}[dtype]


# ---------------------------------------------------------------- GroupNorm + activation
def act(z, kind):
    if kind == 1:
        return np.maximum(z, 0)
    if kind == 2:
        return np.clip(z, 0, 6)
    if kind == 3:
        return z / (1 + np.exp(-z))
    return z


def act_grad(z, kind):
    if kind == 1:
        return (z > 0).astype(np.float64)
    if kind == 2:
        return ((z > 0) & (z < 6)).astype(np.float64)
    if kind == 3:
        s = 1 / (1 + np.exp(-z))
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


def group_norm(x, gamma, beta, groups, eps, kind):
    """x [n, hw, c] -> y, mean [n, g], rstd [n, g], z (the pre-activation), xhat."""
    n, hw, c = x.shape
    xg = x.reshape(n, hw, groups, c // groups)
    mean = xg.mean((1, 3))
    rstd = 1 / np.sqrt(((xg - mean[:, None, :, None]) ** 2).mean((1, 3)) + eps)
    xh = ((xg - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(n, hw, c)
    z = xh * gamma + beta
    return act(z, kind), mean, rstd, z, xh


def group_norm_backward(dy, z, xh, rstd, gamma, groups, kind):
    """dx, dgamma, dbeta, and the scale of dx before its cancellation, [n, 1, c]."""
    n, hw, c = dy.shape
    dz = dy * act_grad(z, kind)
    t = (dz * gamma).reshape(n, hw, groups, c // groups)
    xg = xh.reshape(t.shape)
    m1 = t.mean((1, 3), keepdims=True)
    m2 = (t * xg).mean((1, 3), keepdims=True)
    r = rstd[:, None, :, None]
    dx = (r * (t - m1 - xg * m2)).reshape(n, hw, c)
    size = (r * (np.abs(t) + np.abs(m1) + np.abs(xg) * (np.abs(t * xg).mean((1, 3), keepdims=True))))
    return dx, (dz * xh).sum((0, 1)), dz.sum((0, 1)), size.reshape(n, hw, c), dz


# ---------------------------------------------------------------- dropout
def philox(counter, offset, seed):
    """Philox4x32-10 words [len(counter), 4] in Python integers, from the published round."""
    out = []
    for c in counter:
        x = [c & 0xFFFFFFFF, c >> 32, offset & 0xFFFFFFFF, offset >> 32]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            a, b = 0xD2511F53 * x[0], 0xCD9E8D57 * x[2]
            x = [(b >> 32) ^ x[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ x[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        out.append(x)
    return np.array(out, np.uint64)


def keep_mask(n, p, seed, offset, first=0):
    """Which of elements first .. first + n - 1 are kept (first a multiple of 8), and the scale."""
    t = int(p * 65536 + 0.5)
    words = philox(range(first // 8, (first + n + 7) // 8), offset, seed)
    bits = np.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]
    return bits >= t, 65536.0 / (65536 - t) if t < 65536 else 0.0


# ---------------------------------------------------------------- attention
def visible(sq, sk, ql, kl, causal):
    i, j = np.arange(sq)[:, None], np.arange(sk)[None, :]
    m = (i < ql) & (j < kl)
    return m & (j <= i + kl - ql) if causal else m


def attention(q, k, v, scale, mask):
    """One head: q [sq, d], k, v [sk, d], mask [sq, sk] -> o, lse, p. Rows without keys: 0, -inf.
    What masked-out rows of k and v hold is not used."""
    seen_k = mask.any(0)[:, None]
    k, v = np.where(seen_k, k, 0), np.where(seen_k, v, 0)
    q = np.where(mask.any(1)[:, None], q, 0)
    s = np.where(mask, q @ k.T * scale, -np.inf)
    m = s.max(1, initial=-np.inf, keepdims=True)
    p = np.exp(s - np.where(np.isinf(m), 0, m))
    total = p.sum(1, keepdims=True)
    p = p / np.where(total > 0, total, 1)
    with np.errstate(divide="ignore"):
        lse = np.where(total > 0, np.where(np.isinf(m), 0, m) + np.log(total), -np.inf)[:, 0]
    return p @ v, lse, p


def attention_backward(q, k, v, o, do, p, scale, mask):
    """One head's dq, dk, dv and, for each, the sum of its terms' sizes (what a relative rounding
    of every probability and of every score gradient can move)."""
    seen_k, seen_q = mask.any(0)[:, None], mask.any(1)[:, None]
    k, v = np.where(seen_k, k, 0), np.where(seen_k, v, 0)
    q, do, o = np.where(seen_q, q, 0), np.where(seen_q, do, 0), np.where(seen_q, o, 0)
    dp = do @ v.T
    delta = (do * o).sum(1, keepdims=True)
    ds = p * (dp - delta) * scale
    size = p * (np.abs(do) @ np.abs(v).T + np.abs(do * o).sum(1, keepdims=True)) * abs(scale)
    grads = (ds @ k, ds.T @ q, p.T @ do)
    terms = (np.abs(ds) @ np.abs(k), np.abs(ds).T @ np.abs(q), p.T @ np.abs(do))
    sizes = (size @ np.abs(k), size.T @ np.abs(q), p.T @ np.abs(do))
    return grads, terms, sizes
