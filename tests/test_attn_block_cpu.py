"""The 64-bit references' gradients against central differences, the generator against its
published vectors, and the entry points' refusals without a device."""
import threading

import numpy as np
import pytest

import attn_block_ref as ref


def _directional(f, args, grads, rng):
    """sum(grad . direction) against the central difference of f along the direction."""
    ds = [rng.standard_normal(a.shape) for a in args]
    h = 1e-6
    num = (f(*[a + h * d for a, d in zip(args, ds)]) - f(*[a - h * d for a, d in zip(args, ds)])) / (2 * h)
    ana = sum((g * d).sum() for g, d in zip(grads, ds))
    # truncation h^2 and cancellation 2^-53 / h of a sum of order 1e2
    assert abs(num - ana) <= 1e-6 * max(1.0, abs(ana)), (num, ana)


@pytest.mark.parametrize("kind", [0, 1, 2, 3])
def test_group_norm_gradient_against_differences(kind):
    rng = np.random.Generator(np.random.PCG64(3 + kind))
    x, dy = rng.standard_normal((2, 2, 7, 12))
    gamma, beta = 1 + 0.3 * rng.standard_normal(12), rng.standard_normal(12)

    def loss(x, gamma, beta):
        return (ref.group_norm(x, gamma, beta, 4, 1e-5, kind)[0] * dy).sum()

    _, _, rstd, z, xh = ref.group_norm(x, gamma, beta, 4, 1e-5, kind)
    dx, dg, db, _, _ = ref.group_norm_backward(dy, z, xh, rstd, gamma, 4, kind)
    _directional(loss, (x, gamma, beta), (dx, dg, db), rng)


@pytest.mark.parametrize("sq,sk,ql,kl,causal", [(5, 5, 5, 5, False), (6, 9, 4, 7, True), (9, 4, 9, 4, True),
                                                (3, 1, 2, 1, False)])
def test_attention_gradient_against_differences(sq, sk, ql, kl, causal):
    rng = np.random.Generator(np.random.PCG64(17))
    q, k, v, do = (rng.standard_normal((n, 8)) for n in (sq, sk, sk, sq))
    mask = ref.visible(sq, sk, ql, kl, causal)

    def loss(q, k, v):
        return (ref.attention(q, k, v, 0.4, mask)[0] * do).sum()

    o, _, p = ref.attention(q, k, v, 0.4, mask)
    grads, _, _ = ref.attention_backward(q, k, v, o, do, p, 0.4, mask)
    _directional(loss, (q, k, v), grads, rng)


def test_philox_known_answers():
    # the generator's published test vectors: all zeros, all ones
    got = ref.philox([0], 0, 0)[0]
    assert [int(w) for w in got] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    got = ref.philox([2 ** 64 - 1], 2 ** 64 - 1, 2 ** 64 - 1)[0]
    assert [int(w) for w in got] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_entry_points_without_init():
    from omnimatchdeeplearningtool_b200._lib import lib
    got = []

    def probe():
        got.append(lib.omCudaGroupNormActNhwc(16, 16, None, None, None, None, 16, 1, 4, 8, 8, 1, 1e-5, 0, 1))
        got.append(lib.omCudaGroupNormActNhwcBackward(16, 16, 16, 16, None, None, 16, None, None, 16, 1, 4, 8, 8,
                                                      1, 0, 1))
        got.append(lib.omCudaDropoutAdd(16, None, 16, 8, 0.1, 0, 0, 1))
        got.append(lib.omCudaAttention(16, 16, 16, 16, None, None, None, None, 16, 1, 1, 1, 1, 1, 64, 1.0, 0, 1))
        got.append(lib.omCudaAttentionBackward(16, 16, 16, 16, 16, 16, 16, 16, 16, None, None, None, 16, 1, 1, 1,
                                               1, 1, 64, 1.0, 0, 1))

    t = threading.Thread(target=probe)
    t.start()
    t.join()
    assert got == [-4] * 5


def test_workspace_sizes_refuse_bad_shapes():
    from omnimatchdeeplearningtool_b200._lib import lib
    gn = lib.omCudaGroupNormNhwcWorkspaceBytes
    assert gn(2, 49, 64, 64, 32, 1, 0) >= 0 and gn(2, 49, 64, 64, 32, 1, 1) >= 0
    assert gn(2, 49, 64, 60, 32, 1, 0) == -2      # fewer stored channels than channels
    assert gn(2, 49, 60, 60, 4, 1, 0) == -2       # stored channels not a multiple of 8
    assert gn(2, 49, 64, 64, 7, 1, 0) == -2       # groups do not divide the channels
    assert gn(2, 49, 64, 64, 32, 3, 0) == -3      # dtype
    at = lib.omCudaAttentionWorkspaceBytes
    assert at(2, 8, 8, 197, 197, 64, 0) >= 0 and at(2, 8, 8, 197, 197, 64, 1) > 0
    assert at(2, 8, 3, 197, 197, 64, 0) == -2     # heads not shared evenly
    assert at(2, 8, 8, -1, 197, 64, 0) == -2
    assert at(2, 8, 8, 197, 197, 60, 0) == -3     # head dimension
    assert at(2, 8, 8, 197, 197, 136, 0) == -3
