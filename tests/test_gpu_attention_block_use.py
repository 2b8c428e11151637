"""The attention block in a model: several blocks, several steps, a captured step."""
import ctypes

import numpy as np
import pytest

import attn_block_ref as ref
from attn_block_ref import from_bits, np_type, to_bits

N, H, W, C, HEADS, GROUPS = 2, 5, 7, 64, 2, 8


def _params():
    rng = np.random.Generator(np.random.PCG64(1))
    prm = {"gamma": np.ones(C), "beta": np.zeros(C), "w_qkv": rng.standard_normal((3 * C, C)) / 8,
           "b_qkv": np.zeros(3 * C), "w_out": rng.standard_normal((C, C)) / 8, "b_out": 3 + rng.standard_normal(C)}
    return {k: v.astype(np.float32) for k, v in prm.items()}


def _dropped(blk, x, xd, code, **step):
    """Which elements of the last projection's output the block's next pass drops: there the output is
    the input, as the projection's bias keeps its values away from 0."""
    blk.forward(xd.ptr, **step)
    return from_bits(blk.out.to_numpy((N, H * W, C), np_type(code)), code) == x


@pytest.mark.gpu
def test_blocks_and_steps_have_masks_of_their_own(gpu):
    from omnimatchdeeplearningtool_b200.attention_block import AttentionBlock
    from omnimatchdeeplearningtool_b200.backend import DeviceBuffer
    x = ref.rounded(np.random.Generator(np.random.PCG64(2)).standard_normal((N, H * W, C)), 1)
    xd = DeviceBuffer.from_numpy(to_bits(x, 1))
    blocks = [AttentionBlock(N, H, W, C, HEADS, GROUPS, _params(), dropout=0.5) for _ in range(3)]
    first = [_dropped(b, x, xd, 1) for b in blocks]
    for i, a in enumerate(first):
        assert abs(a.mean() - 0.5) < 0.05
        assert all(abs((a == b).mean() - 0.5) < 0.05 for b in first[:i])    # independent, not equal
    b = blocks[0]
    assert b.step == 0
    second = _dropped(b, x, xd, 1)
    assert b.step == 1 and abs((second == first[0]).mean() - 0.5) < 0.05
    assert (_dropped(b, x, xd, 1, step=0) == first[0]).all() and (_dropped(b, x, xd, 1, step=1) == second).all()
    same = AttentionBlock(N, H, W, C, HEADS, GROUPS, _params(), dropout=0.5, seed=b.seed)
    assert (_dropped(same, x, xd, 1, step=1) == second).all()
    for blk in blocks + [same]:
        blk.close()


@pytest.mark.gpu
def test_captured_step_draws_new_masks(gpu):
    """Forward and backward captured together: each replay has the mask of the step in device memory, in
    both directions, and the results of a pass that is given that step."""
    from omnimatchdeeplearningtool_b200._lib import call, check, lib
    from omnimatchdeeplearningtool_b200.attention_block import AttentionBlock
    from omnimatchdeeplearningtool_b200.backend import DeviceBuffer
    rng = np.random.Generator(np.random.PCG64(3))
    xd, dod = (DeviceBuffer.from_numpy(to_bits(rng.standard_normal((N, H * W, C)), 2)) for _ in range(2))
    step = DeviceBuffer.from_numpy(np.zeros(1, np.uint64))
    blk = AttentionBlock(N, H, W, C, HEADS, GROUPS, _params(), "fp16", dropout=0.3, seed=5)

    def results():
        g = blk._grads
        return [blk.out.to_numpy((N, H * W, C), np.uint16)] + [g["x"].to_numpy((N, H * W, C), np.uint16)] + \
               [g["w_out"].to_numpy((C, C)), g["w_qkv"].to_numpy((3 * C, C))]

    blk.forward(xd.ptr, step_ptr=step.ptr)
    blk.backward(dod.ptr)
    call("omCudaSynchronize")
    call("omCudaGraphBeginCapture")
    try:
        blk.forward(xd.ptr, step_ptr=step.ptr)
        blk.backward(dod.ptr)
    finally:
        graph = ctypes.c_void_p()
        st = lib.omCudaGraphEndCapture(ctypes.byref(graph))
    check(st, "omCudaGraphEndCapture")
    seen = []
    for s in (0, 1, 12345):
        step.upload(np.array([s], np.uint64))
        call("omCudaGraphLaunch", graph)
        call("omCudaSynchronize")
        got = results()
        blk.forward(xd.ptr, step=s)
        blk.backward(dod.ptr)
        assert all((a == b).all() for a, b in zip(got, results()))
        seen.append(got)
    assert all((a != b).any() for a, b in zip(seen[0], seen[1])) and all((a != b).any() for a, b in zip(seen[1], seen[2]))
    call("omCudaGraphDestroy", graph)
    blk.close()


@pytest.mark.parametrize("name", ["gamma", "beta", "w_qkv", "b_qkv", "w_out", "b_out"])
def test_block_refuses_parameters_of_another_size(name):
    """Refused before anything reaches the device, where the kernels would read past the array."""
    from omnimatchdeeplearningtool_b200.attention_block import AttentionBlock
    prm = _params()
    prm[name] = prm[name][:-1]
    with pytest.raises(ValueError, match=name):
        AttentionBlock(N, H, W, C, HEADS, GROUPS, prm)
    del prm[name]
    with pytest.raises(ValueError, match=name):
        AttentionBlock(N, H, W, C, HEADS, GROUPS, prm)


@pytest.mark.parametrize("sizes", [(0, H, W, C, HEADS, GROUPS), (N, -1, W, C, HEADS, GROUPS), (N, H, 0, C, HEADS, GROUPS),
                                   (N, H, W, 0, HEADS, GROUPS), (N, H, W, C, 0, GROUPS), (N, H, W, C, HEADS, -8)])
def test_block_refuses_empty_sizes(sizes):
    from omnimatchdeeplearningtool_b200.attention_block import AttentionBlock
    with pytest.raises(ValueError):
        AttentionBlock(*sizes, _params())
