"""OM_ACT_SILU belongs to the GroupNorm entry points; the other channels-last calls refuse it."""
import pytest

from omnimatchdeeplearningtool_b200._lib import ACT_NONE, ACT_RELU6, ACT_SILU, DTYPE_F32, DTYPE_F16, lib

pytestmark = pytest.mark.gpu

SIZE = 1 << 20


def _conv(b, act):
    return lib.omCudaConv2dBnAct(b[0], b[1], b[2], None, b[3], 1, 4, 4, 16, 16, 1, 1, 1, 0, act, DTYPE_F16, DTYPE_F16)


def _pair_first(b, act):
    return lib.omCudaConvPairBnAct(b[0], b[1], b[2], b[1], b[2], None, b[3], 1, 4, 4, 64, 64, 128, 1, 1, 1, 0, act, 0,
                                   DTYPE_F16)


def _pair_second(b, act):
    return lib.omCudaConvPairBnAct(b[0], b[1], b[2], b[1], b[2], None, b[3], 1, 4, 4, 64, 64, 128, 1, 1, 1, 0, 0, act,
                                   DTYPE_F16)


def _depthwise(b, act):
    return lib.omCudaDepthwiseConv2dNhwc(b[0], b[1], b[2], b[3], 1, 6, 6, 16, 3, 3, 1, 1, act, DTYPE_F16)


def _add(b, act):
    return lib.omCudaAddActNhwc(b[0], b[1], b[3], 1024, act, DTYPE_F16)


def _stem(b, act):
    return lib.omCudaStemConvBnActIn(b[0], DTYPE_F32, b[4], b[1], b[2], b[3], 1, 3, 16, 16, 64, 7, 7, 2, 3, act, DTYPE_F16)


@pytest.mark.parametrize("f", [_conv, _pair_first, _pair_second, _depthwise, _add, _stem])
def test_silu_is_refused(gpu, f):
    from omnimatchdeeplearningtool_b200.backend import DeviceBuffer
    assert 0 < lib.omCudaStemWorkspaceBytes(1, 3, 16, 16, 7, 7, 2, 3) <= SIZE
    assert 0 < lib.omCudaPackedStemWeightElems(64, 3, 7, 7, 2) * 2 <= SIZE
    keep = [DeviceBuffer.zeros(SIZE) for _ in range(5)]
    b = [x.ptr for x in keep]
    assert f(b, ACT_NONE) == 0 and f(b, ACT_RELU6) == 0
    assert f(b, ACT_SILU) == -3
    assert lib.omCudaSynchronize() == 0
