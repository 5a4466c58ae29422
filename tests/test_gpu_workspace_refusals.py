"""A caller's workspace is counted by the memory it spans and has to lie on the
operands' device: what the linears, the decode attention, the LM head and the
argmax refuse before anything is launched."""
import pytest
import torch

from ondeviceinfer_amd import _native

pytestmark = pytest.mark.gpu

BAD = {'expanded': lambda gpu: torch.empty(1, dtype=torch.uint8, device=gpu).expand(1 << 24),
       'strided': lambda gpu: torch.empty(1 << 12, dtype=torch.uint8, device=gpu)[::2],
       'host': lambda gpu: torch.empty(1 << 24, dtype=torch.uint8)}


def half(gpu, *shape):
    return torch.zeros(*shape, dtype=torch.float16, device=gpu)


def int8(gpu, *shape):
    return torch.zeros(*shape, dtype=torch.int8, device=gpu)


CALLS = {
    'w4a16_linear': lambda gpu, ws: _native.w4a16_linear(
        half(gpu, 8, 512), int8(gpu, 256 * 256), half(gpu, 256 * 16), 256, 128, workspace=ws),
    'w8a16_linear': lambda gpu, ws: _native.w8a16_linear(
        half(gpu, 8, 512), int8(gpu, 256, 512), half(gpu, 256), workspace=ws),
    'decode_attention': lambda gpu, ws: _native.decode_attention(
        half(gpu, 8 * 128), 4, 2, None, None, 1e-6, half(gpu, 64, 128), half(gpu, 64, 128),
        torch.zeros(1, dtype=torch.int32, device=gpu), half(gpu, 2, 64, 128), half(gpu, 2, 64, 128), 0.1, workspace=ws),
    'lm_head': lambda gpu, ws: _native.lm_head(half(gpu, 512), half(gpu, 1000, 512), workspace=ws),
    'argmax_f16': lambda gpu, ws: _native.argmax_f16(half(gpu, 1000), workspace=ws),
}


@pytest.mark.parametrize('bad', list(BAD))
@pytest.mark.parametrize('call', list(CALLS))
def test_workspaces_without_memory_of_their_own_are_refused(gpu, call, bad):
    print(call, bad, flush=True)
    with pytest.raises(ValueError, match='contiguous' if bad != 'host' else 'GPU'):
        CALLS[call](gpu, BAD[bad](gpu))
