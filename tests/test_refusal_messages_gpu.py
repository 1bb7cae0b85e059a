"""Refusals whose messages hold numbers: the call raises, the process goes on."""
import pytest
import torch

from gpu_util import native, status_word

pytestmark = pytest.mark.gpu


def test_products_of_unequal_depth_are_refused():
    a, b, d = (torch.zeros(16, k, dtype=torch.bfloat16, device="cuda") for k in (64, 128, 16))
    with pytest.raises(RuntimeError, match="K mismatch 64 vs 128"):
        native().gemm_bf16(a, b, d, False, False, None, 1.0, False, status_word(), None)


@pytest.mark.parametrize("which,offset", [(0, -8), (3, 4), (6, 1 << 40)])
def test_offsets_that_a_layer_cannot_have_are_refused(which, offset):
    from test_layer_call_gpu import Layer

    layer = Layer([16])
    layer.off_list[which] = offset
    with pytest.raises(RuntimeError, match=f"offset of tensor {which}"):
        layer.call_forward(False)
    with pytest.raises(RuntimeError, match=f"offset of tensor {which}"):
        layer.call_backward(torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"), torch.zeros_like(layer.params, dtype=torch.float32))
