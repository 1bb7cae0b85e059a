"""Refusals whose messages hold numbers: the call raises, the process goes on."""
import pytest
import torch

from gpu_util import native, status_word

pytestmark = pytest.mark.gpu


def test_products_of_unequal_depth_are_refused():
    a, b, d = (torch.zeros(16, k, dtype=torch.bfloat16, device="cuda") for k in (64, 128, 16))
    with pytest.raises(RuntimeError, match="K mismatch 64 vs 128"):
        native().gemm_bf16(a, b, d, False, False, None, 1.0, False, status_word(), None)
