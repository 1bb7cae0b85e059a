"""The 8-bit form of the KV cache on the CPU: what its oracle promises, and what the entry points refuse without a GPU."""
import math

import pytest
import torch

from async_grpo_nccl_b200.ops import native
from async_grpo_nccl_b200.ops import reference as R


def vectors(D=64):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(200, D, generator=g) * torch.exp2(torch.randint(-30, 30, (200, 1), generator=g).float())
    x[0] = 0
    x[1] = 2.0 ** -130
    x[2, 0], x[3, 0], x[4, 0] = 448.0, 449.0, 1e38
    return x.bfloat16()


def test_what_is_read_is_the_nearest_code():
    """At most half a step of 3 mantissa bits off, or half the smallest code; exact in bf16; quantising again changes nothing."""
    x = vectors()
    codes, scale = R.kv8_quantise(x)
    y = R.kv8_values(codes, scale)
    step = torch.exp2(scale.double() - 127)[:, None]
    assert bool(((y - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, step * 2.0 ** -10)).all())
    assert torch.equal(y, y.bfloat16().double())
    assert torch.equal(R.kv8_values(*R.kv8_quantise(y.bfloat16())), y)
    top = x.double().abs().amax(-1)
    assert bool((top <= 448 * step[:, 0]).all()) and bool(((top > 224 * step[:, 0]) | (scale == R.KV8_MIN_BYTE)).all())


def test_infinities_and_nans_read_as_nan_and_the_top_stays_finite():
    x = torch.ones(4, 64).bfloat16()
    x[0, 3], x[1, 5] = math.inf, math.nan
    x[2, 0] = torch.finfo(torch.bfloat16).max
    y = R.kv8_values(*R.kv8_quantise(x))
    assert bool(y[:2].isnan().all()) and bool(y[2:].isfinite().all()) and bool(y[2:].bfloat16().isfinite().all())


def test_rows_that_see_nothing_are_zero():
    k = torch.randn(3, 1, 16, 64)
    q = torch.randn(4, 64)
    out, _ = R.paged_chunk_attention(q, k, k, torch.zeros(2, 1, dtype=torch.int32), torch.tensor([2, 0]), torch.tensor([0, 3, 4]), 1, 1, 64, 0.1)
    assert bool((out[0] == 0).all()) and bool((out[3] == 0).all()) and bool((out[1:3] != 0).any(-1).all())
    assert torch.allclose(out[1], k[0, 0, 0].double())


@pytest.mark.parametrize("op", ["write", "read", "attn"])
def test_tensors_on_the_host_are_refused(op):
    C = native()
    rows = torch.zeros(2, 3 * 64, dtype=torch.bfloat16)
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float8_e4m3fn)
    s = torch.zeros(2, 1, 16, dtype=torch.uint8)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        if op == "write":
            C.kv_cache_write(rows, i[:2], k, k, 1, 1, 64, None, 0, s, s)
        elif op == "read":
            C.kv_cache_read(k, k, i[:2], rows, 1, 1, 64, None, s, s)
        else:
            C.paged_chunk_attn(rows, k, k, i[:2, None], i, i, torch.empty(2, 64, dtype=torch.bfloat16), 1, 1, 64, 0.1, None, s, s)


def test_configuration_keys():
    from async_grpo_nccl_b200.config import make_config

    assert make_config({"kv_cache_dtype": "fp8", "prefill_chunk_tokens": 512}).kv_cache_dtype == "fp8"
    for bad in ({"kv_cache_dtype": "int8"}, {"prefill_chunk_tokens": -1},
                {"kv_cache_dtype": "fp8", "generation_tp_size": 2, "num_generation_gpu_workers": 2},
                {"prefill_chunk_tokens": 64, "generation_tp_size": 2, "num_generation_gpu_workers": 2}):
        with pytest.raises(ValueError):
            make_config(bad)
