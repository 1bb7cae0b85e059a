"""The rollout engine over an 8-bit cache against one over a bf16 cache whose keys and values are rounded, by plain torch, as they are written.

Prompts of many rows take the same products in both, so their log-probabilities are equal in every bit: what an 8-bit engine computes is bf16 attention over rounded
keys and values, and nothing else."""
import pytest
import torch

from async_grpo_nccl_b200.ops import reference as R
from test_kv8_engine_gpu import engine, model, prompts_of, run  # noqa: F401 (model is a fixture)

pytestmark = pytest.mark.gpu


class Rounding:
    """The native operators, with what is written to the cache rounded to 8 bits and back."""

    def __init__(self, ops):
        self.ops = ops

    def __getattr__(self, name):
        return getattr(self.ops, name)

    def kv_cache_write(self, qkv, slots, k, v, Hq, Hkv, D, status=None, kv_head0=0, k_scale=None, v_scale=None):
        self.ops.kv_cache_write(qkv, slots, k, v, Hq, Hkv, D, status, kv_head0, k_scale, v_scale)
        at = slots[slots >= 0].long()
        for c in (k, v):
            rows = c[at // c.shape[2], :, at % c.shape[2]]
            c[at // c.shape[2], :, at % c.shape[2]] = R.kv8_values(*R.kv8_quantise(rows)).to(torch.bfloat16)


@pytest.mark.parametrize("kw", [dict(kv_cache_dtype="fp8"), dict(prefill_chunk_tokens=8193)])
def test_more_sequences_than_the_attention_takes_are_refused_at_once(model, kw):  # noqa: F811
    with pytest.raises(ValueError, match="8192"):
        engine(model, max_seqs=8193, **kw)
    if "prefill_chunk_tokens" in kw:
        engine(model, max_seqs=8193, prefill_chunk_tokens=64)


@pytest.mark.parametrize("size", [100, 100000])
def test_prompts_over_8_bits_are_prompts_over_rounded_keys_and_values(model, size):  # noqa: F811
    prompts = prompts_of(model[0], [90, 130, 260, 400])
    eight = run(engine(model, kv_cache_dtype="fp8", prefill_chunk_tokens=size), prompts, new=1)
    sixteen = engine(model, prefill_chunk_tokens=size)
    other = run(sixteen, prompts, new=1)
    sixteen.dec.C = Rounding(sixteen.dec.C)
    rounded = run(sixteen, prompts, new=1)
    assert eight == rounded
    assert eight != other
