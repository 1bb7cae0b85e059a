"""Options of the native rollout engine's cache where there is no such engine: refused, not passed over."""
import pytest
import torch

from async_grpo_nccl_b200.config import make_config
from async_grpo_nccl_b200.launch import DistributedRuntime, build_inprocess_runtime

OPTIONS = [{"kv_cache_dtype": "fp8"}, {"prefill_chunk_tokens": 64}]


@pytest.mark.parametrize("option", OPTIONS)
def test_runtimes_on_the_cpu(option, tmp_path, monkeypatch):
    cfg = make_config(dict(model_name_or_path="tiny", output_dir=str(tmp_path), **option))
    with pytest.raises(ValueError, match="native rollout engine"):
        build_inprocess_runtime(cfg, device="cpu")
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    with pytest.raises(ValueError, match="native rollout engine"):
        DistributedRuntime(cfg)
    assert not torch.distributed.is_initialized()


@pytest.mark.parametrize("option", OPTIONS)
def test_the_engine_of_plain_torch(option):
    from async_grpo_nccl_b200.engine.engine import OracleEngine
    from async_grpo_nccl_b200.models.config import PRESETS
    from async_grpo_nccl_b200.models.layout import ParamLayout

    cfg = PRESETS["tiny"]
    layout = ParamLayout(cfg)
    params = torch.zeros(layout.total)
    with pytest.raises(ValueError, match="native rollout engine"):
        OracleEngine(cfg, layout, params, **option)
    OracleEngine(cfg, layout, params, kv_cache_dtype="auto", prefill_chunk_tokens=0)
