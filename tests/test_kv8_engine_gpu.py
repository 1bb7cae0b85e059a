"""The rollout engine over an 8-bit cache and with prompts in portions: written, rotated, attended and shared as in use.

Two ways to the same logits (decode steps, prompts in portions of other sizes, cached beginnings) round differently: the hidden state passes about 8 bf16
roundings a layer, 2^-9 of its size each, 0.6 % together after two layers; logits here are below 20, so a log-probability is off by less than 2 * 20 * 0.006 =
0.24."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
OFF = 0.24


@pytest.fixture(scope="module")
def model():
    from async_grpo_nccl_b200.models.config import PRESETS
    from async_grpo_nccl_b200.models.layout import ParamLayout

    cfg = PRESETS["tiny128"]
    layout = ParamLayout(cfg)
    p32 = torch.empty(layout.total)
    layout.init_random_(p32, 0)
    return cfg, layout, (p32 * 3.0).to(torch.bfloat16).to(DEV)


def engine(model, **kw):
    from async_grpo_nccl_b200.engine.engine import RolloutEngine

    cfg, layout, params = model
    args = dict(max_seqs=32, max_model_len=512, num_blocks=600)
    args.update(kw)
    eng = RolloutEngine(cfg, layout, params, **args)
    eng.enable_logprobs()
    return eng


def prompts_of(cfg, lens, seed=7):
    rng = np.random.default_rng(seed)
    return [rng.integers(2, cfg.vocab_size, n).astype(np.int32) for n in lens]


def run(eng, prompts, n=1, new=12, temperature=0.0):
    for i, p in enumerate(prompts):
        eng.add_request(i, p, n=n, max_new_tokens=new, temperature=temperature, seed=i, ignore_eos=True)
    out = {(o.request_id, o.child): (o.output_ids.tolist(), o.output_logprobs.tolist()) for o in eng.run_until_done()}
    eng.check_status()
    assert eng.sched.num_running == 0
    return out


def near(a, b, first_only=False):
    """Greedy samples of two engines: log-probabilities agree as long as the tokens do; where they part, the two tokens are nearly tied."""
    assert a.keys() == b.keys()
    for k in a:
        for (x, lx), (y, ly) in [((u, v), (w, z)) for u, v, w, z in zip(*a[k], *b[k])]:
            assert abs(lx - ly) < OFF, (k, lx, ly)
            if x != y:
                break


LENS = [1, 15, 16, 17, 33, 130, 260]


@pytest.mark.parametrize("kind", ["auto", "fp8"])
def test_prompts_in_portions_give_what_whole_prompts_give(model, kind):
    prompts = prompts_of(model[0], LENS)
    base = run(engine(model, kv_cache_dtype=kind), prompts)
    for size in (5, 64, 100000):
        near(run(engine(model, kv_cache_dtype=kind, prefill_chunk_tokens=size), prompts), base)
    near(run(engine(model, kv_cache_dtype=kind, prefill_chunk_tokens=64, max_prefill_tokens=48), prompts), base)


def test_decode_steps_continue_what_a_prompt_began(model):
    """A token's log-probability from a decode step against the same from a prompt that ends before it."""
    prompts = prompts_of(model[0], [20, 90])
    got = run(engine(model, kv_cache_dtype="fp8"), prompts, new=6)
    for (i, _), (toks, lps) in got.items():
        longer = [np.concatenate([prompts[i], np.asarray(toks[:k], dtype=np.int32)]) for k in range(1, 6)]
        for k, (t, lp) in enumerate(run(engine(model, kv_cache_dtype="fp8"), longer, new=1).values(), start=1):
            assert abs(lp[0] - lps[k]) < OFF, (i, k)


def test_captured_steps_give_the_tokens_of_eager_ones(model):
    prompts = prompts_of(model[0], LENS)
    a = run(engine(model, kv_cache_dtype="fp8", use_cuda_graph=False), prompts, n=3, temperature=1.0)
    b = run(engine(model, kv_cache_dtype="fp8", use_cuda_graph=True), prompts, n=3, temperature=1.0)
    assert {k: v[0] for k, v in a.items()} == {k: v[0] for k, v in b.items()}


def test_more_rows_than_one_product_takes(model):
    prompts = prompts_of(model[0], [9] * 150)
    got = run(engine(model, kv_cache_dtype="fp8", max_seqs=320, num_blocks=2600, max_model_len=64), prompts, n=2, new=5)
    few = run(engine(model, kv_cache_dtype="fp8", max_model_len=64), prompts[:4], n=2, new=5)
    near({k: got[k] for k in few}, few)


def test_cached_beginnings_are_read_as_they_were_written(model):
    shared = prompts_of(model[0], [64], seed=1)[0]
    tails = prompts_of(model[0], [10, 30], seed=2)
    prompts = [np.concatenate([shared, t]) for t in tails]
    for kind, size in (("fp8", 0), ("fp8", 24), ("auto", 24), ("auto", 0)):
        plain = run(engine(model, kv_cache_dtype=kind, prefill_chunk_tokens=size), prompts)
        eng = engine(model, kv_cache_dtype=kind, prefill_chunk_tokens=size, prefix_caching=True)
        first = run(eng, prompts[:1])
        second = run(eng, prompts)
        assert eng.prefix_hit_tokens == 64 + 64
        near({(0, 0): first[(0, 0)]}, {(0, 0): plain[(0, 0)]})
        near(second, plain)


def test_an_8_bit_cache_takes_half_the_memory(model):
    a, b = engine(model), engine(model, kv_cache_dtype="fp8")
    assert b._bytes_per_block() * 256 == a._bytes_per_block() * 129
    assert b.cache.numel() + b.cache_scale.numel() == 600 * b._bytes_per_block()


def test_refusals(model):
    for kw in (dict(kv_cache_dtype="fp4"), dict(prefill_chunk_tokens=-1)):
        with pytest.raises(ValueError):
            engine(model, **kw)
    from async_grpo_nccl_b200.models.registry import build_engine, make_layout, resolve_model_config

    cfg = resolve_model_config("dezelorn-1.5b")
    with pytest.raises(ValueError, match="type of their parameters"):
        build_engine(cfg, make_layout(cfg), torch.zeros(1, dtype=torch.bfloat16, device=DEV), kv_cache_dtype="fp8")
