"""Which steps the vLLM hook's dense path takes and what becomes of its errors, without a GPU."""

from types import SimpleNamespace as NS

import pytest
import torch

from pqhsa_release_b200.pq_hsa_vllm import runtime


@pytest.fixture(autouse=True)
def fresh(monkeypatch):
    for k, v in {"PQ_HSA_BATCH": "1", "PQ_HSA_ENABLE": "1", "PQ_HSA_DENSE": "1", "PQ_HSA_MULTI_QUERY": "0", "PQ_HSA_FALLBACK": "0"}.items():
        monkeypatch.setenv(k, v)
    runtime.reset()
    yield
    runtime.reset()


def step(T=1, impl=(), md=(), extra=(), original=None):
    """One step of two short requests through the hook; returns the calls that reached the original forward."""
    i = dict(scale=0.1, num_heads=8, num_kv_heads=2, sliding_window=(-1, -1), logits_soft_cap=0, alibi_slopes=None)
    m = dict(use_cascade=False, max_query_len=T, num_actual_tokens=2 * T, seq_lens=torch.tensor([9, 12], dtype=torch.int32),
             seq_lens_cpu=torch.tensor([9, 12]), max_seq_len=12, block_table=torch.tensor([[0], [1]], dtype=torch.int32))
    i.update(impl)
    m.update(md)
    calls = []

    def forward(impl_, layer_, *a, output=None, **kw):
        calls.append(kw)
        return output

    q = torch.zeros(2 * T, 8, 128, dtype=torch.bfloat16)
    kv = torch.zeros(2 * T, 2, 128, dtype=torch.bfloat16)
    pages = torch.zeros(4, 2, 16, 256, dtype=torch.bfloat16)
    out = torch.zeros_like(q)
    assert runtime.pq_or_dense_forward(original or forward, NS(**i), object(), q, kv, kv, pages, NS(**m), output=out, **dict(extra)) is out
    return calls


@pytest.fixture
def taken(monkeypatch):
    """Steps that reach the library's dense kernel."""
    steps = []
    monkeypatch.setattr(runtime, "run_dense_decode", lambda *a: steps.append(a) or a[-1])
    return steps


def test_steps_that_are_not_causal_stay_with_the_engine(taken):
    assert len(step(T=3, md=dict(causal=False))) == 1 and not taken
    assert runtime.rejects()["dense_not_causal"] == 1
    assert not step(T=3, md=dict(causal=True)) and not step(T=3) and len(taken) == 2
    assert not step(T=1, md=dict(causal=False)) and len(taken) == 3  # one token sees the same either way


@pytest.mark.parametrize("T", [1, 2])
def test_errors_of_the_dense_path_fall_back_when_asked(T, monkeypatch):
    """The pages here lie in host memory, which the dense path refuses."""
    with pytest.raises(RuntimeError, match="no CPU path"):
        step(T)
    assert runtime.STATS["fallbacks"] == 0
    monkeypatch.setenv("PQ_HSA_FALLBACK", "1")
    assert len(step(T)) == 1
    assert runtime.STATS["fallbacks"] == 1 and runtime.STATS.get("library_dense_steps", 0) == 0 and runtime.STATS["dense_steps"] == 0


def test_an_error_of_the_original_forward_is_not_swallowed(monkeypatch):
    monkeypatch.setenv("PQ_HSA_FALLBACK", "1")

    def original(*a, **kw):
        raise KeyError("the engine's own")

    with pytest.raises(KeyError, match="own"):
        step(original=original)


def test_arguments_the_dense_path_does_not_know_stay_with_the_engine(taken):
    scale = torch.ones(1)
    assert step(extra=dict(output_scale=scale)) == [dict(output_scale=scale)] and not taken
    assert runtime.rejects()["dense_arguments"] == 1
    assert not step(extra=dict(output_scale=None, output_block_scale=None)) and len(taken) == 1


def test_layers_that_attend_within_chunks_stay_with_the_engine(taken):
    assert len(step(impl=dict(use_irope=True), md=dict(local_attn_metadata=NS()))) == 1 and not taken
    assert runtime.rejects()["dense_scores"] == 1
    assert not step(impl=dict(use_irope=True), md=dict(local_attn_metadata=None)) and not step(md=dict(local_attn_metadata=NS()))
    assert len(taken) == 2
