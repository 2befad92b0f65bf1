"""Refusals of the dense paged-cache operators, without a GPU: the C ABI's checks come before any CUDA call, and the
Python layer's before it touches a device."""

import ctypes as C

import pytest
import torch

from pqhsa_release_b200 import PagedAttention, _lib
from pqhsa_release_b200._lib import PagedParams

A = 4096  # a non-null, 256-byte aligned address that is never dereferenced


def params(**over):
    p = PagedParams()
    p.abi_version, p.dtype, p.requests, p.kv_heads, p.group, p.query_len = _lib.ABI_VERSION, _lib.BF16, 2, 8, 4, 1
    p.head_dim, p.slot_capacity = 128, 1024
    p.k_base = p.v_base = p.block_table = p.seq_lens = p.q = p.out = p.workspace = A
    p.max_blocks, p.block_size, p.num_blocks = 64, 16, 128
    p.stride_block, p.stride_head, p.stride_row = 16 * 8 * 128, 128, 8 * 128
    p.scale = 128**-0.5
    p.q_stride_request = p.out_stride_request = 32 * 128
    p.q_stride_token = p.out_stride_token = 32 * 128
    p.q_stride_head = p.out_stride_head = 128
    p.workspace_bytes = 1 << 40
    for k, v in over.items():
        setattr(p, k, v)
    return p


ATTENTION = [
    ({"abi_version": 3}, -2, "abi_version"), ({"dtype": 3}, -3, "dtype"), ({"head_dim": 64}, -2, "head_dim"),
    ({"requests": -1}, -2, "requests"), ({"requests": 70000}, -2, "requests"), ({"kv_heads": 0}, -2, "kv_heads"),
    ({"group": 0}, -2, "group"), ({"group": 17}, -2, "group"), ({"query_len": 0}, -2, "query_len"), ({"query_len": 9}, -2, "query_len"),
    ({"group": 16, "query_len": 5}, -2, "group * query_len"), ({"slot_capacity": 0}, -2, "slot_capacity"),
    ({"slot_capacity": (1 << 24) + 1}, -2, "slot_capacity"), ({"kv_heads": 1024, "slot_capacity": 1 << 24}, -2, "2^33"),
    ({"k_base": None}, -1, "k_base"), ({"seq_lens": None}, -1, "seq_lens"), ({"block_size": 0}, -2, "block_size"),
    ({"num_blocks": 0}, -2, "num_blocks"), ({"max_blocks": 0}, -2, "max_blocks"), ({"block_table": None, "num_blocks": 1}, -2, "contiguous"),
    ({"stride_row": 127}, -2, "aligned"), ({"k_base": A + 2}, -2, "aligned"), ({"window": -1}, -2, "window"),
    ({"sink_tokens": -1}, -2, "sink_tokens"), ({"q": None}, -1, "q is null"), ({"out": None}, -1, "out is null"),
    ({"q_stride_head": 4}, -2, "rows of q"), ({"out": A + 8}, -2, "rows of out"), ({"key_pos": A}, -1, "query_pos"),
    ({"scale": float("nan")}, -2, "scale"), ({"softcap": -1.0}, -2, "softcap"), ({"softcap": float("inf")}, -2, "softcap"),
    ({"workspace": None}, -4, "workspace"), ({"workspace": A + 16}, -4, "aligned"), ({"workspace_bytes": 100}, -4, "needed"),
]


@pytest.mark.parametrize("over, code, text", ATTENTION, ids=[t + str(i) for i, (_, _, t) in enumerate(ATTENTION)])
def test_attention_refuses(over, code, text):
    with pytest.raises(_lib.PqhsaError) as e:
        _lib.call("pqhsa_paged_attention", C.byref(params(**over)), None)
    assert e.value.code == code and text in str(e.value)


EVICT = [
    ({"mass": None}, (64, 8, A, A, A, A, A), -1, "mass"), ({"key_pos": None}, (64, 8, A, A, A, A, A), -1, "key_pos"),
    ({"query_pos": None}, (64, 8, A, A, A, A, A), -1, "query_pos"), ({}, (0, 0, A, A, A, A, A), -2, "budget"),
    ({}, (64, 65, A, A, A, A, A), -2, "recent"), ({"sink_tokens": 60}, (64, 8, A, A, A, A, A), -2, "recent"),
    ({}, (64, -1, A, A, A, A, A), -2, "recent"), ({}, (64, 8, None, A, A, A, A), -1, "null"), ({}, (64, 8, A, None, A, A, A), -1, "null"),
    ({}, (64, 8, A, A, None, A, A), -1, "null"), ({}, (64, 8, A, A, A, None, A), -1, "null"), ({}, (64, 8, A, A, A, A, None), -1, "null"),
]


@pytest.mark.parametrize("over, args, code, text", EVICT, ids=[str(i) for i in range(len(EVICT))])
def test_evict_refuses(over, args, code, text):
    p = params(**{"mass": A, "key_pos": A, "query_pos": A, **over})
    with pytest.raises(_lib.PqhsaError) as e:
        _lib.call("pqhsa_paged_evict", C.byref(p), *args, None)
    assert e.value.code == code and text in str(e.value)


def test_append_refuses():
    for k, v, n, code in ((None, A, A, -1), (A, None, A, -1), (A, A, None, -1), (A + 2, A, A, -2)):
        with pytest.raises(_lib.PqhsaError) as e:
            _lib.call("pqhsa_paged_append", C.byref(params()), k, v, n, None)
        assert e.value.code == code


def test_null_params_and_no_requests():
    for name, args in (("attention", ()), ("append", (A, A, A)), ("evict", (64, 8, A, A, A, A, A))):
        with pytest.raises(_lib.PqhsaError) as e:
            _lib.call("pqhsa_paged_" + name, None, *args, None)
        assert e.value.code == -1
        _lib.call("pqhsa_paged_" + name, C.byref(params(requests=0)), *args, None)  # nothing to do, nothing launched
    assert _lib.lib.pqhsa_paged_workspace_bytes(None) == 0


def test_workspace_grows_with_the_scores_only_when_weights_are_wanted():
    size = lambda **o: _lib.lib.pqhsa_paged_workspace_bytes(C.byref(params(**o)))
    plain = size()
    assert 0 < plain < 16 << 20 and size(slot_capacity=1 << 20) == plain
    assert size(mass=A, slot_capacity=1 << 20) >= plain + 2 * 32 * (4 << 20)
    assert size(group=17) == 0


def make(**kw):
    a = dict(num_query_heads=8, num_kv_heads=2, max_requests=2, token_capacity=64, dtype=torch.bfloat16, device="cuda")
    return PagedAttention(**{**a, **kw})


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=torch.float64), "dtype"), (dict(num_query_heads=7), "GQA"), (dict(num_kv_heads=0), "GQA"), (dict(num_query_heads=34), "query heads"),
    (dict(max_query_len=0), "max_query_len"), (dict(max_query_len=9), "max_query_len"), (dict(num_query_heads=32, max_query_len=5), "max_query_len"),
    (dict(max_requests=0), "positive"), (dict(token_capacity=0), "positive"), (dict(scale=float("inf")), "scale"), (dict(softcap=-2.0), "softcap"),
    (dict(window=-1), "window"), (dict(sink_tokens=-1), "sink_tokens"),
])
def test_constructor_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        make(**kw)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        make(device="cpu")


def test_parameter_block_matches_the_header():
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parents[1] / "include" / "pqhsa.h").read_text()
    body = re.search(r"typedef struct pqhsa_paged_params \{(.*?)\} pqhsa_paged_params;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = []
    for decl in body.split(";"):
        words = decl.replace("*", " ").replace("const", " ").split(None, 1)
        if len(words) == 2:
            names += [n.strip() for n in words[1].split(",")]
    assert names == [n for n, _ in PagedParams._fields_]


def test_hook_takes_only_the_steps_it_can_serve():
    from types import SimpleNamespace as NS

    from pqhsa_release_b200.pq_hsa_vllm import runtime

    def ask(impl=(), md=(), kv=None):
        i = dict(num_heads=8, num_kv_heads=2, sliding_window=(-1, -1), logits_soft_cap=0, alibi_slopes=None)
        m = dict(use_cascade=False, max_query_len=1, num_actual_tokens=3, seq_lens=torch.tensor([4, 0, 9], dtype=torch.int32))
        i.update(impl)
        m.update(md)
        return runtime.should_dense_decode(NS(**i), torch.zeros(4, 2, 16, 256, dtype=torch.bfloat16) if kv is None else kv, NS(**m))

    assert ask() and ask(impl=dict(sliding_window=(39, 0))) and ask(md=dict(max_query_len=2, num_actual_tokens=6))
    assert ask(kv=torch.zeros(2, 4, 16, 2, 128))
    assert not runtime.should_dense_decode(NS(num_heads=8, num_kv_heads=2), torch.zeros(4, 2, 16, 256), None)
    for impl in (dict(num_heads=64), dict(num_heads=9), dict(num_kv_heads=4), dict(attn_type="encoder_only"), dict(sliding_window=(5, 5)),
                 dict(sinks=torch.zeros(8)), dict(kv_sharing_target_layer_name="a"), dict(dcp_world_size=2)):
        assert not ask(impl=impl), impl
    for md in (dict(use_cascade=True), dict(seq_lens=None), dict(max_query_len=9, num_actual_tokens=27), dict(num_actual_tokens=2)):
        assert not ask(md=md), md
    for kv in (torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16), torch.zeros(4, 2, 16, 256, dtype=torch.uint8), torch.zeros(4, 2, 256)):
        assert not ask(kv=kv), tuple(kv.shape)
