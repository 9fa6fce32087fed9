"""Refusals of the operators on device memory that need no GPU: the argument checks of the Python
front end (shapes, element types, strides) and of the C ABI without a context, and the workspace
sizes. The checks that need a context are in test_gpu_train_ops.py."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def model(esm):
    m = object.__new__(esm.Model)  # no context: a call that gets past the front end is ESM_EINVAL
    m._ctx = ctypes.c_void_p()
    return m


def refused(esm, fn, *args, match, **kw):
    with pytest.raises(esm.EsmError, match=match) as e:
        fn(*args, **kw)
    assert e.value.code == esm.ESM_EINVAL


def attention_args(T=12, H=2, dh=16, kind=torch.float16):
    d = H * dh
    return {"qkv": torch.zeros(T, 3 * d, dtype=kind), "cu": torch.tensor([0, T], dtype=torch.int32), "max_len": T,
            "H": H, "out": torch.zeros(T, d, dtype=kind), "lse": torch.zeros(H, T),
            "dout": torch.zeros(T, d, dtype=kind), "dqkv": torch.zeros(T, 3 * d, dtype=kind),
            "ws": torch.zeros(4096, dtype=torch.uint8)}


@pytest.mark.parametrize("change, match", [
    ({"qkv": torch.zeros(12, 95, dtype=torch.float16)}, "qkv must have the shape"),
    ({"qkv": torch.zeros(12, 96)}, "qkv has the element type|out has the element type"),
    ({"qkv": torch.zeros(12, 96, dtype=torch.float64)}, "not supported"),
    ({"qkv": torch.zeros(96, 12, dtype=torch.float16).t()}, "rows must be contiguous"),
    ({"cu": torch.tensor([0, 12])}, "not supported"),
    ({"cu": torch.tensor([0.0, 12.0])}, "cu_seqlens has the element type"),
    ({"lse": torch.zeros(12, 2)}, "lse must have the shape"),
    ({"H": 5}, "do not divide"),
    ({"H": 0}, "do not divide"),
    ({}, "null context"),
])
def test_attention_refusals(esm, model, change, match):
    a = {**attention_args(), **change}
    refused(esm, model.attention, a["qkv"], a["cu"], a["max_len"], a["H"], a["out"], a["lse"], match=match)
    refused(esm, model.attention_backward, a["qkv"], a["cu"], a["max_len"], a["H"], a["out"], a["lse"], a["dout"],
            a["dqkv"], a["ws"], match=match)


def test_attention_backward_refuses_mixed_types(esm, model):
    a = attention_args()
    refused(esm, model.attention_backward, a["qkv"], a["cu"], 12, 2, a["out"], a["lse"], a["dout"].bfloat16(),
            a["dqkv"], a["ws"], match="dout has the element type")


def test_layernorm_refusals(esm, model):
    x, w, s = torch.zeros(3, 8), torch.zeros(8), torch.zeros(3)
    refused(esm, model.layernorm, x, w, torch.zeros(7), x.half(), match="b must have the shape")
    refused(esm, model.layernorm, x, w.half(), w, x.half(), match="w has the element type")
    refused(esm, model.layernorm, torch.zeros(8, 3).t(), w, w, x.half(), match="x must be contiguous")
    refused(esm, model.layernorm, x, w, w, x.double(), match="not supported")
    ws = torch.zeros(64)
    refused(esm, model.layernorm_backward, x, x, w, s, torch.zeros(4), x.clone(), w.clone(), w.clone(), ws,
            match="rstd must have the shape")
    refused(esm, model.layernorm_backward, x.half(), x, w, s, s, x.half(), w.clone(), w.clone(), ws,
            match="dx has the element type")
    refused(esm, model.layernorm_backward, x.half(), x, w, s, s, x.clone(), w.clone(), w.clone(), ws,
            match="null context")


def test_logits_refusals(esm, model):
    x, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int32)
    ids, top = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    s = torch.zeros(3)
    refused(esm, model.token_logprobs, x, t.long(), s, match="not supported")
    refused(esm, model.token_logprobs, x, t, s, top_ids=ids, match="go together")
    refused(esm, model.token_logprobs, x, t, s, top_ids=ids, top_logp=torch.zeros(3, 3), match="top_logp must have")
    refused(esm, model.token_logprobs, x, t, s, match="null context")
    refused(esm, model.distill_loss, x, ids.float(), top, s, s, match="top_ids has the element type")
    refused(esm, model.distill_loss, x, ids, top, s, torch.zeros(4), match="lse must have the shape")
    refused(esm, model.distill_backward, x, ids, top, s, s, x.half(), match="dlogits has the element type")
    refused(esm, model.distill_backward, x, ids, top, s, s, x.clone(), match="null context")


def test_workspace_sizes(esm):
    n = ctypes.c_size_t()
    L = esm.lib()
    assert L.esm_attention_backward_workspace(2, 100, 4, None) == esm.ESM_EINVAL
    assert L.esm_attention_backward_workspace(-1, 100, 4, ctypes.byref(n)) == esm.ESM_EINVAL
    assert L.esm_attention_backward_workspace(2, 100, 0, ctypes.byref(n)) == esm.ESM_EINVAL
    assert L.esm_layernorm_backward_workspace(None, 100, 4, ctypes.byref(n)) == esm.ESM_EINVAL
    small, large = (esm.Model.attention_backward_workspace(b, t, 20) for b, t in ((1, 128), (64, 65536)))
    assert small >= 20 * 128 * 4 and large >= 20 * 65536 * 4


def test_null_context(esm):
    L = esm.lib()
    assert L.esm_attention(None, 1, None, 0, None, 0, 0, 0, 1, 8, 1.0, None, 0, None, None) == esm.ESM_EINVAL
    assert L.esm_layernorm(None, 0, 0, None, None, None, 1e-5, 0, 1, None, None, None, None) == esm.ESM_EINVAL
    assert L.esm_token_logprobs(None, 0, None, 0, 0, 1, None, 0, None, None, None, None, None) == esm.ESM_EINVAL


def test_workspaces_are_contiguous(esm, model):
    """nbytes of an expanded or strided tensor says nothing about the memory behind its pointer."""
    a = attention_args()
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 16, dtype=torch.uint8)[::2]):
        refused(esm, model.attention_backward, a["qkv"], a["cu"], 12, 2, a["out"], a["lse"], a["dout"], a["dqkv"], ws,
                match="workspace must be contiguous")
        x, w, s = torch.zeros(3, 8), torch.zeros(8), torch.zeros(3)
        refused(esm, model.layernorm_backward, x, x, w, s, s, x.clone(), w.clone(), w.clone(), ws,
                match="workspace must be contiguous")


def test_score_refuses_an_empty_batch(esm, model):
    refused(esm, model.score, [], match="at least one sequence")
