"""Which attention the backend's prefill runs, and what the one of this package refuses: no vLLM and no GPU needed."""
import sys
import types

import pytest

import aitherkvcache_amd.chunk_attention as ca
from aitherkvcache_amd.vllm import backend as B


def modules(monkeypatch, **attributes):
    """A `vllm` that can be imported, down to the module with the attention, which holds `attributes`; None: no such module."""
    for name in ("vllm", "vllm.v1", "vllm.v1.attention", "vllm.v1.attention.backends"):
        m = types.ModuleType(name)
        m.__path__ = []
        monkeypatch.setitem(sys.modules, name, m)
    if attributes.get("present", True):
        m = types.ModuleType("vllm.v1.attention.backends.triton_attn")
        for k, v in attributes.items():
            setattr(m, k, v)
        monkeypatch.setitem(sys.modules, m.__name__, m)


class Base:
    def __init__(self, *args, **kwargs):
        pass


def metadata(**more):
    return types.SimpleNamespace(**{**dict(block_table="tables", seq_lens="lens", query_start_loc=types.SimpleNamespace(shape=(3,)), max_query_len=5, max_seq_len=9), **more})


def test_without_vllm_it_is_this_packages():
    assert B._make_impl_class()._dense_paged_attention is B._dense_attention


def test_with_vllm_it_is_vllms(monkeypatch):
    seen = {}
    modules(monkeypatch, TritonAttentionImpl=Base, unified_attention=lambda **k: seen.update(k))
    cls = B._make_impl_class()
    assert issubclass(cls, Base) and cls._dense_paged_attention is B._vllm_unified_attention
    impl = types.SimpleNamespace(num_kv_heads=2, scale=0.5, alibi_slopes=None, sliding_window=(-1, -1), logits_soft_cap=0)
    cls._dense_paged_attention(impl, types.SimpleNamespace(device="cpu"), "k", "v", "out", metadata())
    assert seen["k"] == "k" and seen["softmax_scale"] == 0.5


@pytest.mark.parametrize("present", [True, False], ids=["name-moved", "module-moved"])
def test_an_import_that_fails_inside_vllm_is_an_error(monkeypatch, present):
    """vLLM is there, its attention is not where it was: no other kernel takes its place in silence."""
    modules(monkeypatch, present=present, **({"TritonAttentionImpl": Base} if present else {}))
    cls = B._make_impl_class()
    with pytest.raises(ImportError):
        cls._dense_paged_attention(types.SimpleNamespace(num_kv_heads=2), types.SimpleNamespace(device="cpu"), None, None, None, metadata())


def impl(**options):
    return B._StandaloneImplBase(8, 128, 0.25, num_kv_heads=2, **options)


def test_what_it_passes_on(monkeypatch):
    calls = []
    monkeypatch.setattr(ca, "paged_chunk_attention", lambda *a, **k: calls.append((a, k)))
    md = metadata()
    for options, window in ((dict(), 0), (dict(sliding_window=7), 7), (dict(attn_type="decoder", sinks=None, use_irope=False, blocksparse_params=None), 0)):
        B._dense_attention(impl(**options), "q", "k", "v", "out", md)
        assert calls.pop() == (("q", "k", "v", "tables", "lens", md.query_start_loc), dict(scale=0.25, window=window, out="out", max_query_len=5))


@pytest.mark.parametrize("options", [dict(alibi_slopes=[1.0]), dict(logits_soft_cap=30.0), dict(sinks=[0.0]), dict(attn_type="encoder_only"),
                                     dict(attn_type=types.SimpleNamespace(value="encoder")), dict(kv_sharing_target_layer_name="layer.0"),
                                     dict(use_irope=True), dict(a_new_option=3)], ids=str)
def test_what_it_refuses(monkeypatch, options):
    monkeypatch.setattr(ca, "paged_chunk_attention", lambda *a, **k: pytest.fail("computed without the option"))
    with pytest.raises(NotImplementedError):
        B._dense_attention(impl(**options), "q", "k", "v", "out", metadata())


def test_attention_that_is_not_causal_is_refused(monkeypatch):
    monkeypatch.setattr(ca, "paged_chunk_attention", lambda *a, **k: pytest.fail("computed as causal"))
    with pytest.raises(NotImplementedError):
        B._dense_attention(impl(), "q", "k", "v", "out", metadata(causal=False))
