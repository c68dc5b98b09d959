"""Prefill of the attention backend without vLLM: the block buffers and the attention over them are this package's."""
import types

import numpy as np
import pytest
import torch

from aitherkvcache_amd.vllm import backend as B
from tests.test_gpu_backend import BS, KVH, QH, make_layers, meta, slots_of, t
from tests.test_gpu_chunk import BF, check, dense_reference
from tests.util import kv_like

pytestmark = pytest.mark.gpu


@pytest.fixture
def impl_cls():
    cls = B.TurboQuantBackend.get_impl_cls()
    cls.reset_class_state()
    yield cls
    cls.reset_class_state()
    cls._dense_paged_attention = staticmethod(B._vllm_unified_attention)


class Rows:
    """What dense_reference reads of a batch."""

    def __init__(self, lens, tables):
        self.lens, self.tables = lens, tables

    def rows(self, cache, i):
        c = self.lens[i][1]
        return cache[torch.from_numpy(self.tables[i, :-(-c // BS)].astype(np.int64)).to(cache.device)].flatten(0, 1)[:c]


@pytest.mark.parametrize("name", ["tq-t4nc", "tq-t3nc", "tq35"])
@pytest.mark.parametrize("window", [None, 9])
def test_prefill_without_vllm(golden, dev, impl_cls, name, window):
    """A first chunk of two sequences, then a second one beside a decode step: out = attention over the block buffer."""
    layers, tq = make_layers(impl_cls, golden, dev, name)
    impl = layers[1]
    impl.sliding_window = (-1, -1) if window is None else (window - 1, 0)
    rng = np.random.default_rng(5)
    kv_cache = torch.zeros(*B.TurboQuantBackend.get_kv_cache_shape(24, BS, KVH, 128, name), dtype=torch.uint8, device=dev)
    tables = np.array([[5, 11, 2, 9], [20, 7, 1, 0]], dtype=np.int32)
    seen = {}

    def recorder(impl_, q, k_buf, v_buf, out, md):
        B._dense_attention(impl_, q, k_buf, v_buf, out, md)
        seen.update(q=q.clone(), k=k_buf.clone(), v=v_buf.clone())
    impl_cls._dense_paged_attention = staticmethod(recorder)
    done = [0, 0]
    for new in ((37, 20), (20, 1)):
        slots = [s for i in range(2) for s in slots_of(tables, i, done[i], done[i] + new[i])] + [-1, 24 * BS + 3]
        done = [done[i] + new[i] for i in range(2)]
        n = sum(new)
        k, v = kv_like(rng, (n + 2, KVH, 128)), kv_like(rng, (n + 2, KVH, 128))
        q = rng.standard_normal((n + 2, QH, 128)).astype(np.float16)
        md = meta(dev, slots, tables, done, n, max(new), query_lens=list(new))
        impl.do_kv_cache_update(None, t(k[:n], dev), t(v[:n], dev), kv_cache, md.slot_mapping[:n])
        out = torch.full((n + 2, QH * 128), 7.0, dtype=torch.float16, device=dev)
        impl.forward(None, t(q, dev).view(n + 2, -1), t(k, dev), t(v, dev), kv_cache, md, output=out)
        at = torch.tensor(slots[:n], device=dev)
        assert torch.equal(seen["k"].flatten(0, 1)[at], t(k[:n], dev).to(BF)) and torch.equal(seen["v"].flatten(0, 1)[at], t(v[:n], dev).to(BF))
        want, bound = dense_reference(Rows([(new[i], done[i]) for i in range(2)], tables), seen["q"], seen["k"], seen["v"], impl.scale, window or 0)
        got = out.view(n + 2, QH, 128)
        check(got[:n], want, bound + 2.0 ** -11 * want.abs())          # (rounded to float16 at the end)
        assert bool((got[n:] == 7.0).all())


def test_refusals_without_vllm(dev):
    q = torch.zeros(1, 8, 128, dtype=BF, device=dev)
    buf = torch.zeros(1, BS, 2, 128, dtype=BF, device=dev)
    md = meta(dev, [0], [[0]], [1], 1, 1)
    for change in (dict(alibi_slopes=torch.ones(8)), dict(logits_soft_cap=30.0), dict(sliding_window=(4, 4))):
        impl = types.SimpleNamespace(**{**dict(alibi_slopes=None, logits_soft_cap=0, sliding_window=(-1, -1), scale=1.0, num_kv_heads=2), **change})
        with pytest.raises(NotImplementedError):
            B._dense_attention(impl, q, buf, buf, torch.empty_like(q), md)
