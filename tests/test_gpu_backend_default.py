"""Prefill of the backend's class as it is made, nothing replaced in it."""
import numpy as np
import pytest
import torch

from aitherkvcache_amd.vllm import backend as B
from tests.test_gpu_backend import BS, KVH, QH, make_layers, meta, slots_of, t
from tests.test_gpu_chunk import BF, check, dense_reference
from tests.test_gpu_backend_prefill import Rows
from tests.util import kv_like

pytestmark = pytest.mark.gpu


def test_prefill_of_the_class_as_made(golden, dev):
    """A first chunk: out = attention over the chunk's own rows, which the block buffer holds uncompressed."""
    cls = B._make_impl_class()
    cls.reset_class_state()
    try:
        layers, _ = make_layers(cls, golden, dev, "tq-t4nc")
        rng = np.random.default_rng(6)
        kv_cache = torch.zeros(*B.TurboQuantBackend.get_kv_cache_shape(24, BS, KVH, 128, "tq-t4nc"), dtype=torch.uint8, device=dev)
        tables, new = np.array([[5, 11, 2], [20, 7, 1]], dtype=np.int32), (37, 20)
        slots, n = slots_of(tables, 0, 0, 37) + slots_of(tables, 1, 0, 20), sum(new)
        k, v, q = kv_like(rng, (n, KVH, 128)), kv_like(rng, (n, KVH, 128)), rng.standard_normal((n, QH, 128)).astype(np.float16)
        md = meta(dev, slots, tables, new, n, max(new), query_lens=list(new))
        layers[0].do_kv_cache_update(None, t(k, dev), t(v, dev), kv_cache, md.slot_mapping)
        out = torch.empty(n, QH * 128, dtype=torch.float16, device=dev)
        layers[0].forward(None, t(q, dev).view(n, -1), t(k, dev), t(v, dev), kv_cache, md, output=out)
        buffers = [torch.zeros(24, BS, KVH, 128, dtype=BF, device=dev) for _ in range(2)]
        for buf, x in zip(buffers, (k, v)):
            buf.view(-1, KVH, 128)[torch.tensor(slots, device=dev)] = t(x, dev).to(BF)
        want, bound = dense_reference(Rows([(m, m) for m in new], tables), t(q, dev).to(BF), *buffers, layers[0].scale, 0)
        check(out.view(n, QH, 128), want, bound + 2.0 ** -11 * want.abs())      # (rounded to float16 at the end)
    finally:
        cls.reset_class_state()
