"""What the operators on a part of a long context refuse, before any kernel runs: no GPU needed."""
import ctypes as C

import pytest
import torch

import aitherkvcache_amd as akv
from aitherkvcache_amd import _lib

H = torch.float16
I32 = torch.int32


@pytest.fixture
def anywhere(monkeypatch):
    """Tensors of the host pass for the device's; a call that reaches the library says so."""
    class Reached(Exception):
        pass

    class Library:
        def __getattr__(self, name):
            if name.endswith("_workspace_bytes"):
                return lambda *a: 0

            def call(*args):
                raise Reached(name)
            return call

    monkeypatch.setattr(_lib, "require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "lib", Library)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 0)
    return Reached


def batch():
    return dict(block_tables=torch.zeros(2, 2, dtype=I32), context_lens=torch.zeros(2, dtype=I32), query_start_loc=torch.tensor([0, 2, 5]))


BATCH = [
    (ValueError, dict(block_tables=torch.zeros(1, 2, dtype=I32))),
    (ValueError, dict(block_tables=torch.zeros(4, dtype=I32))),
    (ValueError, dict(context_lens=torch.zeros(1, dtype=I32))),
    (ValueError, dict(query_start_loc=torch.zeros(0, dtype=I32))),
    (ValueError, dict(query_start_loc=torch.zeros(4, dtype=I32))),
    (ValueError, dict(block_tables=torch.zeros(2, 2))),
    (ValueError, dict(context_lens=torch.zeros(2, dtype=torch.int16))),
]
QUERY = [
    (NotImplementedError, dict(query=torch.zeros(5, 8, 64))),
    (ValueError, dict(query=torch.zeros(5, 7, 64, dtype=H))),
    (ValueError, dict(query=torch.zeros(40, 64, dtype=H))),
    (ValueError, dict(query=torch.zeros(5, 8, 128, dtype=H))),
]


def update(**change):
    a = dict(key_cache=torch.zeros(3, 16, 2, 64, dtype=H), **batch())
    a.update(change)
    index = a.pop("index", None) or akv.BlockIndex(3, 2, 64, "cpu")
    return index.update(**a)


def odd_index(**attrs):
    index = akv.BlockIndex(3, 2, 64, "cpu")
    for k, v in attrs.items():
        setattr(index, k, v)
    return index


@pytest.mark.parametrize("error,change", BATCH + [
    (NotImplementedError, dict(key_cache=torch.zeros(3, 16, 2, 64))),
    (ValueError, dict(key_cache=torch.zeros(3, 16, 128, dtype=H))),
    (ValueError, dict(key_cache=torch.zeros(4, 16, 2, 64, dtype=H))),
    (ValueError, dict(key_cache=torch.zeros(3, 16, 1, 64, dtype=H))),
    (ValueError, dict(key_cache=torch.zeros(3, 16, 64, 2, dtype=H).transpose(2, 3))),
    (ValueError, dict(index=odd_index(codes=torch.zeros(3, 2, 64)))),
    (ValueError, dict(index=odd_index(scales=torch.zeros(2, 3).t()))),
])
def test_update_refuses(anywhere, error, change):
    with pytest.raises(error):
        update(**change)


def test_calls_in_order_reach_the_library(anywhere):
    for call in (update, lambda: update(query_start_loc=None), select, sparse, weights, packed, evict):
        with pytest.raises(anywhere):
            call()
    for shape in ((-1, 2, 64), (3, 0, 64), (3, 2, 0)):
        with pytest.raises(ValueError):
            akv.BlockIndex(*shape, "cpu")


def select(**change):
    a = dict(query=torch.zeros(5, 8, 64, dtype=H), block_size=16, num_selected=4, **batch())
    a.update(change)
    return akv.BlockIndex(3, 2, 64, "cpu").select(**a)


@pytest.mark.parametrize("error,change", BATCH + QUERY + [
    (ValueError, dict(block_size=0)),
    (ValueError, dict(num_selected=2)),
    (ValueError, dict(num_sink_blocks=-1)),
    (ValueError, dict(num_recent_blocks=0)),
    (ValueError, dict(num_sink_blocks=3)),
    (ValueError, dict(out=torch.zeros(5, 2, 4))),
    (ValueError, dict(out=torch.zeros(5, 2, 5, dtype=I32))),
    (ValueError, dict(out=torch.zeros(5, 4, 2, dtype=I32).transpose(1, 2))),
])
def test_select_refuses(anywhere, error, change):
    with pytest.raises(error):
        select(**change)


def sparse(**change):
    a = dict(query=torch.zeros(5, 8, 64, dtype=H), key_cache=torch.zeros(3, 16, 2, 64, dtype=H), value_cache=torch.zeros(3, 16, 2, 64, dtype=H),
             selected=torch.zeros(5, 2, 4, dtype=I32), **batch())
    a.update(change)
    return akv.paged_sparse_attention(**a)


@pytest.mark.parametrize("error,change", BATCH + QUERY + [
    (ValueError, dict(query=torch.zeros(5, 8, 64, dtype=torch.bfloat16))),
    (ValueError, dict(key_cache=torch.zeros(3, 16, 64, dtype=H))),
    (ValueError, dict(key_cache=torch.zeros(3, 16, 64, 2, dtype=H).transpose(2, 3))),
    (ValueError, dict(value_cache=torch.zeros(3, 8, 2, 64, dtype=H))),
    (ValueError, dict(value_cache=torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16))),
    (ValueError, dict(selected=torch.zeros(5, 2, 4, dtype=torch.int64))),
    (ValueError, dict(selected=torch.zeros(4, 2, 4, dtype=I32))),
    (ValueError, dict(selected=torch.zeros(5, 8, 4, dtype=I32))),
    (ValueError, dict(out=torch.zeros(5, 8, 64))),
    (ValueError, dict(out=torch.zeros(4, 8, 64, dtype=H))),
])
def test_sparse_refuses(anywhere, error, change):
    with pytest.raises(error):
        sparse(**change)


def weights(**change):
    a = dict(query=torch.zeros(5, 8, 64, dtype=H), key_cache=torch.zeros(3, 16, 2, 64, dtype=H), **batch())
    a.update(change)
    return akv.paged_key_weights(**a)


ACCUMULATED = [
    (ValueError, dict(accumulated=torch.zeros(2, 2, 32, dtype=torch.float64))),
    (ValueError, dict(accumulated=torch.zeros(2, 2, 31))),
    (ValueError, dict(accumulated=torch.zeros(1, 2, 32))),
    (ValueError, dict(accumulated=torch.zeros(2, 8, 32))),
    (ValueError, dict(accumulated=torch.zeros(2, 32))),
    (ValueError, dict(accumulated=torch.zeros(2, 32, 2).transpose(1, 2))),
    (ValueError, dict(accumulated=torch.zeros(1, 2, 32).expand(2, -1, -1))),
]


@pytest.mark.parametrize("error,change", BATCH + QUERY + ACCUMULATED + [
    (ValueError, dict(query=torch.zeros(5, 8, 64, dtype=torch.bfloat16))),
    (ValueError, dict(key_cache=torch.zeros(3, 16, 64, dtype=H))),
    (ValueError, dict(key_cache=torch.zeros(3, 16, 64, 2, dtype=H).transpose(2, 3))),
])
def test_weights_refuse(anywhere, error, change):
    with pytest.raises(error):
        weights(**change)


class Quantizer:
    head_dim, bits, num_levels, _packed_dim = 64, 4, 16, 32
    rotation, centroids = torch.eye(64), torch.linspace(-1, 1, 16)

    def prepared_rotation(self):
        class Prepared:
            ptr = 0
        return Prepared


def packed(centroids=None, **change):
    a = dict(query=torch.zeros(5, 8, 64, dtype=H), k_packed=torch.zeros(3, 16, 2, 32, dtype=torch.uint8), k_norms=torch.zeros(3, 16, 2), **batch())
    a.update(change)
    attn = akv.TQPagedAttention(Quantizer(), 8)
    if centroids is not None:
        attn.centroids = centroids
    return attn.key_weights(**a)


@pytest.mark.parametrize("error,change", BATCH + QUERY + ACCUMULATED + [
    (ValueError, dict(k_packed=torch.zeros(3, 16, 2, 31, dtype=torch.uint8))),
    (ValueError, dict(k_packed=torch.zeros(3, 16, 2, 32))),
    (ValueError, dict(k_packed=torch.zeros(3, 16, 32, dtype=torch.uint8))),
    (ValueError, dict(k_norms=torch.zeros(3, 8, 2))),
    (ValueError, dict(k_norms=torch.zeros(3, 16))),
    (ValueError, dict(block_size=32)),
    (ValueError, dict(block_size=0)),
    (ValueError, dict(num_kv_heads=3)),
    (ValueError, dict(num_kv_heads=4)),
    (ValueError, dict(centroids=torch.zeros(8))),
])
def test_packed_weights_refuse(anywhere, error, change):
    with pytest.raises(error):
        packed(**change)


def evict(**change):
    a = dict(weights=torch.zeros(2, 2, 32), block_tables=torch.zeros(2, 2, dtype=I32), context_lens=torch.zeros(2, dtype=I32),
             caches=[torch.zeros(3, 16, 2, 64, dtype=H), torch.zeros(3, 16, 2)], keep=20, num_sink=2, num_recent=8)
    a.update(change)
    return akv.evict_tokens(**a)


@pytest.mark.parametrize("error,change", [
    (ValueError, dict(weights=torch.zeros(2, 2, 32, dtype=torch.float64))),
    (ValueError, dict(weights=torch.zeros(2, 2, 31))),
    (ValueError, dict(weights=torch.zeros(1, 2, 32))),
    (ValueError, dict(weights=torch.zeros(2, 3, 32))),
    (ValueError, dict(weights=torch.zeros(2, 32))),
    (ValueError, dict(block_tables=torch.zeros(1, 2, dtype=I32))),
    (ValueError, dict(block_tables=torch.zeros(2, dtype=I32))),
    (ValueError, dict(block_tables=torch.zeros(2, 2))),
    (ValueError, dict(context_lens=torch.zeros(2, 1, dtype=I32))),
    (ValueError, dict(context_lens=torch.zeros(2))),
    (ValueError, dict(caches=[])),
    (ValueError, dict(caches=[torch.zeros(3, 16, 2)] * 9)),
    (ValueError, dict(caches=[torch.zeros(3, 16)])),
    (ValueError, dict(caches=[torch.zeros(3, 16, 2), torch.zeros(3, 16, 3)])),
    (ValueError, dict(caches=[torch.zeros(3, 16, 2), torch.zeros(3, 17, 2)])),
    (ValueError, dict(caches=[torch.zeros(3, 16, 2, 8, 4).transpose(3, 4)])),
    (ValueError, dict(keep=0)),
    (ValueError, dict(keep=9)),
    (ValueError, dict(num_sink=-1)),
    (ValueError, dict(num_recent=-1)),
    (ValueError, dict(out_tables=torch.zeros(1, 2, dtype=I32))),
    (ValueError, dict(out_tables=torch.zeros(2, 1, dtype=I32))),
    (ValueError, dict(out_tables=torch.zeros(2, 2))),
])
def test_evict_refuses(anywhere, error, change):
    with pytest.raises(error):
        evict(**change)


# ---- the library itself: sizes and pointers that no kernel can take
needs_library = pytest.mark.skipif(not _lib.available(), reason="library not built")
P = 1 << 12          # an address that is aligned and never read


def status(name, *args):
    return getattr(_lib.lib(), name)(*args)


def library_update(d=64, dtype=0, kc=P, tables=P, it=0, S=2, kvh=2, block=16, blocks=3, cols=2, codes=P, stride=64):
    return status("akv_block_index_update", kc, dtype, 2048, 128, stride, tables, it, 2, P, 0, P, 0, codes, P, S, 5, kvh, d, block, blocks, cols, None)


def library_select(d=64, dtype=0, q=P, qh=8, kvh=2, k=4, sinks=1, recent=2, ws=P, size=1 << 30, block=16, T=5, cols=2):
    return status("akv_block_index_select", q, dtype, 512, 64, P, P, P, 0, 2, P, 0, P, 0, P, 2, T, qh, kvh, d, block, 3, cols, k, sinks, recent, ws, size, None)


def library_sparse(d=64, dtype=0, q=P, qh=8, kvh=2, k=4, sel=P, block=16, scale=0.1, cols=2, out=P, T=5, ks_pos=128, vs_pos=128, ws=P, size=1 << 30):
    return status("akv_sparse_attn", q, dtype, 512, 64, P, 2048, ks_pos, 64, P, 2048, vs_pos, 64, P, 0, 2, P, 0, P, 0, sel, 8, 4, k, out, 512, 64, 1, 2, T, qh, kvh, d, block, 3, cols, scale, ws, size, None)


def library_weights(d=64, dtype=0, q=P, qh=8, kvh=2, length=32, ws=P, size=1 << 30, scale=0.1, out=P, S=2):
    return status("akv_key_weights", q, dtype, 512, 64, P, 2048, 128, 64, P, 0, 2, P, 0, P, 0, out, 64, 32, length, 0, S, 5, qh, kvh, d, 16, 3, 2, scale, ws, size, None)


def library_packed(d=64, bits=4, kp=P, prep=P, cen=P, stride=32):
    return status("akv_packed_key_weights", P, 0, 512, 64, kp, 1024, 64, stride, P, 32, 2, 1, P, 0, 2, P, 0, P, 0, prep, cen, bits, P, 64, 32, 32, 0, 2, 5, 8, 2, d, 16, 3, 2, 0.1, P, 1 << 30, None)


def library_evict(w=P, length=32, keep=10, sinks=2, recent=4, S=2, kvh=2, kept=P):
    return status("akv_evict_select", w, 64, 32, length, P, 0, S, kvh, keep, sinks, recent, kept, 20, 10, P, 64, 32, P, None)


def library_move(caches=None, n=None, keep=10, S=2, kvh=2, ot=None, ot_it=0, kept=P):
    caches = [(P, 4096, 256, 128, 128)] if caches is None else caches
    held = (_lib.EvictCache * max(1, len(caches)))(*(_lib.EvictCache(*c) for c in caches))
    return status("akv_evict_move", kept, 20, 10, P, 0, keep, P, 0, 2, 2, ot, ot_it, 2, 2, held, len(caches) if n is None else n, S, kvh, 16, 3, None)


INVALID, UNSUPPORTED, WORKSPACE = _lib.AKV_ERR_INVALID, _lib.AKV_ERR_UNSUPPORTED, _lib.AKV_ERR_WORKSPACE


@needs_library
@pytest.mark.parametrize("call,want,change", [
    (library_update, INVALID, dict(dtype=7)), (library_update, INVALID, dict(kc=None)), (library_update, INVALID, dict(tables=None)), (library_update, INVALID, dict(it=2)),
    (library_update, INVALID, dict(S=-1)), (library_update, INVALID, dict(kvh=0)), (library_update, INVALID, dict(block=0)), (library_update, INVALID, dict(blocks=-1)),
    (library_update, INVALID, dict(codes=None)), (library_update, UNSUPPORTED, dict(d=96)), (library_update, UNSUPPORTED, dict(dtype=2)),
    (library_update, UNSUPPORTED, dict(kc=P + 8)), (library_update, UNSUPPORTED, dict(stride=68)), (library_update, UNSUPPORTED, dict(kvh=1 << 20)),
    (library_update, UNSUPPORTED, dict(blocks=1 << 31)), (library_update, 0, dict(S=0)), (library_update, 0, dict(cols=0)),
    (library_select, INVALID, dict(dtype=7)), (library_select, INVALID, dict(q=None)), (library_select, INVALID, dict(qh=7)), (library_select, INVALID, dict(k=2)),
    (library_select, INVALID, dict(sinks=-1)), (library_select, INVALID, dict(recent=0)), (library_select, INVALID, dict(block=0)), (library_select, INVALID, dict(T=-1)),
    (library_select, UNSUPPORTED, dict(d=96)), (library_select, UNSUPPORTED, dict(dtype=2)), (library_select, UNSUPPORTED, dict(q=P + 4)),
    (library_select, WORKSPACE, dict(ws=None, cols=40000)), (library_select, WORKSPACE, dict(size=8, cols=40000)), (library_select, WORKSPACE, dict(ws=P + 16, cols=40000)), (library_select, 0, dict(T=0)),
    (library_sparse, INVALID, dict(dtype=7)), (library_sparse, INVALID, dict(q=None)), (library_sparse, INVALID, dict(out=None)), (library_sparse, INVALID, dict(sel=None)),
    (library_sparse, INVALID, dict(k=-1)), (library_sparse, INVALID, dict(qh=7)), (library_sparse, INVALID, dict(scale=0.0)), (library_sparse, INVALID, dict(scale=float("inf"))),
    (library_sparse, INVALID, dict(scale=float("nan"))), (library_sparse, UNSUPPORTED, dict(d=96)), (library_sparse, UNSUPPORTED, dict(dtype=2)),
    (library_sparse, UNSUPPORTED, dict(k=4097)), (library_sparse, UNSUPPORTED, dict(block=4097)), (library_sparse, UNSUPPORTED, dict(q=P + 8)),
    (library_sparse, UNSUPPORTED, dict(ks_pos=1 << 27)), (library_sparse, UNSUPPORTED, dict(vs_pos=1 << 27)), (library_sparse, UNSUPPORTED, dict(vs_pos=-128)),
    (library_sparse, WORKSPACE, dict(T=2, k=64, ws=None)), (library_sparse, WORKSPACE, dict(T=2, k=64, size=100)), (library_sparse, WORKSPACE, dict(T=2, k=64, ws=P + 16)), (library_sparse, 0, dict(T=0)),
    (library_weights, INVALID, dict(dtype=7)), (library_weights, INVALID, dict(q=None)), (library_weights, INVALID, dict(out=None)), (library_weights, INVALID, dict(qh=7)),
    (library_weights, INVALID, dict(length=31)), (library_weights, INVALID, dict(scale=-1.0)), (library_weights, UNSUPPORTED, dict(d=32)), (library_weights, UNSUPPORTED, dict(dtype=2)),
    (library_weights, UNSUPPORTED, dict(S=70000)), (library_weights, WORKSPACE, dict(ws=None)), (library_weights, WORKSPACE, dict(size=100)), (library_weights, 0, dict(S=0)),
    (library_packed, INVALID, dict(bits=5)), (library_packed, INVALID, dict(prep=None)), (library_packed, INVALID, dict(cen=None)), (library_packed, INVALID, dict(kp=None)),
    (library_packed, UNSUPPORTED, dict(d=512)), (library_packed, UNSUPPORTED, dict(kp=P + 2)), (library_packed, UNSUPPORTED, dict(stride=33)),
    (library_evict, INVALID, dict(w=None)), (library_evict, INVALID, dict(kept=None)), (library_evict, INVALID, dict(keep=0)), (library_evict, INVALID, dict(keep=5)),
    (library_evict, INVALID, dict(sinks=-1)), (library_evict, INVALID, dict(length=-1)), (library_evict, INVALID, dict(kvh=0)), (library_evict, UNSUPPORTED, dict(length=1 << 31)),
    (library_evict, UNSUPPORTED, dict(S=70000)), (library_evict, 0, dict(S=0)),
    (library_move, INVALID, dict(caches=[(None, 4096, 256, 128, 128)])), (library_move, INVALID, dict(caches=[(P, 4096, 256, 128, 0)])), (library_move, INVALID, dict(keep=0)),
    (library_move, INVALID, dict(n=-1)), (library_move, INVALID, dict(caches=[(P, 4096, 256, 128, 128), (P, 4096, 256, 128, 128)])),
    (library_move, INVALID, dict(caches=[(P, 4096, 256, 128, 64), (P + 256, 4096, 256, 128, 64), (P + 32, 4096, 256, 128, 96)])), (library_move, INVALID, dict(caches=[(P, 4096, 256, 128, 64), (P, 8192, 256, 128, 64)])), (library_move, INVALID, dict(kept=None)), (library_move, INVALID, dict(ot=P, ot_it=3)), (library_move, UNSUPPORTED, dict(n=9)),
    (library_move, UNSUPPORTED, dict(caches=[(P, 4096, 256, 128, 1 << 21)])), (library_move, UNSUPPORTED, dict(S=70000)), (library_move, 0, dict(S=0)), (library_move, 0, dict(caches=[])),
])
def test_library_refuses(call, want, change):
    assert call(**change) == want
    if want:
        assert _lib.lib().akv_last_error()


@needs_library
def test_workspace_sizes():
    L = _lib.lib()
    assert L.akv_block_index_select_workspace_bytes(0, 8, 100) == 0 and L.akv_block_index_select_workspace_bytes(4, 8, 0) == 0
    # scratch of long calls is held to slabs
    assert 0 < L.akv_block_index_select_workspace_bytes(1 << 20, 8, 40000) <= 1 << 28 and L.akv_block_index_select_workspace_bytes(1 << 20, 8, 8192) == 0
    for weights in (L.akv_key_weights_workspace_bytes, L.akv_packed_key_weights_workspace_bytes):
        assert weights(0, 1, 8, 8, 64, 100) == 0 and weights(4, 1, 8, 8, 96, 100) == 0 and weights(4, 0, 8, 8, 64, 100) == 0
        for seqs in (1, 256, 1 << 16):
            assert 0 < weights(1 << 20, seqs, 32, 8, 128, 1 << 17) <= 5 << 27
