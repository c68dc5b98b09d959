"""What the operators on a chunk of new tokens refuse, before any kernel runs: no GPU needed."""
import ctypes as C

import pytest
import torch

import aitherkvcache_amd as akv
from aitherkvcache_amd import _lib
from aitherkvcache_amd import chunk_attention as ca


@pytest.fixture
def anywhere(monkeypatch):
    """Tensors of the host pass for the device's; a call that reaches the library says so."""
    class Reached(Exception):
        pass

    class Library:
        def __getattr__(self, name):
            def call(*args):
                raise Reached(name)
            return call

    monkeypatch.setattr(_lib, "require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "lib", Library)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 0)
    return Reached


def dense_call(**change):
    a = dict(query=torch.zeros(5, 8, 64, dtype=torch.float16), key_cache=torch.zeros(3, 16, 2, 64, dtype=torch.float16),
             value_cache=torch.zeros(3, 16, 2, 64, dtype=torch.float16), block_tables=torch.zeros(2, 2, dtype=torch.int32),
             context_lens=torch.zeros(2, dtype=torch.int32), query_start_loc=torch.tensor([0, 2, 5]))
    a.update(change)
    return akv.paged_chunk_attention(**a)


H = torch.float16


@pytest.mark.parametrize("error,change", [
    (NotImplementedError, dict(query=torch.zeros(5, 8, 64))),
    (ValueError, dict(query=torch.zeros(5, 7, 64, dtype=H))),
    (ValueError, dict(query=torch.zeros(40, 64, dtype=H))),
    (ValueError, dict(query=torch.zeros(5, 8, 64, dtype=torch.bfloat16))),
    (ValueError, dict(query=torch.zeros(5, 8, 128, dtype=H))),
    (ValueError, dict(key_cache=torch.zeros(3, 16, 64, dtype=H))),
    (ValueError, dict(key_cache=torch.zeros(3, 16, 64, 2, dtype=H).transpose(2, 3))),
    (ValueError, dict(value_cache=torch.zeros(3, 8, 2, 64, dtype=H))),
    (ValueError, dict(value_cache=torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16))),
    (ValueError, dict(block_tables=torch.zeros(1, 2, dtype=torch.int32))),
    (ValueError, dict(block_tables=torch.zeros(4, dtype=torch.int32))),
    (ValueError, dict(context_lens=torch.zeros(1, dtype=torch.int32))),
    (ValueError, dict(query_start_loc=torch.zeros(0, dtype=torch.int32))),
    (ValueError, dict(query_start_loc=torch.zeros(4, dtype=torch.int32))),
    (ValueError, dict(out=torch.zeros(5, 8, 64))),
    (ValueError, dict(out=torch.zeros(4, 8, 64, dtype=H))),
])
def test_dense_refuses(anywhere, error, change):
    with pytest.raises(error):
        dense_call(**change)


def test_good_calls_reach_the_library(anywhere):
    with pytest.raises(anywhere, match="workspace"):
        dense_call()
    with pytest.raises(anywhere, match="akv_rope_append"):
        rope_call()


def rope_call(**change):
    a = dict(query=torch.zeros(4, 8, 64), key=torch.zeros(4, 2, 64), value=torch.zeros(4, 2, 64), positions=torch.zeros(4, dtype=torch.int32),
             cos_sin=torch.zeros(10, 64), slot_mapping=torch.zeros(4, dtype=torch.int64), key_cache=torch.zeros(3, 16, 2, 64, dtype=H),
             value_cache=torch.zeros(3, 16, 2, 64, dtype=H))
    a.update(change)
    return akv.rope_append(**a)


@pytest.mark.parametrize("change", [
    dict(key=torch.zeros(4, 128)),
    dict(value=torch.zeros(4, 1, 64)),
    dict(query=torch.zeros(3, 8, 64)),
    dict(query=torch.zeros(4, 8, 64, dtype=H)),
    dict(value=torch.zeros(4, 2, 64, dtype=H)),
    dict(key_cache=torch.zeros(3, 16, 4, 64, dtype=H)),
    dict(value_cache=torch.zeros(3, 8, 2, 64, dtype=H)),
    dict(value_cache=torch.zeros(3, 16, 2, 64)),
    dict(key_cache=torch.zeros(3, 16, 64, 2, dtype=H).transpose(2, 3)),
    dict(positions=None),
    dict(positions=torch.zeros(3, dtype=torch.int32)),
    dict(positions=torch.zeros(3, 4, dtype=torch.int32)),
    dict(sections=(16, 16)),
    dict(sections=(16, 15), positions=torch.zeros(2, 4, dtype=torch.int32)),
    dict(sections=(33, -1), positions=torch.zeros(2, 4, dtype=torch.int32)),
    dict(sections=(1, 1, 1, 1, 28), positions=torch.zeros(5, 4, dtype=torch.int32)),
    dict(cos_sin=torch.zeros(10, 64, dtype=H)),
    dict(cos_sin=torch.zeros(0, 64)),
    dict(cos_sin=torch.zeros(64, 10).T),
    dict(slot_mapping=torch.zeros(3, dtype=torch.int64)),
    dict(query_out=torch.zeros(4, 8, 64, dtype=H)),
])
def test_rope_refuses(anywhere, change):
    with pytest.raises(ValueError):
        rope_call(**change)


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="HIP devices only"):
        dense_call()
    with pytest.raises(RuntimeError, match="HIP devices only"):
        rope_call()


# ---- the C ABI: every refusal comes before the device is touched ------------------------------------------------------------

P = 4096      # an address: nothing is read from it


def c_dense(query=P, dtype=_lib.AKV_F16, d=64, heads=8, kv=2, tokens=5, seqs=2, block=16, blocks=3, width=2, window=0, scale=0.1, strides=64, ws=P, ws_bytes=1 << 40,
            key=P, starts=P, out=P, itype=0):
    return _lib.lib().akv_dense_chunk_attn(query, dtype, strides, strides, key, 64, 64, 64, P, 64, 64, 64, P, itype, 2, P, 0, starts, 0, out, 64, 64, 1,
                                           seqs, tokens, heads, kv, d, block, blocks, width, window, 0, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("rc,change", [
    (_lib.AKV_ERR_INVALID, dict(query=None)), (_lib.AKV_ERR_INVALID, dict(out=None)), (_lib.AKV_ERR_INVALID, dict(starts=None)), (_lib.AKV_ERR_INVALID, dict(key=None)),
    (_lib.AKV_ERR_INVALID, dict(dtype=7)), (_lib.AKV_ERR_INVALID, dict(itype=2)), (_lib.AKV_ERR_INVALID, dict(heads=7)), (_lib.AKV_ERR_INVALID, dict(kv=0)),
    (_lib.AKV_ERR_INVALID, dict(tokens=-1)), (_lib.AKV_ERR_INVALID, dict(seqs=-1)), (_lib.AKV_ERR_INVALID, dict(block=0)), (_lib.AKV_ERR_INVALID, dict(window=-1)),
    (_lib.AKV_ERR_INVALID, dict(scale=0.0)), (_lib.AKV_ERR_INVALID, dict(scale=float("nan"))), (_lib.AKV_ERR_INVALID, dict(scale=float("inf"))),
    (_lib.AKV_ERR_UNSUPPORTED, dict(dtype=_lib.AKV_F32)), (_lib.AKV_ERR_UNSUPPORTED, dict(d=96)), (_lib.AKV_ERR_UNSUPPORTED, dict(d=512)),
    (_lib.AKV_ERR_UNSUPPORTED, dict(strides=65)), (_lib.AKV_ERR_UNSUPPORTED, dict(key=P + 2)), (_lib.AKV_ERR_UNSUPPORTED, dict(tokens=1 << 30)),
    (_lib.AKV_ERR_WORKSPACE, dict(ws=None)), (_lib.AKV_ERR_WORKSPACE, dict(ws_bytes=100)), (_lib.AKV_ERR_WORKSPACE, dict(ws=P + 16)),
    (_lib.AKV_OK, dict(tokens=0)),
])
def test_c_dense_refuses(rc, change):
    assert c_dense(**change) == rc


def c_packed(bits=4, d=64, prep=P, centroids=P, k=P, pitch=32, ws_bytes=1 << 40, tokens=5):
    return _lib.lib().akv_paged_chunk_attn(P, _lib.AKV_BF16, 64, 64, k, pitch, pitch, pitch, P, 1, 1, 1, P, 32, 32, 32, P, 1, 1, 1, P, 0, 2, P, 0, P, 0, prep, centroids, bits,
                                           P, 64, 64, 1, 2, tokens, 8, 2, d, 16, 3, 2, 0, 0.1, P, ws_bytes, None)


@pytest.mark.parametrize("rc,change", [
    (_lib.AKV_ERR_INVALID, dict(bits=5)), (_lib.AKV_ERR_INVALID, dict(bits=1)), (_lib.AKV_ERR_INVALID, dict(prep=None)), (_lib.AKV_ERR_INVALID, dict(centroids=None)),
    (_lib.AKV_ERR_INVALID, dict(k=None)), (_lib.AKV_ERR_UNSUPPORTED, dict(d=512)), (_lib.AKV_ERR_UNSUPPORTED, dict(pitch=33)), (_lib.AKV_ERR_UNSUPPORTED, dict(k=P + 1)),
    (_lib.AKV_ERR_WORKSPACE, dict(ws_bytes=1000)), (_lib.AKV_OK, dict(tokens=0)),
])
def test_c_packed_refuses(rc, change):
    assert c_packed(**change) == rc


def c_rope(d=64, rotary=64, axes=1, sections=None, heads=4, kv=2, dtype=0, cache=0, table=P, positions=P, rows=10, slots=P, key=P, tokens=3, block=16):
    s = (C.c_int * len(sections))(*sections) if sections else None
    return _lib.lib().akv_rope_append(P, 64, 64, P, 64, 64, key, 64, 64, P, 64, 64, dtype, positions, 0, 0, table, rows, rotary, s, axes, 0, slots, 0,
                                      P, 64, 64, 64, P, 64, 64, 64, cache, tokens, heads, kv, d, block, 2, None)


@pytest.mark.parametrize("rc,change", [
    (_lib.AKV_ERR_INVALID, dict(dtype=3)), (_lib.AKV_ERR_INVALID, dict(cache=-1)), (_lib.AKV_ERR_INVALID, dict(rotary=80)), (_lib.AKV_ERR_INVALID, dict(rotary=-16)),
    (_lib.AKV_ERR_INVALID, dict(axes=5)), (_lib.AKV_ERR_INVALID, dict(axes=0)), (_lib.AKV_ERR_INVALID, dict(axes=2)), (_lib.AKV_ERR_INVALID, dict(axes=2, sections=(16, 15))),
    (_lib.AKV_ERR_INVALID, dict(axes=2, sections=(33, -1))), (_lib.AKV_ERR_INVALID, dict(table=None)), (_lib.AKV_ERR_INVALID, dict(positions=None)),
    (_lib.AKV_ERR_INVALID, dict(rows=0)), (_lib.AKV_ERR_INVALID, dict(slots=None)), (_lib.AKV_ERR_INVALID, dict(key=None)), (_lib.AKV_ERR_INVALID, dict(block=0)),
    (_lib.AKV_ERR_UNSUPPORTED, dict(d=72)), (_lib.AKV_ERR_UNSUPPORTED, dict(rotary=24)), (_lib.AKV_ERR_UNSUPPORTED, dict(table=P + 4)),
    (_lib.AKV_OK, dict(tokens=0)), (_lib.AKV_OK, dict(heads=0, kv=0)),
])
def test_c_rope_refuses(rc, change):
    assert c_rope(**change) == rc


def test_forward_chunk_refuses(anywhere):
    class Quantizer:
        rotation, centroids, head_dim, num_levels, bits, _packed_dim = torch.eye(64), torch.zeros(16), 64, 16, 4, 32

    def call(attn=None, **change):
        a = dict(query=torch.zeros(5, 8, 64, dtype=H), k_packed=torch.zeros(3, 16, 2, 32, dtype=torch.uint8), k_norms=torch.zeros(3, 16, 2),
                 v_packed=torch.zeros(3, 16, 2, 32, dtype=torch.uint8), v_norms=torch.zeros(3, 16, 2), block_tables=torch.zeros(2, 2, dtype=torch.int32),
                 context_lens=torch.zeros(2, dtype=torch.int32), query_start_loc=torch.tensor([0, 2, 5]))
        a.update(change)
        return (attn or akv.TQPagedAttention(Quantizer, 8)).forward_chunk(**a)

    with pytest.raises(anywhere, match="workspace"):
        call()
    with pytest.raises(NotImplementedError):
        call(query=torch.zeros(5, 8, 64))
    with pytest.raises(ValueError, match="selector"):
        call(akv.TQPagedAttention(Quantizer, 8, block_selector=object()))
    for change in (dict(query=torch.zeros(5, 4, 64, dtype=H)), dict(query=torch.zeros(5, 8, 128, dtype=H)), dict(query=torch.zeros(5, 512, dtype=H)),
                   dict(k_packed=torch.zeros(3, 16, 2, 31, dtype=torch.uint8)), dict(v_packed=torch.zeros(3, 16, 2, 32)), dict(k_norms=torch.zeros(3, 16)),
                   dict(block_size=32), dict(num_kv_heads=4), dict(num_kv_heads=3), dict(block_tables=torch.zeros(1, 2, dtype=torch.int32)),
                   dict(out=torch.zeros(5, 8, 64)), dict(query_start_loc=torch.zeros(2, 3))):
        with pytest.raises(ValueError):
            call(**change)
    assert ca.check_chunk(torch.zeros(5, 8, 64, dtype=H), 2, torch.zeros(2, 2), torch.zeros(2), torch.zeros(3))[0] == 2
