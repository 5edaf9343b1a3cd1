"""CPU checks of the token mixers' boundary: what the C entries refuse before they touch a device, and what the Python
entries refuse without one."""
import pytest
import torch


def lib():
    from reax_engine_runtime_v3_b200 import _native
    return _native.load()


def prefill(**kw):
    a = dict(rows=0, batch=1, hk=2, hv=4, dk=128, dv=128, slots=1, ldq=256, ldk=256, ldv=512)
    a.update(kw)
    return lib().reax_gdn_prefill(*[None] * 9, a["rows"], a["batch"], a["hk"], a["hv"], a["dk"], a["dv"], a["slots"], a["ldq"],
                                  a["ldk"], a["ldv"], 1.0, 1, 1, None, 0, None)


def test_gated_delta_entry_refuses():
    assert prefill() == 0                                       # no rows: nothing to do
    assert prefill(rows=5, batch=0) == 0
    for bad, word in ((dict(hv=3), b"multiple"), (dict(dk=96), b"64 or 128"), (dict(rows=-1), b"rows -1"),
                      (dict(ldv=500), b"row stride"), (dict(rows=4), b"NULL"), (dict(batch=70000), b"at most")):
        assert prefill(**bad) == 1 and word in lib().reax_last_error(), bad
    assert lib().reax_gdn_decode(*[None] * 8, 0, 2, 4, 128, 128, 1, 256, 256, 512, 1.0, 1, None) == 0
    assert lib().reax_gdn_decode(*[None] * 8, 1, 2, 4, 128, 32, 1, 256, 256, 512, 1.0, 1, None) == 1


def test_cache_entries_refuse():
    L = lib()
    append = lambda rows, batch, pages, heads, page, dim, cu=None: L.reax_kv8_append(
        *[None] * 8, cu, rows, batch, 4, pages, heads, page, dim, heads * dim, heads * dim, None)
    assert append(0, 0, 4, 2, 64, 128) == 0
    assert append(3, 2, 4, 2, 64, 128) == 1 and b"NULL" in L.reax_last_error()
    assert append(-1, 2, 4, 2, 64, 128) == 1 and b"negative" in L.reax_last_error()
    attend = lambda rows, batch: L.reax_kv8_attend(*[None] * 10, rows, 1, batch, 4, 4, 2, 4, 64, 128, 1024, 1.0, None, 0, None)
    assert attend(0, 3) == 0
    assert attend(2, 2) == 1
    assert L.reax_mixer_status(None, 0, None) == 1


def test_python_entries_refuse_without_a_gpu():
    from reax_engine_runtime_v3_b200 import gated_delta
    from reax_engine_runtime_v3_b200.kv_int8 import Int8Cache
    q = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    v = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    g = torch.zeros(3, 4)
    state = torch.zeros(3, 4, 128, 128)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gated_delta.decode(q, q, v, g, g, state)
    with pytest.raises(AssertionError, match="contiguous float32"):
        gated_delta.decode(q, q, v, g, g, state.transpose(2, 3))
    with pytest.raises(AssertionError, match="float32"):
        gated_delta.prefill(q, q, v, g.bfloat16(), g, state)
    with pytest.raises(AssertionError, match="cu_seqlens|slots|states"):
        gated_delta.prefill(q, q, v, g, g, state[:1], cu_seqlens=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        Int8Cache.empty(2, 1, 64, device="cpu")
