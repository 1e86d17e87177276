"""What the decoder operators refuse: checked on the host, before anything is launched."""
from ctypes import byref, c_void_p

import pytest
import torch

from llcompiler_b200 import _capi as C

X = c_void_p(1 << 20)      # an address that is never followed: every call here is refused, or has nothing to do


def _fill(p, **kw):
    for k, v in kw.items():
        if k == "sections":
            for i, n in enumerate(v):
                p.sections[i] = n
        else:
            setattr(p, k, v)
    return p


def _rotary(**kw):
    base = dict(x=X, out=X, positions=X, inv_freq=X, dtype=8, pos_dtype=3, tokens=4, heads=2, d=64, pairs=32, x_st=128, x_sh=64, o_st=128, o_sh=64, pos_sa=4, axes=1,
                interleaved=0, sections=[32, 0, 0, 0])
    return _fill(C.LlcRotaryParams(), **{**base, **kw})


def _append(**kw):
    base = dict(k=X, v=X, k_cache=X, v_cache=X, page_table=X, q_start=X, kv_len=X, dtype=8, pos_dtype=3, tokens=4, batch=1, heads=2, kv_heads=2, d=64, pairs=32, num_pages=4,
                page_size=16, table_width=2, table_s0=2, k_st=128, k_sh=64, v_st=128, v_sh=64, kc_sp=2048, kc_sn=128, kc_sh=64, vc_sp=2048, vc_sn=128, vc_sh=64)
    return _fill(C.LlcKvAppendParams(), **{**base, **kw})


def _attend(**kw):
    base = dict(q=X, k_cache=X, v_cache=X, out=X, page_table=X, q_start=X, kv_len=X, dtype=8, scale=0.125, tokens=4, batch=1, heads=4, kv_heads=2, d=64, max_q=4, num_pages=4,
                page_size=16, table_width=2, table_s0=2, q_st=256, q_sh=64, o_st=256, o_sh=64, kc_sp=2048, kc_sn=128, kc_sh=64, vc_sp=2048, vc_sn=128, vc_sh=64)
    return _fill(C.LlcPagedAttentionParams(), **{**base, **kw})


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), 3), (dict(heads=-1), 3), (dict(d=0), 3), (dict(pairs=0), 3), (dict(pairs=33, sections=[33]), 3), (dict(axes=0), 3), (dict(axes=5), 3),
    (dict(sections=[31]), 3), (dict(axes=2, sections=[33, -1]), 3), (dict(dtype=3), 2), (dict(dtype=5), 2), (dict(pos_dtype=4), 2), (dict(x=None), 3), (dict(out=None), 3),
    (dict(positions=None), 3), (dict(inv_freq=None), 3), (dict(heads=1 << 20), 2), (dict(tokens=1 << 31), 2),
])
def test_rotary_refuses(kw, code):
    assert C.lib().llc_cuda_rotary(byref(_rotary(**kw)), None) == code
    assert b"rotary" in C.lib().llc_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), 3), (dict(batch=-1), 3), (dict(kv_heads=0), 3), (dict(page_size=0), 3), (dict(num_pages=-1), 3), (dict(table_width=-1), 3), (dict(dtype=3), 2),
    (dict(k=None), 3), (dict(v=None), 3), (dict(k_cache=None), 3), (dict(page_table=None), 3), (dict(q_start=None), 3), (dict(kv_len=None), 3), (dict(q=X), 3),
    (dict(inv_freq=X, axes=1, sections=[31]), 3), (dict(inv_freq=X, axes=1, pairs=64, sections=[64]), 3), (dict(inv_freq=X, positions=X, axes=1, sections=[32], pos_dtype=4), 2),
    (dict(tokens=1 << 31), 2), (dict(page_size=1 << 21), 2),
])
def test_append_refuses(kw, code):
    assert C.lib().llc_cuda_kv_append(byref(_append(**kw)), None) == code
    assert b"kv_append" in C.lib().llc_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(tokens=-1), 3), (dict(batch=-1), 3), (dict(heads=0), 3), (dict(kv_heads=0), 3), (dict(heads=5), 3), (dict(d=0), 3), (dict(d=257), 2), (dict(max_q=-1), 3),
    (dict(window=-1), 3), (dict(sinks=-1), 3), (dict(page_size=0), 3), (dict(dtype=3), 2), (dict(q=None), 3), (dict(out=None), 3), (dict(k_cache=None), 3), (dict(v_cache=None), 3),
    (dict(page_table=None), 3), (dict(q_start=None), 3), (dict(kv_len=None), 3), (dict(page_size=1 << 20, table_width=1 << 20), 2), (dict(tokens=1 << 31), 2),
    (dict(workspace=c_void_p((1 << 20) + 8), workspace_bytes=1 << 20), 3),
])
def test_attention_refuses(kw, code):
    p = _attend(**kw)
    assert C.lib().llc_cuda_paged_attention(byref(p), None) == code
    assert b"paged_attention" in C.lib().llc_last_error()


def test_null_blocks_and_calls_with_nothing_to_do():
    L = C.lib()
    assert L.llc_cuda_rotary(None, None) == 3 and L.llc_cuda_kv_append(None, None) == 3 and L.llc_cuda_paged_attention(None, None) == 3
    assert L.llc_cuda_paged_attention_workspace(None) == 0
    assert L.llc_cuda_rotary(byref(_rotary(tokens=0)), None) == 0 and L.llc_cuda_rotary(byref(_rotary(heads=0)), None) == 0
    assert L.llc_cuda_kv_append(byref(_append(tokens=0)), None) == 0 and L.llc_cuda_kv_append(byref(_append(batch=0)), None) == 0
    for kw in (dict(tokens=0), dict(batch=0), dict(max_q=0)):
        assert L.llc_cuda_paged_attention(byref(_attend(**kw)), None) == 0


def test_python_entry_points_refuse_host_tensors_and_wrong_types():
    from llcompiler_b200.executor import kv_append, paged_attention, rotary
    x = torch.zeros(3, 2, 64)
    cache, table, ends, lens = torch.zeros(2, 16, 2, 64), torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3], dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU fallback"):
        rotary(x, torch.arange(3), torch.ones(32, dtype=torch.float64))
    with pytest.raises(ValueError, match="no CPU fallback"):
        kv_append(x, x, cache, cache, table, ends, lens)
    with pytest.raises(ValueError, match="no CPU fallback"):
        paged_attention(x, cache, cache, table, ends, lens)
    with pytest.raises(TypeError):
        rotary([1.0], torch.arange(3), torch.ones(32, dtype=torch.float64))
