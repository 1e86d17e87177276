"""The extension's side of the decoder operators, as far as it needs no GPU."""
import os
import subprocess
import sys
import types

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FIRST_CALLS = """
import builtins, threading, time
import torch
from llcompiler_b200.executor import rotary
real = builtins.__import__
def slow(name, *a, **k):            # another thread gets the interpreter while the first call sets itself up
    if name.startswith("torch"): time.sleep(0.3)
    return real(name, *a, **k)
builtins.__import__ = slow
def call():
    try: rotary(torch.zeros(3, 2, 64), torch.arange(3), torch.ones(32, dtype=torch.float64))
    except ValueError as e: print("refused", flush=True)
threads = [threading.Thread(target=call) for _ in range(3)]
for t in threads: t.start()
for t in threads: t.join()
"""


def test_first_calls_of_several_threads_at_once():
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.count("refused") == 3, r.stderr[-2000:]


@pytest.mark.parametrize("code,said", [(-1, "cannot be read"), (2, "matrix product"), (7, "of attention"), (9, "paged cache"), (12, "paged cache .* 12")])
def test_a_failure_that_a_kernel_recorded_is_raised(monkeypatch, code, said):
    from llcompiler_b200.executor import device_status, paged
    monkeypatch.setattr(paged, "_ops", types.SimpleNamespace(status=lambda: code))
    with pytest.raises(RuntimeError, match=said):
        device_status()
    monkeypatch.setattr(paged, "_ops", types.SimpleNamespace(status=lambda: 0))
    assert device_status() == 0


@pytest.mark.parametrize("d,group", [(64, 4), (128, 16), (128, 32)])
def test_the_workspace_does_not_grow_with_the_batch(d, group):
    """At most two pairs of (sequence, key head) are cut by a warp's share of the keys: a page of sums for each of those, and eight bytes a pair."""
    from ctypes import byref, c_void_p

    from llcompiler_b200 import _capi as C
    sizes = []
    for batch in (1, 64, 4096):
        p = C.LlcPagedAttentionParams()
        at = c_void_p(1 << 20)                                # never followed
        p.q = p.k_cache = p.v_cache = p.out = p.page_table = p.q_start = p.kv_len = at
        p.dtype, p.scale, p.tokens, p.batch, p.heads, p.kv_heads, p.d, p.max_q = 8, 0.125, batch, batch, 8 * group, 8, d, 1
        p.num_pages, p.page_size, p.table_width, p.table_s0 = 1 << 16, 64, 256, 256
        p.q_st = p.o_st = 8 * group * d
        p.q_sh = p.o_sh = d
        p.kc_sp = p.vc_sp = 64 * 8 * d
        p.kc_sn = p.vc_sn = 8 * d
        p.kc_sh = p.vc_sh = d
        sizes.append(C.lib().llc_cuda_paged_attention_workspace(byref(p)) - (8 * 8 * batch + 15) // 16 * 16)
    assert sizes[0] > 0 and sizes[0] == sizes[1] == sizes[2]
