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
