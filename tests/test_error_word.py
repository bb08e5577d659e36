"""The word that kernels record errors in: one to a device, whoever asks for it
first and when."""

import os
import subprocess
import sys
import threading
import time

import pytest
import torch

from flashmap_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_threads_get_one_word(monkeypatch):
    """Calls that ask for a device's word at the same time all get the one that is kept."""
    device, zeros = torch.device("cpu", 7), torch.zeros

    def slow(*a, **k):
        time.sleep(0.05)
        return zeros(*a, **k)

    monkeypatch.setattr(torch, "zeros", slow)
    got, start = [], threading.Barrier(4)

    def ask():
        start.wait()
        got.append(ops.error_word(device))

    threads = [threading.Thread(target=ask) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and len({w.data_ptr() for w in got}) == 1
    assert got[0].data_ptr() == ops.error_word(device).data_ptr() == ops._error_address(device)


def test_word_outlives_inference_mode():
    device = torch.device("cpu", 8)
    with torch.inference_mode():
        w = ops.error_word(device)
    w.zero_()
    assert not w.is_inference()


FIRST = """
import torch
from flashmap_b200 import _lib, cache_ops, ops
x = torch.randn(2, 500, device="cuda")
good, bad = torch.tensor([3, 4], device="cuda"), torch.tensor([3, 900], device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.inference_mode(), torch.cuda.graph(graph):
    held = ops.token_logprobs(x, good, top_k=2)
cache_ops.check_device_errors()  # nothing has run
ops.token_logprobs(x, bad)
graph.replay()  # leaves what was recorded
torch.cuda.synchronize()
want = ops.token_logprobs(x, good, top_k=2)
assert all(torch.equal(a, b) for a, b in zip(held, want))
try:
    cache_ops.check_device_errors()
except _lib.FlashMapError:
    cache_ops.check_device_errors()  # cleared
    print("as it should be")
"""


@pytest.mark.gpu
def test_first_call_of_a_process_is_captured():
    run = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and run.stdout.strip() == "as it should be", run.stdout + run.stderr[-2000:]


@pytest.mark.gpu
def test_words_of_the_library_and_of_calls():
    from flashmap_b200 import cache_ops
    device = torch.device("cuda", torch.cuda.current_device())
    w = ops.error_word("cuda")
    assert w.is_cuda and w.dtype == torch.int32 and w.shape == (1,) and w is ops.error_word(device)
    assert w.data_ptr() == ops._error_address(device) == cache_ops._err_word(device)
    w.fill_(3)
    with pytest.raises(RuntimeError):
        cache_ops.check_device_errors()
    assert int(w) == 0
