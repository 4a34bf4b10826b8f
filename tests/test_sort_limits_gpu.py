"""sort_routes at the sizes whose shared memory needs the function's limit raised."""
import subprocess
import sys
import threading

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


FIRST_CALLS = """
import torch
import gpu_kernels_b200 as g
for dtype in (torch.int64, torch.int32):
    for experts in (360, 359, 361):
        for tokens in (257, 5000):
            ids = torch.randint(-1, experts, (tokens, 1), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
            offsets, position, source = g.sort_routes(ids.to(dtype), experts)
            key = torch.where(ids >= 0, ids, experts).flatten()
            want = torch.argsort(key, stable=True)
            assert torch.equal(source.long(), want)
            assert torch.equal(position.flatten()[want].long(), torch.arange(tokens, device="cuda"))
            assert torch.equal(offsets.long(), torch.searchsorted(key[want], torch.arange(experts + 1, device="cuda")))
"""


def test_first_calls_of_a_process():
    # 360 experts: the counters alone fit the 48 KB that need no limit, with the kernel's static memory they do not
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


def test_threads_with_different_numbers_of_experts():
    # The limit is one for all threads of a process. Through the C ABI: the calls follow each other closely enough to meet.
    from gpu_kernels_b200 import _lib
    lib, routes, refused = _lib.load(), 300, []

    def sort(experts):
        ids = torch.randint(0, experts, (routes,), device="cuda")
        offsets = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
        position, source = (torch.empty(routes, dtype=torch.int32, device="cuda") for _ in range(2))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        args = (ids.data_ptr(), 8, routes, experts, offsets.data_ptr(), position.data_ptr(), source.data_ptr(), None, stream.cuda_stream)
        refused.extend(experts for _ in range(10000) if lib.gpu_kernels_tokens_sort(*args))
        stream.synchronize()
        if not torch.equal(source.long(), torch.argsort(ids, stable=True)):
            refused.append(-experts)

    threads = [threading.Thread(target=sort, args=(experts,)) for experts in (400, 1024, 512, 1024)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not refused
