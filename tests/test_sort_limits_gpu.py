"""sort_routes at the sizes whose shared memory needs the function's limit raised."""
import subprocess
import sys

import pytest

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
