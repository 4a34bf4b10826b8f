"""int8_linear requests its first weights while its own quantiser runs: behind a kernel that writes these weights and lets its
successor start early (as this library's kernels do, and a copy by torch does not), it must not be given the old ones."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def g():
    import gpu_kernels_b200
    return gpu_kernels_b200


@pytest.mark.parametrize("tokens,n,k", ((4, 4096, 8192), (1, 8192, 4096), (200, 4096, 4096), (600, 8192, 2048)))
def test_weights_from_a_kernel_that_triggers_early(g, tokens, n, k):
    from gpu_kernels_b200 import _lib
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn((tokens, k), generator=gen, device="cuda").bfloat16()
    w = [torch.randn((n, k), generator=gen, device="cuda").bfloat16() for _ in range(2)]
    want = [g.int8_linear(x, *g.quantize_int8(v)) for v in w]
    codes, scales = torch.zeros((n, k), dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
    torch.cuda.synchronize()
    got = []
    for i in range(60):
        _lib.run(x.device, _lib.load().gpu_kernels_int8_quantize, w[i % 2].data_ptr(), 0, codes.data_ptr(), scales.data_ptr(), n, k)
        got.append(g.int8_linear(x, codes, scales))
    g.check_int8()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))
