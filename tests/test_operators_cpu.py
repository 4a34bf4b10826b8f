"""The int8 and token-routing operators without a GPU: symbols, and refusals that need none."""
import ctypes
import re

import pytest
import torch

from conftest import ROOT


def declared_symbols():
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "operators_capi.h").read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(gpu_kernels_(?:int8|tokens)_\w+)\s*\(", text)))


def test_symbols_are_exported_and_bound():
    from gpu_kernels_b200 import _lib, build
    lib = ctypes.CDLL(str(build.build()))
    names = declared_symbols()
    assert len(names) == 12 and sorted(_lib.OPERATOR_SIGNATURES) == names
    for name in names:
        assert hasattr(lib, name), name


def test_fails_loudly_without_gpu():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    from gpu_kernels_b200 import _lib
    with pytest.raises(_lib.Nvfp4Error):
        _lib.check(_lib.load().gpu_kernels_int8_quantize(None, 0, None, None, 1, 16, None))
    with pytest.raises(_lib.Nvfp4Error):
        _lib.check(_lib.load().gpu_kernels_tokens_sort(None, 8, 0, 4, None, None, None, None, None))


def test_cpu_tensors_are_refused():
    import gpu_kernels_b200 as g
    i8, f = torch.zeros((16, 32), dtype=torch.int8), torch.zeros(16)
    ids = torch.zeros((4, 2), dtype=torch.int64)
    routes = g.Routes(torch.zeros(3, dtype=torch.int32), torch.zeros((4, 2), dtype=torch.int32), torch.zeros(8, dtype=torch.int32))
    for call in (lambda: g.quantize_int8(torch.zeros(4, 16)), lambda: g.dequantize_int8(i8, f), lambda: g.int8_gemm(i8, i8, f, f),
                 lambda: g.int8_linear(torch.zeros(4, 32), i8, f),
                 lambda: g.int8_grouped_gemm(i8, i8[None], f, f[None], torch.zeros(2, dtype=torch.int32)),
                 lambda: g.sort_routes(ids, 2), lambda: g.gather_tokens(torch.zeros(4, 8), routes),
                 lambda: g.gather_tokens_int8(torch.zeros(4, 16), routes), lambda: g.combine_tokens(torch.zeros(8, 8), routes)):
        with pytest.raises(ValueError):
            call()
