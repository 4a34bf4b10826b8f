"""What the routing operators hand to their kernels, with the launches replaced: no GPU is needed."""
import ctypes
import weakref

import pytest
import torch
import torch.autograd.forward_ad as fw


class Launches:
    """Stands for `_lib.run`: checks, at each launch, that no address it is given lies in memory nobody holds any more.
    `copy` makes the tensors that are looked after, in memory that lives as long as their storage. A size has to fit the type
    it is handed over in, where ctypes would cut it."""

    def __init__(self):
        self.memory, self.calls = [], 0

    def copy(self, t):
        array = t.detach().numpy().copy()
        self.memory.append((array.ctypes.data, array.nbytes, weakref.ref(array)))
        return torch.from_numpy(array)

    def __call__(self, device, fn, *args):
        self.calls += 1
        lost = [a for a in args for at, size, ref in self.memory if ref() is None and isinstance(a, int) and at <= a < at + size]
        assert not lost, "a launch is given memory that nobody holds"
        cut = [a for a, kind in zip(args, fn.argtypes) if kind is ctypes.c_int and kind(a).value != a]
        assert not cut, "a launch is given a size that is cut"


@pytest.fixture
def launches(monkeypatch):
    from gpu_kernels_b200 import _lib, int8, tokens
    stub = Launches()
    monkeypatch.setattr(_lib, "run", stub)
    for module in (int8, tokens):
        monkeypatch.setattr(module, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(int8, "_operand", lambda t, name, dim, device=None: None)
    return stub


def order(tokens, topk):
    """The order of a batch that one expert takes."""
    import gpu_kernels_b200 as g
    routes = torch.arange(tokens * topk, dtype=torch.int32)
    return g.Routes(torch.tensor([0, tokens * topk], dtype=torch.int32), routes.view(tokens, topk).clone(), routes)


@pytest.mark.parametrize("what,weighted", (("gather", None), ("combine", None), ("combine", "rows"), ("combine", "weights"), ("combine", "both")))
def test_backward_holds_what_its_launch_reads(launches, what, weighted):
    # Saved tensors that hooks give back (as save_on_cpu and checkpointing do) belong to the backward pass alone.
    import gpu_kernels_b200 as g
    tokens, topk, hidden = 6, 3, 8
    routes = order(tokens, topk)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, launches.copy):
        if what == "gather":
            leaf = torch.ones((tokens, hidden), requires_grad=True)
            out = g.gather_tokens(leaf, routes)
        else:
            leaf = torch.ones((tokens * topk, hidden), requires_grad=weighted != "weights")
            weights = None if weighted is None else torch.ones((tokens, topk), requires_grad=weighted != "rows")
            out = g.combine_tokens(leaf, routes, weights)
    before = launches.calls
    out.backward(torch.ones_like(out))
    assert launches.calls == before + 1 and len(launches.memory) >= 2


def test_tangents_are_refused(launches):
    import gpu_kernels_b200 as g
    routes = order(6, 3)
    x, rows, w = torch.ones((6, 8)), torch.ones((18, 8)), torch.ones((6, 3))
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: g.gather_tokens(dual(x), routes), lambda: g.combine_tokens(dual(rows), routes, w),
                     lambda: g.combine_tokens(dual(rows), routes), lambda: g.combine_tokens(rows, routes, dual(w)),
                     lambda: g.combine_tokens(rows, routes, dual(w.double()))):
            with pytest.raises(NotImplementedError):
                call()
        # plain tensors inside a level are as they are outside
        assert g.gather_tokens(x, routes).shape == (18, 8) and g.combine_tokens(rows, routes, w).shape == (6, 8)


FAR = (1 << 32) + 16                                            # 16, where it is cut to 32 bits


def test_sizes_beyond_31_bits_are_refused(launches):
    import gpu_kernels_b200 as g
    empty = lambda *shape, dtype=torch.int8: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    routes = g.Routes(empty(9, dtype=i32), empty(FAR, 1, dtype=i32), empty(FAR, dtype=i32))
    few = g.Routes(empty(9, dtype=i32), empty(8, 2, dtype=i32), empty(16, dtype=i32))
    scales = lambda *shape: empty(*shape, dtype=f32)  # noqa: E731
    for call in (lambda: g.quantize_int8(empty(2, FAR, dtype=bf16)),
                 lambda: g.dequantize_int8(empty(2, FAR), scales(2)),
                 lambda: g.int8_gemm(empty(FAR, 16), empty(16, 16), scales(FAR), scales(16)),
                 lambda: g.int8_gemm(empty(16, 16), empty(FAR, 16), scales(16), scales(FAR)),
                 lambda: g.int8_gemm(empty(16, 16), empty(FAR, 16), scales(16), scales(FAR), out=empty(16, FAR, dtype=bf16)),
                 lambda: g.int8_linear(empty(FAR, 16, dtype=bf16), empty(16, 16), scales(16)),
                 lambda: g.int8_linear(empty(16, 16, dtype=bf16), empty(FAR, 16), scales(FAR)),
                 lambda: g.int8_grouped_gemm(empty(FAR, 16), empty(8, 16, 16), scales(FAR), scales(8, 16), empty(9, dtype=i32)),
                 lambda: g.int8_tiles(FAR, 16, 16), lambda: g.int8_tiles(16, FAR, 16), lambda: g.int8_tiles(16, 16, FAR),
                 lambda: g.int8_tiles(16, 16, 16, FAR),
                 lambda: g.sort_routes(empty(FAR, 1, dtype=i32), 8),
                 lambda: g.gather_tokens(empty(FAR, 8, dtype=bf16), routes),
                 lambda: g.gather_tokens(empty(8, FAR, dtype=bf16), few),
                 lambda: g.gather_tokens_int8(empty(8, FAR, dtype=bf16), few),
                 lambda: g.combine_tokens(empty(FAR, 8, dtype=bf16), routes),
                 lambda: g.combine_tokens(empty(16, FAR, dtype=bf16), few, scales(8, 2))):
        with pytest.raises(ValueError):
            call()
