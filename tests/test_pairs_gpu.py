"""Products on CTA pairs, one quantised call behind the other, with weights that come from memory every time: the pairs of a
call are launched while the quantiser in front of them still holds some of the SMs, one CTA later than its partner."""
import pytest
import torch

pytestmark = pytest.mark.gpu

CALLS = 600


@pytest.fixture(scope="module")
def g():
    import gpu_kernels_b200
    return gpu_kernels_b200


@pytest.mark.timeout(60)
def test_int8_linears_in_a_row(g):
    x = torch.randn((1000, 8192), device="cuda").half()
    weights = [torch.randint(-127, 128, (8192, 8192), dtype=torch.int8, device="cuda") for _ in range(3)]
    scales = torch.rand(8192, device="cuda") * 1e-3
    assert g.int8_tiles(1000, 8192, 8192)["pair"] == 1
    want = [g.int8_linear(x, w, scales) for w in weights]
    last = [None] * 3
    for i in range(CALLS):
        last[i % 3] = g.int8_linear(x, weights[i % 3], scales)
    g.check_int8()
    assert all(torch.equal(a, b) for a, b in zip(last, want))


@pytest.mark.timeout(60)
def test_nvfp4_linears_in_a_row(g):
    x = torch.randn((1000, 8192), device="cuda").bfloat16()
    plans = []
    for _ in range(3):
        b, sb = g.quantize(torch.randn((8192, 8192), device="cuda").bfloat16())
        a, sa = g.quantize(x)
        plans.append(g.Nvfp4Gemm(a, b, sa, sb))
    assert plans[0].info()["launch_cta_group"] == 2
    want = [p.linear(x) for p in plans]
    last = [None] * 3
    for i in range(CALLS):
        last[i % 3] = plans[i % 3].linear(x)
    for p in plans:
        p.validate()
        p.close()
    assert all(torch.equal(a, b) for a, b in zip(last, want))


@pytest.mark.timeout(60)
def test_two_streams_at_once(g):
    # products of both kinds, on pairs and on single CTAs, with nothing between the streams
    x = [torch.randn((m, 4096), device="cuda").bfloat16() for m in (600, 8)]
    w, ws = g.quantize_int8(torch.randn((4096, 4096), device="cuda").bfloat16())
    b, sb = g.quantize(torch.randn((4096, 4096), device="cuda").bfloat16())
    plans = [g.Nvfp4Gemm(*(lambda q: (q[0], b, q[1], sb))(g.quantize(v))) for v in x]
    ids = torch.randint(0, 64, (4000, 4), device="cuda")
    calls = [lambda: g.int8_linear(x[0], w, ws), lambda: plans[0].linear(x[0]), lambda: g.int8_linear(x[1], w, ws),
             lambda: g.sort_routes(ids, 64).source]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [None] * len(calls)
    for _ in range(100):
        for i, (call, stream) in enumerate(zip(calls, streams)):
            with torch.cuda.stream(stream):
                got[i] = call()
    torch.cuda.synchronize()
    g.check_int8()
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    for plan in plans:
        plan.close()
