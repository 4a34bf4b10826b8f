"""Int8 quantiser and products against their definitions in 64 bits.

Rounding to a type is off by at most eps / 2 of the value. A product's exact integer sum is converted to FP32 and
multiplied by two scales: three roundings of 2^-24, and one to the output's type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def g():
    import gpu_kernels_b200
    return gpu_kernels_b200


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype, seed, sigma=1.0):
    return (torch.randn(shape, generator=generator(seed), device="cuda") * sigma).to(dtype)


def random_codes(shape, seed):
    return torch.randint(-128, 128, shape, generator=generator(seed), device="cuda", dtype=torch.int8)


def random_scales(shape, seed):
    return torch.rand(shape, generator=generator(seed), device="cuda") * 1e-2 + 1e-4


def codes_of(x):
    """The definition: nearest integers to 127 x / amax, ties to even. 64-bit quotients of 32-bit values that are no tie
    are never rounded onto one."""
    amax = x.abs().amax(1).double()
    quotient = torch.where(amax[:, None] > 0, 127.0 * x.double() / amax[:, None], 0.0)
    return torch.round(quotient).to(torch.int8), (amax / 127.0).float()     # (a 32-bit tensor over a number is a product in torch)


def check_quantised(g, x):
    codes, scales = g.quantize_int8(x)
    want, want_scales = codes_of(x)
    assert torch.equal(codes, want)
    assert torch.equal(scales, want_scales)
    assert torch.equal(g.dequantize_int8(codes, scales), codes.float() * scales[:, None])


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("rows,k", ((1, 1), (3, 7), (9, 16), (5, 17), (33, 63), (17, 512), (10, 513), (4, 2048), (3, 2051),
                                    (3, 4096), (2, 8192), (2, 8191), (3, 16384), (2, 20000), (2, 32768), (2, 40001),
                                    (11, 1040), (3, 1552), (3, 2064), (3, 4112), (2, 4104), (2, 8784), (2, 8200), (2, 12304), (2, 14336),
                                    (2, 16400), (2, 24592), (1, 16), (65, 48), (70, 64), (33, 80), (100, 128), (17, 144), (31, 256), (9, 272), (300, 1), (70, 15),
                                    (65, 31), (33, 100), (37, 127), (33, 143), (35, 145), (50, 250), (17, 271), (18, 273)))
def test_quantise(g, rows, k, dtype):
    check_quantised(g, normal((rows, k), dtype, rows * 7 + k))


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
def test_values_on_the_borders(g, dtype):
    # with amax = 254, 63.5 times a power of two and so on, 127 x / amax is x / 2: a tie at every odd x
    x = torch.arange(-254, 255, device="cuda", dtype=torch.float64).repeat(6, 1)
    for i, power in enumerate((0, 3, -7, 5, -11, 1)):
        x[i] *= 2.0 ** power
    assert torch.equal(x.to(dtype).double(), x)
    check_quantised(g, x.to(dtype))


def test_fp32_neighbours_of_borders(g):
    # amax = 3, 1.7, ...: every tie of the row, and the FP32 values around it
    rows = []
    for amax in (3.0, 1.7, 0.011, 254.0, 12345.678):
        a = torch.tensor(amax, device="cuda", dtype=F32)
        tie = ((torch.arange(127, device="cuda", dtype=torch.float64) + 0.5) * a.double() / 127.0).float()
        near = [tie]
        for toward in (torch.inf, -torch.inf):
            t = tie
            for _ in range(3):
                t = torch.nextafter(t, torch.full_like(t, toward))
                near.append(t)
        near = torch.cat(near).clamp(max=float(a))
        rows.append(torch.cat((near, -near, a[None])))
    check_quantised(g, torch.stack(rows))


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
def test_extreme_rows(g, dtype):
    info = torch.finfo(dtype)
    x = normal((6, 48), dtype, 5)
    x[0] = 0
    x[1] = torch.linspace(-1, 1, 48, device="cuda") * info.max
    x[2] = (torch.linspace(-1, 1, 48, device="cuda", dtype=torch.float64) * info.smallest_normal).to(dtype)
    x[3] = 0
    x[3, 7] = info.smallest_normal * info.eps                   # the smallest subnormal
    x[4, 0] = info.max
    check_quantised(g, x)
    codes, scales = g.quantize_int8(x)
    assert scales[0] == 0 and not codes[0].any()


@pytest.mark.parametrize("bad", (float("nan"), float("inf"), -float("inf")))
@pytest.mark.parametrize("dtype", (BF16, F32))
def test_row_that_is_not_finite(g, dtype, bad):
    x = normal((3, 40), dtype, 3)
    x[1, 13] = bad
    codes, scales = g.quantize_int8(x)
    assert scales.isnan().tolist() == [False, True, False] and not codes[1].any()
    w, ws = g.quantize_int8(normal((16, 48), BF16, 4))
    y = g.int8_linear(torch.nn.functional.pad(x, (0, 8)), w, ws)
    assert y[1].isnan().all() and y[[0, 2]].isfinite().all()


def test_strides_alignment_and_other_types(g):
    x = normal((9, 64), BF16, 6)
    want, scales = g.quantize_int8(x)
    for same in (x.t().contiguous().t(), torch.cat((x, x), 1)[:, :64], x.double(),
                 torch.cat((x.flatten()[:3], x.flatten()))[3:].view(9, 64)):
        codes, s = g.quantize_int8(same)
        assert torch.equal(codes, want) and torch.equal(s, scales)
    none = g.quantize_int8(x[:0])
    assert none[0].shape == (0, 64) and none[1].shape == (0,) and g.dequantize_int8(*none).shape == (0, 64)


# ---- products -----------------------------------------------------------------------------------------------------


def exact(a, b, sa, sb):
    return (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()


def assert_product(c, want):
    """Three roundings of 2^-24 (and 2^-47 for their products), one to c's type (fp16: at least half its smallest step)."""
    own = 0.0 if c.dtype == F32 else torch.finfo(c.dtype).eps / 2
    bound = want.abs() * ((1 + 3.01 * 2.0 ** -24) * (1 + own) - 1) + (2.0 ** -25 if c.dtype == F16 else 0.0)
    off = (c.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / want.abs().clamp(min=1e-30)).max()):.3e} at most"


SIZES = ((1, 8, 16), (1, 128, 128), (2, 136, 4096), (7, 264, 144), (16, 1024, 4096), (17, 512, 2064), (64, 200, 2048),
         (96, 2048, 8192), (128, 1000, 512), (130, 384, 272), (200, 136, 1040), (256, 512, 1024), (257, 520, 400),
         (300, 1000, 992), (513, 2056, 640), (700, 264, 3184), (1024, 1024, 1024),
         (48, 1000, 4096), (65, 1024, 8192), (2885, 64, 4112), (300, 520, 8192), (128, 520, 16384), (130, 2048, 16384), (640, 136, 5008), (9, 8192, 4096), (5, 18944, 1024), (128, 28672, 272), (300, 8200, 528))


@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(g, m, n, k):
    a, b = random_codes((m, k), m + k), random_codes((n, k), n + k + 1)
    sa, sb = random_scales((m,), 1), random_scales((n,), 2)
    want = exact(a, b, sa, sb)
    for dtype in (F32, BF16, F16):
        out = torch.full((m + 2, n), float("nan"), dtype=dtype, device="cuda")
        c = g.int8_gemm(a, b, sa, sb, out=out[1:m + 1])
        g.check_int8()
        assert_product(c, want)
        assert out[0].isnan().all() and out[m + 1].isnan().all()


@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("m, n, k, ahead", ((3, 8, 16, 16), (131, 136, 64, 16), (258, 520, 144, 16), (257, 272, 144, 48), (513, 1048, 256, 32)))
def test_rows_of_c_on_16_byte_boundaries(g, m, n, k, ahead, dtype):
    a, b, sa, sb = random_codes((m, k), m), random_codes((n, k), n), random_scales((m,), 1), random_scales((n,), 2)
    guard = ahead // dtype.itemsize
    memory = torch.full((guard + m * n + 256,), float("nan"), dtype=dtype, device="cuda")
    out = memory[guard:guard + m * n].view(m, n)
    g.int8_gemm(a, b, sa, sb, out=out)
    assert_product(out, exact(a, b, sa, sb))
    assert memory[:guard].isnan().all() and memory[guard + m * n:].isnan().all()


def test_every_kernel_is_reached(g):
    tiles = [g.int8_tiles(*size) for size in SIZES]
    assert {(t["pair"], t["swap"]) for t in tiles} == {(1, 0), (0, 0), (0, 1)}
    assert {t["split"] for t in tiles if t["swap"]} == {1, 2, 4, 8}
    assert {t["split"] for t in tiles if not t["swap"] and not t["pair"]} >= {1, 2, 4, 8}
    assert {t["width"] for t in tiles if t["swap"]} >= {16, 32, 48} and len({t["width"] for t in tiles if t["pair"]}) >= 3


@pytest.mark.parametrize("m", (1, 300))
def test_longest_sum(g, m):
    # K * 128 * 128 just below 2^31, all of one sign
    k = 131056
    a, b = torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.full((16, k), -128, dtype=torch.int8, device="cuda")
    b[8:] = 127
    sa, sb = torch.ones(m, device="cuda"), torch.ones(16, device="cuda")
    c = g.int8_gemm(a, b, sa, sb, out_dtype=F32)
    assert torch.equal(c[:, :8], torch.full((m, 8), float(k * 16384), device="cuda"))
    assert_product(c, exact(a[:1], b, sa[:1], sb).expand(m, 16))


@pytest.mark.parametrize("dtype,out", ((BF16, None), (F16, F32), (F32, BF16)))
@pytest.mark.parametrize("m,n,k", ((1, 4096, 4096), (5, 72, 48), (33, 1024, 8192), (300, 512, 1024), (1000, 1032, 2000), (400, 1536, 8208), (2000, 72, 4112)))
def test_linear_is_quantise_then_product(g, m, n, k, dtype, out):
    x = normal((m, k), dtype, m)
    w, ws = g.quantize_int8(normal((n, k), BF16, n, 0.02))
    c = g.int8_linear(x, w, ws, out_dtype=out)
    codes, scales = g.quantize_int8(x)
    assert c.dtype == (out or dtype)
    assert torch.equal(c, g.int8_gemm(codes, w, scales, ws, out_dtype=c.dtype))
    g.check_int8()


def test_linear_reads_weights_written_just_before(g):
    # the product's early loads must not overtake the kernel in front of the quantiser
    x = normal((4, 8192), BF16, 1)
    w, ws = torch.empty((4096, 8192), dtype=torch.int8, device="cuda"), torch.ones(4096, device="cuda")
    first, second = random_codes(w.shape, 1), random_codes(w.shape, 2)
    codes, scales = g.quantize_int8(x)
    want = [g.int8_gemm(codes, b, scales, ws) for b in (first, second)]
    for i in range(20):
        w.copy_((first, second)[i % 2])
        assert torch.equal(g.int8_linear(x, w, ws), want[i % 2])


def reference_grouped(rows, weights, row_scales, weight_scales, offsets):
    out = torch.zeros((rows.shape[0], weights.shape[1]), dtype=torch.float64, device="cuda")
    for e in range(weights.shape[0]):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        out[lo:hi] = exact(rows[lo:hi], weights[e], row_scales[lo:hi], weight_scales[e])
    return out


GROUPED = (([0, 1], 8, 16), ([0, 0, 3, 3, 20, 20], 136, 144), ([0, 1, 2, 3, 4, 5, 6], 1024, 512), ([0, 40, 41, 200, 333], 264, 400),
           ([0, 700, 700, 1500], 520, 272), ([0] * 100 + [129], 128, 256), ([0, 0, 0, 0], 64, 64), ([3, 10, 17], 64, 64),
           ([0, 300, 600, 1300, 1301], 256, 1040))


@pytest.mark.parametrize("offsets,n,k", GROUPED)
def test_grouped_product(g, offsets, n, k):
    experts, r = len(offsets) - 1, offsets[-1] + 5
    rows, weights = random_codes((r, k), 1), random_codes((experts, n, k), 2)
    sr, sw = random_scales((r,), 3), random_scales((experts, n), 4)
    where = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    want = reference_grouped(rows, weights, sr, sw, offsets)
    for dtype in (F32, BF16):
        out = torch.full((r, n), 7.0, dtype=dtype, device="cuda")
        c = g.int8_grouped_gemm(rows, weights, sr, sw, where, out=out)
        g.check_int8()
        assert_product(c[offsets[0]:offsets[-1]], want[offsets[0]:offsets[-1]])
        assert bool((c[:offsets[0]] == 7.0).all()) and bool((c[offsets[-1]:] == 7.0).all())
    fresh = g.int8_grouped_gemm(rows, weights, sr, sw, where, out_dtype=BF16)
    assert torch.equal(fresh[offsets[0]:offsets[-1]], c[offsets[0]:offsets[-1]])
    assert not fresh[offsets[-1]:].any() and not fresh[:offsets[0]].any()


def test_grouped_takes_both_kernels(g):
    assert not g.int8_tiles(384, 4096, 4096, 256)["pair"] and g.int8_tiles(1505, 520, 272, 3)["pair"]


@pytest.mark.parametrize("experts", (33, 1024))
def test_grouped_many_experts(g, experts):
    counts = torch.randint(0, 4, (experts,), generator=generator(experts), device="cuda")
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0))).int()
    r, n, k = int(offsets[-1]), 40, 160
    rows, weights = random_codes((r, k), 1), random_codes((experts, n, k), 2)
    sr, sw = random_scales((r,), 3), random_scales((experts, n), 4)
    assert_product(g.int8_grouped_gemm(rows, weights, sr, sw, offsets, out_dtype=F32),
                   reference_grouped(rows, weights, sr, sw, offsets.tolist()))


def test_grouped_offsets_that_make_no_sense_stay_in_bounds(g):
    # clipped to the rows, and where they decrease the largest so far counts
    rows, weights = random_codes((50, 64), 1), random_codes((4, 72, 64), 2)
    sr, sw = random_scales((50,), 3), random_scales((4, 72), 4)
    c = g.int8_grouped_gemm(rows, weights, sr, sw, torch.tensor([-5, 20, 10, 90, 30], dtype=torch.int32, device="cuda"), out_dtype=F32)
    g.check_int8()
    assert_product(c, reference_grouped(rows, weights, sr, sw, [0, 20, 20, 50, 50]))


def test_matrices_beyond_31_bits(g):
    # 70001 x 30808 values: the last rows lie behind element 2^31
    rows, k, tail = 70001, 30808, slice(69990, None)
    x = torch.empty((rows, k), dtype=BF16, device="cuda").normal_(generator=generator(1))
    codes, scales = g.quantize_int8(x)
    want, want_scales = codes_of(x[tail])
    del x
    assert torch.equal(codes[tail], want) and torch.equal(scales[tail], want_scales)
    assert torch.equal(g.dequantize_int8(codes, scales)[tail], codes[tail].float() * scales[tail, None])
    del codes
    a, b = random_codes((rows, 32), 2), random_codes((k, 32), 3)
    sa, sb = random_scales((rows,), 4), random_scales((k,), 5)
    assert_product(g.int8_gemm(a, b, sa, sb)[tail], exact(a[tail], b, sa[tail], sb))
    offsets = torch.tensor([0, 30000, 69995, 70001], dtype=torch.int32, device="cuda")
    b3, sb3 = torch.stack((b, b, b.flip(0))), torch.stack((sb, sb, sb.flip(0)))
    c = g.int8_grouped_gemm(a, b3, sa, sb3, offsets)
    assert_product(c[69990:69995], exact(a[69990:69995], b, sa[69990:69995], sb))
    assert_product(c[69995:], exact(a[69995:], b.flip(0), sa[69995:], sb.flip(0)))


def test_no_rows(g):
    b, sb = random_codes((16, 32), 1), random_scales((16,), 1)
    assert g.int8_gemm(random_codes((0, 32), 1), b, random_scales((0,), 1), sb).shape == (0, 16)
    assert g.int8_linear(normal((0, 32), BF16, 1), b, sb).shape == (0, 16)
    none = g.int8_grouped_gemm(random_codes((0, 32), 1), b[None], random_scales((0,), 1), sb[None],
                               torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert none.shape == (0, 16)


def test_captured_and_on_another_stream(g):
    x, y = normal((24, 512), BF16, 1), normal((24, 512), BF16, 2)
    w, ws = g.quantize_int8(normal((264, 512), BF16, 3))
    want = [g.int8_linear(v, w, ws) for v in (x, y)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(g.int8_linear(x, w, ws), want[0])
    side.synchronize()
    held, graphs, outs = x.clone(), [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(g.int8_linear(held, w, ws))
        graphs.append(graph)
    for v, expect in zip((x, y, x), (want[0], want[1], want[0])):
        held.copy_(v)
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
            assert torch.equal(out, expect)


def test_refusals(g):
    a, b = random_codes((4, 32), 1), random_codes((16, 32), 2)
    sa, sb = random_scales((4,), 1), random_scales((16,), 2)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    for call in (lambda: g.quantize_int8(torch.zeros(32, device="cuda")),
                 lambda: g.quantize_int8(torch.zeros(4, 32)),
                 lambda: g.dequantize_int8(a, sb),
                 lambda: g.dequantize_int8(a.float(), sa),
                 lambda: g.int8_gemm(a, random_codes((16, 48), 1), sa, sb),
                 lambda: g.int8_gemm(a, random_codes((12, 32), 1), sa, random_scales((12,), 1)),
                 lambda: g.int8_gemm(a[:, :24], b[:, :24], sa, sb),
                 lambda: g.int8_gemm(a, b, sa.half(), sb),
                 lambda: g.int8_gemm(a, b, sb, sb),
                 lambda: g.int8_gemm(a, b, sa, sb, out_dtype=torch.int32),
                 lambda: g.int8_gemm(a, b, sa, sb, out=torch.empty((4, 24), device="cuda")),
                 lambda: g.int8_gemm(a, b, sa, sb, out=torch.empty((16, 4), device="cuda").t()),
                 lambda: g.int8_gemm(a.cpu(), b, sa, sb),
                 lambda: g.int8_gemm(random_codes((1, 131072), 1), random_codes((8, 131072), 1), sa[:1], sb[:8]),
                 lambda: g.int8_linear(torch.zeros((4, 32), device="cuda"), b.float(), sb),
                 lambda: g.int8_grouped_gemm(a, b[None], sa, sb[None], off),
                 lambda: g.int8_grouped_gemm(a, b[None], sa, sb[None], off[:2].long()),
                 lambda: g.int8_grouped_gemm(a, b, sa, sb, off[:2])):
        with pytest.raises(ValueError):
            call()
    from gpu_kernels_b200 import _lib
    with pytest.raises(_lib.Nvfp4Error, match="aligned"):
        g.int8_gemm(a, b, sa, sb, out=torch.empty(4 * 16 + 1, dtype=BF16, device="cuda")[1:].view(4, 16))
