"""The order of a router's choices, rows to experts and back, and their gradients, against their definitions in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STEP = 2.0 ** -24                                               # half a step of FP32, relative


@pytest.fixture(scope="module")
def g():
    import gpu_kernels_b200
    return gpu_kernels_b200


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, dtype=F32, seed=0):
    return torch.randn(shape, generator=generator(seed), device="cuda").to(dtype)


def choices(tokens, topk, experts, seed=0, dropped=0.0):
    ids = torch.randint(0, experts, (tokens, topk), generator=generator(seed), device="cuda")
    return torch.where(torch.rand((tokens, topk), generator=generator(seed + 1), device="cuda") < dropped, -1, ids)


def check_order(g, ids, experts):
    offsets, position, source = g.sort_routes(ids, experts)
    flat = ids.cpu().reshape(-1).tolist()
    key = [i if 0 <= i < experts else experts for i in flat]
    want = sorted(range(len(key)), key=lambda i: key[i])        # stable
    assert source.tolist() == want
    inverse = [0] * len(want)
    for row, route in enumerate(want):
        inverse[route] = row
    assert position.reshape(-1).tolist() == inverse and position.shape == ids.shape
    counts = torch.bincount(torch.tensor(key, dtype=torch.int64), minlength=experts + 1)[:experts]
    assert offsets.tolist() == [0] + counts.cumsum(0).tolist()


@pytest.mark.parametrize("tokens,topk,experts", ((1, 1, 1), (1, 6, 256), (5, 3, 2), (32, 1, 7), (31, 2, 1024), (333, 6, 255),
                                                 (32, 8, 64), (255, 8, 64), (256, 4, 64),
                                                 (1025, 1, 3), (256, 8, 64), (1000, 4, 1024), (2731, 6, 33), (20000, 3, 257), (80000, 2, 100)))
def test_order(g, tokens, topk, experts):
    check_order(g, choices(tokens, topk, experts, tokens, 0.1), experts)
    check_order(g, choices(tokens, topk, experts, tokens + 5).int(), experts)


@pytest.mark.parametrize("tokens", (9, 3000))
def test_order_of_extreme_choices(g, tokens):
    for ids in (torch.zeros((tokens, 2)), torch.full((tokens, 2), 15.0), torch.full((tokens, 2), -1.0), torch.full((tokens, 2), 16.0)):
        check_order(g, ids.cuda().long(), 16)
    far = choices(tokens, 2, 16, 3)
    far[::3, 0] = 2 ** 40 + 5                                   # truncated to 32 bits it would be an expert
    far[1::3, 1] = -2 ** 35
    check_order(g, far, 16)
    check_order(g, choices(tokens, 4, 16, 4)[:, ::2], 16)


def test_order_of_nothing(g):
    offsets, position, source = g.sort_routes(torch.zeros((0, 4), dtype=torch.int64, device="cuda"), 5)
    assert offsets.tolist() == [0] * 6 and position.shape == (0, 4) and source.shape == (0,)
    routes = g.Routes(offsets, position, source)
    x = torch.zeros((0, 8), device="cuda", requires_grad=True)
    rows = g.gather_tokens(x, routes)
    assert rows.shape == (0, 8) and g.combine_tokens(rows, routes).shape == (0, 8)
    codes, scales = g.gather_tokens_int8(torch.zeros((0, 16), device="cuda"), routes)
    assert codes.shape == (0, 16) and scales.shape == (0,)


def live_routes(routes):
    return routes.position < routes.offsets[-1]


SHAPES = ((1, 1, 1, 1), (9, 4, 8, 1030), (6, 2, 8, 12), (11, 5, 8, 66), (1, 6, 256, 4096), (7, 3, 4, 33), (20, 2, 5, 64), (64, 6, 16, 1000), (33, 9, 40, 257), (5, 17, 20, 2056), (300, 8, 64, 512))


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("tokens,topk,experts,hidden", SHAPES)
def test_gather_and_its_gradient(g, tokens, topk, experts, hidden, dtype):
    routes = g.sort_routes(choices(tokens, topk, experts, hidden, 0.2), experts)
    x = normal((tokens, hidden), dtype, 1).requires_grad_()
    rows = g.gather_tokens(x, routes)
    live = live_routes(routes)
    want = torch.zeros((tokens, topk, hidden), dtype=dtype, device="cuda")
    want[live] = x.detach()[:, None].expand(-1, topk, -1)[live]
    assert torch.equal(rows[routes.position.long()], want)
    assert torch.equal(g.gather_tokens(x.detach(), routes), rows)
    d_rows = normal(rows.shape, dtype, 2)
    d_rows[int(routes.offsets[-1]):] = float("nan")             # behind the live rows: not read
    d_x, = torch.autograd.grad(rows, x, d_rows)
    terms = torch.where(live[..., None], d_rows[routes.position.long()].double(), 0.0)
    # topk additions in FP32, one rounding to the type (none for FP32, whose additions are counted)
    own = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    bound = topk * STEP * terms.abs().sum(1) * (1 + own) + own * terms.sum(1).abs() + (2.0 ** -25 if dtype == F16 else 0.0)
    assert d_x.dtype == dtype and bool(((d_x.double() - terms.sum(1)).abs() <= bound).all())


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("tokens,topk,experts,hidden", SHAPES)
def test_combine_and_its_gradients(g, tokens, topk, experts, hidden, dtype):
    routes = g.sort_routes(choices(tokens, topk, experts, hidden, 0.2), experts)
    live, place = live_routes(routes), routes.position.long()
    rows, w = normal((tokens * topk, hidden), dtype, 1), normal((tokens, topk), F32, 2)
    rows[int(routes.offsets[-1]):] = float("inf")
    w[~live] = float("nan")
    rows.requires_grad_(), w.requires_grad_()
    own = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    small = 2.0 ** -25 if dtype == F16 else 0.0
    y = g.combine_tokens(rows, routes, w)
    terms = torch.where(live[..., None], rows.detach()[place].double() * w.detach().double()[..., None], 0.0)
    bound = topk * STEP * terms.abs().sum(1) * (1 + own) + own * terms.sum(1).abs() + small
    assert y.dtype == dtype and bool(((y.double() - terms.sum(1)).abs() <= bound).all())

    d_y = normal((tokens, hidden), dtype, 3)
    d_rows, d_w = torch.autograd.grad(y, (rows, w), d_y)
    want = torch.where(live[..., None], w.detach().double()[..., None] * d_y.double()[:, None], 0.0)
    bound = want.abs() * ((1 + STEP) * (1 + own) - 1) + small
    assert d_rows.dtype == dtype and bool(((d_rows[place].double() - want).abs() <= bound).all())
    # a sum of `hidden` products: at most as many additions as one thread makes, five between lanes and eight between warps
    products = torch.where(live[..., None], rows.detach()[place].double(), 0.0) * d_y.double()[:, None]
    depth = 8 * -(-hidden // (256 * 8)) + hidden // 256 + 14
    assert d_w.dtype == F32 and bool(((d_w.double() - products.sum(-1)).abs() <= depth * STEP * products.abs().sum(-1)).all())

    # one at a time, and without weights
    assert torch.equal(torch.autograd.grad(g.combine_tokens(rows, routes, w.detach()), rows, d_y)[0], d_rows)
    assert torch.equal(torch.autograd.grad(g.combine_tokens(rows.detach(), routes, w), w, d_y)[0], d_w)
    plain = g.combine_tokens(rows, routes)
    assert torch.equal(plain, g.combine_tokens(rows.detach(), routes, torch.ones_like(w)))
    assert torch.equal(torch.autograd.grad(plain, rows, d_y)[0], g.gather_tokens(d_y, routes))


def test_gradients_against_differences(g):
    # The whole way out and back: y is linear in x and in the weights, so a difference is the derivative but for rounding.
    tokens, topk, experts, hidden = 20, 3, 6, 96
    routes = g.sort_routes(choices(tokens, topk, experts, 1, 0.1), experts)
    x, w = normal((tokens, hidden), F32, 1).requires_grad_(), normal((tokens, topk), F32, 2).requires_grad_()
    d_y = normal((tokens, hidden), F32, 3)
    loss = lambda a, b: (g.combine_tokens(g.gather_tokens(a, routes), routes, b).double() * d_y.double()).sum()  # noqa: E731
    d_x, d_w = torch.autograd.grad(loss(x, w), (x, w))
    with torch.no_grad():
        size = (x.abs()[:, None] * w.abs()[..., None] * d_y.abs()[:, None]).sum().double()
        for leaf, grad, move in ((x, d_x, lambda v: loss(x + v, w)), (w, d_w, lambda v: loss(x, w + v))):
            v = normal(leaf.shape, F32, 4)
            moved = float(move(v) - loss(x, w))
            # every value on the way is one of FP32 with at most topk roundings, the sum of the moved leaf rounds once more;
            # the gradient's own sums have at most `hidden` roundings
            slack = float(size) * 4 * (topk + 2 + hidden) * STEP * float(1 + v.abs().max())
            assert abs(moved - float((grad.double() * v.double()).sum())) <= slack


def test_strides_broadcast_gradients_and_alignment(g):
    tokens, topk, experts, hidden = 12, 2, 4, 64
    routes = g.sort_routes(choices(tokens, topk, experts, 7), experts)
    x = normal((tokens, hidden), BF16, 1)
    rows = g.gather_tokens(x, routes)
    odd = torch.cat((x.flatten()[:1], x.flatten()))[1:].view(tokens, hidden)         # two bytes off a 16-byte boundary
    for same in (x.t().contiguous().t(), torch.cat((x, x), 1)[:, :hidden], odd):
        assert torch.equal(g.gather_tokens(same, routes), rows)
        assert torch.equal(g.gather_tokens_int8(same, routes)[0], g.gather_tokens_int8(x, routes)[0])
    w = normal((topk, tokens), F32, 2).t()
    y = g.combine_tokens(rows, routes, w)
    assert torch.equal(g.combine_tokens(torch.cat((rows, rows), 1)[:, hidden:], routes, w.contiguous()), y)
    assert torch.equal(g.combine_tokens(rows, routes, w.double()), y)
    leaf = x.clone().requires_grad_()
    g.gather_tokens(leaf, routes).sum().backward()              # the rows' gradient is one value, broadcast
    assert bool((leaf.grad == topk).all())
    leaf = rows.clone().requires_grad_()
    weights = w.to(BF16).clone().requires_grad_()
    g.combine_tokens(leaf, routes, weights).sum().backward()
    assert weights.grad.dtype == BF16 and torch.equal(leaf.grad[routes.position.long()], weights.detach()[..., None].expand(-1, -1, hidden))


@pytest.mark.parametrize("dtype", (BF16, F16, F32))
@pytest.mark.parametrize("tokens,topk,experts,k", ((1, 6, 256, 4096), (9, 3, 4, 16), (40, 2, 8, 528), (70, 8, 16, 2064), (2, 2, 4, 33008),
                                                    (11, 2, 8, 1040), (5, 2, 8, 4112), (6, 3, 8, 8784), (4, 2, 8, 14336), (3, 2, 8, 20496), (75, 3, 8, 64), (41, 4, 8, 128),
                                                    (19, 2, 8, 240)))
def test_gather_quantised(g, tokens, topk, experts, k, dtype):
    routes = g.sort_routes(choices(tokens, topk, experts, k, 0.2), experts)
    x = normal((tokens, k), dtype, 1)
    codes, scales = g.gather_tokens_int8(x, routes)
    token_codes, token_scales = g.quantize_int8(x)
    live = live_routes(routes)
    assert torch.equal(codes[routes.position.long()], torch.where(live[..., None], token_codes[:, None], 0))
    assert torch.equal(scales[routes.position.long()], torch.where(live, token_scales[:, None], 0.0))


def test_rows_beyond_31_bits(g):
    # 9000 tokens of eight routes, 30808 values a row: the last rows lie behind element 2^31
    tokens, topk, experts, hidden = 9000, 8, 16, 30808
    routes = g.sort_routes(choices(tokens, topk, experts, 1), experts)
    x = torch.empty((tokens, hidden), dtype=BF16, device="cuda").normal_(generator=generator(2)).requires_grad_()
    rows = g.gather_tokens(x, routes)
    token = routes.source.long() // topk
    assert torch.equal(rows[-50:], x.detach()[token[-50:]])
    w = torch.full((tokens, topk), 0.125, device="cuda")
    y = g.combine_tokens(rows, routes, w)                        # eight times an eighth of each value: exact
    assert torch.equal(y, x)
    d_x, = torch.autograd.grad(y, x, x.detach())
    assert torch.equal(d_x, x)


def test_positions_outside_the_rows_are_skipped(g):
    # an order of the caller's own making: nothing is read or written out of bounds
    d = torch.device("cuda")
    routes = g.Routes(torch.tensor([0, 4], dtype=torch.int32, device=d), torch.tensor([[0, 99], [-3, 2]], dtype=torch.int32, device=d),
                      torch.zeros(4, dtype=torch.int32, device=d))
    x = normal((2, 16), F32, 1)
    rows = g.gather_tokens(x, routes)
    assert torch.equal(rows[0], x[0]) and torch.equal(rows[2], x[1])
    y = g.combine_tokens(rows, routes, torch.ones((2, 2), device=d))
    assert torch.equal(y, x)
    codes, _ = g.gather_tokens_int8(x, routes)
    assert torch.equal(codes[0], g.quantize_int8(x)[0][0])


def test_captured_with_its_backward_pass(g):
    tokens, topk, experts, hidden = 40, 4, 8, 128
    ids = [choices(tokens, topk, experts, s, 0.1) for s in (1, 2)]
    xs = [normal((tokens, hidden), BF16, s) for s in (3, 4)]
    w, d_y = normal((tokens, topk), F32, 5), normal((tokens, hidden), BF16, 6)

    def step(i, x, weights):
        routes = g.sort_routes(i, experts)
        y = g.combine_tokens(g.gather_tokens(x, routes), routes, weights)
        return y, *torch.autograd.grad(y, (x, weights), d_y)

    want = [[t.detach().clone() for t in step(i, x.clone().requires_grad_(), w.clone().requires_grad_())] for i, x in zip(ids, xs)]
    held_i, held_x, held_w = ids[0].clone(), xs[0].clone().requires_grad_(), w.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held_i, held_x, held_w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(held_i, held_x, held_w)
    for turn in (0, 1, 0):
        with torch.no_grad():
            held_i.copy_(ids[turn])
            held_x.copy_(xs[turn])
        graph.replay()
        for a, b in zip(got, want[turn]):
            assert torch.equal(a, b)


def test_int8_expert_layer_end_to_end(g):
    """Router's choices -> rows in int8 -> the experts' two products -> tokens, as a serving program runs it."""
    tokens, topk, experts, hidden, inter = 77, 3, 12, 256, 128
    x = normal((tokens, hidden), BF16, 1)
    ids, weights = g.route(normal((tokens, experts), F32, 2), topk)
    w1, w2 = normal((experts, 2 * inter, hidden), F32, 3) * 0.05, normal((experts, hidden, inter), F32, 4) * 0.05
    q1, s1 = (t.reshape(experts, 2 * inter, -1).squeeze(-1) for t in g.quantize_int8(w1.reshape(-1, hidden)))
    q2, s2 = (t.reshape(experts, hidden, -1).squeeze(-1) for t in g.quantize_int8(w2.reshape(-1, inter)))

    def layer(x):
        routes = g.sort_routes(ids, experts)
        gate_up = g.int8_grouped_gemm(*(lambda c, s: (c, q1, s, s1))(*g.gather_tokens_int8(x, routes)), routes.offsets)
        act = torch.nn.functional.silu(gate_up[:, :inter]) * gate_up[:, inter:]
        codes, scales = g.quantize_int8(act)
        return g.combine_tokens(g.int8_grouped_gemm(codes, q2, scales, s2, routes.offsets), routes, weights), gate_up, act

    y, gate_up, act = layer(x)
    g.check_int8()
    # each step against its definition, from the step before as it came out
    routes = g.sort_routes(ids, experts)
    expert = ids.reshape(-1)[routes.source.long()]
    token = routes.source.long() // topk
    own = 2.0 ** -8
    codes, scales = g.quantize_int8(x)
    first = torch.einsum("rk,rnk->rn", codes[token].double(), q1[expert].double()) * scales[token].double()[:, None] * s1[expert].double()
    assert bool(((gate_up.double() - first).abs() <= first.abs() * (own * 1.001)).all())
    codes, scales = g.quantize_int8(act)
    second = torch.einsum("rk,rnk->rn", codes.double(), q2[expert].double()) * scales.double()[:, None] * s2[expert].double()
    terms = second.bfloat16().double()[routes.position.long()] * weights.double()[..., None]
    # the second product's own rounding moves each term by 2^-8, the sum is rounded once
    bound = terms.abs().sum(1) * (own * 1.01) + terms.sum(1).abs() * (own * 1.01) + terms.abs().sum(1) * own
    assert bool(((y.double() - terms.sum(1)).abs() <= bound).all())
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        layer(x)
    side.synchronize()
    with torch.cuda.graph(graph):
        replayed = layer(x)[0]
    graph.replay()
    assert torch.equal(replayed, y)


def test_refusals(g):
    ids = choices(6, 2, 4, 1)
    routes = g.sort_routes(ids, 4)
    x, rows = normal((6, 32), BF16, 1), normal((12, 32), BF16, 1)
    for call in (lambda: g.sort_routes(ids.cpu(), 4),
                 lambda: g.sort_routes(ids.float(), 4),
                 lambda: g.sort_routes(ids.reshape(-1), 4),
                 lambda: g.sort_routes(ids, 0),
                 lambda: g.sort_routes(ids, 1025),
                 lambda: g.gather_tokens(x[:5], routes),
                 lambda: g.gather_tokens(x.double(), routes),
                 lambda: g.gather_tokens(x.cpu(), routes),
                 lambda: g.gather_tokens(x, g.Routes(routes.offsets.long(), routes.position, routes.source)),
                 lambda: g.gather_tokens(x, g.Routes(routes.offsets, routes.position.cpu(), routes.source)),
                 lambda: g.gather_tokens_int8(x[:, :24].contiguous(), routes),
                 lambda: g.combine_tokens(x, routes),
                 lambda: g.combine_tokens(rows, routes, torch.ones((6, 3), device="cuda")),
                 lambda: g.combine_tokens(rows, routes, torch.ones((6, 2), device="cuda", dtype=torch.int32)),
                 lambda: g.combine_tokens(rows, routes, torch.ones((6, 2)))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):                           # no gradient of the gradient
        leaf = x.clone().requires_grad_()
        d, = torch.autograd.grad(g.gather_tokens(leaf, routes).float().square().sum(), leaf, create_graph=True)
        d.sum().backward()
