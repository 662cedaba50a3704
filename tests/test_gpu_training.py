"""The operators around a training step's products on the device, against plain 64-bit forms
(training_reference.py): the output head's cross entropy, the router, gradient clipping.

Sizes and values are those at which they can go wrong: one token and none, one class, sizes that fit no
tile or vector, strides and addresses without alignment, rows that a mask leaves empty, infinities and
NaN where nothing may read them, ties, gradients of very different sizes.
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from training_reference import ROUNDING, U32, cross_entropy, cross_entropy_grads, route, route_grad  # noqa: E402

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IGNORE = -100


@pytest.fixture(scope="module")
def ft():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a visible device")
    import flash_train.torch as m

    return m


def within(value, exact, bound, what):
    value = value.detach().cpu().double()
    off = (value - exact).abs() - bound
    assert torch.isfinite(value).all() and (off <= 0).all(), (what, float(off.max()), float(exact.abs().max()))


# ------------------------------------------------------------------ cross entropy


def head(tokens, hidden, classes, dtype, ignored=0.0, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(classes, hidden, generator=g) * (spread / math.sqrt(hidden))).to(dtype)
    y = torch.randint(0, classes, (tokens,), generator=g)
    x = (torch.randn(tokens, hidden, generator=g) + 2.0 * torch.rand(tokens, 1, generator=g) * w[y].float()).to(dtype)
    y = torch.where(torch.rand(tokens, generator=g) < ignored, IGNORE, y)
    grad = (torch.rand(tokens, generator=g) + 0.5) / max(1, tokens)
    return x, w, y, grad


def check_head(ft, x, w, y, grad, device=None):
    dx, dw, dy, dg = device or (t.cuda() for t in (x, w, y, grad))
    loss, lse = ft.linear_cross_entropy_forward(dx, dw, dy, ignore_index=IGNORE)
    exact_loss, exact_lse, bound = cross_entropy(x, w, y, IGNORE)
    within(loss, exact_loss, bound, "loss")
    within(lse, exact_lse, bound, "lse")
    saved = exact_lse.float()
    gx, gw = ft.linear_cross_entropy_backward(dg, dx, dw, dy, saved.cuda(), ignore_index=IGNORE)
    ex, ew, bx, bw = cross_entropy_grads(grad, x, w, y, saved, IGNORE)
    assert gx.dtype == x.dtype and gw.dtype == w.dtype and gx.shape == x.shape and gw.shape == w.shape
    within(gx, ex, bx, "grad_hidden")
    within(gw, ew, bw, "grad_weight")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 64, 300), (2, 8, 5), (3, 7, 257), (17, 33, 1000), (64, 128, 512),
                                   (65, 72, 1031), (130, 200, 129), (257, 96, 513), (300, 520, 4099), (40, 64, 8193)])
def test_cross_entropy(ft, shape, dtype):
    check_head(ft, *head(*shape, dtype, ignored=0.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ignored", [0.1, 0.9])
def test_cross_entropy_leaves_ignored_tokens_out(ft, ignored, dtype):
    x, w, y, grad = head(150, 104, 777, dtype, ignored, seed=3)
    y[0], y[-1] = IGNORE, 5
    clean = x.clone()
    # Whatever an ignored token holds, nothing of it reaches a result.
    for i, row in enumerate(torch.nonzero(y == IGNORE)[:, 0].tolist()):
        x[row] = (math.nan, math.inf, -math.inf)[i % 3]
        grad[row] = (math.inf, math.nan, 1.0)[i % 3]
    quiet = torch.where(y == IGNORE, 0.0, grad)
    check_head(ft, clean, w, y, quiet, device=[t.cuda() for t in (x, w, y, grad)])
    gx, _ = ft.linear_cross_entropy_backward(grad.cuda(), x.cuda(), w.cuda(), y.cuda(), torch.zeros(150).cuda())
    assert (gx[(y == IGNORE).cuda()] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_cross_entropy_without_any_token(ft, dtype):
    for tokens in (0, 5):
        x, w, y, grad = head(tokens, 40, 90, dtype)
        y[:] = IGNORE
        loss, lse = ft.linear_cross_entropy_forward(x.cuda(), w.cuda(), y.cuda())
        assert loss.shape == (tokens,) and (loss == 0).all() and (lse == 0).all()
        gx, gw = ft.linear_cross_entropy_backward(grad.cuda(), x.cuda(), w.cuda(), y.cuda(), lse)
        assert gx.shape == x.shape and (gx == 0).all() and gw.shape == w.shape and (gw == 0).all()


def strided(t, pad, offset):
    """The matrix on the device with `pad` columns between its rows, `offset` elements into its buffer."""
    rows, cols = t.shape
    buffer = torch.full((offset + rows * (cols + pad),), float("nan"), dtype=t.dtype, device="cuda")
    out = buffer[offset:].view(rows, cols + pad)[:, :cols]
    out.copy_(t)
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1), (5, 3)])
def test_cross_entropy_takes_any_row_stride_and_address(ft, pad, offset, dtype):
    x, w, y, grad = head(70, 64, 530, dtype, ignored=0.2, seed=5)
    check_head(ft, x, w, y, grad, device=(strided(x, pad, offset), strided(w, pad, offset), y.int().cuda(), grad.cuda()))


def test_cross_entropy_takes_transposed_and_broadcast_inputs(ft):
    x, w, y, grad = head(33, 24, 100, torch.float32, seed=8)
    grad = torch.full((33,), 0.25)
    check_head(ft, x, w, y, grad, device=(x.cuda().t().contiguous().t(), w.cuda().t().contiguous().t(),
                                          torch.stack([y, y], 1).cuda()[:, 0], torch.tensor(0.25).cuda().expand(33)))
    row = x[:1].expand(33, 24)
    check_head(ft, row.contiguous(), w, y, grad, device=(row.cuda(), w.cuda(), y.cuda(), grad.cuda()))


@pytest.mark.parametrize("dtype", TYPES)
def test_cross_entropy_of_extreme_logits(ft, dtype):
    x, w, y, grad = head(64, 32, 300, dtype, seed=11, spread=60.0)  # logits of hundreds: probabilities 0 and 1
    check_head(ft, x, w, y, grad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 100])
def test_cross_entropy_small_losses_are_not_lost_in_lse(ft, tokens, dtype):
    """Logits that are whole numbers, the target's far above: the loss is the logarithm of a sum near 1,
    with an error of a few roundings of 1, not of the logits."""
    x = torch.zeros(tokens, 16, dtype=dtype)
    x[:, 0] = torch.arange(tokens) % 5 + 1.0
    w = torch.zeros(600, 16, dtype=dtype)
    w[7, 0], w[300, 0], w[599, 0] = 24.0, 20.0, 18.0
    y = torch.full((tokens,), 7)
    loss, lse = ft.linear_cross_entropy_forward(x.cuda(), w.cuda(), y.cuda())
    exact = torch.logsumexp(x.double() @ w.double().t(), 1) - 24.0 * x[:, 0].double()
    within(loss, exact, 16 * U32 * (1.0 + exact), "loss")
    within(lse, exact + 24.0 * x[:, 0].double(), 16 * U32 * (1.0 + exact) + U32 * 2 * 24.0 * x[:, 0].double(), "lse")


def test_cross_entropy_keeps_small_probabilities_in_fp16(ft):
    x, w, y, grad = head(48, 64, 6000, torch.float16, seed=12, spread=0.5)
    check_head(ft, x, w, y, grad * 2.0**-12 * 6000)  # every dl far below fp16's smallest normal number
    check_head(ft, x, w, y, grad * 2.0**10)


def test_cross_entropy_target_outside_the_classes_is_nan(ft):
    x, w, y, grad = head(20, 32, 50, torch.float32, seed=13)
    y[3], y[7] = 50, -1
    loss, lse = ft.linear_cross_entropy_forward(x.cuda(), w.cuda(), y.cuda())
    bad = torch.zeros(20, dtype=torch.bool)
    bad[3] = bad[7] = True
    assert torch.equal(torch.isnan(loss).cpu(), bad) and torch.isfinite(lse).all()
    gx, gw = ft.linear_cross_entropy_backward(grad.cuda(), x.cuda(), w.cuda(), y.cuda(), lse)
    assert torch.equal(torch.isnan(gx).all(1).cpu(), bad) and torch.isfinite(gx[~bad.cuda()]).all()
    assert torch.isnan(gw).all()


def test_cross_entropy_classes_of_minus_infinity(ft):
    """Logits of minus infinity (overflowing products) take no part in a row's sum."""
    x, w, y, _ = head(40, 16, 700, torch.float32, seed=14)
    x[:, 0], w[:, 0] = 1.0, 0.0
    w[64:600, 0] = -math.inf
    y = y % 64
    loss, lse = ft.linear_cross_entropy_forward(x.cuda(), w.cuda(), y.cuda())
    kept = torch.cat([w[:64], w[600:]])
    exact, exact_lse, bound = cross_entropy(x, kept, y)
    within(loss, exact, bound, "loss")
    within(lse, exact_lse, bound, "lse")


@pytest.mark.parametrize("dtype", TYPES)
def test_cross_entropy_repeats_bit_for_bit(ft, dtype):
    x, w, y, grad = (t.cuda() for t in head(333, 264, 5001, dtype, ignored=0.2, seed=15))
    first = ft.linear_cross_entropy_forward(x, w, y)
    grads = ft.linear_cross_entropy_backward(grad, x, w, y, first[1])
    for _ in range(2):
        torch.full((64 << 20,), float("nan"), device="cuda")  # what the next workspaces hold
        again = ft.linear_cross_entropy_forward(x, w, y)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        assert all(torch.equal(a, b) for a, b in zip(grads, ft.linear_cross_entropy_backward(grad, x, w, y, first[1])))


def test_cross_entropy_gradient_against_differences(ft):
    x, w, y, _ = (t.cuda() for t in head(24, 40, 130, torch.float32, ignored=0.2, seed=16))
    weights = torch.linspace(-1.0, 1.0, 24).cuda()
    x.requires_grad_(), w.requires_grad_()
    (ft.linear_cross_entropy(x, w, y, reduction="none") * weights).sum().backward()
    g = torch.Generator().manual_seed(17)
    for leaf in (x, w):
        for _ in range(4):
            d = torch.randn(leaf.shape, generator=g).cuda()
            d /= d.norm()
            h = 2.0**-5
            sides = []
            for s in (h, -h):
                args = [(t + s * d if t is leaf else t).detach() for t in (x, w)]
                loss, _ = ft.linear_cross_entropy_forward(*args, y)
                sides.append(float((loss.double() * weights.double()).sum()))
            slope, exact = (sides[0] - sides[1]) / (2 * h), float((leaf.grad.double() * d.double()).sum())
            # 24 losses near 5, each off by a few 2^-23 of that, over 2 h, and h^2 / 6 of a third
            # derivative (at most about the sixth power of the largest |w| or |x| along d).
            assert abs(slope - exact) < 24 * 5 * 4 * U32 / (2 * h) + h * h, (slope, exact)


def test_cross_entropy_reductions(ft):
    x, w, y, _ = head(50, 32, 80, torch.float32, ignored=0.3, seed=18)
    want = torch.nn.functional.cross_entropy
    for reduction in ("none", "sum", "mean"):
        a, b = x.cuda().requires_grad_(), w.cuda().requires_grad_()
        loss = ft.linear_cross_entropy(a, b, y.cuda(), reduction=reduction)
        p, q = x.double().requires_grad_(), w.double().requires_grad_()
        plain = want(p @ q.t(), y, reduction=reduction)
        torch.testing.assert_close(loss.cpu().double(), plain, rtol=1e-5, atol=1e-5)
        loss.sum().backward(), plain.sum().backward()
        torch.testing.assert_close(a.grad.cpu().double(), p.grad, rtol=1e-4, atol=1e-5)
        torch.testing.assert_close(b.grad.cpu().double(), q.grad, rtol=1e-4, atol=1e-5)
    with pytest.raises(RuntimeError, match="reduction"):
        ft.linear_cross_entropy(a, b, y.cuda(), reduction="median")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(16, 2048, 300), (1, 4096, 50), (64, 1500, 700), (33, 1100, 129), (65, 1024, 1000),
                                   (300, 136, 40001), (500, 40, 30000), (1000, 700, 256)])
def test_cross_entropy_on_every_tile(ft, shape, dtype):
    """Few tokens with a long sum (cut across workgroups), and products large enough for the large tiles."""
    check_head(ft, *head(*shape, dtype, ignored=0.1 if shape[0] > 1 else 0.0, seed=20))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 8, 3), (7, 1032, 260), (40, 64, 530), (64, 2048, 300), (64, 512, 5003)])
def test_cross_entropy_of_few_tokens_as_they_lie(ft, shape, dtype):
    """At most 64 tokens are not packed: rows apart, ignored tokens of any content among them, a target
    outside the classes."""
    x, w, y, grad = head(*shape, dtype, ignored=0.3 if shape[0] > 1 else 0.0, seed=31)
    noisy = x.clone()
    for i, row in enumerate(torch.nonzero(y == IGNORE)[:, 0].tolist()):
        noisy[row] = (math.nan, math.inf, -math.inf)[i % 3]
    for wide in (True, False):
        target = (y if wide else y.int()).cuda()
        check_head(ft, x, w, y, grad, device=(strided(noisy, 8, 0), w.cuda(), target, grad.cuda()))
    y[-1] = shape[2]
    loss, lse = ft.linear_cross_entropy_forward(noisy.cuda(), w.cuda(), y.cuda())
    bad = torch.arange(shape[0]) == shape[0] - 1
    assert torch.equal(torch.isnan(loss).cpu(), bad) and (loss.cpu()[y == IGNORE] == 0).all()
    # An ignored index that is a class.
    y[:] = 2
    loss, lse = ft.linear_cross_entropy_forward(noisy.cuda(), w.cuda(), y.cuda(), ignore_index=2)
    assert (loss == 0).all() and (lse == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(65, 520, 1003), (200, 264, 513), (256, 256, 256), (500, 1024, 5003), (600, 72, 300),
                                   (2000, 512, 1500)])
def test_cross_entropy_gradients_in_one_launch(ft, shape, dtype):
    """Sizes where both products of dl share a launch, with slices of the classes and without."""
    check_head(ft, *head(*shape, dtype, ignored=0.1, seed=37))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hidden", [64, 59])
def test_cross_entropy_in_several_pieces(ft, hidden, dtype):
    """dl of 8192 tokens in pieces of 32768 (16-bit) or 16384 classes; 59: the weight's rows are packed too."""
    x, w, y, grad = head(8192, hidden, 40003, dtype, ignored=0.1, seed=23)
    dev = [t.cuda() for t in (x, w, y, grad)]
    loss, lse = ft.linear_cross_entropy_forward(*dev[:3])
    exact, exact_lse, bound = cross_entropy(*dev[:3])
    assert ((loss.double() - exact).abs() <= bound).all() and ((lse.double() - exact_lse).abs() <= bound).all()
    saved = exact_lse.float()
    gx, gw = ft.linear_cross_entropy_backward(dev[3], *dev[:3], saved)
    ex, ew, bx, bw = cross_entropy_grads(dev[3], *dev[:3], saved)
    assert ((gx.double() - ex).abs() <= bx).all() and ((gw.double() - ew).abs() <= bw).all()


def test_cross_entropy_past_32_bit_offsets(ft):
    """A weight of more than 2^32 bytes; classes at both ends of it."""
    tokens, hidden, classes = 6, 8192, 270001
    g = torch.Generator(device="cuda").manual_seed(19)
    w = torch.randn(classes, hidden, generator=g, device="cuda", dtype=torch.bfloat16).mul_(hidden**-0.5)
    x = torch.randn(tokens, hidden, generator=g, device="cuda", dtype=torch.bfloat16)
    y = torch.tensor([0, classes - 1, 262143, 262144, 131072, IGNORE]).cuda()
    loss, lse = ft.linear_cross_entropy_forward(x, w, y)
    logits = torch.cat([x.float() @ p.float().t() for p in w.split(1 << 16)], 1).double()
    want = torch.logsumexp(logits, 1)
    torch.testing.assert_close(lse[:5].double(), want[:5], rtol=0, atol=1e-4)
    torch.testing.assert_close(loss[:5].double(), (want - logits.gather(1, y.clamp(min=0)[:, None])[:, 0])[:5], rtol=0, atol=1e-4)
    grad = torch.ones(tokens, device="cuda")
    gx, gw = ft.linear_cross_entropy_backward(grad, x, w, y, lse)
    assert (gx[5] == 0).all()
    p = torch.exp(logits - want[:, None])
    for v in (0, 131072, 262143, 262144, classes - 1):
        dl = p[:5, v] - (y[:5] == v).double()
        exact = dl @ x[:5].double()
        torch.testing.assert_close(gw[v].double(), exact, rtol=2.0**-6, atol=float(2.0**-7 * dl.abs().max()))


# ------------------------------------------------------------------ router


def router_logits(rows, n, dtype, seed=0, ties=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, n, generator=g) + 0.5 * torch.randn(n, generator=g)
    if ties:
        x = (x * 2).round() / 2
    return x.to(dtype)


def check_route(ft, logits, top_k, normalize, mask=None, device=None):
    dev = device if device is not None else logits.cuda()
    dmask = None if mask is None else mask.cuda()
    experts, gates, slots, counts, routed, loss = ft.moe_route_forward(dev, top_k, normalize, dmask)
    want = route(logits, top_k, normalize, mask)
    assert torch.equal(experts.cpu(), want[0]) and torch.equal(slots.cpu(), want[2])
    assert torch.equal(counts.cpu(), want[3]) and int(routed) == want[4]
    within(gates, want[1], 32 * U32 * (want[1] + 2.0**-100), "gates")
    # f is a ratio of whole numbers, P a mean of values of either size: a few roundings each.
    bound = (16 + 4 * math.sqrt(logits.shape[0] + logits.shape[1])) * U32 * (want[5] + 2.0**-100)
    within(loss, torch.tensor(want[5], dtype=torch.float64), bound, "loss")
    g = torch.Generator().manual_seed(99)
    grad_gates, grad_loss = torch.randn(logits.shape[0], top_k, generator=g), torch.tensor(0.37)
    grad = ft.moe_route_backward(grad_gates.cuda(), grad_loss.cuda(), dev, experts, counts, routed, normalize, dmask)
    exact = route_grad(grad_gates, grad_loss, logits, want[0], want[3], want[4], normalize, want[6])
    u, tiny = ROUNDING[logits.dtype]
    size = grad_gates.abs().sum(1, keepdim=True).double() + 0.37 * logits.shape[1] / max(1, want[4])
    within(grad, exact, u * exact.abs() + tiny + 64 * U32 * size, "grad_logits")
    assert (grad.cpu()[~want[6]] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,top_k", [(1, 1, 1), (1, 8, 2), (5, 3, 3), (64, 8, 2), (67, 13, 4), (129, 16, 1),
                                          (100, 31, 5), (257, 64, 8), (70, 100, 6), (40, 160, 6), (33, 256, 8),
                                          (12, 300, 3), (9, 512, 32), (7, 1000, 9), (5, 1024, 32)])
def test_route(ft, rows, n, top_k, dtype):
    for normalize in (False, True):
        check_route(ft, router_logits(rows, n, dtype, seed=rows + n), top_k, normalize)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,top_k,passes", [(8, 2, 512), (8, 8, 512), (20, 5, 128), (64, 2, 64), (128, 32, 32), (256, 8, 32),
                                            (260, 4, 16), (1024, 32, 8)])
def test_route_in_one_launch_and_in_two(ft, n, top_k, passes, dtype):
    """Around the most rows that one workgroup takes, twice `passes`."""
    for rows in (passes, passes + 1, 2 * passes - 1, 2 * passes, 2 * passes + 1):
        logits = router_logits(rows, n, dtype, seed=rows)
        mask = torch.rand(rows, generator=torch.Generator().manual_seed(rows)) < 0.8
        logits[rows // 2] = -math.inf
        check_route(ft, logits, top_k, True, mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [8, 24, 64, 250])
def test_route_ties_go_to_the_lowest_index(ft, n, dtype):
    check_route(ft, router_logits(90, n, dtype, seed=n, ties=True), min(n, 7), True)
    check_route(ft, torch.zeros(20, n, dtype=dtype), min(n, 7), False)


@pytest.mark.parametrize("dtype", TYPES)
def test_route_rows_and_experts_left_out(ft, dtype):
    logits = router_logits(120, 40, dtype, seed=4)
    mask = torch.rand(120, generator=torch.Generator().manual_seed(5)) < 0.6
    logits[:, 3] = -math.inf                          # an expert nobody may take
    logits[10] = -math.inf                            # a row without an expert
    logits[11, 1:] = -math.inf                        # a row with one
    logits[12] = torch.finfo(dtype).min               # the type's lowest value everywhere
    logits[13, 5:] = torch.finfo(dtype).min
    mask[10:14] = True
    mask[14] = False
    check_route(ft, logits, 4, True, mask)
    check_route(ft, logits, 4, False)
    noisy = logits.clone()
    noisy[~mask] = math.nan                           # what a masked row holds does not matter
    noisy[14] = math.inf
    got = ft.moe_route_forward(noisy.cuda(), 4, True, mask.cuda())
    same = ft.moe_route_forward(logits.cuda(), 4, True, mask.cuda())
    assert all(torch.equal(a, b) for a, b in zip(got, same))
    grad = ft.moe_route_backward(torch.ones(120, 4).cuda(), torch.ones(()).cuda(), noisy.cuda(), got[0], got[3], got[4], True,
                                 mask.cuda())
    assert torch.isfinite(grad).all() and (grad[~mask.cuda()] == 0).all()


def test_route_nothing_to_route(ft):
    for rows in (0, 9):
        logits = router_logits(rows, 12, torch.float32)
        mask = torch.zeros(rows, dtype=torch.bool)
        check_route(ft, logits, 3, True, mask)


def test_route_nan_shows_in_the_loss(ft):
    logits = router_logits(50, 16, torch.float32, seed=6)
    logits[20, 4] = math.nan
    experts, gates, slots, counts, routed, loss = ft.moe_route_forward(logits.cuda(), 2)
    assert torch.isnan(loss) and torch.isnan(gates[20]).all() and torch.isfinite(gates[:20]).all()
    assert ((experts >= 0) & (experts < 16)).all() and int(counts.sum()) == 100 and int(routed) == 50


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(8, 0), (3, 0), (0, 1)])
def test_route_takes_any_row_stride_and_address(ft, pad, offset, dtype):
    logits = router_logits(77, 64, dtype, seed=7)
    check_route(ft, logits, 6, True, device=strided(logits, pad, offset))
    check_route(ft, logits, 6, False, device=logits.cuda().t().contiguous().t())


@pytest.mark.parametrize("rows,n,top_k", [(20011, 64, 8), (70001, 16, 2)])
def test_route_of_many_rows(ft, rows, n, top_k):
    """More rows than one pass of the workgroups: the packing is a stable sort by expert."""
    logits = router_logits(rows, n, torch.bfloat16, seed=9)
    experts, gates, slots, counts, routed, loss = ft.moe_route_forward(logits.cuda(), top_k)
    order = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :top_k].int()
    assert torch.equal(experts.cpu(), order)
    assert torch.equal(counts.cpu().long(), torch.bincount(order.flatten(), minlength=n)) and int(routed) == rows
    packed = torch.full((rows * top_k,), -1, dtype=torch.int64)
    packed[slots.cpu().flatten().long()] = torch.arange(rows * top_k)
    assert torch.equal(packed, torch.sort(order.flatten(), stable=True).indices)
    p = torch.softmax(logits.double(), 1)
    exact = n * float((counts.cpu().double() / (rows * top_k) * p.mean(0)).sum())
    assert abs(float(loss) - exact) < 64 * U32 * exact
    assert all(torch.equal(a, b) for a, b in zip((experts, gates, slots, counts, routed, loss),
                                                 ft.moe_route_forward(logits.cuda(), top_k)))


@pytest.mark.parametrize("normalize", [False, True])
def test_route_gradient_against_differences(ft, normalize):
    logits = router_logits(30, 12, torch.float32, seed=21).cuda().requires_grad_()
    g = torch.Generator().manual_seed(22)
    weights = torch.randn(30, 3, generator=g).cuda()

    def value(r):
        return float((r.gates.double() * weights.double()).sum() + 3.0 * r.balance_loss.double())

    r = ft.moe_route(logits, 3, normalize)
    ((r.gates * weights).sum() + 3.0 * r.balance_loss).backward()
    for _ in range(4):
        d = torch.randn(30, 12, generator=g).cuda()
        d /= d.norm()
        h = 2.0**-8  # too small a step to change a choice, checked below
        up, down = (ft.moe_route(logits.detach() + s * d, 3, normalize) for s in (h, -h))
        assert torch.equal(up.experts, r.experts) and torch.equal(down.experts, r.experts)
        slope = (value(up) - value(down)) / (2 * h)
        exact = float((logits.grad.double() * d.double()).sum())
        # 90 gates off by a few 2^-24 each, over 2 h, and h^2 of a third derivative of a few units.
        assert abs(slope - exact) < 90 * 4 * U32 / (2 * h) + 4 * h * h, (slope, exact)


# ------------------------------------------------------------------ clipping


def check_clip(ft, grads, max_norm, out, eps=1e-6):
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    coef = min(1.0, max_norm / (exact + eps))
    dev = [g.cuda() for g in grads]
    target = [torch.full_like(g, float("nan")) for g in dev] if out else dev
    norm = ft.clip_grad_norm(dev, max_norm, eps=eps, out=target if out else None)
    assert norm.dim() == 0 and abs(float(norm) - exact) <= 2 * U32 * exact
    for i, (g, t) in enumerate(zip(grads, target)):
        u, tiny = ROUNDING[g.dtype]
        want = g.double() * coef
        within(t, want, (u + 8 * U32) * want.abs() + tiny + 2.0**-149, ("clipped", i))
    if out:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, grads))


def gradients(shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * 10.0 ** (i % 5 - 3)).to(TYPES[i % 3]) for i, s in enumerate(shapes)]


@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e6])
@pytest.mark.parametrize("shapes", [[(1,)], [(7,), (0, 5), (3, 3), (129,)], [(127, 97)] * 5, [(16384,), (16385,), (16383,)],
                                    [(i % 37,) for i in range(400)], [(1 << 20,), (5,), (1 << 19, 3)]])
def test_clip(ft, shapes, max_norm, out):
    check_clip(ft, gradients(shapes), max_norm, out)


def test_clip_takes_dense_tensors_of_any_order_and_address(ft):
    base = [g.cuda() for g in gradients([(130, 70), (40, 9, 11), (1001,)], seed=3)]
    grads = [base[0].t(), base[1].permute(2, 0, 1), base[2][1:]]
    exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    want = [g.double() * (0.25 / (exact + 1e-6)) for g in grads]
    norm = ft.clip_grad_norm(grads, 0.25)
    assert abs(float(norm) - exact) <= 2 * U32 * exact
    for g, w in zip(grads, want):
        torch.testing.assert_close(g.double(), w, rtol=2.0**-7, atol=2.0**-24)
    with pytest.raises(RuntimeError, match="dense"):
        ft.clip_grad_norm([torch.zeros(8, 8, device="cuda")[:, ::2]], 1.0)


def test_clip_of_squares_beyond_32_bits(ft):
    for value in (1e30, 1e-30):
        g = [torch.full((1000,), value), torch.full((50,), value).to(torch.bfloat16)]
        check_clip(ft, g, 1.0, True, eps=0.0)


def test_clip_of_infinite_and_nan_gradients(ft):
    a, b = torch.ones(10).cuda(), torch.full((3,), math.inf).cuda()
    assert float(ft.clip_grad_norm([a, b], 1.0)) == math.inf
    assert (a == 0).all() and torch.isnan(b).all()
    c = torch.tensor([1.0, math.nan]).cuda()
    assert math.isnan(float(ft.clip_grad_norm([c], 1.0))) and torch.isnan(c).all()


def test_clip_repeats_bit_for_bit_and_past_32_bit_counts(ft):
    g = torch.full(((1 << 32) + 5,), 2.0**-16, dtype=torch.bfloat16, device="cuda")
    g[-1] = 3.0
    exact = math.sqrt((2**32 + 4) * 2.0**-32 + 9.0)
    norms = [ft.clip_grad_norm([g], 1e9) for _ in range(2)]
    assert torch.equal(*norms) and abs(float(norms[0]) - exact) <= 2 * U32 * exact
    ft.clip_grad_norm([g], exact / 2, eps=0.0)
    assert float(g[-1]) == 1.5 and float(g[0]) == 2.0**-17 and float(g[1 << 32]) == 2.0**-17


# ------------------------------------------------------------------ streams, graphs, refusals


def step(ft, s):
    loss, lse = ft.linear_cross_entropy_forward(s["x"], s["w"], s["y"])
    gx, gw = ft.linear_cross_entropy_backward(s["g"], s["x"], s["w"], s["y"], lse)
    routed = ft.moe_route_forward(s["l"], 2, True)
    gl = ft.moe_route_backward(s["gg"], s["gl"], s["l"], routed[0], routed[3], routed[4], True)
    norm = ft.clip_grad_norm([gx, gw, gl], 0.01, out=s["out"])
    return [loss, lse, *routed, norm, *s["out"]]


def step_state(seed):
    x, w, y, g = (t.cuda() for t in head(90, 72, 700, torch.bfloat16, 0.2, seed))
    l = router_logits(90, 24, torch.bfloat16, seed).cuda()
    return {"x": x, "w": w, "y": y, "g": g, "l": l, "gg": torch.ones(90, 2).cuda() / 90, "gl": torch.ones(()).cuda(),
            "out": [torch.empty_like(t) for t in (x, w, l)]}


def test_training_operators_run_on_the_current_stream(ft):
    s = step_state(31)
    want = [t.clone() for t in step(ft, s)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        late = dict(s, x=s["x"] * 1.0, l=s["l"] * 1.0)  # made on the side stream after the wait
        got = [t * 1 for t in step(ft, late)]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_training_operators_in_a_graph(ft):
    s = step_state(32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ft, s)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = step(ft, s)
    for seed in (33, 34, 35):
        fresh = step_state(seed)
        for key in ("x", "w", "y", "g", "l"):
            s[key].copy_(fresh[key])
        graph.replay()
        got = [t.clone() for t in captured]
        torch.cuda.synchronize()
        want = step(ft, fresh)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_training_operators_in_the_example_step(ft):
    """The example's step (router, grouped products, head, clipping) learns its batch, and its gradients
    are those of the same model written with torch's operators in fp32."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "moe_training_step.py")
    spec = importlib.util.spec_from_file_location("moe_training_step", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.train(12, 512, 128, 1003)
    assert all(math.isfinite(v) for v in losses) and losses[-1] < 0.7 * losses[0], losses

    model = example.Model(64, 307, 6, 2, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    batch = torch.randint(0, 307, (200,), generator=g, device="cuda")
    mask = torch.rand(200, generator=g, device="cuda") < 0.8
    target = torch.where(mask, (batch + 1) % 307, IGNORE)
    loss = model.loss(batch, target, mask)
    loss.backward()
    # The same choices: the router's logits are computed in bf16 in both.
    r = ft.moe_route((model.embedding[batch] @ model.router.t()).detach(), 2, True, mask)
    plain = [p.detach().float().requires_grad_() for p in model.parameters()]
    emb, router, up, down, out = plain
    x = emb[batch]
    p = torch.softmax(x @ router.t(), 1)
    y = x
    for k in range(2):
        e = r.experts[:, k].long().clamp(min=0)
        gate = p.gather(1, e[:, None]) / sum(p.gather(1, r.experts[:, q].long().clamp(min=0)[:, None]) for q in range(2))
        inner = torch.nn.functional.silu((x[:, None, :] * up[e].transpose(1, 2)).sum(2))
        y = y + torch.where(mask[:, None], gate * (inner[:, None, :] * down[e].transpose(1, 2)).sum(2), 0.0)
    counts = r.counts.float()
    balance = 6 * (counts / counts.sum() * p[mask].mean(0)).sum()
    want = torch.nn.functional.cross_entropy(y @ out.t(), target) + 0.01 * balance
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) < 0.02 * float(want.detach())
    for a, b in zip(model.parameters(), plain):
        # bf16 activations and gradients at every step of the model: a few roundings of 2^-9 each.
        assert float((a.grad.float() - b.grad).norm()) < 0.03 * float(b.grad.norm())


def test_training_operators_refuse(ft):
    x, w, y, g = (t.cuda() for t in head(6, 16, 20, torch.float32))
    lse = torch.zeros(6).cuda()
    fwd, bwd = ft.linear_cross_entropy_forward, ft.linear_cross_entropy_backward
    for args in ((x.cpu(), w, y), (x, w.cpu(), y), (x, w, y.cpu()), (x, w[:, :8], y), (x, w.half(), y), (x[0], w, y),
                 (x.double(), w.double(), y), (x, w, y[:3]), (x, w, y.float()), (x, w[:0], y), (x[:, :0], w[:, :0], y)):
        with pytest.raises(RuntimeError):
            fwd(*args)
    for args in ((g[:3], x, w, y, lse), (g.half(), x, w, y, lse), (g, x, w, y, lse[:2]), (g, x, w, y, lse.cpu())):
        with pytest.raises(RuntimeError):
            bwd(*args)
    logits = router_logits(6, 8, torch.float32).cuda()
    for args in ((logits.cpu(), 2), (logits, 0), (logits, 9), (logits[0], 1), (logits.double(), 2), (logits.int(), 2),
                 (torch.zeros(3, 1025).cuda(), 2), (torch.zeros(3, 100).cuda(), 33), (logits, 2, False, torch.ones(5).bool().cuda()),
                 (logits, 2, False, torch.ones(6).cuda()), (logits, 2, False, torch.ones(6).bool())):
        with pytest.raises(RuntimeError):
            ft.moe_route_forward(*args)
    r = ft.moe_route_forward(logits, 2)
    good = [torch.zeros(6, 2).cuda(), torch.zeros(()).cuda(), logits, r[0], r[3], r[4]]
    for i, bad in ((0, torch.zeros(6, 3).cuda()), (1, torch.zeros(2).cuda()), (3, r[0].long()), (3, r[0][:4]),
                   (4, r[3][:7]), (5, r[4].cpu())):
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError):
            ft.moe_route_backward(*args)
    for args, kw in ((([],  1.0), {}), (([x.cpu()], 1.0), {}), (([x], -1.0), {}), (([x], math.nan), {}), (([x.double()], 1.0), {}),
                     (([x], 1.0), {"out": []}), (([x], 1.0), {"out": [x.half()]}), (([x], 1.0), {"out": [x[:3]]}),
                     (([x], 1.0), {"eps": -1.0})):
        with pytest.raises(RuntimeError):
            ft.clip_grad_norm(*args, **kw)
