"""Token routing on the GPU against its definitions in 64 bits (route_ref.py).

Tolerances count roundings.  u = 2^-24 is half a step of a 32-bit number, relative to the value; half(T) that of the
output's type.  They are stated where they are used."""
import pytest
import torch

import route_ref as ref
from route_ref import INF, U32, half_step, smallest

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def mrs():
    import wgpu_morton_code_radix_sort_test_amd as m

    return m


def gates(mrs):
    return {"softmax": mrs.GATE_SOFTMAX, "sigmoid": mrs.GATE_SIGMOID}


def close(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got - want).abs()
    bad = ~(err <= tol)
    if bad.any():
        i = int(torch.argmax((err / tol.clamp(min=1e-300) if torch.is_tensor(tol) else err).nan_to_num(1e300)))
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, e.g. {got.reshape(-1)[i]} for {want.reshape(-1)[i]}")


# ---- select ---------------------------------------------------------------------------------
def spread(scores, bias):
    """Largest distance of scores that take part in a row: the size of the exponents' arguments, beyond 104 of which
    an exponential is below the smallest number."""
    s = torch.where(ref.keys(scores, bias) > -INF, scores.double(), torch.zeros((), dtype=torch.float64))
    return min(104.0, float(2 * s.abs().max()))


def check_select(mrs, ctx, scores, bias, topk, gate, normalize, scale, strided=False):
    """weights: an exponential's argument is off by u times itself (times two for the logarithm of a sigmoid),
    the exponential and logarithm by an ulp or two each, the sum by at most 22 additions, then a division and a product:
    2 * (2 * spread + 30) u covers numerator and denominator.
    gradient: q and p are off by as much relative to 1 (they are at most 1), the slots' sum adds topk roundings, and a product
    with g another two; p is subtracted once more in a softmax over all; the result is rounded to its type."""
    tokens, experts = scores.shape
    dev = ctx.device
    plan = mrs.RoutePlan(ctx, tokens, experts, topk, gate=gates(mrs)[gate], normalize=normalize, scale=scale)
    d_scores = scores.to(dev)
    if strided:
        wide = torch.full((tokens, experts + 3), float("nan"), dtype=scores.dtype, device=dev)
        wide[:, 1 : experts + 1] = d_scores
        d_scores = wide[:, 1 : experts + 1]
    d_bias = bias.to(dev) if bias is not None else None
    ids, w = plan.select(d_scores, d_bias)
    want_ids = ref.select_ids(scores, bias, topk)
    assert torch.equal(ids.cpu(), want_ids)
    want_w = ref.weights(scores, bias, want_ids, gate, normalize, scale)
    rel = 2 * (2 * spread(scores, bias) + 30) * U32
    close(w, want_w, rel * want_w.abs() + 2.0**-149, "weights")
    assert bool((w.cpu()[want_ids < 0] == 0).all())
    g = torch.Generator().manual_seed(9)
    dw = torch.randn(tokens, topk, generator=g)
    ds = plan.select_backward(d_scores, ids, dw.to(dev), d_bias)
    assert ds.dtype == scores.dtype
    want = ref.scores_grad(scores, bias, want_ids, dw, gate, normalize, scale)
    size = (dw.abs().amax(1, keepdim=True) * abs(scale)).double()
    tol = 2 * (rel + (topk + 6) * U32) * size + half_step(scores.dtype) * want.abs() + smallest(scores.dtype)
    close(ds, want, tol, "scores_grad")
    plan.close()


@pytest.mark.parametrize("gate", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,experts,topk", [(1, 1, 1), (1, 8, 2), (3, 7, 7), (5, 16, 16), (17, 60, 6), (33, 64, 8),
                                                 (2, 33, 32), (40, 128, 8), (9, 129, 10), (70, 256, 8), (3, 257, 16), (4, 512, 32),
                                                 (2, 1000, 22), (3, 1024, 32), (6, 300, 4), (5, 512, 8),
                                                 (4, 513, 3), (3, 1024, 8), (7, 600, 1), (9, 33, 9)])
def test_select(ctx, mrs, tokens, experts, topk, dtype, gate, normalize):
    g = torch.Generator().manual_seed(tokens * 1000 + experts)
    scores = (torch.randn(tokens, experts, generator=g) * 2).to(dtype)  # 16-bit scores hold many equal ones
    check_select(mrs, ctx, scores, None, topk, gate, normalize, 1.0, strided=experts % 2 == 1)
    bias = torch.randn(experts, generator=g) * 0.5
    check_select(mrs, ctx, scores, bias, topk, gate, normalize, 2.5)


@pytest.mark.parametrize("gate", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_select_masks(ctx, mrs, dtype, gate, normalize):
    """Rows whose mask leaves nothing, one, fewer than topk; the type's lowest value; NaN; both zeros; ties."""
    experts, topk = 40, 4
    low = torch.finfo(dtype).min
    nan = float("nan")
    g = torch.Generator().manual_seed(5)
    rows = torch.randn(12, experts, generator=g)
    rows[0] = -INF
    rows[1] = -INF
    rows[1, 17] = 0.5
    rows[2] = -INF
    rows[2, [3, 39, 20]] = torch.tensor([1.0, 1.0, -2.0])
    rows[3] = low
    rows[4] = low
    rows[4, 11] = 1.0
    rows[5, 5:30] = nan
    rows[6] = nan
    rows[7] = 0.0
    rows[7, ::2] = -0.0  # equal keys: the lowest columns
    rows[8] = 3.0
    rows[9, :35] = -INF
    rows[9, 35] = nan
    rows[10] = -100.0  # sigmoids near nothing
    rows[10, 1] = -90.0
    check_select(mrs, ctx, rows.to(dtype), None, topk, gate, normalize, 1.0)
    bias = torch.zeros(experts)
    bias[4] = -INF  # an expert switched off for everyone
    bias[7] = nan
    bias[9] = 1e30
    check_select(mrs, ctx, rows.to(dtype), bias, topk, gate, normalize, 1.0)


def test_select_of_infinite_scores(ctx, mrs):
    """+infinity comes first, lowest column first; a sigmoid of it is 1."""
    s = torch.zeros(1, 8, device=ctx.device)
    s[0, [6, 2]] = INF
    s[0, 4] = 1.0
    for gate in (mrs.GATE_SOFTMAX, mrs.GATE_SIGMOID):
        plan = mrs.RoutePlan(ctx, 1, 8, 4, gate=gate, normalize=False)
        ids, w = plan.select(s)
        assert ids.tolist() == [[2, 6, 4, 0]]
        if gate == mrs.GATE_SIGMOID:
            assert w[0, :2].tolist() == [1.0, 1.0] and w[0, 3] == 0.5
        else:
            assert bool(torch.isnan(w[0, 0]))


@pytest.mark.parametrize("gate", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
def test_select_backward_with_repeated_and_odd_ids(ctx, mrs, gate, normalize):
    """Ids a caller made up: repeated, negative, too large, masked ones."""
    g = torch.Generator().manual_seed(2)
    scores = torch.randn(4, 20, generator=g)
    scores[3, 6] = -INF
    ids = torch.tensor([[3, 3, 3, 3, 3], [1, 2, 1, 2, 1], [-1, 20, 7, 1 << 30, 7], [6, 5, -5, 6, 5]], dtype=torch.int32)
    dw = torch.randn(4, 5, generator=g)
    plan = mrs.RoutePlan(ctx, 4, 20, 5, gate=gates(mrs)[gate], normalize=normalize, scale=0.5)
    ds = plan.select_backward(scores.to(ctx.device), ids.to(ctx.device), dw.to(ctx.device))
    want = ref.scores_grad(scores, None, ids, dw, gate, normalize, 0.5)
    tol = 2 * (2 * (2 * spread(scores, None) + 30) * U32 + 11 * U32) * 0.5 * dw.abs().sum(1, keepdim=True).double() + 2.0**-149
    close(ds, want, tol, "scores_grad")


@pytest.mark.parametrize("gate", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
def test_select_backward_matches_differences_of_the_forward(ctx, mrs, gate, normalize):
    """Central differences of the GPU's own weights along a random direction v, |v| <= 1, over scores 1/4 apart so that the choice
    stays.  The third derivative of sum dw w is below 60 sum |dw|: the difference is off by at most 10 h^2 sum |dw|, and by
    the weights' own error, 2 (2 * spread + 30) u sum |dw| / h; h = 2^-7."""
    h = 2.0**-7
    g = torch.Generator().manual_seed(4)
    scores = torch.stack([torch.randperm(16, generator=g).float() * 0.25 - 2 for _ in range(6)])
    v = torch.rand(6, 16, generator=g) * 2 - 1
    dw = torch.rand(6, 3, generator=g) * 2 - 1
    plan = mrs.RoutePlan(ctx, 6, 16, 3, gate=gates(mrs)[gate], normalize=normalize)
    dev = ctx.device
    ids, _ = plan.select(scores.to(dev))
    ds = plan.select_backward(scores.to(dev), ids, dw.to(dev)).cpu().double()
    up_scores, down_scores = scores + h * v, scores - h * v  # as the GPU sees them, with their rounding
    step = (up_scores.double() - down_scores.double()) / 2
    up, down = (plan.select(x.to(dev)) for x in (up_scores, down_scores))
    assert torch.equal(up[0], ids) and torch.equal(down[0], ids)
    diff = ((up[1].cpu().double() - down[1].cpu().double()) * dw.double()).sum(1) / 2
    size = dw.abs().sum(1).double()
    tol = (10 * h * h * h + 2 * (2 * spread(scores, None) + 30) * U32) * size
    close((ds * step).sum(1), diff, 2 * tol, "directional derivative")


# ---- order ----------------------------------------------------------------------------------
def check_order(mrs, ctx, ids, experts, align=1, capacity=0, extra=0, plan=None):
    tokens, topk = ids.shape
    own = plan is None
    if own:
        plan = mrs.RoutePlan(ctx, tokens, experts, topk, align=align, capacity=capacity)
    rows = plan.max_rows + extra
    junk = lambda *shape: torch.full(shape, 0x5A5A5A5A, dtype=torch.int32, device=ctx.device)  # noqa: E731
    out = mrs.RouteMap(junk(max(tokens, 1), topk), junk(rows), junk(experts), junk(experts + 1))
    plan.order(ids.to(ctx.device), out)
    want = ref.order(ids, experts, align, capacity, rows)
    assert torch.equal(out.counts.cpu(), want[2])
    assert torch.equal(out.offsets.cpu(), want[3])
    assert torch.equal(out.row_of_slot.cpu()[:tokens], want[0])
    assert torch.equal(out.slot_of_row.cpu(), want[1])
    if own:
        plan.close()


@pytest.mark.parametrize("align,capacity", [(1, 0), (16, 0), (128, 7), (1, 1), (5, 3)])
@pytest.mark.parametrize("tokens,experts,topk", [(0, 4, 2), (1, 1, 1), (1, 256, 8), (3, 1024, 32), (63, 3, 1), (64, 64, 8),
                                                 (1000, 60, 4), (1023, 8, 8), (1024, 8, 8), (1025, 8, 8), (4099, 17, 3),
                                                 (5000, 1000, 2), (2731, 1024, 3)])
def test_order(ctx, mrs, tokens, experts, topk, align, capacity):
    g = torch.Generator().manual_seed(tokens + experts)
    ids = torch.randint(-1, experts + 1, (tokens, topk), generator=g, dtype=torch.int32)
    check_order(mrs, ctx, ids, experts, align, capacity, extra=3)


@pytest.mark.parametrize("slots", [64, 65, 1024, 1025, 2048, 2049, 4096, 4097, 8193, 16384, 24576, 24577, 65536, 262144, 262145])
def test_order_around_tile_sizes(ctx, mrs, slots):
    g = torch.Generator().manual_seed(slots)
    ids = (torch.randn(slots, 1, generator=g) * 3 + 8).to(torch.int32)  # crowded in the middle, some outside
    for align, capacity in ((1, 0), (32, slots // 16 + 1)):
        check_order(mrs, ctx, ids, 16, align, capacity, extra=1)


@pytest.mark.parametrize("tokens", [400, 9000, 30000])
def test_order_of_odd_ids(ctx, mrs, tokens):
    """One expert has everything; nobody has anything; runs; numbers far outside; one expert after the other."""
    topk, experts = 2, 37
    n = tokens * topk
    i = torch.arange(n, dtype=torch.int64)
    far = torch.tensor([-(1 << 31), (1 << 31) - 1, -1, experts, 1 << 16, 5])
    for flat in (torch.full((n,), 36), torch.full((n,), -1), i // 100 % experts, far[i % 6], i % experts, (n - 1 - i) * experts // n):
        for capacity in (0, 50):
            check_order(mrs, ctx, flat.to(torch.int32).reshape(tokens, topk), experts, 8, capacity)


@pytest.mark.parametrize("slots,experts", [((1 << 20) + 1, 64), (2500000, 257), (1400000, 1024), (65537, 1024), (140000, 1024), (300001, 300), (524289, 8)])
def test_order_of_many_slots(ctx, mrs, slots, experts):
    """More slots than workgroups have tiles: each walks several, and an expert's capacity ends inside one."""
    g = torch.Generator().manual_seed(7)
    ids = (torch.randn(slots, 1, generator=g) * experts / 4 + experts / 2).to(torch.int32)
    check_order(mrs, ctx, ids, experts, 64, slots // experts)


def test_order_is_the_stable_sort(ctx, mrs):
    """Against the library's own sort of (key, index) pairs: the rows are its sorted source indices."""
    n, experts = 50000, 200
    g = torch.Generator(device=ctx.device).manual_seed(1)
    ids = torch.randint(0, experts, (n, 1), generator=g, device=ctx.device, dtype=torch.int32)
    route = mrs.RoutePlan(ctx, n, experts, 1).order(ids)
    sort = mrs.SortPlan(ctx, n, key_words=1, payload_bytes=4, end_bit=8)
    ka, kb, va, vb = ids.reshape(-1).clone(), *(torch.empty(n, dtype=torch.int32, device=ctx.device) for _ in range(3))
    in_b = sort.sort_pairs_indexed(ka, va, kb, vb)
    sort.check()
    assert torch.equal(route.slot_of_row, vb if in_b else va)


def test_order_with_fewer_tokens_than_the_plan(ctx, mrs):
    plan = mrs.RoutePlan(ctx, 9000, 16, 4, align=8)
    g = torch.Generator().manual_seed(3)
    for tokens in (9000, 1, 0, 3000):
        check_order(mrs, ctx, torch.randint(0, 16, (tokens, 4), generator=g, dtype=torch.int32), 16, 8, 0, plan=plan)


# ---- rows -----------------------------------------------------------------------------------
def make_route(mrs, ctx, tokens, experts, topk, align=1, capacity=0, drop=0.2, seed=1):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (tokens, topk), generator=g, dtype=torch.int32)
    ids[torch.rand(tokens, topk, generator=g) < drop] = -1
    if tokens > 2:
        ids[tokens // 2] = -1  # a token without rows
    plan = mrs.RoutePlan(ctx, tokens, experts, topk, align=align, capacity=capacity)
    rows = plan.max_rows + 5  # some behind the last segment in any case
    route = mrs.RouteMap(*(t.to(ctx.device) for t in ref.order(ids, experts, align, capacity, rows)))
    return plan, route, rows, g


def view(t, pad, shift, device):
    """t on the device, inside wider rows from element `shift` on, among NaN (bytes: 255)."""
    rows, hidden = t.shape
    fill = 255 if t.dtype == torch.uint8 else float("nan")
    wide = torch.full((rows, hidden + pad), fill, dtype=t.dtype, device=device)
    wide[:, shift : shift + hidden] = t.to(device)
    return wide[:, shift : shift + hidden], wide


def untouched(wide, hidden, shift):
    rest = torch.cat([wide[:, :shift], wide[:, shift + hidden :]], 1)
    return bool((rest == 255).all()) if wide.dtype == torch.uint8 else bool(torch.isnan(rest).all())


SHAPES = [(1, 1, 1, 1, 1), (1, 4, 2, 8, 4), (2, 3, 3, 7, 1), (5, 8, 2, 64, 16), (7, 5, 5, 15, 3), (9, 4, 1, 16, 1), (33, 8, 4, 100, 8),
          (64, 16, 8, 129, 1), (3, 64, 32, 250, 2), (20, 6, 6, 513, 4), (6, 9, 9, 1024, 128), (11, 8, 8, 1109, 1), (4, 7, 16, 2050, 7),
          (3, 256, 8, 4096, 16), (2, 3, 17, 8200, 1), (300, 8, 3, 33, 64), (2, 4, 8, 6368, 16), (5, 300, 9, 227, 8)]


@pytest.mark.parametrize("pad,shift", [(0, 0), (5, 1), (16, 8)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16, torch.uint8])
@pytest.mark.parametrize("tokens,experts,topk,hidden,align", SHAPES)
def test_dispatch(ctx, mrs, tokens, experts, topk, hidden, align, dtype, pad, shift):
    plan, route, rows, g = make_route(mrs, ctx, tokens, experts, topk, align)
    make = (lambda *s: torch.randint(0, 255, s, generator=g, dtype=torch.uint8)) if dtype == torch.uint8 else (
        lambda *s: torch.randn(*s, generator=g).to(dtype))
    x, before = make(tokens, hidden), make(rows, hidden)
    if dtype != torch.uint8:
        x[0, 0] = float("nan")  # moved like anything else
    d_x, _ = view(x, pad, shift, ctx.device)
    d_rows, wide = view(before, pad, shift, ctx.device)
    plan.dispatch(d_x, route, rows_out=d_rows)
    parts = [t.cpu() for t in (route.row_of_slot, route.counts, route.offsets)]
    want = ref.dispatch(x, *parts, before)
    as_bits = {4: torch.int32, 2: torch.int16, 1: torch.uint8}[x.element_size()]
    assert torch.equal(d_rows.cpu().contiguous().view(as_bits), want.view(as_bits))
    assert untouched(wide, hidden, shift)
    plan.close()


@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("pad,shift", [(0, 0), (5, 1)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,experts,topk,hidden,align", SHAPES)
def test_combine_and_dispatch_backward(ctx, mrs, tokens, experts, topk, hidden, align, dtype, pad, shift, weighted):
    """Each of topk fused multiply-adds (additions) rounds once, off by at most u times the magnitudes' sum so far; then one
    rounding to the type: half(T) of the 32-bit sum."""
    plan, route, rows, g = make_route(mrs, ctx, tokens, experts, topk, align, seed=2)
    x = torch.randn(rows, hidden, generator=g).to(dtype)
    empty = torch.ones(rows, dtype=torch.bool)
    empty[route.row_of_slot.cpu()[route.row_of_slot.cpu() >= 0].long()] = False
    x[empty] = float("nan")  # rows nobody has are not read into anything
    w = torch.randn(tokens, topk, generator=g) if weighted else None
    if weighted:
        w[route.row_of_slot.cpu() < 0] = float("nan")  # nor the weights of slots without a row
    d_x, _ = view(x, pad, shift, ctx.device)
    d_out, wide = view(torch.zeros(tokens, hidden, dtype=dtype), pad, shift, ctx.device)
    if weighted:
        plan.combine(d_x, route, w.to(ctx.device), out=d_out)
    else:
        plan.dispatch_backward(d_x, route, x_grad_out=d_out)
    want, size = ref.combine(x, route.row_of_slot.cpu(), w)
    sums = topk * U32 * 1.01 * size
    close(d_out, want, sums + half_step(dtype) * (want.abs() + sums) + smallest(dtype), "rows")
    assert bool((d_out[tokens // 2] == 0).all()) or tokens <= 2  # a token without rows
    assert untouched(wide, hidden, shift)
    plan.close()


@pytest.mark.parametrize("pad,shift", [(0, 0), (5, 1)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens,experts,topk,hidden,align", SHAPES)
def test_combine_backward(ctx, mrs, tokens, experts, topk, hidden, align, dtype, pad, shift):
    """rows: a product rounded to 32 bits, then to the type.  weights: a lane adds at most hidden / 64 + 8 products (rows of up to 64
    vectors of 16 bytes: 8), the lanes' sums meet in 6 additions more.  Where n of up to 16 waves share a row, that is one of
    n * 64 vectors at least, a lane's part is that much shorter, which makes room for the n - 1 additions of their sums."""
    plan, route, rows, g = make_route(mrs, ctx, tokens, experts, topk, align, seed=3)
    x, dout = torch.randn(rows, hidden, generator=g).to(dtype), torch.randn(tokens, hidden, generator=g).to(dtype)
    w = torch.randn(tokens, topk, generator=g)
    before = torch.randn(rows, hidden, generator=g).to(dtype)
    d_x, _ = view(x, pad, shift, ctx.device)
    d_dout, _ = view(dout, pad, shift, ctx.device)
    d_rows, wide = view(before, pad, shift, ctx.device)
    _, dw = plan.combine_backward(d_dout, d_x, route, w.to(ctx.device), drows_out=d_rows)
    row_of_slot, counts, offsets = (t.cpu() for t in (route.row_of_slot, route.counts, route.offsets))
    want, want_dw, size = ref.combine_backward(dout, x, row_of_slot, w, counts, offsets, before)
    close(d_rows, want, (half_step(dtype) + 1.01 * U32) * want.abs() + smallest(dtype), "rows_grad")
    end = int(offsets[-1])
    assert torch.equal(d_rows.cpu()[end:], before[end:])  # behind the last segment: as it was
    close(dw, want_dw, (hidden / 64 + 16) * U32 * 1.01 * size + 2.0**-149, "weights_grad")
    assert bool((dw.cpu()[row_of_slot < 0] == 0).all())
    assert untouched(wide, hidden, shift)
    plan.close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("hidden", [9, 21, 300, 1109])
def test_columns_a_kernel_visits_twice_count_once(ctx, mrs, dtype, hidden):
    """Rows that no whole number of 16-byte vectors covers: an infinite element near the end makes its weight's gradient
    infinite, not NaN, and comes through combine as it is."""
    plan, route, rows, g = make_route(mrs, ctx, 4, 4, 2, drop=0.0)
    x, dout = torch.rand(rows, hidden, generator=g).to(dtype) + 0.5, torch.rand(4, hidden, generator=g).to(dtype) + 0.5
    for back in (1, 2, 3, min(8, hidden)):
        y = x.clone()
        y[:, hidden - back] = INF
        row_of_slot = route.row_of_slot.cpu()
        w = torch.ones(4, 2, device=ctx.device)
        _, dw = plan.combine_backward(dout.to(ctx.device), y.to(ctx.device), route, w)
        assert bool((dw.cpu()[row_of_slot >= 0] == INF).all())
        out = plan.combine(y.to(ctx.device), route, w).cpu()
        some = (row_of_slot >= 0).any(1)
        assert bool((out[some][:, hidden - back] == INF).all())
        assert int(torch.isinf(out).sum()) == int(some.sum())


def test_rows_past_4_gib(ctx, mrs):
    """Row offsets beyond 32 bits: rows 2 x 65792 bytes apart, 40000 of them."""
    tokens, experts, topk, hidden, stride = 10000, 16, 4, 72, 65792
    plan, route, rows, g = make_route(mrs, ctx, tokens, experts, topk, 4, drop=0.0)
    assert rows * stride * 2 > 1 << 32
    big = torch.zeros(rows, stride, dtype=BF16, device=ctx.device)
    x = torch.randn(tokens, hidden, generator=g).to(BF16)
    part = big[:, 100 : 100 + hidden]
    plan.dispatch(x.to(ctx.device), route, rows_out=part)
    parts = [t.cpu() for t in (route.row_of_slot, route.counts, route.offsets)]
    assert torch.equal(part.cpu(), ref.dispatch(x, *parts, torch.zeros(rows, hidden, dtype=BF16)))
    w = torch.randn(tokens, topk, generator=g)
    out = plan.combine(part, route, w.to(ctx.device))
    want, size = ref.combine(part.cpu(), parts[0], w)
    sums = topk * U32 * 1.01 * size
    close(out, want, sums + half_step(BF16) * (want.abs() + sums) + smallest(BF16), "combine")
    assert int(torch.count_nonzero(big)) == int(torch.count_nonzero(part))
    grads = big[:, 40000 : 40000 + hidden]  # other columns of the same buffer
    dout = torch.randn(tokens, hidden, generator=g).to(BF16)
    _, dw = plan.combine_backward(dout.to(ctx.device), part, route, w.to(ctx.device), drows_out=grads)
    want, want_dw, size = ref.combine_backward(dout, part.cpu(), parts[0], w, parts[1], parts[2], torch.zeros(rows, hidden, dtype=BF16))
    close(grads, want, (half_step(BF16) + 1.01 * U32) * want.abs() + smallest(BF16), "rows_grad")
    close(dw, want_dw, (hidden / 64 + 16) * U32 * 1.01 * size, "weights_grad")


def test_many_small_rows(ctx, mrs):
    """Several tokens share a wave."""
    plan, route, rows, g = make_route(mrs, ctx, 70001, 8, 2, 1, drop=0.1)
    x = torch.randn(70001, 3, generator=g)
    out = torch.full((rows, 3), -1.0, device=ctx.device)
    plan.dispatch(x.to(ctx.device), route, rows_out=out)
    parts = [t.cpu() for t in (route.row_of_slot, route.counts, route.offsets)]
    assert torch.equal(out.cpu(), ref.dispatch(x, *parts, torch.full((rows, 3), -1.0)))
    w = torch.randn(70001, 2, generator=g)
    want, size = ref.combine(out.cpu(), parts[0], w)
    close(plan.combine(out, route, w.to(ctx.device)), want, 3.1 * U32 * size + U32 * want.abs(), "combine")


def test_indices_outside_the_rows_are_passed_over(ctx, mrs):
    """A map somebody else wrote: rows that do not exist count as no row."""
    plan = mrs.RoutePlan(ctx, 4, 4, 2)
    row_of_slot = torch.tensor([[0, 9], [-7, 1], [1 << 30, -(1 << 31)], [8, 2]], dtype=torch.int32)
    route = mrs.RouteMap(*(t.to(ctx.device) for t in (row_of_slot, torch.zeros(9, dtype=torch.int32), torch.zeros(4, dtype=torch.int32),
                                                      torch.zeros(5, dtype=torch.int32))))
    x = torch.arange(4 * 40, dtype=F32).reshape(4, 40) + 1
    out = torch.zeros(9, 40, device=ctx.device)
    plan.dispatch(x.to(ctx.device), route, rows_out=out)
    want = torch.zeros(9, 40)
    want[0], want[1], want[8], want[2] = x[0], x[1], x[3], x[3]
    assert torch.equal(out.cpu(), want)
    ones = torch.ones(4, 2, device=ctx.device)
    back = plan.combine(out, route, ones).cpu()
    assert torch.equal(back, torch.stack([x[0], x[1], torch.zeros(40), 2 * x[3]]))
    drows, dw = plan.combine_backward(x.to(ctx.device), out, route, ones, drows_out=torch.zeros_like(out))
    assert torch.equal(drows.cpu(), want)
    assert bool((dw.cpu()[[0, 1, 2, 2], [1, 0, 0, 1]] == 0).all()) and float(dw[3, 0]) == float((x[3] * x[3]).sum())


# ---- as they are used -------------------------------------------------------------------------
@pytest.mark.parametrize("gate,normalize", [("softmax", True), ("softmax", False), ("sigmoid", True)])
def test_a_layer_forward_and_backward(ctx, mrs, gate, normalize):
    """select, order, dispatch, a product by each expert's factor, combine, and all of it backwards, against torch's gradients
    in 64 bits.  Products and sums round as in the tests above: the rows carry two roundings (factor, weight), the weights
    the relative error r of `check_select`, out adds topk more; the gradients another factor and sum."""
    tokens, experts, topk, hidden = 50, 10, 3, 37
    g = torch.Generator().manual_seed(6)
    scores, x = torch.randn(tokens, experts, generator=g), torch.randn(tokens, hidden, generator=g)
    factor, dout = torch.rand(experts, generator=g) + 0.5, torch.randn(tokens, hidden, generator=g)
    dev = ctx.device
    plan = mrs.RoutePlan(ctx, tokens, experts, topk, align=8, gate=gates(mrs)[gate], normalize=normalize)
    ids, w = plan.select(scores.to(dev))
    route = plan.order(ids)
    rows = plan.dispatch(x.to(dev), route)
    f = torch.zeros(plan.max_rows, 1, device=dev)
    used = route.slot_of_row >= 0
    f[used, 0] = factor.to(dev)[ids.reshape(-1)[route.slot_of_row[used].long()].long()]
    y = torch.where(f > 0, rows * f, torch.zeros((), device=dev))
    out = plan.combine(y, route, w)
    dy, dw = plan.combine_backward(dout.to(dev), y, route, w)
    drows = torch.where(f > 0, dy * f, torch.zeros((), device=dev))
    dx = plan.dispatch_backward(drows, route)
    ds = plan.select_backward(scores.to(dev), ids, dw)

    s64, x64 = scores.double().requires_grad_(), x.double().requires_grad_()
    p = torch.softmax(s64, 1) if gate == "softmax" else torch.sigmoid(s64)
    want_ids = torch.sort(scores, dim=1, descending=True, stable=True).indices[:, :topk]
    assert torch.equal(ids.cpu().long(), want_ids)
    q = torch.gather(p, 1, want_ids)
    if normalize:
        q = q / q.sum(1, keepdim=True)
    scaled = (q * factor.double()[want_ids]).unsqueeze(2)  # [tokens, topk, 1]
    want = (scaled * x64.unsqueeze(1)).sum(1)
    want.backward(dout.double())
    r = 2 * (2 * spread(scores, None) + 30) * U32
    size = (scaled * x64.detach().abs().unsqueeze(1)).sum(1).detach()
    close(out, want.detach(), (r + (topk + 4) * U32) * size, "out")
    size = (scaled.detach() * dout.double().abs().unsqueeze(1)).sum(1)
    close(dx, x64.grad, (r + (topk + 4) * U32) * size, "x_grad")
    # |dw| and its error, (hidden / 64 + 18) u of the magnitudes, go through the gate's derivative, at most 2 in all
    dw_size = 1.5 * (dout.double().abs() * x.double().abs()).sum(1, keepdim=True)
    close(ds, s64.grad, 2 * (2 * r + (topk + 6 + hidden / 64 + 18) * U32) * dw_size, "scores_grad")


def test_calls_replay_from_a_graph(ctx, mrs):
    """The whole chain captured once and replayed on new contents, with eager work of the same plan in between."""
    tokens, experts, topk, hidden = 3000, 32, 4, 200
    dev = ctx.device
    plan = mrs.RoutePlan(ctx, tokens, experts, topk, align=16)
    scores, x = torch.zeros(tokens, experts, device=dev), torch.zeros(tokens, hidden, dtype=BF16, device=dev)
    dout = torch.zeros(tokens, hidden, dtype=BF16, device=dev)
    rows_buf = torch.zeros(plan.max_rows, hidden, dtype=BF16, device=dev)
    drows_buf = torch.zeros_like(rows_buf)

    def chain(rows_out, drows_out):
        ids, w = plan.select(scores)
        route = plan.order(ids)
        rows = plan.dispatch(x, route, rows_out=rows_out)
        out = plan.combine(rows, route, w)
        drows, dw = plan.combine_backward(dout, rows, route, w, drows_out=drows_out)
        dx = plan.dispatch_backward(drows, route)
        ds = plan.select_backward(scores, ids, dw)
        return [ids, w, route.row_of_slot, route.slot_of_row, route.counts, route.offsets, out, dw, dx, ds]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        chain(rows_buf, drows_buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = chain(rows_buf, drows_buf)
    for seed in range(4):
        g = torch.Generator(device=dev).manual_seed(seed)
        scores.copy_(torch.randn(tokens, experts, generator=g, device=dev))
        x.copy_(torch.randn(tokens, hidden, generator=g, device=dev))
        dout.copy_(torch.randn(tokens, hidden, generator=g, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        eager = chain(torch.zeros_like(rows_buf), torch.zeros_like(drows_buf))
        torch.cuda.synchronize()
        for got, want in zip(captured, eager):
            assert torch.equal(got, want)


def test_two_graphs_of_one_plan_and_two_plans_at_once(ctx, mrs):
    """Graphs that share a plan's memory, replayed one after the other; then plans of their own on streams of their own."""
    dev, n, experts = ctx.device, 120000, 50
    g = torch.Generator().manual_seed(12)
    ids = [torch.randint(-1, experts, (n, 1), generator=g, dtype=torch.int32) for _ in range(4)]
    want = [ref.order(i, experts, 8, 0, n + 7 * experts)[0] for i in ids]
    plan = mrs.RoutePlan(ctx, n, experts, 1, align=8)
    buffers, graphs, maps = [], [], []
    side = torch.cuda.Stream()
    for k in range(2):
        buffers.append(ids[k].to(dev))
        maps.append(plan.order(buffers[k]))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            plan.order(buffers[k], maps[k])
        graphs.append(graph)
    for k, new in ((0, 0), (1, 1), (0, 2), (1, 3), (0, 1), (1, 0)):
        buffers[k].copy_(ids[new].to(dev))
        graphs[k].replay()
        graphs[1 - k].replay()
        torch.cuda.synchronize()
        assert torch.equal(maps[k].row_of_slot.cpu(), want[new])
    plans = [plan, mrs.RoutePlan(ctx, n, experts, 1, align=8)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    on_dev = [i.to(dev) for i in ids]
    torch.cuda.synchronize()
    for _ in range(5):
        for k in range(2):
            plans[k].order(on_dev[k + 2], maps[k], stream=streams[k])
    torch.cuda.synchronize()
    for k in range(2):
        assert torch.equal(maps[k].row_of_slot.cpu(), want[k + 2])
    del graphs


def test_calls_take_the_stream_they_are_given(ctx, mrs):
    """Behind slow work on another stream: a call that ran elsewhere would read the old contents."""
    dev = ctx.device
    plan = mrs.RoutePlan(ctx, 2000, 16, 2)
    g = torch.Generator(device=dev).manual_seed(1)
    ids = torch.zeros(2000, 2, dtype=torch.int32, device=dev)
    new_ids = torch.randint(0, 16, (2000, 2), generator=g, device=dev, dtype=torch.int32)
    big = torch.randn(4096, 4096, device=dev)
    other = torch.cuda.Stream()
    route = plan.new_map()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        for _ in range(20):
            big = big @ big * 1e-3
        ids.copy_(new_ids)
    plan.order(ids, route, stream=other)
    other.synchronize()
    want = plan.order(new_ids)
    for name in ("row_of_slot", "slot_of_row", "counts", "offsets"):
        assert torch.equal(getattr(route, name), getattr(want, name))


def test_new_outputs_belong_to_the_stream_that_writes_them(ctx, mrs):
    """Memory just freed on the current stream, where work that writes it is still queued, must not become the output of a call on
    another stream: the queued work would overwrite it afterwards."""
    dev = ctx.device
    plan = mrs.RoutePlan(ctx, 4096, 8, 1)
    ids = torch.zeros(4096, 1, dtype=torch.int32, device=dev)
    route, w = plan.order(ids), torch.ones(4096, 1, device=dev)
    rows = torch.ones(4096, 512, device=dev)
    other = torch.cuda.Stream()
    big = torch.randn(8192, 8192, device=dev)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    scrap = torch.empty(4096, 512, device=dev)
    place = scrap.data_ptr()
    for _ in range(10):
        big = big @ big * 1e-3
    scrap.fill_(7.0)
    del scrap
    out = plan.combine(rows, route, w, stream=other)
    other.synchronize()
    torch.cuda.synchronize()
    assert out.data_ptr() != place and bool((out == 1).all())


def test_eight_bit_floats_are_moved_unseen(ctx, mrs):
    plan, route, rows, g = make_route(mrs, ctx, 40, 8, 2, 4)
    x = torch.randint(0, 256, (40, 50), generator=g, dtype=torch.uint8)
    out = torch.zeros(rows, 50, dtype=torch.uint8, device=ctx.device).view(torch.float8_e4m3fn)
    plan.dispatch(x.to(ctx.device).view(torch.float8_e4m3fn), route, rows_out=out)
    parts = [t.cpu() for t in (route.row_of_slot, route.counts, route.offsets)]
    assert torch.equal(out.view(torch.uint8).cpu(), ref.dispatch(x, *parts, torch.zeros(rows, 50, dtype=torch.uint8)))


def test_results_are_the_same_every_time(ctx, mrs):
    tokens = 20000
    g = torch.Generator(device=ctx.device).manual_seed(8)
    plan = mrs.RoutePlan(ctx, tokens, 64, 8)
    scores = torch.randn(tokens, 64, generator=g, device=ctx.device).to(BF16)
    x = torch.randn(tokens, 300, generator=g, device=ctx.device)
    first = None
    for _ in range(3):
        ids, w = plan.select(scores)
        route = plan.order(ids)
        rows = plan.dispatch(x, route)
        out = plan.combine(rows, route, w)
        drows, dw = plan.combine_backward(x, rows, route, w)
        got = [ids, w, route.row_of_slot, rows, out, drows, dw, plan.select_backward(scores, ids, dw)]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_refusals(ctx, mrs):
    dev = ctx.device
    with pytest.raises(ValueError):
        mrs.RoutePlan(ctx, -1, 8, 2)
    for kw in (dict(experts=0), dict(topk=33), dict(align=0), dict(gate=7), dict(scale=float("inf"))):
        args = dict(tokens=8, experts=8, topk=2)
        args.update(kw)
        with pytest.raises(mrs.MrsError):
            mrs.RoutePlan(ctx, **args)
    plan = mrs.RoutePlan(ctx, 8, 4, 2, align=4)
    route = plan.order(torch.zeros(8, 2, dtype=torch.int32, device=dev))
    rows = plan.max_rows
    x, r, w = torch.zeros(8, 16, device=dev), torch.zeros(rows, 16, device=dev), torch.zeros(8, 2, device=dev)
    with pytest.raises(mrs.MrsError, match="exceed the handle"):
        plan.select(torch.zeros(9, 4, device=dev))
    with pytest.raises(mrs.MrsError, match="exceeds the 1 experts"):
        mrs.RoutePlan(ctx, 8, 1, 2).select(torch.zeros(8, 1, device=dev))
    with pytest.raises(mrs.MrsError, match="need at least"):
        plan.order(torch.zeros(8, 2, dtype=torch.int32, device=dev),
                   mrs.RouteMap(route.row_of_slot, route.slot_of_row[: rows - 1], route.counts, route.offsets))
    with pytest.raises(mrs.MrsError, match="apart"):  # a broadcast row: all rows in one place
        plan.dispatch(torch.zeros(1, 16, device=dev).expand(8, 16), route)
    with pytest.raises(mrs.MrsError, match="apart"):
        plan.combine(r, route, w, out=torch.zeros(1, 16, device=dev).expand(8, 16))
    both = torch.zeros(rows + 4, 16, device=dev)
    with pytest.raises(mrs.MrsError, match="overlap"):
        plan.dispatch(both[:8], route, rows_out=both[4:])
    with pytest.raises(mrs.MrsError, match="overlap"):
        plan.combine(both[4:], route, w, out=both[:8])
    with pytest.raises(mrs.MrsError, match="overlap"):
        plan.combine_backward(x, r, route, w, drows_out=r)
    with pytest.raises(mrs.MrsError, match="overlap"):
        plan.combine_backward(both[:8], r, route, w, drows_out=both[4:])
    half = torch.zeros(rows, 40, device=dev)
    with pytest.raises(mrs.MrsError, match="overlap"):
        plan.combine_backward(x, half[:, :16], route, w, drows_out=half[:, 15:31])
    plan.combine_backward(x, half[:, :16], route, w, drows_out=half[:, 16:32])  # columns beside each other
    s = torch.zeros(8, 4, device=dev)
    with pytest.raises(mrs.MrsError, match="overlap"):
        plan.select_backward(s, torch.zeros(8, 2, dtype=torch.int32, device=dev), w, scores_grad_out=s)
    ids = torch.zeros(8, 2, dtype=torch.int32, device=dev)
    for bad in (mrs.RouteMap(ids, route.slot_of_row, route.counts, route.offsets),
                mrs.RouteMap(route.row_of_slot, route.slot_of_row, route.slot_of_row, route.offsets),
                mrs.RouteMap(route.row_of_slot, route.slot_of_row, route.offsets, route.offsets)):
        with pytest.raises(mrs.MrsError, match="overlap"):
            plan.order(ids, bad)
    with pytest.raises(mrs.MrsError, match="overlap"):
        plan.combine_backward(x, r, route, w, dweights_out=w)
    with pytest.raises(mrs.MrsError, match="overlap"):
        plan.select(s, ids_out=w.view(torch.int32), weights_out=w)
    with pytest.raises(mrs.MrsError, match="overlap"):
        plan.dispatch_backward(r[:, :2], route, x_grad_out=route.row_of_slot.view(torch.float32))
    with pytest.raises(ValueError, match="is on"):
        plan.dispatch(torch.zeros(8, 16), route)
    # no tokens: nothing to do, nothing refused
    none = torch.zeros(0, 4, device=dev)
    assert plan.select(none)[0].shape == (0, 2)
    empty = plan.order(torch.zeros(0, 2, dtype=torch.int32, device=dev))
    assert empty.offsets.tolist() == [0] * 5 and empty.counts.tolist() == [0] * 4
    assert plan.dispatch(torch.zeros(0, 16, device=dev), empty).shape == (rows, 16)
    assert plan.combine(r, empty, torch.zeros(0, 2, device=dev)).shape == (0, 16)
    plan.close()
    with pytest.raises(mrs.MrsError, match="null handle"):
        plan.dispatch(x, route)
