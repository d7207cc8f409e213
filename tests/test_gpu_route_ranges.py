"""Token routing on the GPU at the ends of its ranges: small calls of a large plan, moves of hundreds of MiB, more work
than one grid takes, offsets past 4 GiB."""
import pytest
import torch

import route_ref as ref
from route_ref import U32, half_step, smallest
from test_gpu_route import BF16, F16, F32, check_order, gates, make_route, mrs, untouched, view  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,experts,topk,align,capacity", [(1000, 8, 2, 64, 64), (2048, 64, 8, 128, 128), (1024, 8, 2, 128, 128),
                                                                (9000, 64, 4, 128, 100), (300, 300, 2, 16, 1)])
def test_order_with_a_capacity_and_fewer_tokens_than_the_plan(ctx, mrs, tokens, experts, topk, align, capacity):
    plan = mrs.RoutePlan(ctx, tokens, experts, topk, align=align, capacity=capacity)
    g = torch.Generator().manual_seed(3)
    for few in (tokens, 1, 3, 32, 50, 64, 100, 0):
        ids = torch.randint(-1, experts, (few, topk), generator=g, dtype=torch.int32)
        check_order(mrs, ctx, ids, experts, align, capacity, plan=plan)
        assert plan.order(ids.to(ctx.device)).slot_of_row.numel() == plan.max_rows
        check_order(mrs, ctx, torch.zeros_like(ids), experts, align, capacity, plan=plan)  # all in one segment


def test_one_map_for_batches_of_different_sizes(ctx, mrs):
    """Forward and backward of a large batch, then of smaller and larger ones, through the same map and buffers.  Rows are copies of
    x, so the gradient of x is the sum of a token's topk rows of the gradient: small whole numbers, exact."""
    dev, experts, topk, hidden = ctx.device, 16, 3, 40
    plan = mrs.RoutePlan(ctx, 500, experts, topk, align=4)
    route = plan.new_map()
    g = torch.Generator().manual_seed(5)
    for tokens in (500, 7, 90, 1, 500):
        ids = torch.randint(-1, experts, (tokens, topk), generator=g, dtype=torch.int32)
        assert plan.order(ids.to(dev), route) is route and route.tokens == tokens
        grad = torch.randint(-8, 9, (plan.max_rows, hidden), generator=g).float()
        got = plan.dispatch_backward(grad.to(dev), route)
        row_of_slot = ref.order(ids, experts, 4, 0, plan.max_rows)[0].long()
        want = (grad[row_of_slot.clamp(min=0)] * (row_of_slot >= 0).unsqueeze(2)).sum(1)
        assert torch.equal(got.cpu(), want)
        assert torch.equal(plan.dispatch_backward(grad.to(dev), route, tokens=tokens).cpu(), want)


def test_a_map_that_a_graph_writes_too(ctx, mrs):
    """Replays say nothing to the host: where their number of tokens is not the last eager call's, it has to be given."""
    dev, experts, hidden = ctx.device, 8, 24
    plan = mrs.RoutePlan(ctx, 300, experts, 2)
    route = plan.new_map()
    g = torch.Generator().manual_seed(6)
    ids = torch.randint(0, experts, (300, 2), generator=g, dtype=torch.int32).to(dev)
    grad = torch.randint(-8, 9, (plan.max_rows, hidden), generator=g).float().to(dev)
    few = ids[:50].contiguous()
    plan.order(few, route)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.order(few, route)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got = plan.dispatch_backward(grad, route)
        assert torch.equal(got, plan.dispatch_backward(grad, plan.order(few)))
    plan.order(ids, route)
    with pytest.raises(ValueError, match="tokens"):
        plan.dispatch_backward(grad, route)
    whole = plan.dispatch_backward(grad, route, tokens=300)
    assert torch.equal(whole, plan.dispatch_backward(grad, plan.order(ids)))
    graph.replay()
    assert torch.equal(plan.dispatch_backward(grad, route, tokens=50), got)


def test_matrices_beyond_the_address_range_are_refused(ctx, mrs):
    """2^30 + 1 rows 2^40 floats apart: an extent of 2^72 bytes, which is 0 in 64 bits.  No slot has a row here, so that
    no kernel would touch one."""
    import ctypes

    from wgpu_morton_code_radix_sort_test_amd import _lib

    dev, lib, hidden, far = ctx.device, _lib.load_library(), 16, 1 << 40
    plan = mrs.RoutePlan(ctx, 4, 4, 2)
    none = torch.full((4, 2), -1, dtype=torch.int32, device=dev)
    zeros = torch.zeros(5, dtype=torch.int32, device=dev)
    x, buf, w = (torch.zeros(4, n, device=dev) for n in (hidden, hidden, 2))
    sums = torch.zeros(4, 2, device=dev)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def calls(rows, ld):
        m = ctypes.byref(_lib.RouteMapStruct(none.data_ptr(), None, zeros.data_ptr(), zeros.data_ptr(), rows))
        f32 = 0
        return [
            lib.mrs_route_dispatch(plan._h, 4, m, f32, hidden, p(x), hidden, p(buf), ld, stream),
            lib.mrs_route_dispatch_backward(plan._h, 4, m, f32, hidden, p(buf), ld, p(x), hidden, stream),
            lib.mrs_route_combine(plan._h, 4, m, f32, hidden, p(buf), ld, p(w), p(x), hidden, stream),
            lib.mrs_route_combine_backward(plan._h, 4, m, f32, hidden, p(x), hidden, p(buf), hidden, p(w), p(buf), ld, p(sums), stream),
            lib.mrs_route_combine_backward(plan._h, 4, m, f32, hidden, p(x), hidden, p(buf), ld, p(w), p(buf), hidden, p(sums), stream),
        ]

    assert calls(4, hidden) == [_lib.MRS_OK] * 3 + [_lib.MRS_ERR_INVALID_ARGUMENT] * 2  # the last two: rows over rows_grad
    assert "overlap" in lib.mrs_last_error_string().decode()
    assert calls((1 << 30) + 1, far) == [_lib.MRS_ERR_INVALID_ARGUMENT] * 5
    assert "2^56 bytes" in lib.mrs_last_error_string().decode()
    assert calls((1 << 14) + 1, far) == [_lib.MRS_ERR_INVALID_ARGUMENT] * 5  # 2^56 + 64 bytes
    torch.cuda.synchronize()
    assert lib.mrs_route_destroy(None) == _lib.MRS_OK


# ---- rows in hundreds of MiB --------------------------------------------------------------------
def within(got, want, tol, what):
    """`close` where the tensors are: got in its type, the others in 64 bits."""
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    if bool(bad.any()):
        i = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError(f"{what}: {int(bad.sum())} off, e.g. {got.reshape(-1)[i]} for {want.reshape(-1)[i]} at {i}")


def row_sums(rows, row_of_slot, w):
    """Per token the sum of its rows and of their magnitudes in 64 bits, on the device."""
    total = torch.zeros(row_of_slot.size(0), rows.size(1), dtype=torch.float64, device=rows.device)
    size = torch.zeros_like(total)
    for j in range(row_of_slot.size(1)):
        token = torch.nonzero(row_of_slot[:, j] >= 0).squeeze(1)
        term = rows[row_of_slot[token, j].long()].double()
        if w is not None:
            term *= w[token, j : j + 1].double()
        total[token] += term
        size[token] += term.abs()
    return total, size


STREAMED = [(4500, 32, 8, 4097, 16, BF16), (3500, 20, 10, 4099, 1, F16), (6000, 16, 3, 4101, 4, F32), (9000, 8, 1, 16411, 64, BF16),
            (17000, 40, 4, 2048, 128, BF16)]


@pytest.mark.parametrize("tokens,experts,topk,hidden,align,dtype", STREAMED)
def test_moves_that_go_past_the_caches(ctx, mrs, tokens, experts, topk, hidden, align, dtype):
    """From 256 MiB of rows on.  Strides wider than the rows, a fifth of the slots dropped; roundings as in the tests of small
    rows."""
    plan, route, rows, g = make_route(mrs, ctx, tokens, experts, topk, align, seed=11)
    dev = ctx.device
    assert tokens * topk * hidden * torch.finfo(dtype).bits // 8 >= 256 << 20
    rand = torch.Generator(device=dev).manual_seed(12)
    x, _ = view(torch.randn(rows, hidden, generator=rand, device=dev).to(dtype), 5, 1, dev)
    row_of_slot = route.row_of_slot
    used = torch.zeros(rows, dtype=torch.bool, device=dev)
    used[row_of_slot[row_of_slot >= 0].long()] = True
    x[~used] = float("nan")  # rows nobody has are not read into anything
    w = torch.randn(tokens, topk, generator=rand, device=dev)
    w[row_of_slot < 0] = float("nan")
    for weights in (w, None):
        out, wide = view(torch.zeros(tokens, hidden, dtype=dtype, device=dev), 3, 2, dev)
        if weights is None:
            plan.dispatch_backward(x, route, x_grad_out=out)
        else:
            plan.combine(x, route, weights, out=out)
        want, size = row_sums(x, row_of_slot, weights)
        sums = topk * U32 * 1.01 * size
        within(out, want, sums + half_step(dtype) * (want.abs() + sums) + smallest(dtype), "rows")
        assert untouched(wide, hidden, 2)
    del want, size, sums, out, wide
    dout, _ = view(torch.randn(tokens, hidden, generator=rand, device=dev).to(dtype), 7, 3, dev)
    before = torch.randn(rows, hidden, generator=rand, device=dev).to(dtype)
    drows, wide = view(before, 1, 1, dev)
    _, dw = plan.combine_backward(dout, x, route, w, drows_out=drows)
    want = torch.zeros(rows, hidden, dtype=dtype, device=dev)
    end = int(route.offsets[-1])
    want[end:] = before[end:]
    assert torch.equal(drows[~used], want[~used])  # padding: zeros; behind the last segment: as it was
    assert untouched(wide, hidden, 1)
    for j in range(topk):
        token = torch.nonzero(row_of_slot[:, j] >= 0).squeeze(1)
        r, grad = row_of_slot[token, j].long(), dout[token].double()
        want = grad * w[token, j : j + 1].double()
        within(drows[r], want, (half_step(dtype) + 1.01 * U32) * want.abs() + smallest(dtype), "rows_grad")
        product = grad * x[r].double()
        within(dw[token, j], product.sum(1), (hidden / 64 + 16) * U32 * 1.01 * product.abs().sum(1) + 2.0**-149, "weights_grad")
    assert bool((dw[row_of_slot < 0] == 0).all())
    plan.close()


def test_wide_rows_past_4_gib(ctx, mrs):
    """Rows of more than 64 vectors, and scores, in a buffer whose rows are 2 x 65792 bytes apart: offsets beyond 32 bits on the
    side of the tokens and on that of the rows."""
    tokens, experts, topk, hidden, stride = 33000, 16, 1, 1109, 65792
    dev = ctx.device
    plan, route, rows, g = make_route(mrs, ctx, tokens, experts, topk, 4, drop=0.01)
    assert tokens * stride * 2 > 1 << 32
    row_of_slot = route.row_of_slot[:, 0].long()
    has = row_of_slot >= 0
    here, there = torch.zeros(tokens, stride, dtype=BF16, device=dev), torch.zeros(rows, stride, dtype=BF16, device=dev)
    rand = torch.Generator(device=dev).manual_seed(13)
    x, out, moved, grads = here[:, 7 : 7 + hidden], here[:, 50001 : 50001 + hidden], there[:, 3 : 3 + hidden], there[:, 60000 : 60000 + hidden]
    x.copy_(torch.randn(tokens, hidden, generator=rand, device=dev))
    plan.dispatch(x, route, rows_out=moved)
    assert torch.equal(moved[row_of_slot[has]], x[has])
    w = torch.randn(tokens, 1, generator=rand, device=dev)
    plan.combine(moved, route, w, out=out)
    want = torch.where(has.unsqueeze(1), w.double() * x.double(), 0.0)
    off = (half_step(BF16) + 1.01 * U32) * want.abs() + smallest(BF16)  # a product, rounded to 32 bits and then to the type
    within(out, want, off, "combine")
    _, dw = plan.combine_backward(x, moved, route, w, drows_out=grads)
    within(grads[row_of_slot[has]], want[has], off[has], "rows_grad")
    product = torch.where(has.unsqueeze(1), x.double() * x.double(), 0.0)
    within(dw[:, 0], product.sum(1), (hidden / 64 + 16) * U32 * 1.01 * product.sum(1), "weights_grad")
    plan.dispatch_backward(moved, route, x_grad_out=out)
    assert torch.equal(out, torch.where(has.unsqueeze(1), x, 0.0))
    assert int(torch.count_nonzero(here)) == int(torch.count_nonzero(x)) + int(torch.count_nonzero(out))
    assert int(torch.count_nonzero(there)) == int(torch.count_nonzero(moved)) + int(torch.count_nonzero(grads))
    plan.close()
    del there, moved, grads
    plan = mrs.RoutePlan(ctx, tokens, 100, 2, normalize=True)
    scores, scores_grad = here[:, 31 : 131], here[:, 40000 : 40100]
    scores.copy_(torch.randn(tokens, 100, generator=rand, device=dev))
    ids, weights = plan.select(scores)
    plan.select_backward(scores, ids, torch.cat([w, -w], 1), scores_grad_out=scores_grad)
    apart = scores.contiguous()
    want = plan.select(apart)
    assert torch.equal(ids, want[0]) and torch.equal(weights, want[1])
    assert torch.equal(ids.long(), torch.sort(apart.float(), dim=1, descending=True, stable=True).indices[:, :2])
    assert torch.equal(scores_grad, plan.select_backward(apart, ids, torch.cat([w, -w], 1)))


# ---- more work than one grid takes ----------------------------------------------------------------
def test_more_tokens_than_a_grid_selects_for(ctx, mrs):
    """2^25 tokens and some: a workgroup's rows and then others.  One of two experts by a softmax over both, p = 1 / (1 + exp(-|s0 - s1|)):
    the gradient is p (1 - p) g for the chosen one and its negative for the other.  Roundings as in `check_select`, whose count holds
    for any number of experts."""
    tokens, dev = (1 << 25) + 1001, ctx.device
    plan = mrs.RoutePlan(ctx, tokens, 2, 1, gate=gates(mrs)["softmax"], normalize=False)
    rand = torch.Generator(device=dev).manual_seed(14)
    scores = torch.randn(tokens, 2, generator=rand, device=dev, dtype=F16)
    g = torch.randn(tokens, 1, generator=rand, device=dev)
    ids, w = plan.select(scores)
    assert torch.equal(ids[:, 0] == 1, scores[:, 1] > scores[:, 0])
    apart = (scores[:, 0].double() - scores[:, 1].double()).abs()
    p = 1.0 / (1.0 + torch.exp(-apart))
    rel = 2 * (2 * float(2 * scores.double().abs().max()) + 30) * U32
    within(w[:, 0], p, rel * p, "weights")
    ds = plan.select_backward(scores, ids, g)
    want = p * (1.0 - p) * g[:, 0].double()
    tol = 2 * (rel + 7 * U32) * g[:, 0].abs().double() + half_step(F16) * want.abs() + smallest(F16)
    first = ids[:, 0] == 0
    within(ds[:, 0], torch.where(first, want, -want), tol, "scores_grad")
    within(ds[:, 1], torch.where(first, -want, want), tol, "scores_grad")
    plan.close()


@pytest.mark.parametrize("log2_tokens,hidden,dtype", [(27, 1, F16), (27, 4, F32), (24, 264, F16)])
def test_more_tokens_than_a_grid_moves(ctx, mrs, log2_tokens, hidden, dtype):
    """Rows shorter than a vector, of one vector, and of a wave.  One slot a token, so that rows and their sums come through unchanged
    and a product p is rounded to 32 bits, off by u |p|, and then to its type, off by half(T) (1 + u) |p|: together at most
    (half(T) + 1.01 u) |p|.  The device can also do both at once, to half(T) |p|."""
    tokens, dev = (1 << log2_tokens) + 777, ctx.device
    plan = mrs.RoutePlan(ctx, tokens, 1, 1)
    rand = torch.Generator(device=dev).manual_seed(15)
    row_of_slot = torch.randperm(tokens, generator=rand, device=dev, dtype=torch.int32)
    row_of_slot[torch.rand(tokens, generator=rand, device=dev) < 0.1] = -1
    ends = torch.tensor([tokens], dtype=torch.int32, device=dev)  # align is 1: not read
    route = mrs.RouteMap(row_of_slot.reshape(tokens, 1), torch.empty(tokens, dtype=torch.int32, device=dev), ends, torch.cat([ends, ends]))
    x = torch.randn(tokens, hidden, generator=rand, device=dev, dtype=dtype)
    w = torch.randn(tokens, 1, generator=rand, device=dev)
    rows, grads = torch.zeros_like(x), torch.zeros_like(x)
    plan.dispatch(x, route, rows_out=rows)
    out = plan.combine(rows, route, w)
    back = plan.dispatch_backward(rows, route)
    _, dw = plan.combine_backward(x, rows, route, w, drows_out=grads)
    step = (1 << 28) // hidden
    for lo in range(0, tokens, step):
        part = slice(lo, lo + step)
        r = row_of_slot[part].long()
        has = r >= 0
        r = r[has]
        got, weighted = x[part][has], (w[part].double() * x[part].double())[has]
        off = (half_step(dtype) + 1.01 * U32) * weighted.abs() + smallest(dtype)
        assert torch.equal(rows[r], got) and torch.equal(back[part][has], got)
        within(out[part][has], weighted, off, "combine")
        within(grads[r], weighted, off, "rows_grad")
        lost = ~has
        assert not bool(back[part][lost].any()) and not bool(out[part][lost].any()) and not bool(dw[part][lost].any())
        product = got.double() * got.double()
        within(dw[part][has][:, 0], product.sum(1), (hidden / 64 + 16) * U32 * 1.01 * product.sum(1) + 2.0**-149, "weights_grad")
    kept = row_of_slot >= 0
    assert int(rows.ne(0).any(1).sum()) == int(x[kept].ne(0).any(1).sum())  # no row that no slot has
    plan.close()
