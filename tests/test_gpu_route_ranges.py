"""Token routing on the GPU at the ends of its ranges: small calls of a large plan, moves of hundreds of MiB, more work
than one grid takes, offsets past 4 GiB."""
import pytest
import torch

import route_ref as ref
from test_gpu_route import check_order, mrs  # noqa: F401

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
