"""Token routing on the GPU at the ends of its ranges: small calls of a large plan, moves of hundreds of MiB, more work
than one grid takes, offsets past 4 GiB."""
import pytest
import torch

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
