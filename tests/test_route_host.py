"""Token routing without a GPU: the sizes the library reports, what it refuses, and that the definitions
the GPU tests compare with have the derivatives they say."""
import ctypes

import pytest
import torch

import route_ref as ref
import wgpu_morton_code_radix_sort_test_amd as mrs
from wgpu_morton_code_radix_sort_test_amd import _lib


@pytest.fixture(autouse=True)
def no_message_left_behind():
    """Refusals leave a message with the thread until the next call that succeeds."""
    yield
    assert _lib.load_library().mrs_route_destroy(None) == _lib.MRS_OK


def _desc(**kw):
    d = dict(tokens=100, experts=8, topk=2, align=1, gate=0, capacity=0, normalize=1, scale=1.0)
    d.update(kw)
    return _lib.RouteDesc(*[d[name] for name, _ in _lib.RouteDesc._fields_])


def _max_rows(**kw):
    rows = ctypes.c_uint64()
    return _lib.load_library().mrs_route_max_rows(ctypes.byref(_desc(**kw)), ctypes.byref(rows)), rows.value


@pytest.mark.parametrize("tokens,experts,topk,align,capacity,want", [
    (100, 8, 2, 1, 0, 200),
    (100, 8, 2, 16, 0, 200 + 8 * 15),
    (1, 256, 4, 16, 0, 4 + 4 * 15),  # only experts with a row need filling up
    (0, 8, 2, 16, 0, 0),
    (1000, 8, 2, 1, 10, 80),
    (1000, 8, 2, 16, 10, 8 * 16),
    (10, 8, 2, 1, 1000, 20),  # a capacity that limits nothing
])
def test_max_rows(tokens, experts, topk, align, capacity, want):
    assert _max_rows(tokens=tokens, experts=experts, topk=topk, align=align, capacity=capacity) == (_lib.MRS_OK, want)


def test_max_rows_holds_the_fullest_ordering():
    g = torch.Generator().manual_seed(3)
    for _ in range(50):
        tokens, experts, topk = (int(torch.randint(1, hi, (1,), generator=g)) for hi in (40, 12, 6))
        align, capacity = int(torch.randint(1, 9, (1,), generator=g)), int(torch.randint(0, 12, (1,), generator=g))
        ids = torch.randint(-1, experts, (tokens, topk), generator=g)
        rows = _max_rows(tokens=tokens, experts=experts, topk=topk, align=align, capacity=capacity)[1]
        offsets = ref.order(ids, experts, align, capacity, 10000)[3]
        assert int(offsets[-1]) <= rows


def test_max_rows_never_falls_as_tokens_grow():
    """A plan's buffers hold the ordering of any smaller call."""
    g = torch.Generator().manual_seed(4)
    shapes = [(8, 2, 64, 64), (64, 8, 128, 128), (8, 2, 128, 128), (64, 1, 128, 100), (1024, 32, 1024, 1), (3, 1, 7, (1 << 64) - 1)]
    for _ in range(60):
        experts, topk, align = (int(torch.randint(1, hi, (1,), generator=g)) for hi in (65, 9, 130))
        shapes.append((experts, topk, align, int(torch.randint(1, 200, (1,), generator=g))))
    for experts, topk, align, capacity in shapes:
        before = 0
        for tokens in range(0, 300):
            rc, rows = _max_rows(tokens=tokens, experts=experts, topk=topk, align=align, capacity=capacity)
            assert rc == _lib.MRS_OK and rows >= before, (experts, topk, align, capacity, tokens)
            before = rows


@pytest.mark.parametrize("kw,word", [
    (dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(topk=0), "topk"), (dict(topk=33), "topk"),
    (dict(align=0), "align"), (dict(align=1025), "align"), (dict(gate=2), "gate"), (dict(normalize=2), "normalize"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(tokens=1 << 31), "tokens"),
    (dict(tokens=1 << 30, topk=2), "tokens"), (dict(tokens=(1 << 64) - 1), "tokens"),
])
def test_bad_descriptions_are_refused(kw, word):
    rc, _ = _max_rows(**kw)
    assert rc == _lib.MRS_ERR_INVALID_ARGUMENT
    assert word in _lib.load_library().mrs_last_error_string().decode()


class _ContextOnTheCpu:
    """Enough of a context for the checks before a handle is made."""

    def __init__(self):
        self.lib, self.device, self._h = _lib.load_library(), torch.device("cpu"), None


@pytest.mark.parametrize("name", ["tokens", "experts", "topk", "align", "gate", "capacity"])
def test_numbers_that_do_not_fit_their_field_are_refused(name):
    """A field keeps the low bits of what it is given: 2^32 + 4 would go for 4."""
    wide = 64 if name in ("tokens", "capacity") else 32
    args = dict(tokens=8, experts=8, topk=2, align=1, capacity=0, gate=0)
    with pytest.raises(mrs.MrsError, match="null argument"):  # right ones get as far as the missing context
        mrs.RoutePlan(_ContextOnTheCpu(), **args)
    for off in (1 << wide, -(1 << wide)):
        with pytest.raises(ValueError, match=name):
            mrs.RoutePlan(_ContextOnTheCpu(), **{**args, name: args[name] + off})


def test_null_arguments_are_refused():
    lib = _lib.load_library()
    rows = ctypes.c_uint64()
    bad = _lib.MRS_ERR_INVALID_ARGUMENT
    assert lib.mrs_route_max_rows(None, ctypes.byref(rows)) == bad
    assert lib.mrs_route_create(None, ctypes.byref(_desc()), None) == bad
    assert lib.mrs_route_destroy(None) == _lib.MRS_OK
    assert lib.mrs_route_select(None, 1, None, 8, 0, None, None, None, None) == bad
    assert lib.mrs_route_select_backward(None, 1, None, 8, 0, None, None, None, None, 8, None) == bad
    assert lib.mrs_route_order(None, 1, None, None, None) == bad
    assert lib.mrs_route_dispatch(None, 1, None, 0, 8, None, 8, None, 8, None) == bad
    assert lib.mrs_route_dispatch_backward(None, 1, None, 0, 8, None, 8, None, 8, None) == bad
    assert lib.mrs_route_combine(None, 1, None, 0, 8, None, 8, None, None, 8, None) == bad
    assert lib.mrs_route_combine_backward(None, 1, None, 0, 8, None, 8, None, 8, None, None, 8, None, None) == bad


def _plan_on_the_cpu(tokens=4, experts=8, topk=2):
    """The Python checks alone: a plan without a handle, on CPU tensors."""
    plan = object.__new__(mrs.RoutePlan)
    plan.device, plan.lib, plan._h = torch.device("cpu"), _lib.load_library(), None
    plan.tokens, plan.experts, plan.topk, plan.max_rows = tokens, experts, topk, tokens * topk
    return plan


def test_tensor_checks(monkeypatch):
    from wgpu_morton_code_radix_sort_test_amd import api

    monkeypatch.setattr(api, "_raw_stream", lambda index: 0)
    plan = _plan_on_the_cpu()
    route = plan.new_map()
    x, rows = torch.zeros(4, 6), torch.zeros(8, 6)
    ids, w = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    scores = torch.zeros(4, 8)
    # right arguments get as far as the library, which misses the handle
    for call in (lambda: plan.select(scores), lambda: plan.select_backward(scores, ids, w), lambda: plan.order(ids, route),
                 lambda: plan.dispatch(x, route), lambda: plan.dispatch_backward(rows, route), lambda: plan.combine(rows, route, w),
                 lambda: plan.combine_backward(x, rows, route, w), lambda: plan.dispatch(x.to(torch.uint8), route)):
        with pytest.raises(mrs.MrsError, match="null handle"):
            call()
    wrong = [
        lambda: plan.select(torch.zeros(4, 7)), lambda: plan.select(torch.zeros(4, 8, dtype=torch.float64)),
        lambda: plan.select(torch.zeros(8, 4).t()), lambda: plan.select(scores, torch.zeros(7)),
        lambda: plan.select(scores, torch.zeros(8, dtype=torch.float16)), lambda: plan.select(torch.zeros(8)),
        lambda: plan.select(scores, ids_out=torch.zeros(4, 2, dtype=torch.int64)),
        lambda: plan.select(scores, weights_out=torch.zeros(3, 2)),
        lambda: plan.select_backward(scores, ids.long(), w), lambda: plan.select_backward(scores, ids, w.half()),
        lambda: plan.select_backward(scores, ids, w, scores_grad_out=torch.zeros(4, 8, dtype=torch.float16)),
        lambda: plan.order(ids.long()), lambda: plan.order(ids[:, :1]), lambda: plan.order(ids.t().contiguous().t(), route),
        lambda: plan.order(torch.zeros(5, 2, dtype=torch.int32), route),  # more tokens than the map holds
        lambda: plan.dispatch(x.double(), route), lambda: plan.dispatch(torch.zeros(6, 4).t(), route),
        lambda: plan.dispatch(x, route, rows_out=torch.zeros(8, 5)), lambda: plan.dispatch(x, route, rows_out=rows.half()),
        lambda: plan.dispatch(torch.zeros(5, 6), route), lambda: plan.dispatch(torch.zeros(6), route),
        lambda: plan.dispatch_backward(rows.to(torch.uint8), route), lambda: plan.dispatch_backward(rows[:7], route),
        lambda: plan.combine(rows, route, w.half()), lambda: plan.combine(rows, route, w, out=torch.zeros(4, 7)),
        lambda: plan.combine(rows, route, torch.zeros(2)), lambda: plan.combine(rows.t().contiguous().t(), route, w),
        lambda: plan.combine_backward(x.half(), rows, route, w), lambda: plan.combine_backward(x[:3], rows, route, w),
        lambda: plan.combine_backward(x, rows, route, w, dweights_out=torch.zeros(4, 2, dtype=torch.float16)),
        lambda: plan.dispatch(x, mrs.RouteMap(route.row_of_slot.long(), route.slot_of_row, route.counts, route.offsets)),
        lambda: plan.dispatch(x, mrs.RouteMap(route.row_of_slot, route.slot_of_row, route.counts, route.offsets[:8])),
    ]
    for i, call in enumerate(wrong):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    plan.device = torch.device("cuda", 0)  # tensors elsewhere than the plan
    with pytest.raises(ValueError, match="is on"):
        plan.dispatch(x, route)


class _LibraryThatTakesEverything:
    """Stands in for the library where only the numbers handed to it matter."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args[1]))
            return _lib.MRS_OK

        return call


def test_dispatch_backward_takes_the_tokens_that_were_ordered(monkeypatch):
    """Entries of row_of_slot behind the ordered tokens are not read as rows, whoever ordered how many before."""
    from wgpu_morton_code_radix_sort_test_amd import api

    captured = [False]
    monkeypatch.setattr(api, "_raw_stream", lambda index: 1 if captured[0] else 0)  # the null stream is never captured
    monkeypatch.setattr(api, "_capturing", lambda: captured[0])
    plan = _plan_on_the_cpu(tokens=6)
    plan.lib = _LibraryThatTakesEverything()
    grad = torch.zeros(plan.max_rows, 5)
    ids = torch.zeros(6, 2, dtype=torch.int32)

    def took(route, **kw):
        out = plan.dispatch_backward(grad, route, **kw)
        assert plan.lib.calls[-1] == ("mrs_route_dispatch_backward", out.size(0))
        return out.size(0)

    route = plan.new_map()
    assert took(route) == 6  # nothing known of it: all it holds
    for tokens in (6, 2, 4, 6, 1, 0):
        assert plan.order(ids[:tokens], route) is route
        assert took(route) == tokens
        assert took(route, tokens=3) == 3
    with pytest.raises(ValueError, match="x_grad_out"):
        plan.dispatch_backward(grad, route, x_grad_out=torch.zeros(6, 5))
    assert took(plan.order(ids[:2])) == 2
    # a map somebody else wrote, or a view of one, holds what it has room for
    assert took(mrs.RouteMap(route.row_of_slot[:5], route.slot_of_row, route.counts, route.offsets)) == 5
    # a refused ordering changes nothing
    with pytest.raises(ValueError):
        plan.order(ids.long(), route)
    assert took(route) == 0
    # captured orderings run again when nobody says so: the count stands as long as all agree on it
    route, captured[0] = plan.new_map(), True
    plan.order(ids[:3], route)
    assert took(route) == 3
    captured[0] = False
    plan.order(ids[:3], route)
    assert took(route) == 3
    plan.order(ids[:4], route)
    plan.order(ids[:3], route)
    with pytest.raises(ValueError, match="tokens"):
        plan.dispatch_backward(grad, route)
    assert took(route, tokens=3) == 3


@pytest.mark.parametrize("gate", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
def test_derivative_formula_matches_differences(gate, normalize):
    """Central differences of the definition in 64 bits: an error of h^2 / 6 times the third derivative, which is
    below 60 for |dw| <= 1 (cumulants of at most unit variables), and of 2^-52 / h: together below 1e-7 for h = 2^-14."""
    g = torch.Generator().manual_seed(1)
    s = (torch.randperm(12, generator=g).double() * 0.25 - 1).reshape(1, 12)
    s[0, 3] = -ref.INF
    ids = ref.select_ids(s, None, 4)
    dw = torch.rand(1, 4, generator=g, dtype=torch.float64) * 2 - 1
    got = ref.scores_grad(s, None, ids, dw, gate, normalize, 1.5)
    h = 2.0**-14
    for e in range(12):
        up, down = s.clone(), s.clone()
        up[0, e] += h
        down[0, e] -= h
        f = [float((ref.weights(x, None, ids, gate, normalize, 1.5) * dw).sum()) for x in (up, down)]
        want = 0.0 if e == 3 else (f[0] - f[1]) / (2 * h)
        assert abs(float(got[0, e]) - want) < 1e-7 * 1.5
