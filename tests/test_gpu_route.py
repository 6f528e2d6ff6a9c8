"""infmoe_route_topk against the float64 oracle: ids equal, weights to FP32's roundings."""
import numpy as np
import pytest

from infmoe_amd import capi
from oracle import topk_oracle as O

pytestmark = pytest.mark.gpu

# Weights: expf to 2 ulp on an argument with one rounding (|x| u each, |x| < 24 here), a sum of at most 1024 terms in pairs
# (log2 = 10 roundings), two quotients: below 2 (24 + 2 + 10 + 4) u = 80 u, u = 2^-24, of a weight.  2^-17 is 128 u.
RTOL = 2.0 ** -17


def tensors(torch, x, dtype):
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda().to(getattr(torch, dtype))
    return t, t.float().cpu().numpy()


def check(got, want):
    ids, w = (g.cpu().numpy() for g in got)
    np.testing.assert_array_equal(ids, want[0])
    np.testing.assert_allclose(w, want[1], rtol=RTOL, atol=1e-38)


CASES = [  # T, E, k, groups, top_groups, group_top
    (1, 1, 1, 1, 1, 1), (1, 64, 2, 1, 1, 1), (3, 5, 5, 1, 1, 1), (1000, 8, 2, 1, 1, 1), (333, 32, 2, 1, 1, 1), (65, 60, 6, 1, 1, 1),
    (70, 256, 8, 1, 1, 1), (70, 256, 8, 8, 4, 2), (129, 128, 16, 4, 2, 2), (33, 257, 8, 1, 1, 1), (17, 512, 32, 1, 1, 1),
    (9, 1024, 32, 1, 1, 1), (40, 20, 17, 1, 1, 1), (50, 63, 4, 3, 2, 1), (50, 63, 4, 3, 2, 2), (21, 1023, 8, 3, 1, 2),
    (21, 1020, 9, 5, 3, 2), (15, 64, 3, 64, 7, 1), (15, 128, 3, 64, 7, 2), (12, 1020, 10, 17, 16, 2), (31, 160, 6, 8, 3, 1),
    (11, 990, 7, 33, 5, 1), (2, 6, 4, 2, 2, 2),
]


@pytest.mark.parametrize("T,E,k,groups,top_groups,group_top", CASES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_matches_oracle(lib, torch_cuda, T, E, k, groups, top_groups, group_top, score):
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(T * 7 + E * 3 + k)
    x = (2.0 * rng.standard_normal((T, E))).astype(np.float32)
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    for dtype in ("float32", "bfloat16", "float16"):
        t, exact = tensors(torch, x, dtype)
        for b in (None, bias):
            for renormalize in (True, False):
                kw = dict(score=score, groups=groups, top_groups=top_groups, group_top=group_top, renormalize=renormalize, scale=2.5)
                print(f"route T={T} E={E} k={k} groups={groups}/{top_groups}/{group_top} {dtype} {score} bias={b is not None}", flush=True)
                got = ops.route_topk(t, k, bias=None if b is None else torch.from_numpy(b).cuda(), **kw)
                check(got, O.route_topk(exact, k, bias=b, **kw))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups,group_top", [(1, 1, 1), (4, 2, 1), (4, 2, 2)])
def test_equal_scores_pick_the_lowest_index(lib, torch_cuda, score, groups, top_groups, group_top):
    torch = torch_cuda
    from infmoe_amd import ops
    x = np.random.default_rng(1).integers(-1, 2, size=(200, 48)).astype(np.float32)  # a handful of values: ties everywhere
    x[7] = 0.0
    for bias in (None, np.zeros(48, np.float32), np.full(48, 0.25, np.float32)):
        kw = dict(score=score, groups=groups, top_groups=top_groups, group_top=group_top)
        got = ops.route_topk(torch.from_numpy(x).cuda(), 6, bias=None if bias is None else torch.from_numpy(bias).cuda(), **kw)
        check(got, O.route_topk(x, 6, bias=bias, **kw))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_closer_than_fp32_are_ordered_in_64_bits(lib, torch_cuda, score):
    """Scores plus bias that agree to 1e-9 .. 1e-7 relative: below a rounding of FP32, far above one of 64 bits."""
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(5)
    T, E = 257, 64
    x = rng.standard_normal((T, E)).astype(np.float32)
    x[:, 32:] = x[:, :32]  # pairs of equal scores ...
    bias = np.zeros(E, np.float32)
    bias[32:] = (10.0 ** rng.uniform(-9, -7, 32) * rng.choice([-1, 1], 32)).astype(np.float32)  # ... that the bias sets apart
    for kw in (dict(), dict(groups=4, top_groups=2, group_top=2), dict(groups=2, top_groups=1, group_top=2)):
        got = ops.route_topk(torch.from_numpy(x).cuda(), 8, score=score, bias=torch.from_numpy(bias).cuda(), **kw)
        check(got, O.route_topk(x, 8, score=score, bias=bias, **kw))


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_masked_and_unordered_rows(lib, torch_cuda, score, scored, groups, top_groups):
    torch = torch_cuda
    from infmoe_amd import ops
    inf, nan = np.inf, np.nan
    x = np.random.default_rng(2).standard_normal((12, 32)).astype(np.float32)
    x[0] = -inf                      # nothing left
    x[1, 1:] = -inf                  # one expert left
    x[2, :30] = -inf                 # two, fewer than k
    x[3, 5] = nan
    x[4, 5] = inf                    # the logistic function takes it, softmax cannot
    x[5] = nan
    x[6] = np.finfo(np.float32).min  # the type's lowest value is a score, no mask
    x[7] = -200.0                    # scores below FP32's range
    x[7, 3] = -199.0
    x[8, ::2] = -inf
    x[9] = 120.0
    x[9, 2] = 121.0
    x[10, 0] = np.finfo(np.float32).min
    bias = np.zeros(32, np.float32)
    bias[9] = -inf                   # an expert switched off for all
    kw = dict(score=score, groups=groups, top_groups=top_groups, group_top=1, bias=bias if scored else None)
    for renormalize in (True, False):
        want = O.route_topk(x, 4, renormalize=renormalize, **kw)
        got = ops.route_topk(torch.from_numpy(x).cuda(), 4, renormalize=renormalize,
                             **{**kw, "bias": torch.from_numpy(bias).cuda() if scored else None})
        check(got, want)
    bias[3] = nan
    ids, w = ops.route_topk(torch.from_numpy(x).cuda(), 4, score=score, bias=torch.from_numpy(bias).cuda())
    want = O.route_topk(x, 4, score=score, bias=bias)
    check((ids, w), want)
    assert np.isnan(want[1][11]).all()


@pytest.mark.parametrize("E,k,groups,top_groups,group_top", [
    (256, 8, 8, 4, 2), (256, 15, 1, 1, 1), (200, 6, 1, 1, 1), (128, 8, 4, 1, 2), (96, 2, 3, 2, 1), (250, 16, 1, 1, 1), (72, 10, 8, 2, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_large_batches(lib, torch_cuda, E, k, groups, top_groups, group_top, score):
    """Batches long enough for several rows of many experts per wave, with everything a row can bring on the way: equal scores
    (more of them than a short list holds), masked experts, rows without order, scores closer than FP32 orders."""
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(E + k)
    T = 4101
    x = (2.0 * rng.standard_normal((T, E))).astype(np.float32)
    x[1::7] = np.round(x[1::7])                       # many equal
    x[2] = 0.5                                        # all equal
    x[3, 5:] = -np.inf
    x[4] = -np.inf
    x[5, 1] = np.nan
    x[6, 2] = np.inf
    x[9::11][rng.random((len(x[9::11]), E)) < 0.5] = -np.inf
    x[4100, :E // 2] = x[4100, E // 2:E // 2 * 2]
    near = (10.0 ** rng.uniform(-9, -6, E) * rng.choice([-1, 1], E)).astype(np.float32)
    for dtype, bias in (("float32", None), ("float32", near), ("bfloat16", near), ("float16", None)):
        t, exact = tensors(torch, x, dtype)
        kw = dict(score=score, groups=groups, top_groups=top_groups, group_top=group_top)
        check(ops.route_topk(t, k, bias=None if bias is None else torch.from_numpy(bias).cuda(), **kw), O.route_topk(exact, k, bias=bias, **kw))


def test_strided_rows_offsets_and_given_outputs(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    x = np.random.default_rng(3).standard_normal((100, 70)).astype(np.float32)
    big = torch.full((100, 131), float("nan"), dtype=torch.bfloat16, device="cuda")
    view = big[:, 3:73]  # not on a 16-byte boundary, rows apart
    view.copy_(torch.from_numpy(x))
    want = O.route_topk(view.float().cpu().numpy(), 5)
    check(ops.route_topk(view, 5), want)
    guard_i, guard_w = torch.full((102, 5), 77, dtype=torch.int32, device="cuda"), torch.full((102, 5), 7.0, device="cuda")
    ops.route_topk(view, 5, out=(guard_i[1:101], guard_w[1:101]))
    check((guard_i[1:101], guard_w[1:101]), want)
    assert (guard_i[[0, 101]] == 77).all() and (guard_w[[0, 101]] == 7.0).all()  # rows around the output stay as they were
    ids, w = ops.route_topk(view[:0], 5)
    assert ids.shape == (0, 5) and w.shape == (0, 5)


def test_offsets_beyond_32_bits(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    stride = (1 << 31) + 8
    big = torch.empty(stride + 16, dtype=torch.float16, device="cuda")
    rows = big.as_strided((2, 16), (stride, 1))
    x = np.random.default_rng(4).standard_normal((2, 16)).astype(np.float16)
    rows.copy_(torch.from_numpy(x))
    check(ops.route_topk(rows, 3), O.route_topk(x, 3))


def test_on_another_stream_and_in_a_graph(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(6)
    x = torch.empty(300, 64, device="cuda")
    bias = torch.from_numpy((0.1 * rng.standard_normal(64)).astype(np.float32)).cuda()
    kw = dict(score="sigmoid", groups=8, top_groups=3, group_top=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x.copy_(torch.from_numpy(rng.standard_normal((300, 64)).astype(np.float32)))
        first = ops.route_topk(x, 4, bias=bias, **kw)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    check(first, O.route_topk(x.cpu().numpy(), 4, bias=bias.cpu().numpy(), **kw))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.route_topk(x, 4, bias=bias, **kw)
    for _ in range(3):
        x.copy_(torch.from_numpy(rng.standard_normal((300, 64)).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        check(out, O.route_topk(x.cpu().numpy(), 4, bias=bias.cpu().numpy(), **kw))


def test_python_binding_refuses_what_does_not_fit(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    x = torch.zeros(4, 8, device="cuda")
    for call in (lambda: ops.route_topk(x.double(), 2), lambda: ops.route_topk(x.cpu(), 2), lambda: ops.route_topk(x.t(), 2),
                 lambda: ops.route_topk(x, 2, bias=torch.zeros(7, device="cuda")), lambda: ops.route_topk(x, 2, bias=torch.zeros(8)),
                 lambda: ops.route_topk(x, 2, score="tanh"), lambda: ops.route_topk(x, 9), lambda: ops.route_topk(x, 0),
                 lambda: ops.route_topk(x, 5, groups=2), lambda: ops.route_topk(x, 2, groups=3),
                 lambda: ops.route_topk(x, 2, out=(torch.zeros(4, 3, dtype=torch.int32, device="cuda"), torch.zeros(4, 2, device="cuda"))),
                 lambda: ops.route_topk(x[0], 2)):
        with pytest.raises(capi.InfMoEError) as ei:
            call()
        assert ei.value.status == capi.ERR_INVALID_ARGUMENT
