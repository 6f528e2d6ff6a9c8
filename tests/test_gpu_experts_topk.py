"""infmoe_experts_topk against the float64 oracle, every value within the bound of its roundings."""
import numpy as np
import pytest

from infmoe_amd import capi
from oracle import topk_oracle as O
from tests.topk_util import DTYPES, FFNS, assert_within, draw_experts, typed

pytestmark = pytest.mark.gpu


def call(ops, c, **kw):
    return ops.experts_topk(c["x"], c["ids"], c["weights"], c["wi"], c["wo"], c["wi_1"], ffn=c["ffn"], **kw)


SHAPES = [  # T, k, E, d, h
    (1, 1, 1, 8, 8), (1, 2, 4, 64, 128), (1, 3, 2, 64, 40), (2, 2, 64, 512, 256), (5, 3, 7, 40, 24), (16, 2, 4, 128, 96), (17, 1, 2, 96, 160),
    (64, 2, 8, 256, 512), (130, 4, 16, 72, 200), (300, 2, 3, 128, 64), (33, 2, 5, 13, 29), (3, 2, 5, 131, 77), (70, 8, 64, 100, 52),
    (1100, 1, 2, 64, 96), (517, 3, 300, 32, 40), (9, 32, 40, 48, 64), (600, 2, 4, 264, 520), (1, 1, 1, 1, 1), (900, 1, 1, 136, 72),
    (700, 2, 1024, 8, 16),
]


@pytest.mark.parametrize("T,k,E,d,h", SHAPES)
@pytest.mark.parametrize("ffn", FFNS)
def test_experts_match_oracle(lib, torch_cuda, T, k, E, d, h, ffn):
    from infmoe_amd import ops
    for dtype in DTYPES:
        print(f"experts T={T} k={k} E={E} d={d} h={h} {ffn} {dtype}", flush=True)
        c = draw_experts(torch_cuda, np.random.default_rng(T + 10 * k + d), T, k, E, d, h, ffn, dtype)
        assert_within(call(ops, c), *O.experts_topk(**c["exact"]), what=f"{dtype} {ffn}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 7, 64, 300])
def test_experts_at_long_rows(lib, torch_cuda, dtype, T):
    """Rows of the benchmark's layer, fewer experts."""
    from infmoe_amd import ops
    c = draw_experts(torch_cuda, np.random.default_rng(T), T, 2, 3, 2048, 1536, "gated_silu", dtype)
    assert_within(call(ops, c), *O.experts_topk(**c["exact"]), what=dtype)


@pytest.mark.parametrize("dtype,ffn", [("bfloat16", "gated_silu"), ("float16", "relu"), ("float32", "gated_gelu")])
def test_experts_on_tall_tiles(lib, torch_cuda, dtype, ffn):
    """Enough rows and columns for tiles of up to 256 x 256: experts with no row, one row, a few, and several tiles; row lengths
    that are no whole number of steps.  A sample of the tokens against the oracle, the others by a second call in which the
    tokens stand in another order."""
    torch = torch_cuda
    from infmoe_amd import ops
    T, k, E, d, h = 1280, 3, 16, 2056, 2072
    rng = np.random.default_rng(12)
    c = draw_experts(torch, rng, T, k, E, d, h, ffn, dtype)
    odds = np.array([0, 0.0002, 0.01, 0.02, 0.05, 0.05, 0.06, 0.07, 0.08, 0.08, 0.08, 0.09, 0.1, 0.1, 0.1, 0.1])
    ids = rng.choice(E, size=(T, k), p=odds / odds.sum()).astype(np.int32)
    ids[17] = [1, 1, 15]
    ids[18] = -1
    c["ids"].copy_(torch.from_numpy(ids))
    y = call(ops, c)
    some = np.concatenate([[17, 18], rng.choice(T, 40, replace=False)])
    exact = dict(c["exact"], x=c["exact"]["x"][some], ids=ids[some], weights=c["exact"]["weights"][some])
    assert_within(y[torch.from_numpy(some).cuda()], *O.experts_topk(**exact), what=f"{dtype} {ffn}")
    order = torch.from_numpy(rng.permutation(T)).cuda()
    again = ops.experts_topk(c["x"][order], c["ids"][order], c["weights"][order], c["wi"], c["wo"], c["wi_1"], ffn=ffn)
    assert torch.equal(again, y[order])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,k", [(6, 5, 3), (200, 6, 2), (40, 3, 4)])
def test_ids_that_are_no_expert_and_ids_twice(lib, torch_cuda, dtype, T, E, k):
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(3)
    c = draw_experts(torch, rng, T, k, E, 64, 80, "relu", dtype)
    ids = rng.integers(-2, E + 2, (T, k)).astype(np.int32)
    ids[0] = -1                                      # a token without any
    ids[1] = 1                                       # the same expert k times
    ids[2] = [np.iinfo(np.int32).min, np.iinfo(np.int32).max] * (k // 2) + [0] * (k % 2)
    weights = c["exact"]["weights"].copy()
    weights[3, 0] = np.nan                           # a row the routing could not order
    ids[3] = -1
    c["exact"].update(ids=ids, weights=weights)
    y = ops.experts_topk(c["x"], torch.from_numpy(ids).cuda(), torch.from_numpy(weights).cuda(), c["wi"], c["wo"], ffn="relu")
    want, bound = O.experts_topk(**c["exact"])
    assert (want[0] == 0).all() and np.isnan(want[3]).all()
    assert_within(y, want, bound)
    # no expert at all in the whole call
    y = ops.experts_topk(c["x"], torch.full((T, k), -1, dtype=torch.int32, device="cuda"), c["weights"], c["wi"], c["wo"], ffn="relu")
    assert (y == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [5, 150])
def test_nan_and_infinity_stay_in_their_rows(lib, torch_cuda, dtype, T):
    torch = torch_cuda
    from infmoe_amd import ops
    c = draw_experts(torch, np.random.default_rng(4), T, 2, 4, 64, 96, "gated_gelu", dtype)
    clean = call(ops, c)
    c["x"][2, 5] = float("nan")
    c["x"][4, 7] = float("inf")
    y = call(ops, c)
    others = [t for t in range(T) if t not in (2, 4)]
    assert torch.equal(y[others], clean[others])
    assert y[2].isnan().all() and not y[4].isfinite().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,h", [(64, 96), (50, 70)])
def test_strided_rows_packed_slots_and_guards(lib, torch_cuda, dtype, d, h):
    """Rows of x and y inside larger tensors; the experts as slots [gamma d | wi | wi_1 | wo] of one block."""
    torch = torch_cuda
    from infmoe_amd import ops
    T, E = 70, 5
    c = draw_experts(torch, np.random.default_rng(5), T, 2, E, d, h, "gated_silu", dtype)
    slots = torch.full((E, d + 3 * h * d + 16), float("nan"), dtype=c["x"].dtype, device="cuda")
    views = [slots[:, d + i * h * d:d + (i + 1) * h * d] for i in range(3)]
    wi, wi_1 = views[0].unflatten(1, (h, d)), views[1].unflatten(1, (h, d))
    wo = views[2].unflatten(1, (d, h))
    wi.copy_(c["wi"]), wi_1.copy_(c["wi_1"]), wo.copy_(c["wo"])
    big_x = torch.full((T, d + 24), float("nan"), dtype=c["x"].dtype, device="cuda")
    big_x[:, 8:8 + d] = c["x"]
    big_y = torch.full((T + 2, d + 9), 3.0, dtype=c["x"].dtype, device="cuda")
    y = big_y[1:T + 1, 4:4 + d]
    ops.experts_topk(big_x[:, 8:8 + d], c["ids"], c["weights"], wi, wo, wi_1, ffn="gated_silu", out=y)
    assert_within(y, *O.experts_topk(**c["exact"]))
    big_y[1:T + 1, 4:4 + d] = 3.0
    assert (big_y == 3.0).all()  # nothing around the output was written


def test_calls_repeat_bit_for_bit(lib, torch_cuda):
    from infmoe_amd import ops
    for T in (3, 40, 700):
        c = draw_experts(torch_cuda, np.random.default_rng(6), T, 4, 8, 128, 256, "relu", "bfloat16")
        first = call(ops, c)
        for _ in range(3):
            assert torch_cuda.equal(call(ops, c), first)


def test_weights_beyond_32_bit_offsets(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    T, E, d, h = 9, 3, 64, 64
    c = draw_experts(torch, np.random.default_rng(7), T, 2, E, d, h, "relu", "float16")
    gap = (1 << 31) + 64
    big = torch.empty(2 * gap + h * d, dtype=torch.float16, device="cuda")
    wi = big.as_strided((E, h, d), (gap, d, 1))
    big2 = torch.empty(2 * gap + 2 * h * d, dtype=torch.float16, device="cuda")
    wo = big2.as_strided((E, d, h), (gap, h, 1), h * d)
    wi.copy_(c["wi"]), wo.copy_(c["wo"])
    assert_within(ops.experts_topk(c["x"], c["ids"], c["weights"], wi, wo), *O.experts_topk(**c["exact"]))


def test_empty_batch_streams_and_graphs(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(8)
    for T, dtype in ((4, "bfloat16"), (90, "float32"), (1500, "float16")):
        c = draw_experts(torch, rng, T, 2, 6, 64, 128, "gated_gelu", dtype)
        assert ops.experts_topk(c["x"][:0], c["ids"][:0], c["weights"][:0], c["wi"], c["wo"], c["wi_1"], ffn=c["ffn"]).shape == (0, 64)
        want = call(ops, c)
        sides = [torch.cuda.Stream(), torch.cuda.Stream()]
        got = []
        for s in sides:  # two calls at once
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(call(ops, c))
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)
        graphs, outs = [], []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(call(ops, c))
            graphs.append(g)
        for _ in range(3):
            ids = torch.from_numpy(rng.integers(-1, 6, (T, 2)).astype(np.int32))
            c["ids"].copy_(ids)
            c["x"].copy_(torch.from_numpy(rng.standard_normal((T, 64)).astype(np.float32)))
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            want = call(ops, c)
            torch.cuda.synchronize()
            assert all(torch.equal(o, want) for o in outs)


def test_router_and_experts_together(lib, torch_cuda):
    """A layer's step: logits of a router product, routing, experts; masked experts and an unordered row on the way."""
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(9)
    T, E, d, h, k = 150, 16, 96, 160, 4
    c = draw_experts(torch, rng, T, k, E, d, h, "gated_silu", "bfloat16")
    logits = rng.standard_normal((T, E)).astype(np.float32)
    logits[3, 2:] = -np.inf   # two experts left
    logits[5] = np.nan
    logits[7] = -np.inf
    bias = (0.05 * rng.standard_normal(E)).astype(np.float32)
    kw = dict(score="sigmoid", groups=4, top_groups=2, group_top=2, scale=1.5)
    ids, weights = ops.route_topk(torch.from_numpy(logits).cuda(), k, bias=torch.from_numpy(bias).cuda(), **kw)
    y = ops.experts_topk(c["x"], ids, weights, c["wi"], c["wo"], c["wi_1"], ffn="gated_silu")
    want_ids, want_w = O.route_topk(logits, k, bias=bias, **kw)
    np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
    c["exact"].update(ids=want_ids, weights=weights.cpu().numpy())
    want, bound = O.experts_topk(**c["exact"])
    assert np.isnan(want[5]).all() and (want[7] == 0).all() and (want_ids[3, 2:] == -1).all()
    assert_within(y, want, bound)


def test_python_binding_refuses_what_does_not_fit(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    c = draw_experts(torch, np.random.default_rng(1), 4, 2, 3, 16, 24, "gated_silu", "float32")
    x, ids, w, wi, wo, w1 = c["x"], c["ids"], c["weights"], c["wi"], c["wo"], c["wi_1"]
    f = ops.experts_topk
    for bad in (lambda: f(x.double(), ids, w, wi, wo, w1, ffn="gated_silu"), lambda: f(x, ids.long(), w, wi, wo, w1, ffn="gated_silu"),
                lambda: f(x, ids, w.half(), wi, wo, w1, ffn="gated_silu"), lambda: f(x, ids, w, wi.half(), wo, w1, ffn="gated_silu"),
                lambda: f(x, ids, w, wi, wo, ffn="gated_silu"), lambda: f(x, ids, w, wi, wo, w1), lambda: f(x, ids, w, wi, wo.transpose(1, 2), w1, ffn="gated_silu"),
                lambda: f(x, ids, w, wi.cpu(), wo, w1, ffn="gated_silu"), lambda: f(x, ids, w, wi, wo[:2], w1, ffn="gated_silu"),
                lambda: f(x[:3], ids, w, wi, wo, w1, ffn="gated_silu"), lambda: f(x[:, :15], ids, w, wi, wo, w1, ffn="gated_silu"),
                lambda: f(x, ids, w[:, :1], wi, wo, w1, ffn="gated_silu"), lambda: f(x, ids, w, wi, wo, w1, ffn="swish"),
                lambda: f(x, ids, w, wi, wo, w1, ffn="gated_silu", out=torch.zeros(4, 17, device="cuda")), lambda: f(x.cpu(), ids, w, wi, wo, w1, ffn="gated_silu")):
        with pytest.raises(capi.InfMoEError) as ei:
            bad()
        assert ei.value.status == capi.ERR_INVALID_ARGUMENT
