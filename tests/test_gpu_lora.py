"""infmoe_lora_project against the float64 oracle, every value within the bound of its roundings."""
import numpy as np
import pytest

from infmoe_amd import capi
from oracle import topk_oracle as O
from tests.topk_util import DTYPES, assert_within, draw_lora

pytestmark = pytest.mark.gpu


def call(ops, c, **kw):
    return ops.lora_project(c["x"], c["w"], c["a"], c["b"], c["adapter"], c["scale"], **kw)


SHAPES = [  # T, d, n, r, L
    (1, 8, 8, 1, 1), (1, 64, 96, 16, 4), (1, 1024, 520, 8, 2), (2, 512, 256, 64, 3), (7, 40, 24, 3, 2), (16, 96, 160, 8, 30), (17, 128, 64, 4, 3),
    (64, 256, 512, 16, 64), (130, 72, 200, 8, 5), (300, 128, 64, 64, 3), (33, 13, 29, 5, 4), (3, 131, 77, 7, 2), (200, 64, 300, 256, 3),
    (513, 100, 130, 12, 9), (1, 1, 1, 1, 1), (1000, 264, 520, 32, 4), (260, 136, 272, 100, 40),
]


@pytest.mark.parametrize("T,d,n,r,L", SHAPES)
@pytest.mark.parametrize("order", ["any", "requests"])
def test_lora_matches_oracle(lib, torch_cuda, T, d, n, r, L, order):
    from infmoe_amd import ops
    for dtype in DTYPES:
        print(f"lora T={T} d={d} n={n} r={r} L={L} {order} {dtype}", flush=True)
        c = draw_lora(torch_cuda, np.random.default_rng(T + d + r), T, d, n, r, L, dtype, order)
        assert_within(call(ops, c), *O.lora_project(**c["exact"]), what=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 9, 64, 200])
def test_lora_at_long_rows(lib, torch_cuda, dtype, T):
    from infmoe_amd import ops
    c = draw_lora(torch_cuda, np.random.default_rng(T), T, 4096, 1040, 16, 70, dtype, "any")
    assert_within(call(ops, c), *O.lora_project(**c["exact"]), what=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,d,n,r,L", [(3000, 64, 4500, 16, 5), (1500, 72, 2300, 12, 3), (100, 2048, 520, 16, 5), (30, 4096, 260, 20, 9), (240, 1032, 776, 8, 4)])
@pytest.mark.parametrize("order", ["any", "requests"])
def test_lora_on_tall_tiles(lib, torch_cuda, dtype, T, d, n, r, L, order):
    """Tiles of 256 and of 128 rows, and tiles whose K is cut over workgroups (two, four and eight blocks of rows)."""
    from infmoe_amd import ops
    c = draw_lora(torch_cuda, np.random.default_rng(T + n), T, d, n, r, L, dtype, order)
    assert_within(call(ops, c), *O.lora_project(**c["exact"]), what=dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [3, 20, 150])
def test_one_adapter_cannot_reach_the_rows_of_another(lib, torch_cuda, dtype, T):
    torch = torch_cuda
    from infmoe_amd import ops
    c = draw_lora(torch, np.random.default_rng(2), T, 64, 96, 8, 4, dtype, "any")
    c["adapter"][:] = torch.arange(T, dtype=torch.int32, device="cuda") % 5 - 1
    clean = call(ops, c)
    c["a"][1, 3, 5] = float("nan")
    c["b"][2, 7, 1] = float("inf")
    c["b"][3] = float("nan")
    y = call(ops, c)
    fine = (c["adapter"] <= 0).nonzero()[:, 0]  # (none, or adapter 0)
    assert torch.equal(y[fine], clean[fine])
    assert all(not y[t].isfinite().all() for t in range(T) if int(c["adapter"][t]) > 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,n", [(3000, 4500), (1500, 2300), (90, 264)])
def test_one_adapter_cannot_reach_the_rows_of_another_on_tall_tiles(lib, torch_cuda, dtype, T, n):
    torch = torch_cuda
    from infmoe_amd import ops
    d = 2048 if T < 100 else 64
    c = draw_lora(torch, np.random.default_rng(2), T, d, n, 8, 4, dtype, "any")
    c["adapter"][:] = torch.arange(T, dtype=torch.int32, device="cuda") % 5 - 1
    clean = call(ops, c)
    c["b"][2, 7, 1] = float("inf")
    c["b"][3] = float("nan")
    c["x"][0] = float("nan")  # (a row without an adapter)
    y = call(ops, c)
    fine = ((c["adapter"] >= 0) & (c["adapter"] <= 1)).nonzero()[:, 0]
    assert torch.equal(y[fine], clean[fine])
    assert y[0].isnan().all() and y[3::5].isfinite().all(dim=1).sum() == 0 and y[4::5].isnan().all()


def test_no_adapter_anywhere_no_scale_and_padding_rows(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    for T in (1, 30, 300):
        c = draw_lora(torch, np.random.default_rng(3), T, 72, 56, 6, 3, "float32", "any")
        c["exact"]["scale"] = None
        assert_within(ops.lora_project(c["x"], c["w"], c["a"], c["b"], c["adapter"]), *O.lora_project(**c["exact"]))
        c["adapter"].fill_(-1)
        c["exact"]["adapter"] = np.full(T, -1)
        c["a"].fill_(float("nan"))
        assert_within(call(ops, c), *O.lora_project(**c["exact"]))
        c["x"][T // 2] = float("nan")  # a padding row's contents stay in it
        y = call(ops, c)
        assert y[T // 2].isnan().all() and int(y.isnan().any(dim=1).sum()) == 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [5, 70])
def test_strided_rows_and_guards(lib, torch_cuda, dtype, T):
    torch = torch_cuda
    from infmoe_amd import ops
    for d, n, at in ((64, 96, 8), (50, 71, 3)):
        c = draw_lora(torch, np.random.default_rng(4), T, d, n, 8, 5, dtype, "any")
        big_x = torch.full((T, d + 24), float("nan"), dtype=c["x"].dtype, device="cuda")
        big_x[:, at:at + d] = c["x"]
        c["x"] = big_x[:, at:at + d]
        big_y = torch.full((T + 2, n + 13), 3.0, dtype=c["w"].dtype, device="cuda")
        y = big_y[1:T + 1, 5:5 + n]
        call(ops, c, out=y)
        assert_within(y, *O.lora_project(**c["exact"]))
        big_y[1:T + 1, 5:5 + n] = 3.0
        assert (big_y == 3.0).all()


def test_adapters_beyond_32_bit_offsets(lib, torch_cuda):
    """A store of adapters of more than 2^31 elements; the first and the last are used."""
    torch = torch_cuda
    from infmoe_amd import ops
    T, d, n, r = 6, 2048, 64, 256
    L = (1 << 31) // (r * d) + 2
    rng = np.random.default_rng(5)
    c = draw_lora(torch, rng, T, d, n, r, 2, "float16", "any")
    a = torch.zeros(L, r, d, dtype=torch.float16, device="cuda")
    b = torch.zeros(L, n, r, dtype=torch.float16, device="cuda")
    a[0], a[-1], b[0], b[-1] = c["a"][0], c["a"][1], c["b"][0], c["b"][1]
    small = np.array([0, 1, 1, 0, -1, 1])
    c["exact"].update(adapter=small, scale=None)
    big = torch.from_numpy(np.where(small == 1, L - 1, small).astype(np.int32)).cuda()
    assert_within(ops.lora_project(c["x"], c["w"], a, b, big), *O.lora_project(**c["exact"]))


def test_empty_batch_streams_and_graphs(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    rng = np.random.default_rng(8)
    for T, dtype in ((4, "bfloat16"), (90, "float32"), (600, "float16")):
        c = draw_lora(torch, rng, T, 64, 128, 16, 6, dtype, "any")
        assert ops.lora_project(c["x"][:0], c["w"], c["a"], c["b"], c["adapter"][:0], c["scale"]).shape == (0, 128)
        want = call(ops, c)
        sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
        for s in sides:
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
            c["adapter"].copy_(torch.from_numpy(rng.integers(-1, 6, T).astype(np.int32)))
            c["x"].copy_(torch.from_numpy(rng.standard_normal((T, 64)).astype(np.float32)))
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            want = call(ops, c)
            torch.cuda.synchronize()
            assert all(torch.equal(o, want) for o in outs)


def test_python_binding_refuses_what_does_not_fit(lib, torch_cuda):
    torch = torch_cuda
    from infmoe_amd import ops
    c = draw_lora(torch, np.random.default_rng(1), 4, 16, 24, 4, 3, "float32", "any")
    x, w, a, b, i, s = c["x"], c["w"], c["a"], c["b"], c["adapter"], c["scale"]
    f = ops.lora_project
    for bad in (lambda: f(x.double(), w, a, b, i, s), lambda: f(x, w.half(), a, b, i, s), lambda: f(x, w.t(), a, b, i, s), lambda: f(x, w, a[:2], b, i, s),
                lambda: f(x, w, a, b[:, :, :3], i, s), lambda: f(x, w, a.transpose(1, 2), b, i, s), lambda: f(x, w, a, b, i.long(), s),
                lambda: f(x, w, a, b, i[:3], s), lambda: f(x, w, a, b, i, s[:2]), lambda: f(x, w, a, b, i, s.cpu()), lambda: f(x, w, a[:0], b[:0], i, s[:0]),
                lambda: f(x, w, a, b, i, s, out=torch.zeros(4, 25, device="cuda")), lambda: f(x[0], w, a, b, i, s)):
        with pytest.raises(capi.InfMoEError) as ei:
            bad()
        assert ei.value.status == capi.ERR_INVALID_ARGUMENT
