"""infmoe_lora_project in every form it can take (operator_shapes.py): every value within the bound of its roundings, what one
adapter or row holds kept out of the others, nothing written around y, a call repeated bit for bit."""
import numpy as np
import pytest

from oracle import topk_oracle as O
from tests import operator_exact
from tests import operator_shapes as shapes
from tests.topk_util import assert_within

pytestmark = pytest.mark.gpu
L = 5


def draw(torch, T, d, n, r, dtype, order, shift=()):
    """Tensors on the GPU; those named in `shift` start one element behind a 16-byte boundary."""
    g = torch.Generator(device="cuda").manual_seed(T + d + n + r)

    def normal(name, *shape, std=1.0):
        flat = torch.empty(int(np.prod(shape)) + 1, dtype=getattr(torch, dtype), device="cuda").normal_(0.0, std, generator=g)
        return flat[1:].view(shape) if name in shift else flat[:-1].view(shape)

    c = dict(x=normal("x", T, d), w=normal("w", n, d, std=d ** -0.5), a=normal("a", L, r, d, std=d ** -0.5), b=normal("b", L, n, r, std=r ** -0.5))
    c["adapter"] = torch.randint(-1, L + 1, (T,), device="cuda", generator=g, dtype=torch.int32)  # (L: none, like -1)
    if order == "requests":  # rows of a request side by side, of about 40 rows each
        c["adapter"] = c["adapter"][:T // 40 + 1].repeat_interleave(40)[:T].contiguous()
    c["scale"] = torch.rand(L, device="cuda", generator=g) + 0.5
    return c


def call(ops, c, **kw):
    return ops.lora_project(c["x"], c["w"], c["a"], c["b"], c["adapter"], c["scale"], **kw)


def check(torch, ops, T, d, n, r, dtype, order, shift=()):
    print(f"lora T={T} d={d} n={n} r={r} {dtype} {order} {shift}", flush=True)
    c = draw(torch, T, d, n, r, dtype, order, shift)
    # given output: rows apart and on no boundary, or whole pieces
    pad = 13 if order == "any" else 16
    big = torch.full((T + 2, (n + 7) // 8 * 8 + pad), 3.0, dtype=c["x"].dtype, device="cuda")
    out = big[1:T + 1, pad - 8:pad - 8 + n]
    y = call(ops, c, out=out).clone()
    out.fill_(3.0)
    assert (big == 3.0).all()
    operator_exact.assert_within(y, *operator_exact.lora_project(torch, **c, dtype=dtype), what=dtype)
    rows = np.unique(np.concatenate([[0, T - 1], np.random.default_rng(T).integers(0, T, 30)]))  # the same by numpy
    at = torch.from_numpy(rows).cuda()
    exact = {k: v.double().cpu().numpy() for k, v in c.items() if k not in ("x", "adapter")}
    assert_within(y[at], *O.lora_project(x=c["x"][at].double().cpu().numpy(), adapter=c["adapter"][at].cpu().numpy(), dtype=dtype, **exact), what=dtype)
    assert torch.equal(call(ops, c), y)
    c["b"][2] = float("nan")
    c["a"][3, 0, 0] = float("inf")
    none = (c["adapter"] < 0) | (c["adapter"] >= L)
    c["x"][none] = float("nan")
    again = call(ops, c)
    fine = ~none & (c["adapter"] != 2) & (c["adapter"] != 3)
    assert torch.equal(again[fine], y[fine])
    assert again[none].isnan().all() and again[c["adapter"] == 2].isnan().all() and not again[c["adapter"] == 3].isfinite().all(dim=1).any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("order", ["any", "requests"])
@pytest.mark.parametrize("i", range(len(shapes.LORA[2])))
def test_rows_of_whole_pieces(lib, torch_cuda, i, order, dtype):
    from infmoe_amd import ops
    check(torch_cuda, ops, *shapes.LORA[4 if dtype == "float32" else 2][i], dtype, order)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("order", ["any", "requests"])
@pytest.mark.parametrize("shape", shapes.LORA_ODD)
def test_rows_that_are_not(lib, torch_cuda, shape, order, dtype):
    from infmoe_amd import ops
    check(torch_cuda, ops, *shape, dtype, order)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("shift", ["x", "w", "a", "b"])
@pytest.mark.parametrize("T,d,n,r", [(3, 64, 80, 8), (70, 712, 264, 16), (1100, 72, 2304, 8)])
def test_operands_off_a_boundary(lib, torch_cuda, T, d, n, r, shift, dtype):
    """Row lengths of whole pieces, one operand that starts off a 16-byte boundary."""
    from infmoe_amd import ops
    check(torch_cuda, ops, T, d, n, r, dtype, "any", (shift,))
