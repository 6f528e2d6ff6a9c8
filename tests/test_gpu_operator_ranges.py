"""Values at the ends of a type's range between the two products: what include/infmoe.h says of float16, and that bfloat16 and
float32 have none of it."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [3, 40, 300])
@pytest.mark.parametrize("dtype,held", [("float32", True), ("bfloat16", True), ("float16", False)])
def test_hidden_values_beyond_float16(lib, torch_cuda, T, dtype, held):
    """u = 64 * 32 * 64 = 131072 in every hidden value; y = 64 u / 65536 = 128, exact in every type and sum."""
    torch = torch_cuda
    from infmoe_amd import ops
    full = lambda value, *shape: torch.full(shape, value, dtype=getattr(torch, dtype), device="cuda")
    ids = torch.arange(T, device="cuda", dtype=torch.int32)[:, None] % 2
    y = ops.experts_topk(full(32.0, T, 64), ids, torch.ones(T, 1, device="cuda"), full(64.0, 2, 64, 64), full(2.0 ** -16, 2, 64, 64))
    assert (y == (128.0 if held else float("inf"))).all()


@pytest.mark.parametrize("T", [3, 40, 300])
@pytest.mark.parametrize("dtype,held", [("float32", True), ("bfloat16", True), ("float16", False)])
def test_adapters_first_product_beyond_float16(lib, torch_cuda, T, dtype, held):
    """scale a x = 2 * 64 * 16 * 64 = 131072 in 8 ranks; b = 2^-14: 64 a row.  Rows without an adapter stay at w x = 0."""
    torch = torch_cuda
    from infmoe_amd import ops
    full = lambda value, *shape: torch.full(shape, value, dtype=getattr(torch, dtype), device="cuda")
    adapter = torch.arange(T, device="cuda", dtype=torch.int32) % 2 - 1
    y = ops.lora_project(full(16.0, T, 64), full(0.0, 80, 64), full(64.0, 1, 8, 64), full(2.0 ** -14, 1, 80, 8), adapter, torch.full((1,), 2.0, device="cuda"))
    assert (y[adapter == 0] == (64.0 if held else float("inf"))).all() and (y[adapter < 0] == 0).all()
