"""infmoe_experts_topk in every form it can take (operator_shapes.py): every value within the bound of its roundings, a call
repeated bit for bit."""
import numpy as np
import pytest

from oracle import topk_oracle as O
from tests import operator_exact
from tests import operator_shapes as shapes
from tests.topk_util import assert_within

pytestmark = pytest.mark.gpu


def check(torch, T, k, E, d, h, ffn, dtype, counts=None):
    from infmoe_amd import ops
    print(f"experts T={T} k={k} E={E} d={d} h={h} {ffn} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(T + E + d + h)
    normal = lambda *shape, std=1.0: torch.empty(shape, dtype=getattr(torch, dtype), device="cuda").normal_(0.0, std, generator=g)
    x, wi, wo = normal(T, d), normal(E, h, d, std=d ** -0.5), normal(E, d, h, std=h ** -0.5)
    wi_1 = normal(E, h, d, std=d ** -0.5) if ffn != "relu" else None
    weights = torch.rand(T, k, device="cuda", generator=g)
    rng = np.random.default_rng(T)
    if counts is None:
        ids = rng.integers(-1, E, (T, k)).astype(np.int32)
        ids[rng.random((T, k)) < 0.2] = E // 2  # one expert with more rows than the others
    else:  # so many slots per expert, the rest without one
        ids = np.full(T * k, -1, np.int32)
        ids[rng.permutation(T * k)[:sum(counts)]] = np.repeat(np.arange(E), counts)
        ids = ids.reshape(T, k)
    there = torch.from_numpy(ids).cuda()
    y = ops.experts_topk(x, there, weights, wi, wo, wi_1, ffn=ffn)
    operator_exact.assert_within(y, *operator_exact.experts_topk(torch, x, there, weights, wi, wo, wi_1, ffn, dtype), what=f"{dtype} {ffn}")
    rows = np.unique(np.concatenate([[0, T - 1], rng.integers(0, T, 8)]))  # the same by numpy
    at = torch.from_numpy(rows).cuda()
    wide = lambda t: None if t is None else t.double().cpu().numpy()
    assert_within(y[at], *O.experts_topk(wide(x[at]), ids[rows], wide(weights[at]), wide(wi), wide(wo), wide(wi_1), ffn=ffn, dtype=dtype), what=f"{dtype} {ffn}")
    assert torch.equal(ops.experts_topk(x, there, weights, wi, wo, wi_1, ffn=ffn), y)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("ffn", ["relu", "gated_silu"])
@pytest.mark.parametrize("shape", shapes.EXPERTS + shapes.EXPERTS_ODD)
def test_every_form(lib, torch_cuda, shape, ffn, dtype):
    check(torch_cuda, *shape, ffn, dtype)


@pytest.mark.parametrize("dtype,ffn", [("float32", "gated_gelu"), ("bfloat16", "relu"), ("bfloat16", "gated_gelu"), ("float16", "gated_silu")])
def test_tall_tiles_of_every_height(lib, torch_cuda, dtype, ffn):
    """Experts whose rows are one tile of 1 to 8 blocks of 32, or several of equal heights."""
    counts = [0, 1, 32, 33, 64, 65, 96, 97, 128, 150, 161, 200, 224, 255, 256, 257, 300, 385, 512, 513]
    check(torch_cuda, 1500, 3, len(counts), 2056, 2064, ffn, dtype, counts)
