"""infmoe_lora_project on more rows than one launch has work items for."""
import numpy as np
import pytest

from oracle import topk_oracle as O
from tests.topk_util import draw_lora

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,d,n,r,dtype", [((1 << 31) - 1, 1, 1, 1, "float16"), ((1 << 26) + 77, 8, 8, 8, "bfloat16"), ((1 << 27) + 77, 3, 5, 2, "float16")])
def test_more_rows_than_one_launch_has_work_items_for(lib, torch_cuda, T, d, n, r, dtype):
    """Every row is one of 1000, with one of three adapters or none, so that the whole result is known from 4000 rows."""
    torch = torch_cuda
    from infmoe_amd import ops
    L, step = 3, 1 << 24
    c = draw_lora(torch, np.random.default_rng(d), 1000, d, n, r, L, dtype, "any")
    want, bound = np.zeros((L + 1, 1000, n)), np.zeros((L + 1, 1000, n))
    for a in range(L + 1):
        want[a], bound[a] = O.lora_project(**dict(c["exact"], adapter=np.full(1000, a)))
    want, bound = torch.from_numpy(want).cuda(), torch.from_numpy(bound).cuda()
    row = lambda at: torch.arange(at, min(at + step, T), device="cuda") * 7 % 1000
    of = lambda at: (torch.arange(at, min(at + step, T), device="cuda") // 13 * 5 % 7).clamp(max=L)  # (L: none)
    x, adapter = torch.empty(T, d, dtype=c["x"].dtype, device="cuda"), torch.empty(T, dtype=torch.int32, device="cuda")
    for at in range(0, T, step):
        x[at:at + step], adapter[at:at + step] = c["x"][row(at)], of(at)
    y = ops.lora_project(x, c["w"], c["a"], c["b"], adapter, c["scale"])
    for at in range(0, T, step):
        places = (of(at), row(at))
        assert ((y[at:at + step].double() - want[places]).abs() <= bound[places]).all()
